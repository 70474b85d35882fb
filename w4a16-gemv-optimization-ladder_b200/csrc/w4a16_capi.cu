// extern "C" entry points of libw4a16_b200.so (declared in include/w4a16_b200.h).
// Host-side validation happens here, before anything is launched: a bad pointer,
// shape, alignment or dtype code returns a status and launches nothing.
#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

#include <atomic>
#include <mutex>
#include <unordered_map>

#include "w4a16_b200.h"
#include "w4a16_internal.h"

namespace {

using w4a16::set_error;

constexpr int kVersion = 1 * 10000 + 0 * 100 + 0;

bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

// Tensor-parallel regions known to this process (created by w4a16_tp_region_alloc or
// mapped by w4a16_tp_region_open), with the byte capacity of each one's gathered output.
// The fused all-gather stores every rank's rows into every region, so a call whose rows
// do not fit one of them is rejected before launch.  The capacity also sits in the
// region's header (kTpCapacityOffset), where the opening process reads it.
std::mutex g_region_mu;
std::unordered_map<uintptr_t, size_t> g_region_capacity;

void register_region(void* region, size_t out_bytes) {
  std::lock_guard<std::mutex> lock(g_region_mu);
  g_region_capacity[reinterpret_cast<uintptr_t>(region)] = out_bytes;
}

void forget_region(void* region) {
  std::lock_guard<std::mutex> lock(g_region_mu);
  g_region_capacity.erase(reinterpret_cast<uintptr_t>(region));
}

bool region_capacity(const void* region, size_t* out_bytes) {
  std::lock_guard<std::mutex> lock(g_region_mu);
  const auto it = g_region_capacity.find(reinterpret_cast<uintptr_t>(region));
  if (it == g_region_capacity.end()) return false;
  *out_bytes = it->second;
  return true;
}

// Limit of the fused all-gather's waits on other GPUs (0 = the 2 s default).
std::atomic<unsigned long long> g_peer_wait_ns{0};
constexpr unsigned long long kDefaultPeerWaitNs = 2000000000ull;

// Shape / pointer checks shared by every GEMV-style entry point.
int check_gemv(const void* packed, int packing, const void* scale, int scale_dtype, int group,
               const void* x, int batch, int rows, int cols, const void* out, int out_dtype) {
  if (packing != W4A16_PACK_INTERLEAVED && packing != W4A16_PACK_SIMPLE) {
    set_error("unknown packing code %d", packing);
    return W4A16_ERR_DTYPE;
  }
  if ((scale_dtype != W4A16_DTYPE_F32 && scale_dtype != W4A16_DTYPE_F16) ||
      (out_dtype != W4A16_DTYPE_F32 && out_dtype != W4A16_DTYPE_F16)) {
    set_error("unknown dtype code (scale %d, out %d)", scale_dtype, out_dtype);
    return W4A16_ERR_DTYPE;
  }
  if (group != 0 && group != 128) {
    set_error("group must be 0 (per-row) or 128, got %d", group);
    return W4A16_ERR_DTYPE;
  }
  if (rows < 0 || cols <= 0 || batch < 0) {
    set_error("bad shape rows=%d cols=%d batch=%d", rows, cols, batch);
    return W4A16_ERR_SHAPE;
  }
  if (cols % 8 != 0 || (group && cols % group != 0)) {
    set_error("cols=%d must be a multiple of %d", cols, group ? group : 8);
    return W4A16_ERR_SHAPE;
  }
  if (rows == 0 || batch == 0) return W4A16_OK;
  if (!packed || !scale || !x || !out) {
    set_error("NULL pointer (packed %p, scale %p, x %p, out %p)", packed, scale, x, out);
    return W4A16_ERR_NULL;
  }
  const size_t ssz = scale_dtype == W4A16_DTYPE_F32 ? 4 : 2;
  const size_t osz = out_dtype == W4A16_DTYPE_F32 ? 4 : 2;
  if (!aligned(packed, 4) || !aligned(x, 16) || !aligned(scale, ssz) || !aligned(out, osz)) {
    set_error("misaligned pointer: packed needs 4 B, x 16 B, scale %zu B, out %zu B", ssz, osz);
    return W4A16_ERR_ALIGN;
  }
  return W4A16_OK;
}

int gemv_common(const uint8_t* packed, int packing, const void* scale, int scale_dtype, int group,
                const void* x, int batch, int rows, int cols, void* out, int out_dtype,
                const float* bias, void* workspace, size_t workspace_bytes,
                w4a16_stream_t stream) {
  int rc = check_gemv(packed, packing, scale, scale_dtype, group, x, batch, rows, cols, out,
                      out_dtype);
  if (rc != W4A16_OK || rows == 0 || batch == 0) return rc;
  if (bias && !aligned(bias, 4)) {
    set_error("bias must be 4-byte aligned");
    return W4A16_ERR_ALIGN;
  }
  w4a16::GemvProblem p;
  p.packed = packed;
  p.packing = packing;
  p.scale = scale;
  p.scale_dtype = scale_dtype;
  p.group = group;
  p.x = x;
  p.M = batch;
  p.N = rows;
  p.K = cols;
  p.y = out;
  p.out_dtype = out_dtype;
  p.bias = bias;
  p.workspace = workspace;
  p.workspace_bytes = workspace ? workspace_bytes : 0;
  p.split_k = 0;
  p.stream = reinterpret_cast<cudaStream_t>(stream);
  return w4a16::launch_gemv(p);
}

int ladder(const uint8_t* packed, const float* scale, const void* vec, float* out, int rows,
           int cols, w4a16_stream_t stream) {
  return gemv_common(packed, W4A16_PACK_SIMPLE, scale, W4A16_DTYPE_F32, 0, vec, 1, rows, cols, out,
                     W4A16_DTYPE_F32, nullptr, nullptr, 0, stream);
}

// ---- paged cache: shared checks ----

int check_pool(const w4a16_page_pool* p, w4a16::PagedPool* out) {
  if (!p || !p->k || !p->v) {
    set_error("null page pool");
    return W4A16_ERR_NULL;
  }
  if (p->dtype != W4A16_DTYPE_F16 && p->dtype != W4A16_DTYPE_BF16) {
    set_error("page pool dtype code %d is not fp16 or bf16", p->dtype);
    return W4A16_ERR_DTYPE;
  }
  if (p->pages <= 0 || p->kv_heads <= 0 || p->page_size <= 0 || p->page_size > 4096 ||
      (p->page_size & (p->page_size - 1)) != 0 ||
      (p->head_dim != 64 && p->head_dim != 128 && p->head_dim != 256)) {
    set_error("unsupported page pool: pages %d kv_heads %d page_size %d head_dim %d (page_size a power of "
              "two up to 4096, head_dim 64, 128 or 256)", p->pages, p->kv_heads, p->page_size, p->head_dim);
    return W4A16_ERR_SHAPE;
  }
  if (p->page_stride <= 0 || p->head_stride <= 0 || p->token_stride <= 0 || p->page_stride % 8 ||
      p->head_stride % 8 || p->token_stride % 8 || !aligned(p->k, 16) || !aligned(p->v, 16)) {
    set_error("page pool strides must be positive multiples of 8 elements (page %lld head %lld token %lld), k and v "
              "16-byte aligned", p->page_stride, p->head_stride, p->token_stride);
    return W4A16_ERR_ALIGN;
  }
  out->k = p->k;
  out->v = p->v;
  out->dtype = p->dtype;
  out->pages = p->pages;
  out->kv_heads = p->kv_heads;
  out->head_dim = p->head_dim;
  out->page_shift = __builtin_ctz((unsigned)p->page_size);
  out->page_stride = p->page_stride;
  out->head_stride = p->head_stride;
  out->token_stride = p->token_stride;
  return W4A16_OK;
}

int check_tables(const w4a16_page_tables* t, w4a16::PagedTables* out) {
  if (!t || !t->ids) {
    set_error("null page tables");
    return W4A16_ERR_NULL;
  }
  if (t->sequences <= 0 || t->width <= 0 || t->stride < 0) {
    set_error("bad page tables: %d sequences, width %d, stride %lld", t->sequences, t->width, t->stride);
    return W4A16_ERR_SHAPE;
  }
  if (!aligned(t->ids, 4)) {
    set_error("page tables must be 4-byte aligned");
    return W4A16_ERR_ALIGN;
  }
  out->ids = t->ids;
  out->rows = t->sequences;
  out->width = t->width;
  out->stride = t->stride;
  return W4A16_OK;
}

int check_state(const w4a16_page_state* s, w4a16::PagesState* out) {
  if (!s || !s->tables || !s->lengths || !s->refs) {
    set_error("null page state");
    return W4A16_ERR_NULL;
  }
  if (s->sequences <= 0 || s->width <= 0 || s->pages <= 0 || s->page_size <= 0 || s->page_size > 4096 ||
      (s->page_size & (s->page_size - 1)) != 0 || s->table_stride < s->width || (long long)s->width * s->page_size > (1 << 30)) {
    set_error("bad page state: %d sequences, width %d, stride %lld, %d pages of %d (page_size a power of two up to 4096, at "
              "most 2^30 positions a row)",
              s->sequences, s->width, s->table_stride, s->pages, s->page_size);
    return W4A16_ERR_SHAPE;
  }
  if (!aligned(s->tables, 4) || !aligned(s->lengths, 4) || !aligned(s->refs, 4)) {
    set_error("page state must be 4-byte aligned");
    return W4A16_ERR_ALIGN;
  }
  out->tables = s->tables;
  out->lengths = s->lengths;
  out->refs = s->refs;
  out->sequences = s->sequences;
  out->width = s->width;
  out->pages = s->pages;
  out->page_shift = __builtin_ctz((unsigned)s->page_size);
  out->table_stride = s->table_stride;
  return W4A16_OK;
}

int check_blocks(const w4a16_page_blocks* b, w4a16::PageBlocks* out) {
  if (!b || !b->k || !b->v) {
    set_error("null page blocks");
    return W4A16_ERR_NULL;
  }
  if (b->layers <= 0 || b->pages <= 0 || b->page_bytes <= 0 || b->page_bytes > (1 << 30) || b->page_stride < b->page_bytes || b->layer_stride < 0) {
    set_error("bad page blocks: %d layers of %d pages, layer stride %lld, page stride %lld, %lld bytes a page", b->layers,
              b->pages, b->layer_stride, b->page_stride, b->page_bytes);
    return W4A16_ERR_SHAPE;
  }
  if (!aligned(b->k, 16) || !aligned(b->v, 16) || b->page_bytes % 16 || b->page_stride % 16 || b->layer_stride % 16) {
    set_error("page blocks must be 16-byte aligned, sizes and strides multiples of 16");
    return W4A16_ERR_ALIGN;
  }
  out->k = b->k;
  out->v = b->v;
  out->layers = b->layers;
  out->pages = b->pages;
  out->layer_stride = b->layer_stride;
  out->page_stride = b->page_stride;
  out->page_bytes = b->page_bytes;
  return W4A16_OK;
}

// n requests with their lists: 0 is a no-op for the caller to return.
int check_requests(int n, int most, const void* a, const void* b, const void* ok) {
  if (n < 0 || n > most) {
    set_error("%d requests (0..%d in one call)", n, most);
    return W4A16_ERR_SHAPE;
  }
  if (n == 0) return W4A16_OK;
  if (!a || !b || !ok) {
    set_error("null pointer argument");
    return W4A16_ERR_NULL;
  }
  if (!aligned(a, 4) || !aligned(b, 4) || !aligned(ok, 4)) {
    set_error("request lists must be 4-byte aligned");
    return W4A16_ERR_ALIGN;
  }
  return W4A16_OK;
}

int check_scratch(const void* scratch, size_t bytes, size_t need) {
  if (need == 0) return W4A16_OK;
  if (!scratch) {
    set_error("null scratch");
    return W4A16_ERR_NULL;
  }
  if (!aligned(scratch, 16)) {
    set_error("scratch must be 16-byte aligned");
    return W4A16_ERR_ALIGN;
  }
  if (bytes < need) {
    set_error("scratch of %zu bytes is smaller than the %zu needed", bytes, need);
    return W4A16_ERR_WORKSPACE;
  }
  return W4A16_OK;
}

}  // namespace

extern "C" {

int w4a16_marlin_cuda(const uint8_t* packed, const float* scale, const void* vec, float* out,
                      int rows, int cols, w4a16_stream_t stream) {
  return gemv_common(packed, W4A16_PACK_INTERLEAVED, scale, W4A16_DTYPE_F32, 0, vec, 1, rows, cols,
                     out, W4A16_DTYPE_F32, nullptr, nullptr, 0, stream);
}

int w4a16_marlin_g128_cuda(const uint8_t* packed, const float* scale, const void* vec,
                           float* out, int rows, int cols, w4a16_stream_t stream) {
  return gemv_common(packed, W4A16_PACK_INTERLEAVED, scale, W4A16_DTYPE_F32, 128, vec, 1, rows,
                     cols, out, W4A16_DTYPE_F32, nullptr, nullptr, 0, stream);
}

int w4a16_byte_cuda(const uint8_t* packed, const float* scale, const void* vec, float* out,
                    int rows, int cols, w4a16_stream_t stream) {
  return ladder(packed, scale, vec, out, rows, cols, stream);
}

int w4a16_u32_cuda(const uint8_t* packed, const float* scale, const void* vec, float* out,
                   int rows, int cols, w4a16_stream_t stream) {
  return ladder(packed, scale, vec, out, rows, cols, stream);
}

int w4a16_u32_v4_cuda(const uint8_t* packed, const float* scale, const void* vec, float* out,
                      int rows, int cols, w4a16_stream_t stream) {
  return ladder(packed, scale, vec, out, rows, cols, stream);
}

int w4a16_champ_cuda(const uint8_t* packed, const float* scale, const void* vec, float* out,
                     int rows, int cols, w4a16_stream_t stream) {
  return ladder(packed, scale, vec, out, rows, cols, stream);
}

int w4a16_uint4_cuda(const uint8_t* packed, const float* scale, const void* vec, float* out,
                     int rows, int cols, w4a16_stream_t stream) {
  return ladder(packed, scale, vec, out, rows, cols, stream);
}

int w4a16_h2f32_cuda(const uint8_t* packed, const float* scale, const void* vec, float* out,
                     int rows, int cols, w4a16_stream_t stream) {
  int rc = check_gemv(packed, W4A16_PACK_SIMPLE, scale, W4A16_DTYPE_F32, 0, vec, 1, rows, cols,
                      out, W4A16_DTYPE_F32);
  if (rc != W4A16_OK || rows == 0) return rc;
  return w4a16::launch_h2f32(packed, scale, vec, out, rows, cols,
                             reinterpret_cast<cudaStream_t>(stream));
}

int w4a16_fp16_cuda(const void* mat, const void* vec, float* out, int rows, int cols,
                    w4a16_stream_t stream) {
  if (rows < 0 || cols <= 0 || cols % 8 != 0) {
    set_error("bad shape rows=%d cols=%d (cols must be a positive multiple of 8)", rows, cols);
    return W4A16_ERR_SHAPE;
  }
  if (rows == 0) return W4A16_OK;
  if (!mat || !vec || !out) {
    set_error("NULL pointer");
    return W4A16_ERR_NULL;
  }
  if (!aligned(mat, 16) || !aligned(vec, 16) || !aligned(out, 4)) {
    set_error("mat and vec must be 16-byte aligned, out 4-byte aligned");
    return W4A16_ERR_ALIGN;
  }
  return w4a16::launch_fp16_gemv(mat, vec, out, rows, cols, reinterpret_cast<cudaStream_t>(stream));
}

int w4a16_gemv(const uint8_t* packed, int packing, const void* scale, int scale_dtype, int group,
               const void* x, int batch, int rows, int cols, void* out, int out_dtype,
               const float* bias, void* workspace, size_t workspace_bytes,
               w4a16_stream_t stream) {
  return gemv_common(packed, packing, scale, scale_dtype, group, x, batch, rows, cols, out,
                     out_dtype, bias, workspace, workspace_bytes, stream);
}

int w4a16_gemv_fused(const uint8_t* packed, const void* scale, int scale_dtype, int group,
                     int prologue, const void* src, const float* gamma, float eps, int rows,
                     int cols, void* out, int out_dtype, const float* bias, void* workspace,
                     size_t workspace_bytes, unsigned flags, w4a16_stream_t stream) {
  if (prologue != W4A16_PROLOGUE_NONE && prologue != W4A16_PROLOGUE_RMSNORM &&
      prologue != W4A16_PROLOGUE_SWIGLU) {
    set_error("unknown prologue code %d", prologue);
    return W4A16_ERR_DTYPE;
  }
  if (flags & ~(unsigned)(W4A16_LAUNCH_PDL | W4A16_LAUNCH_SWIGLU_OUT)) {
    set_error("unknown launch flags 0x%x", flags);
    return W4A16_ERR_DTYPE;
  }
  const bool swiglu_out = (flags & W4A16_LAUNCH_SWIGLU_OUT) != 0;
  if (swiglu_out && (prologue != W4A16_PROLOGUE_RMSNORM || bias || rows % 16 != 0)) {
    set_error("W4A16_LAUNCH_SWIGLU_OUT needs the RMSNorm prologue, no bias and rows %% 16 == 0 (got %d)",
              rows);
    return W4A16_ERR_SHAPE;
  }
  // src stands in for x in the shared checks (16-byte alignment, non-NULL)
  int rc = check_gemv(packed, W4A16_PACK_INTERLEAVED, scale, scale_dtype, group, src, 1, rows, cols,
                      out, out_dtype);
  if (rc != W4A16_OK || rows == 0) return rc;
  if (cols % 256 != 0 || !aligned(packed, 16)) {
    set_error("fused prologue needs cols %% 256 == 0 (got %d) and 16-byte aligned weights", cols);
    return cols % 256 != 0 ? W4A16_ERR_SHAPE : W4A16_ERR_ALIGN;
  }
  if (prologue == W4A16_PROLOGUE_RMSNORM && (!gamma || !aligned(gamma, 16))) {
    set_error("rmsnorm prologue needs a 16-byte aligned gamma");
    return gamma ? W4A16_ERR_ALIGN : W4A16_ERR_NULL;
  }
  if (bias && !aligned(bias, 4)) {
    set_error("bias must be 4-byte aligned");
    return W4A16_ERR_ALIGN;
  }
  {  // every CTA reads all of src while rows of out are written
    const uintptr_t s0 = reinterpret_cast<uintptr_t>(src);
    const uintptr_t s1 = s0 + (size_t)cols * (prologue == W4A16_PROLOGUE_NONE ? 2 : 4);
    const uintptr_t o0 = reinterpret_cast<uintptr_t>(out);
    const uintptr_t o1 = o0 + (size_t)(swiglu_out ? rows / 2 : rows) * (out_dtype == W4A16_DTYPE_F32 ? 4 : 2);
    if (s0 < o1 && o0 < s1) {
      set_error("out overlaps the prologue source");
      return W4A16_ERR_SHAPE;
    }
  }
  w4a16::GemvProblem p;
  p.packed = packed;
  p.packing = W4A16_PACK_INTERLEAVED;
  p.scale = scale;
  p.scale_dtype = scale_dtype;
  p.group = group;
  p.x = src;
  p.M = 1;
  p.N = rows;
  p.K = cols;
  p.y = out;
  p.out_dtype = out_dtype;
  p.bias = bias;
  p.workspace = workspace;
  p.workspace_bytes = workspace ? workspace_bytes : 0;
  p.prologue = prologue;
  p.pro_src = src;
  p.pro_gamma = gamma;
  p.pro_eps = eps;
  p.staged = true;
  p.pdl = (flags & W4A16_LAUNCH_PDL) != 0;
  p.out_swiglu = swiglu_out;
  p.stream = reinterpret_cast<cudaStream_t>(stream);
  return w4a16::launch_gemv(p);
}

int w4a16_decode_attention(const void* qkv, const float* cos_t, const float* sin_t,
                           const int64_t* pos, void* k_cache, void* v_cache, void* out,
                           void* scratch, size_t scratch_bytes, int heads, int kv_heads,
                           int head_dim, int max_len, int splits, unsigned flags,
                           w4a16_stream_t stream) {
  if (flags & ~(unsigned)W4A16_LAUNCH_PDL) {
    set_error("unknown launch flags 0x%x", flags);
    return W4A16_ERR_DTYPE;
  }
  if (!qkv || !cos_t || !sin_t || !pos || !k_cache || !v_cache || !out || !scratch) {
    set_error("null pointer argument");
    return W4A16_ERR_NULL;
  }
  if (head_dim != 64 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 ||
      heads / kv_heads > 32 || max_len <= 0 || splits <= 0 || splits > max_len) {
    set_error("unsupported attention shape: heads %d kv_heads %d head_dim %d max_len %d splits %d "
              "(head_dim 64, heads %% kv_heads == 0, heads / kv_heads <= 32, 1 <= splits <= max_len)",
              heads, kv_heads, head_dim, max_len, splits);
    return W4A16_ERR_SHAPE;
  }
  if (!aligned(qkv, 16) || !aligned(k_cache, 16) || !aligned(v_cache, 16) || !aligned(out, 16) ||
      !aligned(cos_t, 4) || !aligned(sin_t, 4) || !aligned(pos, 8) || !aligned(scratch, 4)) {
    set_error("qkv, caches and out must be 16-byte aligned; tables and scratch 4; pos 8");
    return W4A16_ERR_ALIGN;
  }
  if (scratch_bytes < w4a16::decode_attention_scratch_bytes(heads, kv_heads, splits)) {
    set_error("scratch of %zu bytes is smaller than the %zu needed", scratch_bytes,
              w4a16::decode_attention_scratch_bytes(heads, kv_heads, splits));
    return W4A16_ERR_WORKSPACE;
  }
  return w4a16::launch_decode_attention(qkv, cos_t, sin_t, reinterpret_cast<const long long*>(pos),
                                        k_cache, v_cache, out, scratch, heads, kv_heads, head_dim,
                                        max_len, splits, (flags & W4A16_LAUNCH_PDL) != 0,
                                        reinterpret_cast<cudaStream_t>(stream));
}

size_t w4a16_decode_attention_scratch_bytes(int heads, int kv_heads, int splits) {
  if (heads <= 0 || kv_heads <= 0 || splits <= 0) return 0;
  return w4a16::decode_attention_scratch_bytes(heads, kv_heads, splits);
}

size_t w4a16_tp_header_bytes(void) { return w4a16::kTpHeaderBytes; }

size_t w4a16_tp_ipc_handle_bytes(void) { return sizeof(cudaIpcMemHandle_t); }

int w4a16_tp_region_alloc(size_t out_bytes, void** region, void* ipc_handle) {
  if (!region || !ipc_handle) {
    set_error("null pointer argument");
    return W4A16_ERR_NULL;
  }
  *region = nullptr;
  void* p = nullptr;
  cudaError_t e = cudaMalloc(&p, w4a16::kTpHeaderBytes + out_bytes);
  if (e == cudaSuccess) e = cudaMemset(p, 0, w4a16::kTpHeaderBytes + out_bytes);
  if (e == cudaSuccess) {  // the output capacity, for the processes that open the region
    const unsigned long long cap = out_bytes;
    e = cudaMemcpy(static_cast<uint8_t*>(p) + w4a16::kTpCapacityOffset, &cap, sizeof(cap),
                   cudaMemcpyHostToDevice);
  }
  if (e == cudaSuccess) e = cudaDeviceSynchronize();
  cudaIpcMemHandle_t h;
  if (e == cudaSuccess) e = cudaIpcGetMemHandle(&h, p);
  if (e != cudaSuccess) {
    if (p) cudaFree(p);
    set_error("tensor-parallel region of %zu bytes: %s", out_bytes, cudaGetErrorString(e));
    return W4A16_ERR_CUDA;
  }
  memcpy(ipc_handle, &h, sizeof(h));
  register_region(p, out_bytes);
  *region = p;
  return W4A16_OK;
}

int w4a16_tp_region_open(const void* ipc_handle, void** region) {
  if (!region || !ipc_handle) {
    set_error("null pointer argument");
    return W4A16_ERR_NULL;
  }
  cudaIpcMemHandle_t h;
  memcpy(&h, ipc_handle, sizeof(h));
  void* p = nullptr;
  cudaError_t e = cudaIpcOpenMemHandle(&p, h, cudaIpcMemLazyEnablePeerAccess);
  if (e != cudaSuccess) {
    set_error("cudaIpcOpenMemHandle: %s", cudaGetErrorString(e));
    return W4A16_ERR_CUDA;
  }
  unsigned long long cap = 0;  // written into the header by the owner's w4a16_tp_region_alloc
  e = cudaMemcpy(&cap, static_cast<uint8_t*>(p) + w4a16::kTpCapacityOffset, sizeof(cap),
                 cudaMemcpyDeviceToHost);
  if (e != cudaSuccess) {
    cudaIpcCloseMemHandle(p);
    set_error("reading the capacity of an opened region: %s", cudaGetErrorString(e));
    return W4A16_ERR_CUDA;
  }
  register_region(p, (size_t)cap);
  *region = p;
  return W4A16_OK;
}

int w4a16_tp_region_close(void* region, int owned) {
  if (!region) return W4A16_OK;
  forget_region(region);
  const cudaError_t e = owned ? cudaFree(region) : cudaIpcCloseMemHandle(region);
  if (e != cudaSuccess) {
    set_error("closing a tensor-parallel region: %s", cudaGetErrorString(e));
    return W4A16_ERR_CUDA;
  }
  return W4A16_OK;
}

int w4a16_tp_region_timeline(const void* region, unsigned long long* stamps, w4a16_stream_t stream) {
  if (!region || !stamps) {
    set_error("null pointer argument");
    return W4A16_ERR_NULL;
  }
  size_t cap = 0;
  if (!region_capacity(region, &cap)) {
    set_error("region %p was not created by w4a16_tp_region_alloc or mapped by w4a16_tp_region_open in this process", region);
    return W4A16_ERR_SHAPE;
  }
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e = cudaMemcpyAsync(stamps, static_cast<const uint8_t*>(region) + w4a16::kTpTimelineOffset,
                                  4 * sizeof(unsigned long long), cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  if (e != cudaSuccess) {
    set_error("reading a region's step timeline: %s", cudaGetErrorString(e));
    return W4A16_ERR_CUDA;
  }
  return W4A16_OK;
}

int w4a16_gemv_allgather(const uint8_t* packed, const void* scale, int scale_dtype, int group,
                         const void* x, int rows, int cols, int out_dtype, long long row0, int rank,
                         int nranks, void* const* regions, void* workspace, size_t workspace_bytes,
                         unsigned flags, w4a16_stream_t stream) {
  if (flags & ~(unsigned)W4A16_LAUNCH_PDL) {
    set_error("unknown launch flags 0x%x", flags);
    return W4A16_ERR_DTYPE;
  }
  if (!regions) {
    set_error("null pointer argument");
    return W4A16_ERR_NULL;
  }
  if (nranks < 2 || nranks > 8 || rank < 0 || rank >= nranks || row0 < 0 || rows < 1) {
    set_error("fused all-gather needs 2..8 ranks, 0 <= rank < nranks, row0 >= 0 and rows >= 1 "
              "(got rank %d of %d, row0 %lld, rows %d)", rank, nranks, row0, rows);
    return W4A16_ERR_SHAPE;
  }
  for (int k = 0; k < nranks; ++k)
    if (!regions[k] || !aligned(regions[k], 256)) {
      set_error("region %d is null or not 256-byte aligned", k);
      return regions[k] ? W4A16_ERR_ALIGN : W4A16_ERR_NULL;
    }
  uint8_t* mine = static_cast<uint8_t*>(regions[rank]) + w4a16::kTpHeaderBytes;
  int rc = check_gemv(packed, W4A16_PACK_INTERLEAVED, scale, scale_dtype, group, x, 1, rows, cols,
                      mine, out_dtype);
  if (rc != W4A16_OK) return rc;
  {  // rows [row0, row0 + rows) are stored into every region: each must hold them
    const size_t esize = out_dtype == W4A16_DTYPE_F32 ? 4 : 2;
    const unsigned long long end = ((unsigned long long)row0 + (unsigned long long)rows) * esize;
    for (int k = 0; k < nranks; ++k) {
      size_t cap = 0;
      if (!region_capacity(regions[k], &cap)) {
        set_error("region %d was not created by w4a16_tp_region_alloc or mapped by "
                  "w4a16_tp_region_open in this process", k);
        return W4A16_ERR_SHAPE;
      }
      if (end > cap) {
        set_error("rows [%lld, %lld) of %zu-byte outputs do not fit region %d (%zu bytes)", row0,
                  row0 + rows, esize, k, cap);
        return W4A16_ERR_SHAPE;
      }
    }
  }
  if (cols % 256 != 0 || !aligned(packed, 16)) {
    set_error("fused all-gather needs cols %% 256 == 0 (got %d) and 16-byte aligned weights", cols);
    return cols % 256 != 0 ? W4A16_ERR_SHAPE : W4A16_ERR_ALIGN;
  }
  w4a16::GemvProblem p;
  p.packed = packed;
  p.packing = W4A16_PACK_INTERLEAVED;
  p.scale = scale;
  p.scale_dtype = scale_dtype;
  p.group = group;
  p.x = x;
  p.M = 1;
  p.N = rows;
  p.K = cols;
  p.y = mine;
  p.out_dtype = out_dtype;
  p.workspace = workspace;
  p.workspace_bytes = workspace ? workspace_bytes : 0;
  p.tp_n = nranks;
  p.tp_rank = rank;
  p.tp_row0 = row0;
  for (int k = 0; k < nranks; ++k) {
    p.tp_flags[k] = static_cast<unsigned*>(regions[k]);
    p.tp_out[k] = static_cast<uint8_t*>(regions[k]) + w4a16::kTpHeaderBytes;
  }
  const unsigned long long wait = g_peer_wait_ns.load(std::memory_order_relaxed);
  p.tp_wait_ns = wait ? wait : kDefaultPeerWaitNs;
  p.pdl = (flags & W4A16_LAUNCH_PDL) != 0;
  p.stream = reinterpret_cast<cudaStream_t>(stream);
  return w4a16::launch_gemv(p);
}

int w4a16_tp_set_peer_wait_ns(unsigned long long ns) {
  if (ns != 0 && (ns < 1000ull || ns > 60000000000ull)) {
    set_error("peer wait limit %llu ns outside [1 us, 60 s] (0 restores the 2 s default)", ns);
    return W4A16_ERR_SHAPE;
  }
  g_peer_wait_ns.store(ns, std::memory_order_relaxed);
  return W4A16_OK;
}

size_t w4a16_gemv_workspace_bytes(int batch, int rows, int cols) {
  return w4a16::gemv_workspace_bytes(batch, rows, cols);
}

int w4a16_dequant(const uint8_t* packed, int packing, const void* scale, int scale_dtype,
                  int group, int rows, int cols, void* out, w4a16_stream_t stream) {
  int rc = check_gemv(packed, packing, scale, scale_dtype, group, out, 1, rows, cols, out,
                      W4A16_DTYPE_F16);
  if (rc != W4A16_OK || rows == 0) return rc;
  return w4a16::launch_dequant(packed, packing, scale, scale_dtype, group, rows, cols, out,
                               reinterpret_cast<cudaStream_t>(stream));
}

int w4a16_quantize_pack(const void* w, int w_dtype, int rows, int cols, int group, int packing,
                        uint8_t* packed, void* scale, int scale_dtype, w4a16_stream_t stream) {
  if (w_dtype != W4A16_DTYPE_F32 && w_dtype != W4A16_DTYPE_F16) {
    set_error("unknown weight dtype code %d", w_dtype);
    return W4A16_ERR_DTYPE;
  }
  int rc = check_gemv(packed, packing, scale, scale_dtype, group, packed, 1, rows, cols, packed,
                      W4A16_DTYPE_F16);
  if (rc != W4A16_OK || rows == 0) return rc;
  if (!w) {
    set_error("NULL weight pointer");
    return W4A16_ERR_NULL;
  }
  if (!aligned(w, w_dtype == W4A16_DTYPE_F32 ? 4 : 2)) {
    set_error("weight pointer misaligned");
    return W4A16_ERR_ALIGN;
  }
  return w4a16::launch_quantize_pack(w, w_dtype, rows, cols, group, packing, packed, scale,
                                     scale_dtype, reinterpret_cast<cudaStream_t>(stream));
}

int w4a16_read_device_error(int* code, w4a16_stream_t stream) {
  if (!code) {
    set_error("NULL code pointer");
    return W4A16_ERR_NULL;
  }
  int a = 0, b = 0, c = 0;
  int rc = w4a16::read_device_error(&a, reinterpret_cast<cudaStream_t>(stream));
  if (rc == W4A16_OK) rc = w4a16::read_decode_step_error(&b, reinterpret_cast<cudaStream_t>(stream));
  if (rc == W4A16_OK) rc = w4a16::read_gemm_error(&c, reinterpret_cast<cudaStream_t>(stream));
  if (rc != W4A16_OK) return rc;
  *code = a ? a : b ? b : c;
  return W4A16_OK;
}

size_t w4a16_gemm_workspace_bytes(int M, int N, int K) { return w4a16::gemm_workspace_bytes(M, N, K); }

int w4a16_gemm(const uint8_t* packed, const float* scale, int group, const void* x,
               const float* bias, int M, int N, int K, void* y, int out_dtype, void* workspace,
               size_t workspace_bytes, w4a16_stream_t stream) {
  if (out_dtype != W4A16_DTYPE_F32 && out_dtype != W4A16_DTYPE_F16) {
    set_error("unknown output dtype code %d", out_dtype);
    return W4A16_ERR_DTYPE;
  }
  if (group != 0 && group != 128) {
    set_error("group must be 0 (per-row) or 128, got %d", group);
    return W4A16_ERR_DTYPE;
  }
  if (M <= 0 || N <= 0 || K <= 0 || K % 64 != 0 || (group && K % group != 0)) {
    set_error("bad GEMM shape M=%d N=%d K=%d (K a multiple of %d)", M, N, K, group ? 128 : 64);
    return W4A16_ERR_SHAPE;
  }
  if (!packed || !scale || !x || !y) {
    set_error("NULL pointer (packed %p, scale %p, x %p, y %p)", (const void*)packed, (const void*)scale,
              x, y);
    return W4A16_ERR_NULL;
  }
  const size_t osz = out_dtype == W4A16_DTYPE_F32 ? 4 : 2;
  if (!aligned(packed, 16) || !aligned(x, 16) || !aligned(scale, 4) || !aligned(y, osz) ||
      (bias && !aligned(bias, 4)) || (workspace && !aligned(workspace, 256))) {
    set_error("misaligned pointer: packed and x need 16 B, scale and bias 4 B, y %zu B, workspace 256 B", osz);
    return W4A16_ERR_ALIGN;
  }
  return w4a16::launch_gemm(packed, scale, group, x, bias, M, N, K, y, out_dtype, workspace,
                            workspace_bytes, reinterpret_cast<cudaStream_t>(stream));
}

int w4a16_decode_plan_create(const w4a16_llama_desc* desc, w4a16_decode_plan* plan) {
  if (!plan) {
    set_error("null plan pointer");
    return W4A16_ERR_NULL;
  }
  w4a16::DecodePlan* p = nullptr;
  const int rc = w4a16::decode_plan_create(desc, &p);
  *plan = reinterpret_cast<w4a16_decode_plan>(p);
  return rc;
}

int w4a16_decode_plan_destroy(w4a16_decode_plan plan) {
  return w4a16::decode_plan_destroy(reinterpret_cast<w4a16::DecodePlan*>(plan));
}

int w4a16_decode_plan_timeline(w4a16_decode_plan plan, int enable, unsigned long long* host,
                               size_t capacity, size_t* count, w4a16_stream_t stream) {
  if (!plan) {
    set_error("null plan");
    return W4A16_ERR_NULL;
  }
  return w4a16::decode_plan_timeline(reinterpret_cast<w4a16::DecodePlan*>(plan), enable, host, capacity,
                                     count, reinterpret_cast<cudaStream_t>(stream));
}

int w4a16_decode_step(w4a16_decode_plan plan, const int64_t* token, const int64_t* pos,
                      void* k_cache, void* v_cache, float* logits, w4a16_stream_t stream) {
  if (!plan || !token || !pos || !k_cache || !v_cache || !logits) {
    set_error("null pointer argument");
    return W4A16_ERR_NULL;
  }
  if (!aligned(token, 8) || !aligned(pos, 8) || !aligned(k_cache, 16) || !aligned(v_cache, 16) ||
      !aligned(logits, 4)) {
    set_error("token/pos need 8-byte, caches 16-byte, logits 4-byte alignment");
    return W4A16_ERR_ALIGN;
  }
  return w4a16::decode_step_launch(reinterpret_cast<w4a16::DecodePlan*>(plan),
                                   reinterpret_cast<const long long*>(token),
                                   reinterpret_cast<const long long*>(pos), k_cache, v_cache, logits,
                                   reinterpret_cast<cudaStream_t>(stream));
}

int w4a16_paged_append(const void* q, long long q_stride, const void* k, long long k_stride,
                       const void* v, long long v_stride, const int32_t* positions,
                       const int32_t* seqs, int tokens, int heads, const w4a16_page_tables* tables,
                       const float* cos_t, const float* sin_t, int angle_rows,
                       const w4a16_page_pool* pool, void* q_out, long long q_out_stride,
                       w4a16_stream_t stream) {
  w4a16::PagedPool pl;
  w4a16::PagedTables tb;
  int rc = check_pool(pool, &pl);
  if (rc == W4A16_OK) rc = check_tables(tables, &tb);
  if (rc != W4A16_OK) return rc;
  if (tokens < 0 || heads < 0 || (cos_t == nullptr) != (sin_t == nullptr) || (cos_t && angle_rows <= 0)) {
    set_error("bad shape: %d tokens, %d heads, %d rows of angles (cos and sin together)", tokens, heads, angle_rows);
    return W4A16_ERR_SHAPE;
  }
  if (tokens == 0) return W4A16_OK;
  if (!k || !v || !positions || (heads && (!q || !q_out))) {
    set_error("null pointer argument");
    return W4A16_ERR_NULL;
  }
  if (q_stride % 8 || k_stride % 8 || v_stride % 8 || q_out_stride % 8 || q_stride < 0 || k_stride < 0 || v_stride < 0 ||
      (heads && tokens > 1 && q_out_stride < (long long)heads * pl.head_dim) || !aligned(k, 16) || !aligned(v, 16) ||
      (heads && (!aligned(q, 16) || !aligned(q_out, 16))) || !aligned(positions, 4) || (seqs && !aligned(seqs, 4)) ||
      (cos_t && (!aligned(cos_t, 16) || !aligned(sin_t, 16)))) {
    set_error("q, k, v, q_out and the angles must be 16-byte aligned with strides of multiples of 8 elements, indices 4");
    return W4A16_ERR_ALIGN;
  }
  w4a16::PagedAppend a;
  a.q = q;
  a.k = k;
  a.v = v;
  a.q_out = q_out;
  a.q_stride = q_stride;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  a.q_out_stride = q_out_stride;
  a.positions = positions;
  a.seqs = seqs;
  a.cos_t = cos_t;
  a.sin_t = sin_t;
  a.angle_rows = angle_rows;
  a.tokens = tokens;
  a.heads = heads;
  return w4a16::launch_paged_append(a, pl, tb, reinterpret_cast<cudaStream_t>(stream));
}

size_t w4a16_paged_attention_workspace_bytes(int heads, int kv_heads, int head_dim) {
  if (heads <= 0 || kv_heads <= 0 || heads % kv_heads || head_dim <= 0) return 0;
  return w4a16::paged_attention_workspace_bytes(heads, kv_heads, head_dim);
}

size_t w4a16_paged_attention_call_bytes(int dtype, int rows, int heads, int kv_heads, int head_dim, int width, int page_size) {
  if ((dtype != W4A16_DTYPE_F16 && dtype != W4A16_DTYPE_BF16) || rows <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads ||
      (head_dim != 64 && head_dim != 128 && head_dim != 256) || width <= 0 || page_size <= 0)
    return 0;
  return w4a16::paged_attention_needs_workspace(dtype, rows, heads, kv_heads, head_dim, (long long)width * page_size)
             ? w4a16::paged_attention_workspace_bytes(heads, kv_heads, head_dim)
             : 0;
}

int w4a16_paged_attention(const void* q, long long q_stride, const int32_t* lengths,
                          const int32_t* seqs, int rows, int heads, const w4a16_page_tables* tables,
                          const w4a16_page_pool* pool, float scale, void* out, long long out_stride,
                          void* workspace, size_t workspace_bytes, w4a16_stream_t stream) {
  w4a16::PagedPool pl;
  w4a16::PagedTables tb;
  int rc = check_pool(pool, &pl);
  if (rc == W4A16_OK) rc = check_tables(tables, &tb);
  if (rc != W4A16_OK) return rc;
  if (rows < 0 || heads <= 0 || heads % pl.kv_heads || ((long long)tb.width << pl.page_shift) > (1 << 30)) {
    set_error("bad shape: %d rows, %d heads over %d kv heads, tables of %d pages (at most 2^30 positions)", rows, heads,
              pl.kv_heads, tb.width);
    return W4A16_ERR_SHAPE;
  }
  if (!(scale > 0.f) || scale > 0x1p127f) {  // times log2(e) it has to stay a number
    set_error("scale %g is not a positive number up to 2^127", scale);
    return W4A16_ERR_SHAPE;
  }
  if (rows == 0) return W4A16_OK;
  if (!q || !lengths || !out) {
    set_error("null pointer argument");
    return W4A16_ERR_NULL;
  }
  if (q_stride % 8 || out_stride % 8 || q_stride < 0 || (rows > 1 && out_stride < (long long)heads * pl.head_dim) ||
      !aligned(q, 16) || !aligned(out, 16) || !aligned(lengths, 4) || (seqs && !aligned(seqs, 4))) {
    set_error("q and out must be 16-byte aligned with strides of multiples of 8 elements, indices 4");
    return W4A16_ERR_ALIGN;
  }
  const bool none = !workspace && workspace_bytes == 0 &&
                    w4a16_paged_attention_call_bytes(pl.dtype, rows, heads, pl.kv_heads, pl.head_dim, tb.width, 1 << pl.page_shift) == 0;
  if (!none) rc = check_scratch(workspace, workspace_bytes, w4a16::paged_attention_workspace_bytes(heads, pl.kv_heads, pl.head_dim));
  if (rc != W4A16_OK) return rc;
  w4a16::PagedAttention a;
  a.q = q;
  a.out = out;
  a.q_stride = q_stride;
  a.out_stride = out_stride;
  a.lengths = lengths;
  a.seqs = seqs;
  a.rows = rows;
  a.heads = heads;
  a.scale = scale;
  a.workspace = workspace;
  return w4a16::launch_paged_attention(a, pl, tb, reinterpret_cast<cudaStream_t>(stream));
}

int w4a16_pages_extend(const w4a16_page_state* state, const int32_t* seqs, const int32_t* counts,
                       int n, int32_t* ok, w4a16_stream_t stream) {
  w4a16::PagesState st;
  int rc = check_state(state, &st);
  if (rc == W4A16_OK) rc = check_requests(n, w4a16::kPagesMaxRequests, seqs, counts, ok);
  if (rc != W4A16_OK || n == 0) return rc;
  if ((long long)n * st.width > (1 << 30)) {  // the pages that the call may ask for are summed in 32 bits
    set_error("%d requests on rows of %d pages are too many for one call (2^30 pages)", n, st.width);
    return W4A16_ERR_SHAPE;
  }
  return w4a16::launch_pages_extend(st, seqs, counts, n, ok, reinterpret_cast<cudaStream_t>(stream));
}

size_t w4a16_pages_fork_scratch_bytes(int n) { return n > 0 ? (size_t)n * 8 : 0; }

int w4a16_pages_fork(const w4a16_page_state* state, const w4a16_page_blocks* blocks,
                     const int32_t* src, const int32_t* dst, int n, int32_t* ok, void* scratch,
                     size_t scratch_bytes, w4a16_stream_t stream) {
  w4a16::PagesState st;
  w4a16::PageBlocks b;
  int rc = check_state(state, &st);
  if (rc == W4A16_OK) rc = check_blocks(blocks, &b);
  if (rc == W4A16_OK) rc = check_requests(n, w4a16::kPagesMaxRequests, src, dst, ok);
  if (rc != W4A16_OK || n == 0) return rc;
  if (st.pages != b.pages) {
    set_error("the page state has %d pages, the blocks %d", st.pages, b.pages);
    return W4A16_ERR_SHAPE;
  }
  rc = check_scratch(scratch, scratch_bytes, w4a16_pages_fork_scratch_bytes(n));
  if (rc != W4A16_OK) return rc;
  return w4a16::launch_pages_fork(st, b, src, dst, n, ok, scratch, reinterpret_cast<cudaStream_t>(stream));
}

int w4a16_pages_free(const w4a16_page_state* state, const int32_t* seqs, int n, int32_t* ok,
                     w4a16_stream_t stream) {
  w4a16::PagesState st;
  int rc = check_state(state, &st);
  if (rc == W4A16_OK) rc = check_requests(n, 1 << 16, seqs, seqs, ok);
  if (rc != W4A16_OK || n == 0) return rc;
  return w4a16::launch_pages_free(st, seqs, n, ok, reinterpret_cast<cudaStream_t>(stream));
}

int w4a16_pages_copy(const w4a16_page_blocks* blocks, const int32_t* src, const int32_t* dst, int n,
                     w4a16_stream_t stream) {
  w4a16::PageBlocks b;
  int rc = check_blocks(blocks, &b);
  if (rc == W4A16_OK) rc = check_requests(n, 1 << 30, src, dst, src);
  if (rc != W4A16_OK || n == 0) return rc;
  return w4a16::launch_pages_copy(b, src, dst, n, reinterpret_cast<cudaStream_t>(stream));
}

size_t w4a16_pages_compact_scratch_bytes(int pages) {
  return pages > 0 ? w4a16::pages_compact_scratch_bytes(pages) : 0;
}

int w4a16_pages_compact(const w4a16_page_blocks* blocks, const int32_t* tables, int32_t* tables_out,
                        long long entries, const int32_t* refs, int32_t* refs_out, int32_t* moved,
                        void* scratch, size_t scratch_bytes, w4a16_stream_t stream) {
  w4a16::PageBlocks b;
  int rc = check_blocks(blocks, &b);
  if (rc != W4A16_OK) return rc;
  if (entries < 0) {
    set_error("%lld table entries", entries);
    return W4A16_ERR_SHAPE;
  }
  if (!refs || !refs_out || !moved || (entries && (!tables || !tables_out))) {
    set_error("null pointer argument");
    return W4A16_ERR_NULL;
  }
  if (!aligned(refs, 4) || !aligned(refs_out, 4) || !aligned(moved, 4) || (entries && (!aligned(tables, 4) || !aligned(tables_out, 4)))) {
    set_error("tables, refs and moved must be 4-byte aligned");
    return W4A16_ERR_ALIGN;
  }
  rc = check_scratch(scratch, scratch_bytes, w4a16::pages_compact_scratch_bytes(b.pages));
  if (rc != W4A16_OK) return rc;
  return w4a16::launch_pages_compact(b, tables, tables_out, entries, refs, refs_out, moved, scratch,
                                     reinterpret_cast<cudaStream_t>(stream));
}

int w4a16_process_logits(const w4a16_logits_desc* d, w4a16_stream_t stream) {
  if (!d) {
    set_error("null description");
    return W4A16_ERR_NULL;
  }
  if (d->dtype != W4A16_DTYPE_F32 && d->dtype != W4A16_DTYPE_F16 && d->dtype != W4A16_DTYPE_BF16) {
    set_error("unknown logits dtype code %d", d->dtype);
    return W4A16_ERR_DTYPE;
  }
  if (d->tokens && d->token_bytes != 4 && d->token_bytes != 8) {
    set_error("tokens of %d bytes (4 or 8)", d->token_bytes);
    return W4A16_ERR_DTYPE;
  }
  if (d->rows < 0 || d->vocab < 0 || d->vocab > (1 << 30) || d->history < 0 || d->history > (1 << 30) || d->pairs < 0 || d->stride < 0 || d->bias_stride < 0 ||
      d->mask_stride < 0 || d->token_stride < 0 || (d->rows > 1 && d->out_stride < d->vocab)) {
    set_error("bad shape: rows %d vocab %d history %d pairs %d or a negative or overlapping stride", d->rows, d->vocab,
              d->history, d->pairs);
    return W4A16_ERR_SHAPE;
  }
  if (d->rows == 0 || d->vocab == 0) return W4A16_OK;
  if (!d->logits || !d->out || (d->pairs && (!d->bias_ids || !d->bias_values))) {
    set_error("null pointer argument");
    return W4A16_ERR_NULL;
  }
  const size_t size = d->dtype == W4A16_DTYPE_F32 ? 4 : 2;
  if (!aligned(d->logits, size) || !aligned(d->out, size) || (d->tokens && !aligned(d->tokens, d->token_bytes)) ||
      (d->prompt_lens && !aligned(d->prompt_lens, 4)) || (d->total_lens && !aligned(d->total_lens, 4)) ||
      (d->repetition && !aligned(d->repetition, 4)) || (d->frequency && !aligned(d->frequency, 4)) ||
      (d->presence && !aligned(d->presence, 4)) || (d->bias && !aligned(d->bias, 4)) ||
      (d->pairs && (!aligned(d->bias_ids, 4) || !aligned(d->bias_values, 4))) || (d->mask && !aligned(d->mask, 4))) {
    set_error("a pointer is not aligned to its element size");
    return W4A16_ERR_ALIGN;
  }
  {  // in place exactly, or apart
    const uintptr_t i0 = reinterpret_cast<uintptr_t>(d->logits), o0 = reinterpret_cast<uintptr_t>(d->out);
    const uintptr_t i1 = i0 + ((size_t)(d->rows - 1) * d->stride + d->vocab) * size;
    const uintptr_t o1 = o0 + ((size_t)(d->rows - 1) * d->out_stride + d->vocab) * size;
    if (i0 < o1 && o0 < i1 && !(i0 == o0 && (d->rows == 1 || d->stride == d->out_stride))) {
      set_error("out overlaps logits without being them");
      return W4A16_ERR_SHAPE;
    }
  }
  w4a16::LogitsProblem p;
  p.logits = d->logits;
  p.out = d->out;
  p.dtype = d->dtype;
  p.rows = d->rows;
  p.vocab = d->vocab;
  p.stride = d->stride;
  p.out_stride = d->out_stride;
  p.tokens = d->history ? d->tokens : nullptr;
  p.token_bytes = d->token_bytes;
  p.history = d->history;
  p.token_stride = d->token_stride;
  p.prompt_lens = d->prompt_lens;
  p.total_lens = d->total_lens;
  p.repetition = d->repetition;
  p.frequency = d->frequency;
  p.presence = d->presence;
  p.bias = d->bias;
  p.bias_stride = d->bias_stride;
  p.bias_ids = d->bias_ids;
  p.bias_values = d->bias_values;
  p.pairs = d->pairs;
  p.mask = d->mask;
  p.mask_stride = d->mask_stride;
  return w4a16::launch_process_logits(p, reinterpret_cast<cudaStream_t>(stream));
}

const char* w4a16_status_string(int status) {
  switch (status) {
    case W4A16_OK: return "ok";
    case W4A16_ERR_NULL: return "NULL pointer";
    case W4A16_ERR_SHAPE: return "bad shape";
    case W4A16_ERR_ALIGN: return "misaligned pointer";
    case W4A16_ERR_DTYPE: return "unknown dtype, packing or group";
    case W4A16_ERR_WORKSPACE: return "workspace too small";
    case W4A16_ERR_CUDA: return "CUDA error";
    case W4A16_ERR_KERNEL: return "kernel wait timed out";
    default: return "unknown status";
  }
}

const char* w4a16_last_error_string(void) { return w4a16::last_error(); }

int w4a16_version(void) { return kVersion; }

}  // extern "C"
