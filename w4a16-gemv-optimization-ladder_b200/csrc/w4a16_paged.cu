// Decode over a paged key-value cache: the write of new keys and values into the pages of
// their sequences (with the rotary embedding of q and k), and the attention of one new token
// per row over a sequence's pages.  The static-cache counterpart for one sequence is
// w4a16_decode.cu.
//
// A page holds page_size consecutive positions of one sequence, for every kv head; row s of
// `tables` lists the pages of sequence s in order, so position p of sequence s lies in page
// tables[s][p / page_size], row p % page_size.  Pages are looked up with bounds checks: an
// entry outside the pool (or a position past the row's entries) is never dereferenced and
// gives NaN.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <type_traits>

#include "w4a16_device.cuh"
#include "w4a16_internal.h"

namespace w4a16 {

namespace {

// The page that holds position p of sequence s, or -1 (bad sequence, position or entry).
__device__ __forceinline__ int page_of(const PagedTables& t, int s, int p, int page_shift, int pages) {
  if (s < 0 || s >= t.rows || p < 0 || (p >> page_shift) >= t.width) return -1;
  const int page = __ldg(t.ids + (size_t)s * t.stride + (p >> page_shift));
  return page < 0 || page >= pages ? -1 : page;
}

// ---------------------------------------------------------------------------- append
//
// One thread turns 8 pairs (i, i + D/2) of one head of one token: two 16-byte loads, two
// 16-byte stores, angles read as float4 (they stay in L1 across a token's heads).
template <typename T, int D>
__global__ void __launch_bounds__(256) k_paged_append(const PagedAppend a, const PagedPool pool, const PagedTables tab) {
  constexpr int kChunks = D / 16;
  const int per_token = (a.heads + 2 * pool.kv_heads) * kChunks;
  const long long total = (long long)a.tokens * per_token;
  for (long long e = (long long)blockIdx.x * blockDim.x + threadIdx.x; e < total; e += (long long)gridDim.x * blockDim.x) {
    const int t = (int)(e / per_token), r = (int)(e % per_token);
    const int head = r / kChunks, i = (r % kChunks) * 8;
    const int pos = __ldg(a.positions + t);
    const int seq = a.seqs ? __ldg(a.seqs + t) : t;
    int page = pos < 0 ? -1 : page_of(tab, seq, pos, pool.page_shift, pool.pages);
    if (a.cos_t && pos >= a.angle_rows) page = -1;
    const bool is_q = head < a.heads;
    if (!is_q && page < 0) continue;
    uint4 lo, hi;
    T* dst;
    if (is_q) {
      dst = static_cast<T*>(a.q_out) + (size_t)t * a.q_out_stride + head * D;
      if (page < 0) {  // padding: zeros; a bad position, sequence or page: NaN
        const uint32_t w = pos < 0 ? 0u : pack2<T>(__int_as_float(0x7fc00000), __int_as_float(0x7fc00000));
        lo = hi = make_uint4(w, w, w, w);
        *reinterpret_cast<uint4*>(dst + i) = lo;
        *reinterpret_cast<uint4*>(dst + i + D / 2) = hi;
        continue;
      }
      const T* src = static_cast<const T*>(a.q) + (size_t)t * a.q_stride + head * D;
      lo = *reinterpret_cast<const uint4*>(src + i);
      hi = *reinterpret_cast<const uint4*>(src + i + D / 2);
    } else {
      const int kvh = (head - a.heads) % pool.kv_heads;
      const bool is_v = head - a.heads >= pool.kv_heads;
      const T* src = is_v ? static_cast<const T*>(a.v) + (size_t)t * a.v_stride + kvh * D
                          : static_cast<const T*>(a.k) + (size_t)t * a.k_stride + kvh * D;
      dst = static_cast<T*>(is_v ? pool.v : pool.k) + (size_t)page * pool.page_stride + (size_t)kvh * pool.head_stride +
            (size_t)(pos & ((1 << pool.page_shift) - 1)) * pool.token_stride;
      lo = *reinterpret_cast<const uint4*>(src + i);
      hi = *reinterpret_cast<const uint4*>(src + i + D / 2);
      if (is_v) {
        *reinterpret_cast<uint4*>(dst + i) = lo;
        *reinterpret_cast<uint4*>(dst + i + D / 2) = hi;
        continue;
      }
    }
    if (a.cos_t) {
      uint32_t* l = reinterpret_cast<uint32_t*>(&lo);
      uint32_t* h = reinterpret_cast<uint32_t*>(&hi);
      const float* cr = a.cos_t + (size_t)pos * D + i;
      const float* sr = a.sin_t + (size_t)pos * D + i;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 x = unpack2<T>(l[j]), y = unpack2<T>(h[j]);
        const float2 c0 = __ldg(reinterpret_cast<const float2*>(cr) + j), s0 = __ldg(reinterpret_cast<const float2*>(sr) + j);
        const float2 c1 = __ldg(reinterpret_cast<const float2*>(cr + D / 2) + j);
        const float2 s1 = __ldg(reinterpret_cast<const float2*>(sr + D / 2) + j);
        l[j] = pack2<T>(x.x * c0.x - y.x * s0.x, x.y * c0.y - y.y * s0.y);
        h[j] = pack2<T>(y.x * c1.x + x.x * s1.x, y.y * c1.y + x.y * s1.y);
      }
    }
    *reinterpret_cast<uint4*>(dst + i) = lo;
    *reinterpret_cast<uint4*>(dst + i + D / 2) = hi;
  }
}

// ------------------------------------------------------------------------- attention
//
// Bound by the bytes of the keys and values: each is used for the few query heads of its kv
// head only.  One pass over them with a running maximum and sum; the pages go straight from
// global memory into the operand registers of m16n8k16 tensor-core products (no shared memory
// in between), which the freedom to number the contracted index allows:
//   S^T[position][head] = K Q^T    A = K: lane (g = lane / 4, j = lane % 4) loads 16 bytes of
//                                  positions g and g + 8 at dimensions 8j of each block of 32;
//                                  these four words are the k = 2j, 2j+1, 2j+8, 2j+9 operands
//                                  of two products, and Q is loaded by the same numbering
//   O^T[dimension][head] = V^T P   A = V^T: the lane loads 16 bytes (dimensions 8g) of positions
//                                  2j, 2j+1, 2j+8, 2j+9 and pairs two positions with one byte
//                                  permutation per word; P^T comes from S^T by two 8 x 8 matrix
//                                  transpositions
// The 8 (NH = 1) or 16 (NH = 2) query heads of a CTA are the n of the products.
//
// Work is shared out by a count of units of kUnit positions over all (row, kv head, block of
// query heads) items, in that order: worker w (a CTA) takes units [w T / W, (w + 1) T / W) of
// the T there are (W workers, no more than T), wherever that cuts an item.  The lengths are read on the device, so every
// worker first sums them up.  An item that lies within one worker is finished there; the parts
// of one that was cut go to the workspace (slot 2w + 1 if the part begins the item, else 2w)
// and are joined by k_paged_join.
constexpr int kAttnWarps = 4;
constexpr int kAttnMaxWorkers = 592;  // bounds the workspace: 148 SMs with 4 workers

template <int D, int NH>
struct AttnCfg {
  static constexpr int kTiles = D == 64 ? 2 : 1;  // 16-position tiles a warp holds at once
  static constexpr int kUnit = 16 * kTiles * kAttnWarps;
  static constexpr int kHeads = 8 * NH;
  static constexpr int kPerSm = D == 64 ? (NH == 1 ? 4 : 3) : D == 128 ? (NH == 1 ? 3 : 2) : 2;
  static constexpr int kSlot = kHeads * (D + 2);  // floats of a part: m, l, o per head
};

struct AttnDesc {  // the item that worker w began and did not finish
  int row, item, parts, pad;
};

template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__half>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  mma_16816(d, a0, a1, a2, a3, b0, b1);
}
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                                        uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Keys and values are read once: past L1.
__device__ __forceinline__ uint4 ld_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

template <typename T, int D, int NH>
__global__ void __launch_bounds__(kAttnWarps * 32, AttnCfg<D, NH>::kPerSm)
    k_paged_attention(const PagedAttention a, const PagedPool pool, const PagedTables tab, const int group, const int blocks) {
  using C = AttnCfg<D, NH>;
  constexpr int kB = D / 32, kVB = D / 64, kU = C::kTiles, kHeads = C::kHeads, kThreads = kAttnWarps * 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, j = lane & 3;
  const int worker = blockIdx.x, workers = gridDim.x;
  const int items = pool.kv_heads * blocks;
  const float nan = __int_as_float(0x7fc00000);
  __shared__ long long sh_total, sh_base, sh_warp[kAttnWarps];
  __shared__ int sh_row;
  __shared__ float sh_m[kAttnWarps][kHeads], sh_l[kAttnWarps][kHeads];
  extern __shared__ float sh_o[];  // [warp][head][D]

  grid_launch_dependents();  // the join waits for this kernel's end before it reads anything
  AttnDesc* desc = static_cast<AttnDesc*>(a.workspace);
  float* slots = reinterpret_cast<float*>(desc + kAttnMaxWorkers);
  const long long cap = (long long)tab.width << pool.page_shift;
  // a length past the tables keeps one position there, which has no page: NaN
  auto length = [&](int row) {
    const int n = __ldg(a.lengths + row);
    return n <= 0 ? 0 : n > cap ? (int)(cap + 1) : n;
  };
  auto tiles = [](int len) { return (len + C::kUnit - 1) / C::kUnit; };

  // the units of all rows, and the row that holds this worker's first one
  const int per = (a.rows + kThreads - 1) / kThreads;
  const int r0 = min(a.rows, (int)threadIdx.x * per), r1 = min(a.rows, r0 + per);
  long long sum = 0;
  for (int r = r0; r < r1; ++r) sum += tiles(length(r));
  sum *= items;
  long long inc = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long n = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += n;
  }
  if (lane == 31) sh_warp[warp] = inc;
  if (threadIdx.x == 0) sh_row = a.rows;
  __syncthreads();
  long long before = inc - sum, total = 0;
  for (int w = 0; w < kAttnWarps; ++w) {
    if (w < warp) before += sh_warp[w];
    total += sh_warp[w];
  }
  // every worker in use has a unit, so the parts of an item lie with consecutive workers
  const long long used = total < workers ? total : workers;
  const long long u0 = worker < used ? worker * total / used : 0, u1 = worker < used ? (worker + 1LL) * total / used : 0;
  if (u0 < u1 && before <= u0 && u0 < before + sum) {  // one thread
    long long base = before;
    int r = r0;
    for (;; ++r) {
      const long long n = (long long)tiles(length(r)) * items;
      if (u0 < base + n) break;
      base += n;
    }
    sh_row = r;
    sh_base = base;
  }
  if (threadIdx.x == 0) desc[worker].parts = 0;
  // rows of no positions are zero
  for (int r = worker; r < a.rows; r += workers)
    if (length(r) == 0)
      for (int e = threadIdx.x; e < items / blocks * group * D / 8; e += kThreads)
        reinterpret_cast<uint4*>(static_cast<T*>(a.out) + (size_t)r * a.out_stride)[e] = make_uint4(0u, 0u, 0u, 0u);
  __syncthreads();

  int row = sh_row;
  long long base = sh_base;
  const float scale = a.scale * 1.4426950408889634f;  // probabilities as powers of two
  for (long long u = u0; u < u1;) {
    int len = length(row), nt = tiles(len);
    while (u >= base + (long long)nt * items) {  // on to the next row that has units
      base += (long long)nt * items;
      ++row;
      len = length(row);
      nt = tiles(len);
    }
    const int item = (int)((u - base) / nt), t0 = (int)((u - base) % nt);
    const int t1 = (int)min((long long)nt, t0 + (u1 - u));
    const int kvh = item / blocks, h0 = kvh * group + (item % blocks) * kHeads;
    const int nheads = min(kHeads, group - (item % blocks) * kHeads);
    const int seq = a.seqs ? __ldg(a.seqs + row) : row;
    const bool seq_ok = seq >= 0 && seq < tab.rows;
    const int* ids = tab.ids + (seq_ok ? (size_t)seq * tab.stride : 0);
    const T* kp = static_cast<const T*>(pool.k) + (size_t)kvh * pool.head_stride;
    const T* vp = static_cast<const T*>(pool.v) + (size_t)kvh * pool.head_stride;

    uint4 q[NH][kB];
#pragma unroll
    for (int n = 0; n < NH; ++n)
#pragma unroll
      for (int b = 0; b < kB; ++b)
        q[n][b] = n * 8 + g < nheads ? *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + (size_t)row * a.q_stride +
                                                                       (size_t)(h0 + n * 8 + g) * D + 32 * b + 8 * j)
                                     : make_uint4(0u, 0u, 0u, 0u);
    float o[NH][kVB * 4][4];
    float m[NH][2], l[NH][2];
#pragma unroll
    for (int n = 0; n < NH; ++n) {
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
#pragma unroll
      for (int i = 0; i < kVB * 4; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
    }

    // the page of position p + lane (p: the first position of this warp's tiles), -1 for none
    auto look_up = [&](int p) {
      const int at = p + (lane & (16 * kU - 1));
      if (at >= len || !seq_ok || (at >> pool.page_shift) >= tab.width) return -1;
      const int page = __ldg(ids + (at >> pool.page_shift));
      return page < 0 || page >= pool.pages ? -1 : page;
    };
    const int tmask = (1 << pool.page_shift) - 1;
    auto place = [&](int page, int at) {  // element offset of position `at` of this kv head
      return (size_t)page * pool.page_stride + (size_t)(at & tmask) * pool.token_stride;
    };
    uint4 k[kU][kB][2], v[kU][kVB][4];
    auto load_k = [&](int p, int pages) {
#pragma unroll
      for (int t = 0; t < kU; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int i = 16 * t + 8 * h + g;
          const int page = __shfl_sync(0xffffffffu, pages, i);
          const T* src = kp + place(page, p + i) + 8 * j;
          const uint32_t none = p + i < len ? 0x7fff7fffu : 0u;  // a bad page: NaN
#pragma unroll
          for (int b = 0; b < kB; ++b) k[t][b][h] = page >= 0 ? ld_stream(src + 32 * b) : make_uint4(none, none, none, none);
        }
    };
    auto load_v = [&](int p, int pages) {
#pragma unroll
      for (int t = 0; t < kU; ++t)
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          const int i = 16 * t + 2 * j + (h & 1) + 8 * (h >> 1);
          const int page = __shfl_sync(0xffffffffu, pages, i);
          const T* src = vp + place(page, p + i) + 8 * g;
#pragma unroll
          for (int b = 0; b < kVB; ++b) v[t][b][h] = page >= 0 ? ld_stream(src + 64 * b) : make_uint4(0u, 0u, 0u, 0u);
        }
    };

    const int first = t0 * C::kUnit + warp * 16 * kU, end = min(len, t1 * C::kUnit);
    int pages = look_up(first);
    int pages_next = look_up(first + C::kUnit);
    load_k(first, pages);
    for (int p = first; p < end; p += C::kUnit) {
      load_v(p, pages);
      float s[NH][kU][4];
#pragma unroll
      for (int n = 0; n < NH; ++n)
#pragma unroll
        for (int t = 0; t < kU; ++t) {
          s[n][t][0] = s[n][t][1] = s[n][t][2] = s[n][t][3] = 0.f;
#pragma unroll
          for (int b = 0; b < kB; ++b) {
            mma16816<T>(s[n][t], k[t][b][0].x, k[t][b][1].x, k[t][b][0].y, k[t][b][1].y, q[n][b].x, q[n][b].y);
            mma16816<T>(s[n][t], k[t][b][0].z, k[t][b][1].z, k[t][b][0].w, k[t][b][1].w, q[n][b].z, q[n][b].w);
          }
        }
      pages = pages_next;
      if (p + C::kUnit < end) load_k(p + C::kUnit, pages);
      pages_next = look_up(p + 2 * C::kUnit);
#pragma unroll
      for (int n = 0; n < NH; ++n) {
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int t = 0; t < kU; ++t)
#pragma unroll
          for (int c = 0; c < 4; ++c) {  // c: head 2j + (c & 1), position g + 8 (c >> 1)
            s[n][t][c] = p + 16 * t + g + 8 * (c >> 1) < len ? s[n][t][c] * scale : -INFINITY;
            mx[c & 1] = fmaxf(mx[c & 1], s[n][t][c]);
          }
        float corr[2], low[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) mx[c] = fmaxf(mx[c], __shfl_xor_sync(0xffffffffu, mx[c], x));
          mx[c] = fmaxf(mx[c], m[n][c]);
          low[c] = mx[c] == -INFINITY ? 0.f : mx[c];
          corr[c] = exp2_fast(m[n][c] - low[c]);
          m[n][c] = mx[c];
          l[n][c] *= corr[c];
        }
#pragma unroll
        for (int i = 0; i < kVB * 4; ++i) {
          o[n][i][0] *= corr[0];
          o[n][i][1] *= corr[1];
          o[n][i][2] *= corr[0];
          o[n][i][3] *= corr[1];
        }
#pragma unroll
        for (int t = 0; t < kU; ++t) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            s[n][t][c] = exp2_fast(s[n][t][c] - low[c & 1]);
            l[n][c & 1] += s[n][t][c];
          }
          // rounded to 16 bits for the product with V; the sum l keeps fp32
          const uint32_t b0 = transpose_8x8(pack2<T>(s[n][t][0], s[n][t][1]));
          const uint32_t b1 = transpose_8x8(pack2<T>(s[n][t][2], s[n][t][3]));
#pragma unroll
          for (int b = 0; b < kVB; ++b) {
            const uint32_t w[4][4] = {{v[t][b][0].x, v[t][b][0].y, v[t][b][0].z, v[t][b][0].w},
                                      {v[t][b][1].x, v[t][b][1].y, v[t][b][1].z, v[t][b][1].w},
                                      {v[t][b][2].x, v[t][b][2].y, v[t][b][2].z, v[t][b][2].w},
                                      {v[t][b][3].x, v[t][b][3].y, v[t][b][3].z, v[t][b][3].w}};
#pragma unroll
            for (int i = 0; i < 4; ++i)
              mma16816<T>(o[n][b * 4 + i], prmt(w[0][i], w[1][i], 0x5410u), prmt(w[0][i], w[1][i], 0x7632u),
                          prmt(w[2][i], w[3][i], 0x5410u), prmt(w[2][i], w[3][i], 0x7632u), b0, b1);
          }
        }
      }
    }

    // the warps' parts, joined in shared memory
#pragma unroll
    for (int n = 0; n < NH; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], x);
        const int head = 8 * n + 2 * j + c;
        if (g == 0) {
          sh_m[warp][head] = m[n][c];
          sh_l[warp][head] = l[n][c];
        }
#pragma unroll
        for (int b = 0; b < kVB; ++b) {
          float4* dst = reinterpret_cast<float4*>(sh_o + ((size_t)warp * kHeads + head) * D + 64 * b + 8 * g);
          dst[0] = make_float4(o[n][4 * b][c], o[n][4 * b][2 + c], o[n][4 * b + 1][c], o[n][4 * b + 1][2 + c]);
          dst[1] = make_float4(o[n][4 * b + 2][c], o[n][4 * b + 2][2 + c], o[n][4 * b + 3][c], o[n][4 * b + 3][2 + c]);
        }
      }
    __syncthreads();
    const bool whole = t0 == 0 && t1 == nt;
    float* slot = slots + (size_t)(2 * worker + (t0 == 0 ? 1 : 0)) * C::kSlot;
    for (int e = threadIdx.x; e < nheads * (D / 4); e += kThreads) {
      const int head = e / (D / 4), d = (e % (D / 4)) * 4;
      float mm = sh_m[0][head], ll = 0.f;
#pragma unroll
      for (int w = 1; w < kAttnWarps; ++w) mm = fmaxf(mm, sh_m[w][head]);
      const float low = mm == -INFINITY ? 0.f : mm;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kAttnWarps; ++w) {
        const float f = exp2_fast(sh_m[w][head] - low);
        const float4 x = *reinterpret_cast<const float4*>(sh_o + ((size_t)w * kHeads + head) * D + d);
        ll = fmaf(sh_l[w][head], f, ll);
        acc.x = fmaf(x.x, f, acc.x);
        acc.y = fmaf(x.y, f, acc.y);
        acc.z = fmaf(x.z, f, acc.z);
        acc.w = fmaf(x.w, f, acc.w);
      }
      if (whole) {
        uint2 r;
        r.x = pack2<T>(acc.x / ll, acc.y / ll);
        r.y = pack2<T>(acc.z / ll, acc.w / ll);
        *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + (size_t)row * a.out_stride + (size_t)(h0 + head) * D + d) = r;
      } else {
        *reinterpret_cast<float4*>(slot + 2 * kHeads + head * D + d) = acc;
        if (d == 0) {
          slot[head] = mm;
          slot[kHeads + head] = ll;
        }
      }
    }
    if (!whole && t0 == 0 && threadIdx.x == 0) {
      const long long last = base + (long long)(item + 1) * nt - 1;  // the item's last unit
      desc[worker].row = row;
      desc[worker].item = item;
      desc[worker].parts = (int)(((last + 1) * used - 1) / total) - worker + 1;
    }
    __syncthreads();  // shared memory is free for the next item
    u += t1 - t0;
  }
}

// Joins the parts of the item that worker blockIdx.x began, in the workers' order.
template <typename T, int D, int NH>
__global__ void __launch_bounds__(8 * NH * D / 4) k_paged_join(const PagedAttention a, const int group, const int blocks) {
  using C = AttnCfg<D, NH>;
  grid_dependency_wait();
  const AttnDesc* desc = static_cast<const AttnDesc*>(a.workspace);
  const float* slots = reinterpret_cast<const float*>(desc + kAttnMaxWorkers);
  const AttnDesc it = desc[blockIdx.x];
  const int head = threadIdx.x / (D / 4), d = (threadIdx.x % (D / 4)) * 4;
  const int nheads = min(C::kHeads, group - (it.item % blocks) * C::kHeads);
  if (it.parts == 0 || head >= nheads) return;
  const float* mine = slots + (size_t)(2 * blockIdx.x + 1) * C::kSlot;
  float mm = mine[head], ll = mine[C::kHeads + head];
  float4 acc = *reinterpret_cast<const float4*>(mine + 2 * C::kHeads + head * D + d);
#pragma unroll 4
  for (int i = 1; i < it.parts; ++i) {
    const float* part = slots + (size_t)(2 * (blockIdx.x + i)) * C::kSlot;
    const float pm = part[head], pl = part[C::kHeads + head];
    const float4 x = *reinterpret_cast<const float4*>(part + 2 * C::kHeads + head * D + d);
    const float mx = fmaxf(mm, pm), low = mx == -INFINITY ? 0.f : mx;
    const float f = exp2_fast(mm - low), pf = exp2_fast(pm - low);
    mm = mx;
    ll = ll * f + pl * pf;
    acc.x = acc.x * f + x.x * pf;
    acc.y = acc.y * f + x.y * pf;
    acc.z = acc.z * f + x.z * pf;
    acc.w = acc.w * f + x.w * pf;
  }
  uint2 r;
  r.x = pack2<T>(acc.x / ll, acc.y / ll);
  r.y = pack2<T>(acc.z / ll, acc.w / ll);
  const int h = it.item / blocks * group + it.item % blocks * C::kHeads + head;
  *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + (size_t)it.row * a.out_stride + (size_t)h * D + d) = r;
}

template <typename F>
int by_type(int dtype, int head_dim, F&& f) {
  if (dtype == W4A16_DTYPE_F16) {
    if (head_dim == 64) return f(__half(), std::integral_constant<int, 64>());
    if (head_dim == 128) return f(__half(), std::integral_constant<int, 128>());
    return f(__half(), std::integral_constant<int, 256>());
  }
  if (head_dim == 64) return f(__nv_bfloat16(), std::integral_constant<int, 64>());
  if (head_dim == 128) return f(__nv_bfloat16(), std::integral_constant<int, 128>());
  return f(__nv_bfloat16(), std::integral_constant<int, 256>());
}

int launched(const char* what, cudaError_t e) {
  (void)cudaGetLastError();
  if (e == cudaSuccess) return W4A16_OK;
  set_error("%s launch failed: %s", what, cudaGetErrorString(e));
  return W4A16_ERR_CUDA;
}

}  // namespace

int launch_paged_append(const PagedAppend& a, const PagedPool& pool, const PagedTables& tab, cudaStream_t stream) {
  int sms = 0;
  const int rc = current_sm_count(&sms);
  if (rc != W4A16_OK) return rc;
  return by_type(pool.dtype, pool.head_dim, [&](auto t, auto d) {
    using T = decltype(t);
    constexpr int D = decltype(d)::value;
    const long long total = (long long)a.tokens * (a.heads + 2 * pool.kv_heads) * (D / 16);
    const long long blocks = (total + 255) / 256, most = (long long)sms * 8;
    k_paged_append<T, D><<<(unsigned)(blocks < most ? blocks : most), 256, 0, stream>>>(a, pool, tab);
    return launched("k_paged_append", cudaGetLastError());
  });
}

namespace {

// Query heads of a CTA: up to 16 of a kv head's group; 8 with head_dim 256, whose operands
// fill the registers.
bool attn_wide(int group, int head_dim) { return group > 8 && head_dim <= 128; }

template <typename T, int D, int NH>
int launch_attention(const PagedAttention& a, const PagedPool& pool, const PagedTables& tab, cudaStream_t stream) {
  using C = AttnCfg<D, NH>;
  int sms = 0;
  const int rc = current_sm_count(&sms);
  if (rc != W4A16_OK) return rc;
  const int group = a.heads / pool.kv_heads, blocks = (group + C::kHeads - 1) / C::kHeads;
  const int workers = sms * C::kPerSm < kAttnMaxWorkers ? sms * C::kPerSm : kAttnMaxWorkers;
  constexpr size_t smem = (size_t)kAttnWarps * C::kHeads * D * 4;
  static_assert(smem <= 40960, "with the static arrays under the 48 KB that need no opt-in");
  k_paged_attention<T, D, NH><<<workers, kAttnWarps * 32, smem, stream>>>(a, pool, tab, group, blocks);
  const int rc2 = launched("k_paged_attention", cudaGetLastError());
  if (rc2 != W4A16_OK) return rc2;
  return launched("k_paged_join", launch_maybe_pdl(k_paged_join<T, D, NH>, dim3(workers), dim3(C::kHeads * D / 4), 0, stream, true, a,
                                                   group, blocks));
}

}  // namespace

size_t paged_attention_workspace_bytes(int heads, int kv_heads, int head_dim) {
  const size_t h = attn_wide(heads / kv_heads, head_dim) ? 16 : 8;
  return (size_t)kAttnMaxWorkers * (sizeof(AttnDesc) + 2 * h * (head_dim + 2) * 4);
}

int launch_paged_attention(const PagedAttention& a, const PagedPool& pool, const PagedTables& tab, cudaStream_t stream) {
  const bool wide = attn_wide(a.heads / pool.kv_heads, pool.head_dim);
  return by_type(pool.dtype, pool.head_dim, [&](auto t, auto d) {
    using T = decltype(t);
    constexpr int D = decltype(d)::value;
    if constexpr (D <= 128) {
      if (wide) return launch_attention<T, D, 2>(a, pool, tab, stream);
    }
    return launch_attention<T, D, 1>(a, pool, tab, stream);
  });
}

}  // namespace w4a16
