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
//
// Every kernel here is launched with programmatic stream serialisation: its CTAs may be placed
// while the kernel before it in the stream ends, and wait for that one before they read or
// write anything.  What that kernel may have written is read by ordinary loads through pointers
// without __restrict__ (fetch says why).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <type_traits>

#include "w4a16_device.cuh"
#include "w4a16_internal.h"

namespace w4a16 {

namespace {

// The page that holds position p of sequence s, or -1 (bad sequence, position or entry).
__device__ __forceinline__ int page_of(const PagedTables& t, int s, int p, int page_shift, int pages) {
  if (s < 0 || s >= t.rows || p < 0 || (p >> page_shift) >= t.width) return -1;
  const int page = fetch(t.ids + (size_t)s * t.stride + (p >> page_shift));
  return page < 0 || page >= pages ? -1 : page;
}

// ---------------------------------------------------------------------------- append
//
// Bound by the bytes of q, k and v, read once and written once.  A CTA takes a token at a time;
// a thread turns 8 pairs (i, i + D/2) of every 16th head with the angles of its pairs in
// registers, kBatch heads' loads in flight before the token's position and page are known
// (16384 tokens of 32 + 16 heads of 128: 65 us, 0.96 of the copy rate).
template <int D>
constexpr int append_threads() { return 16 * (D / 16); }

template <typename T, int D>
__global__ void __launch_bounds__(append_threads<D>(), 1024 / append_threads<D>())
    k_paged_append(const PagedAppend a, const PagedPool pool, const PagedTables tab) {
  constexpr int kChunks = D / 16, kBatch = 2;
  grid_dependency_wait();
  grid_launch_dependents();
  const int slot = threadIdx.x / kChunks, i = threadIdx.x % kChunks * 8;
  const int keys = a.heads, values = a.heads + pool.kv_heads, all = values + pool.kv_heads;  // heads in the order q, k, v
  for (int t = blockIdx.x; t < a.tokens; t += gridDim.x) {
    const int pos = fetch(a.positions + t);
    const int seq = a.seqs ? fetch(a.seqs + t) : t;
    const T* q = static_cast<const T*>(a.q) + (size_t)t * a.q_stride + i;
    const T* k = static_cast<const T*>(a.k) + (size_t)t * a.k_stride + i;
    const T* v = static_cast<const T*>(a.v) + (size_t)t * a.v_stride + i;
    int page = -1;
    float4 cs[8];  // cos, sin of the pairs' first halves, then of their second
    size_t place = 0;
    for (int h0 = 0; h0 < all; h0 += 16 * kBatch) {
      uint4 lo[kBatch], hi[kBatch];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const int h = h0 + 16 * b + slot;
        if (h >= all) continue;
        const T* src = h < keys ? q + (size_t)h * D : h < values ? k + (size_t)(h - keys) * D : v + (size_t)(h - values) * D;
        lo[b] = *reinterpret_cast<const uint4*>(src);
        hi[b] = *reinterpret_cast<const uint4*>(src + D / 2);
      }
      if (h0 == 0) {
        page = pos < 0 || (a.cos_t && pos >= a.angle_rows) ? -1 : page_of(tab, seq, pos, pool.page_shift, pool.pages);
        if (page >= 0) {
          place = (size_t)page * pool.page_stride + (size_t)(pos & ((1 << pool.page_shift) - 1)) * pool.token_stride + i;
          if (a.cos_t) {
            const float4* c = reinterpret_cast<const float4*>(a.cos_t + (size_t)pos * D + i);
            const float4* s = reinterpret_cast<const float4*>(a.sin_t + (size_t)pos * D + i);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              cs[e] = fetch(c + e);
              cs[2 + e] = fetch(s + e);
              cs[4 + e] = fetch(c + D / 8 + e);
              cs[6 + e] = fetch(s + D / 8 + e);
            }
          }
        }
      }
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const int h = h0 + 16 * b + slot;
        if (h >= all || (page < 0 && h >= keys)) continue;
        if (page < 0) {  // padding: zeros; a bad position, sequence or page: NaN
          const uint32_t w = pos < 0 ? 0u : pack2<T>(__int_as_float(0x7fc00000), __int_as_float(0x7fc00000));
          lo[b] = hi[b] = make_uint4(w, w, w, w);
        } else if (a.cos_t && h < values) {
          uint32_t* l = reinterpret_cast<uint32_t*>(&lo[b]);
          uint32_t* u = reinterpret_cast<uint32_t*>(&hi[b]);
          const float2* c = reinterpret_cast<const float2*>(cs);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 x = unpack2<T>(l[e]), y = unpack2<T>(u[e]);
            const float2 c0 = c[e], s0 = c[4 + e], c1 = c[8 + e], s1 = c[12 + e];
            l[e] = pack2<T>(x.x * c0.x - y.x * s0.x, x.y * c0.y - y.y * s0.y);
            u[e] = pack2<T>(y.x * c1.x + x.x * s1.x, y.y * c1.y + x.y * s1.y);
          }
        }
        T* dst = h < keys     ? static_cast<T*>(a.q_out) + (size_t)t * a.q_out_stride + (size_t)h * D + i
                 : h < values ? static_cast<T*>(pool.k) + place + (size_t)(h - keys) * pool.head_stride
                              : static_cast<T*>(pool.v) + place + (size_t)(h - values) * pool.head_stride;
        *reinterpret_cast<uint4*>(dst) = lo[b];
        *reinterpret_cast<uint4*>(dst + D / 2) = hi[b];
      }
    }
  }
}

// ------------------------------------------------------------------------- attention
//
// Bound by the bytes of the keys and values: each is used for the few query heads of its kv
// head only.  One pass over them with a running maximum and sum.  Every warp copies its own
// tiles of 16 (head_dim 64: 32) positions into its own ring of shared memory stages with
// 16-byte asynchronous copies, so no barrier and no register holds bytes in flight, and reads
// the operands of m16n8k16 tensor-core products with 16-byte shared loads, which the freedom
// to number the contracted index allows:
//   S^T[position][head] = K Q^T    A = K: lane (g = lane / 4, j = lane % 4) reads 16 bytes of
//                                  positions g and g + 8 at dimensions 8j of each block of 32;
//                                  these four words are the k = 2j, 2j+1, 2j+8, 2j+9 operands
//                                  of two products, and Q is loaded by the same numbering
//   O^T[dimension][head] = V^T P   A = V^T: the lane reads 16 bytes (dimensions 8g) of positions
//                                  2j, 2j+1, 2j+8, 2j+9 and pairs two positions with one byte
//                                  permutation per word; P^T comes from S^T by 8 x 8 matrix
//                                  transpositions, in two 16-bit parts (value and remainder) of
//                                  kProb times the probability: fp16's 11 bits leave 2^-23 of it,
//                                  bf16's 8 leave 2^-17, 2^-8 of the rounding of the result.  (With
//                                  a third part for bf16 one value in 2000 was not the nearest bf16,
//                                  with two one in 900, of 2 rows of up to 120001; it took 1% more
//                                  time there and 5% with 16 heads, 64 rows of up to 2000.)
// A tile's part of O starts from zero and is added to the running sum by an ordinary addition: the
// products' own additions cut off what is below the sum's last bit, always towards zero (values of
// 1 over 262144 positions in a warp gave 0.9985 as one long sum; 16 heads of a CTA pay 3% for the
// additions, 64 rows of up to 2000 with 8 kv heads of 128 65.5 us for 63.7, 8 heads under 1%).
// The 16-byte chunks of a row are permuted by swizzle(row), which keeps both reads free of
// bank conflicts.  The 8 (NH = 1) or 16 (NH = 2) query heads of a CTA are the n of the products.
//
// Work is shared out by a count of units over all (row, kv head, block of query heads) items, in
// that order: each worker takes an equal run of them, wherever that cuts an item.  With an item
// for every warp of the grid a worker is a warp and a unit one stage of positions, so the warps
// run without a barrier; with fewer, which warps would cut into many parts, a worker is a CTA,
// a unit one stage of each warp, and the CTA joins its warps' parts itself (256 rows of up to
// 200 positions, 2048 items: 31 us by warps, 36 by CTAs; 32 rows of up to 4096, 256 items: 54
// and 50).  The lengths are read on the device, so every CTA first sums them up.  An item that
// lies within one worker is finished there; the parts of one that was cut go to the workspace
// (slot 2w + 1 if the part begins the item, else 2w) and are joined by k_paged_join.  Calls of few
// rows go another way (kClusterMax).
//
// Measured: 72 rows of up to 8191 positions, 8 kv heads of 128: 168 us, 0.98 of the copy rate;
// 32 rows of up to 4096: 50 us, 0.85, of which about 7 us are the two launches and the way to
// the first key (lengths, table, page) that a single short row takes as well.
constexpr int kAttnWarps = 4;
constexpr int kAttnMaxSms = 148;  // bounds the workspace
// What it costs to begin and end an item, in units of a warp's and of a CTA's work (256 rows of
// up to 200 positions: 31 us with it, 36 without; 32 rows of up to 4096: 50 and 52).
constexpr int kItemCost = 2, kItemCostCta = 1;
// Workers for each item at most: more cost more to join than they save (one sequence of 30000
// positions with one kv head of 64: 9.4 us with 128, 10.6 with 64 or 256).
constexpr int kMaxParts = 128;
// Calls of few rows in short tables: a cluster of CTAs takes one item (the kernel's kCluster form),
// each warp every (4 * cluster)-th stage of it, and joins its warps' parts through distributed shared
// memory, without a look at the other rows, parts in the workspace or a second launch.  A cluster
// has up to 8 CTAs: as many as the device runs at once, and as have 128 positions of a full table
// row each.  It is not for rows longer than cluster_most() for each CTA, where equal shares for all SMs win.
// (32 query heads over 8 kv heads.  head_dim 64: 1 row of 512 positions 4.2 us, cut into parts 7.6; of
// 4096 7.5 and 8.4; of 8192 11.5 and 9.9.  head_dim 128: 16 rows of 64 4.1 and 8.3; 8 rows of 512 7.2
// and 9.7; 1 row of 4096 11.8 and 9.8, 4 rows, whose clusters fill the device, 18.0 and 20.1.)
// In tables of up to kTwiceMost positions CTAs of an item each are faster even if only half of them
// fit at once (8 kv heads: 60 rows of up to 30 positions 7.6 and 10.1, of up to 200 9.4 and 10.8; 74
// rows of exactly 256 with head_dim 128 are the exception, 20.7 and 19.4).
constexpr int kClusterMax = 8, kClusterLeast = 128, kTwiceMost = 256;
constexpr int cluster_most(int head_dim, int nh, bool fill) {
  const int n = 32768 / (head_dim * nh) * (fill ? 2 : 1);
  return n < 512 ? n : 512;
}
// CTAs of an SM.  head_dim 64 has more to compute for a byte and wants more warps, with two
// stages each (64 rows of up to 8000 positions: 86 us with 3 CTAs of 2 stages, 94 with 2 of 3).
constexpr int attn_per_sm(int head_dim) { return head_dim == 64 ? 3 : head_dim == 128 ? 2 : 1; }

// What the probabilities, their sums and the products with V carry until the last division.  fp16's
// smallest step is 2^-24: a probability as it is would lose what lies below 2^-25 of the warp's largest one,
// with 2^14 (the largest is 2^14, of 65504) what lies below 2^-39.  bf16 has fp32's exponents.
template <typename T>
constexpr float kProb = std::is_same<T, __half>::value ? 16384.f : 1.f;

template <int D, int NH>
struct AttnCfg {
  static constexpr int kTiles = D == 64 ? 2 : 1;  // 16-position tiles of a stage
  static constexpr int kPos = 16 * kTiles;        // positions of a stage
  static constexpr int kHeads = 8 * NH;
  static constexpr int kStages = D == 64 ? 2 : 3;
  static constexpr int kPerSm = NH == 2 && D == 64 ? 2 : attn_per_sm(D);  // 16 heads take more registers
  static constexpr int kMaxWorkers = kAttnMaxSms * attn_per_sm(D) * kAttnWarps;
  static constexpr int kSlot = kHeads * (D + 2);  // floats of a part: m, l, o per head
  static constexpr int kHalf = kPos * D * 2;      // bytes of a stage's keys, and of its values
  static constexpr int kRing = kStages * 2 * kHalf;  // bytes of a warp's ring
  static constexpr int kSmem = kAttnWarps * (kRing + 8 * D * 4);  // the rings, then the warps' parts of 8 heads
};

// An item cut into parts (parts 0: none): at the place of the worker that began it, or in calls of
// few items (by_item) at the item's own.
struct __align__(16) AttnDesc {
  int row, item, parts, first;  // first: the worker that began it
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

// 16 bytes to shared memory, past L1 (they are read once); zeros where `any` is false.
__device__ __forceinline__ void copy_async16(uint32_t dst, const void* src, bool any) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(any ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Permutation of a row's 16-byte chunks within 128 bytes.  Rows 2i differ in bits 1 and 2 (the
// reads of V take rows 0, 2, 4, 6 or 1, 3, 5, 7 at two neighbouring chunks), rows 2i and 2i + 1
// in bit 2 (the reads of K take two neighbouring rows at four neighbouring chunks).
__device__ __forceinline__ int swizzle(int row) { return (row & 7) ^ ((row & 1) << 2); }

// a / b for 0 <= a, 0 < b: 64-bit divisions are several times slower than 32-bit ones.
__device__ __forceinline__ long long divide(long long a, long long b) {
  return (a | b) >> 32 ? a / b : (long long)((uint32_t)a / (uint32_t)b);
}

template <typename T, int D, int NH, bool kCluster>
__global__ void __launch_bounds__(kAttnWarps * 32, AttnCfg<D, NH>::kPerSm)
    k_paged_attention(const PagedAttention a, const PagedPool pool, const PagedTables tab, const int group, const int blocks,
                      const bool coop, const int cost, const int cluster,
                      const bool by_item) {
  using C = AttnCfg<D, NH>;
  constexpr int kB = D / 32, kVB = D / 64, kU = C::kTiles, kHeads = C::kHeads, kThreads = kAttnWarps * 32, kPos = C::kPos;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, j = lane & 3;
  const int rank = blockIdx.x & (cluster - 1);
  const int workers = coop ? gridDim.x : gridDim.x * kAttnWarps;
  const int worker = coop ? blockIdx.x : blockIdx.x * kAttnWarps + warp;
  // positions of a unit, and where this warp's stage of them lies
  const int unit = kCluster ? kPos * kAttnWarps * cluster : coop ? kPos * kAttnWarps : kPos;
  const int shift = kCluster ? (rank * kAttnWarps + warp) * kPos : coop ? warp * kPos : 0;
  const int items = pool.kv_heads * blocks;
  const float nan = __int_as_float(0x7fc00000);
  __shared__ long long sh_base[kAttnWarps], sh_warp[kAttnWarps];
  __shared__ int sh_row[kAttnWarps];
  __shared__ float sh_m[kAttnWarps][8], sh_l[kAttnWarps][8];
  extern __shared__ __align__(128) uint8_t sh_raw[];
  const uint32_t ring = smem_addr(sh_raw) + warp * C::kRing;
  float* sh_o = reinterpret_cast<float*>(sh_raw + kAttnWarps * C::kRing);  // [warp][8][D]

  grid_dependency_wait();    // launched early; nothing is read before this
  grid_launch_dependents();  // the join waits for this kernel's end in turn
  AttnDesc* desc = static_cast<AttnDesc*>(a.workspace);
  float* slots = reinterpret_cast<float*>(desc + C::kMaxWorkers);
  const long long cap = (long long)tab.width << pool.page_shift;
  // a length past the tables keeps one position there, which has no page: NaN
  auto length = [&](int row) {
    const int n = fetch(a.lengths + row);
    return n <= 0 ? 0 : n > cap ? (int)(cap + 1) : n;
  };
  // An item's units: those of its positions, then cost more that stand for what it takes to begin
  // and end one
  auto tiles = [&](int len) { return len == 0 ? 0 : (len + unit - 1) / unit + cost; };

  // A span: the tiles [t0, t1) of one item that the worker takes in a row.
  struct Span {
    int row, len, nt, item, t0, t1;
  };
  Span cur;
  long long u0, u1, each = 0;  // this worker's units; units of a worker
  int more = 0, first_page = -2;
  if constexpr (kCluster) {  // one item
    const int at = blockIdx.x / cluster;
    cur.row = at / items;
    cur.item = at - cur.row * items;
    // the sequence's first pages are looked up while its length is on its way
    const int seq = a.seqs ? fetch(a.seqs + cur.row) : cur.row, col = (shift + (lane & (kPos - 1))) >> pool.page_shift;
    cur.len = length(cur.row);
    if (seq >= 0 && seq < tab.rows && col < tab.width) first_page = fetch(tab.ids + (size_t)seq * tab.stride + col);
    cur.nt = tiles(cur.len);
    cur.t0 = 0;
    cur.t1 = cur.nt;
    u0 = 0;
    u1 = cur.nt;
    if (cur.len == 0) {  // a row of no positions is zero
      const int h0 = cur.item / blocks * group + cur.item % blocks * kHeads, n = min(kHeads, group - cur.item % blocks * kHeads) * D / 8;
      for (int e = rank * kThreads + threadIdx.x; e < n; e += kThreads * cluster)
        reinterpret_cast<uint4*>(static_cast<T*>(a.out) + (size_t)cur.row * a.out_stride + (size_t)h0 * D)[e] = make_uint4(0u, 0u, 0u, 0u);
      __syncwarp();
      cluster_sync_all();  // the join's two, though no CTA of this cluster gets there: each takes every barrier, whatever
      cluster_sync_all();  // length it read
      return;
    }
  } else {
    // the units of all rows, and the row that holds each worker's first one
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
    __syncthreads();
    long long before = inc - sum, total = 0;
    for (int w = 0; w < kAttnWarps; ++w) {
      if (w < warp) before += sh_warp[w];
      total += sh_warp[w];
    }
    // every worker in use has a unit, so the parts of an item lie with consecutive workers: the
    // first `more` of them take each + 1 units, the others each
    const long long most = min((long long)workers, (long long)a.rows * items * kMaxParts);
    const int used = (int)min(total, most);
    each = used ? divide(total, used) : 0;
    more = (int)(total - each * used);
    auto first_unit = [&](int w) { return w < used ? w * each + min(w, more) : total; };
    for (int w = 0; w < (coop ? 1 : kAttnWarps); ++w) {
      const long long u = first_unit(coop ? blockIdx.x : blockIdx.x * kAttnWarps + w);
      if (u < total && before <= u && u < before + sum) {  // one thread
        long long base = before;
        int r = r0;
        for (;; ++r) {
          const long long n = (long long)tiles(length(r)) * items;
          if (u < base + n) break;
          base += n;
        }
        sh_row[w] = r;
        sh_base[w] = base;
      }
    }
    if (!by_item && (coop ? threadIdx.x == 0 : lane == 0)) desc[worker].parts = 0;
    // rows of no positions are zero
    for (int r = blockIdx.x; r < a.rows; r += gridDim.x)
      if (length(r) == 0) {
        for (int e = threadIdx.x; e < a.heads * D / 8; e += kThreads)
          reinterpret_cast<uint4*>(static_cast<T*>(a.out) + (size_t)r * a.out_stride)[e] = make_uint4(0u, 0u, 0u, 0u);
        if (by_item)
          for (int e = threadIdx.x; e < items; e += kThreads) desc[r * items + e].parts = 0;
      }
    __syncthreads();
    u0 = first_unit(worker);
    u1 = worker + 1 < used ? first_unit(worker + 1) : total;
    if (u0 >= u1) return;  // the whole CTA if it works as one
    const long long base = sh_base[coop ? 0 : warp];  // units before the row of cur
    cur.row = sh_row[coop ? 0 : warp];
    cur.len = length(cur.row);
    cur.nt = tiles(cur.len);
    cur.item = (int)divide(u0 - base, cur.nt);
    cur.t0 = (int)(u0 - base - (long long)cur.item * cur.nt);
    cur.t1 = (int)min((long long)cur.nt, cur.t0 + (u1 - u0));
  }
  const float scale = a.scale * 1.4426950408889634f;  // probabilities as powers of two

  auto next_span = [&](Span& sp, long long u) {  // the span that begins at unit u < u1, where sp ends
    sp.t0 = 0;
    if (++sp.item == items) {
      sp.item = 0;
      do sp.len = length(++sp.row);
      while (sp.len == 0);
      sp.nt = tiles(sp.len);
    }
    sp.t1 = (int)min((long long)sp.nt, u1 - u);
  };

  // Copies run kStages - 1 units ahead of the products, across items, and the page numbers one
  // unit ahead of the copies.
  Span ahead = cur;
  long long ahead_u = u0;
  int ahead_t = ahead.t0, pos = 0, page = -1, ahead_len = 0;  // pos, page, ahead_len, head_off: of the unit to be copied next
  size_t head_off = 0;
  const int* ids = tab.ids;
  bool seq_ok = false;
  auto enter = [&]() {
    const int seq = a.seqs ? fetch(a.seqs + ahead.row) : ahead.row;
    seq_ok = seq >= 0 && seq < tab.rows;
    ids = tab.ids + (seq_ok ? (size_t)seq * tab.stride : 0);
    head_off = (size_t)(ahead.item / blocks) * pool.head_stride;
  };
  // page of position pos + lane: -1 for none, -2 where a position has none and should
  auto look_up = [&]() {
    page = -1;
    while (ahead_t >= min(ahead.t1, ahead.nt - cost)) {  // the span's positions are done
      ahead_u += ahead.t1 - ahead.t0;
      if (ahead_u >= u1) {
        ahead.t0 = ahead.t1;  // stay here
        pos = ahead_len;      // a stage without positions
        return;
      }
      next_span(ahead, ahead_u);
      ahead_t = 0;
      enter();
    }
    pos = ahead_t * unit + shift;
    ahead_len = ahead.len;
    const int at = pos + (lane & (kPos - 1));
    if (at < ahead.len) {
      if (kCluster && ahead_t == 0)
        page = first_page;
      else if (seq_ok && (at >> pool.page_shift) < tab.width)
        page = fetch(ids + (at >> pool.page_shift));
      if (page < 0 || page >= pool.pages) page = -2;
    }
    ++ahead_t;
  };
  const int tmask = (1 << pool.page_shift) - 1;
  constexpr int kChunks = D / 8, kRows = 32 / kChunks;  // 16-byte chunks of a row; rows of one copy instruction
  const int crow = lane / kChunks, chunk = lane % kChunks;
  const size_t row_step = (size_t)kRows * pool.token_stride;
  const bool tight = pool.token_stride == D;  // a page's rows of one head one after the other: constant steps
  const T* k_chunk = static_cast<const T*>(pool.k) + (size_t)crow * pool.token_stride + 8 * chunk;
  const T* v_chunk = static_cast<const T*>(pool.v) + (size_t)crow * pool.token_stride + 8 * chunk;
  unsigned bad = 0;  // bit: the stage holds a position without a page
  auto load = [&](int stage) {
    const uint32_t dst = ring + stage * 2 * C::kHalf;
    bad = (bad & ~(1u << stage)) | (page == -2 ? 1u << stage : 0u);
    if (pos >= ahead_len) {  // a unit without positions for this warp (and without a bad page)
      copies_commit();
      return;
    }
    const uint32_t here = dst + crow * (D * 2) + (chunk & ~7) * 16;
    auto to = [&](int r0) {  // where this lane's chunk of row r0 + crow goes (r0 a multiple of kRows)
      return here + r0 * (D * 2) + (((chunk & 7) ^ swizzle(r0 + crow)) * 16);
    };
    if (pool.page_shift >= 4) {  // the 16 positions of a tile lie in one page
#pragma unroll
      for (int t = 0; t < kU; ++t) {
        const int pg = __shfl_sync(0xffffffffu, page, 16 * t), p0 = pos + 16 * t;
        const size_t at = (size_t)(pg < 0 ? 0 : pg) * pool.page_stride + (size_t)(p0 & tmask) * pool.token_stride + head_off;
        const T* ks = k_chunk + at;
        const T* vs = v_chunk + at;
        if (pg >= 0 && p0 + 16 <= ahead_len) {  // all tiles but a sequence's last
          if (tight) {
#pragma unroll
            for (int i = 0; i < 16; i += kRows) {
              copy_async16(to(16 * t + i), ks + i * D);
              copy_async16(to(16 * t + i) + C::kHalf, vs + i * D);
            }
          } else {
#pragma unroll
            for (int i = 0; i < 16; i += kRows) {
              copy_async16(to(16 * t + i), ks);
              copy_async16(to(16 * t + i) + C::kHalf, vs);
              ks += row_step;
              vs += row_step;
            }
          }
        } else {
#pragma unroll 1
          for (int i = 0; i < 16; i += kRows) {
            const bool any = pg >= 0 && p0 + i + crow < ahead_len;
            copy_async16(to(16 * t + i), ks, any);
            copy_async16(to(16 * t + i) + C::kHalf, vs, any);
            ks += row_step;
            vs += row_step;
          }
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < kPos; i += kRows) {
        const int r = i + crow;
        const int pg = __shfl_sync(0xffffffffu, page, r);
        const size_t at = (size_t)(pg < 0 ? 0 : pg) * pool.page_stride + (size_t)((pos + r) & tmask) * pool.token_stride -
                          (size_t)crow * pool.token_stride + head_off;
        copy_async16(to(i), k_chunk + at, pg >= 0);
        copy_async16(to(i) + C::kHalf, v_chunk + at, pg >= 0);
      }
    }
    copies_commit();
  };
  enter();
  look_up();
#pragma unroll
  for (int i = 0; i < C::kStages - 1; ++i) {  // units past the last are copied as zeros
    load(i);
    look_up();
  }
  uint4 q[NH][kB];
  auto load_q = [&](const Span& sp) {
    const int h0 = sp.item / blocks * group + sp.item % blocks * kHeads, nheads = min(kHeads, group - sp.item % blocks * kHeads);
    const T* src = static_cast<const T*>(a.q) + (size_t)sp.row * a.q_stride + (size_t)(h0 + g) * D + 8 * j;
#pragma unroll
    for (int n = 0; n < NH; ++n)
#pragma unroll
      for (int b = 0; b < kB; ++b)
        q[n][b] = n * 8 + g < nheads ? *reinterpret_cast<const uint4*>(src + n * 8 * D + 32 * b) : make_uint4(0u, 0u, 0u, 0u);
  };
  load_q(cur);
  int stage = 0;
  for (long long u = u0;;) {
    const int row = cur.row, item = cur.item, t0 = cur.t0, t1 = cur.t1, len = cur.len, nt = cur.nt;
    const int kvh = item / blocks, h0 = kvh * group + (item % blocks) * kHeads;
    const int nheads = min(kHeads, group - (item % blocks) * kHeads);

    float o[NH][kVB * 4][4];
    float m[NH][2], l[NH][2];
#pragma unroll
    for (int n = 0; n < NH; ++n) {
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
#pragma unroll
      for (int i = 0; i < kVB * 4; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
    }

    bool no_page = false;
    for (int tile = t0; tile < min(t1, nt - cost); ++tile) {
      copies_wait<C::kStages - 2>();
      __syncwarp();  // every lane's copies of this stage are in, its reads of the one before done
      load(stage == 0 ? C::kStages - 1 : stage - 1);
      look_up();
      no_page |= (bad >> stage & 1u) != 0;
      const uint32_t kt = ring + stage * 2 * C::kHalf, vt = kt + C::kHalf;
      stage = stage == C::kStages - 1 ? 0 : stage + 1;
      const int p = tile * unit + shift;
      if (p >= len) continue;  // the item's last unit may leave this warp none
      float s[NH][kU][4];
#pragma unroll
      for (int t = 0; t < kU; ++t) {
#pragma unroll
        for (int n = 0; n < NH; ++n) s[n][t][0] = s[n][t][1] = s[n][t][2] = s[n][t][3] = 0.f;
#pragma unroll
        for (int b = 0; b < kB; ++b) {
          const uint32_t from = kt + (16 * t + g) * (D * 2) + (b >> 1) * 128 + (((b & 1) * 4 + j) ^ swizzle(g)) * 16;
          const uint4 k0 = lds128(from), k1 = lds128(from + 8 * D * 2);
#pragma unroll
          for (int n = 0; n < NH; ++n) {
            mma16816<T>(s[n][t], k0.x, k1.x, k0.y, k1.y, q[n][b].x, q[n][b].y);
            mma16816<T>(s[n][t], k0.z, k1.z, k0.w, k1.w, q[n][b].z, q[n][b].w);
          }
        }
      }
      uint32_t ph[NH][kU][2], pl[NH][kU][2];  // P^T: 16-bit values and remainders
#pragma unroll
      for (int n = 0; n < NH; ++n) {
        if (p + kPos > len) {
#pragma unroll
          for (int t = 0; t < kU; ++t)
#pragma unroll
            for (int c = 0; c < 4; ++c)  // c: head 2j + (c & 1), position g + 8 (c >> 1)
              if (p + 16 * t + g + 8 * (c >> 1) >= len) s[n][t][c] = -INFINITY;
        }
        float mx[2] = {m[n][0], m[n][1]};
#pragma unroll
        for (int t = 0; t < kU; ++t)
#pragma unroll
          for (int c = 0; c < 4; ++c) mx[c & 1] = fmaxf(mx[c & 1], s[n][t][c]);
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) mx[c] = fmaxf(mx[c], __shfl_xor_sync(0xffffffffu, mx[c], x));
        if (__any_sync(0xffffffffu, mx[0] > m[n][0] || mx[1] > m[n][1])) {  // rarely, once the maxima have settled
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float corr = m[n][c] == mx[c] ? 1.f : exp2_fast((m[n][c] - mx[c]) * scale);
            m[n][c] = mx[c];
            l[n][c] *= corr;
#pragma unroll
            for (int i = 0; i < kVB * 4; ++i) {
              o[n][i][c] *= corr;
              o[n][i][2 + c] *= corr;
            }
          }
        }
        const float low[2] = {m[n][0] == -INFINITY ? 0.f : m[n][0] * scale, m[n][1] == -INFINITY ? 0.f : m[n][1] * scale};
#pragma unroll
        for (int t = 0; t < kU; ++t) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            s[n][t][c] = exp2_fast(fmaf(s[n][t][c], scale, -low[c & 1])) * kProb<T>;
            l[n][c & 1] += s[n][t][c];
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t hi = pack2<T>(s[n][t][2 * h], s[n][t][2 * h + 1]);
            const float2 f = unpack2<T>(hi);
            ph[n][t][h] = transpose_8x8(hi);
            pl[n][t][h] = transpose_8x8(pack2<T>(s[n][t][2 * h] - f.x, s[n][t][2 * h + 1] - f.y));
          }
        }
      }
#pragma unroll
      for (int t = 0; t < kU; ++t)
#pragma unroll
        for (int b = 0; b < kVB; ++b) {
          uint32_t w[4][4];
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            const int r = 2 * j + (h & 1);  // and + 8 for h >= 2: the same chunk permutation
            const uint4 x = lds128(vt + (16 * t + r + 8 * (h >> 1)) * (D * 2) + b * 128 + (g ^ swizzle(r)) * 16);
            w[h][0] = x.x;
            w[h][1] = x.y;
            w[h][2] = x.z;
            w[h][3] = x.w;
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t a0 = prmt(w[0][i], w[1][i], 0x5410u), a1 = prmt(w[0][i], w[1][i], 0x7632u);
            const uint32_t a2 = prmt(w[2][i], w[3][i], 0x5410u), a3 = prmt(w[2][i], w[3][i], 0x7632u);
#pragma unroll
            for (int n = 0; n < NH; ++n) {
              float d[4] = {0.f, 0.f, 0.f, 0.f};
              mma16816<T>(d, a0, a1, a2, a3, ph[n][t][0], ph[n][t][1]);
              mma16816<T>(d, a0, a1, a2, a3, pl[n][t][0], pl[n][t][1]);
#pragma unroll
              for (int c = 0; c < 4; ++c) o[n][b * 4 + i][c] += d[c];
            }
          }
        }
    }
    const long long begun = u;
    u += t1 - t0;
    if (u < u1) {  // the next span's queries are on their way while this one's parts are joined
      next_span(cur, u);
      load_q(cur);
    }
    if (__any_sync(0xffffffffu, no_page)) {
#pragma unroll
      for (int n = 0; n < NH; ++n) l[n][0] = l[n][1] = nan;
    }

    const bool whole = t0 == 0 && t1 == nt;
    float* slot = slots + (size_t)(2 * worker + (t0 == 0 ? 1 : 0)) * C::kSlot;
    T* out = static_cast<T*>(a.out) + (size_t)row * a.out_stride + (size_t)h0 * D;
#pragma unroll
    for (int n = 0; n < NH; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], x);
#pragma unroll
    for (int n = 0; n < NH; ++n) {  // from here on maxima of the scaled scores, as powers of two
      m[n][0] *= scale;
      m[n][1] *= scale;
    }
    if constexpr (kCluster) {
      // the warps' parts (o, m, l), each where its warp's ring was, joined by the cluster
      auto part = [&](int w) { return reinterpret_cast<const float*>(sh_raw + w * C::kRing); };
      float* mine = reinterpret_cast<float*>(sh_raw + warp * C::kRing);
      copies_wait<0>();
      __syncwarp();
#pragma unroll
      for (int n = 0; n < NH; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int head = 8 * n + 2 * j + c;
          if (g == 0) {
            mine[kHeads * D + head] = m[n][c];
            mine[kHeads * (D + 1) + head] = l[n][c];
          }
#pragma unroll
          for (int b = 0; b < kVB; ++b) {
            float4* dst = reinterpret_cast<float4*>(mine + head * D + 64 * b + 8 * g);
            dst[0] = make_float4(o[n][4 * b][c], o[n][4 * b][2 + c], o[n][4 * b + 1][c], o[n][4 * b + 1][2 + c]);
            dst[1] = make_float4(o[n][4 * b + 2][c], o[n][4 * b + 2][2 + c], o[n][4 * b + 3][c], o[n][4 * b + 3][2 + c]);
          }
        }
      __syncwarp();
      cluster_sync_all();
      // an equal share of the heads' dimensions for each CTA: `cluster` neighbouring threads add up
      // four of them, each its CTA's warps
      const int all = nheads * (D / 4);
#pragma unroll 1
      for (int e0 = warp * 32; e0 < all; e0 += kThreads) {
        const int e = min(e0 + lane, all - 1), c = e & (cluster - 1), at = (rank * all + e) / cluster, h = at / (D / 4), d = at % (D / 4) * 4;
        float top = -INFINITY, ms[kAttnWarps], ls[kAttnWarps], ll = 0.f;
        float4 x[kAttnWarps], acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kAttnWarps; ++w) {
          ms[w] = ld_cluster_f32(part(w) + kHeads * D + h, c);
          ls[w] = ld_cluster_f32(part(w) + kHeads * (D + 1) + h, c);
          x[w] = ld_cluster_f32x4(part(w) + h * D + d, c);
          top = fmaxf(top, ms[w]);
        }
#pragma unroll
        for (int o = 1; o < kClusterMax; o <<= 1)
          if (o < cluster) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float low = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int w = 0; w < kAttnWarps; ++w) {
          const float f = exp2_fast(ms[w] - low);
          ll = fmaf(ls[w], f, ll);
          acc.x = fmaf(x[w].x, f, acc.x);
          acc.y = fmaf(x[w].y, f, acc.y);
          acc.z = fmaf(x[w].z, f, acc.z);
          acc.w = fmaf(x[w].w, f, acc.w);
        }
#pragma unroll
        for (int o = 1; o < kClusterMax; o <<= 1)
          if (o < cluster) {
            ll += __shfl_xor_sync(0xffffffffu, ll, o);
            acc.x += __shfl_xor_sync(0xffffffffu, acc.x, o);
            acc.y += __shfl_xor_sync(0xffffffffu, acc.y, o);
            acc.z += __shfl_xor_sync(0xffffffffu, acc.z, o);
            acc.w += __shfl_xor_sync(0xffffffffu, acc.w, o);
          }
        if (c == 0 && e == e0 + lane) {
          uint2 r;
          r.x = pack2<T>(acc.x / ll, acc.y / ll);
          r.y = pack2<T>(acc.z / ll, acc.w / ll);
          *reinterpret_cast<uint2*>(out + h * D + d) = r;
        }
      }
      __syncwarp();
      cluster_sync_all();  // no CTA leaves while another reads its memory
      return;
    }
    if (!coop) {
#pragma unroll
      for (int n = 0; n < NH; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int head = 8 * n + 2 * j + c;
          if (head >= nheads) continue;
          const float inv = 1.f / l[n][c];
#pragma unroll
          for (int b = 0; b < kVB; ++b) {
            const float x[8] = {o[n][4 * b][c],     o[n][4 * b][2 + c],     o[n][4 * b + 1][c], o[n][4 * b + 1][2 + c],
                                o[n][4 * b + 2][c], o[n][4 * b + 2][2 + c], o[n][4 * b + 3][c], o[n][4 * b + 3][2 + c]};
            if (whole) {
              uint4 r;
              r.x = pack2<T>(x[0] * inv, x[1] * inv);
              r.y = pack2<T>(x[2] * inv, x[3] * inv);
              r.z = pack2<T>(x[4] * inv, x[5] * inv);
              r.w = pack2<T>(x[6] * inv, x[7] * inv);
              *reinterpret_cast<uint4*>(out + head * D + 64 * b + 8 * g) = r;
            } else {
              float4* dst = reinterpret_cast<float4*>(slot + 2 * kHeads + head * D + 64 * b + 8 * g);
              dst[0] = make_float4(x[0], x[1], x[2], x[3]);
              dst[1] = make_float4(x[4], x[5], x[6], x[7]);
            }
          }
          if (!whole && g == 0) {
            slot[head] = m[n][c];
            slot[kHeads + head] = l[n][c];
          }
        }
    } else
#pragma unroll
    for (int n = 0; n < NH; ++n) {  // the warps' parts, joined in shared memory, 8 heads at a time
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int head = 2 * j + c;
        if (g == 0) {
          sh_m[warp][head] = m[n][c];
          sh_l[warp][head] = l[n][c];
        }
#pragma unroll
        for (int b = 0; b < kVB; ++b) {
          float4* dst = reinterpret_cast<float4*>(sh_o + (warp * 8 + head) * D + 64 * b + 8 * g);
          dst[0] = make_float4(o[n][4 * b][c], o[n][4 * b][2 + c], o[n][4 * b + 1][c], o[n][4 * b + 1][2 + c]);
          dst[1] = make_float4(o[n][4 * b + 2][c], o[n][4 * b + 2][2 + c], o[n][4 * b + 3][c], o[n][4 * b + 3][2 + c]);
        }
      }
      __syncthreads();
      for (int e = threadIdx.x; e < min(8, nheads - 8 * n) * (D / 4); e += kThreads) {
        const int h = e / (D / 4), d = (e % (D / 4)) * 4, head = 8 * n + h;
        float mm = sh_m[0][h], ll = 0.f;
#pragma unroll
        for (int w = 1; w < kAttnWarps; ++w) mm = fmaxf(mm, sh_m[w][h]);
        const float low = mm == -INFINITY ? 0.f : mm;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kAttnWarps; ++w) {
          const float f = exp2_fast(sh_m[w][h] - low);
          const float4 x = *reinterpret_cast<const float4*>(sh_o + (w * 8 + h) * D + d);
          ll = fmaf(sh_l[w][h], f, ll);
          acc.x = fmaf(x.x, f, acc.x);
          acc.y = fmaf(x.y, f, acc.y);
          acc.z = fmaf(x.z, f, acc.z);
          acc.w = fmaf(x.w, f, acc.w);
        }
        if (whole) {
          uint2 r;
          r.x = pack2<T>(acc.x / ll, acc.y / ll);
          r.y = pack2<T>(acc.z / ll, acc.w / ll);
          *reinterpret_cast<uint2*>(out + head * D + d) = r;
        } else {
          *reinterpret_cast<float4*>(slot + 2 * kHeads + head * D + d) = acc;
          if (d == 0) {
            slot[head] = mm;
            slot[kHeads + head] = ll;
          }
        }
      }
      __syncthreads();  // the parts' memory is free again
    }
    if (t0 == 0 && (!whole || by_item) && (coop ? threadIdx.x == 0 : lane == 0)) {
      // the worker of the item's last unit, which lies nt - t1 units past this span
      const long long last = begun + nt - 1, whole_ones = more * (each + 1);
      const int w = last < whole_ones ? (int)divide(last, each + 1) : more + (int)divide(last - whole_ones, each);
      AttnDesc& d = desc[by_item ? row * items + item : worker];
      d.row = row;
      d.item = item;
      d.first = worker;
      d.parts = whole ? 0 : w - worker + 1;
    }
    if (u >= u1) break;
  }
  copies_wait<0>();
}

// Joins the parts of the item that worker blockIdx.x began.  A thread adds up four dimensions of
// one head, kJoinFew parts in a round trip to memory, after the description's.
constexpr int kJoinFew = 4;
template <int D, int NH>
constexpr int join_lanes() { return 8 * NH * D / 4; }

template <typename T, int D, int NH>
__global__ void __launch_bounds__(join_lanes<D, NH>()) k_paged_join(const PagedAttention a, const int group, const int blocks) {
  using C = AttnCfg<D, NH>;
  constexpr int kHeads = C::kHeads;
  grid_dependency_wait();  // and no early launch after this: the next attention fills the GPU, and is the slower for odd places
  const AttnDesc* desc = static_cast<const AttnDesc*>(a.workspace);
  const float* slots = reinterpret_cast<const float*>(desc + C::kMaxWorkers);
  const AttnDesc it = desc[blockIdx.x];
  if (it.parts == 0) return;
  const int head = threadIdx.x / (D / 4), d = threadIdx.x % (D / 4) * 4;
  auto part = [&](int i) { return slots + (size_t)(2 * (blockIdx.x + i) + (i == 0 ? 1 : 0)) * C::kSlot; };
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float sum = 0.f, top = -INFINITY;
  for (int i0 = 0; i0 < it.parts; i0 += kJoinFew) {
    float m[kJoinFew], l[kJoinFew];
    float4 x[kJoinFew];
    const float old = top;
#pragma unroll
    for (int i = 0; i < kJoinFew; ++i) {
      m[i] = -INFINITY;
      if (i0 + i < it.parts) {
        const float* p = part(i0 + i);
        m[i] = p[head];
        l[i] = p[kHeads + head];
        x[i] = *reinterpret_cast<const float4*>(p + 2 * kHeads + head * D + d);
      }
      top = fmaxf(top, m[i]);
    }
    const float low = top == -INFINITY ? 0.f : top, corr = exp2_fast(old - low);
    sum *= corr;
    acc.x *= corr;
    acc.y *= corr;
    acc.z *= corr;
    acc.w *= corr;
#pragma unroll
    for (int i = 0; i < kJoinFew; ++i)
      if (i0 + i < it.parts) {
        const float f = exp2_fast(m[i] - low);
        sum = fmaf(l[i], f, sum);
        acc.x = fmaf(x[i].x, f, acc.x);
        acc.y = fmaf(x[i].y, f, acc.y);
        acc.z = fmaf(x[i].z, f, acc.z);
        acc.w = fmaf(x[i].w, f, acc.w);
      }
  }
  if (head >= group - it.item % blocks * kHeads) return;  // a head block's empty places
  uint2 r;
  r.x = pack2<T>(acc.x / sum, acc.y / sum);
  r.y = pack2<T>(acc.z / sum, acc.w / sum);
  const int h = it.item / blocks * group + it.item % blocks * kHeads + head;
  *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + (size_t)it.row * a.out_stride + (size_t)h * D + d) = r;
}

// The same for calls of few items, which may have a hundred parts: a CTA for 64 dimensions of a head
// of an item, groups of threads that take every G-th part, the parts' values on their way while
// the weights are worked out (1 sequence of 104000 positions, 2 kv heads of 128: 26.5 us with the
// attention; 37 with a CTA for all of an item, bound by what one SM can load).
constexpr int kJoinThreads = 256, kJoinDims = 64;
template <typename T, int D, int NH>
__global__ void __launch_bounds__(kJoinThreads) k_paged_join_heads(const PagedAttention a, const int group, const int blocks, const int items) {
  using C = AttnCfg<D, NH>;
  constexpr int kHeads = C::kHeads, kLanes = kJoinDims / 4, kGroups = kJoinThreads / kLanes, kAhead = 8, kWarps = kJoinThreads / 32;
  __shared__ float sh_w[kJoinThreads], sh_top[kWarps], sh_sum[kWarps];
  __shared__ float4 sh_acc[kJoinThreads];
  grid_dependency_wait();
  const int share = blockIdx.x % (D / kJoinDims), head = blockIdx.x / (D / kJoinDims) % kHeads, at = blockIdx.x / (D / kJoinDims * kHeads);
  const int item = at % items;
  if (head >= group - item % blocks * kHeads) return;  // a head block's empty places
  const AttnDesc* desc = static_cast<const AttnDesc*>(a.workspace);
  const float* slots = reinterpret_cast<const float*>(desc + C::kMaxWorkers);
  const AttnDesc it = desc[at];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, grp = tid / kLanes, d = share * kJoinDims + tid % kLanes * 4;
  auto part = [&](int i) { return slots + (size_t)(2 * (it.first + i) + (i == 0 ? 1 : 0)) * C::kSlot; };
  auto value = [&](int i) { return *reinterpret_cast<const float4*>(part(i) + 2 * kHeads + head * D + d); };
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float sum = 0.f, top = -INFINITY;
  for (int c0 = 0; c0 < it.parts; c0 += kJoinThreads) {
    const int n = min(kJoinThreads, it.parts - c0);
    float m = -INFINITY, l = 0.f;
    if (tid < n) {
      m = part(c0 + tid)[head];
      l = part(c0 + tid)[kHeads + head];
    }
    float4 x[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (grp + k * kGroups < n) x[k] = value(c0 + grp + k * kGroups);
    float most = m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    if (lane == 0) sh_top[warp] = most;
    __syncthreads();
    const float old = top;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sh_top[w]);
    const float low = top == -INFINITY ? 0.f : top, corr = exp2_fast(old - low), f = exp2_fast(m - low);
    sh_w[tid] = f;
    float t = l * f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    if (lane == 0) sh_sum[warp] = t;
    __syncthreads();
    sum *= corr;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) sum += sh_sum[w];
    acc.x *= corr;
    acc.y *= corr;
    acc.z *= corr;
    acc.w *= corr;
    auto add = [&](const float4& v, float by) {
      acc.x = fmaf(v.x, by, acc.x);
      acc.y = fmaf(v.y, by, acc.y);
      acc.z = fmaf(v.z, by, acc.z);
      acc.w = fmaf(v.w, by, acc.w);
    };
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (grp + k * kGroups < n) add(x[k], sh_w[grp + k * kGroups]);
#pragma unroll 8
    for (int i = grp + kAhead * kGroups; i < n; i += kGroups) add(value(c0 + i), sh_w[i]);
    __syncthreads();  // the weights' memory is free again
  }
  if (it.parts == 0) return;
  sh_acc[tid] = acc;
  __syncthreads();
  if (grp > 0) return;
#pragma unroll
  for (int i = 1; i < kGroups; ++i) {
    const float4 x = sh_acc[tid + i * kLanes];
    acc.x += x.x;
    acc.y += x.y;
    acc.z += x.z;
    acc.w += x.w;
  }
  uint2 r;
  r.x = pack2<T>(acc.x / sum, acc.y / sum);
  r.y = pack2<T>(acc.z / sum, acc.w / sum);
  const int h = item / blocks * group + item % blocks * kHeads + head;
  *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + (size_t)(at / items) * a.out_stride + (size_t)h * D + d) = r;
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
    constexpr int threads = append_threads<D>();
    const int most = sms * (2048 / threads);  // more than fit at once: the faster SMs take more
    return launched("k_paged_append", launch_maybe_pdl(k_paged_append<T, D>, dim3(a.tokens < most ? a.tokens : most), dim3(threads), 0,
                                                       stream, true, a, pool, tab));
  });
}

namespace {

// Query heads of a CTA: up to 16 of a kv head's group; 8 with head_dim 256, whose operands
// fill the registers.
bool attn_wide(int group, int head_dim) { return group > 8 && head_dim <= 128; }

template <typename T, int D, int NH>
struct ClusterLaunch {  // n clusters, with programmatic stream serialisation
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attrs[2];
  ClusterLaunch(unsigned n, int cluster, cudaStream_t stream) {
    cfg.gridDim = dim3(n * cluster);
    cfg.blockDim = dim3(kAttnWarps * 32);
    cfg.dynamicSmemBytes = kAttnWarps * AttnCfg<D, NH>::kRing;
    cfg.stream = stream;
    attrs[0].id = cudaLaunchAttributeClusterDimension;
    attrs[0].val.clusterDim.x = cluster;
    attrs[0].val.clusterDim.y = attrs[0].val.clusterDim.z = 1;
    attrs[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attrs;
    cfg.numAttrs = 2;
  }
};

// How many clusters of this size the device runs at once (asked once for each device and size).
template <typename T, int D, int NH>
int resident_clusters(int dev, int cluster) {
  static std::atomic<int> known[64][kClusterMax + 1];  // that number and 1; 0: not asked yet
  std::atomic<int>& mine = known[dev & 63][cluster];
  int n = mine.load(std::memory_order_acquire);
  if (n == 0 || dev >= 64) {
    ClusterLaunch<T, D, NH> l(1, cluster, nullptr);
    l.cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, k_paged_attention<T, D, NH, true>, &l.cfg) != cudaSuccess) n = 0;
    (void)cudaGetLastError();
    mine.store(++n, std::memory_order_release);
  }
  return n - 1;
}

// CTAs that fill the current device, and those of the cluster that takes an item, 0 for a call that
// is shared out in parts.  all: items; cap: positions of a full table row.
template <typename T, int D, int NH>
int plan_attention(long long all, long long cap, int* ctas, int* cluster) {
  using C = AttnCfg<D, NH>;
  int sms = 0;
  const int rc = current_sm_count(&sms);
  if (rc != W4A16_OK) return rc;
  *ctas = (sms < kAttnMaxSms ? sms : kAttnMaxSms) * C::kPerSm;
  static std::atomic<uint64_t> configured{0};  // one bit per device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && !(configured.load(std::memory_order_acquire) >> (dev & 63) & 1ull)) {
    e = cudaFuncSetAttribute(k_paged_attention<T, D, NH, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(k_paged_attention<T, D, NH, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kAttnWarps * C::kRing);
    if (e == cudaSuccess && dev < 64) configured.fetch_or(1ull << dev, std::memory_order_acq_rel);
  }
  if (e != cudaSuccess) return launched("configuring k_paged_attention,", e);
  int n = kClusterMax;
  while (n > 1 && (cap <= (long long)n / 2 * kClusterLeast || all > resident_clusters<T, D, NH>(dev, n))) n /= 2;
  const bool few = all * n <= *ctas && cap <= (long long)n * cluster_most(D, NH, all * n * 2 >= *ctas);
  *cluster = few || (all <= 2 * *ctas && cap <= kTwiceMost) ? n : 0;
  return W4A16_OK;
}

template <typename T, int D, int NH>
int launch_attention(const PagedAttention& a, const PagedPool& pool, const PagedTables& tab, cudaStream_t stream) {
  using C = AttnCfg<D, NH>;
  const int group = a.heads / pool.kv_heads, blocks = (group + C::kHeads - 1) / C::kHeads;
  const long long all = (long long)a.rows * pool.kv_heads * blocks;
  int ctas = 0, cluster = 0;
  const int rc = plan_attention<T, D, NH>(all, (long long)tab.width << pool.page_shift, &ctas, &cluster);
  if (rc != W4A16_OK) return rc;
  if (cluster) {
    ClusterLaunch<T, D, NH> l((unsigned)all, cluster, stream);
    return launched("k_paged_attention", cudaLaunchKernelEx(&l.cfg, k_paged_attention<T, D, NH, true>, a, pool, tab, group, blocks, true, 0, cluster, false));
  }
  const bool coop = all < ctas * kAttnWarps;
  const int workers = coop ? ctas : ctas * kAttnWarps;
  // with far fewer items than CTAs a CTA has one at most, and the cost of beginning it is no matter of balance
  const int cost = !coop ? kItemCost : all * 4 >= ctas ? kItemCostCta : 0;
  const bool many = coop && all * 8 < ctas;  // items few enough to be cut into many parts
  const int rc2 = launched("k_paged_attention", launch_maybe_pdl(k_paged_attention<T, D, NH, false>, dim3(ctas), dim3(kAttnWarps * 32), C::kSmem,
                                                                 stream, true, a, pool, tab, group, blocks, coop, cost, 1, many));
  if (rc2 != W4A16_OK) return rc2;
  if (many)
    return launched("k_paged_join_heads", launch_maybe_pdl(k_paged_join_heads<T, D, NH>, dim3((unsigned)all * C::kHeads * (D / kJoinDims)), dim3(kJoinThreads), 0,
                                                           stream, true, a, group, blocks, pool.kv_heads * blocks));
  return launched("k_paged_join", launch_maybe_pdl(k_paged_join<T, D, NH>, dim3(workers), dim3(join_lanes<D, NH>()), 0, stream, true, a, group,
                                                   blocks));
}

template <typename F>
int by_form(int dtype, int head_dim, int group, F&& f) {  // of the kernel: type, head_dim, 8 or 16 heads
  return by_type(dtype, head_dim, [&](auto t, auto d) {
    if constexpr (decltype(d)::value <= 128) {
      if (attn_wide(group, head_dim)) return f(t, d, std::integral_constant<int, 2>());
    }
    return f(t, d, std::integral_constant<int, 1>());
  });
}

}  // namespace

bool paged_attention_needs_workspace(int dtype, int rows, int heads, int kv_heads, int head_dim, long long cap) {
  int ctas = 0, cluster = 0;
  const int rc = by_form(dtype, head_dim, heads / kv_heads, [&](auto t, auto d, auto nh) {
    const int block = 8 * decltype(nh)::value, blocks = (heads / kv_heads + block - 1) / block;
    return plan_attention<decltype(t), decltype(d)::value, decltype(nh)::value>((long long)rows * kv_heads * blocks, cap, &ctas, &cluster);
  });
  return rc != W4A16_OK || cluster == 0;
}

size_t paged_attention_workspace_bytes(int heads, int kv_heads, int head_dim) {
  const size_t h = attn_wide(heads / kv_heads, head_dim) ? 16 : 8;
  return (size_t)kAttnMaxSms * attn_per_sm(head_dim) * kAttnWarps * (sizeof(AttnDesc) + 2 * h * (head_dim + 2) * 4);
}

int launch_paged_attention(const PagedAttention& a, const PagedPool& pool, const PagedTables& tab, cudaStream_t stream) {
  return by_form(pool.dtype, pool.head_dim, a.heads / pool.kv_heads, [&](auto t, auto d, auto nh) {
    return launch_attention<decltype(t), decltype(d)::value, decltype(nh)::value>(a, pool, tab, stream);
  });
}

}  // namespace w4a16
