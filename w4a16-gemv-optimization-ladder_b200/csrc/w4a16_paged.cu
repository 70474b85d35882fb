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
// One warp per (row, query head); a lane holds D / 32 dimensions.  Running maximum, sum and
// output in fp32.
template <typename T, int D>
__global__ void __launch_bounds__(128) k_paged_attention(const PagedAttention a, const PagedPool pool, const PagedTables tab) {
  constexpr int kPer = D / 64;  // 32-bit words (two dimensions) per lane
  const int lane = threadIdx.x & 31;
  const long long w = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (w >= (long long)a.rows * a.heads) return;
  const int row = (int)(w / a.heads), head = (int)(w % a.heads);
  const int kvh = head / (a.heads / pool.kv_heads);
  const int seq = a.seqs ? __ldg(a.seqs + row) : row;
  const int len = __ldg(a.lengths + row);
  const float nan = __int_as_float(0x7fc00000);
  float2 q[kPer], o[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const uint32_t v = *reinterpret_cast<const uint32_t*>(static_cast<const T*>(a.q) + (size_t)row * a.q_stride + head * D + 2 * (lane + 32 * i));
    q[i] = unpack2<T>(v);
    o[i] = make_float2(0.f, 0.f);
  }
  float m = -INFINITY, l = 0.f;
  const int cap = tab.width << pool.page_shift;
  for (int p = 0; p < len; ++p) {
    const int page = page_of(tab, seq, p, pool.page_shift, pool.pages);
    if (page < 0 || p >= cap) {
      l = nan;
      break;
    }
    const size_t at = (size_t)page * pool.page_stride + (size_t)kvh * pool.head_stride +
                      (size_t)(p & ((1 << pool.page_shift) - 1)) * pool.token_stride;
    float d = 0.f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const float2 k = unpack2<T>(*reinterpret_cast<const uint32_t*>(static_cast<const T*>(pool.k) + at + 2 * (lane + 32 * i)));
      d = fmaf(q[i].x, k.x, fmaf(q[i].y, k.y, d));
    }
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) d += __shfl_xor_sync(0xffffffffu, d, x);
    d *= a.scale;
    const float mn = fmaxf(m, d), base = mn == -INFINITY ? 0.f : mn;
    const float corr = __expf(m - base), e = __expf(d - base);
    l = l * corr + e;
    m = mn;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const float2 v = unpack2<T>(*reinterpret_cast<const uint32_t*>(static_cast<const T*>(pool.v) + at + 2 * (lane + 32 * i)));
      o[i].x = fmaf(e, v.x, o[i].x * corr);
      o[i].y = fmaf(e, v.y, o[i].y * corr);
    }
  }
  const float inv = len <= 0 ? 0.f : 1.f / l;
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    *reinterpret_cast<uint32_t*>(static_cast<T*>(a.out) + (size_t)row * a.out_stride + head * D + 2 * (lane + 32 * i)) =
        pack2<T>(o[i].x * inv, o[i].y * inv);
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

size_t paged_attention_workspace_bytes(int, int, int) { return 16; }  // not used yet

int launch_paged_attention(const PagedAttention& a, const PagedPool& pool, const PagedTables& tab, cudaStream_t stream) {
  return by_type(pool.dtype, pool.head_dim, [&](auto t, auto d) {
    using T = decltype(t);
    constexpr int D = decltype(d)::value;
    const long long warps = (long long)a.rows * a.heads;
    k_paged_attention<T, D><<<(unsigned)((warps + 3) / 4), 128, 0, stream>>>(a, pool, tab);
    return launched("k_paged_attention", cudaGetLastError());
  });
}

}  // namespace w4a16
