// What a serving loop does to a step's logits before the next token is chosen, in one pass:
//   x = logits[v]
//   v occurs in the row's tokens:   x = x > 0 ? x / repetition : x * repetition
//   c = occurrences of v among the tokens generated so far (after the prompt):
//                                   x = x - frequency * c - presence * (c > 0)
//   x = x + bias[v] + (values of the row's pairs (v, value), in their order)
//   v not allowed by the row's grammar mask: x = -inf
// in fp32, rounded once to the logits' type.
//
// A CTA takes a slice of one row's vocabulary.  Its logits go to registers first, in 16-byte
// loads; while they are on their way it counts the row's tokens that fall into the slice in
// shared memory (integer atomics: the result does not depend on their order).  The logits are
// read and written once; the history is read once for each slice, from L2.  Bound by bandwidth
// without tokens (64 rows of 128256: 12 us, 0.85 of the copy rate), else by the chain of loads,
// counts and barriers that each CTA goes through at 4 CTAs for an SM (with histories of up to
// 4096, 64 pairs and a mask: 22 us, 0.46).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>

#include "w4a16_device.cuh"
#include "w4a16_internal.h"

namespace w4a16 {

namespace {

constexpr uint32_t kSeen = 0x80000000u, kPair = 0x40000000u, kCount = 0x3fffffffu;

// kLoads: 16-byte pieces of the slice a thread holds.
template <typename T, int kThreads, int kLoads>
struct LogitsCfg {
  static constexpr int kVec = 16 / sizeof(T), kSlice = kThreads * kLoads * kVec;
  static constexpr int kWords = kSlice / 32 + 1;  // mask words that a slice touches
};

template <typename T, int kThreads, int kLoads>
__global__ void __launch_bounds__(kThreads, kThreads == 256 ? 4 : 1) k_process_logits(const LogitsProblem p, const int slices) {
  using C = LogitsCfg<T, kThreads, kLoads>;
  constexpr int kVec = C::kVec, kSlice = C::kSlice;
  // word[token of the slice]: seen in the prompt | occurrences after it; or, for a token with bias
  // pairs: has pairs | its place in paired (its word, the sum of its values)
  extern __shared__ __align__(16) uint32_t word[];
  uint2* paired = reinterpret_cast<uint2*>(word + kSlice);
  __shared__ uint32_t allowed[C::kWords], pairs_here;
  __shared__ int first_ids[kThreads];  // the row's first pairs
  __shared__ float first_values[kThreads];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  grid_dependency_wait();
  grid_launch_dependents();
  const int row = blockIdx.x / slices;
  const T* in = static_cast<const T*>(p.logits) + (size_t)row * p.stride;
  T* out = static_cast<T*>(p.out) + (size_t)row * p.out_stride;
  // the slice starts where 16-byte loads are aligned, at or before the row's start for the first
  const int skew = (int)(reinterpret_cast<uintptr_t>(in) % 16 / sizeof(T));
  const int v0 = (int)(blockIdx.x % slices) * kSlice - skew, lo = max(v0, 0), v1 = min(p.vocab, v0 + kSlice);

  if (v0 >= p.vocab) return;  // room for a skew that this row does not have

  // Everything that comes from memory is asked for first: lengths, the first tokens (whether they
  // count or not), pairs and mask, then the logits.
  const bool full = v0 >= 0 && v0 + kSlice <= p.vocab;
  auto inside = [&](int v) { return full || (v >= 0 && v + kVec <= p.vocab); };
  const int mine = tid * kVec;  // this thread's place in each round of pieces
  const T* in_mine = in + v0 + mine;
  T* out_mine = out + v0 + mine;
  union Piece {
    uint4 all;
    T one[kVec];
  } piece[kLoads];
  int total = 0, prompt = 0;
  auto token_at = [&](int j) {  // -1 for one outside the vocabulary
    const size_t at = (size_t)row * p.token_stride + j;
    if (p.token_bytes == 4) return fetch(static_cast<const int*>(p.tokens) + at);
    const long long t = fetch(static_cast<const long long*>(p.tokens) + at);
    return t < 0 || t >= p.vocab ? -1 : (int)t;
  };
  const int4* tokens4 = nullptr;  // where int32 tokens are aligned for 16-byte loads
  int4 next = make_int4(-1, -1, -1, -1);
  if (p.tokens) {
    total = p.total_lens ? min(max(fetch(p.total_lens + row), 0), p.history) : p.history;
    prompt = p.prompt_lens ? fetch(p.prompt_lens + row) : 0;
    const int* t = static_cast<const int*>(p.tokens) + (size_t)row * p.token_stride;
    if (p.token_bytes == 4 && reinterpret_cast<uintptr_t>(t) % 16 == 0) {
      tokens4 = reinterpret_cast<const int4*>(t);
      if (4 * tid + 4 <= p.history) next = fetch(tokens4 + tid);
    }
  }
  const int* ids = p.bias_ids + (size_t)row * p.pairs;
  const float* values = p.bias_values + (size_t)row * p.pairs;
  if (p.pairs) {
    first_ids[tid] = tid < p.pairs ? fetch(ids + tid) : -1;
    first_values[tid] = tid < p.pairs ? fetch(values + tid) : 0.f;
  }
  const int first_word = lo >> 5;
  if (p.mask)
    for (int i = tid; i <= ((v1 - 1) >> 5) - first_word; i += kThreads)
      allowed[i] = (uint32_t)fetch(p.mask + (size_t)row * p.mask_stride + first_word + i);
  const float rep = p.repetition ? fetch(p.repetition + row) : 1.f, inv_rep = 1.f / rep;
  const float freq = p.frequency ? fetch(p.frequency + row) : 0.f;
  const float pres = p.presence ? fetch(p.presence + row) : 0.f;

#pragma unroll
  for (int c = 0; c < kLoads; ++c) {
    if (inside(v0 + mine + c * kThreads * kVec)) piece[c].all = *reinterpret_cast<const uint4*>(in_mine + c * kThreads * kVec);
  }
  const bool marks = p.tokens || p.pairs;
  if (marks) {
    for (int i = tid; i < kSlice / 4; i += kThreads) reinterpret_cast<uint4*>(word)[i] = make_uint4(0u, 0u, 0u, 0u);
    if (tid == 0) pairs_here = 0u;
    __syncthreads();
    auto count = [&](int t, int j) {
      if ((unsigned)t - (unsigned)lo >= (unsigned)(v1 - lo)) return;
      if (j >= prompt)
        atomicAdd(&word[t - v0], 1u);
      else
        atomicOr(&word[t - v0], kSeen);
    };
    int done = 0;
    if (tokens4) {
#pragma unroll 1
      for (int q = tid; q < total / 4; q += kThreads) {
        const int4 t = next;
        if (q + kThreads < total / 4) next = fetch(tokens4 + q + kThreads);
        count(t.x, 4 * q);
        count(t.y, 4 * q + 1);
        count(t.z, 4 * q + 2);
        count(t.w, 4 * q + 3);
      }
      done = total / 4 * 4;
    }
#pragma unroll 4
    for (int j = done + tid; j < total; j += kThreads) count(token_at(j), j);
    // the first pair of an id adds up all of the id's values, in the pairs' order: a warp for
    // each pair that falls into the slice
    if (p.pairs) __syncthreads();  // the counts are final
    auto id_at = [&](int k) { return k < kThreads ? first_ids[k] : k < p.pairs ? fetch(ids + k) : -1; };
#pragma unroll 1
    for (int j = warp; j < p.pairs; j += kThreads / 32) {
      const int wanted = id_at(j);
      if (wanted < lo || wanted >= v1) continue;
      float sum = 0.f;
      bool first = true;
      for (int k0 = 0; k0 < p.pairs && first; k0 += 32) {
        const bool same = id_at(k0 + lane) == wanted;  // an id in the slice is not -1
        const float value = !same ? 0.f : k0 + lane < kThreads ? first_values[k0 + lane] : fetch(values + k0 + lane);
        unsigned m = __ballot_sync(0xffffffffu, same);
        if (m && k0 + __ffs(m) - 1 < j) first = false;
        for (; m && first; m &= m - 1) sum += __shfl_sync(0xffffffffu, value, __ffs(m) - 1);
      }
      if (first && lane == 0) {
        const uint32_t i = atomicAdd(&pairs_here, 1u);
        paired[i] = make_uint2(word[wanted - v0], __float_as_uint(sum));
        word[wanted - v0] = kPair | i;
      }
    }
  }
  if (marks || p.mask) __syncthreads();
  const float* bias = p.bias ? p.bias + (size_t)row * p.bias_stride : nullptr;
  auto resolve = [&](uint32_t& w, float& add) {  // a token with pairs: its own word, and what they add
    if (w & kPair) {
      const uint2 it = paired[w & kCount];
      w = kPair | it.x;
      add = __uint_as_float(it.y);
    }
  };
  auto penalised = [&](float x, uint32_t w) {
    const float by = x > 0.f ? inv_rep : rep, n = (float)(w & kCount);
    x = w & (kSeen | kCount) ? x * by : x;
    return w & kCount ? x - freq * n - pres : x;
  };
  const bool wide_out = reinterpret_cast<uintptr_t>(out + v0) % 16 == 0, wide_bias = reinterpret_cast<uintptr_t>(bias + v0) % 16 == 0;
#pragma unroll
  for (int c = 0; c < kLoads; ++c) {
    const int at = mine + c * kThreads * kVec, v = v0 + at;
    if (!inside(v)) continue;
    float x[kVec];
#pragma unroll
    for (int e = 0; e < kVec; ++e) x[e] = to_f32<T>(piece[c].one[e]);
    uint32_t w[kVec], any = 0;
    float add[kVec];
    if (marks) {
#pragma unroll
      for (int e = 0; e < kVec; e += 4) *reinterpret_cast<uint4*>(w + e) = *reinterpret_cast<const uint4*>(word + at + e);
#pragma unroll
      for (int e = 0; e < kVec; ++e) any |= w[e];
      if (any & kPair) {
#pragma unroll
        for (int e = 0; e < kVec; ++e) resolve(w[e], add[e]);
      }
      if (any) {
#pragma unroll
        for (int e = 0; e < kVec; ++e) x[e] = penalised(x[e], w[e]);
      }
    }
    if (bias) {
      if (wide_bias) {
#pragma unroll
        for (int e = 0; e < kVec; e += 4) {
          const float4 b = fetch(reinterpret_cast<const float4*>(bias + v + e));
          x[e] += b.x;
          x[e + 1] += b.y;
          x[e + 2] += b.z;
          x[e + 3] += b.w;
        }
      } else {
#pragma unroll
        for (int e = 0; e < kVec; ++e) x[e] += fetch(bias + v + e);
      }
    }
    if (any & kPair) {
#pragma unroll
      for (int e = 0; e < kVec; ++e)
        if (w[e] & kPair) x[e] += add[e];
    }
    if (p.mask) {  // the piece's bits lie in one word or in two neighbours
      const int i = (v >> 5) - first_word;
      const uint32_t bits = __funnelshift_r(allowed[i], allowed[((v + kVec - 1) >> 5) - first_word], v & 31);
#pragma unroll
      for (int e = 0; e < kVec; ++e)
        if (!(bits >> e & 1u)) x[e] = -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < kVec; ++e) piece[c].one[e] = from_f32<T>(x[e]);
    if (wide_out) {
      *reinterpret_cast<uint4*>(out_mine + c * kThreads * kVec) = piece[c].all;
    } else {
#pragma unroll
      for (int e = 0; e < kVec; ++e) out_mine[c * kThreads * kVec + e] = piece[c].one[e];
    }
  }
  // the ends of the row that are no whole piece: under 2 kVec tokens
  auto one = [&](int v) {
    const int at = v - v0;
    float x = to_f32<T>(in[v]);
    uint32_t w = marks ? word[at] : 0u;
    float add;
    resolve(w, add);
    x = penalised(x, w);
    if (bias) x += fetch(bias + v);
    if (w & kPair) x += add;
    if (p.mask && !(allowed[(v >> 5) - first_word] >> (v & 31) & 1u)) x = -INFINITY;
    out[v] = from_f32<T>(x);
  };
  if (v0 < 0 && tid < min(v0 + kVec, p.vocab)) one(tid);  // the piece around the row's start
  const int tail = v1 - (v1 - v0) % kVec;                 // the piece around its end
  if (tail >= max(v0, 0) && tail + tid < v1) one(tail + tid);
}

template <typename T, int kThreads, int kLoads>
int launch_loads(const LogitsProblem& p, cudaStream_t stream) {
  using C = LogitsCfg<T, kThreads, kLoads>;
  const long long slices = ((long long)p.vocab + C::kVec - 1 + C::kSlice - 1) / C::kSlice;  // the skew is at most kVec - 1
  const long long blocks = slices * p.rows;
  if (blocks > 0x7fffffffll) {
    set_error("%d rows of %d logits are too many for one call", p.rows, p.vocab);
    return W4A16_ERR_SHAPE;
  }
  const size_t smem = p.pairs || p.tokens ? (size_t)C::kSlice * 4 + (size_t)(p.pairs < C::kSlice ? p.pairs : C::kSlice) * 8 : 0;
  cudaError_t e = cudaSuccess;
  if (smem > 40960) {
    static std::atomic<uint64_t> configured{0};  // one bit per device
    int dev = 0;
    e = cudaGetDevice(&dev);
    if (e == cudaSuccess && !(configured.load(std::memory_order_acquire) >> (dev & 63) & 1ull)) {
      e = cudaFuncSetAttribute(k_process_logits<T, kThreads, kLoads>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSlice * 12);
      if (e == cudaSuccess && dev < 64) configured.fetch_or(1ull << dev, std::memory_order_acq_rel);
    }
  }
  if (e == cudaSuccess)
    e = launch_maybe_pdl(k_process_logits<T, kThreads, kLoads>, dim3((unsigned)blocks), dim3(kThreads), smem, stream, true, p, (int)slices);
  (void)cudaGetLastError();
  if (e != cudaSuccess) {
    set_error("k_process_logits launch failed: %s", cudaGetErrorString(e));
    return W4A16_ERR_CUDA;
  }
  return W4A16_OK;
}

template <typename T>
int launch_type(const LogitsProblem& p, cudaStream_t stream) {
  int sms = 0;
  const int rc = current_sm_count(&sms);
  if (rc != W4A16_OK) return rc;
  // Slices of 8192 tokens, whose history is read fewer times; of 2048 where those would leave SMs
  // without one (1 row of 128256: 2.6 us by slices of 2048, 4.2 by 8192; 64 rows: 54 and 22.5).
  constexpr int kSize = sizeof(T);
  const long long blocks = ((long long)p.vocab + 8191) / 8192 * p.rows;
  return blocks < sms ? launch_loads<T, 128 * kSize, 1>(p, stream) : launch_loads<T, 256, kSize * 2>(p, stream);
}

}  // namespace

int launch_process_logits(const LogitsProblem& p, cudaStream_t stream) {
  if (p.dtype == W4A16_DTYPE_F32) return launch_type<float>(p, stream);
  if (p.dtype == W4A16_DTYPE_F16) return launch_type<__half>(p, stream);
  return launch_type<__nv_bfloat16>(p, stream);
}

}  // namespace w4a16
