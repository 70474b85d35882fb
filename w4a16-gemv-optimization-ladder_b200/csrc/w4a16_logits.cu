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
// 4096, 64 pairs and a mask: 20.8 us, 0.50).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>

#include "w4a16_device.cuh"
#include "w4a16_internal.h"

namespace w4a16 {

namespace {

constexpr uint32_t kSeen = 0x80000000u, kCount = 0x7fffffffu;

struct Pair {  // a token with bias pairs: the sum of its values, its logit
  int token;
  float sum, logit;
};

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
  // word[token of the slice]: seen in the prompt | occurrences after it
  extern __shared__ __align__(16) uint32_t word[];
  // places[token of the slice]: of more than one round of pairs, 1 + the place in paired
  const bool rounds = p.pairs > kThreads;
  uint32_t* places = word + kSlice;
  Pair* paired = reinterpret_cast<Pair*>(rounds ? places + kSlice : places);
  __shared__ uint32_t allowed[C::kWords], pairs_here;
  __shared__ __align__(16) int ids_here[kThreads];  // a round of the row's pairs
  __shared__ float values_here[kThreads];
  const int tid = threadIdx.x;
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
  auto pair_at = [&](int k) {
    ids_here[tid] = k < p.pairs ? fetch(ids + k) : -1;
    values_here[tid] = k < p.pairs ? fetch(values + k) : 0.f;
  };
  if (p.pairs) pair_at(tid);
  const int first_word = lo >> 5;
  if (p.mask)
    for (int i = tid; i <= ((v1 - 1) >> 5) - first_word; i += kThreads)
      allowed[i] = (uint32_t)fetch(p.mask + (size_t)row * p.mask_stride + first_word + i);
  const float rep = p.repetition ? fetch(p.repetition + row) : 1.f, inv_rep = 1.f / rep;
  const float inv_rest = fmaf(-rep, inv_rep, 1.f) * inv_rep;  // inv_rep + inv_rest is 1 / rep to 2^-47
  const float freq = p.frequency ? fetch(p.frequency + row) : 0.f;
  const float pres = p.presence ? fetch(p.presence + row) : 0.f;

#pragma unroll
  for (int c = 0; c < kLoads; ++c) {
    if (inside(v0 + mine + c * kThreads * kVec)) piece[c].all = *reinterpret_cast<const uint4*>(in_mine + c * kThreads * kVec);
  }
  const bool marks = p.tokens || p.pairs;
  if (marks) {
    for (int i = tid; i < (rounds ? kSlice / 2 : kSlice / 4); i += kThreads) reinterpret_cast<uint4*>(word)[i] = make_uint4(0u, 0u, 0u, 0u);
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
    // A thread for each pair, kThreads of them in a round: the first of an id in the round adds up all
    // of the id's values there, in the pairs' order (nearly always its own).  The token is written
    // once more at the end, so that the others' way is free of it (64 rows with 64 pairs, histories and
    // a mask: 20.7 us; 22.5 with the pairs' places looked up by every token and a warp for each pair).
#pragma unroll 1
    for (int k0 = 0; k0 < p.pairs; k0 += kThreads) {
      if (k0) {
        __syncthreads();
        pair_at(k0 + tid);
        __syncthreads();
      }
      const int wanted = ids_here[tid];
      if (wanted < lo || wanted >= v1) continue;
      int same = 0;
      const int end = min(p.pairs - k0, kThreads);
#pragma unroll 4
      for (int k = 0; k < end; k += 4) {  // an id in the slice is not -1
        const int4 x = *reinterpret_cast<const int4*>(ids_here + k);
        same += (x.x == wanted) + (x.y == wanted) + (x.z == wanted) + (x.w == wanted);
      }
      int k = tid;
      if (same > 1) {
        k = 0;
        while (ids_here[k] != wanted) ++k;
        if (k < tid) continue;
      }
      const int at = rounds ? (int)places[wanted - v0] - 1 : -1;
      float sum = at < 0 ? 0.f : paired[at].sum;
      for (; same; ++k)
        if (ids_here[k] == wanted) {
          sum += values_here[k];
          --same;
        }
      if (at >= 0) {
        paired[at].sum = sum;
      } else {
        const uint32_t i = atomicAdd(&pairs_here, 1u);
        paired[i] = Pair{wanted, sum, to_f32<T>(in[wanted])};
        if (rounds) places[wanted - v0] = i + 1;
      }
    }
  }
  if (marks || p.mask) __syncthreads();
  const float* bias = p.bias ? p.bias + (size_t)row * p.bias_stride : nullptr;
  auto penalised = [&](float x, uint32_t w) {
    // x / rep as the sum of two products, rounded once (64 rows with 64 pairs, histories and a mask: 20.7 us, with a
    // division 23.5); of an infinity one of them is NaN, and the other the quotient
    const float q = x * inv_rep, z = fmaf(x, inv_rep, x * inv_rest), n = (float)(w & kCount);
    const float y = x > 0.f ? (z == z ? z : q) : x * rep;
    x = w & (kSeen | kCount) ? y : x;
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
    if (marks) {
#pragma unroll
      for (int e = 0; e < kVec; e += 4) *reinterpret_cast<uint4*>(w + e) = *reinterpret_cast<const uint4*>(word + at + e);
#pragma unroll
      for (int e = 0; e < kVec; ++e) any |= w[e];
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
  auto one = [&](int v, float x, float sum) {
    x = penalised(x, marks ? word[v - v0] : 0u);
    if (bias) x += fetch(bias + v);
    x += sum;
    if (p.mask && !(allowed[(v >> 5) - first_word] >> (v & 31) & 1u)) x = -INFINITY;
    out[v] = from_f32<T>(x);
  };
  // the ends of the row that are no whole piece: under 2 kVec tokens
  auto end = [&](int v) { one(v, to_f32<T>(in[v]), -0.f); };  // x + -0 is x, of either zero
  if (v0 < 0 && tid < min(v0 + kVec, p.vocab)) end(tid);  // the piece around the row's start
  const int tail = v1 - (v1 - v0) % kVec;                 // the piece around its end
  if (tail >= max(v0, 0) && tail + tid < v1) end(tail + tid);
  if (p.pairs) {
    __syncthreads();  // the plain values are written
    for (int i = tid; i < (int)pairs_here; i += kThreads) one(paired[i].token, paired[i].logit, paired[i].sum);
  }
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
  const size_t smem = p.pairs || p.tokens ? (size_t)C::kSlice * (p.pairs > kThreads ? 8 : 4) +
                                                (size_t)(p.pairs < C::kSlice ? p.pairs : C::kSlice) * sizeof(Pair) : 0;
  cudaError_t e = cudaSuccess;
  if (smem > 40960) {
    static std::atomic<uint64_t> configured{0};  // one bit per device
    int dev = 0;
    e = cudaGetDevice(&dev);
    if (e == cudaSuccess && !(configured.load(std::memory_order_acquire) >> (dev & 63) & 1ull)) {
      e = cudaFuncSetAttribute(k_process_logits<T, kThreads, kLoads>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSlice * (8 + sizeof(Pair)));
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
  // without one (1 row of 128256: 2.6 us by slices of 2048, 4.2 by 8192; 64 rows: 54 and 20).
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
