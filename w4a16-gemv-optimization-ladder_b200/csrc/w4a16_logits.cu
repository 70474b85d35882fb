// What a serving loop does to a step's logits before the next token is chosen, in one pass:
//   x = logits[v]
//   v occurs in the row's tokens:   x = x > 0 ? x / repetition : x * repetition
//   c = occurrences of v among the tokens generated so far (after the prompt):
//                                   x = x - frequency * c - presence * (c > 0)
//   x = x + bias[v] + (values of the row's pairs (v, value), in their order)
//   v not allowed by the row's grammar mask: x = -inf
// in fp32, rounded once to the logits' type.
//
// A CTA takes a slice of one row's vocabulary: it counts the row's tokens that fall into the
// slice in shared memory (integer atomics: the result does not depend on their order), then
// streams the slice's logits once.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "w4a16_device.cuh"
#include "w4a16_internal.h"

namespace w4a16 {

namespace {

constexpr int kSlice = 8192;
constexpr uint32_t kSeen = 0x80000000u, kPair = 0x40000000u, kCount = 0x3fffffffu;

template <typename T>
__global__ void __launch_bounds__(256) k_process_logits(const LogitsProblem p) {
  __shared__ uint32_t word[kSlice];  // seen | has a bias pair | occurrences in the output
  const int row = blockIdx.y, v0 = blockIdx.x * kSlice, n = min(kSlice, p.vocab - v0);
  const bool marks = p.tokens || p.pairs;
  if (marks) {
    for (int i = threadIdx.x; i < n; i += 256) word[i] = 0;
    __syncthreads();
    if (p.tokens) {
      const int total = p.total_lens ? min(max(p.total_lens[row], 0), p.history) : p.history;
      const int prompt = p.prompt_lens ? p.prompt_lens[row] : 0;
      for (int j = threadIdx.x; j < total; j += 256) {
        const size_t at = (size_t)row * p.token_stride + j;
        const long long t = p.token_bytes == 8 ? static_cast<const long long*>(p.tokens)[at] : static_cast<const int*>(p.tokens)[at];
        if (t < v0 || t >= v0 + n) continue;
        atomicOr(&word[t - v0], kSeen);
        if (j >= prompt) atomicAdd(&word[t - v0], 1u);
      }
    }
    for (int j = threadIdx.x; j < p.pairs; j += 256) {
      const int t = p.bias_ids[(size_t)row * p.pairs + j];
      if (t >= v0 && t < v0 + n) atomicOr(&word[t - v0], kPair);
    }
    __syncthreads();
  }
  const float rep = p.repetition ? p.repetition[row] : 1.f;
  const float freq = p.frequency ? p.frequency[row] : 0.f;
  const float pres = p.presence ? p.presence[row] : 0.f;
  const T* in = static_cast<const T*>(p.logits) + (size_t)row * p.stride + v0;
  T* out = static_cast<T*>(p.out) + (size_t)row * p.out_stride + v0;
  for (int i = threadIdx.x; i < n; i += 256) {
    float x = to_f32<T>(in[i]);
    const uint32_t w = marks ? word[i] : 0u;
    if (w & kSeen) {
      x = x > 0.f ? x / rep : x * rep;
      const uint32_t c = w & kCount;
      if (c) x = x - freq * (float)c - pres;
    }
    if (p.bias) x += p.bias[(size_t)row * p.bias_stride + v0 + i];
    if (w & kPair)
      for (int j = 0; j < p.pairs; ++j)
        if (p.bias_ids[(size_t)row * p.pairs + j] == v0 + i) x += p.bias_values[(size_t)row * p.pairs + j];
    if (p.mask && !(p.mask[(size_t)row * p.mask_stride + ((v0 + i) >> 5)] >> ((v0 + i) & 31) & 1)) x = -INFINITY;
    out[i] = from_f32<T>(x);
  }
}

}  // namespace

int launch_process_logits(const LogitsProblem& p, cudaStream_t stream) {
  const dim3 grid((p.vocab + kSlice - 1) / kSlice, p.rows);
  if (p.dtype == W4A16_DTYPE_F32)
    k_process_logits<float><<<grid, 256, 0, stream>>>(p);
  else if (p.dtype == W4A16_DTYPE_F16)
    k_process_logits<__half><<<grid, 256, 0, stream>>>(p);
  else
    k_process_logits<__nv_bfloat16><<<grid, 256, 0, stream>>>(p);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    set_error("k_process_logits launch failed: %s", cudaGetErrorString(e));
    return W4A16_ERR_CUDA;
  }
  return W4A16_OK;
}

}  // namespace w4a16
