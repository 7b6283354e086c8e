// logits.cu — what stands between the LM head's logits and the choice of a
// token: penalties for tokens of the history, sparse biases and a grammar
// mask, in one pass, with the greedy token.
//
// Per row, for token v with c = its count in the row's history:
//   x = logits[v]
//   c > 0:  x = x > 0 ? x / repetition : x * repetition
//           x = x - presence;  x = x - frequency * c
//   x = x + sum of the biases listed for v (in list order)
//   mask bit 0:  x = -inf
// Each operation is rounded to fp32 once, in this order (no fused multiply-add),
// so that the greedy token does not depend on how the compiler combines them.
//
// Bound: HBM, one read and one write of the logits.  A block takes a slice of
// a row's vocabulary, counts the history's tokens that fall into it in shared
// memory (integers: the order of the atomics does not matter) and streams the
// slice once.  Each slice reads the whole history; it is short beside the
// slice and comes from L2.
#include <cuda_bf16.h>
#include <stdint.h>

#include "launch.cuh"
#include "logits.h"
#include "model_ops.h"

namespace nd {
namespace {

constexpr int kThreads = 256;
constexpr int kSlice = 4096;   // tokens of a block

__device__ __forceinline__ float load_f(const float* p) { return *p; }
__device__ __forceinline__ float load_f(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void store_f(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_f(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

template <typename TI, typename TO>
__global__ void __launch_bounds__(kThreads)
    logits_penalty_kernel(const LogitsPenalty a, int* __restrict__ err_word) {
  __shared__ int count[kSlice];
  __shared__ float bias[kSlice];
  pdl_wait();
  pdl_trigger();
  const int row = blockIdx.y;
  const int v0 = blockIdx.x * kSlice;
  const int n = min(kSlice, a.V - v0);
  for (int i = threadIdx.x; i < kSlice; i += kThreads) {
    count[i] = 0;
    bias[i] = 0.f;
  }
  __syncthreads();
  if (a.history != nullptr) {
    const int* hist = a.history + row * a.history_ld;
    int len = a.history_lens ? a.history_lens[row] : a.n_history;
    if (len < 0 || len > a.n_history) {
      if (threadIdx.x == 0 && err_word) atomicCAS(err_word, 0, kModelErrIndex);
      len = len < 0 ? 0 : a.n_history;
    }
    for (int i = threadIdx.x; i < len; i += kThreads) {
      const int t = hist[i];
      if (t >= a.V && err_word) atomicCAS(err_word, 0, kModelErrIndex);
      if (t >= v0 && t < v0 + n) atomicAdd(&count[t - v0], 1);
    }
  }
  // biases: one warp, in list order; entries of a warp's 32 that name the
  // same token are added by the lowest lane that names it
  if (a.bias_ids != nullptr && threadIdx.x < 32) {
    const int lane = threadIdx.x;
    const int* ids = a.bias_ids + static_cast<long long>(row) * a.n_bias;
    const float* val = a.bias + static_cast<long long>(row) * a.n_bias;
    for (int i0 = 0; i0 < a.n_bias; i0 += 32) {
      const int i = i0 + lane;
      const int t = i < a.n_bias ? ids[i] : -1;
      if (t >= a.V && err_word) atomicCAS(err_word, 0, kModelErrIndex);
      const bool in = t >= v0 && t < v0 + n;
      const float x = in ? val[i] : 0.f;
      const unsigned same = __match_any_sync(0xffffffffu, in ? t : -1);
      float sum = in ? bias[t - v0] : 0.f;
      for (int l = 0; l < 32; ++l) {
        const float y = __shfl_sync(0xffffffffu, x, l);
        if (in && (same >> l & 1u)) sum += y;
      }
      __syncwarp();
      if (in) bias[t - v0] = sum;   // every lane of `same` holds the same sum
      __syncwarp();
    }
  }
  __syncthreads();
  const float rep = a.repetition ? a.repetition[row] : 1.f;
  const float pres = a.presence ? a.presence[row] : 0.f;
  const float freq = a.frequency ? a.frequency[row] : 0.f;
  const TI* in = static_cast<const TI*>(a.logits) + row * a.ld + v0;
  TO* out = static_cast<TO*>(a.out) + row * a.out_ld + v0;
  const unsigned int* mask = a.mask ? a.mask + row * a.mask_ld : nullptr;
  for (int i = threadIdx.x; i < n; i += kThreads) {
    float x = load_f(in + i);
    const int c = count[i];
    if (c > 0) {
      if (a.repetition) x = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
      if (a.presence) x = __fsub_rn(x, pres);
      if (a.frequency) x = __fsub_rn(x, __fmul_rn(freq, static_cast<float>(c)));
    }
    if (a.bias_ids) x = __fadd_rn(x, bias[i]);
    if (mask && !(mask[(v0 + i) >> 5] >> ((v0 + i) & 31) & 1u)) x = -INFINITY;
    store_f(out + i, x);
  }
}

}  // namespace

cudaError_t launch_logits_penalty(cudaStream_t stream, const LogitsPenalty& a, int* err_word) {
  if (a.rows == 0 || a.V == 0) return cudaSuccess;
  const dim3 grid((a.V + kSlice - 1) / kSlice, a.rows);
  cudaError_t e;
#define ND_LOGITS(I, O) \
  e = launch_ex(logits_penalty_kernel<I, O>, grid, dim3(kThreads), 0, stream, 1, true, a, err_word)
  if (a.in_f32) {
    if (a.out_f32) ND_LOGITS(float, float); else ND_LOGITS(float, __nv_bfloat16);
  } else {
    if (a.out_f32) ND_LOGITS(__nv_bfloat16, float); else ND_LOGITS(__nv_bfloat16, __nv_bfloat16);
  }
#undef ND_LOGITS
  if (e != cudaSuccess || a.idx == nullptr) return e;
  return launch_argmax(stream, a.out, a.out_f32, a.out_ld, a.rows, a.V, a.idx, nullptr);
}

}  // namespace nd
