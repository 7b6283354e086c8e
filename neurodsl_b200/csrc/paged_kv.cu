// paged_kv.cu — the paged key-value cache outside attention: the prefill's
// store and the eviction by accumulated attention weight.
//
// Both move rows of 128 bytes (64 bf16) and are bound by HBM: the store reads
// and writes every token's K and V row once, the eviction reads 4 bytes of
// weight per position and moves the kept rows once.
#include <cuda_bf16.h>
#include <stdint.h>

#include "launch.cuh"
#include "model_ops.h"
#include "paged_kv.h"

namespace nd {
namespace {

constexpr int kVec = 8;   // 16-byte pieces of a row

__device__ __forceinline__ void raise(int* err_word) {
  if (err_word) atomicCAS(err_word, 0, kModelErrIndex);
}

// The row of position `pos` of sequence b and head h in the pool; -1 if the
// position lies past the table or its page is none of the pool's.
__device__ __forceinline__ long long pool_row(const PagedPool& pool, const int* table,
                                              long long table_ld, int max_pages, int b, int h,
                                              long long pos) {
  if (pos < 0 || pos >= static_cast<long long>(max_pages) * pool.page_size) return -1;
  const int page = static_cast<int>(pos / pool.page_size);
  const int row = static_cast<int>(pos - static_cast<long long>(page) * pool.page_size);
  const int id = table[b * table_ld + page];
  if (id < 0 || id >= pool.n_pages) return -1;
  return (static_cast<long long>(id) * pool.Hkv + h) * pool.page_size + row;
}

// ------------------------------------------------------------------- store
// Thread = 16 bytes of one (token, head) row of K and of V.
__global__ void __launch_bounds__(256)
    paged_store_kernel(const __nv_bfloat16* __restrict__ src, long long ld, int k_col, int v_col,
                       const PagedPool pool, int B, int S, int pos0,
                       const int* __restrict__ pos0_dev, const int* __restrict__ lens,
                       int* __restrict__ err_word) {
  pdl_wait();
  pdl_trigger();
  const long long n = static_cast<long long>(B) * S * pool.Hkv * kVec;
  const long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i >= n) return;
  const int c = static_cast<int>(i % kVec);
  const long long r = i / kVec;
  const int h = static_cast<int>(r % pool.Hkv);
  const long long bs = r / pool.Hkv;
  const int s = static_cast<int>(bs % S);
  const int b = static_cast<int>(bs / S);
  if (lens != nullptr) {
    const int len = lens[b];
    if (len < 0 || len > S) raise(err_word);
    if (s >= len) return;   // padding
  }
  const long long pos = static_cast<long long>(pos0_dev ? pos0_dev[b] : pos0) + s;
  const long long row = pool_row(pool, pool.table, pool.table_ld, pool.max_pages, b, h, pos);
  if (row < 0) {
    raise(err_word);
    return;
  }
  const __nv_bfloat16* x = src + bs * ld + h * 64 + c * 8;
  const uint4 kk = *reinterpret_cast<const uint4*>(x + k_col);
  const uint4 vv = *reinterpret_cast<const uint4*>(x + v_col);
  *reinterpret_cast<uint4*>(pool.k + row * 64 + c * 8) = kk;
  *reinterpret_cast<uint4*>(pool.v + row * 64 + c * 8) = vv;
}

// ---------------------------------------------------------------- eviction
// Weights in an order of unsigned integers: NaN lowest, then -inf to +inf,
// the two zeros equal.
__device__ __forceinline__ uint32_t ordered(float w) {
  if (w != w) return 0u;
  const uint32_t u = w == 0.f ? 0u : __float_as_uint(w);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

constexpr int kSelThreads = 1024;

// Exclusive sum over the block of two counts packed as 32 + 32 bits; `total`
// receives the block's sums.
__device__ __forceinline__ unsigned long long block_scan(unsigned long long v,
                                                         unsigned long long* sm,
                                                         unsigned long long& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned long long x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();   // the last call's readers are done
  if (lane == 31) sm[warp] = x;
  __syncthreads();
  unsigned long long base = 0, all = 0;
  for (int w = 0; w < kSelThreads / 32; ++w) {
    if (w < warp) base += sm[w];
    all += sm[w];
  }
  total = all;
  return base + x - v;
}

// One block per (sequence, kv head): which positions stay.  The first `sinks`
// and the last `recent` always do; the rest of the budget goes to the largest
// weights between, found by their value's digits (four passes of 8 bits), the
// lowest positions first among equals.  Writes the kept positions in order,
// their weights, and the new length.
__global__ void __launch_bounds__(kSelThreads)
    paged_select_kernel(const PagedEvict a, int* __restrict__ err_word) {
  __shared__ unsigned int hist[256];
  __shared__ unsigned long long scan_sm[kSelThreads / 32];
  __shared__ uint32_t s_prefix;
  __shared__ int s_need;
  pdl_wait();
  pdl_trigger();
  const int b = blockIdx.x / a.pool.Hkv, h = blockIdx.x % a.pool.Hkv;
  const long long cap = static_cast<long long>(a.pool.max_pages) * a.pool.page_size;
  int L = a.lens[b];
  if (L < 0 || L > cap) {
    if (threadIdx.x == 0) raise(err_word);
    L = L < 0 ? 0 : static_cast<int>(cap);
  }
  const float* w = a.weights + static_cast<size_t>(blockIdx.x) * a.weights_ld;
  float* w_out = a.weights_out + static_cast<size_t>(blockIdx.x) * a.weights_out_ld;
  int* kept = a.kept + static_cast<size_t>(blockIdx.x) * a.budget;
  const int n = L < a.budget ? L : a.budget;
  const bool all = L <= a.budget;
  const int lo = a.sinks, hi = L - a.recent;         // the positions that compete
  const int need = a.budget - a.sinks - a.recent;    // how many of them stay

  uint32_t threshold = 0;
  int ties = 0;            // of those equal to the threshold
  if (!all && need > 0) {
    uint32_t prefix = 0, mask = 0;
    int left = need;
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = threadIdx.x; i < 256; i += kSelThreads) hist[i] = 0;
      __syncthreads();
      for (int i = lo + threadIdx.x; i < hi; i += kSelThreads) {
        const uint32_t u = ordered(w[i]);
        if ((u & mask) == prefix) atomicAdd(&hist[(u >> shift) & 255u], 1u);
      }
      __syncthreads();
      if (threadIdx.x == 0) {
        int rest = left, d = 255;
        while (static_cast<int>(hist[d]) < rest) rest -= static_cast<int>(hist[d--]);
        s_prefix = prefix | (static_cast<uint32_t>(d) << shift);
        s_need = rest;
      }
      __syncthreads();
      prefix = s_prefix;
      left = s_need;
      mask |= 255u << shift;
      __syncthreads();
    }
    threshold = prefix;
    ties = left;
  }

  int slot0 = 0, tie0 = 0;
  for (int base = 0; base < L; base += kSelThreads) {
    const int i = base + threadIdx.x;
    bool sure = false, tie = false;
    float x = 0.f;
    if (i < L) {
      x = w[i];
      if (all || i < lo || i >= hi) {
        sure = true;
      } else if (need > 0) {
        const uint32_t u = ordered(x);
        sure = u > threshold;
        tie = u == threshold;
      }
    }
    unsigned long long sums;
    const unsigned long long at =
        block_scan((static_cast<unsigned long long>(tie) << 32) | sure, scan_sm, sums);
    const int tie_at = tie0 + static_cast<int>(at >> 32);
    const int ties_before = min(tie_at, ties) - min(tie0, ties);
    if (sure || (tie && tie_at < ties)) {
      const int slot = slot0 + static_cast<int>(at & 0xffffffffu) + ties_before;
      kept[slot] = i;
      w_out[slot] = x;
    }
    const int tie1 = tie0 + static_cast<int>(sums >> 32);
    slot0 += static_cast<int>(sums & 0xffffffffu) + min(tie1, ties) - min(tie0, ties);
    tie0 = tie1;
  }
  for (int i = n + threadIdx.x; i < a.budget; i += kSelThreads) kept[i] = -1;
  for (long long i = n + threadIdx.x; i < a.weights_out_ld; i += kSelThreads) w_out[i] = 0.f;
  if (h == 0 && threadIdx.x == 0) a.new_lens[b] = n;
}

// Thread = 16 bytes of one kept (slot, head) row of K and of V.
__global__ void __launch_bounds__(256)
    paged_gather_kernel(const PagedEvict a, int* __restrict__ err_word) {
  pdl_wait();
  pdl_trigger();
  const long long n = static_cast<long long>(a.B) * a.pool.Hkv * a.budget * kVec;
  const long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i >= n) return;
  const int c = static_cast<int>(i % kVec);
  const long long r = i / kVec;
  const int slot = static_cast<int>(r % a.budget);
  const int bh = static_cast<int>(r / a.budget);
  const int b = bh / a.pool.Hkv, h = bh % a.pool.Hkv;
  const int pos = a.kept[r];
  if (pos < 0) return;
  const long long src =
      pool_row(a.pool, a.pool.table, a.pool.table_ld, a.pool.max_pages, b, h, pos);
  const long long dst = pool_row(a.pool, a.out_table, a.out_table_ld, a.out_pages, b, h, slot);
  if (src < 0 || dst < 0) raise(err_word);
  if (dst < 0) return;
  uint4 kk = make_uint4(0, 0, 0, 0), vv = kk;   // a row without a page reads as zeros
  if (src >= 0) {
    kk = *reinterpret_cast<const uint4*>(a.pool.k + src * 64 + c * 8);
    vv = *reinterpret_cast<const uint4*>(a.pool.v + src * 64 + c * 8);
  }
  *reinterpret_cast<uint4*>(a.pool.k + dst * 64 + c * 8) = kk;
  *reinterpret_cast<uint4*>(a.pool.v + dst * 64 + c * 8) = vv;
}

}  // namespace

cudaError_t launch_paged_store(cudaStream_t stream, const __nv_bfloat16* src, long long ld,
                               int k_col, int v_col, const PagedPool& pool, int B, int S, int pos0,
                               const int* pos0_dev, const int* lens, int* err_word) {
  const long long n = static_cast<long long>(B) * S * pool.Hkv * kVec;
  if (n == 0) return cudaSuccess;
  return launch_ex(paged_store_kernel, dim3(static_cast<unsigned>((n + 255) / 256)), dim3(256), 0,
                   stream, 1, true, src, ld, k_col, v_col, pool, B, S, pos0, pos0_dev, lens,
                   err_word);
}

cudaError_t launch_paged_evict(cudaStream_t stream, const PagedEvict& a, int* err_word) {
  const unsigned heads = static_cast<unsigned>(a.B * a.pool.Hkv);
  if (heads == 0) return cudaSuccess;
  cudaError_t e = launch_ex(paged_select_kernel, dim3(heads), dim3(kSelThreads), 0, stream, 1, true,
                            a, err_word);
  if (e != cudaSuccess) return e;
  const long long n = static_cast<long long>(heads) * a.budget * kVec;
  return launch_ex(paged_gather_kernel, dim3(static_cast<unsigned>((n + 255) / 256)), dim3(256), 0,
                   stream, 1, true, a, err_word);
}

}  // namespace nd
