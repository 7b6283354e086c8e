// paged_kv.cu — the paged key-value cache outside attention: the prefill's
// store and the eviction by accumulated attention weight.
//
// Both move rows of 128 bytes (64 bf16) and are bound by HBM: the store reads
// and writes every token's K and V row once, the eviction reads 4 bytes of
// weight per position and moves the kept rows once.
//
// The kernels that write the cache do not let the next kernel start early: the
// contiguous decode attention, with programmatic launch on, reads cached rows
// before it waits.
#include <cuda_bf16.h>
#include <stdint.h>

#include "launch.cuh"
#include "model_ops.h"
#include "paged_kv.h"

namespace nd {
namespace {

constexpr int kVec = 8;   // 16-byte pieces of a row
constexpr int kMaxShared = 54 * 1024;   // weights in shared memory, beside the histogram

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
// A warp takes 32 pieces of 16 bytes (four heads) of kTokens consecutive tokens
// of one sequence, whose rows of a head are neighbours in a page: a lane looks
// a token's row up, then all K and V loads go out before the first store.  Four
// tokens a warp keep enough bytes in flight for a long prompt (65536 tokens, half of
// them padding, 12 heads: 35.9 us; with a thread for each 16 bytes 43.4); with few tokens, one a warp spreads them over more SMs.
template <int kTokens>
__global__ void __launch_bounds__(256)
    paged_store_kernel(const __nv_bfloat16* __restrict__ src, long long ld, int k_col, int v_col,
                       const PagedPool pool, int B, int S, int pos0,
                       const int* __restrict__ pos0_dev, const int* __restrict__ lens,
                       int* __restrict__ err_word) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const long long w = static_cast<long long>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int per_seq = (S + kTokens - 1) / kTokens, chunks = (pool.Hkv * kVec + 31) / 32;
  const long long group = w / chunks;
  const int p = static_cast<int>(w - group * chunks) * 32 + lane;   // this lane's piece of a token
  const int b = static_cast<int>(group / per_seq);
  if (b >= B) return;
  const int s0 = static_cast<int>(group - static_cast<long long>(b) * per_seq) * kTokens;
  int len = S;
  if (lens != nullptr) {
    len = lens[b];
    if (len < 0 || len > S) {
      if (s0 == 0 && p == 0) raise(err_word);
      len = len < 0 ? 0 : S;
    }
  }
  if (s0 >= len) return;   // padding
  long long row = -1;      // of lane's token, head 0
  if (lane < kTokens && s0 + lane < len) {
    const long long pos = static_cast<long long>(pos0_dev ? pos0_dev[b] : pos0) + s0 + lane;
    row = pool_row(pool, pool.table, pool.table_ld, pool.max_pages, b, 0, pos);
    if (row < 0) raise(err_word);
  }
  long long rows[kTokens];
#pragma unroll
  for (int i = 0; i < kTokens; ++i) rows[i] = __shfl_sync(0xffffffffu, row, i);
  const __nv_bfloat16* x = src + (static_cast<long long>(b) * S + s0) * ld;
  const long long head = static_cast<long long>(pool.page_size) * 64;   // from head to head
  if (p >= pool.Hkv * kVec) return;
  uint4 kk[kTokens], vv[kTokens];
#pragma unroll
  for (int i = 0; i < kTokens; ++i)
    if (rows[i] >= 0) {
      kk[i] = *reinterpret_cast<const uint4*>(x + i * ld + k_col + p * 8);
      vv[i] = *reinterpret_cast<const uint4*>(x + i * ld + v_col + p * 8);
    }
  const long long off = (p / kVec) * head + (p % kVec) * 8;
#pragma unroll
  for (int i = 0; i < kTokens; ++i)
    if (rows[i] >= 0) {
      *reinterpret_cast<uint4*>(pool.k + rows[i] * 64 + off) = kk[i];
      *reinterpret_cast<uint4*>(pool.v + rows[i] * 64 + off) = vv[i];
    }
}

// ---------------------------------------------------------------- eviction
// Weights in an order of unsigned integers: 1 for NaN, the lowest, then -inf to
// +inf, the two zeros equal; 0 is left for "no weight".
__device__ __forceinline__ uint32_t ordered(float w) {
  if (w != w) return 1u;
  const uint32_t u = w == 0.f ? 0u : __float_as_uint(w);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// A warp moves 32 kept rows of one (sequence, kv head), a lane's from position
// `pos` (-1: none) to `slot`: a lane looks its row up, then eight lanes move a row,
// 4 rows of K and V an instruction and 16 in flight.
__device__ __forceinline__ void gather_rows(const PagedEvict& a, int b, int h, int slot, int pos, int* err_word) {
  const int lane = threadIdx.x & 31;
  long long src = -1, dst = -1;
  if (pos >= 0) {
    src = pool_row(a.pool, a.pool.table, a.pool.table_ld, a.pool.max_pages, b, h, pos);
    dst = pool_row(a.pool, a.out_table, a.out_table_ld, a.out_pages, b, h, slot);
    if (src < 0 || dst < 0) raise(err_word);
  }
  if (!__any_sync(0xffffffffu, dst >= 0)) return;
  const int c = (lane & 7) * 8;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    uint4 kk[4], vv[4];
    long long to[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = half * 16 + i * 4 + (lane >> 3);
      const long long from = __shfl_sync(0xffffffffu, src, r);
      to[i] = __shfl_sync(0xffffffffu, dst, r);
      kk[i] = vv[i] = make_uint4(0, 0, 0, 0);   // a row without a page reads as zeros
      if (from >= 0 && to[i] >= 0) {
        kk[i] = *reinterpret_cast<const uint4*>(a.pool.k + from * 64 + c);
        vv[i] = *reinterpret_cast<const uint4*>(a.pool.v + from * 64 + c);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (to[i] >= 0) {
        *reinterpret_cast<uint4*>(a.pool.k + to[i] * 64 + c) = kk[i];
        *reinterpret_cast<uint4*>(a.pool.v + to[i] * 64 + c) = vv[i];
      }
  }
}

// A length between 0 and what the table holds.
__device__ __forceinline__ int cut(const PagedEvict& a, int L) {
  const long long cap = static_cast<long long>(a.pool.max_pages) * a.pool.page_size;
  return L < 0 ? 0 : L > cap ? static_cast<int>(cap) : L;
}

// One block per (sequence, kv head): which positions stay.  The first `sinks`
// and the last `recent` always do; the rest of the budget goes to the largest
// weights between, the lowest positions first among equals.  The weights stay in
// registers (kR a thread) or, for longer caches, in shared memory (kShared) or, for
// the longest, are read again each time, from L2: every warp owns a contiguous span of positions, lane by
// lane, so that ballots and one sum over the warps give each kept position its
// slot.  The smallest weight that stays is found by its digits of 11, 11 and 10
// bits, from the top of an order-preserving integer, with a histogram in shared
// memory each; from the second digit on only the few weights that share the
// digits so far take part.  (Two bits at a time by counting, without
// atomics, is 16 passes over all weights: 36 us for 256 heads of up to 8192
// keys, against 16.5 with these.)
//
// kGather: the block then moves its rows itself (the launcher's rule), from the
// positions left in the histogram's memory, and writes the new length, which is
// then not where the other heads' blocks read the old one.
template <int kThreads, int kR, bool kGather, bool kShared>
__global__ void __launch_bounds__(kThreads, kThreads < 1024 ? 2 : 1)
    paged_select_kernel(const PagedEvict a, int* __restrict__ err_word) {
  constexpr int kW = kThreads / 32;
  constexpr int kBins = 2048, kPer = kBins / kThreads;   // bins a thread
  constexpr int kAll = 1 << 30;
  __shared__ uint32_t hist[kBins];
  __shared__ uint32_t warp_sum[kW];
  __shared__ uint32_t found_digit;
  __shared__ int found_above;
  __shared__ int sure_sm[kW], tie_sm[kW];
  pdl_wait();
  if (!kGather) pdl_trigger();   // what follows a writing of the cache starts when that is done
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int b = blockIdx.x / a.pool.Hkv, h = blockIdx.x % a.pool.Hkv;
  const long long cap = static_cast<long long>(a.pool.max_pages) * a.pool.page_size;
  int L = a.lens[b];
  if (L < 0 || L > cap) {
    if (threadIdx.x == 0) raise(err_word);
    L = cut(a, L);
  }
  const float* w = a.weights + static_cast<size_t>(blockIdx.x) * a.weights_ld;
  float* w_out = a.weights_out + static_cast<size_t>(blockIdx.x) * a.weights_out_ld;
  int* kept = a.kept + static_cast<size_t>(blockIdx.x) * a.budget;
  const int n = L < a.budget ? L : a.budget;
  const bool all = L <= a.budget;
  const int lo = a.sinks, hi = L - a.recent;         // the positions that compete
  const int need = a.budget - a.sinks - a.recent;    // how many of them stay

  // rows of 32 positions a warp takes, and its first position
  const int rows = kR > 0 ? kR : (L + kThreads - 1) / kThreads;
  const int p0 = warp * rows * 32 + lane;
  // a position's ordered weight, 0 where it does not compete
  auto read = [&](int r) -> uint32_t {
    const int p = p0 + 32 * r;
    return p >= lo && p < hi ? ordered(w[p]) : 0u;
  };
  constexpr bool kKeep = kR > 0 && kR <= 16;   // the weights themselves in registers too
  uint32_t x[kR > 0 ? kR : 1];
  constexpr int kStep = kKeep ? kR : 8;        // weights in flight a thread
  float v[kKeep ? kR : kStep];
  if constexpr (kR > 0) {
#pragma unroll
    for (int r0 = 0; r0 < kR; r0 += kStep) {
#pragma unroll
      for (int r = r0; r < r0 + kStep; ++r) v[kKeep ? r : r - r0] = p0 + 32 * r < L ? w[p0 + 32 * r] : 0.f;
#pragma unroll
      for (int r = r0; r < r0 + kStep; ++r)
        x[r] = p0 + 32 * r >= lo && p0 + 32 * r < hi ? ordered(v[kKeep ? r : r - r0]) : 0u;
    }
  }
  extern __shared__ uint32_t x_sm[];
  if constexpr (kShared) {   // each thread reads its own again
    for (int r = 0; r < rows; ++r) x_sm[p0 + 32 * r] = read(r);
  }
  auto weight = [&](int r) -> uint32_t {
    if constexpr (kR > 0) return x[r];
    else if constexpr (kShared) return x_sm[p0 + 32 * r];
    else return read(r);
  };

  // threshold: the largest value with at least `need` weights at or above it
  uint32_t threshold = 0;
  int above = 0;           // weights above the threshold
  if (!all && need > 0) {
#pragma unroll (kR > 16 ? 1 : 3)   // unrolled the 24 would spill
    for (int digit = 0; digit < 3; ++digit) {
      const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0;
      const uint32_t bins = digit == 2 ? 1023u : 2047u;
#pragma unroll
      for (int i = 0; i < kPer; ++i) hist[i * kThreads + threadIdx.x] = 0;
      __syncthreads();
#pragma unroll
      for (int r = 0; r < (kR > 0 ? kR : kAll); ++r) {
        if (kR == 0 && r >= rows) break;
        const uint32_t u = weight(r);
        const uint32_t known = digit == 0 ? 0u : (u ^ threshold) >> (digit == 1 ? 21 : 10);
        if (u != 0 && known == 0) atomicAdd(&hist[u >> shift & bins], 1u);
      }
      __syncthreads();
      // bins from the highest down: thread i takes the kPer below its neighbour's
      const int first = kBins - 1 - static_cast<int>(threadIdx.x) * kPer;
      uint32_t mine = 0;
#pragma unroll
      for (int i = 0; i < kPer; ++i) mine += hist[first - i];
      uint32_t upto = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
      }
      if (lane == 31) warp_sum[warp] = upto;
      __syncthreads();
      upto += __reduce_add_sync(0xffffffffu, lane < warp && lane < kW ? warp_sum[lane] : 0u);
      const uint32_t left = static_cast<uint32_t>(need - above);
      if (upto >= left && upto - mine < left) {      // one thread's bins reach it
        uint32_t c = upto - mine;
        int i = 0;
        while (c + hist[first - i] < left) c += hist[first - i++];
        found_digit = static_cast<uint32_t>(first - i);
        found_above = above + static_cast<int>(c);
      }
      __syncthreads();
      threshold |= found_digit << shift;
      above = found_above;
    }
  }
  const int ties = need - above;   // of the weights equal to the threshold

  // how many each warp keeps for certain, and how many equal the threshold
  // (with the weights in registers, a bit a position)
  auto is_sure = [&](int r) {
    const int p = p0 + 32 * r;
    return p < L && (all || p < lo || p >= hi || (need > 0 && weight(r) > threshold));
  };
  auto is_tie = [&](int r) { return !all && need > 0 && weight(r) == threshold; };   // threshold > 0
  uint32_t sure_bits = 0, tie_bits = 0;
  if constexpr (kR > 0) {
    const uint32_t t_up = !all && need > 0 ? threshold : ~0u;   // nothing lies above, or ties, ~0
#pragma unroll
    for (int r = 0; r < kR; ++r) {
      sure_bits |= static_cast<uint32_t>(x[r] > t_up) << r;
      tie_bits |= static_cast<uint32_t>(x[r] == t_up) << r;
    }
    // the positions that do not compete: rows r with p0 + 32 r below a bound are
    // the lowest bits
    auto lowest = [&](int bound) {
      const int m = min(max((bound - p0 + 31) >> 5, 0), 32);
      return m < 32 ? (1u << m) - 1u : ~0u;
    };
    constexpr uint32_t kRows = kR < 32 ? (1u << kR) - 1u : ~0u;
    sure_bits |= kRows & lowest(L) & (all ? ~0u : lowest(lo) | ~lowest(hi));
  }
  int n_sure = 0, n_tie = 0;
#pragma unroll
  for (int r = 0; r < (kR > 0 ? kR : kAll); ++r) {
    if (kR == 0 && r >= rows) break;
    n_sure += __popc(__ballot_sync(0xffffffffu, kR > 0 ? sure_bits >> r & 1u : is_sure(r)));
    n_tie += __popc(__ballot_sync(0xffffffffu, kR > 0 ? tie_bits >> r & 1u : is_tie(r)));
  }
  if (lane == 0) {
    sure_sm[warp] = n_sure;
    tie_sm[warp] = n_tie;
  }
  __syncthreads();
  const bool before = lane < warp && lane < kW;
  int slot = __reduce_add_sync(0xffffffffu, before ? static_cast<unsigned>(sure_sm[lane]) : 0u);
  int tie_at = __reduce_add_sync(0xffffffffu, before ? static_cast<unsigned>(tie_sm[lane]) : 0u);
  slot += min(tie_at, ties);
  const uint32_t below = (1u << lane) - 1u;
#pragma unroll
  for (int r = 0; r < (kR > 0 ? kR : kAll); ++r) {
    if (kR == 0 && r >= rows) break;
    const bool tie = kR > 0 ? tie_bits >> r & 1u : is_tie(r);
    const uint32_t m_tie = __ballot_sync(0xffffffffu, tie);
    const bool keep = (kR > 0 ? sure_bits >> r & 1u : is_sure(r)) || (tie && tie_at + __popc(m_tie & below) < ties);
    const uint32_t m = __ballot_sync(0xffffffffu, keep);
    if (keep) {
      const int at = slot + __popc(m & below);
      kept[at] = p0 + 32 * r;
      if (kGather) hist[at] = static_cast<uint32_t>(p0 + 32 * r);
      w_out[at] = kKeep ? v[kKeep ? r : 0] : w[p0 + 32 * r];
    }
    slot += __popc(m);
    tie_at += __popc(m_tie);
  }
  if constexpr (kGather) {
    __syncthreads();
    for (int i = warp * 32; i < n; i += kThreads) {
      const int slot = i + lane;
      gather_rows(a, b, h, slot, slot < n ? static_cast<int>(hist[slot]) : -1, err_word);
    }
  }
  for (int i = n + threadIdx.x; i < a.budget; i += kThreads) kept[i] = -1;
  // zeros behind the kept weights, 16 bytes at a time where the rows allow
  long long z = n;
  if (a.weights_out_ld % 4 == 0 && (reinterpret_cast<uintptr_t>(w_out) & 15) == 0) {
    const long long z4 = (z + 3) / 4, e4 = a.weights_out_ld / 4;
    if (z + threadIdx.x < 4 * z4) w_out[z + threadIdx.x] = 0.f;
#pragma unroll 4
    for (long long i = z4 + threadIdx.x; i < e4; i += kThreads)
      reinterpret_cast<float4*>(w_out)[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  } else {
    for (long long i = z + threadIdx.x; i < a.weights_out_ld; i += kThreads) w_out[i] = 0.f;
  }
  if (kGather && h == 0 && threadIdx.x == 0) a.new_lens[b] = n;
}

// The rows of all heads, and the new lengths: every selection has read the old ones
// by now, so they may be written in their place.
__global__ void __launch_bounds__(256)
    paged_gather_kernel(const PagedEvict a, int* __restrict__ err_word) {
  pdl_wait();
  const int per_head = (a.budget + 31) / 32;
  const long long w = static_cast<long long>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const long long bh = w / per_head;
  if (bh >= static_cast<long long>(a.B) * a.pool.Hkv) return;
  const int slot = static_cast<int>(w - bh * per_head) * 32 + (threadIdx.x & 31);
  const int b = static_cast<int>(bh / a.pool.Hkv), h = static_cast<int>(bh % a.pool.Hkv);
  if (h == 0 && slot == 0) a.new_lens[b] = min(cut(a, a.lens[b]), a.budget);   // one thread a sequence
  gather_rows(a, b, h, slot, slot < a.budget ? a.kept[bh * a.budget + slot] : -1, err_word);
}

template <int kThreads, int kR, bool kGather = false, bool kShared = false>
cudaError_t launch_select(cudaStream_t stream, const PagedEvict& a, unsigned heads, int* err_word) {
  auto kern = paged_select_kernel<kThreads, kR, kGather, kShared>;
  size_t smem = 0;
  if (kShared) {
    const size_t cap = static_cast<size_t>(a.pool.max_pages) * a.pool.page_size;
    smem = (cap + kThreads - 1) / kThreads * kThreads * sizeof(uint32_t);
    static SmemOptIn opt_in;
    const cudaError_t e = allow_smem(kern, static_cast<int>(smem), opt_in);
    if (e != cudaSuccess) return e;
  }
  return launch_dependent(kern, dim3(heads), dim3(kThreads), smem, stream, 1, a, err_word);
}

}  // namespace

cudaError_t launch_paged_store(cudaStream_t stream, const __nv_bfloat16* src, long long ld,
                               int k_col, int v_col, const PagedPool& pool, int B, int S, int pos0,
                               const int* pos0_dev, const int* lens, int* err_word) {
  if (B == 0 || S == 0 || pool.Hkv == 0) return cudaSuccess;
  const long long chunks = (static_cast<long long>(pool.Hkv) * kVec + 31) / 32;
  const bool few = B * static_cast<long long>(S) * chunks < 32 * current_sm_count();
  const long long warps = chunks * B * (few ? S : (S + 3) / 4);
  return launch_dependent(few ? paged_store_kernel<1> : paged_store_kernel<4>,
                          dim3(static_cast<unsigned>((warps + 7) / 8)), dim3(256), 0, stream, 1, src,
                          ld, k_col, v_col, pool, B, S, pos0, pos0_dev, lens, err_word);
}

cudaError_t launch_paged_evict(cudaStream_t stream, const PagedEvict& a, int* err_word) {
  const unsigned heads = static_cast<unsigned>(a.B * a.pool.Hkv);
  if (heads == 0) return cudaSuccess;
  // Weights in registers as far as they go without spilling, then in shared memory:
  // for 12 heads of 16000 keys cut to 2000 16.6 us (32 a thread: 42.0), of 24000
  // 22.9 (42.5, from L2 41.0), of 32000 cut to 4000 48.2 (49.6, from L2 62.7).
  const long long cap = static_cast<long long>(a.pool.max_pages) * a.pool.page_size;
  cudaError_t e;
  // One launch, each block moving its head's rows, but where that leaves SMs idle:
  // few heads with many rows, or a third round of blocks (two fit an SM) that is
  // nearly empty.  12 heads, 256 of 500 keys: 6.2 us against 8.1 in two launches; 512
  // of 8192: 12.0 against 12.9; 1024 of 8192: 14.9 against 13.1, with 144 heads 24.7
  // against 27.1, with 240 35.8 against 40.3, with 320 51.5 against 54.0 but 2048 of
  // them 86.9 against 81.0, with 512 67.3 against 76.6.
  // Lengths that are written in place take two launches.
  const unsigned sms = static_cast<unsigned>(current_sm_count());
  if (a.new_lens != a.lens && cap <= 8192 && a.budget <= 2048 && (heads > sms / 2 || a.budget <= 512) && (heads <= 2 * sms || heads > 3 * sms)) {
    if (cap <= 1024) return launch_select<512, 2, true>(stream, a, heads, err_word);
    return heads <= sms ? launch_select<1024, 8, true>(stream, a, heads, err_word)
                        : launch_select<512, 16, true>(stream, a, heads, err_word);
  }
  if (cap <= 1024)
    e = launch_select<256, 4>(stream, a, heads, err_word);
  else if (cap <= 8192)
    e = launch_select<512, 16>(stream, a, heads, err_word);
  else if (cap <= 16384)
    e = launch_select<1024, 16>(stream, a, heads, err_word);
  else if (cap <= 24576)
    e = launch_select<1024, 24>(stream, a, heads, err_word);
  else if (cap <= kMaxShared)
    e = launch_select<1024, 0, false, true>(stream, a, heads, err_word);
  else
    e = launch_select<1024, 0>(stream, a, heads, err_word);
  if (e != cudaSuccess) return e;
  const long long warps = static_cast<long long>(heads) * ((a.budget + 31) / 32);
  return launch_dependent(paged_gather_kernel, dim3(static_cast<unsigned>((warps + 7) / 8)), dim3(256),
                          0, stream, 1, a, err_word);
}

}  // namespace nd
