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
// Bound: HBM, one read and one write of the logits.  A row is one CTA's, or a
// cluster's when there are few rows, each CTA taking a contiguous part of the
// vocabulary.  A CTA first enters the listed tokens of its part (history and
// biases) into a hash table in shared memory, with their counts; the first to
// enter a token takes it off the part's bit map of allowed tokens and sends for
// its logit (an asynchronous copy that no one waits for).  Then the CTA streams its
// part without a barrier, -inf for what the map lacks, and at the end computes and
// writes the listed tokens.  So the stream, which runs at the copy rate (23 us for
// 512 rows of 50257, bf16 to fp32), does not branch, and what precedes it is two
// trips to memory.  Earlier forms: every penalty inside the stream and a count for
// each token of a slice, the lists read once a slice, 161 us for those rows with
// histories of 1024; listed tokens looked up and read again after each round of the
// stream, 45.9; the logits of the listed tokens read at the end, 45.5; now 37.8 (44.0
// where a history's tokens are all different, 46.6 before).  The rest over the
// stream's time: the lists 6 us, the listed tokens' writing 4, four rows on some SMs
// and three on others.  Counts are integers, so the order of the atomics does not
// matter; biases are summed by one warp in list order.  The CTAs' best tokens meet
// in distributed shared memory, so the logits are not read again for the argmax.
#include <cuda_bf16.h>
#include <stdint.h>

#include <type_traits>

#include "argmax.cuh"
#include "launch.cuh"
#include "logits.h"
#include "model_ops.h"
#include "ptx.cuh"

namespace nd {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxPart = 1 << 18;               // tokens of the bit map
constexpr int kCluster = 8;                     // CTAs of a row, at most
constexpr int kMaxTable = 8192;                 // table entries
constexpr int kBiased = 1 << 31;                // flag beside a token in the table
constexpr int kForbidden = -0x7fffffff - 1;     // taken off a forbidden token's count
constexpr int kNone = 0x7fffffff;

template <typename T>
__device__ __forceinline__ float load_f(const T* p) {
  return static_cast<float>(*p);
}
template <typename T>
__device__ __forceinline__ T rounded(float x) {
  if constexpr (sizeof(T) == 4) return x;
  else return __float2bfloat16_rn(x);
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __forceinline__ float warp_max(float x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
  return x;
}
// kN values as they lie in memory (8 or 16 bytes).
template <typename T, int kN>
struct Piece {
  uint32_t w[kN * sizeof(T) / 4];
  template <bool kVec>   // else one by one
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (!kVec) {
#pragma unroll
      for (int e = 0; e < kN; e += 4 / sizeof(T)) {
        if constexpr (sizeof(T) == 4)
          w[e] = __float_as_uint(p[e]);
        else
          w[e / 2] = __bfloat16_as_ushort(p[e]) | static_cast<uint32_t>(__bfloat16_as_ushort(p[e + 1])) << 16;
      }
    } else if constexpr (sizeof(w) == 16) {
      const uint4 v = *reinterpret_cast<const uint4*>(p);
      w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    } else {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      w[0] = v.x, w[1] = v.y;
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (sizeof(w) == 16)
      *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    else
      *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  }
  __device__ __forceinline__ void unpack(float (&x)[kN]) const {
#pragma unroll
    for (int e = 0; e < kN; ++e) {
      if constexpr (sizeof(T) == 4) x[e] = __uint_as_float(w[e]);
      else x[e] = __uint_as_float(e & 1 ? w[e / 2] & 0xFFFF0000u : w[e / 2] << 16);
    }
  }
  __device__ __forceinline__ void pack(const float (&x)[kN]) {
#pragma unroll
    for (int e = 0; e < kN; e += sizeof(T) == 4 ? 1 : 2) {
      if constexpr (sizeof(T) == 4) w[e] = __float_as_uint(x[e]);
      else w[e / 2] = pack_bf16x2(x[e], x[e + 1]);
    }
  }
};

// Values move in groups of kN: 16 bytes of the wider type, so that a warp's
// loads and stores each cover contiguous bytes.  Groups are aligned in the output.
// kVec: a row's input and output have the same place within a group, so that they
// are aligned in the input too (the launcher checks); else their values are loaded
// one by one (a padded input and a tight output, 512 rows of 50257, bf16 to fp32:
// 43 us for 34; all token by token 112).
// In shared memory `table` entries (a multiple of four) for the listed tokens,
// n_sums for those with a bias, and a bit map of `part` tokens (a multiple of 32),
// which a CTA takes at a time.
template <typename TI, typename TO, bool kVec>
__global__ void __launch_bounds__(kThreads, 4)
    logits_penalty_kernel(const LogitsPenalty a, int table, int n_sums, int part, int* __restrict__ err_word) {
  constexpr int kN = sizeof(TI) + sizeof(TO) == 4 ? 8 : 4;   // 8: both bf16
  // groups in flight a thread: four of 16 bytes to load would spill
  constexpr int kUnroll = sizeof(TI) + sizeof(TO) == 6 ? 4 : 3;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  int* key = reinterpret_cast<int*>(smem_raw);                  // token and the flag kBiased, -1: free
  int* count = key + table;                                     // below zero: the mask forbids it
  uint32_t* value = reinterpret_cast<uint32_t*>(count + table); // the word of the token's logit
  int* bias_key = reinterpret_cast<int*>(value + table);        // the biased tokens once more, with
  float* bias = reinterpret_cast<float*>(bias_key + n_sums);    // the sums of their biases
  uint32_t* bits = reinterpret_cast<uint32_t*>(bias + n_sums);  // tokens that the stream keeps
  __shared__ float best_v[kThreads / 32], cta_v;
  __shared__ int best_i[kThreads / 32], cta_i;
  const int nc = static_cast<int>(cluster_nctarank()), rank = static_cast<int>(cluster_ctarank());
  const int row = blockIdx.x / nc;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const TI* in = static_cast<const TI*>(a.logits) + row * a.ld;
  TO* out = static_cast<TO*>(a.out) + row * a.out_ld;
  // tokens before the first aligned group; group k holds tokens head + kN k ...,
  // and group -1, if there are such tokens, them
  const int head = static_cast<int>((kN - (reinterpret_cast<uintptr_t>(out) / sizeof(TO)) % kN) % kN);
  const int first = head > 0 ? -1 : 0;
  const int n_groups = (a.V - head + kN - 1) / kN - first;
  const int per = (n_groups + nc - 1) / nc;
  const int g_begin = first + rank * per, g_end = first + min(n_groups, (rank + 1) * per);
  const bool lists = table > 0;
  const int* hist = a.history ? a.history + row * a.history_ld : nullptr;
  const int* ids = a.bias_ids ? a.bias_ids + static_cast<long long>(row) * a.n_bias : nullptr;
  const int n_bias = ids ? a.n_bias : 0;
  const uint32_t* words = a.mask ? a.mask + row * a.mask_ld : nullptr;
  const int n_words = (a.V + 31) >> 5;
  auto clear_tables = [&]() {
    for (int i = threadIdx.x; i < table / 4; i += kThreads) {
      reinterpret_cast<int4*>(key)[i] = make_int4(-1, -1, -1, -1);
      reinterpret_cast<int4*>(count)[i] = make_int4(0, 0, 0, 0);
    }
    for (int i = threadIdx.x; i < n_sums; i += kThreads) {
      bias_key[i] = -1;
      bias[i] = 0.f;
    }
  };
  clear_tables();
  pdl_wait();
  pdl_trigger();

  // The lists' first entries and the mask before everything else: they are what
  // the stream waits for.  The rows of the history are read whole; its length
  // says which entries count.
  auto read = [&](const int* list, int n, int i, int (&t)[4]) {
#pragma unroll
    for (int u = 0; u < 4; ++u) t[u] = i + u * kThreads < n ? list[i + u * kThreads] : -1;
  };
  int th[4], tb[4];
  read(hist, a.n_history, threadIdx.x, th);
  read(ids, n_bias, threadIdx.x, tb);
  int n_hist = a.n_history;
  if (a.history_lens) n_hist = a.history_lens[row];
  float rep = 1.f, pres = 0.f, freq = 0.f;
  if (a.repetition) rep = a.repetition[row];
  if (a.presence) pres = a.presence[row];
  if (a.frequency) freq = a.frequency[row];

  float bv = -INFINITY;
  int bi = kNone;
  // open addressing in a table of n entries
  auto slot_of = [](int t, int n) { return static_cast<int>(__umulhi(static_cast<uint32_t>(t) * 2654435761u, n)); };
  auto after = [](int s, int n) { return s + 1 < n ? s + 1 : 0; };
  auto finish = [&](int t, float x) {
    out[t] = rounded<TO>(x);
    x = static_cast<float>(rounded<TO>(x));
    if (x == x) better(bv, bi, x, t);
  };
  for (int g0 = g_begin; g0 < g_end; g0 += part / kN) {
    const int g1 = min(g_end, g0 + part / kN);
    const int t0 = max(0, head + kN * g0), t1 = min(a.V, head + kN * g1);   // the part's tokens
    // whole groups [ga, gz); their loads run one round ahead, the first round's
    // while the lists are worked through
    const int ga = max(g0, 0), gz = max(ga, min(g1, (a.V - head) / kN));
    constexpr int kRound = kUnroll * kThreads;
    if (g0 != g_begin) {
      __syncthreads();   // the last part's map and tables have been read
      read(hist, n_hist, threadIdx.x, th);
      read(ids, n_bias, threadIdx.x, tb);
      clear_tables();
    }
    // the map: words w0 ... of the mask, and one behind the last for the shifts
    const int w0 = t0 >> 5, n_map = ((t1 - 1) >> 5) - w0 + 2;
    for (int i = threadIdx.x; i < n_map; i += kThreads) {
      if (words != nullptr && w0 + i < n_words)
        cp_async4(smem_u32(bits + i), words + w0 + i);
      else
        bits[i] = ~0u;
    }
    // the tokens around the whole groups, few but without alignment
    const int n0 = max(0, min(t1, head + kN * ga) - t0), z = max(t0 + n0, head + kN * gz);
    const int n1 = max(0, t1 - z);
    auto around = [&](int i) { return i < n0 ? t0 + i : z + i - n0; };
    const float x_around = threadIdx.x < n0 + n1 ? load_f(in + around(threadIdx.x)) : 0.f;
    Piece<TI, kN> next[kUnroll];
    const TI* src = in + head + static_cast<size_t>(ga + threadIdx.x) * kN;   // of the next round
#pragma unroll
    for (int i = 0; i < kUnroll; ++i)
      if (i * kThreads < gz - ga - static_cast<int>(threadIdx.x)) next[i].template load<kVec>(src + i * kThreads * kN);
    cp_async_wait_all();
    __syncthreads();
    if (n_hist < 0 || n_hist > a.n_history) {
      if (threadIdx.x == 0 && err_word) atomicCAS(err_word, 0, kModelErrIndex);
      n_hist = n_hist < 0 ? 0 : a.n_history;
    }
    if (lists) {
      // ---- the listed tokens of the part.  The tables hold more entries than that:
      // the launcher sizes them by the lists, or else by the part.
      // The first to enter a token sends for the word that holds its logit and
      // takes it off the map.  Half a word beyond an end of the row is none of the
      // caller's: there the two bytes alone are read.
      auto enter = [&](int t, bool biased) {
        int s = slot_of(t, table), k;
        while ((k = atomicCAS(&key[s], -1, t)) != -1 && (k & ~kBiased) != t) s = after(s, table);
        if (k == -1) {
          const uintptr_t at = reinterpret_cast<uintptr_t>(in + t);
          if (sizeof(TI) == 2 && (at & 2 ? t == 0 : t == a.V - 1))
            value[s] = static_cast<uint32_t>(*reinterpret_cast<const unsigned short*>(at)) << (at & 2 ? 16 : 0);
          else
            cp_async4(smem_u32(value + s), reinterpret_cast<const void*>(at & ~uintptr_t{3}));
          const uint32_t bit = 1u << (t & 31);
          if (!(atomicAnd(&bits[(t >> 5) - w0], ~bit) & bit)) atomicAdd(&count[s], kForbidden);
        }
        if (!biased) {
          atomicAdd(&count[s], 1);
          return;
        }
        atomicOr(&key[s], kBiased);
        s = slot_of(t, n_sums);
        while ((k = atomicCAS(&bias_key[s], -1, t)) != -1 && k != t) s = after(s, n_sums);
      };
      auto enter_all = [&](const int (&t)[4], int i, int n, bool biased) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (i + u * kThreads >= n) break;
          if (t[u] >= t0 && t[u] < t1) enter(t[u], biased);
          if (t[u] >= a.V && err_word) atomicCAS(err_word, 0, kModelErrIndex);
        }
      };
      enter_all(th, threadIdx.x, n_hist, false);
      enter_all(tb, threadIdx.x, n_bias, true);
      for (int i = threadIdx.x + 4 * kThreads; i < n_hist; i += 4 * kThreads) {
        read(hist, n_hist, i, th);
        enter_all(th, i, n_hist, false);
      }
      for (int i = threadIdx.x + 4 * kThreads; i < n_bias; i += 4 * kThreads) {
        read(ids, n_bias, i, tb);
        enter_all(tb, i, n_bias, true);
      }
      // in place the stream writes where they come from
      if (static_cast<const void*>(in) == out) cp_async_wait_all();
    }
    __syncthreads();
    // The biases' sums: the last warp, in list order, while the others stream.
    // Entries of a warp's 32 that name one token are summed alike by every lane
    // that names it.
    if (n_bias > 0 && warp == kThreads / 32 - 1) {
      const float* val = a.bias + static_cast<long long>(row) * a.n_bias;
      for (int i0 = 0; i0 < n_bias; i0 += 32) {
        const int i = i0 + lane;
        const int t = i < n_bias ? ids[i] : -1;
        const bool here = t >= t0 && t < t1;
        if (!__any_sync(0xffffffffu, here)) continue;
        const float x = here ? val[i] : 0.f;
        int s = 0;
        if (here)
          for (s = slot_of(t, n_sums); bias_key[s] != t;) s = after(s, n_sums);
        float sum = here ? bias[s] : 0.f;
        const unsigned same = __match_any_sync(0xffffffffu, here ? t : -1 - lane);
        if (__all_sync(0xffffffffu, same == 1u << lane)) {
          sum += x;
        } else {
          for (int l = 0; l < 32; ++l) {
            const float y = __shfl_sync(0xffffffffu, x, l);
            if (same >> l & 1u) sum += y;
          }
        }
        __syncwarp();
        if (here) bias[s] = sum;
        __syncwarp();
      }
    }

    // The value of listed token t, entry s, but for the biases.  (The mask's -inf
    // was streamed: count[s] >= 0 here.)
    auto penalised = [&](int t, int s) {
      float x;
      if constexpr (sizeof(TI) == 4)
        x = __uint_as_float(value[s]);
      else
        x = __uint_as_float(reinterpret_cast<uintptr_t>(in + t) & 2 ? value[s] & 0xffff0000u : value[s] << 16);
      const int c = count[s];
      if (c > 0) {
        if (a.repetition) x = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
        if (a.presence) x = __fsub_rn(x, pres);
        if (a.frequency) x = __fsub_rn(x, __fmul_rn(freq, static_cast<float>(c)));
      }
      return x;
    };
    auto stray = [&](int v, float x) {
      if (!(bits[(v >> 5) - w0] >> (v & 31) & 1u)) x = -INFINITY;
      out[v] = rounded<TO>(x);
      x = static_cast<float>(rounded<TO>(x));
      if (x > -INFINITY) better(bv, bi, x, v);
    };
    if (threadIdx.x < n0 + n1) stray(around(threadIdx.x), x_around);

    // ---- stream the part's whole groups; listed tokens as -inf, so that they
    // take no part in the maximum
    float pv = -INFINITY;        // the largest value of the thread's groups, and
    int pg = -1;                 // the first group with it
    {
      TO* dst = out + head + static_cast<size_t>(ga + threadIdx.x) * kN;
      // a round moves whole words of the map on: one place in a word a thread
      const int v = head + (ga + static_cast<int>(threadIdx.x)) * kN, place = v & 31;
      const uint32_t* map = bits + (v >> 5) - w0;
      auto round = [&](int g, int left, auto all) {   // all: this round and the next are whole
        Piece<TI, kN> raw[kUnroll];
#pragma unroll
        for (int i = 0; i < kUnroll; ++i) raw[i] = next[i];
        src += kRound * kN;
#pragma unroll
        for (int i = 0; i < kUnroll; ++i)
          if (all || i * kThreads < left - kRound) next[i].template load<kVec>(src + i * kThreads * kN);
#pragma unroll
        for (int i = 0; i < kUnroll; ++i) {
          if (!all && i * kThreads >= left) break;
          float x[kN];
          raw[i].unpack(x);
          const uint32_t* m = map + i * kThreads * kN / 32;
          const uint32_t keep = __funnelshift_r(m[0], m[1], place);
#pragma unroll
          for (int e = 0; e < kN; ++e)
            if (!(keep & (1u << e))) x[e] = -INFINITY;
          Piece<TO, kN> y;
          y.pack(x);
          y.store(dst + i * kThreads * kN);
          float top = x[0];        // fmaxf passes over NaN
#pragma unroll
          for (int e = 1; e < kN; ++e) top = fmaxf(top, x[e]);
          top = static_cast<float>(rounded<TO>(top));
          const bool more = top > pv;
          pv = more ? top : pv;
          pg = more ? g + i * kThreads : pg;
        }
        dst += kRound * kN;
        map += kRound * kN / 32;
      };
      int gb = ga;
      for (; gb + 2 * kRound <= gz; gb += kRound) round(gb + threadIdx.x, 0, std::true_type{});
      for (; gb < gz; gb += kRound) round(gb + threadIdx.x, gz - gb - static_cast<int>(threadIdx.x), std::false_type{});
    }
    // Which token it was, for the warp's largest, from what the thread wrote; the
    // loads pass while the listed tokens are finished.  (A listed one of that value
    // may have come to lie before it, and is as good.)
    const float top = warp_max(pv);
    const bool mine = pg >= 0 && pv == top;
    Piece<TO, kN> wrote;
    if (mine) wrote.template load<true>(out + head + static_cast<size_t>(pg) * kN);

    // ---- the listed tokens
    if (lists) {
      cp_async_wait_all();
      __syncthreads();   // streamed, values here, biases summed
      for (int s = threadIdx.x; s < table / 4; s += kThreads) {
        const int4 k = reinterpret_cast<const int4*>(key)[s];
        const int ks[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)   // free and flagged ones are below zero
          if (ks[e] >= 0 && count[4 * s + e] >= 0) finish(ks[e], penalised(ks[e], 4 * s + e));
      }
      if (n_bias > 0) {
        for (int i = threadIdx.x; i < n_sums; i += kThreads) {
          const int t = bias_key[i];
          if (t < 0) continue;
          int s = slot_of(t, table);
          while ((key[s] & ~kBiased) != t) s = after(s, table);
          if (count[s] >= 0) finish(t, __fadd_rn(penalised(t, s), bias[i]));
        }
      }
    }
    if (mine) {
      float x[kN];
      wrote.unpack(x);
      int e = kN - 1;
#pragma unroll
      for (int i = kN - 2; i >= 0; --i)
        if (x[i] == pv) e = i;
      better(bv, bi, pv, head + kN * pg + e);
    }
  }
  if (a.idx == nullptr) return;

  // ---- the greedy token: warp, CTA, cluster
  auto reduce = [&]() {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float v2 = __shfl_xor_sync(0xffffffffu, bv, o);
      const int i2 = __shfl_xor_sync(0xffffffffu, bi, o);
      better(bv, bi, v2, i2);
    }
  };
  auto reduce_cta = [&]() {   // the same in every thread
    reduce();
    if (lane == 0) {
      best_v[warp] = bv;
      best_i[warp] = bi;
    }
    __syncthreads();
    bv = best_v[lane % (kThreads / 32)];
    bi = best_i[lane % (kThreads / 32)];
    reduce();
  };
  reduce_cta();
  // No value above -inf: the first token that is a number.  (The stream looks for
  // values above -inf alone.)
  if (bi == kNone || bv == -INFINITY) {
    const int v0 = max(0, head + kN * g_begin), v1 = min(a.V, head + kN * g_end);
    for (int v = v0 + threadIdx.x; v < v1; v += kThreads) {
      const float x = load_f(out + v);
      if (x == x) {
        better(bv, bi, x, v);
        break;
      }
    }
    __syncthreads();   // every warp has read the first round's
    reduce_cta();
  }
  if (threadIdx.x == 0) {
    cta_v = bv;
    cta_i = bi;
  }
  if (nc > 1) cluster_sync();   // every CTA of the cluster reaches both barriers
  if (rank == 0 && threadIdx.x == 0) {
    for (int q = 1; q < nc; ++q)
      better(bv, bi, ld_dsmem_f32(&cta_v, static_cast<uint32_t>(q)),
             __float_as_int(ld_dsmem_f32(&cta_i, static_cast<uint32_t>(q))));
    a.idx[row] = bi == kNone ? 0 : bi;
  }
  if (nc > 1) cluster_sync();   // rank 0 has read every CTA's result
}

template <typename TI, typename TO>
cudaError_t launch_typed(cudaStream_t stream, const LogitsPenalty& a, int* err_word) {
  // the element offset of input and output rows agrees modulo a group, row by row
  constexpr int kN = sizeof(TI) + sizeof(TO) == 4 ? 8 : 4;
  const uintptr_t x = reinterpret_cast<uintptr_t>(a.logits) / sizeof(TI);
  const uintptr_t y = reinterpret_cast<uintptr_t>(a.out) / sizeof(TO);
  const bool vec = (x - y) % kN == 0 && (a.rows == 1 || (a.ld - a.out_ld) % kN == 0);
  auto kern = vec ? logits_penalty_kernel<TI, TO, true> : logits_penalty_kernel<TI, TO, false>;
  // CTAs of a row: enough to fill the SMs (three each), at least a thousand
  // tokens a CTA
  int nc = 1;
  while (nc < kCluster && static_cast<long long>(a.rows) * nc < 3 * current_sm_count() && a.V / (2 * nc) >= 1024)
    nc *= 2;
  // The tables hold twice the lists (at four thirds a search is so long that 512
  // rows with 1024 different tokens each took 62 us for 4x); lists longer than
  // three quarters of the largest table are worked through part by part, a part no
  // longer than that.  (Small tables leave the L1 cache to the loads in flight:
  // with 26 KB more a row the stream took 27 us for 23.)
  constexpr int kMost = kMaxTable / 4 * 3;
  const long long n_bias = a.bias_ids ? a.n_bias : 0, n = a.n_history + n_bias;
  auto entries = [](long long m) {
    return 2 * m < kMaxTable ? (2 * static_cast<int>(m) + 3) / 4 * 4 : kMaxTable;
  };
  const int table = entries(n), n_sums = entries(n_bias);
  // a CTA's share of the row, at most
  int part = ((a.V + nc - 1) / nc + 24 + 31) / 32 * 32;
  if (n > kMost && part > kMost) part = kMost;
  part = part < kMaxPart ? part : kMaxPart;
  const size_t smem = static_cast<size_t>(table) * 12 + static_cast<size_t>(n_sums) * 8 + static_cast<size_t>(part) / 8 + 16;
  static SmemOptIn opt_in[2];
  const cudaError_t e = allow_smem(kern, static_cast<int>(smem), opt_in[vec]);
  if (e != cudaSuccess) return e;
  return launch_dependent(kern, dim3(static_cast<unsigned>(a.rows) * nc), dim3(kThreads), smem, stream,
                          nc, a, table, n_sums, part, err_word);
}

}  // namespace

cudaError_t launch_logits_penalty(cudaStream_t stream, const LogitsPenalty& a, int* err_word) {
  if (a.rows == 0 || a.V == 0) return cudaSuccess;
  if (a.in_f32)
    return a.out_f32 ? launch_typed<float, float>(stream, a, err_word)
                     : launch_typed<float, __nv_bfloat16>(stream, a, err_word);
  return a.out_f32 ? launch_typed<__nv_bfloat16, float>(stream, a, err_word)
                   : launch_typed<__nv_bfloat16, __nv_bfloat16>(stream, a, err_word);
}

}  // namespace nd
