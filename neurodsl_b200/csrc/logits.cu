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
// biases) into a hash table in shared memory, with their counts, and marks them
// in a bit map; then it streams its part without a barrier, some thousand tokens
// a round, with the mask alone, and after each round every thread computes the
// listed tokens it passed anew, while their lines are in the cache.  The rare
// tokens so cost a few steps a round and not a divergent path a value, nor
// scattered traffic to memory (all of them at the end: 46.8 us for 512 rows of
// 50257 tokens with histories of 1024; with the penalties inside the stream and
// a count for every token of a slice, the lists read once a slice: 161 us; now
// 45.1).  Counts are integers, so the order of the atomics does not matter; biases
// are summed by one warp in list order, their tokens computed last.  The CTAs'
// best tokens meet in distributed shared memory, so the logits are not read
// again for the argmax.
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
constexpr int kMaxPart = 1 << 18;               // tokens of a bit map
constexpr int kCluster = 8;                     // CTAs of a row, at most
constexpr int kMaxTable = 8192;                 // table entries, a power of two
constexpr int kBiased = 1 << 31;                // flag beside a token's count
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
// kN values as they lie in memory (8 or 16 bytes).
template <typename T, int kN>
struct Piece {
  uint32_t w[kN * sizeof(T) / 4];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (sizeof(w) == 16) {
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
// loads and stores each cover contiguous bytes.  kVec: a row's input and output
// have the same place within a group, so that groups aligned in one are aligned
// in the other (the launcher checks); else token by token.
// `table` entries of shared memory, a power of two, for the listed tokens, and
// bit maps of `part` tokens (a multiple of 32), which a CTA takes at a time.
template <typename TI, typename TO, bool kVec>
__global__ void __launch_bounds__(kThreads, 4)
    logits_penalty_kernel(const LogitsPenalty a, int table, int part, int* __restrict__ err_word) {
  constexpr int kN = sizeof(TI) + sizeof(TO) == 4 ? 8 : 4;   // 8: both bf16
  constexpr int kUnroll = sizeof(TI) == 4 || kN == 8 ? 4 : 8;   // groups in flight a thread
  constexpr uint32_t kMaskN = (1u << kN) - 1u;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  int* key = reinterpret_cast<int*>(smem_raw);                  // token, -1: free
  int* count = key + table;                                     // and the flag kBiased
  float* bias = reinterpret_cast<float*>(count + table);
  uint2* bits = reinterpret_cast<uint2*>(bias + table);         // x: allowed, y: listed
  __shared__ float best_v[kThreads / 32], cta_v;
  __shared__ int best_i[kThreads / 32], cta_i;
  const int nc = static_cast<int>(cluster_nctarank()), rank = static_cast<int>(cluster_ctarank());
  const int row = blockIdx.x / nc;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const TI* in = static_cast<const TI*>(a.logits) + row * a.ld;
  TO* out = static_cast<TO*>(a.out) + row * a.out_ld;
  // tokens before the first aligned group; group k holds tokens head + kN k ...,
  // and group -1, if there are such tokens, them
  const int head = kVec ? static_cast<int>((kN - (reinterpret_cast<uintptr_t>(out) / sizeof(TO)) % kN) % kN) : 0;
  const int first = head > 0 ? -1 : 0;
  const int n_groups = (a.V - head + kN - 1) / kN - first;
  const int per = (n_groups + nc - 1) / nc;
  const int g_end = first + min(n_groups, (rank + 1) * per);
  const bool lists = a.history != nullptr || a.bias_ids != nullptr;
  pdl_wait();
  pdl_trigger();

  const int* hist = nullptr;
  const int* ids = nullptr;
  float rep = 1.f, pres = 0.f, freq = 0.f;
  int n_hist = 0, n_bias = 0;
  if (a.history != nullptr) {
    hist = a.history + row * a.history_ld;
    if (a.repetition) rep = a.repetition[row];
    if (a.presence) pres = a.presence[row];
    if (a.frequency) freq = a.frequency[row];
    n_hist = a.history_lens ? a.history_lens[row] : a.n_history;
    if (n_hist < 0 || n_hist > a.n_history) {
      if (threadIdx.x == 0 && err_word) atomicCAS(err_word, 0, kModelErrIndex);
      n_hist = n_hist < 0 ? 0 : a.n_history;
    }
  }
  if (a.bias_ids != nullptr) {
    ids = a.bias_ids + static_cast<long long>(row) * a.n_bias;
    n_bias = a.n_bias;
  }
  const uint32_t* words = a.mask ? a.mask + row * a.mask_ld : nullptr;
  const int n_words = (a.V + 31) >> 5;

  float bv = -INFINITY;
  int bi = kNone;
  auto slot_of = [&](int t) { return (static_cast<uint32_t>(t) * 2654435761u) >> 19 & (table - 1); };
  // Token t, entry s of the table, anew from its logit.  (In place: the stream
  // left that as it was, unless the mask forbids the token.)
  auto finish = [&](int t, uint32_t s, int v0) {
    if (!(bits[(t - v0) >> 5].x >> ((t - v0) & 31) & 1u)) return;   // streamed as -inf
    float x = load_f(in + t);
    const int c = count[s] & ~kBiased;
    if (c > 0) {
      if (a.repetition) x = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
      if (a.presence) x = __fsub_rn(x, pres);
      if (a.frequency) x = __fsub_rn(x, __fmul_rn(freq, static_cast<float>(c)));
    }
    if (count[s] < 0) x = __fadd_rn(x, bias[s]);
    out[t] = rounded<TO>(x);
    x = static_cast<float>(rounded<TO>(x));
    if (x == x) better(bv, bi, x, t);
  };
  // the same for a token the stream passed; one with a bias waits for its sum
  auto finish_listed = [&](int t, int v0) {
    uint32_t s = slot_of(t);
    while (key[s] != t) s = (s + 1) & (table - 1);
    if (count[s] >= 0) finish(t, s, v0);
  };
  const bool maps = lists || words != nullptr;
  for (int g0 = first + rank * per; g0 < g_end; g0 += part / kN) {
    const int g1 = min(g_end, g0 + part / kN);
    const int v0 = head + kN * g0;                      // token of the bit maps' bit 0
    const int t0 = max(v0, 0), t1 = min(a.V, head + kN * g1);   // the part's tokens
    // whole groups [ga, gz); their loads run one round ahead, the first round's
    // while the lists are worked through
    const int ga = kVec ? max(g0, 0) : g1, gz = kVec ? max(ga, min(g1, (a.V - head) / kN)) : g1;
    constexpr int kRound = kUnroll * kThreads;
    Piece<TI, kN> next[kUnroll];
    const TI* src = in + head + static_cast<size_t>(ga + threadIdx.x) * kN;   // of the next round
    auto load_round = [&](int left) {    // left: groups from this thread's next on
#pragma unroll
      for (int i = 0; i < kUnroll; ++i)
        if (i * kThreads < left) next[i].load(src + i * kThreads * kN);
      src += kRound * kN;
    };
    // the lists' first entries too
    auto read = [&](const int* list, int n, int i, int (&t)[4]) {
#pragma unroll
      for (int u = 0; u < 4; ++u) t[u] = i + u * kThreads < n ? list[i + u * kThreads] : -1;
    };
    int th[4], tb[4];
    read(hist, n_hist, threadIdx.x, th);
    read(ids, n_bias, threadIdx.x, tb);
    load_round(gz - ga - threadIdx.x);
    if (maps) {
      __syncthreads();   // the last part's maps and table have been read
      const int n_map = ((t1 - v0) >> 5) + 1, w0 = v0 >> 5;     // w0: -1 before token 0
      for (int i = threadIdx.x; i < n_map; i += 4 * kThreads) {
        uint32_t lo[4], hi[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int w = w0 + i + u * kThreads;
          lo[u] = hi[u] = ~0u;
          if (words != nullptr) {
            lo[u] = w >= 0 && w < n_words ? words[w] : 0u;
            hi[u] = (v0 & 31) != 0 && w + 1 < n_words ? words[w + 1] : 0u;
          }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (i + u * kThreads < n_map)
            bits[i + u * kThreads] = make_uint2(__funnelshift_r(lo[u], hi[u], v0 & 31), 0u);
      }
    }
    if (lists) {
      // ---- the listed tokens of the part.  At most `table` * 3/4 of them: the
      // lists, or else the part, are no longer than that.
      auto enter = [&](int t, bool biased) {
        uint32_t s = slot_of(t);
        for (;; s = (s + 1) & (table - 1)) {
          const int k = atomicCAS(&key[s], -1, t);
          if (k == -1 || k == t) break;
        }
        if (biased)
          atomicOr(&count[s], kBiased);
        else
          atomicAdd(&count[s], 1);
        atomicOr(&bits[(t - v0) >> 5].y, 1u << ((t - v0) & 31));
      };
      auto enter_all = [&](const int (&t)[4], bool biased) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (t[u] >= t0 && t[u] < t1) enter(t[u], biased);
          if (t[u] >= a.V && err_word) atomicCAS(err_word, 0, kModelErrIndex);
        }
      };
      for (int i = threadIdx.x; i < table; i += kThreads) {
        key[i] = -1;
        count[i] = 0;
        bias[i] = 0.f;
      }
      __syncthreads();
      enter_all(th, false);
      enter_all(tb, true);
      for (int i = threadIdx.x + 4 * kThreads; i < n_hist; i += 4 * kThreads) {
        read(hist, n_hist, i, th);
        enter_all(th, false);
      }
      for (int i = threadIdx.x + 4 * kThreads; i < n_bias; i += 4 * kThreads) {
        read(ids, n_bias, i, tb);
        enter_all(tb, true);
      }
    }
    if (maps) __syncthreads();
    if (lists) {
      // The biases' sums: the last warp, in list order, while the others stream.
      // Entries of a warp's 32 that name one token are summed alike by every
      // lane that names it.
      if (n_bias > 0 && warp == kThreads / 32 - 1) {
        const float* val = a.bias + static_cast<long long>(row) * a.n_bias;
        for (int i0 = 0; i0 < n_bias; i0 += 32) {
          const int i = i0 + lane;
          const int t = i < n_bias ? ids[i] : -1;
          const bool here = t >= t0 && t < t1;
          if (!__any_sync(0xffffffffu, here)) continue;
          const float x = here ? val[i] : 0.f;
          uint32_t s = 0;
          if (here)
            for (s = slot_of(t); key[s] != t;) s = (s + 1) & (table - 1);
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
    }

    // ---- stream the part: whole groups, then the tokens around them
    {
      TO* dst = out + head + static_cast<size_t>(ga + threadIdx.x) * kN;
      // a round moves whole words of the maps on: one place in a word a thread
      const uint2* map = bits + (ga - g0 + threadIdx.x) * kN / 32;
      const int place = (ga - g0 + threadIdx.x) * kN & 31;
      float pv = -INFINITY;   // the largest value of the thread's groups, and
      int pg = -1;            // the first group with it
      auto round = [&](int g, int left, auto all) {
        Piece<TI, kN> raw[kUnroll];
#pragma unroll
        for (int i = 0; i < kUnroll; ++i) raw[i] = next[i];
        load_round(left - kRound);
        uint32_t found = 0;      // the round's listed tokens, kN bits a group
#pragma unroll
        for (int i = 0; i < kUnroll; ++i) {
          if (!all && i * kThreads >= left) break;
          float x[kN];
          raw[i].unpack(x);
          uint32_t listed = 0;
          if (maps) {
            const uint2 m = map[i * kThreads * kN / 32];
            listed = m.y >> place & kMaskN;
            found |= listed << (i * kN);
            const uint32_t allowed = m.x >> place;
#pragma unroll
            for (int e = 0; e < kN; ++e)
              if (!(allowed & (1u << e))) x[e] = -INFINITY;
          }
          Piece<TO, kN> y;
          y.pack(x);
          y.store(dst + i * kThreads * kN);
          if (a.idx != nullptr) {
            y.unpack(x);         // as they were stored
            if (listed != 0) {   // listed tokens take part below; fmaxf passes over NaN
#pragma unroll
              for (int e = 0; e < kN; ++e)
                if (listed & (1u << e)) x[e] = __int_as_float(0x7fffffff);
            }
            float top = x[0];
#pragma unroll
            for (int e = 1; e < kN; ++e) top = fmaxf(top, x[e]);
            const bool more = top > pv;
            pv = more ? top : pv;
            pg = more ? g + i * kThreads : pg;
          }
        }
        // while their lines are at hand
        for (; found != 0; found &= found - 1) {
          const int b = __ffs(found) - 1;
          finish_listed(head + (g + b / kN * kThreads) * kN + b % kN, v0);
        }
        dst += kRound * kN;
        map += kRound * kN / 32;
      };
      int gb = ga;
      for (; gb + kRound <= gz; gb += kRound) round(gb + threadIdx.x, gz - gb - threadIdx.x, std::true_type{});
      if (gb < gz) round(gb + threadIdx.x, gz - gb - threadIdx.x, std::false_type{});
      // which of the group's tokens it was: this thread wrote them
      if (pg >= 0) {
        const uint32_t listed = maps ? bits[(pg - g0) * kN >> 5].y >> ((pg - g0) * kN & 31) : 0u;
        const TO* y = out + head + static_cast<size_t>(pg) * kN;
        int e = 0;
        while (e < kN - 1 && (load_f(y + e) != pv || (listed >> e & 1u))) ++e;
        better(bv, bi, pv, head + kN * pg + e);
      }
    }
    {
      const int n0 = max(0, min(t1, head + kN * ga) - t0), z = max(t0 + n0, head + kN * gz);
      const int n1 = max(0, t1 - z);
      for (int i = threadIdx.x; i < n0 + n1; i += kThreads) {
        const int v = i < n0 ? t0 + i : z + i - n0;
        const uint2 m = maps ? bits[(v - v0) >> 5] : make_uint2(~0u, 0u);
        float x = load_f(in + v);
        if (!(m.x >> ((v - v0) & 31) & 1u)) x = -INFINITY;
        out[v] = rounded<TO>(x);
        x = static_cast<float>(rounded<TO>(x));
        if (m.y >> ((v - v0) & 31) & 1u)
          finish_listed(v, v0);
        else if (x == x)
          better(bv, bi, x, v);
      }
    }

    // ---- the tokens with a bias
    if (n_bias > 0) {
      __syncthreads();   // streamed, biases summed
      for (int s = threadIdx.x; s < table; s += kThreads)
        if (count[s] < 0) finish(key[s], s, v0);
    }
  }
  if (a.idx == nullptr) return;

  // A part without a value above -inf: its first token that is a number.  (The
  // stream looks for values above -inf alone.)
  if (__syncthreads_and(bi == kNone || bv == -INFINITY)) {
    const int v0 = max(0, head + kN * (first + rank * per)), v1 = min(a.V, head + kN * g_end);
    for (int v = v0 + threadIdx.x; v < v1; v += kThreads) {
      const float x = load_f(out + v);
      if (x == x) {
        better(bv, bi, x, v);
        break;
      }
    }
  }

  // ---- the greedy token: warp, CTA, cluster
  auto reduce = [&]() {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float v2 = __shfl_xor_sync(0xffffffffu, bv, o);
      const int i2 = __shfl_xor_sync(0xffffffffu, bi, o);
      better(bv, bi, v2, i2);
    }
  };
  reduce();
  if (lane == 0) {
    best_v[warp] = bv;
    best_i[warp] = bi;
  }
  __syncthreads();
  if (warp == 0) {
    bv = lane < kThreads / 32 ? best_v[lane] : -INFINITY;
    bi = lane < kThreads / 32 ? best_i[lane] : kNone;
    reduce();
    if (lane == 0) {
      cta_v = bv;
      cta_i = bi;
    }
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
  // The table holds the lists, filled to three quarters at most; lists longer
  // than the largest table are worked through part by part, a part no longer
  // than what the table holds.
  const long long n = (a.history ? a.n_history : 0) + static_cast<long long>(a.bias_ids ? a.n_bias : 0);
  int table = 0;
  // a CTA's share of the row, at most
  int part = ((a.V + nc - 1) / nc + 24 + 31) / 32 * 32;
  if (n > 0) {
    for (table = 64; table < kMaxTable && table * 3LL / 4 < n; table *= 2) {}
    if (table * 3LL / 4 < n && part > table * 3 / 4) part = table * 3 / 4;
  }
  part = part < kMaxPart ? part : kMaxPart;
  const size_t smem = static_cast<size_t>(table) * 12 + (n > 0 || a.mask ? static_cast<size_t>(part) / 4 + 8 : 0);
  static SmemOptIn opt_in[2];
  const cudaError_t e = allow_smem(kern, static_cast<int>(smem), opt_in[vec]);
  if (e != cudaSuccess) return e;
  return launch_dependent(kern, dim3(static_cast<unsigned>(a.rows) * nc), dim3(kThreads), smem, stream,
                          nc, a, table, part, err_word);
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
