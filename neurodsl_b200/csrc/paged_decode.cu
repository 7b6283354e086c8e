// paged_decode.cu — decode attention of one new token per sequence over a
// paged key-value cache, with grouped query heads, per-sequence lengths read
// on the device, a sliding window with sinks, the append of the new token and
// the accumulation of each key's attention weight.
//
// For sequence b with L = lens[b] keys, key j is visible when
// j >= L - window or j < sinks (window 0: every j < L).  Per query head:
//   s_j = scale * q.k_j,  out = sum_j exp(s_j - lse) v_j,
//   lse = log sum_j exp(s_j)  over the visible j;
// no visible key (L = 0) gives out = 0 and lse = -inf.
//
// Bound: HBM, 256 bytes per visible key and kv head (K and V rows of 64
// bf16), each read once for all the query heads of the group.
//
// Split: the visible keys of a (sequence, kv head) are cut into tiles of 64,
// and the tiles of all heads, laid end to end, are dealt out in equal
// contiguous ranges to one wave of CTAs.  So a ragged batch and a single long
// sequence both keep every SM busy, whatever the lengths.  Every CTA sums the
// lengths itself: they live on the device, and a host-side plan would need a
// synchronisation.  A head wholly inside one range is written at once; a head
// cut by range borders leaves partials (max, sum, unnormalised output) in the
// workspace, and the CTA that draws the head's last ticket joins them in
// range order, so the result does not depend on timing.
//
// Inside a CTA each of four warps takes 16 keys of a tile and keeps its own
// running max and sum; the warps join through shared memory at a head's end.
// Keys and values go from global memory to a ring of per-lane shared-memory
// slots by cp.async (a lane reads back only what it copied, so the ring needs
// no barrier and has no bank conflicts) and feed mma.m16n8k16 directly: the
// 64 dims of Q and K are assigned to fragment slots by one permutation that
// lets a lane read 16 contiguous bytes, and V rows are paired along keys with
// byte permutes.  The matrix unit runs far below its rate here; what counts
// is that one instruction serves the whole group of query heads.
#include <cuda_bf16.h>
#include <stdint.h>

#include "launch.cuh"
#include "model_ops.h"
#include "paged_kv.h"
#include "ptx.cuh"

namespace nd {
namespace {

constexpr int kD = 64;
constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kKeysPerWarp = 16;
constexpr int kTile = kWarps * kKeysPerWarp;    // keys per tile
constexpr int kStages = 4;                      // ring depth, in tiles
constexpr int kStageBytes = 4096;               // one warp's 16 keys, K and V
constexpr int kMaxCtas = 512;                   // CTAs of one launch
constexpr int kMaxRows = 16;                    // query heads of one pass
constexpr int kPartialRow = kD + 2;             // acc[64], max, sum
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct Params {
  const __nv_bfloat16* q;
  const __nv_bfloat16* k_new;
  const __nv_bfloat16* v_new;
  __nv_bfloat16* k;
  __nv_bfloat16* v;
  const int* table;
  long long table_ld;
  const int* lens;
  void* out;
  float* lse;
  float* scores;       // [B][H][cap], log2 units, or null
  float* lse2;         // [B][H], log2 units, with scores
  float* partials;
  unsigned int* tickets;
  int* err_word;
  int B, H, Hkv, G, parts;   // parts: passes of up to 16 query heads per kv head
  int n_pages, page_size, page_shift, max_pages;
  int window, sinks, min_tiles;
  float scale_log2;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool pred) {
  const int n = pred ? 16 : 0;   // 0: the slot is filled with zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint4 ld_shared_v4(uint32_t a) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "r"(a)
               : "memory");
  return r;
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ unsigned int atom_add_acq_rel_gpu(unsigned int* p, unsigned int v) {
  unsigned int old;
  asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], %2;" : "=r"(old) : "l"(p), "r"(v) : "memory");
  return old;
}

// The visible tiles of a sequence of L keys: the tiles of the sinks below the
// window's first tile, then the window's.  A sequence without keys has one
// tile with nothing visible, so that its outputs are written like the others.
struct Span {
  int L;        // keys
  bool ok;      // the length fits the table (else it is cut, and nothing is appended)
  int start;    // first key of the window
  int n_sink;   // sink tiles before the window's
  int lo;       // first tile of the window
  int n;        // tiles in all
};
__device__ __forceinline__ Span span_of(const Params& p, int b) {
  Span s;
  const long long cap = static_cast<long long>(p.max_pages) * p.page_size;
  int L = p.lens[b];
  s.ok = L >= 0 && L <= cap;
  if (!s.ok) {
    if (p.err_word && blockIdx.x == 0) atomicCAS(p.err_word, 0, kModelErrIndex);
    L = L < 0 ? 0 : static_cast<int>(cap);
  }
  s.L = L;
  s.start = (p.window > 0 && p.window < L) ? L - p.window : 0;
  s.lo = s.start / kTile;
  const int sinks = p.sinks < s.start ? p.sinks : s.start;
  s.n_sink = min((sinks + kTile - 1) / kTile, s.lo);
  s.n = max(1, s.n_sink + (L + kTile - 1) / kTile - s.lo);
  return s;
}
__device__ __forceinline__ int key_tile(const Span& s, int j) {
  return j < s.n_sink ? j : s.lo + j - s.n_sink;
}

// A place in the row of all tiles: tile j of pass `hp` (kv head and group of
// query heads) of sequence b.
struct Cursor {
  int b, hp, j;
  Span s;
};

template <int kRows, bool kOutF32, bool kWholePage>
__global__ void __launch_bounds__(kThreads, kRows == 8 ? 3 : 2) paged_decode_kernel(const Params p) {
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ long long sm_sum[kThreads];
  __shared__ long long sm_first;   // tiles before the CTA's first sequence
  __shared__ int sm_b;
  __shared__ float sm_m[kWarps][kRows], sm_l[kWarps][kRows];
  __shared__ float sm_o[kWarps][kRows][kD + 4];
  __shared__ unsigned int sm_ticket;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, q4 = lane & 3;
  const int heads = p.Hkv * p.parts;

  pdl_wait();
  pdl_trigger();

  // ---- this CTA's range: sum every sequence's tiles, deal them out evenly
  const int per = (p.B + kThreads - 1) / kThreads;
  {
    long long mine = 0;
    for (int b = threadIdx.x * per; b < min(p.B, (static_cast<int>(threadIdx.x) + 1) * per); ++b)
      mine += span_of(p, b).n;
    sm_sum[threadIdx.x] = mine;
  }
  __syncthreads();
  // inclusive scan by the first warp, four sums a lane
  if (warp == 0) {
    long long v[4], run = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      run += sm_sum[lane * 4 + i];
      v[i] = run;
    }
    long long base = run;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, base, o);
      if (lane >= o) base += x;
    }
    base -= run;
#pragma unroll
    for (int i = 0; i < 4; ++i) sm_sum[lane * 4 + i] = base + v[i];
  }
  __syncthreads();
  const long long total = sm_sum[kThreads - 1] * heads;
  long long n_cta = (total + p.min_tiles - 1) / p.min_tiles;
  if (n_cta > gridDim.x) n_cta = gridDim.x;
  if (static_cast<long long>(blockIdx.x) >= n_cta) return;
  const long long cta = blockIdx.x;
  const long long lo = total * cta / n_cta, hi = total * (cta + 1) / n_cta;
  {
    const long long before = threadIdx.x == 0 ? 0 : sm_sum[threadIdx.x - 1];
    if (before * heads <= lo && lo < sm_sum[threadIdx.x] * heads) {
      long long at = before;
      int b = threadIdx.x * per;
      for (int n; lo >= (at + (n = span_of(p, b).n)) * heads; ++b) at += n;
      sm_b = b;
      sm_first = at;
    }
  }
  __syncthreads();

  Cursor c;                 // the tile being computed
  c.b = sm_b;
  c.s = span_of(p, c.b);
  long long head_start;     // first tile of the head being computed
  {
    const long long in = lo - sm_first * heads;
    c.hp = static_cast<int>(in / c.s.n);
    c.j = static_cast<int>(in - static_cast<long long>(c.hp) * c.s.n);
    head_start = lo - c.j;
  }
  auto advance = [&](Cursor& x) {
    if (++x.j == x.s.n) {
      x.j = 0;
      if (++x.hp == heads) {
        x.hp = 0;
        if (++x.b < p.B) x.s = span_of(p, x.b);
      }
    }
  };

  // ---- the ring: issue() copies this warp's 16 keys of a tile into a stage
  const uint32_t my_ring = smem_u32(ring) + warp * (kStages * kStageBytes) + lane * 16;
  auto visible = [&](const Span& s, int key) -> bool {
    return key < s.L && (key >= s.start || key < p.sinks);
  };
  auto page_of = [&](int key) -> int {
    return p.page_shift >= 0 ? key >> p.page_shift : key / p.page_size;
  };
  // the row of a key in the pool, -1 if its page is none of the pool's
  auto row_of = [&](int b, int h, int key, int id) -> long long {
    const int row = key - page_of(key) * p.page_size;
    if (id < 0 || id >= p.n_pages) {
      if (p.err_word) atomicCAS(p.err_word, 0, kModelErrIndex);
      return -1;
    }
    return (static_cast<long long>(id) * p.Hkv + h) * p.page_size + row;
  };
  // Whether this warp's keys from key0 hold a visible one: the table is read
  // only for those (a page below the window may have been given back).
  auto any_visible = [&](const Span& s, int key0) -> bool {
    return key0 < s.L && (key0 + kKeysPerWarp > s.start || key0 < p.sinks);
  };
  auto page_id = [&](const Cursor& x) -> int {   // of this warp's keys (kWholePage)
    const int key = key_tile(x.s, x.j) * kTile + warp * kKeysPerWarp;
    return any_visible(x.s, key) ? p.table[x.b * p.table_ld + page_of(key)] : 0;
  };
  auto issue = [&](const Cursor& x, int stage, int id) {
    const int key0 = key_tile(x.s, x.j) * kTile + warp * kKeysPerWarp;
    const int h = x.hp / p.parts;
    const uint32_t dst = my_ring + stage * kStageBytes;
    long long row0 = 0;    // whole page: the row of key0; else the row of key0 + lane
    if constexpr (kWholePage) {
      if (any_visible(x.s, key0)) row0 = row_of(x.b, h, key0, id);
    } else {
      const int key = key0 + (lane & 15);
      row0 = visible(x.s, key)
                 ? row_of(x.b, h, key, p.table[x.b * p.table_ld + page_of(key)]) : -1;
    }
    const bool app = p.k_new != nullptr && x.s.ok && x.s.L - 1 >= key0 && x.s.L - 1 < key0 + kKeysPerWarp;
    const size_t new_off = (static_cast<size_t>(x.b) * p.Hkv + h) * kD;
    auto copy = [&](const __nv_bfloat16* pool, const __nv_bfloat16* fresh, __nv_bfloat16* pool_w,
                    int r, int piece, uint32_t slot) {
      const int key = key0 + r;
      long long row;
      if constexpr (kWholePage)
        row = row0 < 0 ? -1 : row0 + r;
      else
        row = __shfl_sync(0xffffffffu, row0, r);
      const __nv_bfloat16* src = pool + (row < 0 ? 0 : row) * kD + piece * 8;
      bool there = row >= 0 && visible(x.s, key);
      if (app && key == x.s.L - 1) {   // the new token: from k_new / v_new, and into its page
        src = fresh + new_off + piece * 8;
        if (row >= 0 && x.hp % p.parts == 0)
          *reinterpret_cast<uint4*>(pool_w + row * kD + piece * 8) =
              *reinterpret_cast<const uint4*>(src);
        there = true;
      }
      cp_async16(dst + slot * 512, src, there);
    };
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int c2 = 0; c2 < 2; ++c2) copy(p.k, p.k_new, p.k, g + 8 * t, q4 + 4 * c2, t * 2 + c2);
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 2; ++e) copy(p.v, p.v_new, p.v, 8 * t + 2 * q4 + e, g, 4 + t * 2 + e);
  };

  Cursor pre = c;           // the next tile to copy
  long long pre_at = lo;
  int pre_id = 0;
  if constexpr (kWholePage) pre_id = page_id(pre);
  auto issue_next = [&](int stage) {
    if (pre_at < hi) {
      issue(pre, stage, pre_id);
      ++pre_at;
      if (pre_at < hi) {
        advance(pre);
        if constexpr (kWholePage) pre_id = page_id(pre);
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) issue_next(s);

  // ---- heads of the range, one after the other
  long long at = lo;
  int stage = 0;
  while (at < hi) {
    const long long head_end = head_start + c.s.n;
    const long long seg_end = head_end < hi ? head_end : hi;
    const int h = c.hp / p.parts, row_base = (c.hp % p.parts) * kMaxRows;
    const int rows = min(p.G - row_base, kRows);
    const int head0 = h * p.G + row_base;       // query head of row 0

    // Q fragments: rows g and g + 8, dims in the order K is read
    uint32_t qa[2][8];
#pragma unroll
    for (int r = 0; r < (kRows > 8 ? 2 : 1); ++r) {
      uint4 x0 = make_uint4(0, 0, 0, 0), x1 = x0;
      if (g + 8 * r < rows) {
        const uint4* src = reinterpret_cast<const uint4*>(
            p.q + (static_cast<size_t>(c.b) * p.H + head0 + g + 8 * r) * kD);
        x0 = src[q4];
        x1 = src[q4 + 4];
      }
      qa[r][0] = x0.x; qa[r][1] = x0.y; qa[r][2] = x0.z; qa[r][3] = x0.w;
      qa[r][4] = x1.x; qa[r][5] = x1.y; qa[r][6] = x1.z; qa[r][7] = x1.w;
    }
    constexpr int kR = kRows > 8 ? 2 : 1;       // rows per lane
    float m[kR], l[kR], o[8][4];
#pragma unroll
    for (int r = 0; r < kR; ++r) {
      m[r] = -INFINITY;
      l[r] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = 0.f;

    for (; at < seg_end; ++at) {
      issue_next((stage + kStages - 1) % kStages);
      cp_async_wait<kStages - 1>();
      const uint32_t src = my_ring + stage * kStageBytes;
      stage = (stage + 1) % kStages;
      const int key0 = key_tile(c.s, c.j) * kTile + warp * kKeysPerWarp;

      // S = Q K^T: two tiles of 8 keys, four steps of 16 dims
      float sc[2][4];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const uint4 k0 = ld_shared_v4(src + (t * 2) * 512), k1 = ld_shared_v4(src + (t * 2 + 1) * 512);
        sc[t][0] = sc[t][1] = sc[t][2] = sc[t][3] = 0.f;
        const uint32_t z = 0;
        mma_bf16(sc[t], qa[0][0], kR > 1 ? qa[1][0] : z, qa[0][1], kR > 1 ? qa[1][1] : z, k0.x, k0.y);
        mma_bf16(sc[t], qa[0][2], kR > 1 ? qa[1][2] : z, qa[0][3], kR > 1 ? qa[1][3] : z, k0.z, k0.w);
        mma_bf16(sc[t], qa[0][4], kR > 1 ? qa[1][4] : z, qa[0][5], kR > 1 ? qa[1][5] : z, k1.x, k1.y);
        mma_bf16(sc[t], qa[0][6], kR > 1 ? qa[1][6] : z, qa[0][7], kR > 1 ? qa[1][7] : z, k1.z, k1.w);
      }
      bool vis[2][2];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) vis[t][e] = visible(c.s, key0 + 8 * t + 2 * q4 + e);
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < kR; ++r)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            sc[t][2 * r + e] = vis[t][e] ? sc[t][2 * r + e] * p.scale_log2 : -INFINITY;
      if (p.scores != nullptr) {
        const long long cap = static_cast<long long>(p.max_pages) * p.page_size;
#pragma unroll
        for (int r = 0; r < kR; ++r)
          if (g + 8 * r < rows) {
            float* dst = p.scores + (static_cast<size_t>(c.b) * p.H + head0 + g + 8 * r) * cap;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
              for (int e = 0; e < 2; ++e)
                if (vis[t][e]) dst[key0 + 8 * t + 2 * q4 + e] = sc[t][2 * r + e];
          }
      }
      // running max; the accumulators follow where it rose
#pragma unroll
      for (int r = 0; r < kR; ++r) {
        float x = fmaxf(fmaxf(sc[0][2 * r], sc[0][2 * r + 1]), fmaxf(sc[1][2 * r], sc[1][2 * r + 1]));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
        const float m_new = fmaxf(m[r], x);
        const float base = m_new == -INFINITY ? 0.f : m_new;   // no key yet: every p is 2^-inf
        const float alpha = exp2f(m[r] - base);
        m[r] = m_new;
        l[r] *= alpha;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          o[i][2 * r] *= alpha;
          o[i][2 * r + 1] *= alpha;
        }
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float pr = exp2f(sc[t][2 * r + e] - base);
            sc[t][2 * r + e] = pr;
            l[r] += pr;
          }
      }
      // O += P V.  P goes to the matrix unit in bf16 (relative error 2^-9 a
      // weight, below the bf16 output's own rounding); an fp32 output takes
      // P as three bf16 terms, which carry all 24 bits.
      uint4 v0 = ld_shared_v4(src + 4 * 512), v1 = ld_shared_v4(src + 5 * 512);
      uint4 v2 = ld_shared_v4(src + 6 * 512), v3 = ld_shared_v4(src + 7 * 512);
      const uint32_t va[4][4] = {{v0.x, v0.y, v0.z, v0.w}, {v1.x, v1.y, v1.z, v1.w},
                                 {v2.x, v2.y, v2.z, v2.w}, {v3.x, v3.y, v3.z, v3.w}};
#pragma unroll
      for (int term = 0; term < (kOutF32 ? 3 : 1); ++term) {
        uint32_t pa[2][2];   // [key half][row]
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            if (r >= kR) {
              pa[t][r] = 0;
              continue;
            }
            const uint32_t w = pack_bf16x2(sc[t][2 * r], sc[t][2 * r + 1]);
            pa[t][r] = w;
            if constexpr (kOutF32) {   // what the rounding left
              sc[t][2 * r] -= __uint_as_float(w << 16);
              sc[t][2 * r + 1] -= __uint_as_float(w & 0xFFFF0000u);
            }
          }
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          mma_bf16(o[2 * w], pa[0][0], pa[0][1], pa[1][0], pa[1][1],
                   __byte_perm(va[0][w], va[1][w], 0x5410), __byte_perm(va[2][w], va[3][w], 0x5410));
          mma_bf16(o[2 * w + 1], pa[0][0], pa[0][1], pa[1][0], pa[1][1],
                   __byte_perm(va[0][w], va[1][w], 0x7632), __byte_perm(va[2][w], va[3][w], 0x7632));
        }
      }
      if (at + 1 < seg_end) ++c.j;
    }

    // ---- the head's end in this range: join the warps
    __syncthreads();   // the previous head's readers are done
#pragma unroll
    for (int r = 0; r < kR; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      if (q4 == 0) {
        sm_m[warp][g + 8 * r] = m[r];
        sm_l[warp][g + 8 * r] = l[r];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {    // lane q4 holds dims 16 q4 + i and 16 q4 + 8 + i
        sm_o[warp][g + 8 * r][16 * q4 + i] = o[i][2 * r];
        sm_o[warp][g + 8 * r][16 * q4 + 8 + i] = o[i][2 * r + 1];
      }
    }
    __syncthreads();
    const bool whole = head_start >= lo && head_end <= hi;
    // slot 1 of the range where the head begins, slot 0 of every later one
    float* part = p.partials + (cta * 2 + (head_start >= lo ? 1 : 0)) * kRows * kPartialRow;
    for (int i = threadIdx.x; i < rows * kD; i += kThreads) {
      const int r = i / kD, d = i % kD;
      float mm = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, sm_m[w][r]);
      float ll = 0.f, oo = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = sm_m[w][r] == -INFINITY ? 0.f : exp2f(sm_m[w][r] - mm);
        ll += sm_l[w][r] * f;
        oo += sm_o[w][r][d] * f;
      }
      if (whole) {
        const size_t row = static_cast<size_t>(c.b) * p.H + head0 + r;
        const float y = ll > 0.f ? oo / ll : 0.f;
        if constexpr (kOutF32)
          static_cast<float*>(p.out)[row * kD + d] = y;
        else
          static_cast<__nv_bfloat16*>(p.out)[row * kD + d] = __float2bfloat16_rn(y);
        if (d == 0) {
          const float lse2 = ll > 0.f ? mm + log2f(ll) : -INFINITY;
          if (p.lse) p.lse[row] = lse2 * kLn2;
          if (p.scores) p.lse2[row] = lse2;
        }
      } else {
        part[r * kPartialRow + d] = oo;
        if (d == 0) {
          part[r * kPartialRow + kD] = mm;
          part[r * kPartialRow + kD + 1] = ll;
        }
      }
    }
    if (!whole) {
      // The barrier orders this CTA's partial before thread 0's ticket, whose
      // release publishes it; the last ticket's acquire sees all of them.
      const long long c0 = ((head_start + 1) * n_cta + total - 1) / total - 1;
      const long long c1 = (head_end * n_cta + total - 1) / total - 1;
      __syncthreads();
      if (threadIdx.x == 0) sm_ticket = atom_add_acq_rel_gpu(&p.tickets[c0], 1u);
      __syncthreads();
      if (sm_ticket == static_cast<unsigned int>(c1 - c0)) {
        auto slot = [&](long long cc) {
          return p.partials + (cc * 2 + (cc == c0 ? 1 : 0)) * kRows * kPartialRow;
        };
        for (int i = threadIdx.x; i < rows * kD; i += kThreads) {
          const int r = i / kD, d = i % kD;
          float mm = -INFINITY;
          for (long long cc = c0; cc <= c1; ++cc)
            mm = fmaxf(mm, __ldcg(slot(cc) + r * kPartialRow + kD));
          float ll = 0.f, oo = 0.f;
          for (long long cc = c0; cc <= c1; ++cc) {
            const float* x = slot(cc) + r * kPartialRow;
            const float pm = __ldcg(x + kD);
            const float f = pm == -INFINITY ? 0.f : exp2f(pm - mm);
            ll += __ldcg(x + kD + 1) * f;
            oo += __ldcg(x + d) * f;
          }
          const size_t row = static_cast<size_t>(c.b) * p.H + head0 + r;
          const float y = ll > 0.f ? oo / ll : 0.f;
          if constexpr (kOutF32)
            static_cast<float*>(p.out)[row * kD + d] = y;
          else
            static_cast<__nv_bfloat16*>(p.out)[row * kD + d] = __float2bfloat16_rn(y);
          if (d == 0) {
            const float lse2 = ll > 0.f ? mm + log2f(ll) : -INFINITY;
            if (p.lse) p.lse[row] = lse2 * kLn2;
            if (p.scores) p.lse2[row] = lse2;
          }
        }
        if (threadIdx.x == 0) p.tickets[c0] = 0u;   // ready for the next call
      }
    }
    if (at < hi) {
      advance(c);
      head_start = head_end;
    }
  }
}

// weights[b][h][j] += sum over the group's query heads of exp(s_j - lse), for
// every visible key, in the heads' order.  A block takes kWeightKeys keys of
// one (sequence, kv head).
constexpr int kWeightThreads = 256;
constexpr int kWeightKeys = 1024;

__global__ void __launch_bounds__(kWeightThreads)
    paged_weights_kernel(const Params p, float* __restrict__ weights, long long weights_ld) {
  pdl_wait();
  pdl_trigger();
  const int b = blockIdx.y / p.Hkv, h = blockIdx.y % p.Hkv;
  const Span s = span_of(p, b);
  const long long cap = static_cast<long long>(p.max_pages) * p.page_size;
  float* w = weights + static_cast<size_t>(blockIdx.y) * weights_ld;
  const size_t row0 = static_cast<size_t>(b) * p.H + h * p.G;
  for (int i = 0; i < kWeightKeys; i += kWeightThreads) {
    const long long key = static_cast<long long>(blockIdx.x) * kWeightKeys + i + threadIdx.x;
    if (key >= s.L || (key < s.start && key >= p.sinks)) continue;
    float x = 0.f;
    for (int g = 0; g < p.G; ++g)
      x += exp2f(p.scores[(row0 + g) * cap + key] - p.lse2[row0 + g]);
    w[key] += x;
  }
}

size_t round256(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }
size_t tickets_bytes() { return round256(kMaxCtas * sizeof(unsigned int)); }
size_t partials_bytes(int G) {
  const int rows = G <= 8 ? 8 : 16;
  return round256(static_cast<size_t>(kMaxCtas) * 2 * rows * kPartialRow * sizeof(float));
}

template <int kRows, bool kOutF32, bool kWholePage>
cudaError_t launch_typed(cudaStream_t stream, const Params& p, long long max_tiles) {
  auto kern = paged_decode_kernel<kRows, kOutF32, kWholePage>;
  constexpr int smem = kWarps * kStages * kStageBytes;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  long long grid = static_cast<long long>(current_sm_count()) * (kRows == 8 ? 3 : 2);
  if (grid > kMaxCtas) grid = kMaxCtas;
  if (grid > max_tiles) grid = max_tiles;
  return launch_ex(kern, dim3(static_cast<unsigned>(grid)), dim3(kThreads), smem, stream, 1, true, p);
}

}  // namespace

size_t paged_decode_workspace_bytes(int B, int H, int Hkv, long long max_len, bool weights) {
  const int G = Hkv > 0 ? H / Hkv : 0;
  size_t n = tickets_bytes() + partials_bytes(G);
  if (weights) {
    const size_t rows = static_cast<size_t>(B) * H;
    n += round256(rows * sizeof(float)) + rows * static_cast<size_t>(max_len) * sizeof(float);
  }
  return n;
}

cudaError_t launch_paged_decode(cudaStream_t stream, const PagedDecode& a, int* err_word) {
  Params p = {};
  p.q = a.q;
  p.k_new = a.k_new;
  p.v_new = a.v_new;
  p.k = a.pool.k;
  p.v = a.pool.v;
  p.table = a.pool.table;
  p.table_ld = a.pool.table_ld;
  p.lens = a.lens;
  p.out = a.out;
  p.lse = a.lse;
  p.err_word = err_word;
  p.B = a.B;
  p.H = a.H;
  p.Hkv = a.pool.Hkv;
  p.G = a.H / a.pool.Hkv;
  p.parts = (p.G + kMaxRows - 1) / kMaxRows;
  p.n_pages = a.pool.n_pages;
  p.page_size = a.pool.page_size;
  p.page_shift = -1;
  for (int s = 0; s < 31; ++s)
    if ((1 << s) == p.page_size) p.page_shift = s;
  p.max_pages = a.pool.max_pages;
  p.window = a.window;
  p.sinks = a.window > 0 ? a.sinks : 0;
  p.min_tiles = 2;
  p.scale_log2 = a.scale * kLog2e;
  char* ws = static_cast<char*>(a.workspace);
  p.tickets = reinterpret_cast<unsigned int*>(ws);
  ws += tickets_bytes();
  p.partials = reinterpret_cast<float*>(ws);
  ws += partials_bytes(p.G);
  if (a.weights) {
    p.lse2 = reinterpret_cast<float*>(ws);
    p.scores = reinterpret_cast<float*>(ws + round256(static_cast<size_t>(a.B) * a.H * sizeof(float)));
  }
  const long long cap = static_cast<long long>(p.max_pages) * p.page_size;
  const long long per_head = cap > 0 ? (cap + kTile - 1) / kTile : 1;
  const long long max_tiles = static_cast<long long>(a.B) * p.Hkv * p.parts * per_head;
  const bool whole_page = p.page_size % kKeysPerWarp == 0;
  cudaError_t e;
#define ND_PAGED(R, F)                                                        \
  e = whole_page ? launch_typed<R, F, true>(stream, p, max_tiles)             \
                 : launch_typed<R, F, false>(stream, p, max_tiles)
  if (p.G <= 8) {
    if (a.out_f32) ND_PAGED(8, true); else ND_PAGED(8, false);
  } else {
    if (a.out_f32) ND_PAGED(16, true); else ND_PAGED(16, false);
  }
#undef ND_PAGED
  if (e != cudaSuccess || a.weights == nullptr || cap == 0) return e;
  const dim3 grid(static_cast<unsigned>((cap + kWeightKeys - 1) / kWeightKeys),
                  static_cast<unsigned>(a.B * p.Hkv));
  return launch_ex(paged_weights_kernel, grid, dim3(kWeightThreads), 0, stream, 1, true, p,
                   a.weights, a.weights_ld);
}

}  // namespace nd
