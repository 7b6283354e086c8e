// paged_decode.cu — decode attention of one new token per sequence over a
// paged key-value cache, with grouped query heads, per-sequence lengths read
// on the device, a sliding window with sinks, the append of the new token and
// the accumulation of each key's attention weight.
//
// For sequence b with L = lens[b] keys, key j is visible when
// j >= L - window or j < sinks (window 0: every j < L).  Per query head:
//   s_j = scale * q.k_j,  out = sum_j exp(s_j - lse) v_j,
//   lse = log sum_j exp(s_j)  over the visible j;
// no visible key (L = 0) gives out = 0 and lse = -inf.  A score that is NaN or
// +inf leaves no number in its head's row, as in the formula.
//
// Bound: HBM, 256 bytes per visible key and kv head (K and V rows of 64
// bf16), each read once for up to 16 query heads of the group.
//
// Split: the visible keys of a (sequence, kv head) are cut into tiles of 64,
// and the tiles of all heads, laid end to end, are dealt out in equal
// contiguous ranges to one wave of CTAs.  So a ragged batch and a single long
// sequence both keep every SM busy, whatever the lengths; a head counts as
// kHeadCost tiles more than it has, for the joins at its end (without that the
// CTAs that drew the short heads finished last: 47.5 us for 64 sequences of 32 to
// 2048 keys, 12 heads, where it now takes 38.4, 81 % of the copy bandwidth).
// Every CTA sums the lengths itself: they live on the device, and a host-side
// plan would need a synchronisation.  A head wholly inside one range is written at once; a head
// cut by range borders leaves partials (max, sum, unnormalised output) in the
// workspace, and the CTA that draws the head's last ticket joins them in
// range order, so the result does not depend on timing.
//
// Inside a CTA a producer warp keeps a ring of tiles filled, running ahead over
// the range whatever heads its tiles belong to, and four warps take 16 keys
// of a tile each, with their own running max and sum; they join through shared
// memory at a head's end while the next head's tiles are already arriving.
// Two producers, by the page size: where a page holds whole boxes of 8 rows or
// more (the largest power of two that divides it, up to the tile), one TMA box
// each with the 128-byte swizzle; else 16-byte cp.async pieces into the same
// layout, by four warps (two beside 16 query heads, whose consumers need the
// registers).  64 sequences of 2048 keys, 12 heads: 67.8 us at pages of 64 rows,
// 70.2 at 16, 77.4 at 24 (by pieces with one warp 1.6 times as long); by pieces 88.5
// at 100 (in boxes of 4 a seventh longer), 97.2 at 7, 120.7 at 1.
//
// S = Q K^T takes Q as the 16-row operand of mma.m16n8k16 (query head = row)
// and K's rows as they lie (ldmatrix).  The scores' fragment is then, packed to
// bf16, the column operand of O^T = V^T P^T as it stands, with V^T by
// transposing ldmatrix: no data moves between lanes but the row max.  The
// matrix unit runs far below its rate; what counts is that one instruction
// serves the whole group of query heads and that a warp's chain per tile is
// short (an earlier form in which each lane copied its own keys by cp.async
// spent 350 instructions per 16 keys: 85 us for the batch above).  What is left
// beside the bytes is some 7 us a call: the lengths, the first tile's way
// through memory, and the last joins.
#include <cuda.h>
#include <cuda_bf16.h>
#include <stdint.h>

#include "launch.cuh"
#include "model_ops.h"
#include "paged_kv.h"
#include "ptx.cuh"
#include "ring.cuh"
#include "tma.h"

namespace nd {
namespace {

constexpr int kD = 64;
constexpr int kWarps = 4;                       // consumer warps
constexpr int kConsumers = kWarps * 32;
constexpr int kMinBox = 8;                      // rows of a TMA box, at least
constexpr int kKeysPerWarp = 16;
constexpr int kTile = kWarps * kKeysPerWarp;    // keys per tile
// The producer's warps, the ring's depth in tiles and the CTAs of an SM: more
// warps where they copy piece by piece, and so fewer CTAs, with deeper rings.
template <int kRows, bool kTma>
struct Shape {
  static constexpr int kProducers = kTma ? 1 : kRows == 8 ? 4 : 2;
  static constexpr int kThreads = kConsumers + 32 * kProducers;
  static constexpr int kStages = kTma ? 4 : kRows == 8 ? 6 : 5;
  static constexpr int kCtas = kTma && kRows == 8 ? 3 : 2;
};
constexpr int kMaxStages = 6;
constexpr int kRowBytes = kD * 2;
constexpr int kTileBytes = kTile * kRowBytes;   // K or V of a tile
constexpr int kStageBytes = 2 * kTileBytes;
constexpr int kMaxCtas = 512;                   // CTAs of one launch
constexpr int kMaxRows = 16;                    // query heads of one pass
constexpr int kPartialRow = kD + 4;             // acc[64], max, sum (16-byte rows)
constexpr int kHeadCost = 3;                    // what a head costs beside its tiles, in tiles
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
  float* scores;       // [B][H][scores_ld], log2 units, or null
  long long scores_ld; // the table's keys, rounded up to whole tiles
  float* lse2;         // [B][H], log2 units, with scores
  float* partials;
  unsigned int* tickets;
  int* err_word;
  int B, H, Hkv, G, parts;   // parts: passes of up to 16 query heads per kv head
  int n_pages, page_size, page_shift, max_pages;
  int box;             // rows of a TMA box
  int window, sinks;
  float scale_log2;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool there) {
  const int n = there ? 16 : 0;   // 0: the piece is filled with zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n)
               : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
// This thread's copies so far arrive on `bar` when they have landed.
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// A box of K or V rows whose lines L2 may give up first: they are read once a
// step, and would push out what is read again (the scores, the partials).
__device__ __forceinline__ void tma_load_rows(const CUtensorMap* map, uint64_t* bar, void* dst, int row,
                                              uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%3, %4}], [%2], %5;" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(0), "r"(row), "l"(policy)
      : "memory");
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
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
__device__ __forceinline__ Span make_span(const Params& p, int L) {
  Span s;
  const int cap = p.max_pages * p.page_size;
  s.ok = L >= 0 && L <= cap;
  if (!s.ok) L = L < 0 ? 0 : cap;
  s.L = L;
  s.start = (p.window > 0 && p.window < L) ? L - p.window : 0;
  s.lo = s.start / kTile;
  const int sinks = min(p.sinks, s.start);
  s.n_sink = min((sinks + kTile - 1) / kTile, s.lo);
  s.n = max(1, s.n_sink + (L + kTile - 1) / kTile - s.lo);
  return s;
}
__device__ __forceinline__ bool visible(const Params& p, const Span& s, int key) {
  return key < s.L && (key >= s.start || key < p.sinks);
}
// Whether the n keys from key0 on hold a visible one / are all visible.  The
// table is read only for the former: a page below the window may have been
// given back.
__device__ __forceinline__ bool any_visible(const Params& p, const Span& s, int key0, int n) {
  return key0 < s.L && (key0 + n > s.start || key0 < p.sinks);
}
__device__ __forceinline__ bool all_visible(const Params& p, const Span& s, int key0, int n) {
  return key0 + n <= s.L && (key0 >= s.start || key0 + n <= p.sinks);
}

// A place in the row of all tiles: tile j of pass `hp` (kv head and group of
// query heads) of sequence b.
struct Cursor {
  int b, hp, j;
  int next_len;     // of sequence b + 1, read well before it is needed
  Span s;
  __device__ __forceinline__ int key_tile() const {
    return j < s.n_sink ? j : s.lo + j - s.n_sink;
  }
};
__device__ __forceinline__ void next_head(const Params& p, int heads, Cursor& c) {
  c.j = 0;
  if (++c.hp < heads) return;
  c.hp = 0;
  if (++c.b >= p.B) return;
  c.s = make_span(p, c.next_len);
  if (c.b + 1 < p.B) c.next_len = p.lens[c.b + 1];
}
// On to the next tile; returns how far that is in cost.
__device__ __forceinline__ int next_tile(const Params& p, int heads, Cursor& c) {
  if (++c.j < c.s.n) return 1;
  next_head(p, heads, c);
  return 1 + kHeadCost;
}

// What every warp works out for itself: the cost of all heads, how many CTAs
// share it, and this CTA's range [lo, hi) of it.  A head of n tiles takes
// n + kHeadCost places, its tiles the first n.  (No barrier: the warps of a CTA
// read the same few lengths.)
struct Plan {
  long long total, lo, hi;
  int n_cta;
};
// a / b; in 32 bits where that holds both (a 64-bit division is a long call)
__device__ __forceinline__ long long quotient(long long a, long long b) {
  if ((a | b) >> 32 == 0) return static_cast<unsigned>(a) / static_cast<unsigned>(b);
  return a / b;
}
__device__ __forceinline__ Plan make_plan(const Params& p, int heads, Cursor& c) {
  const int lane = threadIdx.x & 31;
  const int per = (p.B + 31) / 32;
  const int b0 = lane * per, b1 = min(p.B, b0 + per);
  long long mine = 0;
  for (int b = b0; b < b1; ++b) {
    const Span s = make_span(p, p.lens[b]);
    if (!s.ok && p.err_word && blockIdx.x == 0) atomicCAS(p.err_word, 0, kModelErrIndex);
    mine += s.n + kHeadCost;
  }
  long long upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += x;
  }
  Plan r;
  r.total = __shfl_sync(0xffffffffu, upto, 31) * heads;
  // A range's time grows with its tiles, the join's with the ranges of a head
  // times its rows (32 partials of one row, or 4 of each of 16, at a time):
  // their sum is least near sqrt(T rows / 32) tiles a range for heads of T.  (At
  // least one: with two, a window of 256 of 700 keys takes 7.0 us for 6.5.)
  const int rows = min(p.G, kMaxRows);
  const float mean = static_cast<float>(r.total) / (static_cast<float>(p.B) * heads);
  const float least = fmaxf(1.f, sqrtf(mean * (rows <= 2 ? 2 : rows <= 4 ? 4 : rows) * (1.f / 32.f)));
  r.n_cta = static_cast<int>(fminf(ceilf(static_cast<float>(r.total) / least), static_cast<float>(gridDim.x)));
  r.lo = r.hi = 0;
  if (static_cast<int>(blockIdx.x) >= r.n_cta) return r;
  r.lo = quotient(r.total * blockIdx.x, r.n_cta);
  r.hi = quotient(r.total * (blockIdx.x + 1), r.n_cta);
  // the sequence of the range's first tile
  long long at = upto - mine;
  const bool here = at * heads <= r.lo && r.lo < upto * heads;
  int b = b0;
  if (here)
    for (int n; r.lo >= (at + (n = make_span(p, p.lens[b]).n + kHeadCost)) * heads; ++b) at += n;
  const int src = __ffs(__ballot_sync(0xffffffffu, here)) - 1;
  c.b = __shfl_sync(0xffffffffu, b, src);
  const long long in = r.lo - __shfl_sync(0xffffffffu, at, src) * heads;
  c.s = make_span(p, p.lens[c.b]);
  c.next_len = c.b + 1 < p.B ? p.lens[c.b + 1] : 0;
  const int places = c.s.n + kHeadCost;
  c.hp = static_cast<int>(quotient(in, places));
  c.j = static_cast<int>(in - static_cast<long long>(c.hp) * places);
  if (c.j >= c.s.n) {      // the range begins behind a head's last tile
    r.lo += places - c.j;
    next_head(p, heads, c);
  }
  return r;
}

// The row of a key in the pool; -1 (and the error word) if its page is none of
// the pool's.
__device__ __forceinline__ long long pool_row(const Params& p, int b, int h, int key) {
  const int page = p.page_shift >= 0 ? key >> p.page_shift : key / p.page_size;
  const int id = p.table[b * p.table_ld + page];
  if (id < 0 || id >= p.n_pages) {
    if (p.err_word) atomicCAS(p.err_word, 0, kModelErrIndex);
    return -1;
  }
  return (static_cast<long long>(id) * p.Hkv + h) * p.page_size + (key - page * p.page_size);
}

struct Bars {
  uint64_t full[kMaxStages];    // a tile has landed
  uint64_t empty[kMaxStages];   // the four consumer warps have read it
  int abort_flag;
};

// ---- the producer warp: every tile of the range into the ring, in order.
// Rows without a visible key are not copied (their stage bytes are whatever was
// there; the consumers mask them), rows of a page outside the pool are zeros.
template <bool kTma, int kStages, int kProducers>
__device__ __forceinline__ void produce(const Params& p, const CUtensorMap* tm_k,
                                        const CUtensorMap* tm_v, int heads, Cursor c, long long at,
                                        long long hi, uint8_t* ring, Bars* bars) {
  const int lane = threadIdx.x & 31;
  volatile int* abort_flag = &bars->abort_flag;
  // what a lane looks up, one tile ahead: with TMA, box `lane` of the tile; else
  // the row `lane` of its warp's share of the tile
  constexpr int kShare = kTile / kProducers;
  static_assert(kTma ? kProducers == 1 : kShare <= 32, "a row a lane");
  const int row0 = kTma ? 0 : (static_cast<int>(threadIdx.x) - kConsumers) / 32 * kShare;
  long long row = -2;     // -2: nothing to copy, -1: zeros
  auto look_up = [&](const Cursor& x) {
    const int key0 = x.key_tile() * kTile, h = x.hp / p.parts;
    if constexpr (kTma) {
      const int key = key0 + lane * p.box;
      row = lane * p.box < kTile && any_visible(p, x.s, key, p.box) ? pool_row(p, x.b, h, key) : -2;
    } else {
      const int key = key0 + row0 + lane;
      row = lane < kShare && visible(p, x.s, key) ? pool_row(p, x.b, h, key) : -2;
    }
  };
  look_up(c);
  uint64_t policy = 0;
  if constexpr (kTma) asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
  auto fill = [&](int s) {
    uint8_t* dst = ring + s * kStageBytes;
    if constexpr (kTma) {
      const bool go = row != -2;
      const unsigned n = __popc(__ballot_sync(0xffffffffu, go));
      if (lane == 0) mbar_arrive_expect_tx(&bars->full[s], n * p.box * 2 * kRowBytes);
      if (go) {
        // a box that starts past the pool's last row reads as zeros
        const int r = static_cast<int>(row < 0 ? static_cast<long long>(p.n_pages) * p.Hkv * p.page_size : row);
        tma_load_rows(tm_k, &bars->full[s], dst + lane * p.box * kRowBytes, r, policy);
        tma_load_rows(tm_v, &bars->full[s], dst + kTileBytes + lane * p.box * kRowBytes, r, policy);
      }
    } else {
      const int piece = lane & 7;
#pragma unroll
      for (int i = 0; i < kShare / 4; ++i) {
        const long long src = __shfl_sync(0xffffffffu, row, 4 * i + (lane >> 3));
        const int r = row0 + 4 * i + (lane >> 3);
        const size_t off = static_cast<size_t>(src < 0 ? 0 : src) * kD + piece * 8;
        const uint32_t to = smem_u32(dst) + r * kRowBytes + ((piece ^ (r & 7)) << 4);
        if (src != -2) {
          cp_async16(to, p.k + off, src >= 0);
          cp_async16(to + kTileBytes, p.v + off, src >= 0);
        }
      }
      cp_async_arrive(&bars->full[s]);
    }
    at += next_tile(p, heads, c);
    if (at < hi) look_up(c);
  };
  ring_produce<kStages>(
      [&]() { return at < hi; },
      [&](int s, uint32_t parity) { return warp_wait(&bars->empty[s], parity, abort_flag); }, fill,
      [&]() { raise_abort(abort_flag, p.err_word, kDevErrTimeoutPaged); },
      [&](int s, uint32_t parity) {
        // the pieces by thread: another warp's may never have been sent off
        if constexpr (kTma) mbar_landed(&bars->full[s], parity);
        else cp_async_wait_all();
      });
}

template <int kRows, bool kOutF32, bool kTma>
__global__ void __launch_bounds__(Shape<kRows, kTma>::kThreads, Shape<kRows, kTma>::kCtas)
    paged_decode_kernel(const Params p, const __grid_constant__ CUtensorMap tm_k,
                        const __grid_constant__ CUtensorMap tm_v) {
  constexpr int kStages = Shape<kRows, kTma>::kStages, kProducers = Shape<kRows, kTma>::kProducers;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Bars bars;
  __shared__ float sm_m[kWarps][kRows], sm_l[kWarps][kRows];
  __shared__ __align__(16) float sm_o[kWarps][kRows][kD + 4];
  __shared__ unsigned int sm_ticket;
  uint8_t* ring = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int heads = p.Hkv * p.parts;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&bars.full[s], kTma ? 1 : 32 * kProducers);
      mbar_init(&bars.empty[s], kWarps);
    }
    bars.abort_flag = 0;
    fence_barrier_init();
  }
  if (kTma && threadIdx.x == kConsumers) {
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  pdl_wait();
  // A call that appends writes the cache, and the contiguous decode attention, with
  // programmatic launch on, reads cached rows before it waits: what follows starts
  // when this kernel is done.
  if (p.k_new == nullptr) pdl_trigger();
  __syncthreads();

  Cursor c;
  const Plan plan = make_plan(p, heads, c);
  const long long lo = plan.lo, hi = plan.hi;   // lo: the range's first tile
  if (lo >= hi) return;
  if (warp >= kWarps) {
    if constexpr (kTma) {
      // rows written by earlier kernels' ordinary stores, read by bulk copies
      asm volatile("fence.proxy.async.global;" ::: "memory");
    }
    produce<kTma, kStages, kProducers>(p, &tm_k, &tm_v, heads, c, lo, hi, ring, &bars);
    return;
  }

  // ---- consumers
  const int g = lane >> 2, q4 = lane & 3;
  volatile int* abort_flag = &bars.abort_flag;
  // ldmatrix: lane's row of the warp's 16 and its 16-byte piece, swizzled;
  // matrices 0/1: keys 0-7, pieces 2s and 2s + 1; matrices 2/3: keys 8-15
  uint32_t mat[4];
  {
    const uint32_t r = (lane & 7) + ((lane >> 4) << 3);
    const uint32_t base = smem_u32(ring) + (warp * kKeysPerWarp + r) * kRowBytes;
#pragma unroll
    for (int s = 0; s < 4; ++s) mat[s] = base + (((2 * s + ((lane >> 3) & 1)) ^ (lane & 7)) << 4);
  }
  constexpr int kR = kRows > 8 ? 2 : 1;       // rows per lane: g, g + 8
  // Q fragments: rows g and g + 8; k step s takes dims 16 s + 2 q4 and + 8.
  // A head's are read while the head before it is computed.
  uint32_t qa[kR][8], qn[kR][8];
  auto load_q = [&](int b, int hp) {
    const int base = (hp % p.parts) * kMaxRows;
#pragma unroll
    for (int r = 0; r < kR; ++r) {
      const int row = base + g + 8 * r;
      const uint32_t* src = reinterpret_cast<const uint32_t*>(
          p.q + (static_cast<size_t>(b) * p.H + (hp / p.parts) * p.G + row) * kD);
#pragma unroll
      for (int s = 0; s < 8; ++s) qn[r][s] = row < p.G ? src[4 * s + q4] : 0u;
    }
  };
  load_q(c.b, c.hp);
  bool ok = true;          // no tile has failed to come
  int it = 0;              // tiles taken from the ring
  long long at = lo;
  long long head_start = lo - c.j;
  while (at < hi) {
    const long long head_end = head_start + c.s.n;
    const long long seg_end = head_end < hi ? head_end : hi;
    const int h = c.hp / p.parts, row_base = (c.hp % p.parts) * kMaxRows;
    const int rows = min(p.G - row_base, kRows);
    const int head0 = h * p.G + row_base;       // query head of row 0

#pragma unroll
    for (int r = 0; r < kR; ++r)
#pragma unroll
      for (int s = 0; s < 8; ++s) qa[r][s] = qn[r][s];
    if (head_end + kHeadCost < hi) load_q(c.hp + 1 < heads ? c.b : c.b + 1, c.hp + 1 < heads ? c.hp + 1 : 0);
    // The new token's K (lanes 0-7) and V (lanes 8-15), and its row in the
    // pool, in hand before the head's last tile is.
    const bool append = p.k_new != nullptr && c.s.ok && c.s.L > 0 && seg_end == head_end;
    uint4 fresh_kv = make_uint4(0, 0, 0, 0);
    long long fresh_row = -1;
    if (append && lane < 16) {
      fresh_kv = *reinterpret_cast<const uint4*>((lane < 8 ? p.k_new : p.v_new) +
                                                 (static_cast<size_t>(c.b) * p.Hkv + h) * kD + (lane & 7) * 8);
      if (c.hp % p.parts == 0) fresh_row = pool_row(p, c.b, h, c.s.L - 1);
    }
    // o[r][i] holds, of rows 8 r + 2 q4 and 8 r + 2 q4 + 1, the dims 16 i + g
    // and 16 i + 8 + g (the C fragment of O^T)
    float m[kR], l[kR], o[kR][4][4];
#pragma unroll
    for (int r = 0; r < kR; ++r) {
      m[r] = -INFINITY;
      l[r] = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[r][i][e] = 0.f;
    }

    const int n = static_cast<int>(seg_end - at);
    for (int k = 0; k < n; ++k, ++it) {
      const int st = it % kStages;
      const uint32_t off = st * kStageBytes;
      const int key0 = c.key_tile() * kTile + warp * kKeysPerWarp;
      if (k + 1 < n) ++c.j;
      if (!ring_take<kStages>(
              ok, it, [&](int s, uint32_t parity) { return warp_wait(&bars.full[s], parity, abort_flag); },
              [&]() { raise_abort(abort_flag, p.err_word, kDevErrTimeoutPaged); })) {
        it += n - k;
        break;
      }
      const bool full = all_visible(p, c.s, key0, kKeysPerWarp);
      const int fresh = c.s.L - 1 - key0;          // the new token's row of the 16
      const bool app = append && fresh >= 0 && fresh < kKeysPerWarp;
      if (!full || app) {
        // The border of the visible range: values of keys outside it become
        // zeros (their weight is zero, but 0 * NaN is not), and the new token
        // goes into the tile and into its page.
        uint8_t* kt = ring + off + warp * kKeysPerWarp * kRowBytes;
        uint8_t* vt = kt + kTileBytes;
        const int piece = lane & 7;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = 4 * i + (lane >> 3);
          if (!visible(p, c.s, key0 + r))
            *reinterpret_cast<uint4*>(vt + r * kRowBytes + ((piece ^ (r & 7)) << 4)) = make_uint4(0, 0, 0, 0);
        }
        if (app && lane < 16) {
          *reinterpret_cast<uint4*>((lane < 8 ? kt : vt) + fresh * kRowBytes + ((piece ^ (fresh & 7)) << 4)) = fresh_kv;
          if (fresh_row >= 0)
            *reinterpret_cast<uint4*>((lane < 8 ? p.k : p.v) + fresh_row * kD + piece * 8) = fresh_kv;
        }
        fence_async_shared();   // before the stage's next bulk copy
        __syncwarp();
      }

      uint32_t kf[4][4], vf[4][4];
#pragma unroll
      for (int s = 0; s < 4; ++s) ldmatrix4(kf[s], mat[s] + off);
#pragma unroll
      for (int s = 0; s < 4; ++s) ldmatrix4_trans(vf[s], mat[s] + off + kTileBytes);
      // S = Q K^T: two tiles of 8 keys, four steps of 16 dims; in log2 units
      float sc[2][4];
#pragma unroll
      for (int t = 0; t < 2; ++t) sc[t][0] = sc[t][1] = sc[t][2] = sc[t][3] = 0.f;
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int t = 0; t < 2; ++t)
          mma_bf16(sc[t], qa[0][2 * s], kR > 1 ? qa[kR - 1][2 * s] : 0u, qa[0][2 * s + 1],
                   kR > 1 ? qa[kR - 1][2 * s + 1] : 0u, kf[s][2 * t], kf[s][2 * t + 1]);
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.empty[st]);
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 2 * kR; ++e) sc[t][e] *= p.scale_log2;
      if (!full) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 2 * kR; ++e)
            if (!visible(p, c.s, key0 + 8 * t + 2 * q4 + (e & 1))) sc[t][e] = -INFINITY;
      }
      if (p.scores != nullptr) {
        // whole tiles: a row of scores has room for them
#pragma unroll
        for (int r = 0; r < kR; ++r)
          if (g + 8 * r < rows) {
            float* dst = p.scores + (static_cast<size_t>(c.b) * p.H + head0 + g + 8 * r) * p.scores_ld +
                         key0 + 2 * q4;
#pragma unroll
            for (int t = 0; t < 2; ++t)
              *reinterpret_cast<float2*>(dst + 8 * t) = make_float2(sc[t][2 * r], sc[t][2 * r + 1]);
          }
      }
      // running max; the accumulators follow where it rose
      float up[kR];
      bool rose = false;
#pragma unroll
      for (int r = 0; r < kR; ++r) {
        float x = fmaxf(fmaxf(sc[0][2 * r], sc[0][2 * r + 1]), fmaxf(sc[1][2 * r], sc[1][2 * r + 1]));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
        up[r] = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
        rose = rose || up[r] > m[r];
      }
      if (__any_sync(0xffffffffu, rose)) {
#pragma unroll
        for (int r = 0; r < kR; ++r) {
          const float m_new = fmaxf(m[r], up[r]);
          const float alpha = m_new == -INFINITY ? 1.f : fast_exp2(m[r] - m_new);
          m[r] = m_new;
          l[r] *= alpha;
          const float a0 = __shfl_sync(0xffffffffu, alpha, 8 * q4);        // row 2 q4
          const float a1 = __shfl_sync(0xffffffffu, alpha, 8 * q4 + 4);    // row 2 q4 + 1
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            o[r][i][0] *= a0;
            o[r][i][1] *= a1;
            o[r][i][2] *= a0;
            o[r][i][3] *= a1;
          }
        }
      }
#pragma unroll
      for (int r = 0; r < kR; ++r) {
        const float base = m[r] == -INFINITY ? 0.f : m[r];   // no key yet: every p is 2^-inf
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float pr = fast_exp2(sc[t][2 * r + e] - base);
            sc[t][2 * r + e] = pr;
            l[r] += pr;
          }
      }
      // O^T += V^T P^T.  The matrix unit takes P in bf16: as two terms for a bf16
      // output (off by 2^-16 of a weight, far below the output's own rounding, as the
      // contiguous decode's fp32 weights are; one term, off by 2^-8, takes 38.1 us for
      // 38.3 with 64 ragged sequences, and 38.9 for 39.9 with 16 heads a kv head).
      // An fp32 output takes three terms, which carry all 24 bits, and adds each
      // step's product in fp32 arithmetic: the matrix unit's own accumulation
      // cuts off low bits, a bias that grows with the number of steps.
      constexpr int kTerms = kOutF32 ? 3 : 2;
      uint32_t pb[kR][kTerms][2];
#pragma unroll
      for (int r = 0; r < kR; ++r)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int x = 0; x < kTerms; ++x) {
            const uint32_t w = pack_bf16x2(sc[t][2 * r], sc[t][2 * r + 1]);
            pb[r][x][t] = w;
            sc[t][2 * r] -= __uint_as_float(w << 16);     // what the rounding left
            sc[t][2 * r + 1] -= __uint_as_float(w & 0xFFFF0000u);
          }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int r = 0; r < kR; ++r) {
          if constexpr (kOutF32) {
            float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int y = kTerms - 1; y >= 0; --y)
              mma_bf16(x, vf[i][0], vf[i][1], vf[i][2], vf[i][3], pb[r][y][0], pb[r][y][1]);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[r][i][e] += x[e];
          } else {
#pragma unroll
            for (int y = kTerms - 1; y >= 0; --y)
              mma_bf16(o[r][i], vf[i][0], vf[i][1], vf[i][2], vf[i][3], pb[r][y][0], pb[r][y][1]);
          }
        }
      }
    }
    at = seg_end;
    // a head that lacks a tile has no result: NaN through all joins, which go on so
    // that the workspace stays as it has to be
    if (!ok) {
#pragma unroll
      for (int r = 0; r < kR; ++r) l[r] = __int_as_float(0x7fffffff);
    }

    // ---- the head's end in this range: join the warps
    named_bar_sync(1, kConsumers);   // the previous head's readers are done
#pragma unroll
    for (int r = 0; r < kR; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      if (q4 == 0) {
        sm_m[warp][g + 8 * r] = m[r];
        sm_l[warp][g + 8 * r] = l[r];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          sm_o[warp][8 * r + 2 * q4 + (e & 1)][16 * i + 8 * (e >> 1) + g] = o[r][i][e];
    }
    named_bar_sync(1, kConsumers);
    const bool whole = head_start >= lo && head_end <= hi;
    // The warps' shares of value d of row r, joined.  A share without a key above
    // -inf has max -inf and sum 0 and is left out; one whose scores are NaN has
    // that max too, but a sum that is NaN and has to come through.
    auto joined = [&](int r, int d, float& mm, float& ll, float& oo) {
      mm = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, sm_m[w][r]);
      ll = oo = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float x = sm_m[w][r];
        const float f = fast_exp2(x - mm);
        if (x != -INFINITY || sm_l[w][r] != 0.f) {   // values of a share left out may not even be written
          ll += sm_l[w][r] * f;
          oo += sm_o[w][r][d] * f;
        }
      }
    };
    auto finish = [&]() {
      for (int i = threadIdx.x; i < rows * kD; i += kConsumers) {
        const int r = i / kD, d = i % kD;
        float mm, ll, oo;
        joined(r, d, mm, ll, oo);
        const size_t row = static_cast<size_t>(c.b) * p.H + head0 + r;
        const float y = c.s.L > 0 ? oo / ll : 0.f;
        if constexpr (kOutF32)
          static_cast<float*>(p.out)[row * kD + d] = y;
        else
          static_cast<__nv_bfloat16*>(p.out)[row * kD + d] = __float2bfloat16_rn(y);
        if (d == 0) {
          const float lse2 = mm + log2f(ll);   // no key: -inf
          if (p.lse) p.lse[row] = lse2 * kLn2;
          if (p.scores) p.lse2[row] = lse2;
        }
      }
    };
    if (whole) {
      finish();
    } else {
      // slot 1 of the range where the head begins, slot 0 of every later one
      float* part = p.partials + (static_cast<size_t>(blockIdx.x) * 2 + (head_start >= lo ? 1 : 0)) *
                                     kRows * kPartialRow;
      for (int i = threadIdx.x; i < rows * kD; i += kConsumers) {
        const int r = i / kD, d = i % kD;
        float mm, ll, oo;
        joined(r, d, mm, ll, oo);
        part[r * kPartialRow + d] = oo;
        if (d == 0) {
          part[r * kPartialRow + kD] = mm;
          part[r * kPartialRow + kD + 1] = ll;
        }
      }
      // The barrier orders this CTA's partial before thread 0's ticket, whose
      // release publishes it; the last ticket's acquire sees all of them.
      const int c0 = static_cast<int>(quotient((head_start + 1) * plan.n_cta + plan.total - 1, plan.total)) - 1;
      const int c1 = static_cast<int>(quotient(head_end * plan.n_cta + plan.total - 1, plan.total)) - 1;
      named_bar_sync(1, kConsumers);
      if (threadIdx.x == 0) sm_ticket = atom_add_acq_rel_gpu(&p.tickets[c0], 1u);
      named_bar_sync(1, kConsumers);
      if (sm_ticket == static_cast<unsigned int>(c1 - c0)) {
        // Join the ranges' partials in an order that only their number sets.
        // Eight groups of 16 threads (four values each): `per` rows at a time,
        // 8 / per groups to a row, eight partials in flight a group; the
        // groups' shares then go the way of the warps'.
        const int n_part = c1 - c0 + 1;
        const int group = threadIdx.x >> 4, l16 = threadIdx.x & 15;
        const int per = rows <= 2 ? 2 : rows <= 4 ? 4 : 8;
        const int share = group / per, shares = 8 / per;
        for (int r = group % per; r < rows; r += per) {
          float mm = -INFINITY, ll = 0.f;
          float4 oo = make_float4(0.f, 0.f, 0.f, 0.f);
          for (int x0 = share; x0 < n_part; x0 += 8 * shares) {
            float pm[8], pl[8];
            float4 po[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
              const int x = x0 + u * shares;
              pm[u] = -INFINITY;
              pl[u] = 0.f;
              po[u] = make_float4(0.f, 0.f, 0.f, 0.f);
              if (x < n_part) {
                const float* s = p.partials + ((static_cast<size_t>(c0 + x) * 2 + (x == 0 ? 1 : 0)) * kRows + r) *
                                                  kPartialRow;
                pm[u] = __ldcg(s + kD);
                pl[u] = __ldcg(s + kD + 1);
                po[u] = __ldcg(reinterpret_cast<const float4*>(s) + l16);
              }
            }
            float top = mm;
#pragma unroll
            for (int u = 0; u < 8; ++u) top = fmaxf(top, pm[u]);
            const float base = top == -INFINITY ? 0.f : top;   // sums that are NaN stay so
            const float a = fast_exp2(mm - base);
            ll *= a;
            oo.x *= a;
            oo.y *= a;
            oo.z *= a;
            oo.w *= a;
#pragma unroll
            for (int u = 0; u < 8; ++u) {
              const float f = fast_exp2(pm[u] - base);
              ll += pl[u] * f;
              oo.x += po[u].x * f;
              oo.y += po[u].y * f;
              oo.z += po[u].z * f;
              oo.w += po[u].w * f;
            }
            mm = top;
          }
          *reinterpret_cast<float4*>(&sm_o[share][r][4 * l16]) = oo;
          if (l16 == 0) {
            for (int w = share; w < kWarps; w += shares) {
              sm_m[w][r] = w == share ? mm : -INFINITY;
              sm_l[w][r] = w == share ? ll : 0.f;
            }
          }
        }
        named_bar_sync(1, kConsumers);
        finish();
        if (threadIdx.x == 0) p.tickets[c0] = 0u;   // ready for the next call
      }
    }
    at = head_start = head_end + kHeadCost;
    if (at < hi) next_head(p, heads, c);
  }
}

// weights[b][h][j] += sum over the group's query heads of exp(s_j - lse), for
// every visible key, in the heads' order.  A thread takes four keys of one
// (sequence, kv head): the scores come in 16-byte pieces.  It lets no successor's
// blocks in before its own are done: the next call's would stand in their way (67
// us a call for 59 with 8 sequences of 32768 keys).
constexpr int kWeightThreads = 256;
constexpr int kWeightKeys = 4 * kWeightThreads;

__global__ void __launch_bounds__(kWeightThreads)
    paged_weights_kernel(const Params p, float* __restrict__ weights, long long weights_ld) {
  pdl_wait();
  const int b = blockIdx.y / p.Hkv, h = blockIdx.y % p.Hkv;
  const Span s = make_span(p, p.lens[b]);
  const int key0 = blockIdx.x * kWeightKeys + threadIdx.x * 4;
  if (!any_visible(p, s, key0, 4)) return;
  float* w = weights + static_cast<size_t>(blockIdx.y) * weights_ld + key0;
  const size_t row0 = static_cast<size_t>(b) * p.H + h * p.G;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int g = 0; g < p.G; ++g) {
    const float4 y = *reinterpret_cast<const float4*>(p.scores + (row0 + g) * p.scores_ld + key0);
    const float lse2 = p.lse2[row0 + g];
    x.x += exp2f(y.x - lse2);
    x.y += exp2f(y.y - lse2);
    x.z += exp2f(y.z - lse2);
    x.w += exp2f(y.w - lse2);
  }
  if (all_visible(p, s, key0, 4) && (reinterpret_cast<uintptr_t>(w) & 15) == 0) {
    float4 y = *reinterpret_cast<float4*>(w);
    y.x += x.x;
    y.y += x.y;
    y.z += x.z;
    y.w += x.w;
    *reinterpret_cast<float4*>(w) = y;
  } else {
    const float v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (visible(p, s, key0 + e)) w[e] += v[e];
  }
}

size_t round256(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }
size_t tickets_bytes() { return round256(kMaxCtas * sizeof(unsigned int)); }
size_t partials_bytes(int G) {
  const int rows = G <= 8 ? 8 : 16;
  return round256(static_cast<size_t>(kMaxCtas) * 2 * rows * kPartialRow * sizeof(float));
}

template <int kRows, bool kOutF32, bool kTma>
cudaError_t launch_typed(cudaStream_t stream, const Params& p, long long max_tiles,
                         const CUtensorMap& tk, const CUtensorMap& tv) {
  auto kern = paged_decode_kernel<kRows, kOutF32, kTma>;
  using S = Shape<kRows, kTma>;
  constexpr int smem = S::kStages * kStageBytes + 1024;   // + alignment
  static SmemOptIn opt_in;
  const cudaError_t e = allow_smem(kern, smem, opt_in);
  if (e != cudaSuccess) return e;
  long long grid = static_cast<long long>(current_sm_count()) * S::kCtas;
  if (grid > kMaxCtas) grid = kMaxCtas;
  if (grid > max_tiles) grid = max_tiles;
  // placed early, before the kernel before it has ended: a call starts 0.3 us sooner
  return launch_dependent(kern, dim3(static_cast<unsigned>(grid)), dim3(S::kThreads), smem, stream, 1, p, tk,
                          tv);
}

long long scores_ld(long long max_len) { return (max_len + kTile - 1) / kTile * kTile; }

}  // namespace

size_t paged_decode_workspace_bytes(int B, int H, int Hkv, long long max_len, bool weights) {
  const int G = Hkv > 0 ? H / Hkv : 0;
  size_t n = tickets_bytes() + partials_bytes(G);
  if (weights) {
    const size_t rows = static_cast<size_t>(B) * H;
    n += round256(rows * sizeof(float)) + rows * static_cast<size_t>(scores_ld(max_len)) * sizeof(float);
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
  p.scale_log2 = a.scale * kLog2e;
  char* ws = static_cast<char*>(a.workspace);
  p.tickets = reinterpret_cast<unsigned int*>(ws);
  ws += tickets_bytes();
  p.partials = reinterpret_cast<float*>(ws);
  ws += partials_bytes(p.G);
  if (a.weights != nullptr && a.pool.max_pages > 0) {
    p.lse2 = reinterpret_cast<float*>(ws);
    p.scores = reinterpret_cast<float*>(ws + round256(static_cast<size_t>(a.B) * a.H * sizeof(float)));
  }
  const long long cap = static_cast<long long>(p.max_pages) * p.page_size;
  p.scores_ld = scores_ld(cap);
  const long long per_head = cap > 0 ? (cap + kTile - 1) / kTile : 1;
  const long long max_tiles = static_cast<long long>(a.B) * p.Hkv * p.parts * per_head;
  // TMA boxes: a page holds whole boxes, row numbers fit 31 bits
  const long long pool_rows = static_cast<long long>(p.n_pages) * p.Hkv * p.page_size;
  const bool tma = p.page_size % kMinBox == 0 && pool_rows < (1LL << 31);
  p.box = kTile;
  while (p.page_size % p.box != 0) p.box /= 2;
  CUtensorMap tk = {}, tv = {};
  cudaError_t e = cudaSuccess;
  if (tma) {
    const uint64_t dims[2] = {kD, static_cast<uint64_t>(pool_rows)};
    const uint64_t strides[1] = {kRowBytes};
    const uint32_t box[2] = {kD, static_cast<uint32_t>(p.box)};
    e = make_tmap_bf16_sw128(&tk, p.k, 2, dims, strides, box, nullptr);
    if (e == cudaSuccess) e = make_tmap_bf16_sw128(&tv, p.v, 2, dims, strides, box, nullptr);
    if (e != cudaSuccess) return e;
  }
#define ND_PAGED(R, F)                                                        \
  e = tma ? launch_typed<R, F, true>(stream, p, max_tiles, tk, tv)            \
          : launch_typed<R, F, false>(stream, p, max_tiles, tk, tv)
  if (p.G <= 8) {
    if (a.out_f32) ND_PAGED(8, true); else ND_PAGED(8, false);
  } else {
    if (a.out_f32) ND_PAGED(16, true); else ND_PAGED(16, false);
  }
#undef ND_PAGED
  if (e != cudaSuccess || a.weights == nullptr || cap == 0) return e;
  const dim3 grid(static_cast<unsigned>((cap + kWeightKeys - 1) / kWeightKeys),
                  static_cast<unsigned>(a.B * p.Hkv));
  return launch_dependent(paged_weights_kernel, grid, dim3(kWeightThreads), 0, stream, 1, p, a.weights,
                          a.weights_ld);
}

}  // namespace nd
