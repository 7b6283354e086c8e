// paged_kv.h — launchers of the paged key-value cache: decode attention,
// prefill store and eviction.
//
// A pool is K and V of [n_pages][Hkv][page_size][64] bf16; position t of
// sequence b is row t % page_size of page table[b][t / page_size].
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stddef.h>

namespace nd {

// A pool and the block table that reads it.
struct PagedPool {
  __nv_bfloat16* k;
  __nv_bfloat16* v;
  int n_pages, Hkv, page_size;
  const int* table;      // [B][table_ld], the first max_pages of a row used
  long long table_ld;
  int max_pages;
};

struct PagedDecode {
  const __nv_bfloat16* q;       // [B][H][64]
  const __nv_bfloat16* k_new;   // [B][Hkv][64] or null
  const __nv_bfloat16* v_new;
  PagedPool pool;
  const int* lens;              // [B], the new token included
  void* out;                    // [B][H][64]
  bool out_f32;
  float* lse;                   // [B][H] or null
  float* weights;               // [B][Hkv][weights_ld] or null
  long long weights_ld;
  int B, H;
  int window, sinks;            // window 0: every key is visible
  float scale;
  void* workspace;
};

// Scratch bytes of one call: tickets (zero before the first call; every call
// leaves them at zero), the partials of heads split over CTAs and, with
// weights, the scores of every key.
size_t paged_decode_workspace_bytes(int B, int H, int Hkv, long long max_len, bool weights);
cudaError_t launch_paged_decode(cudaStream_t stream, const PagedDecode& a, int* err_word);

// Rows of token (b, s), s < lens[b] (null: S), of src [B*S][ld] at columns
// k_col / v_col into position pos0 + s (pos0_dev[b] instead of pos0 if given).
cudaError_t launch_paged_store(cudaStream_t stream, const __nv_bfloat16* src, long long ld,
                               int k_col, int v_col, const PagedPool& pool, int B, int S, int pos0,
                               const int* pos0_dev, const int* lens, int* err_word);

struct PagedEvict {
  PagedPool pool;               // read through pool.table
  const int* lens;              // [B]
  const float* weights;         // [B][Hkv][weights_ld]
  long long weights_ld;
  const int* out_table;         // [B][out_table_ld], the pages the kept rows go to
  long long out_table_ld;
  int out_pages;
  int B, budget, sinks, recent;
  float* weights_out;           // [B][Hkv][weights_out_ld]
  long long weights_out_ld;
  int* kept;                    // [B][Hkv][budget]
  int* new_lens;                // [B], may be lens
};
cudaError_t launch_paged_evict(cudaStream_t stream, const PagedEvict& a, int* err_word);

}  // namespace nd
