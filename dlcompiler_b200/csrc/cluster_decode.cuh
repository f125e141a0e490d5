// Single-token attention split over a thread-block cluster (cluster_decode.cu), as its callers see it.
#pragma once
#include "attention.cuh"

namespace dlb {

// Partial results of the shared prefixes, one row per (token, q-head): unnormalised output, then the reference maximum
// (base-2 domain) and the sum that go with it.
struct PrefixPartials {
  float* o;                    // [splits, tokens * hq, D]
  float2* ml;                  // [splits, tokens * hq]
  const void* lens;            // [groups] tokens of each prefix
  const void* group_start;     // [groups + 1] first token (row of q) of each group
  int groups, lens_is_int64, start_is_int64;
  int max_len;                 // tokens the prefix table has room for
  int chunk;                   // tokens per split, a multiple of 64
};

struct ClusterDecodeParams {
  const void* q;               // [tokens, hq, dk]
  void* out;                   // [tokens, hq, dv]
  const void* block_table;     // [batch, max_pages]
  const void* kv_lens;         // [batch]
  const void* q_start;         // [batch] row of each sequence, with q_lens (none where it is 0); null: row b
  const void* q_lens;
  int64_t q_st, q_sh, o_st, o_sh, bt_stride;
  int64_t tokens;
  int batch, hq, hkv, group, dk, dv;
  int page_shift, max_pages, num_pages;
  int table_is_int64, lens_is_int64, start_is_int64, qlens_is_int64;
  int window, sinks;           // window < 0: every key
  float sm_scale, softcap;     // softcap <= 0: none
  int* status;
  PrefixPartials prefix;       // o == null: none
};

// Records a page that does not exist where a visible token should be.
__device__ __forceinline__ void report_bad_page(int* status, int row, int column, int page) {
  if (status != nullptr && atomicCAS(status, DLB_DEV_OK, DLB_DEV_BAD_PAGE) == DLB_DEV_OK) {
    status[1] = row;
    status[2] = column;
    status[3] = page;
  }
}

// Splits of a prefix of `len` tokens (as many as the table has room for).
__device__ __forceinline__ int prefix_splits(const PrefixPartials& p, int len) {
  return (max(min(len, p.max_len), 0) + p.chunk - 1) / p.chunk;
}

// Rows [start, start + n) of group g, kept inside the rows that exist.
__device__ __forceinline__ void group_rows(const PrefixPartials& p, int64_t tokens, int g, int& start, int& n) {
  const int64_t lo = p.start_is_int64 ? reinterpret_cast<const int64_t*>(p.group_start)[g]
                                      : reinterpret_cast<const int32_t*>(p.group_start)[g];
  const int64_t hi = p.start_is_int64 ? reinterpret_cast<const int64_t*>(p.group_start)[g + 1]
                                      : reinterpret_cast<const int32_t*>(p.group_start)[g + 1];
  const int64_t a = max((int64_t)0, min(lo, tokens));
  start = (int)a;
  n = (int)max((int64_t)0, min(hi, tokens) - a);
}

// `width` is the tile width (64 or 128); key_bound the keys that one sequence can see at most.
int launch_cluster_decode(const ClusterDecodeParams& p, const void* k_cache, const void* v_cache, int64_t k_stride_page,
                          int64_t k_stride_slot, int64_t k_stride_head, int64_t v_stride_page, int64_t v_stride_slot,
                          int64_t v_stride_head, int width, int64_t key_bound, int dtype, cudaStream_t stream);

}  // namespace dlb
