// Arguments of the attention kernels over the paged cache.
#pragma once
#include "paged_tc.cuh"

namespace snl {

struct AttendArgs {
  PagedView c;
  PagedMask m;
  snl_paged_attn_p p;
  const uint16_t* q;
  const void* gate;
  void* out;
  float* lse;
  uint32_t group;                      // query heads per KV head
  uint32_t toks, slots;                // tokens of one tile (128 / group), slots of pairs of tiles
  uint32_t n_split, split_len;         // parts of the keys and keys of one part
  float* part;                         // [row][head][part][D], then [row][head][part][max, sum]
  float2* part_ml;
  uint32_t vrun;                       // keys of a page that one box of V loads
};

// One or two rows a sequence (paged_attend_rows.cu).
bool attend_rows_fits(const snl_paged_cache& c, const snl_paged_batch& b, uint32_t group);
size_t attend_rows_workspace(const snl_paged_cache& c, const snl_paged_batch& b, uint32_t group);
int launch_attend_rows(const snl_paged_cache& c, const snl_paged_batch& b, const AttendArgs& a, void* work, cudaStream_t s);

}  // namespace snl
