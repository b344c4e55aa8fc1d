// Parameters and launches of the grouped-head attention over a cache of 4 bits.
#pragma once

#include "mla_gqa.h"
#include "mla_mx4.h"

namespace mla {

struct GqaMx4Params {
  GqaParams g;  // k and v null; rows of the pools by page_table
  const uint8_t *k_codes, *k_scales, *v_codes, *v_scales;
  int64_t c_page, c_tok, c_head, s_page, s_tok, s_head;  // bytes, of both pools
  // long chunks: values of the batch's keys in pages of 64 rows, [kv_heads][scratch_rows][D], and their page table
  __bf16 *scratch_k, *scratch_v;
  int32_t* scratch_table;  // [batch, scratch_cols]
  int32_t scratch_cols;
  int64_t scratch_rows;
};

hipError_t launch_gqa_mx4(const GqaMx4Params& p, int dim, int rows, hipStream_t stream);  // CTAs of 16 or 32 rows
hipError_t launch_mx4_pages(const GqaMx4Params& p, int dim, hipStream_t stream);
hipError_t launch_gqa_merge(const GqaParams& p, int dim, int rows, hipStream_t stream);

}  // namespace mla
