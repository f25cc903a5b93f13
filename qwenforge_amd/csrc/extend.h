// Attention of new tokens behind cached ones, as the layers of an extension call
// it.
#pragma once

#include "qf_common.h"

namespace qf {

// Attention of packed new tokens whose K and V are in the pages already
// (span_attn.hip), for rows that hold context[b * ctx_sb] slots before them;
// arguments and workspace as in qf_prefill_extend_paged.
struct ExtendCall {
  const int32_t* cu;
  const int64_t* context;
  int64_t ctx_sb;
  const int32_t* table;
  int64_t t_sb;
  int ppr, n_pages, page_size, cap, B, T, QH, KVH;
};
int extend_attention(const ExtendCall& c, const void* q, int64_t q_sh, int64_t q_sn, void* out,
                     int64_t o_sh, int64_t o_sn, const void* k_pool, int64_t kp_sp, int64_t kp_sh,
                     int64_t kp_sn, const void* v_pool, int64_t vp_sp, int64_t vp_sh, int64_t vp_sn,
                     void* ws, int64_t ws_bytes, float scale, hipStream_t st);

}  // namespace qf
