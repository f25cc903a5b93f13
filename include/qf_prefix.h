/*
 * qf_prefix.h -- paged serving with shared prefixes: page copies, decode
 * attention that reads a shared prefix once, and attention of new tokens
 * behind cached ones.
 *
 * The reference prefills every row from slot 0 of its own cache
 * (student_engine.py:679-737, :1162-1204) and attends every row alone
 * (:834-874); rows that share pages of a paged cache (qf_paged.h) have no
 * counterpart there.  Conventions, pools and block tables are those of
 * qf_attn.h and qf_paged.h: fp16, strides in elements, no allocation, no
 * synchronisation, legal under stream capture.
 */
#ifndef QF_PREFIX_H
#define QF_PREFIX_H

#include <stdint.h>

#include "qf_paged.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Copies pages within every one of n_pools * per page pools: for each pair i,
 * slots [0, slots[i]) of all KVH heads of page dst[i] become those of src[i].
 *
 *   pools   HOST array of n_pools device pointers (read during the call); at each
 *           begin `per` pools (n_pages, KVH, page_size, D), `step` elements apart,
 *           with the strides sp, sh, sn
 *   src, dst  int32[n_pairs] on the device; a pair with a page outside
 *           [0, n_pages) copies nothing
 *   slots   int32[n_pairs] on the device, clamped to [0, page_size]; NULL
 *           copies whole pages
 *
 * No page may be written twice, or written and read, by one call: what such a
 * page holds afterwards is unspecified.  n_pairs = 0 launches nothing.
 */
int qf_copy_pages(const void* const* pools, int n_pools, int per, int64_t step,
                  int64_t sp, int64_t sh, int64_t sn, const int32_t* src, const int32_t* dst,
                  const int32_t* slots, int n_pairs, int n_pages, int KVH, int page_size, int D, void* stream);

/*
 * Decode attention of a batch whose rows share prefixes: the result of
 * qf_decode_attn_paged with a kv_last per row and no bias, with the slots that
 * a group of rows shares read once for the whole group.
 *
 *   q, out       (B, KVH, G, D), strides *_sb, *_sh, *_sg
 *   prefix_rows  int32[n_groups + 1] on the device, ascending: rows
 *                [prefix_rows[g], prefix_rows[g + 1]) are group g; rows outside
 *                every group share nothing
 *   prefix_len   int32[n_groups] on the device: slots [0, prefix_len[g]) hold
 *                the same K and V in every row of group g.  They are read from
 *                the group's pages, for each row up to its own kv_last; the slots
 *                behind from the row's own pages
 *   prefix_table NULL: a group's pages are those of its first row.  Else int32
 *                (n_groups, prefix_pages) on the device, row stride pt_sb: group
 *                g's pages (its first row may then have none mapped)
 *   kv_last      int64 on the device, row b reads kv_last[b * kv_last_sb]: its
 *                last slot (inclusive).  A row with kv_last < 0 has none, and
 *                its output is zero
 *   ws           16-byte aligned scratch of at least
 *                qf_decode_attn_prefix_workspace bytes for these sizes (cap =
 *                pages_per_row * page_size), else QF_ERR_SCRATCH_LIMIT; free
 *                again when the call's work is done, and not to be shared by
 *                calls that overlap in time
 *   scale        > 0
 *
 * All device arrays are read when the kernels run; any contents keep every
 * access in bounds.  Infinities and NaN in slots that a row does not see do not
 * reach its output.  Where every score that a query sees is -infinity its output is
 * NaN, here and in the extension, as from qf_decode_attn and qf_prefill_attn.
 */
int64_t qf_decode_attn_prefix_workspace(int B, int KVH, int G, int n_groups, int cap);

int qf_decode_attn_prefix_paged(const void* q, int64_t q_sb, int64_t q_sh, int64_t q_sg,
                                const void* k_pool, int64_t kp_sp, int64_t kp_sh, int64_t kp_sn,
                                const void* v_pool, int64_t vp_sp, int64_t vp_sh, int64_t vp_sn,
                                const int32_t* block_table, int64_t bt_sb, int pages_per_row,
                                int n_pages, int page_size,
                                const int32_t* prefix_rows, const int32_t* prefix_len, int n_groups,
                                const int32_t* prefix_table, int64_t pt_sb, int prefix_pages,
                                const int64_t* kv_last, int64_t kv_last_sb,
                                void* ws, int64_t ws_bytes,
                                void* out, int64_t o_sb, int64_t o_sh, int64_t o_sg,
                                int B, int KVH, int G, int D, float scale, void* stream);

/*
 * New tokens behind cached ones: qf_prefill_varlen_paged for rows that hold
 * slots already.  Row b's tokens, [cu_seqlens[b], cu_seqlens[b + 1]) of the
 * packed q, k, v and out, go to its slots context[b] + i, and token i attends
 * to slots [0, context[b] + i].
 *
 *   q, out (T, QH, D), k, v (T, KVH, D): strides *_sh per head, *_sn per token;
 *          a row may have no tokens; tokens of no row (before cu_seqlens[0],
 *          from cu_seqlens[B] to T = total) are not appended, and their rows of
 *          out are left as they were
 *   context  int64 on the device, row b reads context[b * ctx_sb]; negative:
 *          the row's tokens are not appended and their outputs are zero
 *   cos, sin (T, D), token stride cs_sn, or both NULL: rotate-half RoPE of q
 *          and k as in qf_prefill_varlen_paged
 *   cap    slots of a row that the call may use, at most pages_per_row *
 *          page_size: a bound on every row's context + tokens, from which the
 *          work is split.  Tokens past it are not appended and see the slots
 *          below it
 *   ws     as above, qf_prefill_extend_workspace bytes for these sizes (ws is
 *          not NULL even for 0)
 *   scale  > 0
 *
 * Pages that hold the new slots must not be shared (written by no other row).
 */
int64_t qf_prefill_extend_workspace(int B, int QH, int KVH, int total, int cap);

int qf_prefill_extend_paged(const void* q, int64_t q_sh, int64_t q_sn,
                            const void* k, int64_t k_sh, int64_t k_sn,
                            const void* v, int64_t v_sh, int64_t v_sn,
                            const int32_t* cu_seqlens, int total,
                            const int64_t* context, int64_t ctx_sb,
                            const void* cos, const void* sin, int64_t cs_sn,
                            void* k_pool, int64_t kp_sp, int64_t kp_sh, int64_t kp_sn,
                            void* v_pool, int64_t vp_sp, int64_t vp_sh, int64_t vp_sn,
                            const int32_t* block_table, int64_t bt_sb, int pages_per_row,
                            int n_pages, int page_size, int cap,
                            void* ws, int64_t ws_bytes,
                            void* out, int64_t o_sh, int64_t o_sn,
                            int B, int QH, int KVH, int D, float scale, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* QF_PREFIX_H */
