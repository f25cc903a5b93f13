/*
 * qf_paged8.h -- paged KV caches held in 8 bits: tokens quantised as they are
 * written, slots read back in fp16, and the attention over them.
 *
 * The reference keeps its caches in fp16 (student_engine.py:705-716); this is
 * qf_paged.h's layout at half the bytes.  A page of a kv head holds
 *
 *   k        page_size x D codes, slot by slot
 *   v        page_size / 64 x D x 64 codes: dim by dim within groups of 64 slots
 *   k_scale, v_scale
 *            page_size / QF_BLOCK8 floats, one for every QF_BLOCK8 slots
 *
 * and slot s of row b is slot s % page_size of page table[b][s / page_size].  A
 * code's value is code * scale of its block.  Codes are int8 (QF_CODE_INT8, -127
 * to 127) or e4m3 (QF_CODE_E4M3, the OCP format, largest 448).  Scales are powers
 * of two from 2^-24 on: a code is the nearest one to x / scale without a rounding
 * before it (ties go to the even code), and its value is exact in fp16, as both x
 * and the codes' steps are multiples of powers of two.
 *
 * A block's scale is the least one at which the largest magnitude written to it
 * since its first slot fits its largest code.  Tokens that need a larger one than
 * the block has round the codes already there to it.  Values that the rounding would take past
 * fp16's largest are held at the code below.  Tokens that are not all finite make
 * the block's scale NaN, and all of the block reads as NaN, until its first slot
 * is written again.
 *
 * Conventions are those of qf_attn.h and qf_paged.h: fp16 tensors with strides in
 * elements, D = 64, QF_OK / QF_ERR_* / hipError_t returns, no allocation, no
 * synchronisation, legal under stream capture.  All device arrays are read when
 * the kernels run, and any contents of them keep every access in bounds: page ids
 * outside [0, n_pages) are clamped for reads and skipped by writes.
 */
#ifndef QF_PAGED8_H
#define QF_PAGED8_H

#include <stdint.h>

#include "qf_paged.h"

#ifdef __cplusplus
extern "C" {
#endif

#define QF_CODE_INT8 0
#define QF_CODE_E4M3 1

/* Slots of one scale. */
#define QF_BLOCK8 16

/* The pools of `layers` layers and the rows' pages (HOST struct, read during the
 * call).  Strides of codes in bytes, of scales in floats, alike for K and V; the
 * codes of one page and head are contiguous, and so are its scales.  Code
 * pointers and strides are multiples of 16. */
typedef struct {
  void* k;
  void* v;
  float* k_scale;
  float* v_scale;
  int64_t sl, sp, sh;        /* layer, page, kv head */
  int64_t ssl, ssp, ssh;
  const int32_t* table;      /* (rows, pages_per_row), row stride bt_sb */
  int64_t bt_sb;
  int32_t pages_per_row, n_pages, page_size;
  int32_t layers, KVH, code;
} QfPool8;

/*
 * Quantises new tokens into their pages.  Row b's tokens, [cu_seqlens[b],
 * cu_seqlens[b + 1]) of the packed k and v, go to its slots context[b] + i.
 *
 *   k, v  (layers, T, KVH, D): strides *_sl per layer, *_sn per token, *_sh per
 *         head.  Tokens of no row are not read
 *   context  int64 on the device, row b reads context[b * ctx_sb]; a negative one
 *         appends nothing.  Slots past the row's pages are not written
 *   cos, sin (T, D), token stride cs_sn, or both NULL: rotate-half RoPE of k as in
 *         qf_rope_append, before it is quantised
 *   max_seqlen  the most tokens of a row
 *
 * Slots of the last block behind the row's last token keep their codes.  No page
 * may be written by two rows of a call.
 */
int qf_append_paged8(const void* k, int64_t k_sl, int64_t k_sh, int64_t k_sn,
                     const void* v, int64_t v_sl, int64_t v_sh, int64_t v_sn,
                     const int32_t* cu_seqlens, int total, int max_seqlen,
                     const int64_t* context, int64_t ctx_sb,
                     const void* cos, const void* sin, int64_t cs_sn,
                     const QfPool8* pool, int B, int D, void* stream);

/*
 * Slots first[b] .. of each row back in fp16, packed: token i of row b is slot
 * first[b] + i.
 *
 *   k, v  (layers, T, KVH, D) as above, written.  Tokens of no row are left as they
 *         were; those of a row with a negative first, and of slots past the row's
 *         pages, become zero
 */
int qf_read_paged8(void* k, int64_t k_sl, int64_t k_sh, int64_t k_sn,
                   void* v, int64_t v_sl, int64_t v_sh, int64_t v_sn,
                   const int32_t* cu_seqlens, int total, int max_seqlen,
                   const int64_t* first, int64_t first_sb,
                   const QfPool8* pool, int B, int D, void* stream);

/*
 * Copies whole page records within every layer: page dst[i] becomes page src[i].
 *
 *   store  (layers, n_pages) records of `bytes` bytes, the pages `step` bytes
 *          apart, the layers `layer_step`; all multiples of 16
 *   src, dst  int32[n_pairs] on the device; a pair with a page outside
 *          [0, n_pages) copies nothing.  No page may be written twice, or written
 *          and read
 */
int qf_copy_pages8(void* store, int layers, int64_t layer_step, int64_t step, int64_t bytes,
                   const int32_t* src, const int32_t* dst, int n_pairs, int n_pages, void* stream);

/*
 * Decode attention of single tokens: softmax(scale q K^T) V over each row's slots
 * [0, kv_last], as qf_decode_attn_paged without a bias.
 *
 *   q, out   (B, KVH, G, D), strides *_sb, *_sh, *_sg
 *   kv_last  int64 on the device, row b reads kv_last[b * kv_last_sb]: its last
 *            slot (inclusive).  A row with kv_last < 0 (parked) gets zeros
 *   pool     of one layer
 *   ws       16-byte aligned scratch of at least qf_decode_attn_paged8_workspace
 *            bytes for these sizes (cap = pages_per_row * page_size; NULL where
 *            that is 0), else QF_ERR_SCRATCH_LIMIT; free again when the call's work
 *            is done, and not to be shared by calls that overlap in time
 *   scale    > 0
 *
 * Slots that a row does not see may hold anything.  A block that reads as NaN makes
 * NaN of the rows that see any of it; where every score is -infinity the output is NaN.
 */
int64_t qf_decode_attn_paged8_workspace(int B, int KVH, int G, int cap);

int qf_decode_attn_paged8(const void* q, int64_t q_sb, int64_t q_sh, int64_t q_sg,
                          const QfPool8* pool, const int64_t* kv_last, int64_t kv_last_sb,
                          void* ws, int64_t ws_bytes, void* out, int64_t o_sb, int64_t o_sh,
                          int64_t o_sg, int B, int G, int D, float scale, void* stream);

/*
 * Its split phase alone: the partials acc (B, KVH, splits, G, D), m and l (B, KVH,
 * splits, G) of qf_decode_split_paged, for qf_decode_combine or qf_attn_merge_o_proj
 * (m in natural units; a range without a slot leaves acc = l = 0 and m = -infinity).
 * acc is 16-byte aligned.
 */
int qf_decode_split_paged8(const void* q, int64_t q_sb, int64_t q_sh, int64_t q_sg,
                           const QfPool8* pool, const int64_t* kv_last, int64_t kv_last_sb,
                           float* acc, float* m, float* l, int splits, int B, int G, int D,
                           float scale, void* stream);

/*
 * New tokens behind cached ones: qf_append_paged8 of a layer's k and v, then token i of
 * row b attends to slots [0, context[b] + i] of its pages -- all of them as the pages
 * hold them, the new ones too.
 *
 *   q, out  (T, QH, D), strides *_sh per head, *_sn per token, QH a multiple of the
 *           pool's KVH.  Rows of out for tokens of no row are left as they were; those
 *           of a parked row (context < 0) become zero
 *   cos, sin  as in the append; q is rotated with them too
 *   max_seqlen  the most tokens of a row; further ones get no output
 *   cap     slots of a row that the call may use, at most pages_per_row *
 *           page_size: a bound on every row's context + tokens, from which the
 *           work is split.  Tokens past it are not appended and see the slots below
 *   ws      as above, qf_prefill_extend_paged8_workspace bytes
 */
int64_t qf_prefill_extend_paged8_workspace(int B, int QH, int KVH, int total, int max_seqlen, int cap);

int qf_prefill_extend_paged8(const void* q, int64_t q_sh, int64_t q_sn,
                             const void* k, int64_t k_sh, int64_t k_sn,
                             const void* v, int64_t v_sh, int64_t v_sn,
                             const int32_t* cu_seqlens, int total, int max_seqlen,
                             const int64_t* context, int64_t ctx_sb,
                             const void* cos, const void* sin, int64_t cs_sn,
                             const QfPool8* pool, int cap, void* ws, int64_t ws_bytes,
                             void* out, int64_t o_sh, int64_t o_sn,
                             int B, int QH, int D, float scale, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* QF_PAGED8_H */
