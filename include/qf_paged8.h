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

/* Arguments come in HOST structs of 8-byte fields, read during the call: a caller
 * whose language is slow at passing many arguments packs them into one buffer.
 *
 * The pools of `layers` layers and the rows' pages.  Strides of codes in bytes, of
 * scales in floats, alike for K and V; the codes of one page and head are contiguous,
 * and so are its scales.  Code pointers and strides are multiples of 16. */
typedef struct {
  void* k;
  void* v;
  float* k_scale;
  float* v_scale;
  int64_t sl, sp, sh;        /* layer, page, kv head */
  int64_t ssl, ssp, ssh;
  const int32_t* table;      /* (rows, pages_per_row), row stride bt_sb */
  int64_t bt_sb;
  int64_t pages_per_row, n_pages, page_size;
  int64_t layers, KVH, code;
} QfPool8;

/* Packed tokens of B rows: row b has tokens [cu_seqlens[b], cu_seqlens[b + 1]) of
 * `total`, at most max_seqlen (of a longer row the first max_seqlen; the others are tokens
 * of no row), and they are its slots first[b * first_sb] + i. */
typedef struct {
  QfPool8 pool;
  void* k;                   /* (layers, T, KVH, D): strides per layer, head, token */
  int64_t k_sl, k_sh, k_sn;
  void* v;
  int64_t v_sl, v_sh, v_sn;
  const int32_t* cu_seqlens;
  int64_t total, max_seqlen;
  const int64_t* first;
  int64_t first_sb;
  const void* cos;           /* (T, D), token stride cs_sn, or both NULL */
  const void* sin;
  int64_t cs_sn;
  int64_t B, D;
} QfRows8;

/*
 * Quantises new tokens into their pages.  A row with a negative first slot (parked)
 * appends nothing; slots past the row's pages are not written; tokens of no row are
 * not read.  With cos and sin k gets the rotate-half RoPE of qf_rope_append before it
 * is quantised.
 *
 * Slots of the last block behind the row's last token keep their codes.  No page
 * may be written by two rows of a call.
 */
int qf_append_paged8(const QfRows8* rows, void* stream);

/*
 * The rows' slots back in fp16: k and v are written (cos and sin NULL).  Tokens of no
 * row are left as they were; those of a row with a negative first slot, and of slots
 * past the row's pages, become zero.
 */
int qf_read_paged8(const QfRows8* rows, void* stream);

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

/* Queries of single tokens: q and out (B, KVH, G, D), G at most 16, one layer's pool. */
typedef struct {
  QfPool8 pool;
  const void* q;
  int64_t q_sb, q_sh, q_sg;
  const int64_t* kv_last;    /* row b's last slot: kv_last[b * kv_last_sb] */
  int64_t kv_last_sb;
  void* out;
  int64_t o_sb, o_sh, o_sg;
  void* ws;
  int64_t ws_bytes;
  int64_t B, G, D;
  const void* k_new;         /* (B, KVH, D): strides per row and head; or both NULL */
  int64_t kn_sb, kn_sh;
  const void* v_new;
  int64_t vn_sb, vn_sh;
  double scale;              /* > 0 */
} QfDecode8;

/*
 * Decode attention of single tokens: softmax(scale q K^T) V over each row's slots
 * [0, kv_last], as qf_decode_attn_paged without a bias.  A row with kv_last < 0
 * (parked) gets zeros.  With k_new and v_new row b's token is appended at slot
 * kv_last first, as by qf_append_paged8 (a slot past the row's pages appends nothing).
 *
 * ws is 16-byte aligned scratch of at least qf_decode_attn_paged8_workspace bytes for
 * these sizes (cap = pages_per_row * page_size; NULL where that is 0), else
 * QF_ERR_SCRATCH_LIMIT; free again when the call's work is done, and not to be shared
 * by calls that overlap in time.
 *
 * Slots that a row does not see may hold anything.  A block that reads as NaN makes
 * NaN of the rows that see any of it; where every score is -infinity the output is NaN.
 */
int64_t qf_decode_attn_paged8_workspace(int B, int KVH, int G, int cap);

int qf_decode_attn_paged8(const QfDecode8* args, void* stream);

/*
 * Its split phase alone (out and ws unused): the partials acc (B, KVH, splits, G, D),
 * m and l (B, KVH, splits, G) of qf_decode_split_paged, for qf_decode_combine or
 * qf_attn_merge_o_proj (m in natural units; a range without a slot leaves acc = l = 0
 * and m = -infinity).  acc is 16-byte aligned.
 */
int qf_decode_split_paged8(const QfDecode8* args, float* acc, float* m, float* l, int splits,
                           void* stream);

/* New tokens with their queries: q and out (T, QH, D), QH a multiple of the pool's KVH, at
 * most 16 times it. */
typedef struct {
  QfRows8 rows;              /* k and v appended at first[b] + i, one layer */
  const void* q;
  int64_t q_sh, q_sn;
  void* out;
  int64_t o_sh, o_sn;
  int64_t cap;               /* slots of a row that the call may use */
  void* ws;
  int64_t ws_bytes;
  int64_t QH;
  double scale;              /* > 0 */
} QfExtend8;

/*
 * New tokens behind cached ones: qf_append_paged8 of a layer's k and v, then token i of
 * row b attends to slots [0, first[b] + i] of its pages -- all of them as the pages
 * hold them, the new ones too.  cos and sin rotate q as well.
 *
 * Rows of out for tokens of no row are left as they were; those of a parked row become
 * zero.  cap is at most pages_per_row * page_size, a
 * bound on every row's first + tokens, from which the work is split; tokens past it
 * are not appended and see the slots below.  ws as above,
 * qf_prefill_extend_paged8_workspace bytes.
 */
int64_t qf_prefill_extend_paged8_workspace(int B, int QH, int KVH, int total, int max_seqlen, int cap);

int qf_prefill_extend_paged8(const QfExtend8* args, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* QF_PAGED8_H */
