/*
 * qf_verify.h -- drafted tokens against the target model's logits (gfx950).
 *
 * The reference decodes greedily, one token a step (argmax,
 * student_engine.py:980-982, :1126-1132).  Here a row's last token and the
 * tokens drafted after it have run together (qf_prefill_extend_paged), and the
 * drafts are kept while the target would have drawn them.  Conventions as in
 * qf_attn.h.
 */
#ifndef QF_VERIFY_H
#define QF_VERIFY_H

#include <stdint.h>

#include "qf_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

#define QF_F16 0
#define QF_F32 1

/*
 * Rows packed along the token axis as in qf_prefill_varlen: row b's positions
 * are [cu_seqlens[b], cu_seqlens[b + 1]), n of them, of which the first n - 1
 * judge the row's drafts: position j the token at position j + 1.
 *
 *   logits      (T, V) fp16 or fp32 (dtype), row stride lg_sn: after each position
 *   tokens      int64[T]: each row's last token, then its drafts
 *   accept_u    fp32[T] in [0, 1): position j's number for its draft
 *   sample_u    fp32[B] in [0, 1): for the row's last new token
 *   draft_probs NULL, or fp32 (T, V), row stride dp_sn: the distribution q_j that
 *               position j's draft was drawn from
 *   temperature T > 0 (1 / T a normal fp32 number): p_j = softmax(logits[j] / T).  Draft d is accepted while
 *               accept_u q_j(d) < p_j(d) (q_j(d) = 1 without draft_probs).  After
 *               the first rejection the row's next token is drawn from
 *               max(p_j - q_j, 0) (without draft_probs from p_j without d; from
 *               p_j where nothing is left), after the last draft from p: the
 *               lowest token i with sum_{k <= i} w_k > sample_u sum_k w_k.
 *               T = 0: drafts are accepted while they are the argmax, and the
 *               argmax (ties: the lowest) comes next; the numbers and draft_probs
 *               are not read.
 *   out         int64 (B, width): the accepted drafts, the next token, then -1
 *   count       int64[B]: tokens in each row of out
 *
 * A draft outside [0, V) is rejected.  A position whose logits give no
 * distribution (NaN, or with T > 0 an infinity of +; nothing above -infinity)
 * rejects its draft and draws nothing.  A row without positions gets 0 tokens; no
 * row uses more than `width` positions.  Every new token, accepted or drawn, is
 * the one that exponentials and sums in 64 bits give.  ws: 16-byte aligned, of
 * qf_verify_workspace bytes, else QF_ERR_SCRATCH_LIMIT; not to be shared by calls
 * that overlap in time.
 */
int64_t qf_verify_workspace(int T, int B, int V);

int qf_verify_drafts(const void* logits, int dtype, int64_t lg_sn, const int64_t* tokens,
                     const int32_t* cu_seqlens, const float* accept_u, const float* sample_u,
                     const float* draft_probs, int64_t dp_sn, double temperature,
                     int64_t* out, int width, int64_t* count, void* ws, int64_t ws_bytes,
                     int T, int B, int V, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* QF_VERIFY_H */
