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
 * Copies pages within every one of n_pools page pools: for each pair i, slots
 * [0, slots[i]) of all KVH heads of page dst[i] become those of page src[i].
 *
 *   pools   HOST array of n_pools device pointers (read during the call), each
 *           a pool (n_pages, KVH, page_size, D) with the strides sp, sh, sn
 *   src, dst  int32[n_pairs] on the device; a pair with a page outside
 *           [0, n_pages) copies nothing
 *   slots   int32[n_pairs] on the device, clamped to [0, page_size]; NULL
 *           copies whole pages
 *
 * No page may be written twice, or written and read, by one call: what such a
 * page holds afterwards is unspecified.  n_pairs = 0 launches nothing.
 */
int qf_copy_pages(const void* const* pools, int n_pools, int64_t sp, int64_t sh, int64_t sn,
                  const int32_t* src, const int32_t* dst, const int32_t* slots, int n_pairs,
                  int n_pages, int KVH, int page_size, int D, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* QF_PREFIX_H */
