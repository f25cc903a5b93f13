// Codes, scales and pages of the caches held in 8 bits (qf_paged8.h).
#pragma once

#include "qf_common.h"
#include "../../include/qf_paged8.h"

namespace qf {
namespace kv8 {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

constexpr int kD = 64;
constexpr int kBlock = QF_BLOCK8;
constexpr int kMinExp = -24;   // of a scale: fp16's least step

// Two codes, bytes 2 kHi and 2 kHi + 1 of w, as halves: the codes themselves for
// int8 (signed bytes given with their top bit flipped, see flip8), their values
// times `scale` for e4m3, which the conversion multiplies in.
template <bool kE4m3, bool kHi>
__device__ __forceinline__ f16x2 code_pair(unsigned w, float scale) {
  if constexpr (kE4m3) {
    return __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, kHi));
  } else {
    // 0x6400 | u is 1024 + u in fp16, u = code + 128.
    const unsigned p = __builtin_amdgcn_perm(0x64646464u, w, kHi ? 0x04030402u : 0x04010400u);
    return __builtin_bit_cast(f16x2, p) - f16x2{(f16)1152.f, (f16)1152.f};
  }
}

// int8 codes offset by 128, four at a time; e4m3 codes as they are.
template <bool kE4m3>
__device__ __forceinline__ unsigned flip8(unsigned w) {
  return kE4m3 ? w : w ^ 0x80808080u;
}

// Eight codes (two words) as the halves of a matrix operand: codes for int8, values
// times `scale` for e4m3.
template <bool kE4m3>
__device__ __forceinline__ f16x8 codes8(unsigned lo, unsigned hi, float scale) {
  lo = flip8<kE4m3>(lo);
  hi = flip8<kE4m3>(hi);
  const f16x2 a = code_pair<kE4m3, false>(lo, scale), b = code_pair<kE4m3, true>(lo, scale);
  const f16x2 c = code_pair<kE4m3, false>(hi, scale), d = code_pair<kE4m3, true>(hi, scale);
  return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Eight codes as their values.  Exact: a code has at most 7 bits, and the scale is
// a power of two that keeps it within fp16.
template <bool kE4m3>
__device__ __forceinline__ f16x8 values8(unsigned lo, unsigned hi, float scale) {
  f16x8 x = codes8<kE4m3>(lo, hi, scale);
  if constexpr (!kE4m3) x *= (f16)scale;
  return x;
}

// The pool's side of a kernel's arguments.
struct Pool {
  uint8_t* k;
  uint8_t* v;
  float* ks;
  float* vs;
  int64_t sl, sp, sh, ssl, ssp, ssh;
  const int32_t* table;
  int64_t t_sb;
  int ppr, n_pages, log2p, kvh;
};

// Checks a caller's pool and fills p; QF_OK or the error.
inline int make_pool(const QfPool8* h, Pool& p) {
  if (!h) return QF_ERR_INVALID_ARG;
  const int l2 = page_log2(h->page_size, h->pages_per_row, h->n_pages);
  if (l2 < 0 || (h->code != QF_CODE_INT8 && h->code != QF_CODE_E4M3)) return QF_ERR_UNSUPPORTED;
  if (!h->k || !h->v || !h->k_scale || !h->v_scale || !h->table || h->KVH < 1 || h->layers < 1 ||
      h->bt_sb < h->pages_per_row)
    return QF_ERR_INVALID_ARG;
  const uintptr_t all = reinterpret_cast<uintptr_t>(h->k) | reinterpret_cast<uintptr_t>(h->v) |
                        (uintptr_t)h->sl | (uintptr_t)h->sp | (uintptr_t)h->sh;
  if ((all & 15u) != 0 || ((reinterpret_cast<uintptr_t>(h->k_scale) |
                            reinterpret_cast<uintptr_t>(h->v_scale)) & 3u) != 0)
    return QF_ERR_INVALID_ARG;
  if (h->sp < 0 || h->sh < 0 || h->sl < 0 || h->ssp < 0 || h->ssh < 0 || h->ssl < 0 ||
      h->KVH > 65535 / h->layers)
    return QF_ERR_UNSUPPORTED;
  p = {static_cast<uint8_t*>(h->k), static_cast<uint8_t*>(h->v), h->k_scale, h->v_scale,
       h->sl, h->sp, h->sh, h->ssl, h->ssp, h->ssh, h->table, h->bt_sb,
       h->pages_per_row, h->n_pages, l2, h->KVH};
  return QF_OK;
}

// qf_append_paged8 into the rows' slots below cap (paged8.hip).
int append(const void* k, int64_t k_sl, int64_t k_sh, int64_t k_sn, const void* v, int64_t v_sl,
           int64_t v_sh, int64_t v_sn, const int32_t* cu_seqlens, int total, int max_seqlen,
           const int64_t* context, int64_t ctx_sb, const void* cos, const void* sin, int64_t cs_sn,
           const QfPool8* pool, int cap, int B, int D, hipStream_t st);

__device__ __forceinline__ int clampi(int64_t x, int lo, int hi) {
  return (int)(x < lo ? lo : x > hi ? hi : x);
}

}  // namespace kv8
}  // namespace qf
