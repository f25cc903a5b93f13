// Codes, scales and pages of the caches held in 8 bits (qf_paged8.h).
#pragma once

#include "qf_common.h"
#include "kv8_pieces.h"
#include "../../include/qf_paged8.h"

namespace qf {
namespace kv8 {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

constexpr int kD = 64;
constexpr int kBlock = QF_BLOCK8;
constexpr int kMinExp = -24;   // of a scale: fp16's least step

// Two codes, bytes 2 kHi and 2 kHi + 1 of w, as halves of one word: e4m3 codes as
// their values times `scale`, which the conversion multiplies in; int8 codes, given
// with their top bit flipped (flip8), plus 1152 -- 0x6400 | u is 1024 + u in fp16, and
// u = code + 128.
template <bool kE4m3, bool kHi>
__device__ __forceinline__ f16x2 code_pair(unsigned w, float scale) {
  if constexpr (kE4m3)
    return __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, kHi));
  else
    return __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w, kHi ? 0x04030402u : 0x04010400u));
}

// int8 codes offset by 128, four at a time; e4m3 codes as they are.
template <bool kE4m3>
__device__ __forceinline__ unsigned flip8(unsigned w) {
  return kE4m3 ? w : w ^ 0x80808080u;
}

// Eight codes (two words) as the halves of a matrix operand, int8 ones through `fix`,
// which takes the 1152 off a pair.  The halves stay pairs in 32-bit words: put
// together one by one they are taken apart and packed again.
template <bool kE4m3, typename Fix>
__device__ __forceinline__ f16x8 convert8(unsigned lo, unsigned hi, float scale, Fix&& fix) {
  lo = flip8<kE4m3>(lo);
  hi = flip8<kE4m3>(hi);
  f16x2 x[4] = {code_pair<kE4m3, false>(lo, scale), code_pair<kE4m3, true>(lo, scale),
                code_pair<kE4m3, false>(hi, scale), code_pair<kE4m3, true>(hi, scale)};
  u32x4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = __builtin_bit_cast(unsigned, kE4m3 ? x[i] : fix(x[i]));
  return __builtin_bit_cast(f16x8, w);
}

// Eight codes: int8 codes themselves, e4m3 values times `scale`.
template <bool kE4m3>
__device__ __forceinline__ f16x8 codes8(unsigned lo, unsigned hi, float scale) {
  const f16x2 off = {(f16)1152.f, (f16)1152.f};
  return convert8<kE4m3>(lo, hi, scale, [&](f16x2 x) { return x - off; });
}

// What takes 1152 off int8 codes and multiplies them by a scale in one fma, which is
// exact: scales up to 2^5, past which 1152 * scale is more than fp16 holds.
struct Affine {
  f16x2 mul, sub;
};
constexpr float kAffineMost = 32.f;

__device__ __forceinline__ Affine affine(float scale) {
  const f16 s = (f16)scale, o = (f16)(-1152.f * scale);
  return {{s, s}, {o, o}};
}

// Eight codes as their values.  Exact: a code has at most 7 bits, and the scale is
// a power of two that keeps it within fp16.
template <bool kE4m3>
__device__ __forceinline__ f16x8 values8(unsigned lo, unsigned hi, float scale) {
  const f16x2 off = {(f16)1152.f, (f16)1152.f}, s = {(f16)scale, (f16)scale};
  return convert8<kE4m3>(lo, hi, scale, [&](f16x2 x) { return (x - off) * s; });
}

template <bool kE4m3>
__device__ __forceinline__ f16x8 values8(unsigned lo, unsigned hi, float scale, const Affine& f) {
  return convert8<kE4m3>(lo, hi, scale, [&](f16x2 x) { return __builtin_elementwise_fma(x, f.mul, f.sub); });
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
inline int make_pool(const QfPool8& h, Pool& p) {
  constexpr int64_t kInt = 0x7fffffff;
  if (h.page_size < 0 || h.page_size > kInt || h.pages_per_row < 0 || h.pages_per_row > kInt ||
      h.n_pages < 0 || h.n_pages > kInt)
    return QF_ERR_UNSUPPORTED;
  const int l2 = page_log2((int)h.page_size, (int)h.pages_per_row, (int)h.n_pages);
  if (l2 < 0 || (h.code != QF_CODE_INT8 && h.code != QF_CODE_E4M3)) return QF_ERR_UNSUPPORTED;
  if (!h.k || !h.v || !h.k_scale || !h.v_scale || !h.table || h.KVH < 1 || h.layers < 1 ||
      h.bt_sb < h.pages_per_row)
    return QF_ERR_INVALID_ARG;
  const uintptr_t all = reinterpret_cast<uintptr_t>(h.k) | reinterpret_cast<uintptr_t>(h.v) |
                        (uintptr_t)h.sl | (uintptr_t)h.sp | (uintptr_t)h.sh;
  if ((all & 15u) != 0 || ((reinterpret_cast<uintptr_t>(h.k_scale) |
                            reinterpret_cast<uintptr_t>(h.v_scale)) & 3u) != 0)
    return QF_ERR_INVALID_ARG;
  if (h.sp < 0 || h.sh < 0 || h.sl < 0 || h.ssp < 0 || h.ssh < 0 || h.ssl < 0 || h.layers > 65535 ||
      h.KVH > 65535 / h.layers)
    return QF_ERR_UNSUPPORTED;
  p = {static_cast<uint8_t*>(h.k), static_cast<uint8_t*>(h.v), h.k_scale, h.v_scale,
       h.sl, h.sp, h.sh, h.ssl, h.ssp, h.ssh, h.table, h.bt_sb,
       (int)h.pages_per_row, (int)h.n_pages, l2, (int)h.KVH};
  return QF_OK;
}

inline int row_cap(const Pool& p) { return p.ppr << p.log2p; }

// What a call has to say about packed tokens, but for its pool (paged8.hip).
int check_rows(const QfRows8& rows);

// qf_append_paged8 into the rows' slots below cap (paged8.hip).
int append(const QfRows8& rows, int cap, hipStream_t st);

// The sum of x >= 0 over the lanes up to this one, held at the largest int.
__device__ __forceinline__ int scan_sum(int x) {
  const int lane = threadIdx.x & 63;
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(x, d);
    if (lane >= d) x = add_capped(x, y);
  }
  return x;
}

__device__ __forceinline__ int clampi(int64_t x, int lo, int hi) {
  return (int)(x < lo ? lo : x > hi ? hi : x);
}

}  // namespace kv8
}  // namespace qf
