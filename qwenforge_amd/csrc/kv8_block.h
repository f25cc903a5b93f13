// One block of the caches held in 8 bits, written by a wave (qf_paged8.h):
//   scale = max(the scale of the slots already there, 2^e), the least e >= -24 with
//           max |x| <= Q 2^e (Q = 127 or 448), read off the exponent and mantissa
//           of the largest magnitude;
//   code  = rne(x 2^-e), which is exact before the rounding.
// K goes through it as four lanes a slot, each with the dims [8c, 8c + 8) and
// [32 + 8c, 40 + 8c) that a rotate-half pair needs; V as two dims and eight slots a
// lane: a token's two dims are one word, and a dim's eight slots 8 bytes of the
// dim-major page.
#pragma once

#include "kv8.h"

namespace qf {
namespace kv8 {

// The least scale of a block whose largest magnitude has these fp16 bits.
template <bool kE4m3>
__device__ __forceinline__ float scale_for(unsigned top) {
  if (top >= 0x7C00u) return __builtin_nanf("");
  const unsigned f = __float_as_uint((float)__builtin_bit_cast(f16, (unsigned short)top));
  // Q = 1.984375 * 2^6 or 1.75 * 2^8.
  const int e = (int)(f >> 23) - 127 - (kE4m3 ? 8 : 6) +
                ((f & 0x7FFFFFu) > (kE4m3 ? 0x600000u : 0x7E0000u) ? 1 : 0);
  return __uint_as_float((unsigned)(max(e, kMinExp) + 127) << 23);
}

// Largest magnitude at scale s whose value fp16 holds: 65504 / s rounded down to a
// code.  It is below Q where the scale is the largest there is alone.
template <bool kE4m3>
__device__ __forceinline__ float code_top(float s) {
  if (kE4m3) return s >= 256.f ? 240.f : 448.f;
  return s >= 1024.f ? 63.f : 127.f;
}

// Four codes of y[0..3] = x / scale.
template <bool kE4m3>
__device__ __forceinline__ unsigned encode4(const float (&y)[4], float top) {
  float z[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) z[i] = __builtin_amdgcn_fmed3f(y[i], -top, top);
  if constexpr (kE4m3) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(z[0], z[1], 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(z[2], z[3], w, true);
  } else {
    // Adding 1.5 * 2^23 rounds to a whole number, ties to even, in the low bits.
    unsigned b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = __float_as_uint(z[i] + 12582912.f);
    const unsigned lo = __builtin_amdgcn_perm(b[1], b[0], 0x0C0C0400u);
    const unsigned hi = __builtin_amdgcn_perm(b[3], b[2], 0x0C0C0400u);
    return lo | hi << 16;
  }
}

template <bool kE4m3>
__device__ __forceinline__ unsigned encode4(f16 a, f16 b, f16 c, f16 d, float inv, float top) {
  return encode4<kE4m3>({(float)a * inv, (float)b * inv, (float)c * inv, (float)d * inv}, top);
}

// Four codes at the ratio old scale / new scale.
template <bool kE4m3>
__device__ __forceinline__ unsigned recode4(unsigned w, float ratio, float top) {
  const f16x8 x = codes8<kE4m3>(w, w, 1.f);
  return encode4<kE4m3>({(float)x[0] * ratio, (float)x[1] * ratio, (float)x[2] * ratio,
                         (float)x[3] * ratio}, top);
}

__device__ __forceinline__ unsigned magnitudes(f16x8 x) {
  const u32x4 w = __builtin_bit_cast(u32x4, x);
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) top = max(top, max(w[i] & 0x7FFFu, (w[i] >> 16) & 0x7FFFu));
  return top;
}

// By lanes' neighbours within rows of 16 (quads, half rows, rows), then across rows:
// no trip through LDS.
template <int kCtrl>
__device__ __forceinline__ unsigned dpp_max(unsigned x) {
  return max(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, kCtrl, 0xF, 0xF, true));
}

__device__ __forceinline__ unsigned wave_max(unsigned x) {
  x = dpp_max<0xB1>(x);    // quad_perm 1 0 3 2
  x = dpp_max<0x4E>(x);    // quad_perm 2 3 0 1
  x = dpp_max<0x141>(x);   // row_half_mirror
  x = dpp_max<0x140>(x);   // row_mirror
  const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = max(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return max(b[0], b[1]);
}

// The block's new scale, and what its old codes are multiplied by (1: left alone).
struct Scales {
  float s, inv, top, ratio;
  bool bad;
};

template <bool kE4m3>
__device__ __forceinline__ Scales new_scale(unsigned top, float old, bool begun) {
  Scales r;
  const float need = scale_for<kE4m3>(top);
  r.s = need;
  if (begun && !(old < need)) r.s = need == need ? old : need;  // NaN of either stays
  r.bad = !(r.s == r.s);
  r.inv = r.bad ? 0.f : 1.f / r.s;
  r.top = code_top<kE4m3>(r.s);
  r.ratio = begun && old < r.s ? old * r.inv : 1.f;
  return r;
}

// Tokens of one kv head that go to neighbouring slots.
struct Tokens {
  const f16* k;
  int64_t k_sn;
  const f16* v;
  int64_t v_sn;
  const f16* cos;      // of the first token, or null
  const f16* sin;
  int64_t cs_sn;
};

// Where the block of 16 whose first slot is slot0 of a row begins in `page` of the layer.
struct BlockAt {
  int64_t code, scale;
  int in_page;
};

__device__ __forceinline__ BlockAt block_at(const Pool& p, int layer, int hk, int page, int slot0) {
  const int in_page = slot0 & ((1 << p.log2p) - 1);
  return {layer * p.sl + page * p.sp + hk * p.sh, layer * p.ssl + page * p.ssp + hk * p.ssh + (in_page >> 4),
          in_page};
}

// One wave quantises tokens into slots [lo, end) of that block, their keys, their values or
// both; without such a page nothing is written.  All is loaded before any of it is used.
template <bool kE4m3, bool kKeys, bool kValues>
__device__ __forceinline__ void append_block(const Pool& p, int layer, int hk, int page, int slot0, int lo,
                                             int end, const Tokens& tokens) {
  const int lane = threadIdx.x & 63;
  const bool begun = lo > 0;
  // K: slot t, dims c and 32 + c.
  const int t = lane >> 2, c = 8 * (lane & 3);
  const bool fresh = t >= lo && t < end;
  const int64_t tok = fresh ? t - lo : 0;
  f16x8 klo, khi;
  if (kKeys) {
    const f16* src = tokens.k + tok * tokens.k_sn + c;
    klo = load16(src);
    khi = load16(src + 32);
  }
  // V: dims 2d and 2d + 1, slots j0 .. j0 + 7.
  const int d = lane & 31, j0 = lane >> 5 << 3;
  unsigned x[8];
  if (kValues) {
    const f16* src = tokens.v + 2 * d;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const bool in = j0 + j >= lo && j0 + j < end;
      x[j] = 0;
      if (in) x[j] = *reinterpret_cast<const unsigned*>(src + (j0 + j - lo) * tokens.v_sn);
    }
  }
  if (page < 0 || page >= p.n_pages) return;
  const BlockAt at = block_at(p, layer, hk, page, slot0);
  uint8_t* kp = p.k + at.code + (int64_t)at.in_page * kD + t * kD + c;     // 16 slots x 64
  uint8_t* vp = p.v + at.code + (int64_t)(at.in_page >> 6) * 64 * kD + (at.in_page & 63) + 128 * d + j0;
  float ks_old, vs_old;
  u32x2 old_lo = {0, 0}, old_hi = {0, 0}, old_v[2] = {{0, 0}, {0, 0}};
  if (kKeys) ks_old = p.ks[at.scale];
  if (kValues) vs_old = p.vs[at.scale];
  if (begun || end < kBlock) {
    if (kKeys) {
      old_lo = *reinterpret_cast<const u32x2*>(kp);
      old_hi = *reinterpret_cast<const u32x2*>(kp + 32);
    }
    if (kValues) {
      old_v[0] = *reinterpret_cast<const u32x2*>(vp);
      old_v[1] = *reinterpret_cast<const u32x2*>(vp + 64);
    }
  }
  Scales ks, vs;
  if (kKeys) {
    if (tokens.cos != nullptr) {
      const int64_t co = tok * tokens.cs_sn + c;
      rope_pair(klo, khi, load16(tokens.cos + co), load16(tokens.sin + co), load16(tokens.cos + co + 32),
                load16(tokens.sin + co + 32));
    }
    ks = new_scale<kE4m3>(wave_max(fresh ? max(magnitudes(klo), magnitudes(khi)) : 0u), ks_old, begun);
  }
  if (kValues) {
    unsigned top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, max(x[j] & 0x7FFFu, (x[j] >> 16) & 0x7FFFu));
    vs = new_scale<kE4m3>(wave_max(top), vs_old, begun);
  }
  if (kKeys) {
    const Scales s = ks;
    if (fresh || (t < lo && s.ratio != 1.f)) {
      u32x2 lo8, hi8;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (fresh) {
          lo8[i] = s.bad ? 0u : encode4<kE4m3>(klo[4 * i], klo[4 * i + 1], klo[4 * i + 2], klo[4 * i + 3], s.inv, s.top);
          hi8[i] = s.bad ? 0u : encode4<kE4m3>(khi[4 * i], khi[4 * i + 1], khi[4 * i + 2], khi[4 * i + 3], s.inv, s.top);
        } else {
          lo8[i] = recode4<kE4m3>(old_lo[i], s.ratio, s.top);
          hi8[i] = recode4<kE4m3>(old_hi[i], s.ratio, s.top);
        }
      }
      *reinterpret_cast<u32x2*>(kp) = lo8;
      *reinterpret_cast<u32x2*>(kp + 32) = hi8;
    }
  }
  if (kValues) {
    const Scales s = vs;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      u32x2 out;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        f16 y[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = __builtin_bit_cast(f16, (unsigned short)(x[4 * i + j] >> (16 * h)));
        const unsigned w = s.bad ? 0u : encode4<kE4m3>(y[0], y[1], y[2], y[3], s.inv, s.top);
        // Bytes of slots that are new, and of those before them.
        const int n0 = min(max(lo - j0 - 4 * i, 0), 4), n1 = min(max(end - j0 - 4 * i, 0), 4);
        const unsigned below = n0 == 4 ? ~0u : (1u << (8 * n0)) - 1u;
        const unsigned upto = n1 == 4 ? ~0u : (1u << (8 * n1)) - 1u;
        const unsigned old = old_v[h][i];
        const unsigned had = s.ratio != 1.f ? recode4<kE4m3>(old, s.ratio, s.top) : old;
        out[i] = (w & upto & ~below) | (had & below) | (old & ~upto);
      }
      *reinterpret_cast<u32x2*>(vp + 64 * h) = out;
    }
  }
  if (lane == 0) {
    if (kKeys) p.ks[at.scale] = ks.s;
    if (kValues) p.vs[at.scale] = vs.s;
  }
}

}  // namespace kv8
}  // namespace qf
