// Tokens quantised into paged caches held in 8 bits, slots read back, pages copied
// (gfx950; the format is qf_paged8.h's).
//
// A wave takes one block of 16 slots of one kv head, K and V:
//   scale = max(the scale of the slots already there, 2^e), the least e >= -24 with
//           max |x| <= Q 2^e (Q = 127 or 448), read off the exponent and mantissa
//           of the largest magnitude;
//   code  = rne(x 2^-e), which is exact before the rounding.
// K goes through it as four lanes a slot, each with the dims [8c, 8c + 8) and
// [32 + 8c, 40 + 8c) that a rotate-half pair needs; V as a lane a dim, whose 16
// slots of the block are 16 bytes of the dim-major page.  Four waves are a
// workgroup, so a page's 64-byte lines of V are written on one CU.
#include <algorithm>

#include "kv8.h"

namespace qf {
namespace kv8 {

constexpr int kWaves = 4;

struct RowsArgs {
  Pool p;
  f16* k;                    // packed tokens: the append's input, the read's output
  int64_t k_sl, k_sh, k_sn;
  f16* v;
  int64_t v_sl, v_sh, v_sn;
  const int32_t* cu;
  const int64_t* first;      // first slot of each row's tokens
  int64_t first_sb;
  int B, total, cap;         // slots of a row from cap on are not there
  const f16* cos;
  const f16* sin;
  int64_t cs_sn;
};

// A wave's work: tokens [tok, tok + n) of a row at slots lo .. lo + n - 1 of its
// block `block`; n = 0: none.  lo < 0: the row is parked.
struct Unit {
  int row, tok, n, lo, block;
};

__device__ __forceinline__ int scan_sum(int x) {
  const int lane = threadIdx.x & 63;
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(x, d);
    if (lane >= d) x += y;
  }
  return x;
}

// Blocks that n slots from `first` touch.
__device__ __forceinline__ int blocks_of(int64_t first, int n) {
  return n <= 0 ? 0 : (int)(((first < 0 ? 0 : first) % kBlock + n + kBlock - 1) / kBlock);
}

// Tokens [lo, hi) of row r, any contents of cu kept within the tokens.
__device__ __forceinline__ void row_tokens(const RowsArgs& a, int r, int& lo, int& hi) {
  lo = clampi(a.cu[r], 0, a.total);
  hi = clampi(a.cu[r + 1], lo, a.total);
}

// The id-th of the blocks that the rows' tokens touch, counted row by row.
__device__ __forceinline__ Unit find_unit(const RowsArgs& a, int id) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int i0 = 0; i0 < a.B; i0 += 64) {
    const int r = min(i0 + lane, a.B - 1);
    int lo, hi;
    row_tokens(a, r, lo, hi);
    const int64_t first = a.first[r * a.first_sb];
    const int mine = i0 + lane < a.B ? blocks_of(first, hi - lo) : 0;
    const int upto = scan_sum(mine);
    const uint64_t hit = __ballot(id < before + upto);
    if (hit != 0) {
      const int j = __builtin_ctzll(hit);
      const int64_t f = ((int64_t)__builtin_amdgcn_readlane((int)(first >> 32), j) << 32) |
                        (unsigned)__builtin_amdgcn_readlane((int)first, j);
      const int l = __builtin_amdgcn_readlane(lo, j), h = __builtin_amdgcn_readlane(hi, j);
      const int k = id - before - __builtin_amdgcn_readlane(upto - mine, j);
      const int64_t at = f < 0 ? 0 : f;           // slot of the row's first token
      const int64_t s0 = at / kBlock * kBlock + (int64_t)k * kBlock;
      const int64_t from = s0 < at ? at : s0;
      const int tok = l + (int)(from - at);
      const int64_t end = s0 + kBlock - from;
      Unit u;
      u.row = i0 + j;
      u.tok = tok;
      u.n = min((int)end, h - tok);
      u.lo = f < 0 ? -1 : (int)(from - s0);
      const int64_t block = s0 / kBlock;
      u.block = (int)(block < 0x7fffffff / kBlock ? block : 0x7fffffff / kBlock);
      return u;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  return {0, 0, 0, 0, 0};
}

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
  const unsigned u = flip8<kE4m3>(w);
  const f16x2 a = code_pair<kE4m3, false>(u, 1.f), b = code_pair<kE4m3, true>(u, 1.f);
  return encode4<kE4m3>({(float)a[0] * ratio, (float)a[1] * ratio, (float)b[0] * ratio,
                         (float)b[1] * ratio}, top);
}

__device__ __forceinline__ unsigned magnitudes(f16x8 x) {
  const u32x4 w = __builtin_bit_cast(u32x4, x);
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) top = max(top, max(w[i] & 0x7FFFu, (w[i] >> 16) & 0x7FFFu));
  return top;
}

__device__ __forceinline__ unsigned wave_max(unsigned x) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) x = max(x, (unsigned)__shfl_xor((int)x, d));
  return x;
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

template <bool kE4m3>
__global__ __launch_bounds__(64 * kWaves) void append_kernel(RowsArgs a) {
  const int lane = threadIdx.x & 63;
  const int id = __builtin_amdgcn_readfirstlane(blockIdx.x * kWaves + (threadIdx.x >> 6));
  const int hk = blockIdx.y % a.p.kvh, layer = blockIdx.y / a.p.kvh;
  const Unit u = find_unit(a, id);
  if (u.n <= 0 || u.lo < 0) return;
  const int slot0 = u.block << 4;                       // of the block
  const int lp = slot0 >> a.p.log2p;
  if (lp >= a.p.ppr) return;
  const int page = a.p.table[u.row * a.p.t_sb + lp];
  if (page < 0 || page >= a.p.n_pages) return;
  const int in_page = slot0 & ((1 << a.p.log2p) - 1);
  const int64_t at = layer * a.p.sl + page * a.p.sp + hk * a.p.sh;
  const int64_t sat = layer * a.p.ssl + page * a.p.ssp + hk * a.p.ssh + (in_page >> 4);
  uint8_t* kp = a.p.k + at + (int64_t)in_page * kD;     // 16 slots x 64
  uint8_t* vp = a.p.v + at + (int64_t)(in_page >> 6) * 64 * kD + (in_page & 63);
  const bool begun = u.lo > 0;
  const int end = min(u.lo + u.n, a.cap - slot0);       // slots [lo, end) of the block are new
  if (end <= u.lo) return;
  const float ks_old = a.p.ks[sat], vs_old = a.p.vs[sat];

  // K: slot t, dims 8c and 32 + 8c.
  const int t = lane >> 2, c = 8 * (lane & 3);
  const bool fresh = t >= u.lo && t < end;
  const int64_t tok = u.tok + (fresh ? t - u.lo : 0);
  const f16* src = a.k + layer * a.k_sl + hk * a.k_sh + tok * a.k_sn + c;
  f16x8 klo = load16(src), khi = load16(src + 32);
  // V: dim `lane`, the block's 16 slots.
  const f16* vsrc = a.v + layer * a.v_sl + hk * a.v_sh + (int64_t)u.tok * a.v_sn + lane;
  f16 x[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const bool in = j >= u.lo && j < end;
    x[j] = in ? vsrc[(j - u.lo) * a.v_sn] : (f16)0.f;
  }
  u32x2 old_lo = {0, 0}, old_hi = {0, 0};
  u32x4 old_v = {0, 0, 0, 0};
  if (begun || end < kBlock) {
    old_lo = *reinterpret_cast<const u32x2*>(kp + t * kD + c);
    old_hi = *reinterpret_cast<const u32x2*>(kp + t * kD + c + 32);
    old_v = *reinterpret_cast<const u32x4*>(vp + lane * 64);
  }
  if (a.cos != nullptr) {
    const int64_t co = tok * a.cs_sn + c;
    rope_pair(klo, khi, load16(a.cos + co), load16(a.sin + co), load16(a.cos + co + 32),
              load16(a.sin + co + 32));
  }
  const Scales k = new_scale<kE4m3>(
      wave_max(fresh ? max(magnitudes(klo), magnitudes(khi)) : 0u), ks_old, begun);
  unsigned vtop = 0;
#pragma unroll
  for (int j = 0; j < 16; ++j)
    vtop = max(vtop, (unsigned)__builtin_bit_cast(unsigned short, x[j]) & 0x7FFFu);
  const Scales v = new_scale<kE4m3>(wave_max(vtop), vs_old, begun);

  if (fresh || (t < u.lo && k.ratio != 1.f)) {
    u32x2 lo, hi;
    if (fresh) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        lo[i] = k.bad ? 0u : encode4<kE4m3>(klo[4 * i], klo[4 * i + 1], klo[4 * i + 2], klo[4 * i + 3], k.inv, k.top);
        hi[i] = k.bad ? 0u : encode4<kE4m3>(khi[4 * i], khi[4 * i + 1], khi[4 * i + 2], khi[4 * i + 3], k.inv, k.top);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        lo[i] = recode4<kE4m3>(old_lo[i], k.ratio, k.top);
        hi[i] = recode4<kE4m3>(old_hi[i], k.ratio, k.top);
      }
    }
    *reinterpret_cast<u32x2*>(kp + t * kD + c) = lo;
    *reinterpret_cast<u32x2*>(kp + t * kD + c + 32) = hi;
  }
  u32x4 out;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned w = v.bad ? 0u : encode4<kE4m3>(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3], v.inv, v.top);
    // Bytes of slots that are new, and of those before them.
    const int n0 = min(max(u.lo - 4 * i, 0), 4), n1 = min(max(end - 4 * i, 0), 4);
    const unsigned below = n0 == 4 ? ~0u : (1u << (8 * n0)) - 1u;
    const unsigned upto = n1 == 4 ? ~0u : (1u << (8 * n1)) - 1u;
    const unsigned had = v.ratio != 1.f ? recode4<kE4m3>(old_v[i], v.ratio, v.top) : old_v[i];
    out[i] = (w & upto & ~below) | (had & below) | (old_v[i] & ~upto);
  }
  *reinterpret_cast<u32x4*>(vp + lane * 64) = out;
  if (lane == 0) {
    a.p.ks[sat] = k.s;
    a.p.vs[sat] = v.s;
  }
}

template <bool kE4m3>
__global__ __launch_bounds__(64 * kWaves) void read_kernel(RowsArgs a) {
  const int lane = threadIdx.x & 63;
  const int id = __builtin_amdgcn_readfirstlane(blockIdx.x * kWaves + (threadIdx.x >> 6));
  const int hk = blockIdx.y % a.p.kvh, layer = blockIdx.y / a.p.kvh;
  const Unit u = find_unit(a, id);
  if (u.n <= 0) return;
  const int slot0 = u.block << 4;
  const int lp = slot0 >> a.p.log2p;
  const bool none = u.lo < 0 || lp >= a.p.ppr;
  const int lo = max(u.lo, 0);
  const int page = none ? 0 : min(max(a.p.table[u.row * a.p.t_sb + lp], 0), a.p.n_pages - 1);
  const int in_page = none ? 0 : slot0 & ((1 << a.p.log2p) - 1);
  const int64_t at = layer * a.p.sl + page * a.p.sp + hk * a.p.sh;
  const int64_t sat = layer * a.p.ssl + page * a.p.ssp + hk * a.p.ssh + (in_page >> 4);
  const float ks = a.p.ks[sat], vs = a.p.vs[sat];
  // Four lanes a slot, 16 dims each.
  const int t = lane >> 2, c = 16 * (lane & 3);
  const u32x4 kw = *reinterpret_cast<const u32x4*>(a.p.k + at + (int64_t)in_page * kD + t * kD + c);
  const u32x4 vw = *reinterpret_cast<const u32x4*>(a.p.v + at + (int64_t)(in_page >> 6) * 64 * kD +
                                                   (in_page & 63) + lane * 64);
  const f16 nan = (f16)__builtin_nanf("");
  f16x8 k0 = values8<kE4m3>(kw[0], kw[1], ks), k1 = values8<kE4m3>(kw[2], kw[3], ks);
  f16x8 v0 = values8<kE4m3>(vw[0], vw[1], vs), v1 = values8<kE4m3>(vw[2], vw[3], vs);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    k0[i] = none ? (f16)0.f : ks == ks ? k0[i] : nan;
    k1[i] = none ? (f16)0.f : ks == ks ? k1[i] : nan;
    v0[i] = none ? (f16)0.f : vs == vs ? v0[i] : nan;
    v1[i] = none ? (f16)0.f : vs == vs ? v1[i] : nan;
  }
  if (t >= lo && t < lo + u.n) {
    f16* dst = a.k + layer * a.k_sl + hk * a.k_sh + (int64_t)(u.tok + t - lo) * a.k_sn + c;
    store16(dst, k0);
    store16(dst + 8, k1);
  }
  f16* dst = a.v + layer * a.v_sl + hk * a.v_sh + (int64_t)u.tok * a.v_sn + lane;
#pragma unroll
  for (int j = 0; j < 16; ++j)
    if (j >= lo && j < lo + u.n) dst[(j - lo) * a.v_sn] = j < 8 ? v0[j & 7] : v1[j & 7];
}

constexpr int kCopyThreads = 256, kCopyUnroll = 4;

// 16 KB of one page of one layer; blockIdx = (piece, pair, layer).
__global__ __launch_bounds__(kCopyThreads) void copy_kernel(uint8_t* store, int64_t layer_step,
                                                            int64_t step, int64_t bytes,
                                                            const int32_t* src, const int32_t* dst,
                                                            int n_pages) {
  const int from = src[blockIdx.y], to = dst[blockIdx.y];
  if (from < 0 || from >= n_pages || to < 0 || to >= n_pages || from == to) return;
  uint8_t* base = store + blockIdx.z * layer_step;
  const uint8_t* s = base + from * step;
  uint8_t* d = base + to * step;
  const int64_t first = ((int64_t)blockIdx.x * kCopyThreads * kCopyUnroll + threadIdx.x) * 16;
  u32x4 w[kCopyUnroll];
#pragma unroll
  for (int i = 0; i < kCopyUnroll; ++i) {
    const int64_t o = first + i * kCopyThreads * 16;
    if (o < bytes) w[i] = *reinterpret_cast<const u32x4*>(s + o);
  }
#pragma unroll
  for (int i = 0; i < kCopyUnroll; ++i) {
    const int64_t o = first + i * kCopyThreads * 16;
    if (o < bytes) *reinterpret_cast<u32x4*>(d + o) = w[i];
  }
}

// Checks and fills what the append and the read share, and the launch's size.
int make_rows(RowsArgs& a, dim3& grid, const void* k, int64_t k_sl, int64_t k_sh, int64_t k_sn,
              const void* v, int64_t v_sl, int64_t v_sh, int64_t v_sn, const int32_t* cu, int total,
              int max_seqlen, const int64_t* first, int64_t first_sb, const QfPool8* pool, int B, int D) {
  if (D != kD) return QF_ERR_UNSUPPORTED;
  if (!pool || !k || !v || !cu || !first || B < 1 || total < 1 || max_seqlen < 1 || max_seqlen > total)
    return QF_ERR_INVALID_ARG;
  if (((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15u) != 0 ||
      ((k_sl | k_sh | k_sn | v_sl | v_sh | v_sn) & 7) != 0)
    return QF_ERR_INVALID_ARG;
  if (B > 0x3fffffff || total > 0x3fffffff) return QF_ERR_UNSUPPORTED;
  a = RowsArgs{};
  const int rc = make_pool(pool, a.p);
  if (rc != QF_OK) return rc;
  a.k = static_cast<f16*>(const_cast<void*>(k));
  a.k_sl = k_sl; a.k_sh = k_sh; a.k_sn = k_sn;
  a.v = static_cast<f16*>(const_cast<void*>(v));
  a.v_sl = v_sl; a.v_sh = v_sh; a.v_sn = v_sn;
  a.cu = cu;
  a.first = first;
  a.first_sb = first_sb;
  a.B = B; a.total = total;
  a.cap = pool->pages_per_row * pool->page_size;
  // A row's n tokens touch at most n / 16 + 2 blocks, one of them if n is 1.
  const int64_t blocks = max_seqlen == 1 ? B : (int64_t)total / kBlock + 2 * (int64_t)std::min(B, total);
  grid = dim3((unsigned)((blocks + kWaves - 1) / kWaves), (unsigned)(pool->KVH * pool->layers));
  return QF_OK;
}

}  // namespace kv8
}  // namespace qf

int qf::kv8::append(const void* k, int64_t k_sl, int64_t k_sh, int64_t k_sn, const void* v, int64_t v_sl,
                    int64_t v_sh, int64_t v_sn, const int32_t* cu_seqlens, int total, int max_seqlen,
                    const int64_t* context, int64_t ctx_sb, const void* cos, const void* sin,
                    int64_t cs_sn, const QfPool8* pool, int cap, int B, int D, hipStream_t st) {
  RowsArgs a;
  dim3 grid;
  const int rc = make_rows(a, grid, k, k_sl, k_sh, k_sn, v, v_sl, v_sh, v_sn, cu_seqlens, total,
                           max_seqlen, context, ctx_sb, pool, B, D);
  if (rc != QF_OK) return rc;
  if ((cos == nullptr) != (sin == nullptr) ||
      ((reinterpret_cast<uintptr_t>(cos) | reinterpret_cast<uintptr_t>(sin)) & 15u) != 0 ||
      (cos != nullptr && (cs_sn & 7) != 0))
    return QF_ERR_INVALID_ARG;
  a.cos = static_cast<const f16*>(cos);
  a.sin = static_cast<const f16*>(sin);
  a.cs_sn = cs_sn;
  a.cap = std::min(a.cap, cap);
  if (pool->code == QF_CODE_E4M3)
    hipLaunchKernelGGL(append_kernel<true>, grid, dim3(64 * kWaves), 0, st, a);
  else
    hipLaunchKernelGGL(append_kernel<false>, grid, dim3(64 * kWaves), 0, st, a);
  return (int)hipGetLastError();
}

extern "C" int qf_append_paged8(const void* k, int64_t k_sl, int64_t k_sh, int64_t k_sn,
                                const void* v, int64_t v_sl, int64_t v_sh, int64_t v_sn,
                                const int32_t* cu_seqlens, int total, int max_seqlen,
                                const int64_t* context, int64_t ctx_sb, const void* cos,
                                const void* sin, int64_t cs_sn, const QfPool8* pool, int B, int D,
                                void* stream) {
  return qf::kv8::append(k, k_sl, k_sh, k_sn, v, v_sl, v_sh, v_sn, cu_seqlens, total, max_seqlen, context,
                         ctx_sb, cos, sin, cs_sn, pool, 0x7fffffff, B, D, static_cast<hipStream_t>(stream));
}

extern "C" int qf_read_paged8(void* k, int64_t k_sl, int64_t k_sh, int64_t k_sn, void* v, int64_t v_sl,
                              int64_t v_sh, int64_t v_sn, const int32_t* cu_seqlens, int total,
                              int max_seqlen, const int64_t* first, int64_t first_sb,
                              const QfPool8* pool, int B, int D, void* stream) {
  using namespace qf;
  using namespace qf::kv8;
  RowsArgs a;
  dim3 grid;
  const int rc = make_rows(a, grid, k, k_sl, k_sh, k_sn, v, v_sl, v_sh, v_sn, cu_seqlens, total,
                           max_seqlen, first, first_sb, pool, B, D);
  if (rc != QF_OK) return rc;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (pool->code == QF_CODE_E4M3)
    hipLaunchKernelGGL(read_kernel<true>, grid, dim3(64 * kWaves), 0, st, a);
  else
    hipLaunchKernelGGL(read_kernel<false>, grid, dim3(64 * kWaves), 0, st, a);
  return (int)hipGetLastError();
}

extern "C" int qf_copy_pages8(void* store, int layers, int64_t layer_step, int64_t step, int64_t bytes,
                              const int32_t* src, const int32_t* dst, int n_pairs, int n_pages,
                              void* stream) {
  using namespace qf::kv8;
  if (!store || layers < 1 || bytes < 16 || n_pairs < 0 || n_pages < 1 || step < bytes)
    return QF_ERR_INVALID_ARG;
  if (((reinterpret_cast<uintptr_t>(store) | (uintptr_t)layer_step | (uintptr_t)step |
        (uintptr_t)bytes) & 15u) != 0)
    return QF_ERR_INVALID_ARG;
  if (layers > 65535 || bytes > 0x7fffffff) return QF_ERR_UNSUPPORTED;
  if (n_pairs == 0) return QF_OK;
  if (!src || !dst) return QF_ERR_INVALID_ARG;
  constexpr int kPiece = kCopyThreads * kCopyUnroll * 16, kMaxPairs = 65535;
  for (int i0 = 0; i0 < n_pairs; i0 += kMaxPairs) {
    const int n = n_pairs - i0 < kMaxPairs ? n_pairs - i0 : kMaxPairs;
    hipLaunchKernelGGL(copy_kernel, dim3((unsigned)((bytes + kPiece - 1) / kPiece), n, layers),
                       dim3(kCopyThreads), 0, static_cast<hipStream_t>(stream),
                       static_cast<uint8_t*>(store), layer_step, step, bytes, src + i0, dst + i0,
                       n_pages);
    const int rc = (int)hipGetLastError();
    if (rc != 0) return rc;
  }
  return QF_OK;
}
