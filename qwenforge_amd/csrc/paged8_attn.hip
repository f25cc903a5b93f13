// Attention over paged caches held in 8 bits (gfx950; the format is qf_paged8.h's):
// single tokens of a batch, and new tokens behind cached ones.
//
// softmax(q K^T) V over slots [0, lim) of a row's pages, lim differing by query, is
// cut into units: up to 16 kNC query rows (token, query head of one kv head) times
// a range of slots.  The waves of a unit's workgroup take tiles of 64 slots in turn and
// join their states in LDS; what several ranges of a query leave is joined by
// merge_kernel.
//
// A tile is 8 KB of codes, K and V both loaded straight into matrix-core operands,
// 16 bytes a lane: with lane group g = lane / 16,
//   K  lane r + 16 g of load (u, j) has dims [16 g, 16 g + 16) of slot
//      16 (r / 4) + 8 u + 4 j + r % 4, so that element i of score tile (u, j) is
//      slot 16 g + 8 u + 4 j + i;
//   V  lane r + 16 g of load t has slots [16 g, 16 g + 16) of dim 16 t + r, which the
//      dim-major pages hold side by side: no transposition anywhere.
// So all 16 slots whose scores and values a lane has are one block of the cache, and a
// tile's scales are two floats a lane.  K's scale goes into the factor that the scores
// have anyway; V's into the conversion of its codes to fp16, which is exact.
#include <algorithm>

#include "kv8_block.h"
#include "lds_tile.h"

namespace qf {
namespace kv8 {

constexpr int kTile = 64;                    // slots
constexpr int kMaxSplits = 64;

typedef float f32x8 __attribute__((ext_vector_type(8)));

struct AttnArgs {
  Pool p;
  const f16* q;
  int64_t q_st, q_sh, q_sg;                  // token, kv head, query head of the kv head
  const int32_t* cu;                         // extension: the rows' tokens
  const int64_t* last;                       // decode: last slot; extension: cached slots
  int64_t last_sb;
  int B, tokens, G, cap;
  int longest;                               // extension: tokens of a row that get an output
  int n_tiles, splits;                       // query tiles of a row, splits of a row's slots
  float* acc;                                // (token, kv head, split, query head, 64)
  float* m;                                  // (token, kv head, split, query head), times m_unit
  float* l;
  float m_unit;                              // ln 2 where a caller's own merge reads m
  int fill;                                  // ranges without a slot leave partials too
  f16* out;
  int64_t o_st, o_sh, o_sg;
  float scale_log2;
  const f16* cos;
  const f16* sin;
  int64_t cs_sn;
  // New tokens that the attention itself appends, or null.  Decode: a row's for its slot
  // `last`.  Extension: the packed ones, where a unit has all of a row's queries.
  const f16* kn;
  int64_t kn_st, kn_sh;
  const f16* vn;
  int64_t vn_st, vn_sh;
};

// Slots [k0, k1) of split s of [0, end): cut at multiples of `least` and 64.
__device__ __forceinline__ void cut(int end, int s, int n, int& k0, int& k1) {
  const int tiles = (end + kTile - 1) / kTile;
  const int len = (tiles + n - 1) / n * kTile;
  const int64_t at = (int64_t)s * len;
  k0 = (int)(at < end ? at : end);
  k1 = (int)(at + len < end ? at + len : end);
}

struct Unit {
  int tok0, rows, r0;     // the row's first token, its query rows, the unit's first one
  int row, hk, split;
  int ctx;                // extension: cached slots, -1 parked
  int k0, k1;
};

struct Raw {
  u32x4 k[4], v[4];
  float ks, vs;
};

// A row's pages of one kv head, read tile by tile in ascending order.
struct Source {
  const uint8_t* k;
  const uint8_t* v;
  const float* ks;
  const float* vs;
  const int32_t* row;
  int64_t sp, ssp;
  int pid, pwin;          // lane j: page of logical page pwin + j
  int log2p, ppr, n_pages;
  int koff, voff;         // of the lane within a tile
};

__device__ __forceinline__ void load_pids(Source& s, int win) {
  const int j = min(win + (int)(threadIdx.x & 63), s.ppr - 1);
  s.pid = min(max(s.row[j], 0), s.n_pages - 1);
  s.pwin = win;
}

// Loads the tile at slot0 where `valid`; without it nothing is fetched, but the loads
// count: what a wave waits for then does not depend on where its tiles end.
template <bool kNt>
__device__ __forceinline__ void load_tile(Raw& r, Source& s, int slot0, bool valid) {
  const int lp = valid ? slot0 >> s.log2p : s.pwin;
  if (lp - s.pwin >= 64) load_pids(s, lp);
  const int64_t page = __builtin_amdgcn_readlane(s.pid, lp - s.pwin);
  const int in_page = slot0 & ((1 << s.log2p) - 1);
  const int64_t at = page * s.sp + in_page * kD, sat = page * s.ssp + (in_page >> 4);
  const int g = (threadIdx.x & 63) >> 4;
  constexpr int aux = kNt ? 2 : 0;
  const __amdgpu_buffer_rsrc_t rk = buffer_rsrc(s.k + at, valid ? kTile * kD : 0);
  const __amdgpu_buffer_rsrc_t rv = buffer_rsrc(s.v + at, valid ? kTile * kD : 0);
  const __amdgpu_buffer_rsrc_t rks = buffer_rsrc(s.ks + sat, valid ? 16 : 0);
  const __amdgpu_buffer_rsrc_t rvs = buffer_rsrc(s.vs + sat, valid ? 16 : 0);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    r.k[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rk, s.koff + i * 4 * kD, 0, aux));
  r.ks = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rks, 4 * g, 0, 0));
#pragma unroll
  for (int i = 0; i < 4; ++i)
    r.v[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rv, s.voff + i * 16 * kTile, 0, aux));
  r.vs = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rvs, 4 * g, 0, 0));
}

// The softmax state of kNC blocks of 16 query columns.
template <int kNC>
struct State {
  f16x8 q[kNC][2];      // dims 16 g + 8 h ..
  int lim[kNC];
  int seen;             // every column sees [0, seen)
  float m[kNC];         // log2 units
  f32x4 l[kNC];
  f32x4 o[kNC][4];
};

// The unit's query rows from `first` on; what each sees is set_limits'.
template <int kNC, bool kDecode>
__device__ __forceinline__ void load_queries(State<kNC>& s, const AttnArgs& a, const Unit& u, int first) {
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
#pragma unroll
  for (int b = 0; b < kNC; ++b) {
    const int rr = min(first + 16 * b + col, u.rows - 1);
    const int token = kDecode ? u.tok0 : u.tok0 + rr / a.G, h = kDecode ? rr : rr % a.G;
    const f16* qp = a.q + token * a.q_st + u.hk * a.q_sh + h * a.q_sg + 16 * g;
#pragma unroll
    for (int i = 0; i < 2; ++i) s.q[b][i] = load16(qp + 8 * i);
    if (!kDecode && a.cos != nullptr) {
      // The other half of the rotated pairs is the lane's 32 away.
      const f16* other = qp + (g < 2 ? 32 : -32);
      const int64_t co = token * a.cs_sn + 16 * (g & 1);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        f16x8 x = g < 2 ? s.q[b][i] : load16(other + 8 * i);
        f16x8 y = g < 2 ? load16(other + 8 * i) : s.q[b][i];
        rope_pair(x, y, load16(a.cos + co + 8 * i), load16(a.sin + co + 8 * i),
                  load16(a.cos + co + 8 * i + 32), load16(a.sin + co + 8 * i + 32));
        s.q[b][i] = g < 2 ? x : y;
      }
    }
    s.m[b] = kNegInf;
    s.l[b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int t = 0; t < 4; ++t) s.o[b][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
}

template <int kNC, bool kDecode>
__device__ __forceinline__ void set_limits(State<kNC>& s, const AttnArgs& a, const Unit& u, int first) {
  const int col = threadIdx.x & 15;
  int least = u.k1;
#pragma unroll
  for (int b = 0; b < kNC; ++b) {
    s.lim[b] = u.k1;
    if (!kDecode) {
      const int r = first + 16 * b + col;
      if (r < u.rows) s.lim[b] = min(u.ctx + r / a.G + 1, u.k1);
      least = min(least, s.lim[b]);
    }
  }
  if (!kDecode) {
    for (int d = 8; d > 0; d >>= 1) least = min(least, __shfl_xor(least, d));
    least = __builtin_amdgcn_readfirstlane(least);
  }
  s.seen = least;
}

// What a tile's scales mean for a lane's 16 slots: the scores' factor, the values' scale
// (1 where the lane has no slot below k1), and whether they read as NaN.
struct Block {
  float ks2, vs;
  bool bad;
};

__device__ __forceinline__ Block block_scales(float ks, float vs, int have, float scale_log2) {
  Block r;
  r.ks2 = ks * scale_log2;
  r.vs = have <= 0 ? 1.f : vs;
  r.bad = !(r.vs == r.vs);
  if (r.bad) r.vs = 0.f;   // zeros, and NaN probabilities for who sees them
  return r;
}

// Slots behind the last one may hold anything: of the lane's 16 the first `have` keep
// their codes, the others become zeros.
__device__ __forceinline__ u32x4 keep_slots(u32x4 w, int have) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int n = min(max(have - 4 * i, 0), 4);
    w[i] &= n == 4 ? ~0u : (1u << (8 * n)) - 1u;
  }
  return w;
}

// Online softmax and PV product from a tile's scores; `values` gives operand (t, u) of
// V^T.  `left`: how many of the lane's 16 slots, from the first on, a column sees.
template <int kNC, typename Values>
__device__ __forceinline__ void attend_tile(State<kNC>& s, f32x4 (&sc)[kNC][4], const Block& blk, int key0,
                                            Values&& values) {
  const int g = (threadIdx.x & 63) >> 4;
  const bool masked = key0 + kTile > s.seen;
  float f[kNC], mx[kNC];
  bool grew = false;
#pragma unroll
  for (int b = 0; b < kNC; ++b) {
    f[b] = blk.ks2;
    if (masked) {
      const int left = s.lim[b] - key0 - 16 * g;
      if (left <= 0) f[b] = 1.f;   // whatever scale an unseen block has
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (i >= left) sc[b][i / 4][i % 4] = kNegInf;
    }
    mx[b] = max16(sc[b]) * f[b];
    grew = grew || mx[b] > s.m[b] + kRescaleSlack;
  }
  // Moves the references of the columns whose own scores grew past them.
  if (__any(grew)) {
#pragma unroll
    for (int b = 0; b < kNC; ++b) {
      const float top = col_max(mx[b]);
      const float m_new = top > s.m[b] + kRescaleSlack ? top : s.m[b];
      const float c = m_new == s.m[b] ? 1.f : fast_exp2(s.m[b] - m_new);
      s.l[b] *= c;
#pragma unroll
      for (int t = 0; t < 4; ++t) s.o[b][t] *= c;
      s.m[b] = m_new;
    }
  }
  const f16x8 ones = {(f16)1.f, (f16)1.f, (f16)1.f, (f16)1.f, (f16)1.f, (f16)1.f, (f16)1.f, (f16)1.f};
  f16x8 p[kNC][2];
#pragma unroll
  for (int b = 0; b < kNC; ++b) {
    // p is rounded to fp16 for the matrix cores (2^-12 of it at most, as much as the
    // output's own rounding), and the sum adds the rounded ones: the weights add to one.
    const float neg_m = s.m[b] == kNegInf ? 0.f : -s.m[b];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      f32x8 x;
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = fast_exp2(__builtin_fmaf(sc[b][2 * u + e / 4][e % 4], f[b], neg_m));
      p[b][u] = __builtin_convertvector(x, f16x8);
    }
  }
  if (__any(blk.bad)) {
#pragma unroll
    for (int b = 0; b < kNC; ++b)
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (blk.bad && s.lim[b] > key0 + 16 * g) p[b][u][e] = (f16)__builtin_nanf("");
  }
#pragma unroll
  for (int b = 0; b < kNC; ++b)
#pragma unroll
    for (int u = 0; u < 2; ++u) s.l[b] = mfma16x16x32(ones, p[b][u], s.l[b]);
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const f16x8 v = values(t, u);
#pragma unroll
      for (int b = 0; b < kNC; ++b) s.o[b][t] = mfma16x16x32(v, p[b][u], s.o[b][t]);
    }
}

// Scores, softmax and PV product of the tile at key0.  `next` loads what comes after
// it, once the tile's codes are in fp16.
template <bool kE4m3, int kNC, typename Next>
__device__ __forceinline__ void tile_step(State<kNC>& s, Raw& r, int key0, int k1, float scale_log2,
                                          Next&& next) {
  const int g = (threadIdx.x & 63) >> 4;
  const int have = k1 - key0 - 16 * g;  // of the lane's 16 slots
  const Block blk = block_scales(r.ks, r.vs, have, scale_log2);
  if (key0 + kTile > k1) {
#pragma unroll
    for (int t = 0; t < 4; ++t) r.v[t] = keep_slots(r.v[t], have);
  }
  f16x8 k[4][2], v[4][2];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int h = 0; h < 2; ++h) k[i][h] = codes8<kE4m3>(r.k[i][2 * h], r.k[i][2 * h + 1], 1.f);
  if (kE4m3 || !__any(blk.vs > kAffineMost)) {
    const Affine f = affine(blk.vs);
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int u = 0; u < 2; ++u) v[t][u] = values8<kE4m3>(r.v[t][2 * u], r.v[t][2 * u + 1], blk.vs, f);
  } else {
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int u = 0; u < 2; ++u) v[t][u] = values8<kE4m3>(r.v[t][2 * u], r.v[t][2 * u + 1], blk.vs);
  }
  next();
  f32x4 sc[kNC][4];
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int b = 0; b < kNC; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        sc[b][i] = mfma16x16x32(k[i][h], s.q[b][h], h == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : sc[b][i]);
  attend_tile<kNC>(s, sc, blk, key0, [&](int t, int u) { return v[t][u]; });
}

__device__ __forceinline__ void store_out(const AttnArgs& a, int token, int hk, int g, int d, f32x4 o,
                                          float l, bool sees) {
  const float inv = sees ? 1.f / l : 0.f;
  const f16x4 r = {(f16)(o[0] * inv), (f16)(o[1] * inv), (f16)(o[2] * inv), (f16)(o[3] * inv)};
  *reinterpret_cast<f16x4*>(a.out + token * a.o_st + hk * a.o_sh + g * a.o_sg + d) = r;
}

__device__ __forceinline__ int64_t part_index(const AttnArgs& a, const Unit& u, int token, int g) {
  return (((int64_t)token * a.p.kvh + u.hk) * a.splits + u.split) * a.G + g;
}

// A unit without a slot.
__device__ __forceinline__ void empty_unit(const AttnArgs& a, const Unit& u, int n_rows) {
  if (a.splits > 1 && !a.fill) return;
  for (int i = threadIdx.x; i < n_rows * 16; i += blockDim.x) {
    const int r = u.r0 + (i >> 4), d = 4 * (i & 15);
    if (r >= u.rows) break;
    const int token = u.tok0 + r / a.G, g = r % a.G;
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    if (a.splits == 1 && !a.fill) {
      store_out(a, token, u.hk, g, d, zero, 0.f, false);
    } else {
      const int64_t p = part_index(a, u, token, g);
      *reinterpret_cast<f32x4*>(a.acc + p * kD + d) = zero;
      if (d == 0) {
        a.m[p] = kNegInf;
        a.l[p] = 0.f;
      }
    }
  }
}

// The row's pages, with the first 64 table entries on their way.
__device__ __forceinline__ Source make_source(const AttnArgs& a, const Unit& u) {
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  Source s;
  s.row = a.p.table + u.row * a.p.t_sb;
  s.ppr = a.p.ppr; s.n_pages = a.p.n_pages;
  load_pids(s, 0);
  s.k = a.p.k + u.hk * a.p.sh;
  s.v = a.p.v + u.hk * a.p.sh;
  s.ks = a.p.ks + u.hk * a.p.ssh;
  s.vs = a.p.vs + u.hk * a.p.ssh;
  s.sp = a.p.sp;
  s.ssp = a.p.ssp;
  s.log2p = a.p.log2p;
  s.koff = (16 * (col >> 2) + (col & 3)) * kD + 16 * g;
  s.voff = col * kTile + 16 * g;
  return s;
}

// A unit whose queries are in s.
template <bool kE4m3, int kNC, bool kDecode>
__device__ __forceinline__ void run_unit(const AttnArgs& a, const Unit& u, Source& src, State<kNC>& s,
                                         f32x4* lds) {
  if (u.k1 <= u.k0) {
    empty_unit(a, u, 16 * kNC);
    return;
  }
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = blockDim.x >> 6;
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int n = (u.k1 - u.k0 + kTile - 1) / kTile;
  const int mine = (n - w + nw - 1) / nw;      // tiles of this wave, from w on every nw-th
  const auto slot = [&](int j) { return u.k0 + (w + j * nw) * kTile; };
  if constexpr (kNC == 1) {
    // Two tiles ahead: a wave that is alone on its SIMD takes a tile in less time than
    // memory answers in.
    Raw r0, r1;
    load_tile<kDecode>(r0, src, slot(0), 0 < mine);
    load_tile<kDecode>(r1, src, slot(1), 1 < mine);
    set_limits<kNC, kDecode>(s, a, u, u.r0);
    int j = 0;
    for (; j + 2 <= mine; j += 2) {
      tile_step<kE4m3, kNC>(s, r0, slot(j), u.k1, a.scale_log2,
                            [&] { load_tile<kDecode>(r0, src, slot(j + 2), j + 2 < mine); });
      tile_step<kE4m3, kNC>(s, r1, slot(j + 1), u.k1, a.scale_log2,
                            [&] { load_tile<kDecode>(r1, src, slot(j + 3), j + 3 < mine); });
    }
    if (j < mine) tile_step<kE4m3, kNC>(s, r0, slot(j), u.k1, a.scale_log2, [] {});
  } else {
    Raw r;
    load_tile<kDecode>(r, src, slot(0), 0 < mine);
    set_limits<kNC, kDecode>(s, a, u, u.r0);
    for (int j = 0; j < mine; ++j)
      tile_step<kE4m3, kNC>(s, r, slot(j), u.k1, a.scale_log2,
                            [&] { load_tile<kDecode>(r, src, slot(j + 1), j + 1 < mine); });
  }
  // The waves' states, a block of columns at a time.
  f32x4* so = lds;                                          // [wave][d tile][lane]
  float2* sml = reinterpret_cast<float2*>(lds + nw * 256);  // [wave][column]
#pragma unroll
  for (int b = 0; b < kNC; ++b) {
    if (b > 0) __syncthreads();
#pragma unroll
    for (int t = 0; t < 4; ++t) so[(w * 4 + t) * 64 + lane] = s.o[b][t];
    if (g == 0) sml[w * 16 + col] = float2{s.m[b], s.l[b][0]};
    __syncthreads();
    const int rr = u.r0 + 16 * b + col;
    const int t = w;   // dims 16 t ..
    if (w < 4 && rr < u.rows) {
      float top = kNegInf;
      for (int i = 0; i < nw; ++i) top = fmaxf(top, sml[i * 16 + col].x);
      float sum = 0.f;
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
      for (int i = 0; i < nw; ++i) {
        const float2 x = sml[i * 16 + col];
        const float c = x.x == top ? 1.f : fast_exp2(x.x - top);
        sum += x.y * c;
        o += so[(i * 4 + t) * 64 + lane] * c;
      }
      const int token = u.tok0 + rr / a.G, h = rr % a.G;
      if (a.splits == 1 && !a.fill) {
        store_out(a, token, u.hk, h, 16 * t + 4 * g, o, sum, true);
      } else {
        const int64_t p = part_index(a, u, token, h);
        *reinterpret_cast<f32x4*>(a.acc + p * kD + 16 * t + 4 * g) = o;
        if (t == 0 && g == 0) {
          a.m[p] = top * a.m_unit;
          a.l[p] = sum;
        }
      }
    }
  }
}

// The unit's row's new tokens into its slots [first, end), a wave a block.  The waves of
// a workgroup share a first-level cache: past the barrier they see what was written.
template <bool kE4m3, bool kDecode>
__device__ __forceinline__ void append_tokens(const AttnArgs& a, const Unit& u, const Source& src, int first,
                                              int end) {
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = blockDim.x >> 6;
  for (int s0 = (first / kBlock + w) * kBlock; s0 < end; s0 += nw * kBlock) {
    const int from = max(s0, first);
    const int64_t token = u.tok0 + from - first;
    const bool turn = !kDecode && a.cos != nullptr;
    const Tokens t = {a.kn + token * a.kn_st + u.hk * a.kn_sh, a.kn_st, a.vn + token * a.vn_st + u.hk * a.vn_sh,
                      a.vn_st, turn ? a.cos + token * a.cs_sn : nullptr, turn ? a.sin + token * a.cs_sn : nullptr,
                      a.cs_sn};
    append_block<kE4m3>(a.p, 0, u.hk, src.row[s0 >> a.p.log2p], s0, from - s0, min(end - s0, kBlock), t);
  }
  s_waitcnt_vm(0);
  __threadfence_block();
  __syncthreads();
}

template <bool kE4m3>
__global__ __launch_bounds__(512, 2) void decode_kernel(AttnArgs a) {
  extern __shared__ f32x4 lds[];
  Unit u;
  int id = blockIdx.x;
  u.split = id % a.splits;
  id /= a.splits;
  u.hk = id % a.p.kvh;
  u.row = u.tok0 = id / a.p.kvh;
  u.rows = a.G;
  u.r0 = 0;
  u.ctx = -1;
  // The table and the queries are loaded while the row's length is.
  const int64_t last = a.last[u.row * a.last_sb];
  Source src = make_source(a, u);
  State<1> s;
  load_queries<1, true>(s, a, u, 0);
  cut(clampi(last, -1, a.cap - 1) + 1, u.split, a.splits, u.k0, u.k1);
  if (a.kn != nullptr && last >= u.k0 && last < u.k1) {
    // The unit that sees the new token writes it; its block is in no other unit.
    append_tokens<kE4m3, true>(a, u, src, (int)last, (int)last + 1);
  }
  run_unit<kE4m3, 1, true>(a, u, src, s, lds);
}

// The extension's unit of this workgroup, of kRows query rows; false: none.
template <int kRows>
__device__ __forceinline__ bool extend_unit(const AttnArgs& a, Unit& u) {
  // Query tiles that read the same slots share an XCD (workgroups go to the XCDs in
  // turn) and its L2, where there are XCDs enough.
  const int groups = a.B * a.p.kvh * a.splits;
  int id = blockIdx.x;
  if (groups >= 8) id = (id / (8 * a.n_tiles) * 8 + id % 8) * a.n_tiles + id / 8 % a.n_tiles;
  const int tile = id % a.n_tiles;
  id /= a.n_tiles;
  if (id >= groups) return false;
  u.split = id % a.splits;
  id /= a.splits;
  u.hk = id % a.p.kvh;
  u.row = id / a.p.kvh;
  const int lo = clampi(a.cu[u.row], 0, a.tokens);
  const int new_tokens = min(clampi(a.cu[u.row + 1], lo, a.tokens) - lo, a.longest);
  u.tok0 = lo;
  u.rows = new_tokens * a.G;
  u.r0 = tile * kRows;
  if (u.r0 >= u.rows) return false;
  u.ctx = clampi(a.last[u.row * a.last_sb], -1, a.cap);
  // All tiles of a row are cut alike; a tile stops where its newest token does.
  const int end = u.ctx < 0 ? 0 : min(u.ctx + new_tokens, a.cap);
  cut(end, u.split, a.splits, u.k0, u.k1);
  if (u.ctx >= 0) {
    const int newest = (min(u.r0 + kRows, u.rows) - 1) / a.G;
    u.k1 = min(u.k1, min(u.ctx + newest + 1, a.cap));
  }
  return true;
}

// Few query rows: the waves take the tiles in turn.
template <bool kE4m3, int kNC>
__global__ __launch_bounds__(512, 2) void extend_kernel(AttnArgs a) {
  extern __shared__ f32x4 lds[];
  Unit u;
  if (!extend_unit<16 * kNC>(a, u)) return;
  Source src = make_source(a, u);
  State<kNC> s;
  load_queries<kNC, false>(s, a, u, u.r0);
  if (a.kn != nullptr && u.ctx >= 0) append_tokens<kE4m3, false>(a, u, src, u.ctx, u.k1);
  run_unit<kE4m3, kNC, false>(a, u, src, s, lds);
}

// Many query rows: the waves take 32 of them each and share the tiles.  A wave
// turns a quarter of each tile's codes into operands, in LDS, a tile ahead of their
// use: a quarter of the conversions that a wave by itself has for as many queries.
template <bool kE4m3>
__global__ __launch_bounds__(256, 3) void extend_wide_kernel(AttnArgs a) {
  constexpr int kWaves = 4, kQB = 2;
  // [stage][operand: K (i, h), then V (t, u)][lane]
  __shared__ f16x8 lds[2][16][64];
  Unit u;
  if (!extend_unit<16 * kQB * kWaves>(a, u)) return;
  if (u.k1 <= u.k0) {
    empty_unit(a, u, 16 * kQB * kWaves);
    return;
  }
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  Source src = make_source(a, u);
  src.koff += w * 4 * kD;
  src.voff += w * 16 * kTile;
  const int n = (u.k1 - u.k0 + kTile - 1) / kTile;
  struct Part {
    u32x4 k, v;
    float ks, vs;
  };
  const auto load = [&](Part& r, int i) {
    const bool valid = i < n;
    const int slot0 = u.k0 + i * kTile;
    const int lp = valid ? slot0 >> src.log2p : src.pwin;
    if (lp - src.pwin >= 64) load_pids(src, lp);
    const int64_t page = __builtin_amdgcn_readlane(src.pid, lp - src.pwin);
    const int in_page = slot0 & ((1 << src.log2p) - 1);
    const int64_t at = page * src.sp + in_page * kD, sat = page * src.ssp + (in_page >> 4);
    r.k = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
        buffer_rsrc(src.k + at, valid ? kTile * kD : 0), src.koff, 0, 0));
    r.v = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
        buffer_rsrc(src.v + at, valid ? kTile * kD : 0), src.voff, 0, 0));
    r.ks = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(
        buffer_rsrc(src.ks + sat, valid ? 16 : 0), 4 * g, 0, 0));
    r.vs = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(
        buffer_rsrc(src.vs + sat, valid ? 16 : 0), 4 * g, 0, 0));
  };
  // Tile i's part into its stage; returns the scales' meaning for the lane.
  const auto convert = [&](const Part& r, int i) {
    const int key0 = u.k0 + i * kTile, have = u.k1 - key0 - 16 * g;
    const Block blk = block_scales(r.ks, r.vs, have, a.scale_log2);
    const u32x4 vw = key0 + kTile > u.k1 ? keep_slots(r.v, have) : r.v;
    f16x8(&to)[16][64] = lds[i & 1];
    to[2 * w][lane] = codes8<kE4m3>(r.k[0], r.k[1], 1.f);
    to[2 * w + 1][lane] = codes8<kE4m3>(r.k[2], r.k[3], 1.f);
    to[8 + 2 * w][lane] = values8<kE4m3>(vw[0], vw[1], blk.vs);
    to[9 + 2 * w][lane] = values8<kE4m3>(vw[2], vw[3], blk.vs);
    return blk;
  };
  // Every wave's LDS writes are there, and its reads done; loads from memory go on.
  const auto meet = [] {
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_barrier();
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
  };
  Part r0, r1;
  load(r0, 0);
  load(r1, 1);
  State<kQB> s;
  const int first = u.r0 + w * 16 * kQB;
  load_queries<kQB, false>(s, a, u, first);
  set_limits<kQB, false>(s, a, u, first);
  Block blk = convert(r0, 0);
  load(r0, 2);
  meet();
  const auto step = [&](int i, Part& r) {
    const f16x8(&at)[16][64] = lds[i & 1];
    f16x8 k[4][2];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) k[j][h] = at[2 * j + h][lane];
    // Past the last tile: zeros that nobody reads.
    const Block next = convert(r, i + 1);
    load(r, i + 3);
    f32x4 sc[kQB][4];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int b = 0; b < kQB; ++b)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          sc[b][j] = mfma16x16x32(k[j][h], s.q[b][h], h == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : sc[b][j]);
    attend_tile<kQB>(s, sc, blk, u.k0 + i * kTile, [&](int t, int e) { return at[8 + 2 * t + e][lane]; });
    blk = next;
    meet();
  };
  for (int i = 0; i < n; i += 2) {
    step(i, r1);
    if (i + 1 < n) step(i + 1, r0);
  }
#pragma unroll
  for (int b = 0; b < kQB; ++b) {
    const int rr = first + 16 * b + col;
    if (rr >= u.rows) continue;
    const int token = u.tok0 + rr / a.G, h = rr % a.G;
    const float l = s.l[b][0];
    const int64_t p = part_index(a, u, token, h);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      if (a.splits == 1) store_out(a, token, u.hk, h, 16 * t + 4 * g, s.o[b][t], l, true);
      else *reinterpret_cast<f32x4*>(a.acc + p * kD + 16 * t + 4 * g) = s.o[b][t];
    }
    if (a.splits > 1 && g == 0) {
      a.m[p] = s.m[b];
      a.l[p] = l;
    }
  }
}

// Joins the at most kSubs * kEach partials of each (token, kv head, query head).  kSubs
// groups of 16 lanes, a lane for 4 dims, share a query.
template <int kSubs, int kEach, bool kDecode>
__global__ __launch_bounds__(256) void merge_kernel(AttnArgs a) {
  constexpr int kLanes = 16 * kSubs;
  const int tid = threadIdx.x, lane = tid & 63;
  const int64_t id = (int64_t)blockIdx.x * (256 / kLanes) + tid / kLanes;
  const bool in = id < (int64_t)a.tokens * a.p.kvh * a.G;
  const int64_t id0 = in ? id : 0;
  const int g = (int)(id0 % a.G);
  const int64_t th = id0 / a.G;
  const int hk = (int)(th % a.p.kvh), token = (int)(th / a.p.kvh);
  int end, lim;
  bool mine = in;
  if (kDecode) {
    end = lim = clampi(a.last[token * a.last_sb], -1, a.cap - 1) + 1;
  } else {
    // The token's row: the last one that starts at or before it.
    int lo = 0, hi = a.B;
    while (lo + 1 < hi) {
      const int mid = (lo + hi) / 2;
      if (a.cu[mid] <= token) lo = mid;
      else hi = mid;
    }
    const int t0 = clampi(a.cu[lo], 0, a.tokens);
    const int new_tokens = min(clampi(a.cu[lo + 1], t0, a.tokens) - t0, a.longest);
    mine = mine && token >= t0 && token < t0 + new_tokens;
    const int ctx = clampi(a.last[lo * a.last_sb], -1, a.cap);
    end = ctx < 0 ? 0 : min(ctx + new_tokens, a.cap);
    lim = ctx < 0 ? 0 : min(ctx + token - t0 + 1, a.cap);
  }
  int n = 0;   // splits that hold a slot below lim
  if (lim > 0) {
    const int len = ((end + kTile - 1) / kTile + a.splits - 1) / a.splits * kTile;
    n = (lim + len - 1) / len;
  }
  const int64_t p0 = th * a.splits * a.G + g;
  // All of a lane's partials at once.  Those past n hold anything, but are there.
  const int sub = (tid >> 4) & (kSubs - 1), d0 = 4 * (lane & 15);
  float mv[kEach], lv[kEach], top = kNegInf;
  f32x4 x[kEach];
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int64_t p = p0 + (int64_t)min(sub + kSubs * e, a.splits - 1) * a.G;
    mv[e] = a.m[p];
    lv[e] = a.l[p];
    x[e] = *reinterpret_cast<const f32x4*>(a.acc + p * kD + d0);
  }
#pragma unroll
  for (int e = 0; e < kEach; ++e)
    if (sub + kSubs * e < n) top = fmaxf(top, mv[e]);
  if constexpr (kSubs > 1) top = col_max(top);
  float sum = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    if (sub + kSubs * e >= n) continue;
    const float c = mv[e] == top ? 1.f : fast_exp2(mv[e] - top);
    sum += lv[e] * c;
    o += x[e] * c;
  }
  if constexpr (kSubs > 1) {
    sum = col_sum(sum);
#pragma unroll
    for (int c = 0; c < 4; ++c) o[c] = col_sum(o[c]);
  }
  if (mine && (kSubs == 1 || lane < 16)) store_out(a, token, hk, g, d0, o, sum, lim > 0);
}

// ---------------------------------------------------------------------------
// host side

constexpr int kCus = 256;

int64_t part_bytes(int64_t queries, int n) { return n <= 1 ? 0 : queries * n * (kD + 2) * 4; }

struct Plan {
  int waves, splits, cols, n_tiles;   // cols: blocks of 16 query rows of a unit
  bool wide, appends;                // appends: the attention writes the new tokens
};

// Rows of at most 1024 slots whole, by one launch; longer ones in ranges of at least a
// tile a wave, as many as let two workgroups a CU run at once, at least two from 4096
// slots on.  MI355X, 2 kv heads of 7 queries, us in a replayed graph, in one piece /
// in the best number of pieces: one row of 512 slots 5.5 / 7.3, 1024 7.6 / 7.5, 2048
// 10.2 / 7.6, 16384 51.8 / 9.8; 16 rows of 1024 8.8 / 8.5; 64 of 512 7.0 / 8.7, of 32768
// 169 / 87.  Two pieces a row where there are more pairs of a row and a kv head than
// CUs: 160 rows of 8192 slots 72 / 65, 128 rows of 200 to 8192 36 / 31, but 200 rows of
// 8192 79 / 84.  Eight waves to a row in one piece take one of 512 slots in 5.5 where
// four take 6.1, but 200 rows of 1024 in 17.6 where those take 15.7.
Plan decode_plan(int B, int KVH, int cap) {
  const int64_t pairs = (int64_t)B * KVH, tiles = ((int64_t)cap + kTile - 1) / kTile;
  if (tiles <= 16) return {pairs <= kCus / 2 ? 8 : 4, 1, 1, 1, false, false};
  const int64_t fill = std::max<int64_t>(2 * kCus / pairs, tiles >= 64 ? 2 : 1);
  return {4, (int)std::min<int64_t>({(tiles + 3) / 4, fill, kMaxSplits}), 1, 1, false, false};
}

// A workgroup has 128 query rows and its waves share the tiles (wide), or 16 cols query
// rows and its waves take the tiles in turn.  MI355X, 7 queries to each of 2 kv heads, us
// in a replayed graph, int8:
// - where one unit of up to 32 query rows has all of a short row's queries, it appends the
//   row's tokens too: 4 rows of 3 tokens behind 1000 slots 12.0, by a launch of its own
//   13.0 (calls from Python 12.4 and 15.3); 32 of 2 behind 2000 15.3 and 17.8.  48 query
//   rows take a wave longer than the launch unless the units fill the CUs: 4 of 5 behind
//   2000 18.8 and 15.9, 64 of 5 behind 1000 16.2 and 18.6;
// - wide where its units give most CUs two workgroups or more, if need be cut along
//   slots as long as each piece keeps 90 tiles: 4 rows of 2048 tokens 73, 89 with two
//   column blocks and 82 with three; 32 of 100 behind 500 slots 30, 36 and 34; 2048
//   tokens behind 16384 slots in three pieces 199, 232 and 236; but 2 rows of 1024
//   behind 8000 in one piece 170, 133 and 129, 16 of 9 to 301 behind 2048 65, 57, 55;
// - three column blocks, for which a wave turns codes into halves once, where there are
//   units enough and most slots are old ones: 8 rows of 512 behind 4000 slots 110, with
//   two 120; but 2048 tokens from slot 0 on 40 and 35, one row of 300 behind 2000 25, 21;
// - one for a single token's heads and for short rows of up to 64 (4 rows of 5 tokens
//   behind 1000 slots 12.9, with two 14.3; behind 8000 in 16 pieces 17.5 and 17.1).
// Rows of at most 2048 slots whole.  Longer ones in as many pieces as let two workgroups a
// CU run at once; of 32 tiles at least where there are 64 units, whose partials are many.
// Eight waves where a piece is all of a row and units are few (one row of 300 behind
// 2000 slots 18.4, with four waves 21.1; 4 rows 43 and 38).
Plan extend_plan(int B, int KVH, int G, int total, int max_seqlen, int cap) {
  const int64_t rows = (int64_t)max_seqlen * G, tiles = ((int64_t)cap + kTile - 1) / kTile;
  const auto units = [&](int64_t tr) {   // of tr query rows, at most
    return KVH * std::min<int64_t>(B * ((rows + tr - 1) / tr), (int64_t)total * G / tr + B);
  };
  const auto plan = [&](int cols, int64_t splits, bool wide) {
    return Plan{4, (int)std::max<int64_t>(1, std::min<int64_t>(splits, kMaxSplits)), cols,
                (int)((rows + 16 * cols - 1) / (16 * cols)), wide, false};
  };
  const int64_t wide_units = units(128), pieces = std::min<int64_t>(3 * kCus / wide_units, tiles / 90);
  if (rows > 64 && wide_units * std::max<int64_t>(pieces, 1) >= 3 * kCus / 2) return plan(8, pieces, true);
  const int cols = rows <= 16 || (rows <= 64 && tiles <= 64) ? 1
                   : units(48) >= kCus && cap >= 4 * (int64_t)max_seqlen ? 3 : 2;
  if (tiles <= 32 && (rows <= 32 || (rows <= 48 && (int64_t)B * KVH >= kCus / 2))) {
    Plan p = plan((int)((rows + 15) / 16), 1, false);
    p.appends = true;
    p.waves = 8;
    return p;
  }
  const int64_t n = units(16 * cols);
  Plan p = plan(cols, tiles <= 32 ? 1 : std::min<int64_t>(tiles / (n >= 64 ? 32 : 4), 2 * kCus / n), false);
  if (p.splits == 1 && n <= kCus) p.waves = 8;
  return p;
}

size_t lds_bytes(int waves) { return waves * (256 * sizeof(f32x4) + 16 * sizeof(float2)); }

template <bool kDecode>
int launch_merge(const AttnArgs& a, hipStream_t st) {
  const int64_t queries = (int64_t)a.tokens * a.p.kvh * a.G;
  const dim3 all((unsigned)((queries + 15) / 16)), quarter((unsigned)((queries + 3) / 4)), b(256);
  if (a.splits <= 4) hipLaunchKernelGGL((merge_kernel<1, 4, kDecode>), all, b, 0, st, a);
  else if (a.splits <= 16) hipLaunchKernelGGL((merge_kernel<4, 4, kDecode>), quarter, b, 0, st, a);
  else hipLaunchKernelGGL((merge_kernel<4, 16, kDecode>), quarter, b, 0, st, a);
  return (int)hipGetLastError();
}

int launch_decode(const AttnArgs& a, int code, int waves, hipStream_t st) {
  const int64_t grid = (int64_t)a.B * a.p.kvh * a.splits;
  if (grid > 0x7fffffff) return QF_ERR_UNSUPPORTED;
  const dim3 g((unsigned)grid), b(64 * waves);
  if (code == QF_CODE_E4M3) hipLaunchKernelGGL(decode_kernel<true>, g, b, lds_bytes(waves), st, a);
  else hipLaunchKernelGGL(decode_kernel<false>, g, b, lds_bytes(waves), st, a);
  return (int)hipGetLastError();
}

template <bool kE4m3>
int launch_extend(const AttnArgs& a, const Plan& p, hipStream_t st) {
  const int64_t grid = (((int64_t)a.B * a.p.kvh * a.splits + 7) & ~(int64_t)7) * a.n_tiles;
  if (grid > 0x7fffffff) return QF_ERR_UNSUPPORTED;
  const dim3 g((unsigned)grid), b(64 * p.waves);
  if (p.wide) hipLaunchKernelGGL(extend_wide_kernel<kE4m3>, g, b, 0, st, a);
  else if (p.cols == 1) hipLaunchKernelGGL((extend_kernel<kE4m3, 1>), g, b, lds_bytes(p.waves), st, a);
  else if (p.cols == 3) hipLaunchKernelGGL((extend_kernel<kE4m3, 3>), g, b, lds_bytes(p.waves), st, a);
  else hipLaunchKernelGGL((extend_kernel<kE4m3, 2>), g, b, lds_bytes(p.waves), st, a);
  return (int)hipGetLastError();
}

// Checks and fills what the entry points share.
int fill_args(AttnArgs& a, const void* q, const QfPool8& pool, const int64_t* last, int64_t last_sb,
              int64_t B, int64_t tokens, int64_t G, int64_t D, double scale) {
  if (D != kD || G < 1 || G > 16) return QF_ERR_UNSUPPORTED;
  a = AttnArgs{};
  const int rc = make_pool(pool, a.p);
  if (rc != QF_OK) return rc;
  if (!q || !last || B < 1 || tokens < 1 || pool.layers != 1 || !(scale > 0.) || !(scale < 1e30) ||
      (reinterpret_cast<uintptr_t>(q) & 15u) != 0)
    return QF_ERR_INVALID_ARG;
  a.cap = row_cap(a.p);
  if (B > 0x3fffffff || tokens > 0x3fffffff / G || tokens * G > 0x7fffffff / a.p.kvh ||
      a.cap + tokens > 0x7fffffff - kTile)
    return QF_ERR_UNSUPPORTED;
  a.q = static_cast<const f16*>(q);
  a.last = last;
  a.last_sb = last_sb;
  a.B = (int)B; a.tokens = (int)tokens; a.G = (int)G;
  a.scale_log2 = (float)scale * kLog2e;
  a.m_unit = 1.f;
  return QF_OK;
}

bool bad_out(const void* out, int64_t st, int64_t sh, int64_t sg) {
  return !out || (reinterpret_cast<uintptr_t>(out) & 7u) != 0 || ((st | sh | sg) & 3) != 0;
}

int set_parts(AttnArgs& a, void* ws, int64_t ws_bytes) {
  if (a.splits <= 1) return QF_OK;
  const int64_t queries = (int64_t)a.tokens * a.p.kvh * a.G;
  if (!ws || (reinterpret_cast<uintptr_t>(ws) & 15u) != 0) return QF_ERR_INVALID_ARG;
  if (ws_bytes < part_bytes(queries, a.splits)) return QF_ERR_SCRATCH_LIMIT;
  a.acc = static_cast<float*>(ws);
  a.m = a.acc + queries * a.splits * kD;
  a.l = a.m + queries * a.splits;
  return QF_OK;
}

int decode_args(AttnArgs& a, const QfDecode8* h) {
  if (!h) return QF_ERR_INVALID_ARG;
  const int rc = fill_args(a, h->q, h->pool, h->kv_last, h->kv_last_sb, h->B, h->B, h->G, h->D, h->scale);
  if (rc != QF_OK) return rc;
  if (((h->q_sb | h->q_sh | h->q_sg) & 7) != 0) return QF_ERR_INVALID_ARG;
  a.q_st = h->q_sb; a.q_sh = h->q_sh; a.q_sg = h->q_sg;
  if ((h->k_new == nullptr) != (h->v_new == nullptr) ||
      ((reinterpret_cast<uintptr_t>(h->k_new) | reinterpret_cast<uintptr_t>(h->v_new)) & 15u) != 0 ||
      (h->k_new != nullptr && ((h->kn_sb | h->kn_sh | h->vn_sb | h->vn_sh) & 7) != 0))
    return QF_ERR_INVALID_ARG;
  a.kn = static_cast<const f16*>(h->k_new);
  a.kn_st = h->kn_sb; a.kn_sh = h->kn_sh;
  a.vn = static_cast<const f16*>(h->v_new);
  a.vn_st = h->vn_sb; a.vn_sh = h->vn_sh;
  return QF_OK;
}

}  // namespace kv8
}  // namespace qf

extern "C" int64_t qf_decode_attn_paged8_workspace(int B, int KVH, int G, int cap) {
  using namespace qf::kv8;
  if (B < 1 || KVH < 1 || cap < 1) return QF_ERR_INVALID_ARG;
  if (G < 1 || G > 16 || (int64_t)B * KVH * G > 0x7fffffff) return QF_ERR_UNSUPPORTED;
  return part_bytes((int64_t)B * KVH * G, decode_plan(B, KVH, cap).splits);
}

extern "C" int qf_decode_attn_paged8(const QfDecode8* h, void* stream) {
  using namespace qf;
  using namespace qf::kv8;
  AttnArgs a;
  int rc = decode_args(a, h);
  if (rc != QF_OK) return rc;
  if (bad_out(h->out, h->o_sb, h->o_sh, h->o_sg)) return QF_ERR_INVALID_ARG;
  a.out = static_cast<f16*>(h->out);
  a.o_st = h->o_sb; a.o_sh = h->o_sh; a.o_sg = h->o_sg;
  const Plan p = decode_plan(a.B, a.p.kvh, a.cap);
  a.splits = p.splits;
  rc = set_parts(a, h->ws, h->ws_bytes);
  if (rc != QF_OK) return rc;
  hipStream_t st = static_cast<hipStream_t>(stream);
  rc = launch_decode(a, (int)h->pool.code, p.waves, st);
  return rc == 0 && a.splits > 1 ? launch_merge<true>(a, st) : rc;
}

extern "C" int qf_decode_split_paged8(const QfDecode8* h, float* acc, float* m, float* l, int splits,
                                      void* stream) {
  using namespace qf;
  using namespace qf::kv8;
  AttnArgs a;
  const int rc = decode_args(a, h);
  if (rc != QF_OK) return rc;
  if (!acc || (reinterpret_cast<uintptr_t>(acc) & 15u) != 0 || !m || !l || splits < 1 || splits > 1024)
    return QF_ERR_INVALID_ARG;
  a.acc = acc;
  a.m = m;
  a.l = l;
  a.m_unit = kLn2;
  a.fill = 1;
  a.splits = splits;
  return launch_decode(a, (int)h->pool.code, 4, static_cast<hipStream_t>(stream));
}

extern "C" int64_t qf_prefill_extend_paged8_workspace(int B, int QH, int KVH, int total, int max_seqlen,
                                                      int cap) {
  using namespace qf::kv8;
  if (B < 1 || KVH < 1 || QH < KVH || QH % KVH != 0 || total < 1 || max_seqlen < 1 || cap < 1)
    return QF_ERR_INVALID_ARG;
  if (QH / KVH > 16 || (int64_t)total * QH > 0x7fffffff || B > 0x3fffffff) return QF_ERR_UNSUPPORTED;
  return part_bytes((int64_t)total * QH, extend_plan(B, KVH, QH / KVH, total, max_seqlen, cap).splits);
}

extern "C" int qf_prefill_extend_paged8(const QfExtend8* h, void* stream) {
  using namespace qf;
  using namespace qf::kv8;
  if (!h) return QF_ERR_INVALID_ARG;
  const QfRows8& r = h->rows;
  if (r.pool.KVH < 1 || h->QH < r.pool.KVH || h->QH % r.pool.KVH != 0) return QF_ERR_INVALID_ARG;
  const int64_t G = h->QH / r.pool.KVH;
  AttnArgs a;
  int rc = fill_args(a, h->q, r.pool, r.first, r.first_sb, r.B, r.total, G, r.D, h->scale);
  if (rc != QF_OK) return rc;
  if (!r.cu_seqlens || r.max_seqlen < 1 || r.max_seqlen > r.total || h->cap < 1 || h->cap > a.cap ||
      ((h->q_sh | h->q_sn) & 7) != 0 || bad_out(h->out, h->o_sn, h->o_sh, 0))
    return QF_ERR_INVALID_ARG;
  a.cap = (int)h->cap;
  a.q_st = h->q_sn; a.q_sh = G * h->q_sh; a.q_sg = h->q_sh;
  a.out = static_cast<f16*>(h->out);
  a.o_st = h->o_sn; a.o_sh = G * h->o_sh; a.o_sg = h->o_sh;
  a.cu = r.cu_seqlens;
  a.cos = static_cast<const f16*>(r.cos);
  a.sin = static_cast<const f16*>(r.sin);
  a.cs_sn = r.cs_sn;
  const Plan p = extend_plan(a.B, a.p.kvh, a.G, a.tokens, (int)r.max_seqlen, a.cap);
  a.splits = p.splits;
  a.n_tiles = p.n_tiles;
  a.longest = (int)r.max_seqlen;
  rc = set_parts(a, h->ws, h->ws_bytes);
  if (rc != QF_OK) return rc;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (p.appends) {
    rc = check_rows(r);
    a.kn = static_cast<const f16*>(r.k);
    a.kn_st = r.k_sn; a.kn_sh = r.k_sh;
    a.vn = static_cast<const f16*>(r.v);
    a.vn_st = r.v_sn; a.vn_sh = r.v_sh;
  } else {
    rc = append(r, a.cap, st);
  }
  if (rc != QF_OK) return rc;
  rc = r.pool.code == QF_CODE_E4M3 ? launch_extend<true>(a, p, st) : launch_extend<false>(a, p, st);
  return rc == 0 && a.splits > 1 ? launch_merge<false>(a, st) : rc;
}
