// Attention over paged caches held in 8 bits (gfx950; the format is qf_paged8.h's):
// single tokens of a batch, and new tokens behind cached ones.
//
// softmax(q K^T) V over slots [0, lim) of a row's pages, lim differing by query, is
// cut into units: query rows (token, query head of one kv head) times a range of slots.
// With few query rows, 16 kNC of them, the waves of a unit's workgroup take tiles of 64
// slots in turn and join their states in LDS (decode_kernel, extend_kernel); with many,
// 128, each wave has 32 of its own and the tiles are shared (extend_wide_kernel).
// What several ranges of a query leave is joined by merge_kernel.
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
// have anyway; V's into the conversion of its codes to fp16, which is exact (taken into
// P instead it would round small P below fp16's normal range).
//
// New tokens are appended by the attention itself where one workgroup has all that a
// row and kv head attend with: in decoding the unit that sees the token's slot, in short
// extensions the row's only one.  A launch less is 1 to 3 us less.
#include <algorithm>

#include "kv8_block.h"
#include "kv8_pieces.h"
#include "lds_tile.h"

namespace qf {
namespace kv8 {

constexpr int kTile = 64;                    // slots
constexpr int kMaxSplits = 64;
// Least factor of the scores: no scores of finite halves are told apart by it, and times a
// block's scale (2^-24 or more) it is not zero, by which masked ones would become NaN.
constexpr float kLeastFactor = 0x1p-100f;

// Weights are held in fp16 for the matrix cores, as 2^(score - reference).  A reference is
// set kHeadroom below the score that moves it and moved when scores come to be more than
// kSlack above that again, so the largest weight of a state is 2^7 to 2^13, and the absolute
// steps of others, 2^-24 below fp16's normal range, are 2^-31 of it or less.  (With the
// largest at 1 slots 18 nats below it round to nothing: of 5400 slots beside one such, all
// that they weigh together, 1e-4, was lost.)  The 3 bits up to fp16's largest are for the
// rounding of the scores, which is 2 at 2^25.  A slack of 4 moves references often enough to
// take 2% longer where rows are many and short, one of 8 half a percent less.
constexpr float kHeadroom = 7.f, kSlack = 6.f;

typedef float f32x8 __attribute__((ext_vector_type(8)));

// A unit of 128 query rows that pieces have to be joined for: `more` partials behind the
// first; 0: none.
struct Join {
  int more, tok0, rows, r0, hk, pad[3];
};

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
  int share;                                 // query tiles that read the same slots share an XCD
  int pieces, shift;                         // even pieces: how many, and the costs' quantum
  Join* joins;                               // even pieces: one for each
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

// Slots [k0, k1) of split s of n of [0, end): n ranges of whole tiles, the last ones shorter
// or empty.
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
  float m[kNC];         // references, log2 units
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
// V^T.
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
      const int left = s.lim[b] - key0 - 16 * g;   // of the lane's 16 slots, what the column sees
      if (left <= 0) f[b] = 1.f;   // whatever scale an unseen block has
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (i >= left) sc[b][i / 4][i % 4] = kNegInf;
    }
    mx[b] = max16(sc[b]) * f[b];
    grew = grew || mx[b] > s.m[b] + (kHeadroom + kSlack);
  }
  // Moves the references of the columns whose own scores grew past them.
  if (__any(grew)) {
#pragma unroll
    for (int b = 0; b < kNC; ++b) {
      const float top = col_max(mx[b]);
      const float m_new = top > s.m[b] + (kHeadroom + kSlack) ? top - kHeadroom : s.m[b];
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
    // p is rounded to fp16 for the matrix cores (off by 2^-11 of it, as the output is by its own
    // rounding, or by 2^-25: see kHeadroom), and the sum adds the rounded ones: the weights
    // add to one.
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

// The unit's row's new tokens into its slots [first, end), one wave for a block's keys and one
// for its values.  The waves of a workgroup share a first-level cache: past the barrier they
// see what was written.
template <bool kE4m3, bool kDecode>
__device__ __forceinline__ void append_tokens(const AttnArgs& a, const Unit& u, const Source& src, int first,
                                              int end) {
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = blockDim.x >> 6;
  for (int s0 = (first / kBlock + w / 2) * kBlock; s0 < end; s0 += nw / 2 * kBlock) {
    const int from = max(s0, first), to = min(end - s0, kBlock);
    const int64_t token = u.tok0 + from - first;
    const bool turn = !kDecode && a.cos != nullptr;
    const Tokens t = {a.kn + token * a.kn_st + u.hk * a.kn_sh, a.kn_st, a.vn + token * a.vn_st + u.hk * a.vn_sh,
                      a.vn_st, turn ? a.cos + token * a.cs_sn : nullptr, turn ? a.sin + token * a.cs_sn : nullptr,
                      a.cs_sn};
    const int page = src.row[s0 >> a.p.log2p];
    if (w & 1) append_block<kE4m3, false, true>(a.p, 0, u.hk, page, s0, from - s0, to, t);
    else append_block<kE4m3, true, false>(a.p, 0, u.hk, page, s0, from - s0, to, t);
  }
  s_waitcnt_vm(0);
  __threadfence_block();
  __syncthreads();
}

// One unit a workgroup: a row's queries of a kv head over a range of its slots.  Long rows
// are bound by memory (64 rows of some 31400 slots, 516 MB, in 87 us: 5.9 TB/s), short ones
// by three loads that wait for each other and some 1 us a tile (one row of 1024 slots, 16
// tiles on 8 waves, 7.0 us).
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
  // Workgroups go to the XCDs in turn: neighbouring tiles to all of them, or with `share` the
  // tiles that read the same slots to one, and its L2.
  const int groups = a.B * a.p.kvh * a.splits;
  int id = blockIdx.x;
  if (a.share) id = (id / (8 * a.n_tiles) * 8 + id % 8) * a.n_tiles + id / 8 % a.n_tiles;
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

// Few query rows: the waves take the tiles in turn.  Bound by the vector unit and by
// latency: 16 rows of 9 to 301 tokens behind 2048 slots, in e4m3, issue it 37% of the time
// with 1.1 waves a SIMD on average (50 us; their products alone 16), as rows end unevenly.
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

// ---- many query rows: even pieces of units of 128 (kv8_pieces.h)

// What all lanes have alike, in scalar registers, where the loop over a piece's units is to
// keep its state.
__device__ __forceinline__ int same(int x) { return __builtin_amdgcn_readfirstlane(x); }

__device__ __forceinline__ RowUnits load_units(const AttnArgs& a, int r) {
  return row_units(a.cu[r], a.cu[r + 1], a.last[r * a.last_sb], a.G, a.tokens, a.longest, a.cap, a.shift);
}

__device__ __forceinline__ RowUnits of_lane(const RowUnits& w, int lane) {
  const auto get = [&](int x) { return __builtin_amdgcn_readlane(x, lane); };
  return {get(w.tok0), get(w.rows), get(w.ctx), get(w.n), get(w.first), get(w.step)};
}

// A unit and its part of the line.
struct Place {
  RowUnits w;
  int r, hk, q, seen, x0, x1;
};

__device__ __forceinline__ void set_place(const AttnArgs& a, Place& u, int x0) {
  u.x0 = x0;
  u.x1 = x0 + u.w.first + u.w.step * u.q;
  u.seen = same(slots_seen(u.w, u.q, a.G, a.cap));
}

// Finds the piece's part [x, end) of the line and the unit that has x; false: none.
__device__ __forceinline__ bool find_piece(const AttnArgs& a, int& piece, int& x, int& end, int& len, Place& u) {
  const int lane = threadIdx.x & 63;
  // 64 rows at a time; with no more of them all is there after one pass.
  RowUnits w;
  int mine, upto;
  const auto rows_from = [&](int i0) {
    w = load_units(a, min(i0 + lane, a.B - 1));
    mine = i0 + lane < a.B ? cost_before(w, w.n) * a.p.kvh : 0;
    upto = scan_sum(mine);
    return __builtin_amdgcn_readlane(upto, 63);
  };
  int work = rows_from(0);
  for (int i0 = 64; i0 < a.B; i0 += 64) work = add_capped(work, rows_from(i0));
  work = line_length(work);
  len = same(piece_length(work, a.pieces, a.G, a.shift));
  piece = same(piece_of((int)blockIdx.x, a.pieces, work, len));
  x = piece * len;
  end = min(x + len, work);
  if (x >= work) return false;
  int before = 0, i0 = 0;
  if (a.B > 64) rows_from(0);
  for (;;) {
    const uint64_t hit = __ballot(x < add_capped(before, upto));
    if (hit != 0) {
      const int j = __builtin_ctzll(hit);
      int base = before + __builtin_amdgcn_readlane(upto - mine, j);
      u.r = i0 + j;
      u.w = of_lane(w, j);
      const int row = cost_before(u.w, u.w.n);
      u.hk = same((int)min((unsigned)(x - base) / (unsigned)row, (unsigned)a.p.kvh - 1u));
      base += u.hk * row;
      u.q = unit_at(u.w, x - base);
      set_place(a, u, base + cost_before(u.w, u.q));
      return true;
    }
    before = add_capped(before, __builtin_amdgcn_readlane(upto, 63));
    i0 += 64;
    if (i0 >= a.B) return false;
    rows_from(i0);
  }
}

// The unit behind u; false: none.
__device__ __forceinline__ bool next_place(const AttnArgs& a, Place& u) {
  if (++u.q >= u.w.n) {
    u.q = 0;
    if (++u.hk >= a.p.kvh) {
      u.hk = 0;
      do {
        if (++u.r >= a.B) return false;
        u.w = of_lane(load_units(a, u.r), 0);
      } while (u.w.n == 0);
    }
  }
  set_place(a, u, u.x1);
  return true;
}

// Tiles that a workgroup has done, of about how many, and when its priority changes next.
struct Progress {
  int done, tiles, quarter, level;
};

// The waves take 32 query rows of a unit each and share its tiles.  A wave turns a
// quarter of each tile's codes into operands, in LDS, a tile ahead of their use: a
// quarter of the conversions that a wave by itself has for as many queries.  lds:
// [stage][operand: K (i, h), then V (t, u)][lane].  The result goes to the output, or to
// partial `part` if that is one.
//
// What bounds it: a wave-step (32 query rows x 64 slots) is 36 matrix instructions of 16
// cycles and some 180 vector ones, 32 of them exponentials; with three waves a SIMD the
// vector unit issues 55% of the time, the matrix cores run 32% of it, and the clock is
// lowered (2.0 GHz with int8 codes, 2.4 without load).  In even pieces the 168 registers of
// three waves a SIMD are too few for the walk from unit to unit: 26 are spilled in int8, 21
// in e4m3.  A reload behind each tile's exponentials waits for all loads that are out, and
// in int8 every second tile waits for the K codes that it has just asked for, to spill them.
// 2048 tokens behind 16384 slots: 620 to 660 TF/s in int8, 730 in e4m3.
template <bool kE4m3, bool kEven>
__device__ __forceinline__ void wide_unit(const AttnArgs& a, const Unit& u, int part, Progress& pr,
                                          f16x8 (&lds)[2][16][64]) {
  constexpr int kQB = 2;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int lane = threadIdx.x & 63;
  if (kEven) asm volatile("" : "+v"(lane));   // what hangs on it is not kept from one unit to the next
  const int col = lane & 15, g = lane >> 4;
  Source src = make_source(a, u);
  src.koff += w * 4 * kD;
  src.voff += w * 16 * kTile;
  const int n = (u.k1 - u.k0 + kTile - 1) / kTile;
  struct Part {
    u32x4 k, v;
    float ks, vs;
  };
  // Tiles are loaded in order; a tile's page is fetched, into a scalar register, while the
  // one before it is loaded.
  typedef const __attribute__((address_space(4))) int32_t* Table;
  const auto fetch = [&](int i) {
    const int lp = min((u.k0 + i * kTile) >> src.log2p, src.ppr - 1);
    return ((Table)src.row)[lp];
  };
  int pid = fetch(0);
  const auto load = [&](Part& r, int i) {
    const bool valid = i < n;
    const int slot0 = u.k0 + i * kTile;
    const int64_t page = min(max(pid, 0), src.n_pages - 1);
    pid = fetch(min(i + 1, n - 1));
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
    if (kEven && pr.done + i >= pr.quarter) {
      // Of the three waves of a SIMD the eldest goes first, so the workgroups of a CU would end
      // one after the other (115 to 195 us where the mean is 155), the last with the CU for
      // itself: the further a piece is, the lower its priority (121 to 179; 2048 tokens
      // behind 16384 slots 216 -> 205 us).
      if (pr.level == 0) __builtin_amdgcn_s_setprio(2);
      else if (pr.level == 1) __builtin_amdgcn_s_setprio(1);
      else __builtin_amdgcn_s_setprio(0);
      ++pr.level;
      pr.quarter += pr.tiles / 4 + 1;
    }
    step(i, r1);
    if (i + 1 < n) step(i + 1, r0);
  }
  if (kEven) pr.done += n;
#pragma unroll
  for (int b = 0; b < kQB; ++b) {
    const int rr = first + 16 * b + col;
    if (rr >= u.rows) continue;
    const float l = s.l[b][0];
    if (part < 0) {
      const int token = u.tok0 + rr / a.G, h = rr % a.G;
#pragma unroll
      for (int t = 0; t < 4; ++t) store_out(a, token, u.hk, h, 16 * t + 4 * g, s.o[b][t], l, true);
    } else {
      const int64_t p = (int64_t)part * kUnitRows + rr - u.r0;
#pragma unroll
      for (int t = 0; t < 4; ++t) *reinterpret_cast<f32x4*>(a.acc + p * kD + 16 * t + 4 * g) = s.o[b][t];
      if (g == 0) {
        a.m[p] = s.m[b];
        a.l[p] = l;
      }
    }
  }
}

// A unit to a workgroup.
template <bool kE4m3>
__global__ __launch_bounds__(256, 3) void extend_wide_kernel(AttnArgs a) {
  __shared__ f16x8 lds[2][16][64];
  Unit u;
  if (!extend_unit<kUnitRows>(a, u)) return;
  Progress none;
  if (u.k1 > u.k0) wide_unit<kE4m3, false>(a, u, -1, none, lds);
  else empty_unit(a, u, kUnitRows);
}

// The kernel's arguments, loaded again: nothing of them is kept in registers from one unit
// to the next.
__device__ __forceinline__ AttnArgs arguments() {
  typedef const __attribute__((address_space(4))) AttnArgs* Pointer;
  Pointer p = (Pointer)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const AttnArgs*)p;
}

// A piece to a workgroup.  Piece p leaves at most two partials: 2 p of the unit that it takes up
// inside, 2 p + 1 of one that it begins and does not end.  Finding the piece takes 2 us.
template <bool kE4m3>
__global__ __launch_bounds__(256, 3) void extend_even_kernel(AttnArgs a) {
  __shared__ f16x8 lds[2][16][64];
  __shared__ Place held;
  int piece, x, end, len, k0 = 0;
  Place at;
  Join join = {};
  const bool any = find_piece(a, piece, x, end, len, at);
  if (any) {
    const auto cut_at = [&](int y) { return same(cut_slot(y - at.x0, at.seen, a.G, a.shift)); };
    k0 = cut_at(x);
    if (k0 > 0 && k0 < at.seen && (x - len < at.x0 || cut_at(x - len) == 0)) {
      // The unit's first cut.
      join = {1, at.w.tok0, at.w.rows, at.q * kUnitRows, at.hk};
      for (int y = x + len; join.more < a.pieces - piece && y < at.x1 && cut_at(y) < at.seen; y += len) ++join.more;
    }
  }
  if (threadIdx.x == 0) a.joins[piece] = join;
  if (!any) return;
  Progress progress = {0, len / a.G, len / a.G / 4, 0};
  __builtin_amdgcn_s_setprio(3);
  for (;;) {
    const int k1 = end >= at.x1 ? at.seen : same(cut_slot(end - at.x0, at.seen, a.G, a.shift));
    const bool more = at.x1 < end;
    if (threadIdx.x == 0) held = at;
    {
      const AttnArgs b = arguments();
      const Unit u = {at.w.tok0, at.w.rows, at.q * kUnitRows, at.r, at.hk, 0, at.w.ctx, k0, k1};
      const bool whole = k0 == 0 && k1 == at.seen;
      if (k1 > k0) wide_unit<kE4m3, true>(b, u, whole ? -1 : 2 * piece + (k0 == 0), progress, lds);
      else if (at.seen == 0) empty_unit(b, u, kUnitRows);
    }
    if (!more) return;
    __syncthreads();
    at.w = of_lane(held.w, 0);
    at.r = same(held.r);
    at.hk = same(held.hk);
    at.q = same(held.q);
    at.x1 = same(held.x1);
    __syncthreads();
    if (!next_place(arguments(), at)) return;
    k0 = 0;
  }
}

// Joins the partials of the unit that piece blockIdx.x + 1 cuts first; 16 lanes, 4 dims
// each, share a query row.  7 us behind 224 units in 768 pieces (the pieces leave the
// places: finding them here again took 30).
__global__ __launch_bounds__(256) void join_kernel(AttnArgs a) {
  const int piece = blockIdx.x + 1;
  const Join u = a.joins[piece];
  const int more = u.more;
  const int rr = blockIdx.y * 16 + (threadIdx.x >> 4), d0 = 4 * (threadIdx.x & 15), r = u.r0 + rr;
  if (more == 0 || r >= u.rows) return;
  constexpr int kEach = 6;
  float top = kNegInf, sum = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int j0 = 0; j0 <= more; j0 += kEach) {
    float mv[kEach], lv[kEach], t = top;
    f32x4 acc[kEach];
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const int j = min(j0 + e, more);
      const int64_t p = (int64_t)(j == 0 ? 2 * piece - 1 : 2 * (piece + j - 1)) * kUnitRows + rr;
      mv[e] = a.m[p];
      lv[e] = a.l[p];
      acc[e] = *reinterpret_cast<const f32x4*>(a.acc + p * kD + d0);
    }
#pragma unroll
    for (int e = 0; e < kEach; ++e) t = fmaxf(t, mv[e]);
    const float c = top == t ? 1.f : fast_exp2(top - t);
    sum *= c;
    o *= c;
    top = t;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      if (j0 + e > more) continue;
      const float f = mv[e] == top ? 1.f : fast_exp2(mv[e] - top);
      sum += lv[e] * f;
      o += acc[e] * f;
    }
  }
  store_out(a, u.tok0 + r / a.G, u.hk, r % a.G, d0, o, sum, true);
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
    n = (lim - 1) / len + 1;
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

constexpr int kCus = 256, kPieces = 3 * kCus;   // as many as run at once

// Partials of a plan's call.
int64_t part_rows(int64_t queries, int splits, int pieces) {
  return pieces > 0 ? 2 * (int64_t)pieces * kUnitRows : splits <= 1 ? 0 : queries * splits;
}

int64_t part_bytes(int64_t rows, int pieces) { return rows * (kD + 2) * 4 + pieces * (int64_t)sizeof(Join); }

struct Plan {
  int waves, splits, cols, n_tiles;   // cols: blocks of 16 query rows of a unit, 8: wide
  int pieces, shift;                 // of a wide extension in even pieces, else 0
  bool appends;                      // the attention writes the new tokens
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
  if (tiles <= 16) return {pairs <= kCus / 2 ? 8 : 4, 1, 1, 1, 0, 0, false};
  const int64_t fill = std::max<int64_t>(2 * kCus / pairs, tiles >= 64 ? 2 : 1);
  return {4, (int)std::min<int64_t>({(tiles + 3) / 4, fill, kMaxSplits}), 1, 1, 0, 0, false};
}

// A workgroup has 128 query rows and its waves share the tiles (wide, cols 8), or 16 cols
// query rows and its waves take the tiles in turn.  MI355X, 7 queries to each of 2 kv
// heads, us in a replayed graph, int8:
// - where one unit of up to 32 query rows has all of a short row's queries, it appends the
//   row's tokens too: 4 rows of 3 tokens behind 1000 slots 12.0, by a launch of its own
//   13.0 (calls from Python 12.4 and 15.3); 32 of 2 behind 2000 15.3 and 17.8.  48 query
//   rows take a wave longer than the launch unless there are units enough: 4 of 5 behind
//   2000 18.4 and 15.6, 16 behind 1000 14.4 and 14.4, 32 15.0 and 16.0, 64 16.2 and 18.6;
// - wide, in even pieces of all units (kv8_pieces.h), where those have 48 tiles or more, or
//   24 of rows of 120: 2048 tokens behind 16384 slots 205, with each unit in as many equal
//   ranges as fill the CUs once 214; 1750 tokens 169 and 193, 2400 218 and 289, 1024 behind
//   65536 343 and 477; with two column blocks one row of 700 behind 16000 91 and 113, of
//   1024 114 and 150; but of 512 behind 16000 83 and 73, 8 of 512 behind 4000 129 and with
//   three 124, 4 of 400 71 and 53;
// - wide, a workgroup a unit, where there are units for most CUs and a half: 4 rows of 2048
//   tokens 71, in even pieces 89, with two column blocks 89 and with three 82; 32 of 100
//   behind 500 slots 30, 49, 36 and 34; but 2 rows of 1024 behind 8000 170, 133 and 129 with
//   two and three column blocks, 16 of 9 to 301 behind 2048 65, 57, 55;
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
  const auto plan = [&](int cols, int64_t splits) {
    return Plan{4, (int)std::max<int64_t>(1, std::min<int64_t>(splits, kMaxSplits)), cols,
                (int)((rows + 16 * cols - 1) / (16 * cols)), 0, 0, false};
  };
  const int64_t n_units = units(kUnitRows);
  if (rows > 64 && n_units * tiles >= (tiles >= 120 ? 24 : 48) * kPieces) {
    Plan p = plan(8, 1);
    p.pieces = kPieces;
    while (p.shift < 20 && most_cost(n_units, G, cap, max_seqlen, p.shift) >= 1 << 30) ++p.shift;
    if (p.shift < 20) return p;
  }
  if (rows > 64 && n_units >= 3 * kCus / 2) return plan(8, 1);
  const int cols = rows <= 16 || (rows <= 64 && tiles <= 64) ? 1
                   : units(48) >= kCus && cap >= 4 * (int64_t)max_seqlen ? 3 : 2;
  if (tiles <= 32 && (rows <= 32 || (rows <= 48 && (int64_t)B * KVH >= kCus / 4))) {
    Plan p = plan((int)((rows + 15) / 16), 1);
    p.appends = true;
    p.waves = 8;
    return p;
  }
  const int64_t n = units(16 * cols);
  Plan p = plan(cols, tiles <= 32 ? 1 : std::min<int64_t>(tiles / (n >= 64 ? 32 : 4), 2 * kCus / n));
  if (p.splits == 1 && n <= kCus) p.waves = 8;
  return p;
}

// Whether the query tiles of a row, kv head and split go to one XCD: where those are eight or
// more and must be of like size, as rows are one or have about as many new tokens and no
// more old ones.  MI355X, us in a replayed graph: 4 rows of 2048 tokens 72, spread 78; 16
// of 301 behind 2048 slots 80 and 83; but 5 rows of 9 to 301 behind 16000 slots 140 and 98.
bool share_xcd(const AttnArgs& a, int splits, int max_seqlen) {
  return (int64_t)a.B * a.p.kvh * splits >= 8 &&
         (a.B == 1 || ((int64_t)a.tokens * 4 >= (int64_t)a.B * max_seqlen * 3 && a.cap <= 2 * (int64_t)max_seqlen));
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
  if (p.pieces > 0) {
    hipLaunchKernelGGL(extend_even_kernel<kE4m3>, dim3(p.pieces), dim3(256), 0, st, a);
    const int rc = (int)hipGetLastError();
    if (rc != 0) return rc;
    hipLaunchKernelGGL(join_kernel, dim3(p.pieces - 1, kUnitRows / 16), dim3(256), 0, st, a);
    return (int)hipGetLastError();
  }
  const int64_t grid = (((int64_t)a.B * a.p.kvh * a.splits + 7) & ~(int64_t)7) * a.n_tiles;
  if (grid > 0x7fffffff) return QF_ERR_UNSUPPORTED;
  const dim3 g((unsigned)grid), b(64 * p.waves);
  if (p.cols == 8) hipLaunchKernelGGL(extend_wide_kernel<kE4m3>, g, b, 0, st, a);
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
  a.scale_log2 = std::max((float)scale * kLog2e, kLeastFactor);
  a.m_unit = 1.f;
  return QF_OK;
}

bool bad_out(const void* out, int64_t st, int64_t sh, int64_t sg) {
  return !out || (reinterpret_cast<uintptr_t>(out) & 7u) != 0 || ((st | sh | sg) & 3) != 0;
}

int set_parts(AttnArgs& a, const Plan& p, void* ws, int64_t ws_bytes) {
  a.splits = p.splits;
  a.pieces = p.pieces;
  a.shift = p.shift;
  const int64_t rows = part_rows((int64_t)a.tokens * a.p.kvh * a.G, p.splits, p.pieces);
  if (rows == 0) return QF_OK;
  if (!ws || (reinterpret_cast<uintptr_t>(ws) & 15u) != 0) return QF_ERR_INVALID_ARG;
  if (ws_bytes < part_bytes(rows, p.pieces)) return QF_ERR_SCRATCH_LIMIT;
  a.acc = static_cast<float*>(ws);
  a.m = a.acc + rows * kD;
  a.l = a.m + rows;
  a.joins = reinterpret_cast<Join*>(a.l + rows);
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
  return part_bytes(part_rows((int64_t)B * KVH * G, decode_plan(B, KVH, cap).splits, 0), 0);
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
  rc = set_parts(a, p, h->ws, h->ws_bytes);
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
  const Plan p = extend_plan(B, KVH, QH / KVH, total, max_seqlen, cap);
  return part_bytes(part_rows((int64_t)total * QH, p.splits, p.pieces), p.pieces);
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
  a.n_tiles = p.n_tiles;
  a.share = share_xcd(a, p.splits, (int)r.max_seqlen);
  a.longest = (int)r.max_seqlen;
  rc = set_parts(a, p, h->ws, h->ws_bytes);
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
