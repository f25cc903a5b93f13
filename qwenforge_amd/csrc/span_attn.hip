// Attention over spans of paged caches for gfx950: decode of a batch whose rows
// share long prefixes, and new tokens behind cached ones.
//
// Both are softmax(q K^T) V over slots [0, lim) of a row's pages with a lim for
// every query, and both are cut into units: up to kQB * 64 query rows (token,
// query head of one kv head; the heads of a token are neighbours) times a range
// of slots.  A unit leaves (sum p v, max, sum p), and span_merge_kernel joins
// the ranges of each query:
//   softmax over a union = sum_i 2^(m_i - M) acc_i / sum_i 2^(m_i - M) l_i.
// Decode has two kinds of unit.  The shared slots of a group of rows are read
// once per query tile of the whole group, the rows of a tile being the matrix
// cores' columns; the slots behind them belong to one row, whose at most 16
// queries are one column block, and the four waves of the workgroup take the
// key tiles in turn.  New tokens are units of the first kind whose lim grows
// with the token.
//
// Tiles of 64 keys go HBM -> LDS with direct-to-LDS loads and are read as in
// lds_tile.h; scores and output are computed transposed (qf_common.h).  Slots
// past a unit's last one read as zero, and masked slots count for nothing
// whatever K and V hold there (masked_values).
//
// A wave's step of 32 queries and 64 keys is 36 matrix products of 16 cycles and
// some 120 vector instructions, 32 of them exponentials of 16 cycles.  No unit is
// full, and memory is not the bound: counted over 2048 tokens behind 16384 slots
// (96 rows of a 32768-slot prefix), the vector unit issues in 44% (42%) of the SIMDs'
// cycles and the matrix cores are busy in 33% (23%); a wave spends 23% (38%) of its
// time waiting for tiles and barriers and 29% (24%) for its turn to issue, with 1.5
// waves to a SIMD.  MI355X, 14 query heads on 2 kv heads, GPU time of the whole call
// in a replayed graph: that chunk 189 us (680 TF/s; 111 us at the rate of a large
// fp16 product), 16 rows of 9 to 301 tokens behind 2048 slots 56 us (its 286 units
// leave most CUs one workgroup of the two that they hold), four times five tokens
// behind 2000 slots 12.2 us (three launches and their dependent loads).  Decode,
// and in brackets each row alone over the shared pages (flash_decode_attention_paged):
// 96 rows of the 32768-slot prefix 36 us (235), 24 rows in three groups of up to
// 4096 shared slots 12.8 (14.1), four rows of a 512-slot prefix 9.4 (6.3): the two
// launches, of which the merge is 3 us, pay from long prefixes or many rows on.
#include <algorithm>

#include "extend.h"
#include "lds_tile.h"
#include "../../include/qf_prefix.h"

namespace qf {
namespace span {

constexpr int kD = 64;
constexpr int kBN = 64;                      // keys per tile
constexpr int kWaves = 4;
constexpr int kThreads = kWaves * 64;
constexpr int kTileBytes = kBN * kRowBytes;  // of K or V
constexpr int kStages = 4;                   // ring of the wide units
constexpr int kMaxSplits = 64;               // of either kind of unit
constexpr int kMinKeys = 128;                // least keys of a split
constexpr int kStepKeys = kWaves * kBN;      // a step of a narrow unit's waves
constexpr float kHuge = 3.402823466e38f;

struct Args {
  const f16* q;
  int64_t q_st, q_sh, q_sg;                  // token, kv head, query head of the kv head
  const f16* k;
  int64_t k_sp, k_sh, k_sn;
  const f16* v;
  int64_t v_sp, v_sh, v_sn;
  const int32_t* table;
  int64_t t_sb;
  int log2p, n_pages, ppr;
  // Segments: tokens [bounds[i], bounds[i + 1]) share their tiles.  Decode: a
  // group of rows (a token is a row) with plen[i] shared slots, at most pcap, in
  // the pages of ptable's row i, or without it of the group's first row;
  // last[token] is the row's last slot.  Extension: the new tokens of row i
  // behind last[i] cached slots.
  const int32_t* bounds;
  const int32_t* plen;
  const int32_t* ptable;
  int64_t pt_sb;
  int pcap, pppr;
  const int64_t* last;
  int64_t last_sb;
  int n_seg, tokens, KVH, G, cap;
  int n_tiles, splits;                       // query tiles and splits of the grid's first units
  int own_splits;                            // splits of each row's own slots (decode)
  float* acc;                                // (token, kv head, split, query head, 64)
  float2* ml;                                // (token, kv head, split, query head): max, sum
  f16* out;
  int64_t o_st, o_sh, o_sg;
  float scale_log2;
  const f16* cos;                            // per token: Q is rotated on its way in
  const f16* sin;
  int64_t cs_sn;
};

// The kernel's arguments read anew from the argument block.  What only the end
// of a unit needs would otherwise stay in scalar registers through its loop,
// which has none to spare (the compiler then parks them in vector registers).
__device__ __forceinline__ const Args& late_args() {
  auto p = __builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const Args*)p;
}

__device__ __forceinline__ int clampi(int64_t x, int lo, int hi) {
  return (int)(x < lo ? lo : x > hi ? hi : x);
}

__device__ __forceinline__ int scan_max(int x, int n) {
  const int lane = threadIdx.x & 63;
  for (int d = 1; d < n; d <<= 1) {
    const int y = __shfl_up(x, d);
    if (lane >= d) x = max(x, y);
  }
  return x;
}

__device__ __forceinline__ int scan_sum(int x, int n) {
  const int lane = threadIdx.x & 63;
  for (int d = 1; d < n; d <<= 1) {
    const int y = __shfl_up(x, d);
    if (lane >= d) x += y;
  }
  return x;
}

// One segment: its tokens [lo, hi), its index, -1 if there is none, and its plen
// or cached slots (-1: none, parked), clamped.
struct Segment {
  int index, lo, hi, slots;
};

// Walks the segments 64 at a time and takes the first one for which `pick(lo,
// hi, tiles ahead, its tiles)` is true, tiles holding tr query rows; `before`
// becomes the tiles ahead of it.  Any contents of bounds give segments that
// ascend, do not overlap and stay within the tokens.
template <bool kDecode, typename Pick>
__device__ __forceinline__ Segment find_segment(const Args& a, int tr, int& before, Pick&& pick) {
  const int lane = threadIdx.x & 63;
  int top = 0;
  before = 0;
  for (int i0 = 0; i0 < a.n_seg; i0 += 64) {
    const int n = min(a.n_seg - i0, 64);
    const int i = i0 + min(lane, n - 1);
    // Loaded with the bounds: the walk waits for memory once.
    const int slots = kDecode ? clampi(a.plen[i], 0, a.pcap) : clampi(a.last[i * a.last_sb], -1, a.cap);
    const int hi = scan_max(max(top, clampi(a.bounds[i + 1], 0, a.tokens)), n);
    int lo = clampi(a.bounds[i], 0, a.tokens);
    lo = max(max(top, scan_max(lo, n)), 0);
    const int end = max(lo, hi);
    const int tiles = lane < n ? ((end - lo) * a.G + tr - 1) / tr : 0;
    const int upto = scan_sum(tiles, n);
    const uint64_t hit = __ballot(lane < n && pick(lo, end, before + upto - tiles, tiles));
    if (hit != 0) {
      const int j = __builtin_ctzll(hit);
      before += __builtin_amdgcn_readlane(upto - tiles, j);
      return {i0 + j, __builtin_amdgcn_readlane(lo, j), __builtin_amdgcn_readlane(end, j),
              __builtin_amdgcn_readlane(slots, j)};
    }
    before += __builtin_amdgcn_readlane(upto, n - 1);
    top = __builtin_amdgcn_readlane(end, n - 1);
  }
  return {-1, 0, 0, 0};
}

// A range of slots of a row's pages, read tile by tile.  A tile's address takes a
// dozen scalar instructions per wave, so they are 32-bit ones (the host refuses
// strides past them); tiles come in ascending order.
struct Source {
  const unsigned char* k;  // pool + kv head
  const unsigned char* v;
  const int32_t* row;      // block table row
  unsigned k_sp, v_sp;     // page strides, 16 bytes
  int k_sn, v_sn;          // slot strides, bytes
  int pid, pwin;           // lane j: page of logical page pwin + j
  int log2p, ppr, n_pages;
  int end;                 // slots from here on read as zero
};

__device__ __forceinline__ void load_pids(Source& s, int win) {
  const int j = min(win + (int)(threadIdx.x & 63), s.ppr - 1);
  s.pid = min(max(s.row[j], 0), s.n_pages - 1);
  s.pwin = win;
}

// Async loads of kRows rows from row r0 of the tile at slot0 (a multiple of 64,
// below s.end) into the K and V tiles at Kd and Vd.
template <int kRows>
__device__ __forceinline__ void issue(Source& s, int slot0, int r0, unsigned char* Kd,
                                      unsigned char* Vd) {
  const int lane = threadIdx.x & 63;
  const int lp = slot0 >> s.log2p;
  if (lp - s.pwin >= 64) load_pids(s, lp);
  const unsigned page = __builtin_amdgcn_readlane(s.pid, lp - s.pwin);
  const int in_page = slot0 & ((1 << s.log2p) - 1), rows = min(s.end - slot0, kBN);
  const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<unsigned char*>(s.k + ((uint64_t)page * s.k_sp << 4) + in_page * s.k_sn), (short)0,
      rows * s.k_sn, 0x00020000);
  const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<unsigned char*>(s.v + ((uint64_t)page * s.v_sp << 4) + in_page * s.v_sn), (short)0,
      rows * s.v_sn, 0x00020000);
#pragma unroll
  for (int i = 0; i < kRows / 8; ++i) {
    const int r = r0 + 8 * i + (lane >> 3);
    const int c = 16 * ((lane & 7) ^ swz(r));
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, (lds_void*)(Kd + (r0 + 8 * i) * kRowBytes), 16,
                                             r * s.k_sn + c, 0, 0, 0);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, (lds_void*)(Vd + (r0 + 8 * i) * kRowBytes), 16,
                                             r * s.v_sn + c, 0, 0, 0);
  }
}

// The softmax state of kQB blocks of 16 query columns of one wave.
template <int kQB>
struct State {
  f16x8 q[kQB][2];
  int lim[kQB];     // the column sees slots [lo, lim)
  int lo, seen;     // every column of the wave sees [lo, seen)
  float m[kQB];     // running reference, log2 units
  f32x4 l[kQB];     // running sum of p, in every row of the column
  f32x4 o[kQB][4];
  float ks2;
  int koff[2], voff[4];  // operand addresses within a tile
};

template <int kQB>
__device__ __forceinline__ void init_state(State<kQB>& s, int lo, float scale_log2) {
  const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
  s.lo = lo;
  s.ks2 = scale_log2;
  const int rk = 8 * (col >> 2) + (col & 3);
#pragma unroll
  for (int kk = 0; kk < 2; ++kk) s.koff[kk] = rk * kRowBytes + 16 * ((grp + 4 * kk) ^ swz(rk));
  const int rv = 8 * grp + (col >> 2);
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int d = 16 * t + 4 * (col & 3);
    s.voff[t] = rv * kRowBytes + 16 * ((d >> 3) ^ swz(rv)) + 2 * (d & 7);
  }
#pragma unroll
  for (int b = 0; b < kQB; ++b) {
    s.m[b] = kNegInf;
    s.l[b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int t = 0; t < 4; ++t) s.o[b][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
}

// Bits 15 and 31 set for halves of w that are infinities or NaN (an exponent of
// ones carries into the sign's place).
__device__ __forceinline__ unsigned special2(unsigned w) {
  return (w & 0x7FFF7FFFu) + 0x04000400u;
}

// The infinities and NaNs of a masked tile's V: out of the operands, so that a
// masked slot's zero probability meets zeros, and into the output only where
// the column sees the slot.  p of key 32 ch + 8 g + e of the tile is element e
// of pb[ch] in the column's lane of group g.
template <int kQB>
__device__ __forceinline__ void masked_values(u32x2 (&vr)[2][4][2], const State<kQB>& s,
                                              const f16x8 (&pb)[kQB][2], int key0, f32x4 (&o)[kQB][4],
                                              const unsigned char* Vs) {
#pragma unroll
  for (int ch = 0; ch < 2; ++ch)
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const unsigned bad = (special2(vr[ch][t][h][x]) & 0x80008000u) >> 15;
          vr[ch][t][h][x] &= ~(bad * 0xFFFFu);
        }
  const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
#pragma unroll
  for (int ch = 0; ch < 2; ++ch)
#pragma unroll
    for (int e = 0; e < 8; ++e)
      for (int g = 0; g < 4; ++g) {
        const int j = 32 * ch + 8 * g + e;
#pragma unroll
        for (int b = 0; b < kQB; ++b) {
          const float p = __shfl((float)pb[b][ch][e], col + 16 * g);
          if (key0 + j < s.lo || key0 + j >= s.lim[b]) continue;
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int d = 16 * t + 4 * grp + i;
              const f16 v = *reinterpret_cast<const f16*>(Vs + j * kRowBytes +
                                                          16 * ((d >> 3) ^ swz(j)) + 2 * (d & 7));
              const float x = (float)v;
              if (!(__builtin_fabsf(x) < __builtin_huge_valf())) o[b][t][i] += p * x;
            }
        }
      }
}

// The K operands of a tile, waited for.
struct KTile {
  u32x4 r[2][2][2];  // [32 keys][4-key half][32 dims]
};

__device__ __forceinline__ void read_k(KTile& k, const int (&koff)[2], const unsigned char* Ks) {
  const unsigned ks = lds_addr(Ks);
#pragma unroll
  for (int kk = 0; kk < 2; ++kk) {
    const unsigned at = ks + koff[kk];
    k.r[0][0][kk] = lds_read_b128<0>(at);
    k.r[0][1][kk] = lds_read_b128<4 * kRowBytes>(at);
    k.r[1][0][kk] = lds_read_b128<32 * kRowBytes>(at);
    k.r[1][1][kk] = lds_read_b128<36 * kRowBytes>(at);
  }
}

__device__ __forceinline__ void wait_k(KTile& k) {
  asm volatile("s_waitcnt lgkmcnt(0)"
               : "+v"(k.r[0][0][0]), "+v"(k.r[0][0][1]), "+v"(k.r[0][1][0]), "+v"(k.r[0][1][1]),
                 "+v"(k.r[1][0][0]), "+v"(k.r[1][0][1]), "+v"(k.r[1][1][0]), "+v"(k.r[1][1][1]));
}

// The V^T operands of a tile: [32 keys][16 dims][4-key half].
struct VTile {
  u32x2 r[2][4][2];
};

__device__ __forceinline__ void read_v(VTile& v, const int (&voff)[4], const unsigned char* Vs) {
  const unsigned vs = lds_addr(Vs);
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const unsigned at = vs + voff[t];
    v.r[0][t][0] = lds_read_tr_b64<0>(at);
    v.r[0][t][1] = lds_read_tr_b64<4 * kRowBytes>(at);
    v.r[1][t][0] = lds_read_tr_b64<32 * kRowBytes>(at);
    v.r[1][t][1] = lds_read_tr_b64<36 * kRowBytes>(at);
  }
}

__device__ __forceinline__ void wait_v(VTile& v) {
  asm volatile("s_waitcnt lgkmcnt(0)"
               : "+v"(v.r[0][0][0]), "+v"(v.r[0][0][1]), "+v"(v.r[0][1][0]), "+v"(v.r[0][1][1]),
                 "+v"(v.r[0][2][0]), "+v"(v.r[0][2][1]), "+v"(v.r[0][3][0]), "+v"(v.r[0][3][1]),
                 "+v"(v.r[1][0][0]), "+v"(v.r[1][0][1]), "+v"(v.r[1][1][0]), "+v"(v.r[1][1][1]),
                 "+v"(v.r[1][2][0]), "+v"(v.r[1][2][1]), "+v"(v.r[1][3][0]), "+v"(v.r[1][3][1]));
}

// S^T of a tile: block 2 ch + j holds keys 32 ch + 8 grp + 4 j + i in element i.
template <int kQB>
__device__ __forceinline__ void scores(f32x4 (&sc)[kQB][4], const KTile& k, const State<kQB>& s) {
  // All of the first 32 dims before the second: no product waits for the last.
#pragma unroll
  for (int kk = 0; kk < 2; ++kk)
#pragma unroll
    for (int b = 0; b < kQB; ++b)
#pragma unroll
      for (int ch = 0; ch < 2; ++ch)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const f32x4 acc = kk == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : sc[b][2 * ch + j];
          sc[b][2 * ch + j] = mfma16x16x32(__builtin_bit_cast(f16x8, k.r[ch][j][kk]), s.q[b][kk], acc);
        }
}

// Drops the scores of keys past each column's bound, and below the unit's first
// slot where its first tile holds such keys (narrow units only: the others
// start on a tile's edge).
template <int kQB, bool kLow>
__device__ __forceinline__ void mask(f32x4 (&sc)[kQB][4], const State<kQB>& s, int key0) {
  const int grp = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int b = 0; b < kQB; ++b) {
    const int left = s.lim[b] - key0 - 8 * grp, skip = s.lo - key0 - 8 * grp;
#pragma unroll
    for (int blk = 0; blk < 4; ++blk)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = 32 * (blk >> 1) + 4 * (blk & 1) + i;
        if (key >= left || (kLow && key < skip)) sc[b][blk][i] = kNegInf;
      }
  }
}

// Largest score of each lane, log2 units.
template <int kQB>
__device__ __forceinline__ void tops(float (&mx)[kQB], f32x4 (&sc)[kQB][4], float ks2) {
#pragma unroll
  for (int b = 0; b < kQB; ++b) mx[b] = max16(sc[b]) * ks2;
}

// Moves the references of the columns whose scores grew past them.  A column
// moves only for scores of its own, so that a query's result does not depend on
// the others of its wave.
template <int kQB>
__device__ __forceinline__ void raise(State<kQB>& s, const float (&mx)[kQB]) {
  bool grew = false;
#pragma unroll
  for (int b = 0; b < kQB; ++b) grew = grew || mx[b] > s.m[b] + kRescaleSlack;
  if (__any(grew)) {
#pragma unroll
    for (int b = 0; b < kQB; ++b) {
      const float top = col_max(mx[b]);
      const float m_new = top > s.m[b] + kRescaleSlack ? top : s.m[b];
      const float r = m_new == s.m[b] ? 1.f : fast_exp2(s.m[b] - m_new);
      s.l[b] *= r;
#pragma unroll
      for (int t = 0; t < 4; ++t) s.o[b][t] *= r;
      s.m[b] = m_new;
    }
  }
}

typedef float f32x8 __attribute__((ext_vector_type(8)));

// p of block b, rounded to fp16 for the matrix cores (relative error 2^-11, as
// large as that of the fp16 V it meets).
template <int kQB>
__device__ __forceinline__ void weights(f16x8 (&pb)[kQB][2], const f32x4 (&sc)[kQB][4],
                                        const State<kQB>& s, int b) {
  const float neg_m = s.m[b] == kNegInf ? 0.f : -s.m[b];
#pragma unroll
  for (int ch = 0; ch < 2; ++ch) {
    f32x8 p;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      p[e] = fast_exp2(__builtin_fmaf(sc[b][2 * ch + e / 4][e % 4], s.ks2, neg_m));
    pb[b][ch] = __builtin_convertvector(p, f16x8);
  }
}

// o += V^T P^T, l += ones P^T: the sum adds the rounded p, so that the weights
// add to one.
template <int kQB>
__device__ __forceinline__ void add_values(State<kQB>& s, const f16x8 (&pb)[kQB][2], const VTile& v) {
  const f16x8 ones = {(f16)1.f, (f16)1.f, (f16)1.f, (f16)1.f, (f16)1.f, (f16)1.f, (f16)1.f, (f16)1.f};
#pragma unroll
  for (int ch = 0; ch < 2; ++ch) {
#pragma unroll
    for (int b = 0; b < kQB; ++b) s.l[b] = mfma16x16x32(ones, pb[b][ch], s.l[b]);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const u32x4 w = {v.r[ch][t][0][0], v.r[ch][t][0][1], v.r[ch][t][1][0], v.r[ch][t][1][1]};
      const f16x8 va = __builtin_bit_cast(f16x8, w);
#pragma unroll
      for (int b = 0; b < kQB; ++b) s.o[b][t] = mfma16x16x32(va, pb[b][ch], s.o[b][t]);
    }
  }
}

template <int kQB>
__device__ __forceinline__ void check_values(VTile& v, State<kQB>& s, const f16x8 (&pb)[kQB][2],
                                             int key0, const unsigned char* Vs) {
  unsigned bad = 0;
#pragma unroll
  for (int ch = 0; ch < 2; ++ch)
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int h = 0; h < 2; ++h) bad |= special2(v.r[ch][t][h][0]) | special2(v.r[ch][t][h][1]);
  if (__any((bad & 0x80008000u) != 0)) {
    masked_values<kQB>(v.r, s, pb, key0, s.o, Vs);
    // lgkmcnt(0) where the compiler sees it: it would wait for these LDS reads at
    // the end of the branch's other side too, among reads it does not know.
    __builtin_amdgcn_s_waitcnt(0xC07F);
  }
}

// Scores, online softmax and PV product of the tile of keys [key0, key0 + 64)
// in (Ks, Vs), whose loads have landed.
template <int kQB>
__device__ __forceinline__ void tile_step(State<kQB>& s, int key0, const unsigned char* Ks,
                                          const unsigned char* Vs) {
  KTile k;
  read_k(k, s.koff, Ks);
  wait_k(k);
  f32x4 sc[kQB][4];
  scores(sc, k, s);
  const bool masked = key0 < s.lo || key0 + kBN > s.seen;
  if (masked) mask<kQB, true>(sc, s, key0);
  float mx[kQB];
  tops(mx, sc, s.ks2);
  raise(s, mx);
  VTile v;
  read_v(v, s.voff, Vs);
  f16x8 pb[kQB][2];
#pragma unroll
  for (int b = 0; b < kQB; ++b) weights(pb, sc, s, b);
  wait_v(v);
  if (masked) check_values(v, s, pb, key0, Vs);
  add_values(s, pb, v);
}

// All but this wave's newest `ahead` tiles of loads (0 or 1, of four) have
// landed, and after the barrier that holds for every wave.
__device__ __forceinline__ void stage_ready(int ahead) {
  s_waitcnt_vm(ahead == 0 ? 0 : 4);
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __builtin_amdgcn_s_barrier();
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
}

// One unit: query rows r0 .. of a segment's (token, query head) rows against
// slots [k0, k1) of a block table row.
struct Unit {
  int tok0, rows;     // the segment's first token, its query rows
  int r0, hk;
  const int32_t* pages;
  int n_pages;        // entries of `pages`
  int k0, k1;
  int ctx;            // extension: cached slots of the row; decode: -1
  int split, n_split; // place among each query's partials; n_split = 0: the output itself
};

__device__ __forceinline__ Source make_source(const Args& a, const Unit& u) {
  Source s;
  s.k = reinterpret_cast<const unsigned char*>(a.k + u.hk * a.k_sh);
  s.v = reinterpret_cast<const unsigned char*>(a.v + u.hk * a.v_sh);
  s.row = u.pages;
  s.k_sp = (unsigned)(a.k_sp >> 3); s.k_sn = (int)a.k_sn * 2;
  s.v_sp = (unsigned)(a.v_sp >> 3); s.v_sn = (int)a.v_sn * 2;
  s.log2p = a.log2p; s.ppr = u.n_pages; s.n_pages = a.n_pages;
  s.end = u.k1;
  return s;
}

// Query row r of the unit's segment: its token, query head, and bound.
__device__ __forceinline__ int row_limit(const Args& a, const Unit& u, int token) {
  if (u.ctx >= 0) return min(u.ctx + (token - u.tok0) + 1, u.k1);
  return min(clampi(a.last[token * a.last_sb], -1, a.cap - 1) + 1, u.k1);
}

__device__ __forceinline__ int64_t part_index(const Args& a, const Unit& u, int token, int g) {
  return (((int64_t)token * a.KVH + u.hk) * u.n_split + u.split) * a.G + g;
}

template <int kQB>
__device__ __forceinline__ void load_queries(State<kQB>& s, const Args& a, const Unit& u, int first) {
  const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
#pragma unroll
  for (int b = 0; b < kQB; ++b) {
    const int r = first + 16 * b + col;
    const int rr = min(r, u.rows - 1);
    const int token = u.tok0 + rr / a.G, g = rr % a.G;
    const f16* qp = a.q + token * a.q_st + u.hk * a.q_sh + g * a.q_sg + 8 * grp;
    s.q[b][0] = load16(qp);
    s.q[b][1] = load16(qp + 32);
    if (a.cos != nullptr) {
      const int64_t co = token * a.cs_sn + 8 * grp;
      rope_pair(s.q[b][0], s.q[b][1], load16(a.cos + co), load16(a.sin + co),
                load16(a.cos + co + 32), load16(a.sin + co + 32));
    }
    s.lim[b] = r < u.rows ? row_limit(a, u, token) : u.k1;
  }
  int least = s.lim[0];
#pragma unroll
  for (int b = 1; b < kQB; ++b) least = min(least, s.lim[b]);
  for (int d = 8; d > 0; d >>= 1) least = min(least, __shfl_xor(least, d));  // columns: 16 lanes
  s.seen = __builtin_amdgcn_readfirstlane(least);
}

// o / l of a column.  Where all that it sees scored -infinity, o and l are 0 and
// the quotient, as the softmax, is NaN; `sees` is false where it sees nothing, and
// the output zero.
__device__ __forceinline__ void store_out(const Args& a, int token, int hk, int g, int d, f32x4 o,
                                          float l, bool sees) {
  const float inv = sees ? 1.f / l : 0.f;
  const f16x4 r = {(f16)(o[0] * inv), (f16)(o[1] * inv), (f16)(o[2] * inv), (f16)(o[3] * inv)};
  *reinterpret_cast<f16x4*>(a.out + token * a.o_st + hk * a.o_sh + g * a.o_sg + d) = r;
}

__device__ __forceinline__ void store_part(const Args& a, const Unit& u, int r, int t, f32x4 o,
                                           float m, float l, bool stats) {
  const int grp = (threadIdx.x & 63) >> 4;
  if (r >= u.rows) return;
  const int token = u.tok0 + r / a.G, g = r % a.G;
  if (u.n_split == 0) {
    store_out(a, token, u.hk, g, 16 * t + 4 * grp, o, l, true);
    return;
  }
  const int64_t p = part_index(a, u, token, g);
  *reinterpret_cast<f32x4*>(a.acc + p * kD + 16 * t + 4 * grp) = o;
  // New tokens all see their split 0, which says to the merge that they see
  // something where it holds scores of -infinity alone.
  if (stats && grp == 0) a.ml[p] = float2{l == 0.f && u.split == 0 ? -kHuge : m, l};
}

// A unit with no slot: every query's partial is absent (l = 0), the output zero.
__device__ __forceinline__ void empty_unit(const Args& a, const Unit& u, int n_rows) {
  for (int i = threadIdx.x; i < n_rows * 16; i += kThreads) {
    const int r = u.r0 + (i >> 4), d = 4 * (i & 15);
    if (r >= u.rows) break;
    const int token = u.tok0 + r / a.G, g = r % a.G;
    if (u.n_split == 0) store_out(a, token, u.hk, g, d, f32x4{0.f, 0.f, 0.f, 0.f}, 0.f, false);
    else if (d == 0) a.ml[part_index(a, u, token, g)] = float2{kNegInf, 0.f};
  }
}

// Places [from, to) of a unit's queries hold nothing.
__device__ __forceinline__ void no_parts(const Args& a, const Unit& u, int n_rows, int from, int to) {
  n_rows = min(n_rows, u.rows - u.r0);
  for (int i = threadIdx.x; i < (to - from) * n_rows; i += kThreads) {
    const int split = from + i / n_rows, r = u.r0 + i % n_rows;
    const int64_t th = (int64_t)(u.tok0 + r / a.G) * a.KVH + u.hk;
    a.ml[(th * u.n_split + split) * a.G + r % a.G] = float2{kNegInf, 0.f};
  }
}

// kQB * 64 query rows, kQB * 16 per wave; the waves share the key tiles, on a
// ring of kStages.  A step takes tile i's probabilities while the matrix cores
// form tile i + 1's scores (its K came into registers during the step before),
// then reads tile i + 2's K behind tile i's output product; tile i + 3 is on its
// way (one more stage, and tile i + 4 too, took 194 us where this takes 189: a
// 2048-token chunk behind 16384 slots).
template <int kQB>
__device__ __forceinline__ void wide_unit(const Args& a, const Unit& u, unsigned char* lds) {
  if (u.k1 <= u.k0) {
    empty_unit(a, u, kQB * 64);
    return;
  }
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const auto stage = [&](int st, int kv) { return lds + (st * 2 + kv) * kTileBytes; };
  const auto after = [](int st, int d) { return st + d < kStages ? st + d : st + d - kStages; };
  Source src = make_source(a, u);
  const int first = u.k0 & ~(kBN - 1);
  const int n = (u.k1 - first + kBN - 1) / kBN;
  const auto load = [&](int i, int st) {
    if (i < n) issue<16>(src, first + i * kBN, 16 * w, stage(st, 0), stage(st, 1));
  };
  load_pids(src, first >> a.log2p);
  load(0, 0);
  State<kQB> s;
  init_state(s, u.k0, a.scale_log2);
  const int row0 = u.r0 + w * kQB * 16;
  load_queries(s, a, u, row0);
  load(1, 1);
  load(2, 2);
  f32x4 sc[kQB][4];
  float mx[kQB];
  KTile k;
  stage_ready(n > 2 ? 1 : 0);  // tiles 0 and, if there is one, 1
  read_k(k, s.koff, stage(0, 0));
  wait_k(k);
  scores(sc, k, s);
  tops(mx, sc, s.ks2);
  if (n > 1) {
    read_k(k, s.koff, stage(1, 0));
    wait_k(k);
  }
  int st = 0;
  // Step i from its scores `sc`; `next` becomes step i + 1's.
  const auto step = [&](int i, f32x4 (&sc)[kQB][4], f32x4 (&next)[kQB][4]) __attribute__((always_inline)) {
    const int key0 = first + i * kBN;
    const bool masked = key0 + kBN > s.seen;
    if (masked) {
      mask<kQB, false>(sc, s, key0);
      tops(mx, sc, s.ks2);
    }
    raise(s, mx);
    // From here to wait_v, and from read_k to wait_k, nothing may branch: the
    // reads in flight are not the compiler's.
    VTile v;
    read_v(v, s.voff, stage(st, 1));
    __builtin_amdgcn_sched_barrier(0);
    f16x8 pb[kQB][2];
    scores(next, k, s);  // past the last tile: of its K again, unused
#pragma unroll
    for (int b = 0; b < kQB; ++b) weights(pb, sc, s, b);
    // One matrix product, then vector work for the 16 cycles that it takes.
#pragma unroll
    for (int j = 0; j < 8 * kQB; ++j) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // MFMA
      __builtin_amdgcn_sched_group_barrier(0x002, 3, 0);  // fma, conversion
      __builtin_amdgcn_sched_group_barrier(0x400, 2, 0);  // exp
    }
    // Keeps the exponentials here, with the matrix products (left alone, they
    // sink behind the branches to their use).
#pragma unroll
    for (int b = 0; b < kQB; ++b) asm volatile("" : "+v"(pb[b][0]), "+v"(pb[b][1]));
    wait_v(v);
    // Tile i + 2 is there, and every wave is past tile i - 1, whose stage takes
    // tile i + 3.
    stage_ready(0);
    load(i + 3, after(st, 3));
    if (masked) check_values(v, s, pb, key0, stage(st, 1));
    read_k(k, s.koff, stage(i + 2 < n ? after(st, 2) : st, 0));
    __builtin_amdgcn_sched_barrier(0);
    add_values(s, pb, v);
    tops(mx, next, s.ks2);
    wait_k(k);
    st = after(st, 1);
  };
  f32x4 next[kQB][4];
  for (int i = 0; i < n; i += 2) {  // in pairs, so that no scores are copied
    step(i, sc, next);
    if (i + 1 < n) step(i + 1, next, sc);
  }
  const int col = threadIdx.x & 15;
  const Args& late = late_args();
#pragma unroll
  for (int b = 0; b < kQB; ++b)
#pragma unroll
    for (int t = 0; t < 4; ++t)
      store_part(late, u, row0 + 16 * b + col, t, s.o[b][t], s.m[b], s.l[b][0], t == 0);
}

// At most 16 query rows; the waves take the key tiles in turn and join their
// states in LDS.
__device__ __forceinline__ void narrow_unit(const Args& a, const Unit& u, unsigned char* lds) {
  if (u.k1 <= u.k0) {
    empty_unit(a, u, 16);
    return;
  }
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  unsigned char* Ks = lds + w * 2 * kTileBytes;
  unsigned char* Vs = Ks + kTileBytes;
  Source src = make_source(a, u);
  const int first = u.k0 & ~(kBN - 1);
  const int n = (u.k1 - first + kBN - 1) / kBN;
  if (w < n) {
    load_pids(src, (first + w * kBN) >> a.log2p);
    issue<64>(src, first + w * kBN, 0, Ks, Vs);
  }
  State<1> s;
  init_state(s, u.k0, a.scale_log2);
  load_queries(s, a, u, u.r0);
  for (int i = w; i < n; i += kWaves) {
    s_waitcnt_vm(0);
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    tile_step(s, first + i * kBN, Ks, Vs);
    // The tile's reads are done: its LDS takes the wave's next one.
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (i + kWaves < n) issue<64>(src, first + (i + kWaves) * kBN, 0, Ks, Vs);
  }
  __syncthreads();
  f32x4* so = reinterpret_cast<f32x4*>(lds);                              // [wave][d tile][lane]
  float2* sml = reinterpret_cast<float2*>(lds + kWaves * 4 * 64 * 16);    // [wave][lane]
#pragma unroll
  for (int t = 0; t < 4; ++t) so[(w * 4 + t) * 64 + lane] = s.o[0][t];
  sml[w * 64 + lane] = float2{s.m[0], s.l[0][0]};
  __syncthreads();
  // Wave w joins dims 16 w .. 16 w + 15.
  float m[kWaves], l[kWaves], top = kNegInf;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    const float2 x = sml[i * 64 + lane];
    m[i] = x.x;
    l[i] = x.y;
    top = fmaxf(top, x.x);
  }
  float sum = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    if (l[i] == 0.f) continue;
    const float r = m[i] == top ? 1.f : fast_exp2(m[i] - top);
    sum += l[i] * r;
    o += so[(i * 4 + w) * 64 + lane] * r;
  }
  store_part(late_args(), u, u.r0 + (lane & 15), w, o, top, sum, w == 0);
}

// Slots [k0, k1) of split s of `n` splits of at least `least` over [lo, hi), cut at
// multiples of 64.
__device__ __forceinline__ void cut(int lo, int hi, int s, int n, int least, int& k0, int& k1) {
  const int first = lo & ~(kBN - 1);
  const int len = max((int)(((int64_t)hi - first + n * kBN - 1) / (n * kBN)) * kBN, least);
  const int64_t at = first + (int64_t)s * len;
  k0 = (int)(at < hi ? (s == 0 ? lo : at) : hi);
  k1 = (int)(at + len < hi ? at + len : hi);
}

// kForm: 0 narrow units, 1 and 2 wide ones of 64 kForm query rows.  Decode: the
// grid's first n_tiles * KVH * splits workgroups take the shared slots, the
// others one row's own slots each.
template <int kForm, bool kDecode>
__global__ __launch_bounds__(kThreads, 2) void span_kernel(Args a) {
  static_assert(kStages >= kWaves, "the narrow units' four tiles fit too");
  __shared__ __attribute__((aligned(16))) unsigned char lds[kStages * 2 * kTileBytes];
  constexpr int kTr = kForm == 0 ? 16 : 64 * kForm;
  const int n_first = a.n_tiles * ((a.KVH * a.splits + 7) & ~7);
  Unit u;
  u.ctx = -1;
  u.n_split = kDecode ? a.splits + a.own_splits : a.splits > 1 ? a.splits : 0;
  int before;
  if (!kDecode || (int)blockIdx.x < n_first) {
    // Workgroups go to the XCDs in turn.  Query tiles that read the same keys
    // share an XCD and its L2: pairs of a kv head and a split are dealt out in
    // turn, where there are XCDs enough for that.
    int id = blockIdx.x;
    if (a.KVH * a.splits >= 8) id = (id / (8 * a.n_tiles) * 8 + id % 8) * a.n_tiles + id / 8 % a.n_tiles;
    const int tile = id % a.n_tiles, rest = id / a.n_tiles;
    u.hk = rest % a.KVH;
    u.split = rest / a.KVH;
    if (u.split >= a.splits) return;
    const Segment g = find_segment<kDecode>(a, kTr, before, [&](int, int, int ahead, int tiles) {
      return tile < ahead + tiles;
    });
    if (g.index < 0) return;
    u.tok0 = g.lo;
    u.rows = (g.hi - g.lo) * a.G;
    u.r0 = (tile - before) * kTr;
    int end;
    if (kDecode) {
      const bool given = a.ptable != nullptr;
      u.pages = given ? a.ptable + (int64_t)g.index * a.pt_sb : a.table + (int64_t)g.lo * a.t_sb;
      u.n_pages = given ? a.pppr : a.ppr;
      end = g.slots;
    } else {
      u.pages = a.table + (int64_t)g.index * a.t_sb;
      u.n_pages = a.ppr;
      u.ctx = g.slots;
      const int newest = (min(u.r0 + kTr, u.rows) - 1) / a.G;   // last token of the tile
      end = u.ctx < 0 ? 0 : min(u.ctx + newest + 1, a.cap);
    }
    cut(0, end, u.split, a.splits, kMinKeys, u.k0, u.k1);
    if constexpr (kForm == 0) narrow_unit(a, u, lds);
    else wide_unit<kForm>(a, u, lds);
  } else {
    const int id = blockIdx.x - n_first;
    const int s = id % a.own_splits, rest = id / a.own_splits;
    u.hk = rest % a.KVH;
    const int token = rest / a.KVH;
    const int64_t last = a.last[token * a.last_sb];
    const Segment g = find_segment<true>(a, kTr, before, [&](int lo, int hi, int, int) {
      return lo <= token && token < hi;
    });
    const int end = clampi(last, -1, a.cap - 1) + 1;
    const int lo = min(g.slots, end);  // 0 in no group
    u.tok0 = token;
    u.pages = a.table + (int64_t)token * a.t_sb;
    u.n_pages = a.ppr;
    u.rows = a.G;
    u.r0 = 0;
    if (g.index < 0) {  // in no group: no workgroup reports on its shared slots
      if (s == 0) no_parts(a, u, 16, 0, a.splits);
    }
    u.split = a.splits + s;
    cut(lo, end, s, a.own_splits, kStepKeys, u.k0, u.k1);
    narrow_unit(a, u, lds);
  }
}

// Joins the `n` partials of each (token, kv head, query head).  kSubs groups of 16
// lanes, a lane for 4 dims, share a query: one where there are few partials (four
// queries to a wave: the two of each of a 2048-token chunk's 28672 queries, 202 ->
// 195 us for the call), four where there are many (24 rows in three groups, 17.4 ->
// 15.0).  A lane loads the statistics of
// a partial of its own, kEach times, and hands the weights around; then each
// group takes every kSubs-th partial, eight loads in flight together.
template <int kSubs, int kEach, bool kDecode>
__global__ __launch_bounds__(256) void span_merge_kernel(Args a, int n) {
  constexpr int kLanes = 16 * kSubs;  // of one query
  const int tid = threadIdx.x, lane = tid & 63;
  const int64_t id = (int64_t)blockIdx.x * (16 / kSubs) + tid / (16 * kSubs);
  bool in = id < (int64_t)a.tokens * a.KVH * a.G;
  const int64_t id0 = in ? id : 0;
  const int g = (int)(id0 % a.G);
  const int64_t th = id0 / a.G;
  const int hk = (int)(th % a.KVH), token = (int)(th / a.KVH);
  // New tokens outside every row were no unit's.
  if (!kDecode) in = in && token >= a.bounds[0] && token < a.bounds[a.n_seg];
  const int64_t p0 = th * n * a.G + g;
  const int mine = lane & (kLanes - 1), base = lane & ~(kLanes - 1);
  float2 x[kEach];
  float top = kNegInf;
#pragma unroll
  for (int h = 0; h < kEach; ++h) {
    const int j = mine + kLanes * h;
    x[h] = j < n ? a.ml[p0 + (int64_t)j * a.G] : float2{kNegInf, 0.f};
    top = fmaxf(top, x[h].x);
  }
  for (int d = kLanes / 2; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
  float sum = 0.f;
#pragma unroll
  for (int h = 0; h < kEach; ++h) {
    // Absent partials have l = 0, whatever their accumulators hold.
    const float w = x[h].y == 0.f ? 0.f : x[h].x == top ? 1.f : fast_exp2(x[h].x - top);
    sum += x[h].y == 0.f ? 0.f : w * x[h].y;
    x[h].x = w;
  }
  for (int d = kLanes / 2; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
  const int sub = (tid >> 4) & (kSubs - 1), d0 = 4 * (lane & 15);
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  constexpr int kRounds = kLanes * kEach / kSubs;  // partials of a group
#pragma unroll 1
  for (int i0 = 0; i0 < kRounds; i0 += 8) {
    if (i0 * kSubs >= n) break;
    f32x4 v[8];
    float w[8];
#pragma unroll
    for (int i = 0; i < 8 && i0 + i < kRounds; ++i) {
      const int j = sub + kSubs * (i0 + i);
      float l = 0.f;
      w[i] = 0.f;
#pragma unroll
      for (int h = 0; h < kEach; ++h) {
        const float wh = __shfl(x[h].x, base + (j & (kLanes - 1)));
        const float lh = __shfl(x[h].y, base + (j & (kLanes - 1)));
        if (j / kLanes == h) {
          w[i] = wh;
          l = lh;
        }
      }
      v[i] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (l != 0.f)
        v[i] = *reinterpret_cast<const f32x4*>(a.acc + (p0 + (int64_t)j * a.G) * kD + d0);
    }
#pragma unroll
    for (int i = 0; i < 8 && i0 + i < kRounds; ++i) o += v[i] * w[i];
  }
  if constexpr (kSubs > 1) {
#pragma unroll
    for (int c = 0; c < 4; ++c) o[c] = col_sum(o[c]);
  }
  const bool sees = kDecode ? a.last[token * a.last_sb] >= 0 : top > kNegInf;
  if (in && (kSubs == 1 || lane < 16)) store_out(a, token, hk, g, d0, o, sum, sees);
}

// K (rotated with cos / sin if given) and V of every new token into its slot:
// 16 tokens of one kv head per workgroup, 16 threads a token, four for K's
// rotate-half chunk pairs and eight for V's chunks.
struct AppendArgs {
  const f16* k;
  int64_t k_sh, k_sn;
  const f16* v;
  int64_t v_sh, v_sn;
  f16* kp;
  f16* vp;
};

__global__ __launch_bounds__(256) void extend_append_kernel(Args a, AppendArgs p) {
  const int token = blockIdx.x * 16 + (threadIdx.x >> 4);
  const int sub = threadIdx.x & 15, h = blockIdx.y;
  if (token >= a.tokens || sub >= 12) return;
  int lo = 0, hi = a.n_seg;  // the token's row: the last one that starts at or before it
  while (lo + 1 < hi) {
    const int mid = (lo + hi) / 2;
    if (a.bounds[mid] <= token) lo = mid;
    else hi = mid;
  }
  const int start = a.bounds[lo];
  if (start < 0 || start > token || a.bounds[lo + 1] <= token) return;
  const int64_t ctx = a.last[lo * a.last_sb];
  if (ctx < 0 || ctx > a.cap) return;
  const int slot = (int)ctx + token - start;
  if (slot >= a.cap) return;
  const int page = a.table[(int64_t)lo * a.t_sb + (slot >> a.log2p)];
  if (page < 0 || page >= a.n_pages) return;
  const int in_page = slot & ((1 << a.log2p) - 1);
  if (sub < 4) {
    const f16* src = p.k + h * p.k_sh + token * p.k_sn + 8 * sub;
    f16x8 x = load16(src), y = load16(src + 32);
    if (a.cos != nullptr) {
      const int64_t co = token * a.cs_sn + 8 * sub;
      rope_pair(x, y, load16(a.cos + co), load16(a.sin + co), load16(a.cos + co + 32),
                load16(a.sin + co + 32));
    }
    f16* dst = p.kp + page * a.k_sp + h * a.k_sh + in_page * a.k_sn + 8 * sub;
    store16(dst, x);
    store16(dst + 32, y);
  } else {
    const int c = 8 * (sub - 4);
    store16(p.vp + page * a.v_sp + h * a.v_sh + in_page * a.v_sn + c,
            load16(p.v + h * p.v_sh + token * p.v_sn + c));
  }
}

// ---------------------------------------------------------------------------
// host side

constexpr int kCus = 256;

struct Plan {
  int form, n_tiles, splits, own_splits;
};

int64_t part_bytes(int64_t queries, int n) { return queries * n * (kD * 4 + (int64_t)sizeof(float2)); }

// Units of the larger forms read a tile's K and V for more query rows, those of
// the smaller ones leave fewer columns empty and make more workgroups.  MI355X, 7
// queries to a kv head, us in a replayed graph, this rule / the next larger form:
// 32 rows of 2 tokens behind 4000 slots 23.6 / 27.0, of 8 tokens 26.1 / 34.5, two
// rows of a 4096-slot prefix 9.1 / 10.9; the next smaller one: 16 rows of 9 to 301
// tokens behind 2048 slots 56 / 61, 2048 tokens behind 16384 190 / 245.
int pick_form(int64_t rows_per_segment) {
  return rows_per_segment <= 16 ? 0 : rows_per_segment <= 64 ? 1 : 2;
}

// Splits of at least `least` keys, so that these units are no more than the two
// workgroups per CU that run at once: some more would take a second round (286
// units of 16 ragged rows behind 2048 slots: 56 us whole, 62 cut in two).  A decode's
// own slots are counted by themselves, though they share the launch: 96 rows of a
// 32768-slot prefix are 504 wide and 384 narrow workgroups.
int pick_splits(int64_t units, int cap, int least) {
  const int64_t by_len = std::min<int64_t>(kMaxSplits, ((int64_t)cap + least - 1) / least);
  return (int)std::max<int64_t>(1, std::min<int64_t>(by_len, 2 * kCus / units));
}

Plan decode_plan(int B, int KVH, int G, int n_groups, int cap) {
  Plan p;
  const int64_t rows = (int64_t)B * G;
  p.form = pick_form((rows + n_groups - 1) / n_groups);
  const int tr = p.form == 0 ? 16 : 64 * p.form;
  p.n_tiles = (int)(rows / tr) + n_groups;
  // Half as many as kMinKeys allows: the merge reads them all (24 rows in three
  // groups behind up to 4096 shared slots: 14.9 us with all, 14.3 with these).
  p.splits = pick_splits((int64_t)p.n_tiles * KVH, cap, 2 * kMinKeys);
  p.own_splits = pick_splits((int64_t)B * KVH, cap, kStepKeys);
  return p;
}

Plan extend_plan(int B, int KVH, int G, int total, int cap) {
  Plan p;
  const int64_t rows = (int64_t)total * G;
  p.form = pick_form((rows + B - 1) / B);
  const int tr = p.form == 0 ? 16 : 64 * p.form;
  p.n_tiles = (int)(rows / tr) + B;
  p.splits = pick_splits((int64_t)p.n_tiles * KVH, cap, kMinKeys);
  p.own_splits = 0;
  return p;
}

template <bool kDecode>
int launch(const Args& a, const Plan& p, hipStream_t st) {
  const int64_t grid = a.n_tiles * (((int64_t)a.KVH * a.splits + 7) & ~(int64_t)7) +
                       (kDecode ? (int64_t)a.tokens * a.KVH * a.own_splits : 0);
  if (grid > 0x7fffffff) return QF_ERR_UNSUPPORTED;
  const dim3 g((unsigned)grid), b(kThreads);
  if (p.form == 0) hipLaunchKernelGGL((span_kernel<0, kDecode>), g, b, 0, st, a);
  else if (p.form == 1) hipLaunchKernelGGL((span_kernel<1, kDecode>), g, b, 0, st, a);
  else hipLaunchKernelGGL((span_kernel<2, kDecode>), g, b, 0, st, a);
  int rc = (int)hipGetLastError();
  const int n = kDecode ? a.splits + a.own_splits : a.splits;
  if (rc == 0 && (kDecode || n > 1)) {
    const int64_t queries = (int64_t)a.tokens * a.KVH * a.G;
    const dim3 all((unsigned)((queries + 15) / 16)), quarter((unsigned)((queries + 3) / 4));
    if (n <= 8) hipLaunchKernelGGL((span_merge_kernel<1, 1, kDecode>), all, dim3(256), 0, st, a, n);
    else if (n <= 64) hipLaunchKernelGGL((span_merge_kernel<4, 1, kDecode>), quarter, dim3(256), 0, st, a, n);
    else if (kDecode) hipLaunchKernelGGL((span_merge_kernel<4, 2, true>), quarter, dim3(256), 0, st, a, n);
    rc = (int)hipGetLastError();
  }
  return rc;
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Checks and fills what both entry points share; the query rows' strides and
// the segments are the caller's.
int fill(Args& a, const void* q, const void* k_pool, int64_t kp_sp, int64_t kp_sh, int64_t kp_sn,
         const void* v_pool, int64_t vp_sp, int64_t vp_sh, int64_t vp_sn,
         const int32_t* block_table, int64_t bt_sb, int pages_per_row, int n_pages, int page_size,
         const int32_t* bounds, const int64_t* last, int64_t last_sb, void* ws, void* out, int n_seg,
         int tokens, int KVH, int G, int D, int cap, float scale) {
  const int l2 = page_log2(page_size, pages_per_row, n_pages);
  if (D != kD || G < 1 || G > 16 || l2 < 0) return QF_ERR_UNSUPPORTED;
  if (!q || !k_pool || !v_pool || !block_table || !bounds || !last || !ws || !out)
    return QF_ERR_INVALID_ARG;
  if (n_seg < 1 || tokens < 1 || KVH < 1 || bt_sb < pages_per_row || cap < 1 ||
      cap > pages_per_row * page_size || !(scale > 0.f) || !(scale < 1e30f))
    return QF_ERR_INVALID_ARG;
  if (!al16(q) || !al16(k_pool) || !al16(v_pool) || !al16(ws) ||
      (reinterpret_cast<uintptr_t>(out) & 7u) != 0 ||
      ((kp_sp | kp_sh | kp_sn | vp_sp | vp_sh | vp_sn) & 7) != 0)
    return QF_ERR_INVALID_ARG;
  // A page's rows are addressed with 32-bit byte offsets, pages with 32-bit
  // strides of 16 bytes.
  if (kp_sn < kD || vp_sn < kD || kp_sn > 0x3fffffff / page_size || vp_sn > 0x3fffffff / page_size ||
      kp_sp < 0 || vp_sp < 0 || kp_sp >> 3 > 0x7fffffff || vp_sp >> 3 > 0x7fffffff)
    return QF_ERR_UNSUPPORTED;
  if (n_seg > 0x3fffffff || (int64_t)tokens * G > 0x3fffffff || (int64_t)tokens * KVH * G > 0x7fffffff ||
      (int64_t)cap + tokens > 0x7fffffff)
    return QF_ERR_UNSUPPORTED;
  a = Args{};
  a.q = static_cast<const f16*>(q);
  a.k = static_cast<const f16*>(k_pool);
  a.k_sp = kp_sp; a.k_sh = kp_sh; a.k_sn = kp_sn;
  a.v = static_cast<const f16*>(v_pool);
  a.v_sp = vp_sp; a.v_sh = vp_sh; a.v_sn = vp_sn;
  a.table = block_table;
  a.t_sb = bt_sb;
  a.log2p = l2; a.n_pages = n_pages; a.ppr = pages_per_row;
  a.bounds = bounds;
  a.last = last;
  a.last_sb = last_sb;
  a.n_seg = n_seg; a.tokens = tokens; a.KVH = KVH; a.G = G; a.cap = cap;
  a.out = static_cast<f16*>(out);
  a.scale_log2 = scale * kLog2e;
  return QF_OK;
}

void set_parts(Args& a, const Plan& p, void* ws) {
  a.n_tiles = p.n_tiles;
  a.splits = p.splits;
  a.own_splits = p.own_splits;
  a.acc = static_cast<float*>(ws);
  a.ml = reinterpret_cast<float2*>(a.acc + (int64_t)a.tokens * a.KVH * a.G *
                                               (p.splits + p.own_splits) * kD);
}

}  // namespace span
}  // namespace qf

extern "C" int64_t qf_decode_attn_prefix_workspace(int B, int KVH, int G, int n_groups, int cap) {
  using namespace qf::span;
  if (B < 1 || KVH < 1 || n_groups < 1 || cap < 1) return QF_ERR_INVALID_ARG;
  if (G < 1 || G > 16 || (int64_t)B * KVH * G > 0x7fffffff || n_groups > 0x3fffffff)
    return QF_ERR_UNSUPPORTED;
  const Plan p = decode_plan(B, KVH, G, n_groups, cap);
  return part_bytes((int64_t)B * KVH * G, p.splits + p.own_splits);
}

extern "C" int qf_decode_attn_prefix_paged(
    const void* q, int64_t q_sb, int64_t q_sh, int64_t q_sg, const void* k_pool, int64_t kp_sp,
    int64_t kp_sh, int64_t kp_sn, const void* v_pool, int64_t vp_sp, int64_t vp_sh, int64_t vp_sn,
    const int32_t* block_table, int64_t bt_sb, int pages_per_row, int n_pages, int page_size,
    const int32_t* prefix_rows, const int32_t* prefix_len, int n_groups, const int32_t* prefix_table,
    int64_t pt_sb, int prefix_pages, const int64_t* kv_last, int64_t kv_last_sb, void* ws,
    int64_t ws_bytes, void* out, int64_t o_sb, int64_t o_sh, int64_t o_sg, int B,
    int KVH, int G, int D, float scale, void* stream) {
  using namespace qf;
  using namespace qf::span;
  Args a;
  const int cap = page_log2(page_size, pages_per_row, n_pages) < 0 ? 0 : pages_per_row * page_size;
  const int rc = fill(a, q, k_pool, kp_sp, kp_sh, kp_sn, v_pool, vp_sp, vp_sh, vp_sn, block_table,
                      bt_sb, pages_per_row, n_pages, page_size, prefix_rows, kv_last, kv_last_sb, ws,
                      out, n_groups, B, KVH, G, D, cap, scale);
  if (rc != QF_OK) return rc;
  if (prefix_table != nullptr &&
      (prefix_pages < 1 || pt_sb < prefix_pages || (int64_t)prefix_pages * page_size > 0x7fffffff - B))
    return QF_ERR_INVALID_ARG;
  if (!prefix_len || ((q_sb | q_sh | q_sg) & 7) != 0 || ((o_sb | o_sh | o_sg) & 3) != 0)
    return QF_ERR_INVALID_ARG;
  a.q_st = q_sb; a.q_sh = q_sh; a.q_sg = q_sg;
  a.o_st = o_sb; a.o_sh = o_sh; a.o_sg = o_sg;
  a.plen = prefix_len;
  a.ptable = prefix_table;
  a.pt_sb = pt_sb;
  a.pppr = prefix_pages;
  a.pcap = prefix_table == nullptr ? cap : std::min(cap, prefix_pages * page_size);
  const Plan p = decode_plan(B, KVH, G, n_groups, cap);
  if (ws_bytes < part_bytes((int64_t)B * KVH * G, p.splits + p.own_splits)) return QF_ERR_SCRATCH_LIMIT;
  set_parts(a, p, ws);
  return launch<true>(a, p, static_cast<hipStream_t>(stream));
}

extern "C" int64_t qf_prefill_extend_workspace(int B, int QH, int KVH, int total, int cap) {
  using namespace qf::span;
  if (B < 1 || KVH < 1 || QH < KVH || QH % KVH != 0 || total < 1 || cap < 1) return QF_ERR_INVALID_ARG;
  if (QH / KVH > 16 || (int64_t)total * QH > 0x7fffffff || B > 0x3fffffff) return QF_ERR_UNSUPPORTED;
  const Plan p = extend_plan(B, KVH, QH / KVH, total, cap);
  return p.splits > 1 ? part_bytes((int64_t)total * QH, p.splits) : 0;
}

int qf::extend_attention(const ExtendCall& c, const void* q, int64_t q_sh, int64_t q_sn, void* out,
                         int64_t o_sh, int64_t o_sn, const void* k_pool, int64_t kp_sp, int64_t kp_sh,
                         int64_t kp_sn, const void* v_pool, int64_t vp_sp, int64_t vp_sh,
                         int64_t vp_sn, void* ws, int64_t ws_bytes, float scale, hipStream_t st) {
  using namespace qf::span;
  const int G = c.QH / c.KVH;
  Args a;
  const int rc = fill(a, q, k_pool, kp_sp, kp_sh, kp_sn, v_pool, vp_sp, vp_sh, vp_sn, c.table, c.t_sb,
                      c.ppr, c.n_pages, c.page_size, c.cu, c.context, c.ctx_sb, ws, out, c.B, c.T, c.KVH,
                      G, kD, c.cap, scale);
  if (rc != QF_OK) return rc;
  a.q_st = q_sn; a.q_sh = G * q_sh; a.q_sg = q_sh;
  a.o_st = o_sn; a.o_sh = G * o_sh; a.o_sg = o_sh;
  const Plan p = extend_plan(c.B, c.KVH, G, c.T, c.cap);
  if (p.splits > 1 && ws_bytes < part_bytes((int64_t)c.T * c.QH, p.splits)) return QF_ERR_SCRATCH_LIMIT;
  set_parts(a, p, ws);
  return launch<false>(a, p, st);
}

extern "C" int qf_prefill_extend_paged(
    const void* q, int64_t q_sh, int64_t q_sn, const void* k, int64_t k_sh, int64_t k_sn,
    const void* v, int64_t v_sh, int64_t v_sn, const int32_t* cu_seqlens, int total,
    const int64_t* context, int64_t ctx_sb, const void* cos, const void* sin, int64_t cs_sn,
    void* k_pool, int64_t kp_sp, int64_t kp_sh, int64_t kp_sn, void* v_pool, int64_t vp_sp,
    int64_t vp_sh, int64_t vp_sn, const int32_t* block_table, int64_t bt_sb, int pages_per_row,
    int n_pages, int page_size, int cap, void* ws, int64_t ws_bytes, void* out, int64_t o_sh,
    int64_t o_sn, int B, int QH, int KVH, int D, float scale, void* stream) {
  using namespace qf;
  using namespace qf::span;
  if (KVH < 1 || QH < KVH || QH % KVH != 0) return QF_ERR_INVALID_ARG;
  const int G = QH / KVH;
  Args a;
  const int rc = fill(a, q, k_pool, kp_sp, kp_sh, kp_sn, v_pool, vp_sp, vp_sh, vp_sn, block_table,
                      bt_sb, pages_per_row, n_pages, page_size, cu_seqlens, context, ctx_sb, ws, out,
                      B, total, KVH, G, D, cap, scale);
  if (rc != QF_OK) return rc;
  if (!k || !v || !al16(k) || !al16(v) || ((q_sh | q_sn | k_sh | k_sn | v_sh | v_sn) & 7) != 0 ||
      ((o_sh | o_sn) & 3) != 0 || (cos == nullptr) != (sin == nullptr) || !al16(cos) || !al16(sin) ||
      (cos != nullptr && (cs_sn & 7) != 0))
    return QF_ERR_INVALID_ARG;
  if (KVH > 65535) return QF_ERR_UNSUPPORTED;
  a.q_st = q_sn; a.q_sh = G * q_sh; a.q_sg = q_sh;
  a.o_st = o_sn; a.o_sh = G * o_sh; a.o_sg = o_sh;
  a.cos = static_cast<const f16*>(cos);
  a.sin = static_cast<const f16*>(sin);
  a.cs_sn = cs_sn;
  const Plan p = extend_plan(B, KVH, G, total, cap);
  if (p.splits > 1 && ws_bytes < part_bytes((int64_t)total * QH, p.splits)) return QF_ERR_SCRATCH_LIMIT;
  set_parts(a, p, ws);
  const AppendArgs ap = {static_cast<const f16*>(k), k_sh, k_sn, static_cast<const f16*>(v), v_sh, v_sn,
                         static_cast<f16*>(k_pool), static_cast<f16*>(v_pool)};
  hipStream_t st = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(extend_append_kernel, dim3((total + 15) / 16, KVH), dim3(256), 0, st, a, ap);
  const int err = (int)hipGetLastError();
  return err != 0 ? err : launch<false>(a, p, st);
}
