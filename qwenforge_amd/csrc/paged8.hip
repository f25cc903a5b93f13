// Tokens quantised into paged caches held in 8 bits, slots read back, pages copied
// (gfx950; the format is qf_paged8.h's).
//
// A wave takes one block of 16 slots of one kv head, K and V or one of them
// (kv8_block.h).  Four waves are a workgroup.
#include <algorithm>
#include <type_traits>

#include "kv8_block.h"

namespace qf {
namespace kv8 {

constexpr int kWaves = 4;
constexpr int64_t kApartMost = 1500;   // blocks of one kv head

struct RowsArgs {
  Pool p;
  f16* k;                    // packed tokens: the append's input, the read's output
  int64_t k_sl, k_sh, k_sn;
  f16* v;
  int64_t v_sl, v_sh, v_sn;
  const int32_t* cu;
  const int64_t* first;      // first slot of each row's tokens
  int64_t first_sb;
  int B, total, longest;     // no row has more than `longest` tokens
  int cap;                   // slots of a row from cap on are not there
  const f16* cos;
  const f16* sin;
  int64_t cs_sn;
};

// A wave's work: tokens [tok, tok + n) of a row at slots lo .. lo + n - 1 of its
// block `block`; n = 0: none.  lo < 0: the row is parked.
struct Unit {
  int row, tok, n, lo, block;
};

// Blocks that n slots from `first` touch.
__device__ __forceinline__ int blocks_of(int64_t first, int n) {
  return n <= 0 ? 0 : (int)(((first < 0 ? 0 : first) % kBlock + n + kBlock - 1) / kBlock);
}

// Tokens [lo, hi) of row r, any contents of cu kept within the tokens and the longest row.
__device__ __forceinline__ void row_tokens(const RowsArgs& a, int r, int& lo, int& hi) {
  lo = clampi(a.cu[r], 0, a.total);
  hi = clampi(a.cu[r + 1], lo, min(a.total, lo + a.longest));
}

// The id-th of the blocks that the rows' tokens touch, counted row by row.  kSingle: no
// row has more than one token, and row id has the block.
template <bool kSingle>
__device__ __forceinline__ Unit find_unit(const RowsArgs& a, int id) {
  if constexpr (kSingle) {
    if (id >= a.B) return {0, 0, 0, 0, 0};
    int lo, hi;
    row_tokens(a, id, lo, hi);
    const int64_t first = a.first[id * a.first_sb];
    if (first < 0) return {id, lo, hi - lo, -1, 0};
    const int64_t block = first / kBlock;
    return {id, lo, hi - lo, (int)(first % kBlock),
            (int)(block < 0x7fffffff / kBlock ? block : 0x7fffffff / kBlock)};
  }
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
      // Slot of the row's first token; none is past 2^40.
      const int64_t at = f < 0 ? 0 : f < ((int64_t)1 << 40) ? f : (int64_t)1 << 40;
      const int64_t s0 = at / kBlock * kBlock + (int64_t)k * kBlock;
      const int64_t from = s0 < at ? at : s0;
      if (from - at >= h - l) return {0, 0, 0, 0, 0};
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

// Bound by the loads that wait for each other -- the rows' offsets, the table, tokens and old
// codes.  kApart: a wave has a block's keys or its values, else both (one token of 32 rows
// 4.2 us, with both 4.8; one row of 2048 tokens 5.0 and 5.3; 4 rows of 8192, 25 MB, 10.9
// and 9.3, 2.7 TB/s).
template <bool kE4m3, bool kSingle, bool kApart>
__global__ __launch_bounds__(64 * kWaves) void append_kernel(RowsArgs a) {
  const int w = __builtin_amdgcn_readfirstlane(blockIdx.x * kWaves + (threadIdx.x >> 6));
  const int hk = blockIdx.y % a.p.kvh, layer = blockIdx.y / a.p.kvh;
  const Unit u = find_unit<kSingle>(a, kApart ? w >> 1 : w);
  if (u.n <= 0 || u.lo < 0) return;
  const int slot0 = u.block << 4;                       // of the block
  const int lp = slot0 >> a.p.log2p;
  if (lp >= a.p.ppr) return;
  const int end = min(u.lo + u.n, a.cap - slot0);
  if (end <= u.lo) return;
  const Tokens t = {a.k + layer * a.k_sl + hk * a.k_sh + u.tok * a.k_sn, a.k_sn,
                    a.v + layer * a.v_sl + hk * a.v_sh + u.tok * a.v_sn, a.v_sn,
                    a.cos == nullptr ? nullptr : a.cos + u.tok * a.cs_sn,
                    a.cos == nullptr ? nullptr : a.sin + u.tok * a.cs_sn, a.cs_sn};
  const int page = a.p.table[u.row * a.p.t_sb + lp];
  if (!kApart) append_block<kE4m3, true, true>(a.p, layer, hk, page, slot0, u.lo, end, t);
  else if (w & 1) append_block<kE4m3, false, true>(a.p, layer, hk, page, slot0, u.lo, end, t);
  else append_block<kE4m3, true, false>(a.p, layer, hk, page, slot0, u.lo, end, t);
}

// A wave a block, the heads of a block side by side, so that a token's heads are written
// together, past the caches (203000 slots of 2 heads: 41.8 -> 35.4 us; 43.7 with the
// heads apart, 44 then also with four blocks a wave): 4.5 TB/s, two bytes written for each
// read.
template <bool kE4m3>
__global__ __launch_bounds__(64 * kWaves) void read_kernel(RowsArgs a) {
  const int lane = threadIdx.x & 63;
  const int id = __builtin_amdgcn_readfirstlane(blockIdx.x * kWaves + (threadIdx.x >> 6));
  const int hk = id % a.p.kvh, layer = blockIdx.y;
  const Unit u = find_unit<false>(a, id / a.p.kvh);
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
  // K: four lanes a slot, 16 dims each.  V: dims 2d and 2d + 1, slots j0 .. j0 + 7.
  const int t = lane >> 2, c = 16 * (lane & 3);
  const int d = lane & 31, j0 = lane >> 5 << 3;
  const u32x4 kw = *reinterpret_cast<const u32x4*>(a.p.k + at + (int64_t)in_page * kD + t * kD + c);
  const uint8_t* vp = a.p.v + at + (int64_t)(in_page >> 6) * 64 * kD + (in_page & 63) + 128 * d + j0;
  const u32x2 vw0 = *reinterpret_cast<const u32x2*>(vp), vw1 = *reinterpret_cast<const u32x2*>(vp + 64);
  u32x4 k0 = __builtin_bit_cast(u32x4, values8<kE4m3>(kw[0], kw[1], ks));
  u32x4 k1 = __builtin_bit_cast(u32x4, values8<kE4m3>(kw[2], kw[3], ks));
  u32x4 v0 = __builtin_bit_cast(u32x4, values8<kE4m3>(vw0[0], vw0[1], vs));
  u32x4 v1 = __builtin_bit_cast(u32x4, values8<kE4m3>(vw1[0], vw1[1], vs));
  const unsigned ksay = none ? 0u : ks == ks ? ~0u : 0x7E007E00u, vsay = none ? 0u : vs == vs ? ~0u : 0x7E007E00u;
  if (t >= lo && t < lo + u.n) {
    f16* dst = a.k + layer * a.k_sl + hk * a.k_sh + (int64_t)(u.tok + t - lo) * a.k_sn + c;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      k0[i] = ksay == ~0u ? k0[i] : ksay;
      k1[i] = ksay == ~0u ? k1[i] : ksay;
    }
    __builtin_nontemporal_store(k0, reinterpret_cast<u32x4*>(dst));
    __builtin_nontemporal_store(k1, reinterpret_cast<u32x4*>(dst + 8));
  }
  f16* dst = a.v + layer * a.v_sl + hk * a.v_sh + (int64_t)u.tok * a.v_sn + 2 * d;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    // Slot j of both dims, as one word.
    const unsigned w = __builtin_amdgcn_perm(v1[j / 2], v0[j / 2], j & 1 ? 0x07060302u : 0x05040100u);
    if (j0 + j >= lo && j0 + j < lo + u.n)
      __builtin_nontemporal_store(vsay == ~0u ? w : vsay,
                                  reinterpret_cast<unsigned*>(dst + (j0 + j - lo) * a.v_sn));
  }
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

// Checks and fills what the append and the read share; `blocks`: how many the tokens may
// touch.
int make_rows(RowsArgs& a, int64_t& blocks, const QfRows8& h) {
  int rc = check_rows(h);
  if (rc != QF_OK) return rc;
  a = RowsArgs{};
  rc = make_pool(h.pool, a.p);
  if (rc != QF_OK) return rc;
  a.k = static_cast<f16*>(h.k);
  a.k_sl = h.k_sl; a.k_sh = h.k_sh; a.k_sn = h.k_sn;
  a.v = static_cast<f16*>(h.v);
  a.v_sl = h.v_sl; a.v_sh = h.v_sh; a.v_sn = h.v_sn;
  a.cu = h.cu_seqlens;
  a.first = h.first;
  a.first_sb = h.first_sb;
  a.B = (int)h.B; a.total = (int)h.total; a.longest = (int)h.max_seqlen;
  a.cap = row_cap(a.p);
  // A row's n tokens touch at most n / 16 + 2 blocks, one of them if n is 1.
  blocks = h.max_seqlen == 1 ? h.B : h.total / kBlock + 2 * std::min(h.B, h.total);
  if (blocks > 0x7fffffff / h.pool.KVH) return QF_ERR_UNSUPPORTED;
  return QF_OK;
}

}  // namespace kv8
}  // namespace qf

int qf::kv8::check_rows(const QfRows8& h) {
  if (h.D != kD) return QF_ERR_UNSUPPORTED;
  if (!h.k || !h.v || !h.cu_seqlens || !h.first || h.B < 1 || h.total < 1 || h.max_seqlen < 1 ||
      h.max_seqlen > h.total)
    return QF_ERR_INVALID_ARG;
  if (((reinterpret_cast<uintptr_t>(h.k) | reinterpret_cast<uintptr_t>(h.v)) & 15u) != 0 ||
      ((h.k_sl | h.k_sh | h.k_sn | h.v_sl | h.v_sh | h.v_sn) & 7) != 0)
    return QF_ERR_INVALID_ARG;
  if (h.B > 0x3fffffff || h.total > 0x3fffffff) return QF_ERR_UNSUPPORTED;
  if ((h.cos == nullptr) != (h.sin == nullptr) ||
      ((reinterpret_cast<uintptr_t>(h.cos) | reinterpret_cast<uintptr_t>(h.sin)) & 15u) != 0 ||
      (h.cos != nullptr && (h.cs_sn & 7) != 0))
    return QF_ERR_INVALID_ARG;
  return QF_OK;
}

int qf::kv8::append(const QfRows8& h, int cap, hipStream_t st) {
  RowsArgs a;
  int64_t blocks;
  const int rc = make_rows(a, blocks, h);
  if (rc != QF_OK) return rc;
  a.cos = static_cast<const f16*>(h.cos);
  a.sin = static_cast<const f16*>(h.sin);
  a.cs_sn = h.cs_sn;
  a.cap = std::min(a.cap, cap);
  // Apart until the waves are more than run at once.
  const int64_t pairs = h.pool.KVH * h.pool.layers;
  const bool e4m3 = h.pool.code == QF_CODE_E4M3, apart = blocks * pairs <= kApartMost;
  const dim3 grid((unsigned)(((apart ? 2 : 1) * blocks + kWaves - 1) / kWaves), (unsigned)pairs), block(64 * kWaves);
  const auto launch = [&](auto code, auto single) {
    if (apart) hipLaunchKernelGGL((append_kernel<code.value, single.value, true>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((append_kernel<code.value, single.value, false>), grid, block, 0, st, a);
  };
  const auto by_code = [&](auto single) {
    if (e4m3) launch(std::true_type{}, single);
    else launch(std::false_type{}, single);
  };
  if (h.max_seqlen == 1) by_code(std::true_type{});
  else by_code(std::false_type{});
  return (int)hipGetLastError();
}

extern "C" int qf_append_paged8(const QfRows8* rows, void* stream) {
  if (!rows) return QF_ERR_INVALID_ARG;
  return qf::kv8::append(*rows, 0x7fffffff, static_cast<hipStream_t>(stream));
}

extern "C" int qf_read_paged8(const QfRows8* rows, void* stream) {
  using namespace qf::kv8;
  RowsArgs a;
  int64_t blocks;
  if (!rows || rows->cos || rows->sin) return QF_ERR_INVALID_ARG;
  const int rc = make_rows(a, blocks, *rows);
  if (rc != QF_OK) return rc;
  const dim3 grid((unsigned)((blocks * rows->pool.KVH + kWaves - 1) / kWaves), (unsigned)rows->pool.layers);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (rows->pool.code == QF_CODE_E4M3)
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
