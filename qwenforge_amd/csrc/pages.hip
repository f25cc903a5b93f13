// Page copies of the paged KV cache (gfx950): the partly filled last page of a
// forked row, the pages a row takes for itself before it writes to them, the
// moves of a compaction.
//
// Every byte is read and written once, by 16-byte loads, four in flight per
// thread, all layers' K and V in one launch, so memory bounds it: 700 pages of 64
// slots in 24 layers (1.1 GB read and written) take 213 us, 5.2 TB/s, where a
// copy of 1 GiB runs at 4.8.  A partly filled page of one row takes 2.7 us, the
// launch; called from Python 8.6 us with indices on the device and 30 with lists,
// which are checked and copied there (700 pages 211 and 229).
#include "qf_common.h"
#include "../../include/qf_prefix.h"

namespace qf {
namespace pages {

constexpr int kD = 64;
constexpr int kRowChunks = kD * 2 / 16;           // 16-byte chunks of a slot
constexpr int kThreads = 256;
constexpr int kUnroll = 4;                        // 16-byte loads in flight per thread
constexpr int kRows = kThreads / kRowChunks * kUnroll;  // slots of one workgroup: 128
constexpr int kPools = 128;                       // pool pointers in one launch's arguments

struct Args {
  f16* pool[kPools];
  int per;                   // pools from each pointer on, `step` elements apart
  int64_t step, sp, sh, sn;
  const int32_t* src;
  const int32_t* dst;
  const int32_t* slots;
  int n_pages, log2p, rows;  // rows = KVH * page_size
};

// One workgroup copies kRows consecutive (head, slot) rows of one page of one
// pool; blockIdx = (block of rows, pair, pool).
__global__ __launch_bounds__(kThreads) void copy_pages_kernel(Args a) {
  const int pair = blockIdx.y;
  const int from = a.src[pair], to = a.dst[pair];
  const int page = 1 << a.log2p;
  const int n = a.slots == nullptr ? page : min(max(a.slots[pair], 0), page);
  if (from < 0 || from >= a.n_pages || to < 0 || to >= a.n_pages || from == to) return;
  f16* pool = a.pool[blockIdx.z / a.per] + (int)(blockIdx.z % a.per) * a.step;
  const f16* s = pool + from * a.sp;
  f16* d = pool + to * a.sp;
  const int sub = threadIdx.x / kRowChunks, c = 8 * (threadIdx.x % kRowChunks);
  const int row0 = blockIdx.x * kRows + sub;
  f16x8 v[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int row = row0 + u * (kRows / kUnroll);
    const int h = row >> a.log2p, slot = row & (page - 1);
    if (row < a.rows && slot < n) v[u] = load16(s + h * a.sh + slot * a.sn + c);
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int row = row0 + u * (kRows / kUnroll);
    const int h = row >> a.log2p, slot = row & (page - 1);
    if (row < a.rows && slot < n) store16(d + h * a.sh + slot * a.sn + c, v[u]);
  }
}

}  // namespace pages
}  // namespace qf

extern "C" int qf_copy_pages(const void* const* pools, int n_pools, int per, int64_t step,
                             int64_t sp, int64_t sh, int64_t sn, const int32_t* src, const int32_t* dst,
                             const int32_t* slots, int n_pairs, int n_pages, int KVH,
                             int page_size, int D, void* stream) {
  using namespace qf;
  using namespace qf::pages;
  const int l2 = page_log2(page_size, 1, n_pages);
  if (D != kD || l2 < 0) return QF_ERR_UNSUPPORTED;
  if (!pools || n_pools < 1 || per < 1 || per > 65535 || KVH < 1 || n_pairs < 0)
    return QF_ERR_INVALID_ARG;
  if ((int64_t)KVH * page_size > 0x7fffffff - kRows) return QF_ERR_UNSUPPORTED;
  if (((step | sp | sh | sn) & 7) != 0) return QF_ERR_INVALID_ARG;
  for (int i = 0; i < n_pools; ++i)
    if (!pools[i] || (reinterpret_cast<uintptr_t>(pools[i]) & 15u)) return QF_ERR_INVALID_ARG;
  if (n_pairs == 0) return QF_OK;
  if (!src || !dst) return QF_ERR_INVALID_ARG;
  hipStream_t st = static_cast<hipStream_t>(stream);
  Args a;
  a.per = per;
  a.step = step;
  a.sp = sp; a.sh = sh; a.sn = sn;
  a.n_pages = n_pages;
  a.log2p = l2;
  a.rows = KVH * page_size;
  constexpr int kMaxPairs = 65535;  // gridDim.y
  const int bases = 65535 / per < kPools ? 65535 / per : kPools;  // gridDim.z
  for (int p0 = 0; p0 < n_pools; p0 += bases) {
    const int np = n_pools - p0 < bases ? n_pools - p0 : bases;
    for (int i = 0; i < np; ++i) a.pool[i] = static_cast<f16*>(const_cast<void*>(pools[p0 + i]));
    for (int i0 = 0; i0 < n_pairs; i0 += kMaxPairs) {
      const int n = n_pairs - i0 < kMaxPairs ? n_pairs - i0 : kMaxPairs;
      a.src = src + i0;
      a.dst = dst + i0;
      a.slots = slots ? slots + i0 : nullptr;
      hipLaunchKernelGGL(copy_pages_kernel, dim3((a.rows + kRows - 1) / kRows, n, np * per),
                         dim3(kThreads), 0, st, a);
      const int rc = (int)hipGetLastError();
      if (rc != 0) return rc;
    }
  }
  return QF_OK;
}
