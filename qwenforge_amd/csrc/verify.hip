// Verification of drafted tokens on gfx950 (include/qf_verify.h): rejection of a
// draft d ~ q against p with u q(d) < p(d) and a draw from max(p - q, 0) at the
// first rejection leave exactly p.
//
// stats_kernel reads every logit once: maximum and sum of exponentials (or the
// argmax) of each chunk of each position, in fp32.  decide_kernel, a workgroup per
// row, finds the row's first rejection from those; where an acceptance is closer
// than fp32 sums tell (2e-5 of it at 151936 logits), it takes that position's
// sum again in 64 bits.  draw_kernel, a workgroup per row and chunk of 2048 tokens,
// goes over the logits of the last position once more.  Its weights and sums are in
// 64 bits: the token drawn is where a running sum over the vocabulary crosses a
// number, and a sum off by 2^-24 would move that crossing past a token in some draws
// out of a hundred.  The workgroup that completes a row adds up its chunks and
// searches the one of the crossing.  With draft probabilities the sum of
// exponentials has to be known in 64 bits before max(p - q, 0) can be formed, so a
// first launch of the kernel takes it.
//
// MI355X, 151936 fp16 logits a position: 32 rows of 8 positions with draft
// probabilities 47.5 us in a replayed graph (fp32 logits 59).  Traced one by one,
// which adds 0.5 to 2 us to each: stats_kernel 18.2 (78 MB, 4.3 TB/s: memory; four
// groups in flight or twice the parts were slower), decide_kernel 4.8 (6 with four
// waves), the sums of exponentials 8.2, the draw 18.9 (exps in 64 bits, 29 MB, and
// the last workgroup's search, some 5 us of dependent steps).  One row of 5
// positions 14.6 us, 8 rows at temperature 0 8.5 us: the launches and each one's
// chain of dependent loads.
#include <algorithm>
#include <cmath>

#include "qf_common.h"
#include "../../include/qf_verify.h"

namespace qf {
namespace verify {

constexpr int kThreads = 256;
constexpr int kDecide = 512;               // of decide_kernel
constexpr int kGroup = 8;                  // consecutive logits of a thread
constexpr int kChunk = kThreads * kGroup;  // tokens of a draw_kernel workgroup
constexpr int kMaxParts = 64;              // chunks of a position in stats_kernel
constexpr int kMinPart = 256;              // least groups of one
// Counters of the rows, each on a 128-byte line of its own: counts of one line
// are taken one after the other, 32 rows' 2400 of them in some 20 us.
constexpr int kTicket = 32;

struct Args {
  const void* logits;
  int64_t lg_sn;
  const int64_t* tokens;
  const int32_t* cu;
  const float* accept_u;
  const float* sample_u;
  const float* probs;
  int64_t dp_sn;
  double inv_t;
  float k2;            // log2(e) / temperature
  double slack;        // sides of an acceptance that are closer than this factor are close
  int64_t* out;
  int64_t* count;
  float2* stats;       // (T, parts): max, sum (argmax: max, index)
  double2* sums;       // (B, chunks): weights left after the draft, all weights
  double* total;       // (B, chunks): sums of exponentials (draft probabilities)
  int4* rows;          // (B): first position, positions, accepted drafts, maximum there
  int32_t* ticket;     // one in every kTicket, zeroed by decide_kernel
  int width, T, B, V, parts, chunks;
};

// Eight consecutive values from element `at` of a row of n, `fill` outside it;
// 16-byte loads where all eight exist (the caller aligns `at`).
__device__ __forceinline__ void load8(const f16* row, int at, int n, float fill, float (&x)[kGroup]) {
  if (at >= 0 && at + kGroup <= n) {
    const f16x8 v = load16(row + at);
#pragma unroll
    for (int e = 0; e < kGroup; ++e) x[e] = (float)v[e];
  } else {
#pragma unroll
    for (int e = 0; e < kGroup; ++e) x[e] = at + e >= 0 && at + e < n ? (float)row[at + e] : fill;
  }
}

__device__ __forceinline__ void load8(const float* row, int at, int n, float fill, float (&x)[kGroup]) {
  if (at >= 0 && at + kGroup <= n) {
    const f32x4 a = *reinterpret_cast<const f32x4*>(row + at);
    const f32x4 b = *reinterpret_cast<const f32x4*>(row + at + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[e] = a[e];
      x[4 + e] = b[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < kGroup; ++e) x[e] = at + e >= 0 && at + e < n ? row[at + e] : fill;
  }
}

// Elements by which groups of eight start before the row, so that they start on
// 16-byte boundaries (rows of odd length start anywhere).
template <typename E>
__device__ __forceinline__ int lead(const E* row) {
  return (int)(reinterpret_cast<uintptr_t>(row) & 15u) / (int)sizeof(E);
}

// Maximum and sum of exponentials of one part of a position (kArgmax: the
// maximum and its lowest index; with a NaN, index -1 and a maximum that none
// exceeds).
template <typename E, bool kArgmax>
__global__ __launch_bounds__(kThreads) void stats_kernel(Args a) {
  __shared__ float sm[4], sl[4];
  __shared__ int si[4];
  const int part = blockIdx.x % a.parts, pos = blockIdx.x / a.parts;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const E* row = static_cast<const E*>(a.logits) + pos * a.lg_sn;
  const int before = lead(row);
  const int groups = (int)(((int64_t)a.V + before + kGroup - 1) / kGroup);
  const int per = (groups + a.parts - 1) / a.parts;
  const int end = min((part + 1) * per, groups);
  float m = kNegInf, l = 0.f;
  int at = 0x7fffffff;
  bool nan = false;
#pragma unroll 2
  for (int g = part * per + tid; g < end; g += kThreads) {
    float x[kGroup];
    const int first = g * kGroup - before;
    load8(row, first, a.V, kNegInf, x);
    if (kArgmax) {
#pragma unroll
      for (int e = 0; e < kGroup; ++e)
        if (x[e] > m) {
          m = x[e];
          at = first + e;
        }
#pragma unroll
      for (int e = 0; e < kGroup; e += 2) nan |= __builtin_isunordered(x[e], x[e + 1]);
    } else {
      float top = m;
#pragma unroll
      for (int e = 0; e < kGroup; ++e) top = fmaxf(top, x[e]);
      const float ref = top == kNegInf ? 0.f : top;
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < kGroup; ++e) s += fast_exp2((x[e] - ref) * a.k2);
      l = l * fast_exp2((m - ref) * a.k2) + s;   // m = -inf: l is 0 (or NaN and stays so)
      m = top;
    }
  }
  if (kArgmax && nan) {
    m = __builtin_huge_valf();
    at = -1;
  }
  for (int d = 32; d > 0; d >>= 1) {
    const float m2 = __shfl_xor(m, d);
    if (kArgmax) {
      const int i2 = __shfl_xor(at, d);
      if (m2 > m || (m2 == m && i2 < at)) {
        m = m2;
        at = i2;
      }
    } else {
      const float l2 = __shfl_xor(l, d);
      const float top = fmaxf(m, m2), ref = top == kNegInf ? 0.f : top;
      l = l * fast_exp2((m - ref) * a.k2) + l2 * fast_exp2((m2 - ref) * a.k2);
      m = top;
    }
  }
  if (lane == 0) {
    sm[w] = m;
    sl[w] = l;
    si[w] = at;
  }
  __syncthreads();
  if (tid != 0) return;
  for (int i = 1; i < 4; ++i) {
    if (kArgmax) {
      if (sm[i] > m || (sm[i] == m && si[i] < at)) {
        m = sm[i];
        at = si[i];
      }
    } else {
      const float top = fmaxf(m, sm[i]), ref = top == kNegInf ? 0.f : top;
      l = l * fast_exp2((m - ref) * a.k2) + sl[i] * fast_exp2((sm[i] - ref) * a.k2);
      m = top;
    }
  }
  a.stats[(int64_t)pos * a.parts + part] = float2{m, kArgmax ? __int_as_float(at) : l};
}

// A row's first position and positions, within [0, T) whatever cu holds.
__device__ __forceinline__ void row_span(const Args& a, int b, int& lo, int& n) {
  lo = min(max(a.cu[b], 0), a.T);
  const int hi = min(max(a.cu[b + 1], lo), a.T);
  n = min(hi - lo, a.width);
}

// The accepted drafts of row b, the next token (-1: none) and -1 behind.
__device__ __forceinline__ void write_row(const Args& a, int b, int lo, int taken, int64_t token) {
  for (int j = threadIdx.x; j < a.width; j += blockDim.x)
    a.out[(int64_t)b * a.width + j] = j < taken ? a.tokens[lo + j + 1] : j == taken ? token : -1;
  if (threadIdx.x == 0) a.count[b] = taken + (token >= 0 ? 1 : 0);
}

__device__ __forceinline__ float wave_max(float x) {
  for (int d = 32; d > 0; d >>= 1) x = fmaxf(x, __shfl_xor(x, d));
  return x;
}

__device__ __forceinline__ double wave_sum(double x) {
  for (int d = 32; d > 0; d >>= 1) x += __shfl_xor(x, d);
  return x;
}

// Argmax of a position from its parts (one per lane), -1 if nothing is above -inf
// or there is a NaN.
__device__ __forceinline__ int best_token(const Args& a, int pos) {
  const int lane = threadIdx.x & 63;
  const float2 x = lane < a.parts ? a.stats[(int64_t)pos * a.parts + lane]
                                  : float2{kNegInf, __int_as_float(0x7fffffff)};
  const float top = wave_max(x.x);
  int at = x.x == top ? __float_as_int(x.y) : 0x7fffffff;
  for (int d = 32; d > 0; d >>= 1) at = min(at, __shfl_xor(at, d));
  return top == kNegInf ? -1 : at;
}

// Temperature 0: one wave per row.
__global__ __launch_bounds__(64) void greedy_kernel(Args a) {
  const int b = blockIdx.x;
  int lo, n;
  row_span(a, b, lo, n);
  int taken = 0, best = -1;
  for (; taken < n; ++taken) {
    best = best_token(a, lo + taken);
    if (taken + 1 == n || best < 0 || a.tokens[lo + taken + 1] != best) break;
  }
  write_row(a, b, lo, taken, best);
}

__device__ __forceinline__ double exp_of(const Args& a, float x, float top) {
  return exp(((double)x - (double)top) * a.inv_t);
}

// Drafts of the row that are accepted: waves take the positions in turn, each
// three dependent loads.  The statistics' sum of exponentials decides where it is
// certain to (Args::slack); the few positions whose two sides are closer take
// their sum anew in 64 bits, one after the other.
template <typename E>
__global__ __launch_bounds__(kDecide) void decide_kernel(Args a) {
  constexpr int kWaves = kDecide / 64;
  __shared__ int first, close;  // refused, too close to say: the first of each
  __shared__ double part[kWaves];
  const int b = blockIdx.x, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int lo, n;
  row_span(a, b, lo, n);
  if (threadIdx.x == 0) {
    first = n - 1;
    close = n;
    a.ticket[b * kTicket] = 0;
  }
  if (n == 0) {
    if (threadIdx.x == 0) a.rows[b] = int4{lo, 0, 0, 0};
    write_row(a, b, lo, 0, -1);
    return;
  }
  __syncthreads();
  int from = 0;
  for (;;) {
    for (int j = from + w; j < n - 1; j += kWaves) {
      const int64_t pos = lo + j;
      const int64_t d = a.tokens[pos + 1];
      const bool known = d >= 0 && d < a.V;
      const float2 x = lane < a.parts ? a.stats[pos * a.parts + lane] : float2{kNegInf, 0.f};
      const float xd = known ? (float)static_cast<const E*>(a.logits)[pos * a.lg_sn + d] : kNegInf;
      const float qd = a.probs == nullptr ? 1.f : known ? a.probs[pos * a.dp_sn + d] : 0.f;
      const float top = wave_max(x.x), ref = top == kNegInf ? 0.f : top;
      // An absent part (-inf, 0) adds 0; a NaN sum stays.
      const double sum = wave_sum((double)x.y * (double)fast_exp2((x.x - ref) * a.k2));
      const bool fine = sum > 0. && sum < (double)__builtin_huge_valf();
      // u q < e / sum, both sides times the sum.
      const double e = fine && known ? exp_of(a, xd, top) : 0.;
      const double uq = (double)a.accept_u[pos] * (double)qd, lhs = uq * sum;
      if (lane == 0) {
        if (e > 0. && lhs <= e * a.slack && e <= lhs * a.slack) atomicMin(&close, j);
        else if (!(e > 0. && lhs < e)) atomicMin(&first, j);
      }
    }
    __syncthreads();
    const int j = close;
    if (j >= first) break;
    const int64_t pos = lo + j, d = a.tokens[pos + 1];
    const E* row = static_cast<const E*>(a.logits) + pos * a.lg_sn;
    const float top = wave_max(lane < a.parts ? a.stats[pos * a.parts + lane].x : kNegInf);
    double s = 0.;
    for (int i = threadIdx.x; i < a.V; i += kDecide) s += exp_of(a, (float)row[i], top);
    s = wave_sum(s);
    if (lane == 0) part[w] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
      double sum = 0.;
      for (int i = 0; i < kWaves; ++i) sum += part[i];
      const float qd = a.probs == nullptr ? 1.f : a.probs[pos * a.dp_sn + d];
      if (!((double)a.accept_u[pos] * (double)qd < exp_of(a, (float)row[d], top) / sum)) first = j;
      close = n;
    }
    __syncthreads();
    from = j + 1;  // once one is refused, no position from here on comes before it
  }
  if (w != 0) return;
  const int taken = first;
  const float top = wave_max(lane < a.parts ? a.stats[(int64_t)(lo + taken) * a.parts + lane].x : kNegInf);
  if (lane == 0) a.rows[b] = int4{lo, n, taken, __float_as_int(top)};
}

// x of another lane by a DPP move, 0 where the move names none.
template <int kCtrl, int kRowMask>
__device__ __forceinline__ double dpp(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const unsigned lo = __builtin_amdgcn_update_dpp(0, (int)u, kCtrl, kRowMask, 0xF, true);
  const unsigned hi = __builtin_amdgcn_update_dpp(0, (int)(u >> 32), kCtrl, kRowMask, 0xF, true);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// Inclusive sums over the lanes of a wave: within rows of 16 lanes, then across
// them (a lane that a move leaves out adds 0).
__device__ __forceinline__ double wave_scan(double x) {
  x += dpp<0x111, 0xF>(x);  // row_shr:1
  x += dpp<0x112, 0xF>(x);  // row_shr:2
  x += dpp<0x114, 0xF>(x);  // row_shr:4
  x += dpp<0x118, 0xF>(x);  // row_shr:8
  x += dpp<0x142, 0xA>(x);  // row_bcast:15 into rows 1 and 3
  x += dpp<0x143, 0xC>(x);  // row_bcast:31 into rows 2 and 3
  return x;
}

// Inclusive sums over the workgroup's threads; `all` their total.  `part` is this
// call's own.
__device__ __forceinline__ double block_scan(double x, double (&part)[4], double& all) {
  const int w = threadIdx.x >> 6;
  x = wave_scan(x);
  if ((threadIdx.x & 63) == 63) part[w] = x;
  __syncthreads();
  double ahead = 0.;
  all = 0.;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (i < w) ahead += part[i];
    all += part[i];
  }
  return ahead + x;
}

// The first thread with `hit`, or the last one with `some`, or -1.  `at` is this
// call's own.
__device__ __forceinline__ int find_thread(bool hit, bool some, int2 (&at)[4]) {
  const uint64_t h = __ballot(hit), m = __ballot(some);
  if ((threadIdx.x & 63) == 0)
    at[threadIdx.x >> 6] = int2{h ? __builtin_ctzll(h) : -1, m ? 63 - __builtin_clzll(m) : -1};
  __syncthreads();
  int last = -1;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (at[i].x >= 0) return 64 * i + at[i].x;
    if (at[i].y >= 0) last = 64 * i + at[i].y;
  }
  return last;
}

// kTotal: only the sums of exponentials of the drawn position.  Else its
// weights, and the draw by the row's last workgroup.
template <typename E, bool kTotal>
__global__ __launch_bounds__(kThreads) void draw_kernel(Args a) {
  __shared__ double part[5][4];
  __shared__ int2 at[2][4];
  __shared__ int found_chunk, token;
  __shared__ double found_ahead;
  __shared__ bool mine;
  const int b = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
  const int tid = threadIdx.x;
  const int4 r = a.rows[b];
  if (r.y == 0) return;
  const int taken = r.z;
  const float top = __int_as_float(r.w);
  const int64_t pos = r.x + taken;
  const E* row = static_cast<const E*>(a.logits) + pos * a.lg_sn;
  const bool refused = taken < r.y - 1;
  if (kTotal && !refused) return;
  const int64_t draft = refused && a.probs == nullptr ? a.tokens[pos + 1] : -1;
  const float* q = refused && a.probs != nullptr ? a.probs + pos * a.dp_sn : nullptr;
  const int before = lead(row);
  double sum_exp = 0.;
  if (!kTotal && q != nullptr) {
    double s = 0.;
    for (int i = tid; i < a.chunks; i += kThreads) s += a.total[(int64_t)b * a.chunks + i];
    block_scan(s, part[0], sum_exp);
  }
  // Weights of this thread's eight tokens of chunk c: left after the draft, all.
  const auto weights = [&](int c, double (&left)[kGroup], double (&all)[kGroup]) {
    const int start = c * kChunk + tid * kGroup - before;
    float x[kGroup], y[kGroup];
    load8(row, start, a.V, kNegInf, x);
    if (q != nullptr) {
      // Aligned like the logits only if the rows are.
      if ((reinterpret_cast<uintptr_t>(q + start) & 15u) == 0) load8(q, start, a.V, 0.f, y);
      else
#pragma unroll
        for (int e = 0; e < kGroup; ++e) y[e] = start + e >= 0 && start + e < a.V ? q[start + e] : 0.f;
    }
#pragma unroll
    for (int e = 0; e < kGroup; ++e) {
      const int i = start + e;
      all[e] = i >= 0 && i < a.V ? exp_of(a, x[e], top) : 0.;
      left[e] = all[e];
      if (q != nullptr) left[e] = fmax(all[e] - (double)y[e] * sum_exp, 0.);
      if (i == draft) left[e] *= 0.;  // a NaN stays: no distribution, nothing drawn
    }
  };
  double left[kGroup], all[kGroup], sl = 0., sa = 0.;
  weights(chunk, left, all);
#pragma unroll
  for (int e = 0; e < kGroup; ++e) {
    sl += left[e];
    sa += all[e];
  }
  double chunk_left, chunk_all;
  block_scan(sa, part[1], chunk_all);
  if (kTotal) {
    if (tid == 0) a.total[(int64_t)b * a.chunks + chunk] = chunk_all;
    return;
  }
  block_scan(sl, part[2], chunk_left);
  if (tid == 0) {
    double2* s = a.sums + (int64_t)b * a.chunks + chunk;
    __hip_atomic_store(&s->x, chunk_left, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store(&s->y, chunk_all, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    // The sums go past the L2 (agent-scope accesses) and have arrived before the
    // count; their readers use such accesses too.  No fence: releasing every
    // workgroup's L2 took four times the rest of the kernel.
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    s_waitcnt_vm(0);
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    mine = __hip_atomic_fetch_add(&a.ticket[b * kTicket], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
           a.chunks - 1;
  }
  __syncthreads();
  if (!mine) return;
  // The chunk of the crossing: a thread adds up `per` neighbouring chunks, the
  // thread of the crossing walks them.
  const int per = (a.chunks + kThreads - 1) / kThreads;
  const auto chunk_sum = [&](int c, bool use_left) {
    double2* s = a.sums + (int64_t)b * a.chunks + c;
    return __hip_atomic_load(use_left ? &s->x : &s->y, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  };
  bool use_left = true;
  double total, s, upto;
  for (int pass = 0;; ++pass) {
    s = 0.;
    for (int c = tid * per; c < min((tid + 1) * per, a.chunks); ++c) s += chunk_sum(c, use_left);
    upto = block_scan(s, part[3 + pass], total);
    if (total > 0. && total < (double)__builtin_huge_val()) break;
    if (pass == 1) {
      write_row(a, b, r.x, taken, -1);
      return;
    }
    use_left = false;  // nothing left after the draft: from all of p
  }
  const double mark = (double)a.sample_u[b] * total;
  if (tid == find_thread(upto > mark && s > 0., s > 0., at[0])) {
    double ahead = upto - s, passed = 0.;
    // One chunk to a thread: no second trip to memory for it.
    if (per == 1) found_chunk = tid;
    else for (int c = tid * per; c < min((tid + 1) * per, a.chunks); ++c) {
      const double here = chunk_sum(c, use_left);
      if (!(here > 0.)) continue;
      ahead += passed;
      passed = here;
      found_chunk = c;
      if (ahead + here > mark) break;
    }
    found_ahead = ahead;
  }
  __syncthreads();
  const int found = found_chunk;
  weights(found, left, all);
  s = 0.;
#pragma unroll
  for (int e = 0; e < kGroup; ++e) s += use_left ? left[e] : all[e];
  double whole;
  upto = found_ahead + block_scan(s, part[1], whole);
  if (tid == find_thread(upto > mark && s > 0., s > 0., at[1])) {
    double sum = upto - s;
    int here = -1;
    bool crossed = false;
#pragma unroll
    for (int e = 0; e < kGroup; ++e) {
      const double w = use_left ? left[e] : all[e];
      sum += w;
      if (!crossed && w > 0.) {
        here = found * kChunk + tid * kGroup - before + e;
        crossed = sum > mark;
      }
    }
    token = here;
  }
  __syncthreads();
  write_row(a, b, r.x, taken, token);
}

int parts_of(int T, int V) {
  const int64_t groups = ((int64_t)V + kGroup - 1) / kGroup;
  const int64_t by_len = (groups + kMinPart - 1) / kMinPart;
  return (int)std::max<int64_t>(1, std::min<int64_t>({by_len, kMaxParts, 2048 / T}));
}

// By which factor the two sides of an acceptance have to be apart for the fp32 sums to
// say which is larger; u = 2^-24.  An exponential's argument of -a log2 units comes of
// three roundings, 3 u a ln 2 of its value, and the weighted mean of a is at most
// log2 V < 31: 65 u of the sum.  The exponential and a thread's eight terms are 9
// more; each of the nine joins of threads and waves, the join of parts and each
// further group of a thread 4 (exponential, product, sum).  That is less than x =
// (128 + 4 groups) u, and 1 / (1 - x) < 1 + 2.5 x below 0.1; from there on every
// position is looked at again.
double slack_of(int V, int parts) {
  const int64_t groups = ((int64_t)V + 2 * kGroup - 1) / kGroup;
  const int64_t per = (groups + parts - 1) / parts;
  const double x = (128. + 4. * (double)((per + kThreads - 1) / kThreads)) * 0x1p-24;
  return x < 0.1 ? 1. + 2.5 * x : HUGE_VAL;
}

// With the elements that groups may start before the row.
int chunks_of(int V) { return (int)(((int64_t)V + kGroup - 1 + kChunk - 1) / kChunk); }

int64_t round16(int64_t x) { return (x + 15) / 16 * 16; }

}  // namespace verify
}  // namespace qf

extern "C" int64_t qf_verify_workspace(int T, int B, int V) {
  using namespace qf::verify;
  if (T < 1 || B < 1 || V < 1) return QF_ERR_INVALID_ARG;
  if (V > 0x7fffffff - 2 * kChunk || (int64_t)T * kMaxParts > 0x7fffffff ||
      (int64_t)B * chunks_of(V) > 0x7fffffff || B > 0x7fffffff / kTicket)
    return QF_ERR_UNSUPPORTED;
  const int64_t sums = (int64_t)B * chunks_of(V);
  return round16((int64_t)T * parts_of(T, V) * 8) + sums * 16 + round16(sums * 8) +
         (int64_t)B * (16 + 4 * kTicket);
}

namespace qf {
namespace verify {

template <typename E>
int launch(const Args& a, bool greedy, hipStream_t st) {
  const dim3 all((unsigned)(a.T * a.parts)), block(kThreads);
  if (greedy) {
    hipLaunchKernelGGL((stats_kernel<E, true>), all, block, 0, st, a);
    hipLaunchKernelGGL(greedy_kernel, dim3(a.B), dim3(64), 0, st, a);
    return (int)hipGetLastError();
  }
  hipLaunchKernelGGL((stats_kernel<E, false>), all, block, 0, st, a);
  hipLaunchKernelGGL(decide_kernel<E>, dim3(a.B), dim3(kDecide), 0, st, a);
  const dim3 draw((unsigned)(a.B * a.chunks));
  if (a.probs != nullptr) hipLaunchKernelGGL((draw_kernel<E, true>), draw, block, 0, st, a);
  hipLaunchKernelGGL((draw_kernel<E, false>), draw, block, 0, st, a);
  return (int)hipGetLastError();
}

}  // namespace verify
}  // namespace qf

extern "C" int qf_verify_drafts(const void* logits, int dtype, int64_t lg_sn, const int64_t* tokens,
                                const int32_t* cu_seqlens, const float* accept_u,
                                const float* sample_u, const float* draft_probs, int64_t dp_sn,
                                double temperature, int64_t* out, int width, int64_t* count, void* ws,
                                int64_t ws_bytes, int T, int B, int V, void* stream) {
  using namespace qf;
  using namespace qf::verify;
  const int64_t need = qf_verify_workspace(T, B, V);
  if (need < 0) return (int)need;
  const bool greedy = temperature == 0.;
  if (dtype != QF_F16 && dtype != QF_F32) return QF_ERR_UNSUPPORTED;
  if (!logits || !tokens || !cu_seqlens || !out || !count || !ws || width < 1 || lg_sn < V ||
      !(temperature >= 0.) || !std::isfinite(temperature))
    return QF_ERR_INVALID_ARG;
  // Past the normal fp32 numbers a masked logit times k2 would be no number.
  const float k2 = greedy ? 0.f : (float)(1.4426950408889634 / temperature);
  if (!greedy && (!accept_u || !sample_u || (draft_probs != nullptr && dp_sn < V) || !std::isnormal(k2)))
    return QF_ERR_INVALID_ARG;
  if ((reinterpret_cast<uintptr_t>(logits) & (dtype == QF_F16 ? 1u : 3u)) != 0 ||
      (reinterpret_cast<uintptr_t>(ws) & 15u) != 0)
    return QF_ERR_INVALID_ARG;
  if (ws_bytes < need) return QF_ERR_SCRATCH_LIMIT;
  Args a = {};
  a.logits = logits;
  a.lg_sn = lg_sn;
  a.tokens = tokens;
  a.cu = cu_seqlens;
  a.accept_u = accept_u;
  a.sample_u = sample_u;
  a.probs = greedy ? nullptr : draft_probs;
  a.dp_sn = dp_sn;
  a.inv_t = greedy ? 0. : 1. / temperature;
  a.k2 = k2;
  a.out = out;
  a.count = count;
  a.width = width;
  a.T = T; a.B = B; a.V = V;
  a.parts = parts_of(T, V);
  a.slack = slack_of(V, a.parts);
  a.chunks = chunks_of(V);
  unsigned char* p = static_cast<unsigned char*>(ws);
  const int64_t sums = (int64_t)B * a.chunks;
  a.sums = reinterpret_cast<double2*>(p);
  p += sums * 16;
  a.stats = reinterpret_cast<float2*>(p);
  p += verify::round16((int64_t)T * a.parts * 8);
  a.total = reinterpret_cast<double*>(p);
  p += verify::round16(sums * 8);
  a.rows = reinterpret_cast<int4*>(p);
  a.ticket = reinterpret_cast<int32_t*>(p + (int64_t)B * 16);
  hipStream_t st = static_cast<hipStream_t>(stream);
  return dtype == QF_F16 ? launch<f16>(a, greedy, st) : launch<float>(a, greedy, st);
}
