// A long extension's work in even pieces (gfx950).
//
// A unit is 128 query rows of a row and kv head and the slots that they see.  Units come
// in a line -- by row, kv head, query rows -- and each takes as much of it as it costs; the
// line is cut into pieces of one length, a workgroup for each.  What a workgroup has may
// begin and end inside units: those are joined from partials.  Every workgroup finds its
// piece from the rows' lengths by itself, and all find the same cuts, which depend on
// where the line is cut alone.
//
// Costs are counted in quanta of 64 << shift slots, over G: 32 bits hold them, as
// 64-bit products, comparisons and divisions would take longer than short pieces.
#pragma once

#include <cstdint>

#ifndef QF_HD
#define QF_HD __host__ __device__ __forceinline__
#endif

namespace qf {
namespace kv8 {

constexpr int kUnitRows = 128;
constexpr int kUnitTiles = 2;      // what a unit's beginning and end cost, in tiles of 64 slots
constexpr int kLeastCut = 4 * 64;  // slots on either side of a cut
constexpr int kLeastTiles = 8;     // of a piece
constexpr int kMostWork = (1 << 30) - 1;   // of a call's line

// A sum of what is not negative, held at the largest int.  Offsets of rows are read on the
// device, and those that overlap give sums that no check on the host bounds: one that
// wrapped would make places out of range.
QF_HD int add_capped(int a, int b) {
  const unsigned s = (unsigned)a + (unsigned)b;
  return (int)(s < 0x7fffffffu ? s : 0x7fffffffu);
}

// A row's units: unit q of a kv head costs first + 2 q (its newest token is number
// 128 (q + 1) / G or so).
struct RowUnits {
  int tok0, rows, ctx, n;          // first token, query rows of a kv head, cached slots, units
  int first, step;
};

QF_HD RowUnits row_units(int lo, int hi, int64_t ctx, int G, int tokens, int longest, int cap, int shift) {
  RowUnits r;
  lo = lo < 0 ? 0 : lo > tokens ? tokens : lo;
  hi = hi < lo ? lo : hi > tokens ? tokens : hi;
  const int n = hi - lo < longest ? hi - lo : longest;
  r.tok0 = lo;
  r.rows = n * G;
  r.n = (r.rows + kUnitRows - 1) / kUnitRows;
  r.ctx = (int)(ctx < 0 ? -1 : ctx > cap ? cap : ctx);
  r.first = r.ctx < 0 ? kUnitTiles * G : G * ((r.ctx >> (6 + shift)) + kUnitTiles) + 2;
  r.step = r.ctx < 0 || shift > 0 ? 0 : 2;
  return r;
}

// Units before the q-th.
QF_HD int cost_before(const RowUnits& r, int q) { return r.first * q + (r.step >> 1) * q * (q - 1); }

// More than all units of a call can cost.
QF_HD int64_t most_cost(int64_t units, int G, int64_t cap, int64_t longest, int shift) {
  return units * (G * ((cap >> (6 + shift)) + kUnitTiles) + 2 + (shift > 0 ? 0 : longest * G / 64));
}

// Slots that unit q sees.
QF_HD int slots_seen(const RowUnits& r, int q, int G, int cap) {
  if (r.ctx < 0) return 0;
  const int end = (q + 1) * kUnitRows < r.rows ? (q + 1) * kUnitRows : r.rows;
  const int new_slots = (end - 1) / G + 1;
  return new_slots < cap - r.ctx ? r.ctx + new_slots : cap;
}

// The slot at which a cut of the line `off` behind a unit's beginning cuts the unit: 0 or
// `seen` where it leaves it whole.
QF_HD int cut_slot(int off, int seen, int G, int shift) {
  const int quanta = off / G - kUnitTiles;
  if (quanta <= 0) return 0;
  if (quanta >= seen >> (6 + shift)) return seen;
  const int s = quanta << (6 + shift);
  return s < kLeastCut ? 0 : seen - s < kLeastCut ? seen : s;
}

// The line of a call whose units cost `sum` (add_capped).  Rows that do not overlap cost no
// more than kMostWork; of others what lies past it is left out.
QF_HD int line_length(int sum) { return sum < kMostWork ? sum : kMostWork; }

QF_HD int piece_length(int work, int pieces, int G, int shift) {
  const int even = (int)((unsigned)(work + pieces - 1) / (unsigned)pieces);
  const int least = shift > 0 ? G : kLeastTiles * G;
  return even > least ? even : least;
}

// The piece of a workgroup, `pieces` being a multiple of 8: neighbouring pieces share an XCD
// (workgroups go to the XCDs in turn) and its L2; those that have work are spread over all XCDs.
QF_HD int piece_of(int workgroup, int pieces, int work, int len) {
  const int eighth = (int)((unsigned)((work + len - 1) / len + 7) / 8u), nth = workgroup / 8;
  return nth < eighth ? workgroup % 8 * eighth + nth
                      : 8 * eighth + workgroup % 8 * (pieces / 8 - eighth) + nth - eighth;
}

// The unit of a row's kv head that has `x` of its line.
QF_HD int unit_at(const RowUnits& r, int x) {
  int lo = 0, hi = r.n;
  while (lo + 1 < hi) {
    const int mid = lo + (hi - lo) / 2;
    if (cost_before(r, mid) <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

}  // namespace kv8
}  // namespace qf
