// The walk of every workgroup of a long extension in even pieces (csrc/kv8_pieces.h), on the
// host: pieces, units, slots, partials and joins that any offsets and contexts give, and
// where they would lie.  Prints what is out of range and returns 1, or "ok" and the cases.
#define QF_HD inline
#include "../qwenforge_amd/csrc/kv8_pieces.h"

#include <algorithm>
#include <cstdio>
#include <random>
#include <vector>

using namespace qf::kv8;

struct Call {
  int G, kvh, tokens, longest, cap, shift, pieces;
  std::vector<int> cu;
  std::vector<int64_t> ctx;
  bool apart;   // rows that do not overlap: nothing may be left out
};

static bool fail(const char* what, long a, long b) {
  std::printf("%s %ld %ld\n", what, a, b);
  return false;
}

// As the launch chooses it; < 0: not in pieces.
static int choose_shift(const Call& c) {
  const int64_t B = (int64_t)c.ctx.size(), rows = (int64_t)c.longest * c.G;
  const int64_t units = c.kvh * std::min<int64_t>(B * ((rows + 127) / 128), (int64_t)c.tokens * c.G / 128 + B);
  for (int s = 0; s < 20; ++s)
    if (most_cost(units, c.G, c.cap, c.longest, s) < 1 << 30) return s;
  return -1;
}

static bool walk(const Call& c) {
  const int B = (int)c.ctx.size();
  const auto row = [&](int r) {
    return row_units(c.cu[r], c.cu[r + 1], c.ctx[r], c.G, c.tokens, c.longest, c.cap, c.shift);
  };
  std::vector<RowUnits> w(B);
  std::vector<int> before(B + 1, 0);
  int64_t exact = 0;
  for (int r = 0; r < B; ++r) {
    w[r] = row(r);
    const int mine = cost_before(w[r], w[r].n) * c.kvh;
    if (mine < 0 || mine > kMostWork) return fail("row", r, mine);
    before[r + 1] = add_capped(before[r], mine);
    exact += mine;
  }
  const int work = line_length(before[B]);
  if (c.apart && exact != work) return fail("work", exact, work);
  const int len = piece_length(work, c.pieces, c.G, c.shift);
  if (len < 1) return fail("length", work, len);
  std::vector<char> there(c.pieces, 0);
  for (int b = 0; b < c.pieces; ++b) {
    const int piece = piece_of(b, c.pieces, work, len);
    if (piece < 0 || piece >= c.pieces || there[piece]++) return fail("piece", b, piece);
    const int x = piece * len, end = std::min(x + len, work);
    if (x >= work) continue;
    int r = 0;
    while (r < B && !(x < before[r + 1])) ++r;
    if (r == B) return fail("no row", piece, x);
    const int one = cost_before(w[r], w[r].n);
    if (one <= 0) return fail("empty row", r, one);
    int base = before[r + 1] - one * c.kvh;
    if (base < 0 || base > x) return fail("base", base, x);
    int hk = (int)std::min((unsigned)(x - base) / (unsigned)one, (unsigned)c.kvh - 1u);
    base += hk * one;
    int q = unit_at(w[r], x - base), x0 = base + cost_before(w[r], q), x1 = x0 + w[r].first + w[r].step * q;
    int seen = slots_seen(w[r], q, c.G, c.cap), k0 = cut_slot(x - x0, seen, c.G, c.shift);
    if (k0 > 0 && k0 < seen && (x - len < x0 || cut_slot(x - len - x0, seen, c.G, c.shift) == 0)) {
      int more = 1;
      for (int64_t y = (int64_t)x + len; more < c.pieces - piece && y < x1 &&
                                         cut_slot((int)(y - x0), seen, c.G, c.shift) < seen; y += len) ++more;
      if (piece < 1 || 2 * (piece + more - 1) >= 2 * c.pieces) return fail("join", piece, more);
    }
    for (;;) {
      if (hk < 0 || hk >= c.kvh || q < 0 || q >= w[r].n) return fail("unit", hk, q);
      if (seen < 0 || seen > c.cap) return fail("seen", seen, c.cap);
      if (w[r].tok0 < 0 || w[r].tok0 + w[r].rows / c.G > c.tokens || q * kUnitRows >= w[r].rows)
        return fail("tokens", w[r].tok0, w[r].rows);
      const int k1 = end >= x1 ? seen : cut_slot(end - x0, seen, c.G, c.shift);
      if (k0 < 0 || k1 < 0 || k0 > seen || k1 > seen) return fail("slots", k0, k1);
      if (x1 <= x0) return fail("line", x0, x1);
      if (x1 >= end) break;
      if (++q >= w[r].n) {
        q = 0;
        if (++hk >= c.kvh) {
          hk = 0;
          do ++r; while (r < B && w[r].n == 0);
          if (r == B) {
            if (c.apart) return fail("line's end", piece, x1);
            break;
          }
        }
      }
      k0 = 0;
      x0 = x1;
      x1 = x0 + w[r].first + w[r].step * q;
      seen = slots_seen(w[r], q, c.G, c.cap);
    }
  }
  return true;
}

int main() {
  // 64 rows of all tokens or none, behind 130000 slots: 2.2e9 in all.
  Call c{16, 2, 8192, 8192, 131072, 0, 768, {}, {}, false};
  for (int r = 0; r <= 64; ++r) c.cu.push_back(r % 2 ? 8192 : 0);
  for (int r = 0; r < 64; ++r) c.ctx.push_back(130000);
  c.shift = choose_shift(c);
  if (c.shift != 0 || !walk(c)) return 1;
  std::mt19937_64 g(17);
  const auto rnd = [&](int64_t lo, int64_t hi) { return lo + (int64_t)(g() % (uint64_t)(hi - lo + 1)); };
  int cases = 1, capped = 0;
  for (int it = 0; it < 1500; ++it) {
    const int B = (int)rnd(1, it % 3 ? 12 : 200);
    c.G = (int)rnd(1, 16);
    c.kvh = (int)rnd(1, 8);
    c.tokens = (int)rnd(1, it % 2 ? 9000 : 900);
    c.cap = (int)rnd(c.tokens, it % 5 ? 200000 : 2000000);
    c.apart = it % 4 == 0;
    c.cu.assign(B + 1, 0);
    c.ctx.assign(B, 0);
    const int64_t wild[] = {0, 1, c.tokens, 2147483647, -2147483647 - 1, -4, 100, c.tokens / 2};
    const int64_t far[] = {INT64_MAX, INT64_MIN, (1ll << 40) + 5, 1ll << 31, c.cap, 100, 0, -1};
    for (int r = 1; r <= B; ++r)
      c.cu[r] = (int)(c.apart ? c.tokens * (int64_t)r / B
                      : it % 4 == 1 ? (r % 2 ? c.tokens : 0)
                      : rnd(0, 1) ? wild[rnd(0, 7)] : rnd(0, c.tokens));
    for (auto& x : c.ctx) x = it % 3 == 1 ? rnd(c.cap / 2, c.cap) : rnd(0, 2) ? rnd(-1, c.cap) : far[rnd(0, 7)];
    c.longest = it % 4 == 2 ? (int)rnd(1, c.tokens) : c.tokens;
    c.shift = choose_shift(c);
    if (c.shift < 0) continue;
    ++cases;
    int64_t sum = 0;
    for (int r = 0; r < B; ++r) {
      const RowUnits u = row_units(c.cu[r], c.cu[r + 1], c.ctx[r], c.G, c.tokens, c.longest, c.cap, c.shift);
      sum += (int64_t)cost_before(u, u.n) * c.kvh;
    }
    capped += sum > kMostWork;
    if (!walk(c)) {
      std::printf("case %d\n", it);
      return 1;
    }
  }
  std::printf("ok %d cases, %d past the line\n", cases, capped);
  return capped > 50 ? 0 : 1;
}
