// Host-side check of the places of block lists and of the shares of an attention over
// them (lvsa_paged.h), over random batches, half of them with garbage for row ranges:
//   - p / Divisor is the exact quotient for every p below 2^31;
//   - a tile's list lies among the batch's, no two tiles have the same one, and the rows
//     of a tile are its sequence's, whatever the device arrays hold;
//   - the work-groups' shares (share_of over a grid rounded up to the XCDs) cover every
//     step of every row tile once, partials go to slots of their own, and decode_slots
//     finds exactly those of a row tile.
// Prints "paged lists ok" and exits 0, or names the first failure.
#include "lvsa_paged.h"

#include <cstdio>
#include <map>
#include <random>
#include <set>
#include <vector>

using namespace lvsa;

#define CHECK(cond, ...)                              \
  do {                                                \
    if (!(cond)) {                                    \
      printf("trial %d: %s: ", trial, #cond);         \
      printf(__VA_ARGS__);                            \
      printf("\n");                                   \
      return 1;                                       \
    }                                                 \
  } while (0)

int main() {
  std::mt19937_64 rng(11);
  auto upto = [&](int64_t n) { return (int64_t)(rng() % (uint64_t)(n + 1)); };
  for (int trial = 0; trial < 20000; ++trial) {
    const int by = trial < 3000 ? 1 + trial : (int)(1 + upto(trial % 2 ? 100000 : INT32_MAX - 1));
    const Divisor d = divisor(by);
    for (int k = 0; k < 20; ++k) {
      int64_t p = upto(INT32_MAX);
      if (k % 2) p = p / by * by - (k % 4 == 1);
      if (p < 0) p = 0;
      CHECK((int)p / d == p / by, "%lld / %d = %d", (long long)p, by, (int)p / d);
    }
  }
  for (int trial = 0; trial < 20000; ++trial) {
    const bool garbage = trial % 2;
    PagedView c{};
    set_page_size(&c, 16);
    c.max_pages = 8;
    c.B = (int)upto(trial % 5 ? 7 : 150);
    c.N = (int)upto(trial % 7 ? 300 : 5);
    std::vector<int32_t> cu(c.B + 1), lens(c.B);
    for (int b = 0; b < c.B; ++b) lens[b] = (int32_t)upto(128);
    for (int b = 1; b <= c.B; ++b) cu[b] = (int32_t)(cu[b - 1] + upto(c.N) / (c.B + 1));
    if (trial % 4 == 2)
      for (auto& x : cu) x += (int32_t)upto(c.N > cu[c.B] ? (c.N - cu[c.B]) / 2 : 0), x = x > c.N ? c.N : x;
    bool valid = true;
    for (int b = 0; b < c.B; ++b) valid = valid && cu[b] <= cu[b + 1];
    if (garbage)
      for (auto& x : cu) x = upto(2) ? x : (int32_t)(uint32_t)rng();
    c.cu = cu.data();
    c.lens = lens.data();
    ListView v{};
    v.tile = divisor(trial % 3 ? (int)(1 + upto(40)) : trial % 2 ? 1 : (int)(1 + upto(INT32_MAX - 1)));
    v.lists = v.tile.by == 1 ? c.N : c.N / v.tile.by + c.B;
    std::set<int64_t> seen;
    for (int s = 0; s < c.B; ++s) {
      const PagedSeq q = paged_seq(c, s);
      CHECK(q.t0 >= 0 && q.n >= 0 && (q.n == 0 || q.t0 + q.n <= c.N), "rows %d + %d of %d", q.t0, q.n, c.N);
      const int n = list_count(v, q);
      for (int i = 0; i < n; ++i) {
        const int64_t li = first_list(v, s, q) + i;
        const int i0 = i * v.tile.by, i1 = tile_end(v, q, i0);
        CHECK(i0 >= 0 && i0 < i1 && i1 <= q.n && i1 - i0 <= v.tile.by, "tile %d: rows %d .. %d of %d", i, i0, i1, q.n);
        if (i) CHECK(tile_end(v, q, i0 - v.tile.by) == i0, "tile %d does not start where the one before ends", i);
        if (garbage || !valid) continue;
        CHECK(li >= 0 && li < v.lists, "list %lld of %d", (long long)li, v.lists);
        CHECK(seen.insert(li).second, "list %lld twice", (long long)li);
      }
      if (n) CHECK(tile_end(v, q, (n - 1) * v.tile.by) == q.n, "rows behind the last tile");
    }
  }
  for (int trial = 0; trial < 3000; ++trial) {
    const int64_t units = 1 + upto(trial % 3 ? 40 : 700);
    const int steps = (int)(1 + upto(30));
    const int64_t work = units * steps;
    const int most = (int)(1 + upto(900));
    const int grid = trial % 4 ? (int)(work < most ? work : most) : (int)units;
    std::vector<int> done((size_t)work);
    std::map<int64_t, std::vector<int64_t>> slots;      // of a unit, in the order of its steps
    std::set<int64_t> used;
    std::map<int64_t, std::map<int64_t, int64_t>> by_step;
    std::set<int> shares;
    for (int wg = 0; wg < 8 * ((grid + 7) / 8); ++wg) {
      const int share = share_of(wg, grid);
      if (share < 0) continue;
      CHECK(share < grid && shares.insert(share).second, "share %d", share);
      const int64_t first = unit_start(work, grid, share), end = unit_start(work, grid, share + 1);
      for (int64_t w = first; w < end;) {
        const int64_t unit = quotient(w, steps), w0 = unit * steps;
        const int s0 = (int)(w - w0), s1 = end - w0 < steps ? (int)(end - w0) : steps;
        for (int s = s0; s < s1; ++s) ++done[(size_t)(w0 + s)];
        if (s0 != 0 || s1 != steps) {
          const int64_t slot = 2 * (int64_t)share + (first < w0 ? 1 : 0);
          CHECK(used.insert(slot).second && slot < 2 * (int64_t)grid, "slot %lld", (long long)slot);
          by_step[unit][s0] = slot;
        }
        w = w0 + s1;
      }
    }
    CHECK((int)shares.size() == grid, "%zu of %d shares", shares.size(), grid);
    for (int x : done) CHECK(x == 1, "a step is done %d times", x);
    for (int64_t u = 0; u < units; ++u) {
      const DecodeSlots d = decode_slots(work, grid, u * steps, steps);
      CHECK(d.count == (int)by_step[u].size(), "unit %lld: %d partials, %zu written", (long long)u, d.count, by_step[u].size());
      int i = 0;
      for (auto& x : by_step[u]) {
        CHECK(x.second == (i == 0 ? d.first : d.rest + 2 * i), "unit %lld, partial %d", (long long)u, i);
        ++i;
      }
    }
  }
  printf("paged lists ok\n");
  return 0;
}
