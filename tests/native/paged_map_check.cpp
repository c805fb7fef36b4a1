// Host-side check of the paged cache's lookups and of the decode kernel's work
// shares (lvsa_paged.h), over random batches and over batches whose lengths,
// row ranges and page numbers are garbage:
//   - page_of is the exact quotient for every position below 2^31;
//   - no row, page-table entry or page outside what the caller allocated is
//     named, whatever the device arrays hold;
//   - the work-groups' shares cover every unit once, partial sums go to slots
//     of their own, and decode_slots finds exactly those of a row tile;
//   - quotient is the quotient.
// Prints "paged map ok" and exits 0, or names the first failure.
#include "lvsa_paged.h"

#include <cstdio>
#include <map>
#include <random>
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
  std::mt19937_64 rng(7);
  auto upto = [&](int64_t n) { return (int64_t)(rng() % (uint64_t)(n + 1)); };
  for (int trial = 0; trial < 20000; ++trial) {
    PagedView v{};
    set_page_size(&v, trial < 5000 ? 1 + trial : (int)(1 + upto(trial % 2 ? 5000 : INT32_MAX - 2)));
    const int64_t d = v.page_size;
    for (int k = 0; k < 40; ++k) {
      int64_t pos = upto(INT32_MAX);
      if (k % 2) pos = pos / d * d - (k % 4 == 1);       // around multiples
      if (pos < 0) pos = 0;
      CHECK(page_of(v, (int)pos) == pos / d, "%lld / %lld = %d", (long long)pos, (long long)d, page_of(v, (int)pos));
    }
  }
  for (int trial = 0; trial < 20000; ++trial) {
    const bool garbage = trial % 2;
    PagedAttnParams p{};
    PagedView& c = p.c;
    set_page_size(&c, (int)(1 + upto(trial % 3 ? 40 : 2000)));
    c.n_pages = (int)(1 + upto(50));
    c.max_pages = (int)upto(30);
    c.B = (int)upto(trial % 5 ? 6 : 150);
    c.N = (int)upto(200);
    c.Hkv = (int)(1 + upto(5));
    p.group = (int)(1 + upto(8));
    std::vector<int32_t> cu(c.B + 1), lens(c.B), table((size_t)c.B * c.max_pages + 1);
    const int64_t cap = (int64_t)c.max_pages * c.page_size;
    auto junk = [&]() { return (int32_t)(uint32_t)(upto(3) ? rng() : rng() % 300); };
    for (int b = 0; b < c.B; ++b) lens[b] = garbage && upto(1) ? junk() : (int32_t)upto(cap);
    for (int b = 1; b <= c.B; ++b) cu[b] = garbage && upto(1) ? junk() : (int32_t)(cu[b - 1] + upto(c.N) / (c.B + 1));
    if (garbage && upto(1)) cu[0] = junk();
    for (auto& x : table) x = garbage && upto(1) ? junk() : (int32_t)upto(c.n_pages - 1);
    c.cu = cu.data();
    c.lens = lens.data();
    c.table = table.data();
    c.table_str = c.max_pages;
    const int rows = upto(1) ? 16 : 32, keys = upto(1) ? 64 : 128;
    int64_t U = 0;
    std::vector<int64_t> base(c.B + 1, 0);
    for (int b = 0; b < c.B; ++b) {
      const PagedSeq q = paged_seq(c, b);
      CHECK(q.n >= 0 && (q.n == 0 || (q.t0 >= 0 && (int64_t)q.t0 + q.n <= c.N)), "rows %d + %d of %d", q.t0, q.n, c.N);
      CHECK(q.L >= 0 && q.L <= cap, "length %d of %lld", q.L, (long long)cap);
      if (!garbage) CHECK(q.flags == 0 && q.L == lens[b] && q.n == cu[b + 1] - cu[b] && q.first == lens[b] - q.n, "sequence %d", b);
      for (int k = 0; q.L > 0 && k < 50; ++k) {
        const int pos = key_within((int)upto((int64_t)q.L + 200), q.L);
        const int pi = page_of(c, pos);
        CHECK(pos >= 0 && pi >= 0 && pi < c.max_pages, "position %d of %d: entry %d of %d", pos, q.L, pi, c.max_pages);
        const PagedRow r = paged_row(c, pos, table[(size_t)b * c.max_pages + pi]);
        CHECK(r.page >= 0 && r.page < c.n_pages && r.slot >= 0 && r.slot < c.page_size, "page %lld slot %lld",
              (long long)r.page, (long long)r.slot);
        CHECK(r.ok == (table[(size_t)b * c.max_pages + pi] >= 0 && table[(size_t)b * c.max_pages + pi] < c.n_pages), "ok");
      }
      U += decode_units(p, q, rows, keys);
      base[b + 1] = U;
    }
    if (U == 0) continue;
    const int G = unit_shares(U, (int)(1 + upto(upto(3) ? 40 : 600)));
    // walk the shares as the kernel does
    std::map<int64_t, std::vector<int64_t>> slots;      // first unit of a row tile -> slots of its partials
    std::vector<char> used(2 * G, 0);
    int64_t covered = 0;
    for (int w = 0; w < G; ++w) {
      int64_t u = unit_start(U, G, w);
      const int64_t end = unit_start(U, G, w + 1);
      CHECK(u == covered && end > u, "share %d starts at %lld, %lld covered", w, (long long)u, (long long)covered);
      covered = end;
      const int64_t first = u;
      int b = 0;
      while (u < end) {
        while (u >= base[b + 1]) ++b;
        const PagedSeq q = paged_seq(c, b);
        const int nb = (int)(((int64_t)q.L + keys - 1) / keys);
        const int64_t run = (u - base[b]) / nb, u0 = base[b] + run * nb;
        const int blk0 = (int)(u - u0), blk1 = (int)(end - u < nb - blk0 ? blk0 + (end - u) : nb);
        CHECK(wg_of_unit(U, G, u) == w && wg_of_unit(U, G, u0 + blk1 - 1) == w, "owner of unit %lld", (long long)u);
        if (blk0 > 0 || blk1 < nb) {
          const int piece = first < u0 ? 1 : 0;
          CHECK(!used[2 * w + piece], "share %d: two partials in slot %d", w, piece);
          used[2 * w + piece] = 1;
          slots[u0].push_back(2 * (int64_t)w + piece);
        } else {
          CHECK(decode_slots(U, G, u0, nb).count == 0, "whole tile at %lld has partials", (long long)u0);
        }
        u += blk1 - blk0;
      }
    }
    CHECK(covered == U, "%lld units of %lld", (long long)covered, (long long)U);
    for (int b = 0; b < c.B; ++b) {
      const PagedSeq q = paged_seq(c, b);
      const int nb = (int)(((int64_t)q.L + keys - 1) / keys);
      for (int64_t u0 = base[b]; u0 < base[b + 1]; u0 += nb) {
        const DecodeSlots s = decode_slots(U, G, u0, nb);
        const auto it = slots.find(u0);
        CHECK(s.count == (it == slots.end() ? 0 : (int)it->second.size()), "row tile at %lld: %d partials", (long long)u0, s.count);
        for (int i = 0; i < s.count; ++i)
          CHECK((i == 0 ? s.first : s.rest + 2 * i) == it->second[i], "row tile at %lld: slot of partial %d", (long long)u0, i);
      }
    }
  }
  // quotients in 32 bits where both operands fit, in 64 elsewhere
  int trial = 0;
  for (; trial < 200000; ++trial) {
    const int64_t x = upto((INT64_MAX >> 1) >> upto(61)), y = 1 + upto((INT64_MAX >> 1) >> upto(61));
    CHECK(quotient(x, y) == x / y, "%lld / %lld", (long long)x, (long long)y);
  }
  for (int64_t x : {0xffffffffLL, 0x100000000LL, 0x100000001LL})
    for (int64_t y : {1LL, 2LL, 0xffffffffLL, 0x100000000LL, 0x100000001LL})
      CHECK(quotient(x, y) == x / y, "%lld / %lld", (long long)x, (long long)y);
  printf("paged map ok\n");
  return 0;
}
