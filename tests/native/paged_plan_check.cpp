// Host-side check of the shares of a prefill launch over the paged cache
// (lvsa_paged.h), over random batches:
//   - the row tiles of a batch are no more than the launch's bound;
//   - every work unit (key block of a tile and key head) is in one share, every
//     share belongs to one work-group, and walking a share from its end reaches
//     its first unit exactly;
//   - partial sums go to slots of their own; the share that a divided tile starts
//     in ends inside it and names exactly the tile's partials, in order.
// Prints "paged plan ok" and exits 0, or names the first failure.
#include "lvsa_paged.h"

#include <algorithm>
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
  std::mt19937_64 rng(11);
  auto upto = [&](int64_t n) { return (int64_t)(rng() % (uint64_t)(n + 1)); };
  for (int trial = 0; trial < 6000; ++trial) {
    PagedAttnParams p{};
    PagedView& c = p.c;
    set_page_size(&c, (int)(1 + upto(40)));
    c.max_pages = (int)(1 + upto(trial % 3 ? 200 : 5000));
    c.B = (int)(1 + upto(trial % 50 ? 6 : 6000));
    c.Hkv = (int)(1 + upto(8));
    p.group = (int)(1 + upto(5));
    p.causal = (int)upto(1);
    const int rows = upto(1) ? kPagedTile : kPagedTall;
    const int64_t cap = (int64_t)c.max_pages * c.page_size;
    std::vector<int32_t> cu(c.B + 1, 0), lens(c.B);
    for (int b = 0; b < c.B; ++b) {
      lens[b] = (int32_t)(upto(6) ? upto(cap) : 0);
      const int64_t most = upto(3) ? 20 : 2000;
      cu[b + 1] = cu[b] + (int32_t)(upto(4) ? upto(c.B > 10 ? 3 : most) : 0);     // more rows than keys too
    }
    c.N = cu[c.B] + (int32_t)upto(3);
    c.cu = cu.data();
    c.lens = lens.data();
    const int64_t bound = ((int64_t)c.N * p.group + rows - 1) / rows + std::min(c.B, c.N);
    // the plan's list
    struct Tile { int seq, r0, units, blocks, n; };
    std::vector<Tile> tiles;
    std::vector<int64_t> before;
    int64_t per_head = 0;
    for (int b = 0; b < c.B; ++b) {
      const PagedSeq q = paged_seq(c, b);
      CHECK(q.flags == 0, "sequence %d: flags %d", b, q.flags);
      for (int64_t r0 = 0; r0 < (int64_t)q.n * p.group; r0 += rows) {
        const int blocks = tile_blocks(p, q, (int)r0, rows);
        CHECK(blocks >= 0 && (int64_t)blocks * kPagedBlock < q.L + kPagedBlock, "%d blocks of %d keys", blocks, q.L);
        tiles.push_back({b, (int)r0, std::max(blocks, 1), blocks, q.n});
        before.push_back(per_head);
        per_head += tiles.back().units;
      }
    }
    CHECK((int64_t)tiles.size() <= bound, "%zu tiles, bound %lld", tiles.size(), (long long)bound);
    const int64_t U = per_head * c.Hkv, pairs = (int64_t)tiles.size() * c.Hkv;
    const int grid = 8 * (int)(1 + upto(upto(1) ? 63 : 3));
    const int shares = plan_shares(U, pairs, grid);
    CHECK(shares <= grid && shares <= U && (shares > 0) == (U > 0), "%d shares of %lld units for %d work-groups", shares,
          (long long)U, grid);
    std::vector<int> taken(shares, 0);
    for (int wg = 0; wg < grid; ++wg) {
      const int s = share_of(wg, shares);
      CHECK(s >= -1 && s < shares, "work-group %d has share %d", wg, s);
      if (s >= 0) taken[s]++;
    }
    for (int s = 0; s < shares; ++s) CHECK(taken[s] == 1, "share %d is %d work-groups'", s, taken[s]);
    if (U == 0) continue;
    std::vector<char> covered(U, 0), used(2 * (size_t)shares, 0);
    std::map<int64_t, std::vector<std::pair<int64_t, int64_t>>> parts;   // first unit of a (head, tile) -> (first block, slot)
    std::map<int64_t, DecodeSlots> joins;
    for (int w = 0; w < shares; ++w) {
      int64_t left = unit_start(U, shares, w + 1) - unit_start(U, shares, w);
      const int64_t u = unit_start(U, shares, w + 1) - 1;
      int h = (int)quotient(u, per_head);
      int ti = (int)(std::upper_bound(before.begin(), before.end(), u - h * per_head) - before.begin()) - 1;
      int end = (int)(u - h * per_head - before[ti]) + 1;
      CHECK(left > 0 && end >= 1 && end <= tiles[ti].units, "share %d ends at block %d of %d", w, end, tiles[ti].units);
      const int64_t u0 = h * per_head + before[ti];
      if (end < tiles[ti].units && wg_of_unit(U, shares, u0) == w) joins[u0] = decode_slots(U, shares, u0, tiles[ti].units);
      for (;;) {
        CHECK(h >= 0, "share %d walks past the first head", w);
        const int blk0 = left < end ? end - (int)left : 0;
        const int64_t first = h * per_head + before[ti];
        for (int k = blk0; k < end; ++k) {
          CHECK(!covered[first + k], "unit %lld twice", (long long)(first + k));
          covered[first + k] = 1;
        }
        if (blk0 > 0 || end < tiles[ti].units) {
          const int64_t slot = 2 * (int64_t)w + (left > end ? 1 : 0);
          CHECK(!used[slot], "slot %lld twice", (long long)slot);
          used[slot] = 1;
          parts[first].push_back({blk0, slot});
        }
        left -= end - blk0;
        if (left <= 0) break;
        if (--ti < 0) {
          ti = (int)tiles.size() - 1;
          --h;
        }
        end = tiles[ti].units;
      }
      CHECK(left == 0, "share %d: %lld units left", w, (long long)left);
    }
    for (int64_t k = 0; k < U; ++k) CHECK(covered[k], "unit %lld in no share", (long long)k);
    CHECK(parts.size() == joins.size(), "%zu divided tiles, %zu joins", parts.size(), joins.size());
    for (auto& [first, slots] : parts) {
      std::sort(slots.begin(), slots.end());
      const auto j = joins.find(first);
      CHECK(j != joins.end() && j->second.count == (int)slots.size(), "tile at %lld: %zu partials", (long long)first, slots.size());
      for (int i = 0; i < j->second.count; ++i)
        CHECK((i == 0 ? j->second.first : j->second.rest + 2 * i) == slots[i].second, "tile at %lld: slot of partial %d",
              (long long)first, i);
    }
  }
  printf("paged plan ok\n");
  return 0;
}
