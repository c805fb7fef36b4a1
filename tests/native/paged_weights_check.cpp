// Host-side check of the workspace of the accumulated weights (lvsa_paged.h) over
// random batches, most of them with garbage for row ranges: work-groups that share
// their rows write 128 sums for every unit of the sequences that have work, and none
// of a batch that is refused; all of them lie within the bytes that the library asks
// for.  Also counts the batches that would not fit if each sequence were judged by
// its own range, which is why they are refused whole.  Argument: the built library.
// Prints "paged weights ok" and exits 0, or names the first failure.
#include "lvsa_paged.h"

#include <cstdio>
#include <dlfcn.h>
#include <random>
#include <vector>

using namespace lvsa;

int main(int argc, char** argv) {
  void* lib = argc > 1 ? dlopen(argv[1], RTLD_NOW | RTLD_LOCAL) : nullptr;
  auto query = lib ? (int (*)(const lvsa_paged_weights_args*, int64_t*))dlsym(lib, "lvsa_paged_weights_workspace_query") : nullptr;
  if (!query) {
    printf("no library: %s\n", dlerror());
    return 1;
  }
  std::mt19937_64 rng(5);
  auto upto = [&](int64_t n) { return (int64_t)(rng() % (uint64_t)(n + 1)); };
  int shared = 0, refused = 0, would_not_fit = 0;
  for (int trial = 0; trial < 40000; ++trial) {
    lvsa_paged_weights_args a{};
    a.cache.k = a.cache.v = (void*)4096;
    for (int i = 0; i < 3; ++i) a.cache.k_str[i] = a.cache.v_str[i] = 128;
    a.cache.n_pages = 10;
    a.cache.page_size = (int)(1 + upto(40));
    a.cache.Hkv = (int)(1 + upto(3));
    a.cache.D = 64;
    a.cache.bits = 16;
    a.cache.dtype = LVSA_BF16;
    a.batch.B = (int)(1 + upto(trial % 5 ? 70 : 300));
    a.batch.N = (int)(1 + upto(trial % 3 ? 100 : 6));
    a.batch.max_pages = (int)upto(60);
    a.batch.table_stride = a.batch.max_pages;
    a.q = (void*)4096;
    a.q_str[0] = a.q_str[1] = 64;
    a.H = a.cache.Hkv * (int)(1 + upto(trial % 2 ? 7 : 200));
    a.scale = 1.f;
    a.max_q_len = (int)upto(2 * a.batch.N);
    std::vector<int32_t> cu(a.batch.B + 1), lens(a.batch.B);
    const int cap = a.batch.max_pages * a.cache.page_size;
    for (auto& x : lens) x = trial % 7 ? cap : (int32_t)upto(cap + cap / 8 + 1);
    if (trial % 4 == 0) {              // ranges that ascend
      for (int b = 1; b <= a.batch.B; ++b) cu[b] = cu[b - 1] + (int32_t)upto((a.batch.N - cu[b - 1]) / 2);
    } else if (trial % 4 == 1) {       // every second one all rows
      for (int b = 0; b <= a.batch.B; ++b) cu[b] = b % 2 ? a.batch.N : 0;
    } else {
      for (auto& x : cu) x = upto(30) ? (int32_t)upto(a.batch.N) : (int32_t)(uint32_t)rng();
    }
    a.batch.cu_seqlens = cu.data();
    a.batch.kv_lens = lens.data();
    a.batch.page_table = (const int32_t*)4096;
    PagedView c{};
    set_page_size(&c, a.cache.page_size);
    c.max_pages = a.batch.max_pages;
    c.B = a.batch.B;
    c.N = a.batch.N;
    c.cu = cu.data();
    c.lens = lens.data();
    int64_t bytes = -1, units = 0;
    if (query(&a, &bytes)) {
      printf("trial %d: the query fails\n", trial);
      return 1;
    }
    int flags = 0;
    for (int s = 0; s < c.B; ++s) {
      const PagedSeq q = paged_seq(c, s);
      flags |= q.flags;
      units += weight_units(q, a.cache.Hkv, kWeightKeys);
    }
    if (bytes == 0) continue;          // nothing is shared, nothing written there
    int64_t most = (int64_t)(c.B < c.N ? c.B : c.N) * ((cap + kWeightKeys - 1) / kWeightKeys) * a.cache.Hkv;
    if (most < 1) most = 1;            // a table of no pages
    const int64_t splits = bytes / (4 * kWeightKeys * most);
    if (splits < 2 || splits * 4 * kWeightKeys * most != bytes) {
      printf("trial %d: %lld bytes are no whole sums of %lld units\n", trial, (long long)bytes, (long long)most);
      return 1;
    }
    ++shared;
    const bool fits = units * splits * kWeightKeys * 4 <= bytes;
    if (flags & LVSA_PAGED_BAD_CU) {
      ++refused;
      would_not_fit += !fits;
    } else if (!fits) {
      printf("trial %d: %lld units of %lld splits, %lld bytes\n", trial, (long long)units, (long long)splits, (long long)bytes);
      return 1;
    }
  }
  printf("%d batches share rows, %d of them refused, of which %d would not fit\n", shared, refused, would_not_fit);
  if (shared - refused < 100 || would_not_fit < 100) return 1;
  printf("paged weights ok\n");
  return 0;
}
