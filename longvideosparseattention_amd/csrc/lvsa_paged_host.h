// What the paged cache's entry points share on the host: checks of a cache and a
// batch, and the choice of an instantiation.
#pragma once
#include "lvsa_paged.h"

#include <mutex>

namespace lvsa {
namespace {

inline int cu_count() {
  static std::mutex mu;
  static int cached[64] = {0};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) {
    (void)hipGetLastError();       // no device: sizes are still answered
    return 256;
  }
  std::lock_guard<std::mutex> lock(mu);
  if (cached[dev] == 0) {
    int n = 0;
    cached[dev] = hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) == hipSuccess && n > 0 ? n : 256;
  }
  return cached[dev];
}

inline bool aligned16(int64_t x) { return (x & 15) == 0; }

// Whether two [N, heads, D] tensors of 16-bit elements (strides in bytes) lie within
// each other's bounds.
inline bool share_memory(const void* a, const int64_t* as, int ah, const void* b, const int64_t* bs, int bh, int N, int D) {
  auto bound = [&](const void* at, const int64_t* str, int heads, bool high) {
    int64_t x = (int64_t)(uintptr_t)at + (high ? 2 * (int64_t)D : 0);
    const int64_t far[2] = {(N - 1) * str[0], (heads - 1) * str[1]};
    for (int64_t f : far) x += high == (f > 0) ? f : 0;
    return x;
  };
  return bound(a, as, ah, false) < bound(b, bs, bh, true) && bound(b, bs, bh, false) < bound(a, as, ah, true);
}

// Checks a cache and a batch and forms the device's view of them.
inline int paged_view(const char* what, const lvsa_paged_cache* c, const lvsa_paged_batch* b, bool rows, PagedView* v) {
  LVSA_REQUIRE(c->D == 64 || c->D == 96 || c->D == 128 || c->D == 192 || c->D == 256, LVSA_ERR_UNSUPPORTED,
               "%s: head_dim %d not supported (64, 96, 128, 192, 256)", what, c->D);
  LVSA_REQUIRE(c->bits == 16 || c->bits == 4, LVSA_ERR_UNSUPPORTED, "%s: caches hold 16 or 4 bits, not %d", what, c->bits);
  LVSA_REQUIRE(c->dtype == LVSA_BF16 || c->dtype == LVSA_FP16, LVSA_ERR_UNSUPPORTED, "%s: dtype %d: bf16 or fp16", what,
               c->dtype);
  LVSA_REQUIRE(c->n_pages >= 1 && c->page_size >= 1 && c->Hkv >= 1, LVSA_ERR_INVALID_ARG,
               "%s: %d pages of %d slots, %d heads", what, c->n_pages, c->page_size, c->Hkv);
  LVSA_REQUIRE(c->k && c->v && (c->bits == 16 || (c->k_scale && c->v_scale)), LVSA_ERR_INVALID_ARG,
               "%s: null cache pointer", what);
  LVSA_REQUIRE(b->B >= 0 && b->max_pages >= 0 && b->N >= 0 && b->table_stride >= b->max_pages, LVSA_ERR_INVALID_ARG,
               "%s: batch of %d sequences, %d pages (rows %lld apart), %d rows", what, b->B, b->max_pages,
               (long long)b->table_stride, b->N);
  LVSA_REQUIRE(b->B == 0 || (b->kv_lens && (b->page_table || b->max_pages == 0) && (!rows || b->cu_seqlens)),
               LVSA_ERR_INVALID_ARG, "%s: null batch pointer", what);
  LVSA_REQUIRE((int64_t)b->max_pages * c->page_size < (1LL << 31) - 4096, LVSA_ERR_UNSUPPORTED,
               "%s: %d pages of %d slots: positions must stay below 2^31 - 4096", what, b->max_pages, c->page_size);
  const int64_t unit = c->bits == 16 ? 2 : 1;
  v->k = (char*)c->k;
  v->v = (char*)c->v;
  v->ks = (uint8_t*)c->k_scale;
  v->vs = (uint8_t*)c->v_scale;
  bool ok = aligned16((int64_t)(uintptr_t)c->k) && aligned16((int64_t)(uintptr_t)c->v);
  for (int i = 0; i < 3; ++i) {
    v->k_str[i] = c->k_str[i] * unit;
    v->v_str[i] = c->v_str[i] * unit;
    v->ks_str[i] = c->ks_str[i];
    v->vs_str[i] = c->vs_str[i];
    ok = ok && aligned16(v->k_str[i]) && aligned16(v->v_str[i]);
  }
  LVSA_REQUIRE(ok, LVSA_ERR_INVALID_ARG, "%s: cache rows must start at multiples of 16 bytes", what);
  v->n_pages = c->n_pages;
  v->Hkv = c->Hkv;
  set_page_size(v, c->page_size);
  v->status = c->status;
  v->cu = b->cu_seqlens;
  v->lens = b->kv_lens;
  v->table = b->page_table;
  v->table_str = b->table_stride;
  v->B = b->B;
  v->max_pages = b->max_pages;
  v->N = b->N;
  return LVSA_OK;
}

template <template <int, typename, int> class L, typename... A>
int by_type(int D, int dtype, int bits, A&&... a) {
#define LVSA_PAGED_CASE(d)                                                             \
  case d:                                                                              \
    if (dtype == LVSA_BF16) return bits == 16 ? L<d, __bf16, 16>::go(a...) : L<d, __bf16, 4>::go(a...); \
    return bits == 16 ? L<d, _Float16, 16>::go(a...) : L<d, _Float16, 4>::go(a...);
  switch (D) {
    LVSA_PAGED_CASE(64)
    LVSA_PAGED_CASE(96)
    LVSA_PAGED_CASE(128)
    LVSA_PAGED_CASE(192)
    LVSA_PAGED_CASE(256)
  }
#undef LVSA_PAGED_CASE
  return LVSA_ERR_UNSUPPORTED;
}

}  // namespace
}  // namespace lvsa
