// What the kernels over the paged key/value cache share (lvsa_paged.hip:
// append, gather, merge and the C ABI; lvsa_paged_attn.h: attention, one unit
// per head size; lvsa_paged_blocks.hip, lvsa_paged_list.h, lvsa_paged_weights.h and
// lvsa_paged_evict.hip: parts of a cache): the cache and batch as the device sees
// them, the lookup of rows through the page table, and the number format of 4-bit
// pages.
//
// Nothing read from device memory is trusted: page numbers, lengths and row
// ranges are checked where they are used, so that no address leaves the
// cache's pages or the batch's rows; what is found is reported in the cache's
// status word (LVSA_PAGED_*).
#pragma once
#include "lvsa_common.h"

namespace lvsa {

struct PagedView {
  // 16-bit elements or E2M1 codes and their scales; strides in bytes
  char* k; char* v;
  uint8_t* ks; uint8_t* vs;
  int64_t k_str[3], v_str[3], ks_str[3], vs_str[3];
  int32_t n_pages, page_size, Hkv;
  uint32_t ps_mul, ps_shift;     // p / page_size = (p * ps_mul) >> ps_shift for 0 <= p < 2^31
  int32_t* status;
  const int32_t* cu;
  const int32_t* lens;
  const int32_t* table;
  int64_t table_str;
  int32_t B, max_pages, N;
};

// Sequence s: its rows [t0, t0 + n) of the packed ones, its cached length, and
// the position of row t0 (paged_seq).
struct PagedSeq {
  int t0, n, L, first;
  int flags;
};

// What paged_plan_kernel writes for the prefill kernels, at the start of the
// workspace: the row tiles of all sequences (each is done once per key head),
// the units (key blocks) before each, where each share of the launch's units
// ends, and what the tile it ends in is to be joined from.  Units are ordered
// by key head, tile and key block; a tile without keys counts as one.
struct PlanHead {
  int64_t per_head;              // units of one key head
  int32_t tiles, shares;
  int32_t bad_cu, pad;           // the row ranges do not ascend within the rows: the whole result is NaN
};
struct PlanTile {
  int32_t seq, r0, units, blocks;
  PagedSeq sq;
  int32_t pad[3];
};
struct PlanEnd {
  int32_t h, tile, blk, pad;     // the share's last unit is unit blk - 1 of this tile
};
struct PlanJoin {
  int64_t first, rest;           // see DecodeSlots
  int32_t count;                 // 0: nothing to join
  int32_t h, r0, rows, t0, pad[3];
};

struct PagedAttnParams {
  PagedView c;
  const char* q; char* o; float* lse;
  int64_t q_str[2], o_str[2];    // bytes
  float scale_log2;              // scale * log2(e)
  int32_t H, group, causal, fill_tail;
  int32_t short_rows;            // 16 slots of a page lie within 2^31 bytes
  // The launch's key blocks are cut into equal shares for `grid` work-groups,
  // each with two slots of row-tile partials: fp32 O [slot][rows][D], then
  // (max, sum) pairs.  Prefill kernels: `tiles` bounds the row tiles.
  int32_t grid, tiles;
  float* ws_o; float* ws_ml;
  PlanHead* head;
  PlanTile* plan_tiles;
  int64_t* before;               // [tiles + 1]
  PlanEnd* ends;                 // [grid]
  PlanJoin* joins;               // [grid]
};

// Attention launches per head size.  rows: 16 or 32 (decode kernel, row tiles
// of that many rows), 128 or 256 (prefill kernels).
int paged_attn_d64(const PagedAttnParams& p, int bits, int rows, bool bf16, hipStream_t stream);
int paged_attn_d96(const PagedAttnParams& p, int bits, int rows, bool bf16, hipStream_t stream);
int paged_attn_d128(const PagedAttnParams& p, int bits, int rows, bool bf16, hipStream_t stream);
int paged_attn_d192(const PagedAttnParams& p, int bits, int rows, bool bf16, hipStream_t stream);
int paged_attn_d256(const PagedAttnParams& p, int bits, int rows, bool bf16, hipStream_t stream);

// Keys that the four waves of a decode work-group take per step.
__host__ __device__ constexpr int paged_decode_keys(int D) { return 4 * (D >= 192 ? 16 : 32); }
// Decode work-groups that a compute unit holds at once: what the registers
// allow (the kernels are compiled for it), and what a launch starts of them, so
// that equal shares end together.  16-bit caches are read at 5.7 TB/s by one
// group as by four (40 sequences of 12000 keys, 8 heads of 128: 341, 342, 342,
// 346 us with 1 to 4), 4-bit ones need waves to decode behind the loads (180,
// 122, 111, 128 us; of 64: 123, 85, 75, 72).
__host__ __device__ constexpr int paged_decode_groups(int D, int bits, int rows) {
  if (bits == 16) return D == 64 || (D <= 128 && rows == 16) ? 2 : 1;
  if (rows == 16) return D == 64 ? 4 : D <= 128 ? 3 : 2;
  return D == 64 ? 3 : D <= 192 ? 2 : 1;
}
constexpr int kPagedTile = 128;        // rows of a prefill tile
constexpr int kPagedTall = 256;        // rows of a tall one (head sizes up to 128)
constexpr int kPagedBlock = 64;        // its keys per step
// Chunks run on the decode kernel, too, where their rows (of all heads) and twice
// its steps come to no more than this per compute unit: latency counts there, and
// it needs no plan.  Prefill and decode kernel, us, head size 128, causal:
//   tokens, heads / key heads, keys   rows + 2 steps per unit    16 bits     4 bits
//   20, 16 / 4, 2000                        1.3 +  2             33   17     32   17
//   256, 16 / 4, 300                       16   +  3             43   30     40   30
//   256, 16 / 4, 1000                      16   +  8             51   34     49   33
//   512, 16 / 4, 512                       32   +  8             57   40     54   45
//   384, 16 / 16, 600                      24   +  8             45   47     43   42
//   512, 16 / 16, 1000                     32   + 17             44   47     41   50
//   4 times 256, 16 / 4, 256               64   +  8             47   66     45   55
// and with D = 256 and 2000 tokens of 2 heads over themselves, 16 + 32: 65, 80 us.
constexpr int kPagedShort = 40;
// Fewest steps of a prefill share that is worth its partials (two sequences of 256
// rows, 16 heads of 128, over 600 keys: 63, 50, 76 us with 1, 4, 16; over 1200: 64,
// 54, 65; over 300: 43, 50, 92).
constexpr int kPagedLeast = 4;

// The running maximum of a row that has seen no key: below every finite score,
// and still finite, so that differences to it are never NaN.
constexpr float kNoKeys = -3.0e38f;

// ── lookups, alike on host and device (tests/native/paged_map_check.cpp) ─────

__host__ __device__ inline int page_of(const PagedView& c, int pos) {
  return (int)(((uint64_t)(uint32_t)pos * c.ps_mul) >> c.ps_shift);
}

// The sequence of rows [a, e) with `len` keys.  Ranges and lengths outside what
// the caller allocated are cut to it and flagged.
__host__ __device__ inline PagedSeq paged_seq(const PagedView& c, int a, int e, int len) {
  PagedSeq r;
  const int64_t cap = (int64_t)c.max_pages * c.page_size;
  r.flags = 0;
  r.L = len;
  if (len < 0) r.L = 0;
  if (len > cap) r.L = (int)cap;
  if (r.L != len) r.flags |= LVSA_PAGED_BAD_LENGTH;
  const int lo = a < 0 ? 0 : a, hi = e > c.N ? c.N : e;
  if (a < 0 || e > c.N || e < a) r.flags |= LVSA_PAGED_BAD_CU;
  r.t0 = lo;
  r.n = hi > lo ? hi - lo : 0;
  const int64_t first = (int64_t)r.L - ((int64_t)e - lo);
  r.first = first < -(1 << 30) ? -(1 << 30) : first > INT32_MAX ? INT32_MAX : (int)first;
  return r;
}

__host__ __device__ inline PagedSeq paged_seq(const PagedView& c, int s) {
  return paged_seq(c, c.cu[s], c.cu[s + 1], c.lens[s]);
}

// Key position that a kernel reads for `pos`: past the end the last key, whose
// weight is masked away.  L >= 1.
__host__ __device__ inline int key_within(int pos, int L) { return pos < L ? pos : L - 1; }

// Page and slot of position `pos` whose table entry is `page`; a page outside
// the cache is read as page 0.
struct PagedRow {
  int64_t page, slot;
  bool ok;
};
__host__ __device__ inline PagedRow paged_row(const PagedView& c, int pos, int page) {
  PagedRow r;
  r.slot = pos - page_of(c, pos) * c.page_size;
  r.ok = (uint32_t)page < (uint32_t)c.n_pages;
  r.page = r.ok ? page : 0;
  return r;
}

// Work units of a sequence in the decode kernel: (row tiles) x (key heads) x
// (key steps), key steps innermost.
__host__ __device__ inline int64_t decode_units(const PagedAttnParams& p, const PagedSeq& q, int rows, int keys) {
  const int64_t rt = ((int64_t)q.n * p.group + rows - 1) / rows;
  return rt * p.c.Hkv * (((int64_t)q.L + keys - 1) / keys);
}

// Shares of U > 0 units over a grid, of at least `least` units each: none is
// empty, so that the work-groups a row tile spans all have a partial of it.
__host__ __device__ inline int unit_shares(int64_t U, int grid, int least = 1) {
  const int64_t n = U / least;
  return n < 1 ? 1 : n < grid ? (int)n : grid;
}
// a / b for a >= 0, b > 0: in 32 bits where both fit (64-bit division is 150
// instructions on the device, and these are at the head of a latency chain).
__host__ __device__ inline int64_t quotient(int64_t a, int64_t b) {
  return ((uint64_t)a | (uint64_t)b) >> 32 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b);
}
// First unit of share w of G over U units, and the share of unit u.
__host__ __device__ inline int64_t unit_start(int64_t U, int G, int w) { return quotient(w * U, G); }
__host__ __device__ inline int wg_of_unit(int64_t U, int G, int64_t u) { return (int)quotient((u + 1) * G - 1, U); }

// Shares of a prefill launch: one for every (tile, key head), whatever its keys,
// where there are work-groups for it, else of kPagedLeast units at least.
__host__ __device__ inline int plan_shares(int64_t U, int64_t pairs, int grid) {
  if (U <= 0) return 0;
  const int least = unit_shares(U, grid, kPagedLeast);
  return pairs <= least ? least : pairs < grid ? (int)pairs : grid;
}
// Share of a work-group.  Consecutive work-groups go to the eight XCDs in turn:
// an XCD gets consecutive shares, few key heads' tiles, whose keys its L2 then
// serves to all of them.
__host__ __device__ inline int share_of(int wg, int shares) {
  const int per = (shares + 7) / 8, s = (wg & 7) * per + (wg >> 3);
  return (wg >> 3) < per && s < shares ? s : -1;
}

// Partials of the row tile whose key steps are units [u0, u0 + nb): none if one
// work-group has them all, else one per work-group, in the first of its two
// slots but where it came to the tile from another one.
struct DecodeSlots {
  int count;
  int64_t first, rest;      // slot of partial 0; slot of partial i > 0: rest + 2 i
};
__host__ __device__ inline DecodeSlots decode_slots(int64_t U, int G, int64_t u0, int nb) {
  const int wa = wg_of_unit(U, G, u0), wb = wg_of_unit(U, G, u0 + nb - 1);
  if (wa == wb) return DecodeSlots{0, 0, 0};
  return DecodeSlots{wb - wa + 1, 2 * (int64_t)wa + (unit_start(U, G, wa) < u0 ? 1 : 0), 2 * (int64_t)wa};
}

// p / d as (p * mul) >> shift, exact for 0 <= p < 2^31: with 2^l >= d and mul =
// floor(2^(31 + l) / d) + 1, mul * d exceeds 2^(31 + l) by at most 2^l.
struct Divisor {
  uint32_t mul, shift;
  int32_t by;
};
inline Divisor divisor(int d) {
  int l = 0;
  while ((1LL << l) < d) ++l;
  return Divisor{(uint32_t)((1ULL << (31 + l)) / (uint64_t)d + 1), (uint32_t)(31 + l), d};
}
__host__ __device__ inline int operator/(int p, const Divisor& d) { return (int)(((uint64_t)(uint32_t)p * d.mul) >> d.shift); }

inline void set_page_size(PagedView* v, int page_size) {
  const Divisor d = divisor(page_size);
  v->page_size = page_size;
  v->ps_mul = d.mul;
  v->ps_shift = d.shift;
}

// ── tiles of rows and blocks of keys (lvsa_paged_list.h) ─────────────────────

// Blocks of `block` slots, `parts` to a page; rows of a sequence in tiles of `tile`,
// `lists` of which the batch may have, each with up to `top` blocks a key head.
struct ListView {
  Divisor block, parts, tile;
  int32_t lists, top;
};
constexpr int kListMax = 1024;         // blocks of a list: what a work-group keeps of it is 12 KB of LDS

// Tiles of sequence `s`: from where on, and how many.
__host__ __device__ inline int64_t first_list(const ListView& v, int s, const PagedSeq& q) {
  return v.tile.by == 1 ? q.t0 : (int64_t)(q.t0 / v.tile) + s;
}
// End of the rows of a tile that starts at row i0 < q.n of its sequence.
__host__ __device__ inline int tile_end(const ListView& v, const PagedSeq& q, int i0) {
  return q.n - i0 > v.tile.by ? i0 + v.tile.by : q.n;
}
__host__ __device__ inline int list_count(const ListView& v, const PagedSeq& q) { return (int)(((int64_t)q.n + v.tile.by - 1) / v.tile.by); }

struct BlockAttnParams {
  ListView v;
  const int32_t* blocks;               // [lists][Hkv][top]
  // The launch's work is key heads x lists x row tiles of a list (`subs`), each of
  // `steps` steps, as many as the longest list has (a shorter one's keys are spread
  // over them); it is cut into equal shares for `grid` work-groups, see DecodeSlots.
  int32_t subs, steps;
  int64_t work;
};
int paged_block_attn_d64(const PagedAttnParams& p, const BlockAttnParams& l, int bits, int rows, bool bf16, hipStream_t stream);
int paged_block_attn_d96(const PagedAttnParams& p, const BlockAttnParams& l, int bits, int rows, bool bf16, hipStream_t stream);
int paged_block_attn_d128(const PagedAttnParams& p, const BlockAttnParams& l, int bits, int rows, bool bf16, hipStream_t stream);
int paged_block_attn_d192(const PagedAttnParams& p, const BlockAttnParams& l, int bits, int rows, bool bf16, hipStream_t stream);
int paged_block_attn_d256(const PagedAttnParams& p, const BlockAttnParams& l, int bits, int rows, bool bf16, hipStream_t stream);

// Accumulated weights (lvsa_paged_weights.h).
struct WeightsParams {
  const float* lse;
  char* w;
  int64_t w_str[3];                    // bytes
  int32_t accumulate, many;            // many: rows of a sequence, more than a tile or two
  int32_t splits;                      // work-groups that share the rows of 128 keys
  float* ws;                           // their sums: [128 keys][splits][128]
};
constexpr int kWeightKeys = 128;
// Work-groups of few rows' weights on a compute unit at once (255, 187, 182 us with 1 to
// 3 for 45 sequences of up to 16000 keys, 8 heads of 128).
constexpr int kWeightGroups = 3;
// Work of a sequence: its key heads x blocks of `keys` keys.  Over row ranges that
// ascend there are no more sequences with work than rows or sequences, for which the
// workspace has room; other batches are refused whole, since each of their ranges may
// be fine by itself and all of them together more (tests/native/paged_weights_check.cpp).
__host__ __device__ inline int64_t weight_units(const PagedSeq& s, int Hkv, int keys) {
  return s.n && !s.flags ? ((int64_t)s.L + keys - 1) / keys * Hkv : 0;
}
int paged_weights_d64(const PagedAttnParams& p, const WeightsParams& w, int bits, bool bf16, hipStream_t stream);
int paged_weights_d96(const PagedAttnParams& p, const WeightsParams& w, int bits, bool bf16, hipStream_t stream);
int paged_weights_d128(const PagedAttnParams& p, const WeightsParams& w, int bits, bool bf16, hipStream_t stream);
int paged_weights_d192(const PagedAttnParams& p, const WeightsParams& w, int bits, bool bf16, hipStream_t stream);
int paged_weights_d256(const PagedAttnParams& p, const WeightsParams& w, int bits, bool bf16, hipStream_t stream);

// End of the keys that row r attends, and the key blocks of the tile of rows
// [r0, r1].
__host__ __device__ inline int key_limit(const PagedAttnParams& p, const PagedSeq& s, int r) {
  if (!p.causal) return s.L;
  const int64_t e = (int64_t)s.first + r / p.group + 1;
  return e < 0 ? 0 : e > s.L ? s.L : (int)e;
}
__host__ __device__ inline int tile_blocks(const PagedAttnParams& p, const PagedSeq& s, int r0, int rows) {
  const int end = s.n * p.group, last = r0 + rows < end ? r0 + rows - 1 : end - 1;
  return (int)(((int64_t)key_limit(p, s, last) + kPagedBlock - 1) / kPagedBlock);
}

namespace {

// A value that is the same in every lane, in a scalar register.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ PagedSeq uniform(const PagedSeq& s) {
  return PagedSeq{uniform(s.t0), uniform(s.n), uniform(s.L), uniform(s.first), uniform(s.flags)};
}

__device__ __forceinline__ void paged_flag(const PagedView& c, int bit) {
  if (c.status) atomicOr(c.status, bit);
}

// The first sequence whose row range holds row t (the same for every lane of the
// wave; t uniform), or -1.  Every lane reads one sequence, so that a batch of up to 64
// costs one trip to memory.
__device__ __forceinline__ int paged_seq_of_row(const PagedView& c, int t, int lane, PagedSeq* q) {
  for (int s0 = 0; s0 < c.B; s0 += 64) {
    const int s = s0 + lane;
    int a = 0, e = 0, len = 0;
    if (s < c.B) {
      a = c.cu[s];
      e = c.cu[s + 1];
      len = c.lens[s];
    }
    const uint64_t m = __builtin_amdgcn_ballot_w64(a <= t && t < e);
    if (m) {
      const int i = __builtin_ctzll(m);
      *q = paged_seq(c, __builtin_amdgcn_readlane(a, i), __builtin_amdgcn_readlane(e, i), __builtin_amdgcn_readlane(len, i));
      return s0 + i;
    }
  }
  return -1;
}

// The sequence that lane `from` holds, for every lane.
__device__ __forceinline__ PagedSeq from_lane(const PagedSeq& s, int from) {
  return PagedSeq{__builtin_amdgcn_readlane(s.t0, from), __builtin_amdgcn_readlane(s.n, from),
                  __builtin_amdgcn_readlane(s.L, from), __builtin_amdgcn_readlane(s.first, from),
                  __builtin_amdgcn_readlane(s.flags, from)};
}
__device__ __forceinline__ int64_t from_lane(int64_t x, int from) {
  return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), from) << 32 |
                   (uint32_t)__builtin_amdgcn_readlane((int)x, from));
}

// Inclusive sum over the first `count` lanes of a wave.
__device__ __forceinline__ int64_t wave_scan(int64_t x, int lane, int count = 64) {
  for (int d = 1; d < 64 && d < count; d <<= 1) {
    const int64_t y = __shfl_up(x, d);
    if (lane >= d) x += y;
  }
  return x;
}

// Work-groups take the units of all sequences in turn: `count` says how many a
// sequence has, `work` does unit i of sequence s, the u-th of all.  WHOLE: row ranges
// that do not ascend leave the batch no units at all, else those sequences alone.
template <bool WHOLE, typename Count, typename Work>
__device__ __forceinline__ void walk_units(const PagedView& c, Count count, Work work) {
  const int lane = threadIdx.x & 63;
  int64_t base = 0, u = blockIdx.x;            // units before these sequences, the next one of this work-group
  int flags = 0;
  if (WHOLE)                                   // the first 64 are read before any unit
    for (int s = 64 + lane; s < c.B; s += 64) flags |= paged_seq(c, s).flags;
  for (int s0 = 0; s0 < c.B; s0 += 64) {
    PagedSeq mine = {};
    int64_t n = 0;
    if (s0 + lane < c.B) {
      mine = c.cu ? paged_seq(c, s0 + lane) : paged_seq(c, 0, 0, c.lens[s0 + lane]);
      flags |= mine.flags;
      if (!mine.flags) n = count(mine);
    }
    if (WHOLE && __builtin_amdgcn_ballot_w64(flags & LVSA_PAGED_BAD_CU)) break;
    const int64_t upto = wave_scan(n, lane), end = base + from_lane(upto, 63);
    for (; u < end; u += gridDim.x) {
      const int at = __builtin_ctzll(__builtin_amdgcn_ballot_w64(base + upto > u));
      work(s0 + at, from_lane(mine, at), u - base - from_lane(upto - n, at), u);
    }
    base = end;
  }
  if (blockIdx.x == 0 && threadIdx.x < 64 && flags) paged_flag(c, flags);
}

}  // namespace
}  // namespace lvsa
