// Weights that the newest rows give to the cached tokens (gfx950): w_j (+)= sum_i
// exp(scale q_i.k_j - lse_i) over the rows of a sequence and the query heads of a key
// head.  The scores are formed as S^T = K Q^T, so that a row of the matrix is a key and
// its sum runs over the lanes; nothing is shared between keys.
#pragma once
#include "lvsa_paged_attn.h"

namespace lvsa {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

// Few rows (a tile of 16, or some of them one after the other): bound by the bytes of
// the keys.  The launch's work, sum over sequences of key heads x key steps, is cut
// into equal shares, as in paged_decode_kernel; a wave has 16 T keys of a step and the
// next step's on their way.  Lane (g = lane / 16, x = lane % 16) holds elements of key
// x, and the sums of keys 4 g .. + 3, of which it keeps key x's where x / 4 = g.  The
// sums of 2048 keys wait in LDS and go to the weights together: written step by step,
// 64 bytes a wave, a fortieth of the bytes took a quarter of the time (157 us without
// the writes, 208 with them, 187 together; 45 sequences of up to 16000 keys, 8 heads of
// 128).
template <int D, typename E, int BITS>
__global__ __launch_bounds__(256, kWeightGroups) void paged_weights_kernel(PagedAttnParams p, WeightsParams wp) {
  constexpr int T = D >= 192 ? 1 : 2, ND = D / 32, KW = 16 * T, KEYS = 4 * KW;
  constexpr int HELD = 2048 / KEYS;        // steps whose sums LDS holds
  constexpr bool kTwoScales = D == 96 || D >= 192;
  __shared__ float sum_s[HELD * KEYS];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int g = lane >> 4, x = lane & 15;
  const bool keeps = (x >> 2) == g;
  const int B = p.c.B;
  PagedSeq mine = {};
  int64_t n_mine = 0, upto = 0, U = 0;
  int flags = 0;
  auto units_of = [&](const PagedSeq& s) __attribute__((always_inline)) { return weight_units(s, p.c.Hkv, KEYS); };
  auto read_batch = [&](int s0) __attribute__((always_inline)) {
    n_mine = 0;
    if (s0 + lane < B) {
      mine = paged_seq(p.c, s0 + lane);
      n_mine = units_of(mine);
      flags |= mine.flags;
    }
    upto = wave_scan(n_mine, lane, B - s0);
  };
  for (int s0 = 0; s0 < B; s0 += 64) {
    read_batch(s0);
    U += from_lane(upto, B - s0 < 64 ? B - s0 - 1 : 63);
  }
  if (blockIdx.x == 0 && wave == 0 && flags) paged_flag(p.c, flags);
  if (U == 0 || __builtin_amdgcn_ballot_w64(flags & LVSA_PAGED_BAD_CU)) return;
  const int shares = unit_shares(U, p.grid);
  if ((int)blockIdx.x >= shares) return;
  int64_t u = unit_start(U, shares, blockIdx.x);
  const int64_t u_end = unit_start(U, shares, blockIdx.x + 1);
  int seq = 0, held = 0;
  int64_t base = 0;
  for (int s0 = 0; s0 < B; s0 += 64) {
    if (B > 64) read_batch(s0);
    held = s0;
    const uint64_t above = __builtin_amdgcn_ballot_w64(s0 + lane < B && base + upto > u);
    if (above) {
      const int at = __builtin_ctzll(above);
      seq = s0 + at;
      base += from_lane(upto - n_mine, at);
      break;
    }
    base += from_lane(upto, 63);
  }

  struct Keys {
    u32x4 k[BITS == 16 ? T : 1][ND];
    uint32_t c[BITS == 4 ? T : 1][ND], s[T][2];
  };
  while (u < u_end && seq < B) {
    if (seq >= held + 64) read_batch(held += 64);
    const PagedSeq sq = from_lane(mine, seq - held);
    const int64_t units = units_of(sq);
    if (u >= base + units) {
      base += units;
      ++seq;
      continue;
    }
    const int nb = (int)(((int64_t)sq.L + KEYS - 1) / KEYS);
    const int h = (int)quotient(u - base, nb), blk0 = (int)(u - base - (int64_t)h * nb);
    const int blk1 = u_end - u < nb - blk0 ? blk0 + (int)(u_end - u) : nb;
    const int nrows = sq.n * p.group;
    const int32_t* table = p.c.table + seq * p.c.table_str;
    const char* kbase = p.c.k + h * p.c.k_str[2];
    const uint8_t* sbase = BITS == 4 ? p.c.ks + h * p.c.ks_str[2] : nullptr;
    char* wbase = wp.w + h * wp.w_str[2];
    bool bad = false;
    int held_from = blk0;

    shortx8 qf[ND];
    float lse = 0.f;                       // times log2(e)
    int lim = 0;                           // keys that the lane's row gives anything to
    auto load_rows = [&](int r0) __attribute__((always_inline)) {
      const int r = r0 + x < nrows ? r0 + x : nrows - 1;
      const RowRef ref = row_ref(p, sq, h, r);
      const char* qp = p.q + ref.tok * p.q_str[0] + ref.head * p.q_str[1];
#pragma unroll
      for (int i = 0; i < ND; ++i) qf[i] = *reinterpret_cast<const shortx8*>(qp + 2 * (BITS == 16 ? 32 * i + 8 * g : (D / 4) * g + 8 * i));
      lse = wp.lse[ref.tok * p.H + ref.head] * kLog2e;
      lim = r0 + x < nrows && __builtin_fabsf(lse) < __builtin_inff() ? key_limit(p, sq, r) : 0;
    };
    load_rows(0);

    auto key_pos = [&](int b, int j) __attribute__((always_inline)) { return key_within(b * KEYS + wave * KW + 16 * j + x, sq.L); };
    auto load_pages = [&](int b, int* page) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < T; ++j) page[j] = table[page_of(p.c, key_pos(b, j))];
    };
    auto load = [&](int b, const int* page, Keys& st) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < T; ++j) {
        const int pos = key_pos(b, j);
        const PagedRow at = paged_row(p.c, pos, page[j]);
        bad |= !at.ok;
        const char* kr = kbase + at.page * p.c.k_str[0] + at.slot * p.c.k_str[1];
        if constexpr (BITS == 16) {
#pragma unroll
          for (int i = 0; i < ND; ++i) st.k[j][i] = *reinterpret_cast<const u32x4*>(kr + 64 * i + 16 * g);
        } else {
#pragma unroll
          for (int i = 0; i < ND; ++i) st.c[j][i] = reinterpret_cast<const uint32_t*>(kr + (D / 8) * g)[i];
          const uint8_t* s = sbase + at.page * p.c.ks_str[0] + at.slot * p.c.ks_str[1];
          st.s[j][0] = s[(D / 4) * g / 32];
          st.s[j][1] = kTwoScales ? s[((D / 4) * g + D / 4 - 1) / 32] : 0;
        }
      }
    };
    auto compute = [&](int b, const Keys& st) __attribute__((always_inline)) {
      const int key0 = b * KEYS + wave * KW;
      if (key0 >= sq.L) return;
      shortx8 kf[T][ND];
#pragma unroll
      for (int j = 0; j < T; ++j)
#pragma unroll
        for (int i = 0; i < ND; ++i) {
          if constexpr (BITS == 16) kf[j][i] = __builtin_bit_cast(shortx8, st.k[j][i]);
          else kf[j][i] = decode8<E>(st.c[j][i], kTwoScales && ((D / 4) * g + 8 * i) / 32 != (D / 4) * g / 32 ? st.s[j][1] : st.s[j][0]);
        }
      floatx4 acc[T];
#pragma unroll
      for (int j = 0; j < T; ++j) acc[j] = floatx4{0.f, 0.f, 0.f, 0.f};
      int from = 0;                        // the first rows that attend key0
      if (p.causal && key0 > sq.first) from = (key0 - sq.first) * p.group / 16 * 16;
      for (int r0 = nrows > 16 ? from : 0; r0 < nrows; r0 += 16) {
        if (nrows > 16) load_rows(r0);
#pragma unroll
        for (int j = 0; j < T; ++j) {
          floatx4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int i = 0; i < ND; ++i) s = Mat<E>::mfma16(kf[j][i], qf[i], s);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(s[k], p.scale_log2, -lse));
            acc[j][k] += key0 + 16 * j + 4 * g + k < lim ? w : 0.f;
          }
        }
      }
#pragma unroll
      for (int j = 0; j < T; ++j) {
        // sums over the 16 lanes of a group; of the four keys the lane keeps x % 4
        const float a = (x & 1 ? acc[j][1] : acc[j][0]) + __shfl_xor(x & 1 ? acc[j][0] : acc[j][1], 1);
        const float c = (x & 1 ? acc[j][3] : acc[j][2]) + __shfl_xor(x & 1 ? acc[j][2] : acc[j][3], 1);
        float sum = (x & 2 ? c : a) + __shfl_xor(x & 2 ? a : c, 2);
        sum += __shfl_xor(sum, 4);
        sum += __shfl_xor(sum, 8);
        if (keeps) sum_s[(b - held_from) * KEYS + wave * KW + 16 * j + x] = sum;
      }
    };
    // The sums of steps [held_from, b) to the weights, by all waves
    auto flush = [&](int b) __attribute__((always_inline)) {
      __syncthreads();
      for (int k = threadIdx.x; k < (b - held_from) * KEYS; k += 256) {
        const int key = held_from * KEYS + k;
        if (key >= sq.L) break;
        const PagedRow at = paged_row(p.c, key, table[page_of(p.c, key)]);
        if (!at.ok) continue;
        float* w = reinterpret_cast<float*>(wbase + at.page * wp.w_str[0] + at.slot * wp.w_str[1]);
        *w = (wp.accumulate && key < sq.first ? *w : 0.f) + sum_s[k];
      }
      __syncthreads();
      held_from = b;
    };

    // Page numbers are asked for before the keys of the step ahead of theirs: loads come
    // back in order, and behind those keys a wait for them would be one for the keys, with
    // one step on its way instead of two (263 -> 208 us with one work-group on a unit).
    Keys a, z;
    int pa[T], pz[T];
    load_pages(blk0, pa);
    load_pages(blk0 + 1, pz);
    load(blk0, pa, a);
    for (int b = blk0; b < blk1; b += 2) {
      if (b + 1 < blk1) {
        load_pages(b + 2, pa);
        load(b + 1, pz, z);
      }
      __builtin_amdgcn_sched_barrier(0);
      compute(b, a);
      if (b + 1 < blk1) {
        if (b + 2 < blk1) {
          load_pages(b + 3, pz);
          load(b + 2, pa, a);
        }
        __builtin_amdgcn_sched_barrier(0);
        compute(b + 1, z);
      }
      if (b + 2 - held_from >= HELD) flush(b + 2 < blk1 ? b + 2 : blk1);
    }
    flush(blk1);
    if (bad) paged_flag(p.c, LVSA_PAGED_BAD_PAGE);
    u += blk1 - blk0;
  }
}

// Many rows: bound by the exponentials (a lane's 16 per 32 keys and rows take longer
// than their products).  A work-group has 128 keys of a key head, a wave 32 of them in
// registers as its matrix operand; the rows come through LDS for all four, 64 at a
// time (32 of the large heads), and of two tiles of 32 one's exponentials run beside
// the other's products.  A key's sum stays in a register from the first row to the
// last; where there are few keys for the card, work-groups share their rows and
// paged_weights_merge_kernel adds what they found, in their order.
//
// 6500 tokens of prompts over up to 5200 keys, 16 heads over 4 of 64, causal: 78 to 84 us
// and 5 for the sums (181 with a tile of 16 rows at a time from memory, 97 with a division
// per row instead of the next row's address): VALU issuing 63%, MFMA 15%.
template <int D, typename E, int BITS>
__global__ __launch_bounds__(256, D <= 96 ? 3 : 2) void paged_weights_rows_kernel(PagedAttnParams p, WeightsParams wp) {
  constexpr int NK = D / 16, KEYS = kWeightKeys, RB = 2 * D;       // RB: bytes of a row
  constexpr int CH = D / 8, NT = D <= 128 ? 2 : 1, ROWS = 32 * NT, NL = (ROWS * CH + 255) / 256;
  __shared__ __attribute__((aligned(16))) char q_s[2][ROWS * RB];
  __shared__ float lse_s[2][ROWS];
  __shared__ int lim_s[2][ROWS];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int half = lane >> 5, i32 = lane & 31;
  // chunk c (16 bytes) of row r: sixteen rows' reads of one chunk cover the 64 banks once
  auto at_lds = [](int r, int c) __attribute__((always_inline)) {
    return RB * r + 16 * (c ^ (D == 96 ? r >> 2 & 3 : D == 64 || D == 192 ? r >> 1 & 7 : r & 15));
  };
  auto count = [&](const PagedSeq& s) __attribute__((always_inline)) { return weight_units(s, p.c.Hkv, KEYS) * wp.splits; };
  walk_units<true>(p.c, count, [&](int seq, const PagedSeq& sq, int64_t u, int64_t id) __attribute__((always_inline)) {
    const int64_t unit = quotient(u, wp.splits);
    const int split = (int)(u - unit * wp.splits);
    const int chunk = (int)quotient(unit, p.c.Hkv), h = (int)(unit - (int64_t)chunk * p.c.Hkv);
    const int key_wg = chunk * KEYS, key0 = key_wg + 32 * wave;
    const int32_t* table = p.c.table + seq * p.c.table_str;
    shortx8 kf[NK];
    const int pos = key_within(key0 + i32, sq.L);
    const PagedRow at = paged_row(p.c, pos, table[page_of(p.c, pos)]);
    {
      const char* kr = p.c.k + h * p.c.k_str[2] + at.page * p.c.k_str[0] + at.slot * p.c.k_str[1];
      if constexpr (BITS == 16) {
#pragma unroll
        for (int c = 0; c < NK; ++c) kf[c] = *reinterpret_cast<const shortx8*>(kr + 32 * c + 16 * half);
      } else {
        const uint8_t* s = p.c.ks + h * p.c.ks_str[2] + at.page * p.c.ks_str[0] + at.slot * p.c.ks_str[1];
#pragma unroll
        for (int c = 0; c < NK; ++c) kf[c] = decode8<E>(*reinterpret_cast<const uint32_t*>(kr + 8 * c + 4 * half), s[c / 2]);
      }
    }
    if (!at.ok) paged_flag(p.c, LVSA_PAGED_BAD_PAGE);
    const int nrows = sq.n * p.group;
    int from = 0, to = nrows;              // from the first rows that attend any of these keys on
    if (p.causal && key_wg > sq.first) from = (key_wg - sq.first) * p.group / ROWS * ROWS;
    if (wp.splits > 1) {
      const int tiles = (nrows - from + ROWS - 1) / ROWS;
      const int64_t end = quotient((int64_t)tiles * (split + 1), wp.splits) * ROWS;
      to = from + end < nrows ? from + (int)end : nrows;
      from += (int)quotient((int64_t)tiles * split, wp.splits) * ROWS;
    }
    // Each thread's rows of the next tiles, and its lse and limit: ROWS on is step_i
    // tokens and step_j heads, one token more where the heads pass the group's.
    const int step_i = ROWS / p.group, step_j = ROWS - step_i * p.group;
    const int64_t q_step = step_i * p.q_str[0] + step_j * p.q_str[1], q_wrap = p.q_str[0] - p.group * p.q_str[1];
    const char* q0 = p.q + sq.t0 * p.q_str[0] + (int64_t)h * p.group * p.q_str[1];
    struct At {
      int i, j;
    };
    auto start = [&](int row) __attribute__((always_inline)) {
      const int r = from + row, i = (uint32_t)r / (uint32_t)p.group;
      return At{i, r - i * p.group};
    };
    int row[NL], qj[NL];
    const char* qp[NL];
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      row[i] = (threadIdx.x + 256 * i) / CH % ROWS;
      const At at = start(row[i]);
      qj[i] = at.j;
      qp[i] = q0 + at.i * p.q_str[0] + at.j * p.q_str[1] + 16 * ((threadIdx.x + 256 * i) % CH);
    }
    At l_at = start(threadIdx.x % ROWS);
    u32x4 next[NL];
    float lse_next = 0.f;
    int lim_next = 0;
    auto load = [&](int r0) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < NL; ++i) {       // behind the last row: the first one
        next[i] = *reinterpret_cast<const u32x4*>(r0 + row[i] < nrows ? qp[i] : q0);
        qp[i] += q_step;
        qj[i] += step_j;
        if (qj[i] >= p.group) {
          qj[i] -= p.group;
          qp[i] += q_wrap;
        }
      }
      if (wave < NT) {                     // a wave has 32 of them twice
        const int r = threadIdx.x % ROWS;
        const bool in = r0 + r < to;
        lse_next = wp.lse[(int64_t)(sq.t0 + (in ? l_at.i : 0)) * p.H + h * p.group + (in ? l_at.j : 0)] * kLog2e;
        const int64_t e = (int64_t)sq.first + l_at.i + 1;
        lim_next = !in || !(__builtin_fabsf(lse_next) < __builtin_inff()) ? 0 : p.causal && e < sq.L ? (int)e : sq.L;
        l_at.i += step_i;
        l_at.j += step_j;
        if (l_at.j >= p.group) {
          l_at.j -= p.group;
          ++l_at.i;
        }
      }
    };
    auto store = [&](int s) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const int k = threadIdx.x + 256 * i;
        if (ROWS * CH % 256 == 0 || k < ROWS * CH) *reinterpret_cast<u32x4*>(q_s[s] + at_lds(k / CH, k % CH)) = next[i];
      }
      if (threadIdx.x < ROWS) {
        lse_s[s][threadIdx.x] = lse_next;
        lim_s[s][threadIdx.x] = lim_next;
      }
    };
    floatx16 acc = floatx16{0};
    __syncthreads();                       // LDS of the unit before has been read
    if (from < to) {
      load(from);
      store(0);
    }
    __syncthreads();
    int s = 0;
    for (int r0 = from; r0 < to; r0 += ROWS, s ^= 1) {
      if (r0 + ROWS < to) load(r0 + ROWS);
      __builtin_amdgcn_sched_barrier(0);
      floatx16 z[NT];
      float lse[NT];
      int lim[NT];
      bool partly = false;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        lse[t] = lse_s[s][32 * t + i32];
        lim[t] = lim_s[s][32 * t + i32] - key0 - 4 * half;
        partly |= lim[t] < 32 - 4 * half;
        z[t] = floatx16{0};
#pragma unroll
        for (int c = 0; c < NK; ++c)
          z[t] = Mat<E>::mfma32(kf[c], *reinterpret_cast<const shortx8*>(q_s[s] + at_lds(32 * t + i32, 2 * c + half)), z[t]);
      }
      if (__builtin_amdgcn_ballot_w64(partly)) {         // keys behind a row, or a row without weights
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(z[t][k], p.scale_log2, -lse[t]));
            acc[k] += 8 * (k >> 2) + (k & 3) < lim[t] ? w : 0.f;
          }
      } else {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int k = 0; k < 16; ++k) acc[k] += __builtin_amdgcn_exp2f(__builtin_fmaf(z[t][k], p.scale_log2, -lse[t]));
      }
      if (r0 + ROWS < to) store(s ^ 1);
      __syncthreads();
    }
    // Sums over the 32 lanes of a half, in halves of what a lane holds: it ends with key
    // 8 (i32 >> 3) + 4 half + (i32 & 3) of the tile, which is key i32 where bit 2 of i32
    // is the half, and that is the key whose page it looked up.
    float v[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) v[k] = acc[k];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = (i32 & 16 ? v[k + 8] : v[k]) + __shfl_xor(i32 & 16 ? v[k] : v[k + 8], 16);
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = (i32 & 8 ? v[k + 4] : v[k]) + __shfl_xor(i32 & 8 ? v[k] : v[k + 4], 8);
#pragma unroll
    for (int k = 0; k < 2; ++k) v[k] = (i32 & 2 ? v[k + 2] : v[k]) + __shfl_xor(i32 & 2 ? v[k] : v[k + 2], 2);
    float sum = (i32 & 1 ? v[1] : v[0]) + __shfl_xor(i32 & 1 ? v[0] : v[1], 1);
    sum += __shfl_xor(sum, 4);
    const int key = key0 + i32;
    if (((i32 >> 2) & 1) != half || key >= sq.L) return;
    if (wp.splits > 1) {
      wp.ws[id * KEYS + 32 * wave + i32] = sum;
    } else if (at.ok) {
      float* w = reinterpret_cast<float*>(wp.w + at.page * wp.w_str[0] + at.slot * wp.w_str[1] + h * wp.w_str[2]);
      *w = (wp.accumulate && key < sq.first ? *w : 0.f) + sum;
    }
  });
}

// Adds the sums of work-groups that share their rows: a thread per key.
__global__ __launch_bounds__(kWeightKeys) void paged_weights_merge_kernel(PagedAttnParams p, WeightsParams wp) {
  auto count = [&](const PagedSeq& s) __attribute__((always_inline)) { return weight_units(s, p.c.Hkv, kWeightKeys); };
  walk_units<true>(p.c, count, [&](int seq, const PagedSeq& sq, int64_t u, int64_t id) __attribute__((always_inline)) {
    const int chunk = (int)quotient(u, p.c.Hkv), h = (int)(u - (int64_t)chunk * p.c.Hkv);
    const int key = chunk * kWeightKeys + (int)threadIdx.x;
    if (key >= sq.L) return;
    const PagedRow at = paged_row(p.c, key, p.c.table[seq * p.c.table_str + page_of(p.c, key)]);
    float sum = 0.f;
    for (int s = 0; s < wp.splits; ++s) sum += wp.ws[(id * wp.splits + s) * kWeightKeys + threadIdx.x];
    if (!at.ok) return;
    float* w = reinterpret_cast<float*>(wp.w + at.page * wp.w_str[0] + at.slot * wp.w_str[1] + h * wp.w_str[2]);
    *w = (wp.accumulate && key < sq.first ? *w : 0.f) + sum;
  });
}

template <int D, typename E, int BITS>
int paged_weights_launch(const PagedAttnParams& p, const WeightsParams& w, hipStream_t stream) {
  if (w.many) {
    hipLaunchKernelGGL((paged_weights_rows_kernel<D, E, BITS>), dim3((unsigned)p.grid), dim3(256), 0, stream, p, w);
    const int rc = launch_status("lvsa_paged_weights");
    if (rc || w.splits == 1) return rc;
    hipLaunchKernelGGL(paged_weights_merge_kernel, dim3((unsigned)p.grid), dim3(kWeightKeys), 0, stream, p, w);
  } else {
    hipLaunchKernelGGL((paged_weights_kernel<D, E, BITS>), dim3((unsigned)p.grid), dim3(256), 0, stream, p, w);
  }
  return launch_status("lvsa_paged_weights");
}

template <int D>
int paged_weights_launch(const PagedAttnParams& p, const WeightsParams& w, int bits, bool bf16, hipStream_t stream) {
  if (bf16) return bits == 16 ? paged_weights_launch<D, __bf16, 16>(p, w, stream) : paged_weights_launch<D, __bf16, 4>(p, w, stream);
  return bits == 16 ? paged_weights_launch<D, _Float16, 16>(p, w, stream) : paged_weights_launch<D, _Float16, 4>(p, w, stream);
}

}  // namespace
}  // namespace lvsa
