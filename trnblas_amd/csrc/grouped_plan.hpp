// Which kernel a grouped product runs on: from its sizes, types and alignment
// only (the group sizes are on the device), by estimated times.
#pragma once

#include <algorithm>
#include <cmath>

#include "common.hpp"

namespace trnblas {

// Times of the ring kernels (us), fitted to sweeps of 1 .. 64 groups and 1 .. 16384
// rows over matrices of 512 x 512 .. 2048 x 4096 (bf16 / fp4): a tile takes `start`
// and, per k-tile, from `alone` (an empty GPU) to `full` (all slots taken). Of 228
// sizes, each run on all three, the choice is the fastest within 10 % at all but 12,
// and within 30 % at all. 256 rows, 4096 x 1024: 27.3, 27.4 and 21.4 us (64 x 128 has
// the most tiles); 4096 rows: 62, 51 and 55; 16384 rows, 2048 x 4096: 225, 256, 316.
// 4-bit tiles of 64 x 128 fit twice into a CU's LDS with their scales; over 263 sizes of
// quantised operands the choice is within 10 % of the fastest kernel at all but 8.
struct RingCost {
  int fm, fn;      // MFMA blocks of a wave: tile 32 fm x 32 fn
  int per_cu;      // workgroups of a CU
  double start, alone, full;
};
constexpr RingCost kRing16[] = {{8, 8, 1, 10.0, 0.95, 1.5}, {4, 4, 2, 4.0, 0.38, 1.12}, {2, 4, 3, 3.3, 0.36, 1.08}};
constexpr RingCost kRing4[] = {{8, 8, 1, 11.0, 1.2, 1.6}, {4, 4, 2, 5.5, 0.5, 1.12}, {2, 4, 2, 4.2, 0.42, 0.86}};

inline double ring_time(const RingCost& c, double tiles, double k_tiles) {
  const double t = tiles / (c.per_cu * device_cus());
  // several workgroups of a CU drift apart; one runs in whole rounds, what is left of the last cut into quarters (tile_of)
  const double part = t - std::floor(t);
  if (c.per_cu == 1 && t <= 0.75) return 1e30;  // nothing but quarters: the 128 x 128 kernel's tiles, one per CU
  const double rounds = c.per_cu > 1 ? std::max(1.0, t <= 1.0 ? 1.0 : t + 0.3)
                                     : std::floor(t) + (part > 0.75 ? 1.0 : 0.45 * std::ceil(4.0 * part));
  return rounds * (c.start + k_tiles * (c.alone + (c.full - c.alone) * std::min(1.0, t)));
}

// Row tiles of BM rows that `rows` rows in `groups` groups are likely to take: each
// group that has any rows ends in a tile half full.
inline double likely_row_tiles(double rows, double groups, int bm) {
  if (groups <= 1) return std::ceil(rows / bm);
  const double g = std::min(groups, rows);
  return std::max(g, rows / bm + 0.5 * g);
}

struct GroupedChoice {
  int ring;    // index into kRing16 / kRing4 (fp32: 2 or kAnyTiles), or -1: rows_kernel
  int mf, ks;  // rows_kernel: row blocks, waves along K
};

// grouped_gemm and mx_gemm. row_bytes: of A along K; elem: bytes per value of B.
inline GroupedChoice choose_grouped(const RingCost (&ring)[3], double rows, double groups, double N, double K, double row_bytes,
                                    double elem, bool kc) {
  const double g = std::min(groups, rows), weights = g * K * N * elem, nk = std::ceil(row_bytes / 128.0);
  GroupedChoice best{-1, 1, 8};
  // Few rows: rows_kernel reads the weights once per 16 mf rows at about 4.5 TB/s
  // (two row blocks of a K-contiguous B: 3.2), its waves splitting K; the rings
  // need a tile per CU to read as fast, and read K-contiguous values at 3.9 TB/s. 8
  // groups of one row, 4096 x 1536: 19 us, the rings 27 (96 tiles); 16 groups of one,
  // 2048 x 4096, K-contiguous 58 and 73, otherwise 60 and 54.
  double time = 1e30;
  if (rows <= 64.0 * g) {
    best.mf = rows <= 8.0 * g ? 1 : 2;
    const double again = likely_row_tiles(rows, groups, 16 * best.mf) / g;
    time = 4.5 + row_bytes / 8192.0 + weights * again / (best.mf == 2 && kc ? 3.2e6 : 4.5e6);
    // the fewest waves along K that leave two workgroups per CU: one block of rows of a K-contiguous
    // B, and every 4-bit form, have kernels for it (elsewhere the rings mostly have enough tiles before)
    if (kc && (best.mf == 1 || elem < 2))
      while (best.ks > 1 && again * g * std::ceil(N * (best.ks / 2) / 128.0) >= 2.0 * device_cus()) best.ks /= 2;
  }
  for (int i = 0; i < 3; ++i) {
    const RingCost& c = ring[i];
    const double t = std::max(3.0 + weights / (kc && elem >= 2 ? 3.9e6 : 4.6e6),
                              ring_time(c, likely_row_tiles(rows, groups, 32 * c.fm) * std::ceil(N / (32 * c.fn)), nk));
    // bound by the weights alike: the smaller tiles keep more loads under way (32
    // groups of 32 rows, 4096 x 1024 of 4-bit values: 37.0, 18.6 and 17.0 us)
    if (i ? t <= time : t < time) {
      time = t;
      best.ring = i;
    }
  }
  return best;
}

// mx_gemm: rows_kernel's costs and the rings' over bytes of codes.
inline GroupedChoice choose_mx(double rows, double groups, double N, double K) {
  const double bytes = std::ceil(K / 32.0) * 16.0;
  return choose_grouped(kRing4, rows, groups, N, bytes, bytes, 17.0 / 16.0, true);
}

// Whether rows_kernel quantises a K-contiguous A of values itself: one block of rows, and no more
// than kInPlace values in it (its LDS).
constexpr int kInPlace = 32768;
inline bool quantised_in_place(const GroupedChoice& c, int64_t rows, int64_t K) {
  return c.ring < 0 && c.mf == 1 && std::min<int64_t>(rows, 16) * K <= kInPlace;
}

// fp32: its MFMAs take eight times as long, so its kernels have costs of their own, fitted to 266
// sizes of 1 .. 64 groups and 1 .. 8192 rows in either layout, each run on all kernels (of 532,
// the choice is within 10 % of the fastest at all but 62, and 1.9 % slower over all): the
// rings' 64 x 128 tiles; grouped_any_kernel's 32 x 64, by layout of B (column-, K-contiguous),
// which spread better below two or three rounds; rows_kernel on one block of rows. 32 rows in 2
// groups, 4096 x 1536: 138, 66 and 42 us; 128 in 64, 1024 x 2048: 141, 111 and 121; 8192 in 4, 2048 x
// 4096: 1023 and 1392.
constexpr RingCost kRing32 = {2, 4, 3, 6.7, 0.86, 2.7};
constexpr RingCost kAny32[] = {{1, 2, 4, 4.7, 0.43, 1.25}, {1, 2, 4, 4.0, 0.41, 1.1}};
constexpr int kAnyTiles = 3;  // GroupedChoice::ring: grouped_any_kernel

inline GroupedChoice choose_f32(double rows, double groups, double N, double K, bool kc) {
  const double g = std::min(groups, rows), weights = 4.0 * g * K * N, nk = std::ceil(K / 32.0);
  GroupedChoice best{2, 1, 8};
  double time = std::max(3.0 + weights / 3.2e6, ring_time(kRing32, likely_row_tiles(rows, groups, 64) * std::ceil(N / 128), nk));
  const double any = std::max(3.0 + weights / (kc ? 4.45e6 : 4.6e6),
                              ring_time(kAny32[kc], likely_row_tiles(rows, groups, 32) * std::ceil(N / 64), nk));
  if (any < time) time = any, best.ring = kAnyTiles;
  if (rows <= 64.0 * g) {
    const double tiles = likely_row_tiles(rows, groups, 16), again = tiles / g - 1.0;  // weights read again
    if ((kc ? 6.6 + K * 7.8e-4 + weights * (1.0 / 4.35e6 + again / 4.2e6)
            : 5.1 + K * 4.8e-3 + weights * (1.0 / 5.6e6 + again / 8.7e6)) < time) {
      best.ring = -1;
      for (int ks : {4, 1})  // two: sizes that the 32 x 64 tiles serve
        if (kc && tiles * std::ceil(N * ks / 128.0) >= 2.0 * device_cus()) best.ks = ks;
    }
  }
  return best;
}

// grouped_gemm of aligned operands
inline GroupedChoice choose_gemm(int elem_bytes, double rows, double groups, double N, double K, bool kc) {
  return elem_bytes == 4 ? choose_f32(rows, groups, N, K, kc)
                         : choose_grouped(kRing16, rows, groups, N, K, K * elem_bytes, elem_bytes, kc);
}

// gated_gemm: by the costs of a product of all 2 N columns. rows_kernel: a workgroup takes half
// as many columns of H, hence the fewest waves along K that leave two workgroups per CU of
// these (fp32: eight or one, the sizes between run on the ring).
inline GroupedChoice choose_gated(int elem_bytes, double rows, double groups, double N, double K, bool kc) {
  GroupedChoice c = choose_gemm(elem_bytes, rows, groups, 2.0 * N, K, kc);
  if (c.ring == kAnyTiles) c.ring = 2;
  c.ks = 8;
  if (c.ring < 0 && kc && c.mf == 1)
    for (const int step = elem_bytes == 4 ? 8 : 2;
         c.ks > 1 && likely_row_tiles(rows, groups, 16) * std::ceil(N * (c.ks / step) / 128.0) >= 2.0 * device_cus();)
      c.ks /= step;
  return c;
}

// int4_gemm: the tile kernel's rows (0: the few-rows kernel) and parts of K, or blocks of 16 rows and of 16 columns
// of a wave, and waves along K, of the few-rows kernel.
struct Int4Choice {
  int mf, nf, ks, tile, splits;
};
constexpr int kInt4Reach = 0x7ffffff0;  // bytes of scales that the tile kernel reads from one address

// Times (us) fitted to sweeps of 1 .. 2048 rows over matrices of 2048 .. 8192 squared and of 130 random sizes, dense and
// of up to 64 groups, where the choice took 1.05 times what the best of all forms did. The few-rows kernel: a workgroup
// alone on its CU takes `alone` for each chunk of a wave, several take `busy`; of a block's sixteen rows those count
// that are there, the others are read from the first level's cache. The tile kernel's tiles as in ring_time; parts of K:
// what writes and reads their sums. steps: of 32 values per group: a group's sums are taken at its end. 64 rows,
// 8192 x 8192: few rows 36, tiles of 64 in four parts 28, in one 52, of 128 106; 2048 rows: 1025, 376, 285, 237.
inline Int4Choice choose_int4(double rows, double groups, double N, double K, int steps, int pieces, bool gated) {
  const double cus = device_cus(), chunks = std::ceil(K / 128.0), columns = gated ? 2.0 * N : N, chain = chunks * pieces;
  const double per = rows / std::max(1.0, std::min(groups, rows)), folds = steps == 4 ? 0.0 : steps == 2 ? 0.15 : 0.45;
  Int4Choice best{1, 2, 8, 0, 1};
  double time = 1e30;
  for (int mf : {1, 2, 4}) {
    if (mf == 4 && pieces == 3) break;
    const double filled = std::min(1.0, per / (16.0 * mf));
    for (int nf : {2, 1}) {
      if (nf == 1 && (mf > 1 || gated)) continue;
      double alone = nf == 1 ? 0.35 + 0.45 * filled : 0.72 + 0.33 * filled, busy = nf == 1 ? 0.42 + 0.58 * filled : 0.15 + 0.95 * filled;
      if (mf > 1) alone = 0.45 * mf + 0.45 * mf * filled, busy = 0.15 * mf + 0.85 * mf * filled;
      alone += 0.3 * folds * mf, busy += folds * mf;
      if (pieces == 3) alone *= 2.5, busy *= 2.5;
      for (int ks : {8, 4, 2, 1}) {
        const double r = likely_row_tiles(rows, groups, 16 * mf) * std::ceil(columns * ks / (128.0 * nf)) / cus, n = std::ceil(chunks / ks);
        const double rounds = r <= 1.0 ? 0.0 : r < 4.0 ? std::ceil(r) : r + 0.5;
        const double t = 2.0 + std::max(2.6 + n * alone, rounds * (1.3 + n * busy));
        if (t < time) time = t, best = {mf, nf, ks, 0, 1};
      }
    }
  }
  // (gates and ups: whole row blocks of each, and the ups' scales within the one buffer that starts at the gates')
  const bool tiles = !gated || (std::fmod(N, 16.0) == 0.0 && (N / 16.0 * chunks + 1.0) * (128 / steps) <= kInt4Reach);
  for (int tile : {64, 128})
    for (int splits : {1, 2, 4, 8}) {
      const double sums = splits * rows * columns * 4.0;
      if (!tiles || (splits > 1 && (tile == 128 || chain < 2.0 * splits || sums > 256e6))) break;
      const double slots = tile == 64 ? 2.0 * cus : cus;
      const double r = likely_row_tiles(rows, groups, tile) * std::ceil(columns / (2.0 * tile)) * splits / slots;
      const double busy = tile == 64 ? std::min(1.0, std::max(0.0, 2.0 * r - 1.0)) : std::min(1.0, r);
      const double each = (tile == 64 ? 0.75 + 0.43 * busy : 1.58 + 0.3 * busy) * (1.0 + 0.7 * folds);
      const double rounds = r <= 1.0 ? 1.0 : tile == 64 ? r + 0.3 : std::ceil(r);
      const double t = rounds * (4.2 + std::ceil(chain / splits) * each) + (splits > 1 ? 2.5 + sums / 2.7e6 : 0.0);
      if (t < time) time = t, best = {1, 2, 8, tile, splits};
    }
  return best;
}

// grouped_rank_k of aligned operands: groups x (M x N), over the average group's k-tiles. fp32 has
// the 64 x 128 tiles alone: three workgroups per CU hide its longer MFMAs' steps.
inline int choose_rank_k(int elem_bytes, double groups, double rows, double M, double N) {
  if (elem_bytes == 4) return 2;
  const double k_tiles = rows / groups * elem_bytes / 128.0;
  int best = 0;
  double time = 1e30;
  for (int i = 0; i < 3; ++i) {
    const RingCost& c = kRing16[i];
    const double t = ring_time(c, groups * std::ceil(M / (32 * c.fm)) * std::ceil(N / (32 * c.fn)), k_tiles + 0.5);
    if (t < time) {
      time = t;
      best = i;
    }
  }
  return best;
}

}  // namespace trnblas
