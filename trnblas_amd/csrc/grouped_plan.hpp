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
  int ring;    // index into kRing16 / kRing4, or -1: rows_kernel
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
    while (best.ks > 1 && kc && (best.mf == 1 || elem < 2) && again * g * std::ceil(N * (best.ks / 2) / (kc ? 128.0 : 512.0)) >= 2.0 * device_cus()) best.ks /= 2;
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

// fp32 (its MFMAs take eight times as long): below two 64 x 128 tiles per CU the 32 x
// 64 ones of grouped_any_kernel spread better, aligned or not. 300 rows in 4 groups by
// 2048 x 1024 35 us, the rings 72; 2000 in 8 by 1024^2 60 and 72; 4096 in 8 by 2048^2
// (1088 tiles) 370 and 310.
inline bool f32_small_tiles(double rows, double groups, double N) {
  return likely_row_tiles(rows, groups, 64) * std::ceil(N / 128) < 2.0 * device_cus();
}

// grouped_rank_k: groups x (M x N), k_tiles of the average group.
inline int choose_rank_k(double groups, double M, double N, double k_tiles) {
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
