// The launches of gated projections for one element type; gated_f32.hip, gated_bf16.hip
// and gated_f16.hip compile them side by side.
#pragma once

#include "grouped_run.hpp"

namespace trnblas {

static const char* const kGated = "trnblas_hip_gated_gemm";

template <typename T>
static bool gated_ready(const GroupedArgs& g, bool bkc) {
  return dma_ready<T>(g, bkc, false) && g.sU * (int64_t)sizeof(T) % 16 == 0;
}

template <typename T, int FM, int FN, bool BKC>
static int run_gated_ring(GroupedArgs g, hipStream_t s) {
  g.tiles_n = (g.N + 16 * FN - 1) / (16 * FN);
  unsigned grid;
  if (int rc = grid_of(ring_grid<FM, FN>(g, row_tiles(g.rows, g.groups, 32 * FM) * g.tiles_n), kGated, &grid)) return rc;
  hipLaunchKernelGGL((gated_ring_kernel<T, FM, FN, BKC>), dim3(grid), dim3(256), 0, s, g);
  return check_launch(kGated);
}

template <typename T, int MF, int NF, int KS, bool BKC>
static int run_gated_rows(GroupedArgs g, hipStream_t s) {
  constexpr int BN = 128 * NF / KS;
  g.tiles_n = (g.N + BN - 1) / BN;
  unsigned grid;
  if (int rc = grid_of(row_tiles(g.rows, g.groups, 16 * MF) * g.tiles_n, kGated, &grid)) return rc;
  grid = (grid + kNumXcd - 1) / kNumXcd * kNumXcd;
  hipLaunchKernelGGL((rows_kernel<T, MF, NF, KS, BKC, void, false, true>), dim3(grid), dim3(512), 0, s, g, MxScales{});
  return check_launch(kGated);
}

template <typename T, bool BKC>
static int run_gated(const GroupedArgs& g, hipStream_t s) {
  const GroupedChoice c = choose_gated(sizeof(T), g.rows, g.groups, g.N, g.K, BKC);
  if constexpr (sizeof(T) == 2) {
    if (c.ring == 0) return run_gated_ring<T, 8, 8, BKC>(g, s);
    if (c.ring == 1) return run_gated_ring<T, 4, 4, BKC>(g, s);
  }
  if (c.ring >= 0) return run_gated_ring<T, 2, 4, BKC>(g, s);
  constexpr int NF = BKC ? 1 : 4;
  if constexpr (sizeof(T) == 2) {  // the fp32 plan has one block of rows
    if (c.mf == 2) return run_gated_rows<T, 2, NF, 8, BKC>(g, s);
  }
  if constexpr (BKC) {
    if constexpr (sizeof(T) == 2) {
      if (c.ks == 4) return run_gated_rows<T, 1, NF, 4, BKC>(g, s);
      if (c.ks == 2) return run_gated_rows<T, 1, NF, 2, BKC>(g, s);
    }
    if (c.ks == 1) return run_gated_rows<T, 1, NF, 1, BKC>(g, s);
  }
  return run_gated_rows<T, 1, NF, 8, BKC>(g, s);
}

template <typename T>
int gated_gemm_run(const GroupedArgs& g, bool bkc, hipStream_t s) {
  TRNBLAS_CHECK_ARG(bkc ? gated_ready<T>(g, true) : gated_ready<T>(g, false),
                    "%s: operands must start and continue on 16 bytes (or be padded), a tile's rows within 2^31 bytes", kGated);
  return bkc ? run_gated<T, true>(g, s) : run_gated<T, false>(g, s);
}

}  // namespace trnblas
