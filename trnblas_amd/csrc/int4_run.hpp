// The launches of the products of 4-bit integer weights for one type of rows.
#pragma once

#include <algorithm>

#include "int4_rows.hpp"

namespace trnblas {

static const char* const kInt4Gemm = "trnblas_hip_int4_gemm";

// Bound on the tiles of bm rows (see ragged_tile), in whole rounds of the XCDs.
static int int4_grid(const GroupedArgs& g, int bm, unsigned* grid) {
  const int64_t tiles = (g.rows / bm + std::min<int64_t>(g.groups + 2, g.rows)) * g.tiles_n;
  TRNBLAS_CHECK_ARG(tiles < ((int64_t)1 << 31) - 4096, "%s: too many tiles", kInt4Gemm);
  *grid = (unsigned)((tiles + kNumXcd - 1) / kNumXcd * kNumXcd);
  return TRNBLAS_OK;
}

template <typename T, int P, int MF, bool GATED>
static int run_int4_rows(GroupedArgs g, const Int4Args& q, int ks, hipStream_t s) {
  g.tiles_n = (g.N + 128 / ks - 1) / (128 / ks);
  unsigned grid;
  if (int rc = int4_grid(g, 16 * MF, &grid)) return rc;
  auto kernel = q.zeros ? int4_rows_kernel<T, P, MF, true, GATED> : int4_rows_kernel<T, P, MF, false, GATED>;
  hipLaunchKernelGGL(kernel, dim3(grid), dim3(512), 0, s, g, q, ks);
  return check_launch(kInt4Gemm);
}

template <typename T, int P, bool GATED>
static int run_int4(const GroupedArgs& g, const Int4Args& q, hipStream_t s) {
  const Int4Choice c = choose_int4(g.rows, g.groups, g.N, g.K, P);
  if constexpr (P == 1) {
    if (c.mf == 4) return run_int4_rows<T, P, 4, GATED>(g, q, c.ks, s);
  }
  if (c.mf >= 2) return run_int4_rows<T, P, 2, GATED>(g, q, c.ks, s);
  return run_int4_rows<T, P, 1, GATED>(g, q, c.ks, s);
}

template <typename T>
int int4_gemm_run(const GroupedArgs& g, const Int4Args& q, int pieces, bool gated, hipStream_t s) {
  if constexpr (std::is_same_v<T, __bf16>) {
    if (pieces == 3) return gated ? run_int4<T, 3, true>(g, q, s) : run_int4<T, 3, false>(g, q, s);
  }
  return gated ? run_int4<T, 1, true>(g, q, s) : run_int4<T, 1, false>(g, q, s);
}

}  // namespace trnblas
