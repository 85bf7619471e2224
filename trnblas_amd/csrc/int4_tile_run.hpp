// The launches of the tile kernel of 4-bit integer weights for one type of rows.
#pragma once

#include "int4_tile.hpp"

namespace trnblas {

template <typename T, int FM, int WAVES, int STEPS, bool SF16, bool GATED>
static int run_int4_tile(GroupedArgs g, const Int4Args& q, int pieces, hipStream_t s) {
  constexpr int BN = GATED ? 16 * WAVES : 32 * WAVES;
  g.tiles_n = (g.N + BN - 1) / BN;
  unsigned grid;
  if (int rc = int4_grid(g, 16 * FM, &grid)) return rc;
  auto kernel = q.zeros ? int4_tile_kernel<T, FM, WAVES, STEPS, true, SF16, GATED> : int4_tile_kernel<T, FM, WAVES, STEPS, false, SF16, GATED>;
  hipLaunchKernelGGL(kernel, dim3(grid, q.splits), dim3(64 * WAVES), 0, s, g, q, pieces);
  return check_launch(kInt4Gemm);
}

template <typename T, int STEPS, bool SF16, bool GATED>
static int run_int4_tiles(const GroupedArgs& g, const Int4Args& q, int pieces, int rows, hipStream_t s) {
  return rows == 64 ? run_int4_tile<T, 4, 4, STEPS, SF16, GATED>(g, q, pieces, s) : run_int4_tile<T, 8, 8, STEPS, SF16, GATED>(g, q, pieces, s);
}

template <typename T, int STEPS>
static int run_int4_tile_steps(const GroupedArgs& g, const Int4Args& q, int pieces, bool gated, int rows, hipStream_t s) {
  if (gated)
    return q.scale_f16 ? run_int4_tiles<T, STEPS, true, true>(g, q, pieces, rows, s) : run_int4_tiles<T, STEPS, false, true>(g, q, pieces, rows, s);
  return q.scale_f16 ? run_int4_tiles<T, STEPS, true, false>(g, q, pieces, rows, s) : run_int4_tiles<T, STEPS, false, false>(g, q, pieces, rows, s);
}

template <typename T>
int int4_tile_run(const GroupedArgs& g, const Int4Args& q, int pieces, bool gated, int rows, hipStream_t s) {
  return q.steps == 1   ? run_int4_tile_steps<T, 1>(g, q, pieces, gated, rows, s)
         : q.steps == 2 ? run_int4_tile_steps<T, 2>(g, q, pieces, gated, rows, s)
                        : run_int4_tile_steps<T, 4>(g, q, pieces, gated, rows, s);
}

}  // namespace trnblas
