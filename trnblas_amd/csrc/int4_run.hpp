// The launches of the products of 4-bit integer weights for one type of rows.
#pragma once

#include <algorithm>

#include "int4_rows.hpp"

namespace trnblas {

template <typename T, int P, int MF, int NF, int STEPS, bool GATED>
static int run_int4_rows(GroupedArgs g, const Int4Args& q, int ks, hipStream_t s) {
  constexpr int BN = GATED ? 128 : 128 * NF;
  g.tiles_n = (g.N + BN / ks - 1) / (BN / ks);
  unsigned grid;
  if (int rc = int4_grid(g, 16 * MF, &grid)) return rc;
  auto kernel = q.zeros ? int4_rows_kernel<T, P, MF, NF, STEPS, true, GATED> : int4_rows_kernel<T, P, MF, NF, STEPS, false, GATED>;
  hipLaunchKernelGGL(kernel, dim3(grid), dim3(512), 0, s, g, q, ks);
  return check_launch(kInt4Gemm);
}

template <typename T, int P, int STEPS, bool GATED>
static int run_int4(const GroupedArgs& g, const Int4Args& q, hipStream_t s) {
  const Int4Choice c = choose_int4(g.rows, g.groups, g.N, 128.0 * q.chunks, STEPS, P, GATED);
  if constexpr (P == 1) {
    if (c.mf == 4) return run_int4_rows<T, P, 4, 2, STEPS, GATED>(g, q, c.ks, s);
  }
  if (c.mf >= 2) return run_int4_rows<T, P, 2, 2, STEPS, GATED>(g, q, c.ks, s);
  if constexpr (!GATED) {
    if (c.nf == 1) return run_int4_rows<T, P, 1, 1, STEPS, GATED>(g, q, c.ks, s);
  }
  return run_int4_rows<T, P, 1, 2, STEPS, GATED>(g, q, c.ks, s);
}

template <typename T, int P>
static int run_int4_steps(const GroupedArgs& g, const Int4Args& q, bool gated, hipStream_t s) {
  if (q.steps == 1) return gated ? run_int4<T, P, 1, true>(g, q, s) : run_int4<T, P, 1, false>(g, q, s);
  if (q.steps == 2) return gated ? run_int4<T, P, 2, true>(g, q, s) : run_int4<T, P, 2, false>(g, q, s);
  return gated ? run_int4<T, P, 4, true>(g, q, s) : run_int4<T, P, 4, false>(g, q, s);
}

template <typename T>
int int4_gemm_run(const GroupedArgs& g, const Int4Args& q, int pieces, bool gated, hipStream_t s) {
  if constexpr (std::is_same_v<T, __bf16>) {
    if (pieces == 3) return run_int4_steps<T, 3>(g, q, gated, s);
  }
  return run_int4_steps<T, 1>(g, q, gated, s);
}

}  // namespace trnblas
