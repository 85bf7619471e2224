// Products of 4-bit integer weights with few rows.
#pragma once

#include "int4.hpp"

namespace trnblas {

// Tiles of 16 MF rows by 128 / ks columns. ks of the eight waves split K (chunk c of 128 values to wave c % ks)
// and add their sums through LDS in wave order; 8 / ks such sets take 16 columns each. Codes go from
// memory into registers as the matrix instruction takes them, U chunks under way per wave. A
// group's products are summed by themselves, exact weights, and enter the sum times their
// scale in fp32. P: A is so many pieces whose sum it is. GATED: gates and, N rows of the
// matrix later, ups.
template <typename T, int P, int MF, bool ZERO, bool GATED>
__global__ __launch_bounds__(512) void int4_rows_kernel(GroupedArgs g, Int4Args q, int ks) {
  constexpr int BM = 16 * MF, HALVES = GATED ? 2 : 1, U = 4;
  __shared__ __attribute__((aligned(16))) float part[HALVES][8][BM * 16];
  Segment s;
  if (!ragged_tile<BM>(g, blockIdx.x, 8, s)) return;
  const bool of_group = s.group >= 0 && s.group < g.groups;
  const int lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kw = wave % ks, set = wave / ks, sets = 8 / ks;
  const int n0 = (s.tn * sets + set) * 16;
  const int nc = of_group && n0 < g.N ? q.chunks : 0;
  const int64_t grp = of_group ? s.group : 0;
  const int per_chunk = 4 / q.steps;  // groups
  const uint8_t* pb[HALVES];
  int64_t ps[HALVES];  // of the first group's scale
#pragma unroll
  for (int h = 0; h < HALVES; ++h) {
    const int64_t n = min(n0 + li, g.N - 1) + (h ? g.N : 0);
    pb[h] = q.codes + grp * q.codes_step + (n >> 4) * q.chunks * kInt4Chunk + 16 * (16 * lg + (int)(n & 15));
    ps[h] = grp * q.groups_step + (n >> 4) * q.chunks * per_chunk * 16 + (n & 15);
  }
  const T* pa[P][MF];
#pragma unroll
  for (int a = 0; a < MF; ++a) {
    const int64_t m = min(s.row + 16 * a + li, s.end - 1);
#pragma unroll
    for (int p = 0; p < P; ++p) pa[p][a] = static_cast<const T*>(g.A) + p * q.a_step + m * g.lda + 8 * lg;
  }
  f32x4 sum[HALVES][MF], acc[HALVES][MF];
#pragma unroll
  for (int h = 0; h < HALVES; ++h)
#pragma unroll
    for (int a = 0; a < MF; ++a) sum[h][a] = acc[h][a] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  struct Chunk {
    i32x4 w[HALVES];
    uint16_t scale[HALVES][4];
    uint8_t zero[HALVES][4];
  } c[U];
  auto load = [&](Chunk& v, int i) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < HALVES; ++h) {
      v.w[h] = *reinterpret_cast<const i32x4*>(pb[h] + (int64_t)i * kInt4Chunk);
#pragma unroll
      for (int t = 0; t < 4; ++t)  // a group's stand with its last step
        if (((t + 1) & (q.steps - 1)) == 0) {
          const int64_t at = ps[h] + ((int64_t)i * per_chunk + (t >> (q.steps >> 1))) * 16;
          v.scale[h][t] = q.scales[at];
          if constexpr (ZERO) v.zero[h][t] = q.zeros[at];
        }
    }
  };
  auto multiply = [&](const Chunk& v, int i) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int k = 128 * i + 32 * t;
      i32x4 fa[P][MF];
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int a = 0; a < MF; ++a)
          fa[p][a] = k + 8 * lg < g.K ? *reinterpret_cast<const i32x4*>(pa[p][a] + k) : i32x4{0, 0, 0, 0};
      const bool ends = ((t + 1) & (q.steps - 1)) == 0;
#pragma unroll
      for (int h = 0; h < HALVES; ++h) {
        uint32_t z = 8;
        if constexpr (ZERO) {
          const uint32_t z1 = v.zero[h][t], z2 = v.zero[h][t | 1], z4 = v.zero[h][3];
          z = q.steps == 1 ? z1 : q.steps == 2 ? z2 : z4;
        }
        const i32x4 fb = int4_values<T, ZERO>(v.w[h][t], int4_zero<T>(z));
#pragma unroll
        for (int a = 0; a < MF; ++a)
#pragma unroll
          for (int p = 0; p < P; ++p) acc[h][a] = int4_mma<T>(fa[p][a], fb, acc[h][a]);
        if (ends) {
          const float f = int4_scale(v.scale[h][t], q.scale_f16);
#pragma unroll
          for (int a = 0; a < MF; ++a) {
#pragma unroll
            for (int r = 0; r < 4; ++r) sum[h][a][r] = __builtin_fmaf(f, acc[h][a][r], sum[h][a][r]);
            acc[h][a] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
          }
        }
      }
    }
  };
  for (int i = kw; i < nc; i += ks * U) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i + ks * u < nc) load(c[u], i + ks * u);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i + ks * u < nc) multiply(c[u], i + ks * u);
  }
#pragma unroll
  for (int h = 0; h < HALVES; ++h)
#pragma unroll
    for (int a = 0; a < MF; ++a)
#pragma unroll
      for (int r = 0; r < 4; ++r) part[h][wave][(16 * a + 4 * lg + r) * 16 + li] = kInt4Unit<T> * sum[h][a][r];
  __syncthreads();
  for (int i = threadIdx.x; i < sets * BM * 4; i += 512) {
    const int w = i / (BM * 4), e = i % (BM * 4);
    f32x4 v[HALVES];
#pragma unroll
    for (int h = 0; h < HALVES; ++h) {
      v[h] = *reinterpret_cast<const f32x4*>(&part[h][w * ks][4 * e]);
      for (int p = 1; p < ks; ++p) v[h] += *reinterpret_cast<const f32x4*>(&part[h][w * ks + p][4 * e]);
    }
    const int m = s.row + e / 4, n = (s.tn * sets + w) * 16 + 4 * (e % 4);
    if (m >= s.end) continue;
    int4_store<GATED>(g, m, n, v[0], v[HALVES - 1]);
  }
}

}  // namespace trnblas
