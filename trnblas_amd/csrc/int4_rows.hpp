// Products of 4-bit integer weights with few rows.
#pragma once

#include "int4.hpp"

namespace trnblas {

// A lane's scales and zero points of a chunk: 4 / STEPS of each, loaded at once.
template <int STEPS, bool ZERO>
struct Int4Groups {
  using scales = std::conditional_t<STEPS == 1, u32x2, std::conditional_t<STEPS == 2, uint32_t, uint16_t>>;
  using zeros = std::conditional_t<STEPS == 1, uint32_t, std::conditional_t<STEPS == 2, uint16_t, uint8_t>>;
  scales s;
  zeros z;
  // at: bytes from the buffer's start to the first scale
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t of_scales, __amdgpu_buffer_rsrc_t of_zeros, uint32_t at) {
    if constexpr (STEPS == 1)
      s = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(of_scales, at, 0, 0));
    else if constexpr (STEPS == 2)
      s = __builtin_amdgcn_raw_buffer_load_b32(of_scales, at, 0, 0);
    else
      s = __builtin_amdgcn_raw_buffer_load_b16(of_scales, at, 0, 0);
    if constexpr (ZERO) {
      at = at & kPastEnd | at >> 1;
      if constexpr (STEPS == 1)
        z = __builtin_amdgcn_raw_buffer_load_b32(of_zeros, at, 0, 0);
      else if constexpr (STEPS == 2)
        z = __builtin_amdgcn_raw_buffer_load_b16(of_zeros, at, 0, 0);
      else
        z = __builtin_amdgcn_raw_buffer_load_b8(of_zeros, at, 0, 0);
    }
  }
  __device__ __forceinline__ float scale(int step, int f16) const {
    uint32_t w;
    if constexpr (STEPS == 1)
      w = s[step / 2] >> 16 * (step & 1);
    else if constexpr (STEPS == 2)
      w = s >> 16 * (step / 2);
    else
      w = s;
    return int4_scale((uint16_t)w, f16);
  }
  __device__ __forceinline__ uint32_t zero(int step) const {
    if constexpr (ZERO) return (uint32_t)z >> 8 * (step / STEPS) & 255u;
    return 8;
  }
};

// Tiles of 16 MF rows by 128 NF / ks columns of D (GATED: 128 / ks, NF = 2, gates and, N rows of the
// matrix later, ups). ks of the eight waves split K (chunk c of 128 values to wave c % ks)
// and add their sums through LDS in wave order; 8 / ks such sets take NF blocks of 16 columns each. Codes
// go from memory into registers as the matrix instruction takes them, U chunks under way per wave, the
// rows one chunk ahead. A group's products are summed by themselves, exact weights, and
// enter the sum times their scale in fp32. P: A is so many pieces whose sum it is.
template <typename T, int P, int MF, int NF, int STEPS, bool ZERO, bool GATED>
__global__ __launch_bounds__(512) void int4_rows_kernel(GroupedArgs g, Int4Args q, int ks) {
  constexpr int BM = 16 * MF, BW = GATED ? 16 : 16 * NF, U = P * MF * NF == 1 ? 8 : 4, PRE = P * MF <= 2 ? 2 : 1;
  __shared__ __attribute__((aligned(16))) float part[NF][8][BM * 16];
  Segment s;
  if (!ragged_tile<BM>(g, blockIdx.x, 8, s)) return;
  const bool of_group = s.group >= 0 && s.group < g.groups;
  const int lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kw = wave % ks, set = wave / ks, sets = 8 / ks;
  const int n0 = (s.tn * sets + set) * BW;
  const int nc = of_group && n0 < g.N ? q.chunks : 0;
  const int64_t grp = of_group ? s.group : 0;
  // buffers at the tile's first row block and row; the lane's offsets in them
  __amdgpu_buffer_rsrc_t rb[NF], rs[NF], rz[NF], ra[P];
  uint32_t ob[NF], os[NF], oa[MF];
#pragma unroll
  for (int b = 0; b < NF; ++b) {
    const int64_t first = GATED ? (b ? (int64_t)g.N + n0 : n0) : n0 + 16 * b, last = GATED && b ? 2 * (int64_t)g.N - 1 : g.N - 1;
    const int64_t block = __builtin_amdgcn_readfirstlane((int)(min(first, last) >> 4)), n = min(first + li, last);
    rb[b] = buffer_at(q.codes + grp * q.codes_step + block * q.chunks * kInt4Chunk);
    rs[b] = buffer_at(q.scales + grp * q.groups_step + block * q.chunks * (64 / STEPS));
    if constexpr (ZERO) rz[b] = buffer_at(q.zeros + grp * q.groups_step + block * q.chunks * (64 / STEPS));
    const uint32_t row = (uint32_t)(n >> 4) - (uint32_t)block ? q.chunks * 16 : 0;
    ob[b] = row * 64 + 16 * (16 * lg + (uint32_t)(n & 15));
    os[b] = (row + (uint32_t)(n & 15)) * (8 / STEPS);
  }
#pragma unroll
  for (int p = 0; p < P; ++p) ra[p] = buffer_at(static_cast<const T*>(g.A) + p * q.a_step + s.row * g.lda);
#pragma unroll
  for (int a = 0; a < MF; ++a) oa[a] = (uint32_t)(min(16 * a + li, s.end - 1 - s.row) * (int)g.lda + 8 * lg) * 2;
  f32x4 sum[NF][MF];
#pragma unroll
  for (int b = 0; b < NF; ++b)
#pragma unroll
    for (int a = 0; a < MF; ++a) sum[b][a] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  struct Chunk {
    i32x4 w[NF];
    Int4Groups<STEPS, ZERO> of[NF];
  } c[U];
  struct Rows {
    i32x4 v[P][MF][4];
  } x[PRE];
  // chunk i, or zeros where it is not inside; no branch, so that all loads stay under way
  auto load = [&](Chunk& v, int i, bool inside) __attribute__((always_inline)) {
    const uint32_t at = inside ? (uint32_t)i * kInt4Chunk : kPastEnd, groups = inside ? (uint32_t)i * (128 / STEPS) : kPastEnd;
#pragma unroll
    for (int b = 0; b < NF; ++b) {
      v.w[b] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(rb[b], ob[b] + at, 0, 0));
      v.of[b].load(rs[b], rz[b], os[b] + groups);
    }
  };
  auto load_rows = [&](Rows& v, uint32_t at) __attribute__((always_inline)) {
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int a = 0; a < MF; ++a)
#pragma unroll
        for (int t = 0; t < 4; ++t)
          v.v[p][a][t] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(ra[p], oa[a] + at + 64 * t, 0, 0));
  };
  auto multiply = [&](const Chunk& v, const Rows& r) __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < NF; ++b)
#pragma unroll
      for (int t0 = 0; t0 < 4; t0 += STEPS) {
        const uint32_t z = int4_zero<T>(v.of[b].zero(t0));
        f32x4 acc[MF];
#pragma unroll
        for (int t = t0; t < t0 + STEPS; ++t) {
          const i32x4 fb = int4_values<T, ZERO>(v.w[b][t], z);
#pragma unroll
          for (int a = 0; a < MF; ++a)
#pragma unroll
            for (int p = 0; p < P; ++p)
              acc[a] = int4_mma<T>(r.v[p][a][t], fb, t == t0 && p == 0 ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : acc[a]);
        }
        const float f = v.of[b].scale(t0, q.scale_f16);
#pragma unroll
        for (int a = 0; a < MF; ++a)
#pragma unroll
          for (int e = 0; e < 4; ++e) sum[b][a][e] = __builtin_fmaf(f, acc[a][e], sum[b][a][e]);
      }
  };
  const int whole = nc > 0 ? g.K / 128 : 0;
  for (int i = kw; i < whole; i += ks * U) {
#pragma unroll
    for (int u = 0; u < U; ++u) load(c[u], i + ks * u, i + ks * u < whole);
    load_rows(x[0], (uint32_t)i * 256);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int next = i + ks * (u + 1);
      if (PRE == 2 && u + 1 < U) load_rows(x[(u + 1) & 1], next < whole ? (uint32_t)next * 256 : kPastEnd);
      if (i + ks * u < whole) multiply(c[u], x[u & (PRE - 1)]);
      if (PRE == 1 && u + 1 < U) load_rows(x[0], next < whole ? (uint32_t)next * 256 : kPastEnd);
    }
  }
  if (whole < nc && kw == whole % ks) {  // the last chunk, of fewer values: those past the rows' end are read as zeros
    load(c[0], whole, true);
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int a = 0; a < MF; ++a) {
          const int k = 128 * whole + 32 * t;
          x[0].v[p][a][t] =
              __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(ra[p], k + 8 * lg < g.K ? oa[a] + 2 * k : kPastEnd, 0, 0));
        }
    multiply(c[0], x[0]);
  }
#pragma unroll
  for (int b = 0; b < NF; ++b)
#pragma unroll
    for (int a = 0; a < MF; ++a)
#pragma unroll
      for (int r = 0; r < 4; ++r) part[b][wave][(16 * a + 4 * lg + r) * 16 + li] = kInt4Unit<T> * sum[b][a][r];
  __syncthreads();
  constexpr int BLOCKS = GATED ? 1 : NF;
  for (int i = threadIdx.x; i < sets * BLOCKS * BM * 4; i += 512) {
    const int w = i / (BLOCKS * BM * 4), b = i / (BM * 4) % BLOCKS, e = i % (BM * 4);
    auto total = [&](int block) __attribute__((always_inline)) {
      f32x4 v = *reinterpret_cast<const f32x4*>(&part[block][w * ks][4 * e]);
      for (int p = 1; p < ks; ++p) v += *reinterpret_cast<const f32x4*>(&part[block][w * ks + p][4 * e]);
      return v;
    };
    const int m = s.row + e / 4, n = (s.tn * sets + w) * BW + 16 * b + 4 * (e % 4);
    if (m >= s.end) continue;
    if constexpr (GATED)
      int4_store<true>(g, m, n, total(0), total(1));
    else
      int4_store<false>(g, m, n, total(b), f32x4{});
  }
}

}  // namespace trnblas
