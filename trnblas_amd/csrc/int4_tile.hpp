// Products of 4-bit integer weights with many rows.
#pragma once

#include "int4_rows.hpp"

namespace trnblas {

// The LDS of a tile of 128 rows by 256 columns: stages of a chunk, 128 values of k: rows in two
// panels of 64 values, codes, scales, zero points.
template <int STEPS>
struct Int4Stage {
  static constexpr int PANEL = 128 * 128, B = 2 * PANEL, S = B + 16 * kInt4Chunk, Z = S + 16 * 128 / STEPS, BYTES = Z + 16 * 64 / STEPS;
  static constexpr int STAGES = 3;
};

// Tiles of 128 rows by 256 columns (GATED: 128 of gates and, N rows of the matrix later, 128 of ups; N a multiple of 16), eight waves
// of 64 x 64: sums of a group in one set of registers, those of all groups in another. All operands
// come by LDS DMA, chunk c + 2 behind the barrier that says that every wave has read chunk c - 1 and that c
// has landed. Codes become operands in registers, once in each of the two waves that share them.
// pieces: K is walked so many times, each time with another piece of A.
template <typename T, int STEPS, bool ZERO, bool GATED>
__global__ __launch_bounds__(512) void int4_tile_kernel(GroupedArgs g, Int4Args q, int pieces) {
  using L = Int4Stage<STEPS>;
  using DA = PanelDma<T, 128, true, 8>;
  using PA = typename DA::P;
  constexpr int FM = 4, FN = 4, HALVES = GATED ? 2 : 1, FH = FN / HALVES, BN = 256 / HALVES;
  constexpr int ND = 2 * DA::NB + 2 + 1 + ZERO;  // DMAs per wave and chunk
  __shared__ __attribute__((aligned(16))) char lds[L::STAGES * L::BYTES];
  Segment s;
  if (!ragged_tile<128>(g, blockIdx.x, 8, s)) return;
  const bool of_group = s.group >= 0 && s.group < g.groups;
  const int lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave & 1, wn = wave >> 1;
  const int64_t grp = of_group ? s.group : 0;
  const int n0 = s.tn * BN;
  const int chunks = of_group ? q.chunks : 0, nc = chunks * pieces;
  TileJob j;
  j.m = s.row, j.n = n0 + wn * (16 * FH);
  j.rows_a = min(128, s.end - s.row);
  j.C = g.C, j.D = g.D;

  // the two blocks of columns that this wave moves: 2 wave, 2 wave + 1 of the tile's sixteen, where waves wn's four are
  // 4 wn .. (GATED: two of gates, then two of ups)
  const int first = GATED ? 2 * (wave >> 1) : 2 * wave;
  const bool ups = GATED && (wave & 1);
  const int have = __builtin_amdgcn_readfirstlane(min(max((g.N - n0 + 15) / 16 - first, 0), 2));  // of them inside
  const int64_t block = (n0 >> 4) + first + (ups ? g.N >> 4 : 0);
  const uint8_t* codes = q.codes + grp * q.codes_step + block * q.chunks * kInt4Chunk;
  const uint8_t* scales = reinterpret_cast<const uint8_t*>(q.scales + grp * q.groups_step + block * q.chunks * (64 / STEPS));
  const uint8_t* zeros = ZERO ? q.zeros + grp * q.groups_step + block * q.chunks * (64 / STEPS) : nullptr;
  constexpr int SP = 8 / STEPS, ZP = 4 / STEPS;  // 16-byte pieces of a block's scales, zero points
  const uint32_t os = lane / SP < have ? (uint32_t)(lane / SP) * q.chunks * (128 / STEPS) + 16 * (lane % SP) : kPastEnd;
  const uint32_t oz = lane / ZP < have ? (uint32_t)(lane / ZP) * q.chunks * (64 / STEPS) + 16 * (lane % ZP) : kPastEnd;
  const char* corner = static_cast<const char*>(g.A) + s.row * g.lda * (int64_t)sizeof(T);
  DA da;
  da.init(corner, g.lda, j.rows_a, wave, lane);
  const uint32_t lds0 = lds_offset(lds);
  int piece = 0, at = 0;  // of the next chunk to move
  auto dma_chunk = [&](int c) __attribute__((always_inline)) {
    const bool inside = c < nc;
    const uint32_t st = lds0 + (uint32_t)c % L::STAGES * L::BYTES;
    if (at == chunks && piece + 1 < pieces) {
      ++piece, at = 0;
      da.base = corner + piece * q.a_step * (int64_t)sizeof(T);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int left = g.K - 128 * at - 64 * h;
      if (left > 0 && left < 64) da.last(left, wave, lane);
      const i32x4 ra = dma_rsrc(da.base, inside && left > 0 ? kRecords : 0);
      each<DA::NB>([&](auto uc) __attribute__((always_inline)) {
        constexpr int u = decltype(uc)::value;
        lds_dma<1024 * u>(ra, st + h * L::PANEL + DA::NB * 1024 * wave, da.off[u]);
      });
      da.base += da.step;
    }
    const i32x4 b0 = dma_rsrc(codes + (int64_t)at * kInt4Chunk, inside && have > 0 ? kRecords : 0);
    const i32x4 b1 = dma_rsrc(codes + ((int64_t)q.chunks + at) * kInt4Chunk, inside && have > 1 ? kRecords : 0);
    lds_dma<0>(b0, st + L::B + 2048 * wave, 16 * lane);
    lds_dma<1024>(b1, st + L::B + 2048 * wave, 16 * lane);
    // of the lanes that have a piece: the others would write zeros to what is next to it
    if (lane < 2 * SP) lds_dma<0>(dma_rsrc(scales + at * (128 / STEPS), inside ? kRecords : 0), st + L::S + wave * (256 / STEPS), os);
    if constexpr (ZERO) {
      if (lane < 2 * ZP) lds_dma<0>(dma_rsrc(zeros + at * (64 / STEPS), inside ? kRecords : 0), st + L::Z + wave * (128 / STEPS), oz);
    }
    ++at;
  };

  f32x4 sum[HALVES][FM][FH];
#pragma unroll
  for (int b = 0; b < FN; ++b)
#pragma unroll
    for (int a = 0; a < FM; ++a) sum[b / FH][a][b % FH] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  if (nc > 0) {
    dma_chunk(0);
    dma_chunk(1);
  }
  uint32_t oa[PA::NV];
  PA::lane_offsets(64 * wm, lane, oa);
  for (int c = 0; c < nc; ++c) {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(ND) : "memory");
    dma_chunk(c + 2);
    const char* st = lds + (uint32_t)c % L::STAGES * L::BYTES;
    i32x4 w[FN];
    uint32_t z[FN];
    uint16_t sc[FN][4][4 / STEPS] __attribute__((aligned(16)));
#pragma unroll
    for (int b = 0; b < FN; ++b) {
      const int blk = 4 * wn + b;
      w[b] = *reinterpret_cast<const i32x4*>(st + L::B + blk * kInt4Chunk + 16 * lane);
      const char* ps = st + L::S + blk * (128 / STEPS) + lg * (32 / STEPS);
      if constexpr (STEPS == 4) {
        *reinterpret_cast<u32x2*>(sc[b]) = *reinterpret_cast<const u32x2*>(ps);
      } else {
#pragma unroll
        for (int h = 0; h < 2 / STEPS; ++h) reinterpret_cast<i32x4*>(sc[b])[h] = reinterpret_cast<const i32x4*>(ps)[h];
      }
      if constexpr (ZERO) {
        const char* pz = st + L::Z + blk * (64 / STEPS) + li * (4 / STEPS);
        z[b] = STEPS == 4   ? *reinterpret_cast<const uint8_t*>(pz)
               : STEPS == 2 ? *reinterpret_cast<const uint16_t*>(pz)
                            : *reinterpret_cast<const uint32_t*>(pz);
      }
    }
    f32x4 acc[FM][FN];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const char* pa[PA::NV];
#pragma unroll
      for (int v = 0; v < PA::NV; ++v) pa[v] = st + (t >> 1) * L::PANEL + oa[v];
      i32x4 fa[FM];
#pragma unroll
      for (int a = 0; a < FM; ++a) fa[a] = PA::frag(pa, a, t & 1);
#pragma unroll
      for (int b = 0; b < FN; ++b) {
        const i32x4 fb = int4_values<T, ZERO>(w[b][t], int4_zero<T>(ZERO ? z[b] >> 8 * (t / STEPS) & 255u : 8u));
#pragma unroll
        for (int a = 0; a < FM; ++a) {
          if (t % STEPS == 0) acc[a][b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
          mma_tile<T>(acc[a][b], fb, fa[a]);
        }
      }
      if ((t + 1) % STEPS == 0) {
#pragma unroll
        for (int b = 0; b < FN; ++b) {
          float f[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) f[r] = int4_scale(sc[b][r][t / STEPS], q.scale_f16);
#pragma unroll
          for (int a = 0; a < FM; ++a)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              sum[b / FH][a][b % FH][r] = __builtin_fmaf(f[r], acc[a][b][r], sum[b / FH][a][b % FH][r]);
        }
      }
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no DMA into the LDS of the next workgroup
  if constexpr (GATED) {
#pragma unroll
    for (int a = 0; a < FM; ++a)
#pragma unroll
      for (int b = 0; b < FH; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          sum[0][a][b][r] = gate(g.act, kInt4Unit<T> * sum[0][a][b][r]) * (kInt4Unit<T> * sum[1][a][b][r]);
  } else {
    g.alpha *= kInt4Unit<T>;
  }
  char* own = lds + wave * kStoreLds<FH>;
  static_assert(8 * kStoreLds<FH> <= sizeof(lds));
  __syncthreads();  // the other waves' reads
  if (g.out32)
    store_wave<FM, FH, float, !GATED>(g, j, sum[0], 64 * wm, 0, lane, own);
  else if (g.out_f16)
    store_wave<FM, FH, _Float16, !GATED>(g, j, sum[0], 64 * wm, 0, lane, own);
  else
    store_wave<FM, FH, __bf16, !GATED>(g, j, sum[0], 64 * wm, 0, lane, own);
}

}  // namespace trnblas
