// Products of 4-bit integer weights with many rows.
#pragma once

#include "int4_rows.hpp"

namespace trnblas {

// lds_dma without a memory clobber.
template <int AT>
__device__ __forceinline__ void lds_dma_free(const i32x4& rsrc, uint32_t lds, uint32_t voff) {
  asm volatile("s_add_u32 m0, %0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(voff), "s"(rsrc), "n"(AT)
               : "m0", "scc");
}

// The same for the wave's first LANES lanes, with no branch; the others write nothing.
template <int AT, int LANES>
__device__ __forceinline__ void lds_dma_few(const i32x4& rsrc, uint32_t lds, uint32_t voff) {
  asm volatile("s_add_u32 m0, %0, %3\n\ts_mov_b64 exec, %4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds\n\ts_mov_b64 exec, -1" ::"s"(lds),
               "v"(voff), "s"(rsrc), "n"(AT), "n"((1 << LANES) - 1)
               : "m0", "scc");
}

// The LDS of a tile of 16 FM rows by 32 WAVES columns: stages of a chunk, 128 values of k: rows in two
// panels of 64 values, codes, scales, zero points.
template <int FM, int WAVES, int STEPS>
struct Int4Stage {
  static constexpr int PANEL = 16 * FM * 128, B = 2 * PANEL, S = B + 2 * WAVES * kInt4Chunk, Z = S + 2 * WAVES * 128 / STEPS,
                       BYTES = Z + 2 * WAVES * 64 / STEPS;
  static constexpr int STAGES = 3;
};

// Tiles of 16 FM rows by 32 WAVES columns (GATED: half of them gates and, N rows of the matrix later, as many ups; N a multiple of 16),
// waves of all rows by 32 columns, so that each code becomes an operand once. All operands come by LDS DMA, chunk c + 2 behind the barrier that says that
// every wave has read chunk c - 1 and that c has landed. A group's sums are in one set of registers, those of all
// groups in another. What bounds it is the vector unit: a matrix instruction of 16 cycles keeps it out for 8 of them, and
// eight values of codes take 13 instructions (fp16: 11) of 4 cycles, a group's 64 sums of a lane one each: 2048 rows by
// 8192^2 in groups of 128 237 us, 1.16 PFLOP/s. (Waves of 64 x 64, which make each operand twice: 286.)
// pieces: K is walked so many times, each time with another piece of A. q.splits > 1: the grid's y takes so many parts
// of that walk; their sums go to q.partial (g.rows rows of q.ldp values each), for int4_join_kernel.
template <typename T, int FM, int WAVES, int STEPS, bool ZERO, bool SF16, bool GATED>
__global__ __launch_bounds__(64 * WAVES, 2) void int4_tile_kernel(GroupedArgs g, Int4Args q, int pieces) {
  using L = Int4Stage<FM, WAVES, STEPS>;
  using DA = PanelDma<T, 16 * FM, true, WAVES>;
  using PA = typename DA::P;
  constexpr int BM = 16 * FM, FN = 2, HALVES = GATED ? 2 : 1, FH = FN / HALVES, BN = 32 * WAVES / HALVES;
  constexpr int ND = 2 * DA::NB + 2 + 1 + ZERO;  // DMAs per wave and chunk
  __shared__ __attribute__((aligned(16))) char lds[L::STAGES * L::BYTES];
  Segment s;
  if (!ragged_tile<BM>(g, blockIdx.x, 8, s)) return;
  const bool of_group = s.group >= 0 && s.group < g.groups;
  const int lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t grp = of_group ? s.group : 0;
  const int n0 = s.tn * BN;
  const int chunks = of_group ? q.chunks : 0;
  // this part of the chunks (of all pieces)
  const int per = (chunks * pieces + q.splits - 1) / q.splits, begin = min((int)blockIdx.y * per, chunks * pieces);
  const int nc = min(per, chunks * pieces - begin);
  TileJob j;
  j.m = s.row, j.n = n0 + wave * (16 * FH);
  j.rows_a = min(BM, s.end - s.row);
  j.C = g.C, j.D = g.D;

  // the wave's two blocks of columns, which it moves and multiplies (GATED: one of gates, one of ups)
  const int have = __builtin_amdgcn_readfirstlane(min(max((g.N - n0 + 15) / 16 - FH * wave, 0), FH)) * HALVES;  // of them inside
  const int64_t block = (n0 >> 4) + FH * wave;
  const int apart = GATED ? g.N >> 4 : 1;  // blocks from the first to the second
  const uint8_t* codes = q.codes + grp * q.codes_step + block * q.chunks * kInt4Chunk;
  const uint8_t* scales = reinterpret_cast<const uint8_t*>(q.scales + grp * q.groups_step + block * q.chunks * (64 / STEPS));
  const uint8_t* zeros = ZERO ? q.zeros + grp * q.groups_step + block * q.chunks * (64 / STEPS) : nullptr;
  constexpr int SP = 8 / STEPS, ZP = 4 / STEPS;  // 16-byte pieces of a block's scales, zero points
  static_assert(kInt4Reach <= kRecords);         // (choose_int4)
  const uint32_t os = lane / SP < have ? (uint32_t)(lane / SP) * apart * q.chunks * (128 / STEPS) + 16 * (lane % SP) : kPastEnd;
  const uint32_t oz = lane / ZP < have ? (uint32_t)(lane / ZP) * apart * q.chunks * (64 / STEPS) + 16 * (lane % ZP) : kPastEnd;
  const char* corner = static_cast<const char*>(g.A) + s.row * g.lda * (int64_t)sizeof(T);
  DA da;
  da.init(corner, g.lda, j.rows_a, wave, lane);
  const uint32_t lds0 = lds_offset(lds);
  // buffers at the next chunk to move; of a chunk past the last one zeros are read
  i32x4 ra = dma_rsrc(corner, nc > 0 ? kRecords : 0);
  i32x4 rb[2] = {dma_rsrc(codes, have > 0 ? kRecords : 0), dma_rsrc(codes + (int64_t)apart * q.chunks * kInt4Chunk, have > 1 ? kRecords : 0)};
  i32x4 rs = dma_rsrc(scales, kRecords), rz = dma_rsrc(zeros, kRecords);
  auto advance = [](i32x4& r, int64_t bytes) __attribute__((always_inline)) {
    const uint64_t p = ((uint64_t)(uint32_t)r[1] << 32 | (uint32_t)r[0]) + bytes;
    r[0] = (int)(uint32_t)p, r[1] = (int)(uint32_t)(p >> 32);
  };
  uint32_t off[2][DA::NB];
#pragma unroll
  for (int u = 0; u < DA::NB; ++u) off[0][u] = da.off[u], off[1][u] = da.off[u] == kPastEnd ? kPastEnd : da.off[u] + 128;
  int piece = chunks ? begin / chunks : 0, at = begin - piece * chunks;  // of the next chunk to move
  advance(ra, (piece * q.a_step + 128 * (int64_t)at) * (int64_t)sizeof(T));
  advance(rb[0], (int64_t)at * kInt4Chunk), advance(rb[1], (int64_t)at * kInt4Chunk);
  advance(rs, (int64_t)at * (128 / STEPS)), advance(rz, (int64_t)at * (64 / STEPS));
  uint32_t to = lds0;                                                     // its stage
  // before the first DMA of a chunk
  auto dma_turn = [&](int c) __attribute__((always_inline)) {
    const int left = g.K - 128 * at;  // values of k
    if (left < 128) {
      if (c >= nc) {
        ra[2] = rb[0][2] = rb[1][2] = rs[2] = rz[2] = 0;
      } else if (left > 0) {
#pragma unroll
        for (int u = 0; u < DA::NB; ++u) {
          int r, k;
          PA::where((DA::NB * wave + u) * 64 + lane, r, k);
          if (k >= left) off[0][u] = kPastEnd;
          if (k + 64 >= left) off[1][u] = kPastEnd;
        }
      }
    }
  };
  // DMA i of a chunk; without a memory clobber: LDS reads may pass it, they are of other stages
  auto dma = [&](auto ic) __attribute__((always_inline)) {
    constexpr int i = decltype(ic)::value;
    if constexpr (i < 2 * DA::NB)
      lds_dma_free<i / DA::NB * L::PANEL + 1024 * (i % DA::NB)>(ra, to + DA::NB * 1024 * wave, off[i / DA::NB][i % DA::NB]);
    else if constexpr (i < 2 * DA::NB + 2)
      lds_dma_free<L::B + 1024 * (i - 2 * DA::NB)>(rb[i - 2 * DA::NB], to + 2048 * wave, 16 * lane);
    else if constexpr (i == 2 * DA::NB + 2)  // the lanes that have a piece: others would write zeros to what is next to it
      lds_dma_few<L::S, 2 * SP>(rs, to + wave * (256 / STEPS), os);
    else if constexpr (i < ND)
      lds_dma_few<L::Z, 2 * ZP>(rz, to + wave * (128 / STEPS), oz);
  };
  // after its last
  auto dma_done = [&](int c) __attribute__((always_inline)) {
    to = to == lds0 + (L::STAGES - 1) * L::BYTES ? lds0 : to + L::BYTES;
    if (++at == chunks && piece + 1 < pieces) {
      ++piece, at = 0;
      const i32x4 r = dma_rsrc(corner + piece * q.a_step * (int64_t)sizeof(T), kRecords);
      ra[0] = r[0], ra[1] = r[1];
      const int64_t back = -(int64_t)(chunks - 1);
      advance(rb[0], back * kInt4Chunk), advance(rb[1], back * kInt4Chunk);
      advance(rs, back * (128 / STEPS)), advance(rz, back * (64 / STEPS));
    } else {
      advance(ra, 256), advance(rb[0], kInt4Chunk), advance(rb[1], kInt4Chunk), advance(rs, 128 / STEPS), advance(rz, 64 / STEPS);
    }
  };

  f32x4 sum[HALVES][FM][FH];
#pragma unroll
  for (int b = 0; b < FN; ++b)
#pragma unroll
    for (int a = 0; a < FM; ++a) sum[b / FH][a][b % FH] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  if (nc > 0) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      dma_turn(c);
      each<ND>(dma);
      dma_done(c);
    }
  }
  uint32_t oa[PA::NV];
  PA::lane_offsets(0, lane, oa);
  const char* st = lds;
  for (int c = 0; c < nc; ++c) {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(ND) : "memory");
    dma_turn(c + 2);
    i32x4 w[FN];
    uint32_t z[FN];
    uint16_t sc[FN][4][4 / STEPS] __attribute__((aligned(16)));
#pragma unroll
    for (int b = 0; b < FN; ++b) {
      const int blk = 2 * wave + b;
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
    i32x4 fa[2][FM];
    auto read_rows = [&](int t) __attribute__((always_inline)) {
#pragma unroll
      for (int a = 0; a < FM; ++a) fa[t & 1][a] = *reinterpret_cast<const i32x4*>(st + oa[t & 1] + (t >> 1) * L::PANEL + 2048 * a);
    };
    read_rows(0);
    each<4>([&](auto tc) __attribute__((always_inline)) {
      constexpr int t = decltype(tc)::value;
      if constexpr (t < 3) read_rows(t + 1);
      dma(std::integral_constant<int, 2 * t>{});  // two a step
      dma(std::integral_constant<int, 2 * t + 1>{});
#pragma unroll
      for (int b = 0; b < FN; ++b) {
        const i32x4 fb = int4_values<T, ZERO>(w[b][t], int4_zero<T>(ZERO ? z[b] >> 8 * (t / STEPS) & 255u : 8u));
#pragma unroll
        for (int a = 0; a < FM; ++a) acc[a][b] = int4_mma<T>(fb, fa[t & 1][a], t % STEPS == 0 ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : acc[a][b]);
      }
      if constexpr ((t + 1) % STEPS == 0) {
#pragma unroll
        for (int b = 0; b < FN; ++b) {
          float f[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) f[r] = int4_scale(sc[b][r][t / STEPS], SF16);
#pragma unroll
          for (int a = 0; a < FM; ++a) {
            f32x4& v = sum[b / FH][a][b % FH];
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] = __builtin_fmaf(f[r], acc[a][b][r], v[r]);
            asm volatile("" : "+v"(v));  // here: the compiler would put all of a chunk's behind its last step
          }
        }
      }
      __builtin_amdgcn_sched_barrier(0);  // a step's registers at a time
    });
    dma_done(c + 2);
    st = st == lds + (L::STAGES - 1) * L::BYTES ? lds : st + L::BYTES;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no DMA into the LDS of the next workgroup
  char* own = lds + wave * kStoreLds<FH>;
  static_assert(WAVES * kStoreLds<FH> <= sizeof(lds));
  __syncthreads();  // the other waves' reads
  if (q.splits > 1) {
    GroupedArgs p = g;
    p.alpha = kInt4Unit<T>, p.ldd = q.ldp, p.vec4 = q.ldp % 4 == 0;
    j.D = q.partial + blockIdx.y * (g.rows * q.ldp);
    store_wave<FM, FH, float, false>(p, j, sum[0], 0, 0, lane, own);
    if constexpr (GATED) {
      j.D = static_cast<float*>(j.D) + g.N;
      store_wave<FM, FH, float, false>(p, j, sum[1], 0, 0, lane, own);
    }
    return;
  }
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
  if (g.out32)
    store_wave<FM, FH, float, !GATED>(g, j, sum[0], 0, 0, lane, own);
  else if (g.out_f16)
    store_wave<FM, FH, _Float16, !GATED>(g, j, sum[0], 0, 0, lane, own);
  else
    store_wave<FM, FH, __bf16, !GATED>(g, j, sum[0], 0, 0, lane, own);
}

}  // namespace trnblas
