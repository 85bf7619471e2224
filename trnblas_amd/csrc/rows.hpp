// The grouped products of few rows per group (serving): the weights are read
// once, straight into registers.
#pragma once

#include "gemm.hpp"
#include "grouped_plan.hpp"
#include "mx_block.hpp"
#include "ring.hpp"

namespace trnblas {

typedef i32x4 __attribute__((aligned(2))) i32x4_at2;
typedef i32x4 __attribute__((aligned(4))) i32x4_at4;

// 16 bytes at any alignment of T.
template <typename T>
__device__ __forceinline__ i32x4 load16(const char* p) {
  using loose = std::conditional_t<sizeof(T) == 1, i32x4, std::conditional_t<sizeof(T) == 2, i32x4_at2, i32x4_at4>>;
  return *reinterpret_cast<const loose*>(p);
}

// Steps of a chunk, and chunks that a wave loads before it multiplies.
template <typename T>
constexpr int rows_steps = sizeof(T) == 1 ? 4 : 2;
template <typename T>
constexpr int rows_ahead(int mf, int nf) {
  return (mf + nf <= 3 ? 8 : 4) / rows_steps<T>;
}

// NF MFMA operands of 16 columns over one step of 64 bytes of k, as loaded from
// a B whose columns are contiguous: lane (li, lg) loads columns 4 li .. + 3 of the k
// rows of its group, so operand j is columns 4 li + j.
template <typename T>
struct ColumnStep {
  static constexpr int ES = sizeof(T), KR = 16 / ES;  // k rows of a lane
  using word = std::conditional_t<ES == 2, u32x2, i32x4>;
  word w[KR];
  // p: B at (k of the lane's first row, its first column); rows of k inside
  __device__ __forceinline__ void load(const char* p, int64_t ld) {
#pragma unroll
    for (int e = 0; e < KR; ++e) w[e] = *reinterpret_cast<const word*>(p + e * ld * ES);
  }
  __device__ __forceinline__ void load_last(const char* p, int64_t ld, int rows) {
#pragma unroll
    for (int e = 0; e < KR; ++e) w[e] = e < rows ? *reinterpret_cast<const word*>(p + e * ld * ES) : word{};
  }
  __device__ __forceinline__ i32x4 operand(int j) const {
    i32x4 v;
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      if constexpr (ES == 4)
        v[d] = w[d][j];
      else  // halves j of rows 2 d and 2 d + 1
        v[d] = (int)__builtin_amdgcn_perm(w[2 * d + 1][j / 2], w[2 * d][j / 2], j % 2 ? 0x07060302u : 0x05040100u);
    }
    return v;
  }
};

// Quantises nr rows of x.x from row `row` on into LDS, one block of 32 values per
// thread at a time: rows of g.lda bytes of codes, 16 bytes apart, and scale
// dwords (row, chunk of 512 values, quarter q: the blocks 4 h + q, h = 0 .. 3).
template <typename X>
__device__ __forceinline__ void quantize_rows(const GroupedArgs& g, const MxScales& x, int row, int nr, char* codes, char* scales) {
  const int blocks = x.chunks * 16, have = (int)g.lda / 16;
  for (int i = threadIdx.x; i < nr * blocks; i += 512) {
    const int r = i / blocks, b = i - r * blocks;
    uint32_t byte = 0;
    if (b < have) {
      const X* p = static_cast<const X*>(x.x) + (row + r) * x.ldx + 32 * b;
      const int left = x.kx - 32 * b;
      float v[4][8];
      if (x.vec && left >= 32) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          union {
            i32x4 w[sizeof(X) / 2];
            X e[8];
          } u;
#pragma unroll
          for (int h = 0; h < (int)sizeof(X) / 2; ++h) u.w[h] = reinterpret_cast<const i32x4*>(p + 8 * q)[h];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[q][e] = (float)u.e[e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e / 8][e % 8] = e < left ? (float)p[e] : 0.0f;
      }
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < 32; ++e) top = max(top, __builtin_bit_cast(uint32_t, v[e / 8][e % 8]) & 0x7fffffffu);
      byte = scale_byte(top);
      i32x4 c = {0, 0, 0, 0};
      if (byte != 255) {
#pragma unroll
        for (int q = 0; q < 4; ++q) c[q] = (int)codes8(v[q], inverse_scale(byte));
      }
      *reinterpret_cast<i32x4*>(codes + r * ((int)g.lda + 16) + 16 * b) = c;
    }
    scales[r * x.chunks * 16 + (b >> 4) * 16 + 4 * (b & 3) + ((b >> 2) & 3)] = (char)byte;
  }
}

// Tiles of 16 MF rows by BN columns. KS of the eight waves split K between them
// (chunks of CH bytes per row, chunk c to wave c % KS) and add their sums through
// LDS in wave order; 8 / KS such sets take 16 NF columns each. What bounds it is
// reading B: each wave has U chunks of loads in flight before it multiplies, no
// LDS and no barrier in the loop; KS is chosen so that a wave has U chunks or
// more, or the GPU enough workgroups (choose_grouped).
// K-contiguous B: one row of 64 bytes per lane quad and step. Column-contiguous B: NF
// = 4, whole 128-byte lines of 16-bit values. Rows of A past the segment and columns past
// N repeat the last ones (not stored). Operands as for the ring kernels: groups of 16
// bytes along a row lie inside it, or in its padding, or outside as a whole (operands
// that start anywhere: 8 groups of a row, 4095 x 1535, 69 us here with a branch per
// load, 33 on grouped_any_kernel). One row of bf16 by 4096 x 1536 9 us, 16 groups of a
// row by 2048 x 4096 58 us (4.6 TB/s); 4-bit 8192^2 and one row 9.4 (3.8). fp32 and CHAINS (see kChain16): the
// sums restart every 512 values of k per wave.
//
// X (4-bit floats only): A comes as values of that type, at most kInPlace in the
// tile's rows; the workgroup quantises them into LDS behind its first loads of B,
// which saves a launch of its own (one row of 8192 by 8192^2: 5 us).
template <typename T, int MF, int NF, int KS, bool BKC, typename X = void, bool CHAINS = false>
__global__ __launch_bounds__(512) void rows_kernel(GroupedArgs g, MxScales x) {
  constexpr bool MX = std::is_same_v<T, fp4x2>, FOLD = std::is_same_v<T, float> || CHAINS;
  constexpr int ES = sizeof(T), EV = 16 / ES, BM = 16 * MF, BW = 16 * NF, BN = 8 / KS * BW;
  constexpr int STEPS = rows_steps<T>, CH = 64 * STEPS, CK = CH / ES;  // a chunk: bytes, values of k
  constexpr int U = rows_ahead<T>(MF, NF);
  static_assert(BKC || NF == 4, "four columns of a lane");
  constexpr bool QUANT = !std::is_void_v<X>;
  __shared__ __attribute__((aligned(16))) f32x4 part[8][BM * BW / 4];
  Segment s;
  if (!ragged_tile<BM>(g, blockIdx.x, 8, s)) return;
  const bool of_group = s.group >= 0 && s.group < g.groups;
  const int lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kw = wave % KS, set = wave / KS;
  const int n0 = s.tn * BN + set * BW, K = of_group && n0 < g.N ? g.K : 0;
  const int grp = of_group ? s.group : 0;
  // quantised rows: codes, 16 bytes between rows (LDS banks); then scale dwords by row, chunk and quarter
  __shared__ __attribute__((aligned(16))) char qlds[QUANT ? kInPlace / 2 + kInPlace / 32 + 64 * BM : 16];
  [[maybe_unused]] const int nr = min(s.end - s.row, BM);
  const char* pa[MF];
  const char* pb[BKC ? NF : 1];
  [[maybe_unused]] const uint8_t *qa[MF], *qb[NF];
#pragma unroll
  for (int a = 0; a < MF; ++a) {
    if constexpr (QUANT) {
      const int r = min(16 * a + li, nr - 1);
      pa[a] = qlds + r * ((int)g.lda + 16) + 16 * lg;
      qa[a] = reinterpret_cast<const uint8_t*>(qlds) + nr * ((int)g.lda + 16) + r * x.chunks * 16 + 4 * lg;
    } else {
      const int64_t m = min(s.row + 16 * a + li, s.end - 1);
      pa[a] = static_cast<const char*>(g.A) + m * g.lda * ES + 16 * lg;
      if constexpr (MX) qa[a] = x.a + (m >> 4) * x.chunks * kChunk + 64 * lg + 4 * (m & 15);
    }
  }
  if constexpr (BKC) {
#pragma unroll
    for (int b = 0; b < NF; ++b) {
      const int64_t n = min(n0 + 16 * b + li, g.N - 1);
      pb[b] = static_cast<const char*>(g.B) + (grp * g.sB + n * g.ldb) * ES + 16 * lg;
      if constexpr (MX) qb[b] = x.b + grp * x.b_step + (n >> 4) * x.chunks * kChunk + 64 * lg + 4 * (n & 15);
    }
  } else {
    pb[0] = static_cast<const char*>(g.B) + (grp * g.sB + (int64_t)(EV * lg) * g.ldb + min(n0 + 4 * li, ((g.N + 3) & ~3) - 4)) * ES;
  }
  const int64_t kstep = (BKC ? 64 : 64 / ES * g.ldb * ES);  // bytes of B per step
  struct Chunk {
    i32x4 a[MF][STEPS];
    i32x4 b[BKC ? NF : 1][STEPS];
    ColumnStep<std::conditional_t<MX, __bf16, T>> c[BKC ? 1 : STEPS];
    int sa[MF], sb[NF];
  } w[U];
  f32x4 acc[MF][NF], sum[FOLD ? MF : 1][FOLD ? NF : 1];
#pragma unroll
  for (int a = 0; a < MF; ++a)
#pragma unroll
    for (int b = 0; b < NF; ++b) {
      acc[a][b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      if constexpr (FOLD) sum[a][b] = acc[a][b];
    }
  auto load_a = [&](Chunk& v, int c) __attribute__((always_inline)) {
#pragma unroll
    for (int a = 0; a < MF; ++a) {
#pragma unroll
      for (int h = 0; h < STEPS; ++h) v.a[a][h] = load16<T>(pa[a] + (int64_t)c * CH + 64 * h);
      if constexpr (MX) v.sa[a] = *reinterpret_cast<const int*>(qa[a] + (int64_t)c * (QUANT ? 16 : kChunk));
    }
  };
  auto load_b = [&](Chunk& v, int c) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < STEPS; ++h) {
      if constexpr (BKC) {
#pragma unroll
        for (int b = 0; b < NF; ++b) v.b[b][h] = load16<T>(pb[b] + (int64_t)c * CH + 64 * h);
      } else {
        v.c[h].load(pb[0] + (int64_t)(STEPS * c + h) * kstep, g.ldb);
      }
    }
    if constexpr (MX) {
#pragma unroll
      for (int b = 0; b < NF; ++b) v.sb[b] = *reinterpret_cast<const int*>(qb[b] + (int64_t)c * kChunk);
    }
  };
  // the last, partial chunk
  auto load_last = [&](Chunk& v, int c) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < STEPS; ++h) {
      const int left = K - c * CK - (64 / ES) * h - EV * lg;  // values of k from this lane's group on
#pragma unroll
      for (int a = 0; a < MF; ++a) v.a[a][h] = left > 0 ? load16<T>(pa[a] + (int64_t)c * CH + 64 * h) : i32x4{0, 0, 0, 0};
      if constexpr (BKC) {
#pragma unroll
        for (int b = 0; b < NF; ++b) v.b[b][h] = left > 0 ? load16<T>(pb[b] + (int64_t)c * CH + 64 * h) : i32x4{0, 0, 0, 0};
      } else {
        v.c[h].load_last(pb[0] + (int64_t)(STEPS * c + h) * kstep, g.ldb, left);
      }
    }
    if constexpr (MX) {
#pragma unroll
      for (int a = 0; a < MF; ++a) v.sa[a] = *reinterpret_cast<const int*>(qa[a] + (int64_t)c * (QUANT ? 16 : kChunk));
#pragma unroll
      for (int b = 0; b < NF; ++b) v.sb[b] = *reinterpret_cast<const int*>(qb[b] + (int64_t)c * kChunk);
    }
  };
  auto multiply = [&](const Chunk& v) __attribute__((always_inline)) {
    each<STEPS>([&](auto hc) __attribute__((always_inline)) {
      constexpr int h = decltype(hc)::value;
#pragma unroll
      for (int b = 0; b < NF; ++b) {
        i32x4 fb;
        if constexpr (BKC)
          fb = v.b[b][h];
        else
          fb = v.c[h].operand(b);
#pragma unroll
        for (int a = 0; a < MF; ++a) {
          if constexpr (MX) {
            const i32x8 p = {fb[0], fb[1], fb[2], fb[3], 0, 0, 0, 0};
            const i32x8 q = {v.a[a][h][0], v.a[a][h][1], v.a[a][h][2], v.a[a][h][3], 0, 0, 0, 0};
            acc[a][b] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(p, q, acc[a][b], 4, 4, h, v.sb[b], h, v.sa[a]);
          } else {
            mma_tile<T>(acc[a][b], fb, v.a[a][h]);
          }
        }
      }
    });
  };
  const int nc = K / CK;
  int chain = 0;
  auto batch = [&](int c, auto f) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (c + KS * u < nc) f(w[u], c + KS * u);
  };
  if constexpr (QUANT) {
    batch(kw, load_b);
    quantize_rows<X>(g, x, s.row, of_group ? nr : 0, qlds, qlds + nr * ((int)g.lda + 16));
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  }
  for (int c = kw; c < nc; c += KS * U) {
    if (!QUANT || c != kw) batch(c, load_b);
    batch(c, load_a);
    batch(c, [&](const Chunk& v, int) __attribute__((always_inline)) { multiply(v); });
    if constexpr (FOLD) {
      if ((chain += U) >= 512 / CK) {
        chain = 0;
#pragma unroll
        for (int a = 0; a < MF; ++a)
#pragma unroll
          for (int b = 0; b < NF; ++b) {
            sum[a][b] += acc[a][b];
            acc[a][b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
          }
      }
    }
  }
  if (kw == nc % KS && nc * CK < K) {
    load_last(w[0], nc);
    multiply(w[0]);
  }
  // operand j of a column-contiguous B holds columns 4 li + j, so its register r is column 4 (4 lg + r) + j
#pragma unroll
  for (int a = 0; a < MF; ++a)
#pragma unroll
    for (int b = 0; b < NF; ++b) {
      if constexpr (FOLD) acc[a][b] += sum[a][b];
      if constexpr (BKC) {
        part[wave][(16 * a + li) * (BW / 4) + 4 * b + lg] = acc[a][b];
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          reinterpret_cast<float*>(&part[wave][(16 * a + li) * (BW / 4) + 4 * lg + r])[b] = acc[a][b][r];
      }
    }
  __syncthreads();
  constexpr int PER = BM * BW / 4;
  for (int i = threadIdx.x; i < 8 / KS * PER; i += 512) {
    const int q = i / PER, e = i % PER;
    f32x4 v = part[q * KS][e];
#pragma unroll
    for (int p = 1; p < KS; ++p) v += part[q * KS + p][e];
    const int m = s.row + e / (BW / 4), n = s.tn * BN + q * BW + 4 * (e % (BW / 4));
    if (m >= s.end) continue;
    if (g.out32)
      store_quad<float>(g, static_cast<const float*>(g.C), static_cast<float*>(g.D), m, n, v);
    else if (MX && g.out_f16)
      store_quad<_Float16>(g, static_cast<const _Float16*>(g.C), static_cast<_Float16*>(g.D), m, n, v);
    else
      store_quad<std::conditional_t<MX, __bf16, T>>(g, static_cast<const std::conditional_t<MX, __bf16, T>*>(g.C),
                                                    static_cast<std::conditional_t<MX, __bf16, T>*>(g.D), m, n, v);
  }
}

}  // namespace trnblas
