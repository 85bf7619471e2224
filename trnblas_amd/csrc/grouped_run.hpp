// The launches of the grouped products for one element type, and their kernel for
// operands of any alignment; grouped_f32.hip, grouped_bf16.hip and grouped_f16.hip
// compile them side by side.
#pragma once

#include <algorithm>

#include "gemm.hpp"
#include "grouped.hpp"
#include "grouped_plan.hpp"
#include "ring.hpp"
#include "rows.hpp"

namespace trnblas {

// 16 bytes of values at any alignment, only the first n of them inside (n <= 0: none);
// the rest zeros.
template <typename T>
__device__ __forceinline__ i32x4 load_any(const char* p, int n) {
  constexpr int EV = 16 / sizeof(T);
  if (n >= EV) return load16<T>(p);
  union {
    T e[EV];
    i32x4 v;
  } u;
  u.v = i32x4{0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < EV; ++i)
    if (i < n) u.e[i] = reinterpret_cast<const T*>(p)[i];
  return u.v;
}

// 16 bytes of values ending at a row's end, loaded in the place of n values that start
// that much later: moved down, zeros behind them (n <= 0: zeros).
template <typename T>
__device__ __forceinline__ i32x4 end_of_row(i32x4 v, int n) {
  constexpr int EV = 16 / sizeof(T);
  const int s = (EV - n) * (int)sizeof(T);  // bytes
  if (s & 8) v = i32x4{v[2], v[3], 0, 0};
  if (s & 4) v = i32x4{v[1], v[2], v[3], 0};
  if constexpr (sizeof(T) == 2) {
    if (s & 2) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = (int)__builtin_amdgcn_alignbit(i < 3 ? v[i + 1] : 0, v[i], 16);
    }
  }
  return n > 0 ? v : i32x4{0, 0, 0, 0};
}

// One operand's loads of a k-tile, 16 bytes per lane and 256 groups, in Panel's order:
// with no branch, so that those of two k-tiles stay under way. Of a group that passes
// its row's end the row's last 16 bytes are loaded and moved down behind a uniform
// branch (put); what lies outside is loaded from some place inside and stored as zeros
// (rows of a K-contiguous operand past the tile's end: as they are, their sums are not
// stored). TINY: rows shorter than 16 bytes, one value at a time.
template <typename T, int ROWS, bool KC, bool TINY>
struct Loads {
  using P = Panel<T, ROWS, KC>;
  static constexpr int ES = sizeof(T), EV = 16 / ES, BK = P::BK, H = P::BYTES / 4096;
  const char* p[H];   // KC: the row's start; else the group's of the first k-tile
  const char* first;  // the first row's first values
  int64_t step;       // bytes per k-tile
  int K, at, inside;  // KC: the group's k; else its first k (16-byte groups h: k_of), values inside
  int slot;
  bool edge;          // the tile passes the rows' end

  // base: the panel's corner, `before` values after its row's start
  __device__ __forceinline__ Loads(const char* base, int64_t before, int64_t ld, int rows, int k, int tid) : K(k) {
    first = base - before * ES;
    slot = 16 * tid;
    edge = !KC && rows < ROWS;
    step = (KC ? BK : BK * ld) * ES;
#pragma unroll
    for (int h = 0; h < H; ++h) {
      int r, q;
      P::where(tid + 256 * h, r, q);  // the same q (KC) or r for all h
      if constexpr (KC) {
        at = q;
        inside = r < rows;
        p[h] = base + (TINY ? r : min(r, rows - 1)) * ld * ES;
        if constexpr (TINY) inside = rows;
      } else {
        if (h == 0) at = q;
        inside = rows - r;
        p[h] = (TINY || inside >= EV ? base + r * ES : inside > 0 ? base + (rows - EV) * ES : first) + q * ld * ES;
      }
    }
  }
  static __device__ __forceinline__ int k_of(int h) { return h * (256 / P::GPR); }
  __device__ __forceinline__ void load(int kt, i32x4 (&v)[H]) const {
    const int left = K - kt * BK;
#pragma unroll
    for (int h = 0; h < H; ++h) {
      if constexpr (TINY && KC)
        v[h] = load_any<T>(p[h] + kt * step + at * ES, (slot >> 7) + 32 * h < inside ? left - at : 0);
      else if constexpr (TINY)
        v[h] = load_any<T>(p[h] + kt * step, at + k_of(h) < left ? inside : 0);
      else if constexpr (KC)
        v[h] = load16<T>(p[h] + (int64_t)min(kt * BK + at, K - EV) * ES);
      else
        v[h] = load16<T>(at + k_of(h) < left ? p[h] + kt * step : first);
    }
  }
  __device__ __forceinline__ void put(char* st, int kt, i32x4 (&v)[H]) const {
    const int left = K - kt * BK;
    if (!TINY && (left < BK || edge)) {
#pragma unroll
      for (int h = 0; h < H; ++h) {
        const int n = KC ? left - at : at + k_of(h) < left ? inside : 0;
        v[h] = n < EV ? end_of_row<T>(v[h], n) : v[h];
      }
    }
#pragma unroll
    for (int h = 0; h < H; ++h) *reinterpret_cast<i32x4*>(st + slot + 4096 * h) = v[h];
  }
};

// Operands of any alignment and any strides: the panels go through registers.
// 256 threads on a 64 x 64 tile, each wave 32 x 32; the loads of k-tile t + 2 are in
// flight behind the MFMAs of t. fp32 and CHAINS (see kChain16): the sums restart every
// chain_length(K) values of k (gemm.hpp). fp32 gemm takes 32 x 64: its MFMAs are eight
// times as long, so that the last round's idle CUs cost more than the smaller tile's loads (1501 rows in 6 groups
// by 515 x 771: 360 tiles 31 us, 720 tiles 27; 4093 by 2047^2 385 and 393). 16-bit:
// bound by the loads of rows that start anywhere (16 bytes two bytes past a word take
// several times as long; the five words around them, shifted, longer still): bf16 4093
// rows in 8 groups by 1023 x 2047 61 us (281 TFLOP/s), 16383 by 2047 x 4095 678 (405);
// 512 rows in 16 groups by 1023 x 2047 21 us, 64 when each load was a branch whose
// merge waited for all loads. Larger products are packed first.
template <typename T, bool RK>
constexpr int any_fm = std::is_same_v<T, float> && !RK ? 1 : 2;
template <typename T, bool BKC, bool RK, bool TINY, bool CHAINS = false>
__global__ __launch_bounds__(256, 3) void grouped_any_kernel(GroupedArgs g) {
  constexpr int FM = any_fm<T, RK>, FN = 2, BM = 32 * FM, BN = 32 * FN, AHEAD = 2;
  using PA = Panel<T, BM, !RK>;
  using PB = Panel<T, BN, BKC>;
  constexpr int BK = PA::BK, ES = sizeof(T), HA = PA::BYTES / 4096, HB = PB::BYTES / 4096;
  constexpr bool F32 = std::is_same_v<T, float>, FOLD = F32 || CHAINS;
  __shared__ __attribute__((aligned(16))) char lds[2][PA::BYTES + PB::BYTES];
  TileJob j;
  if (!tile_job<T, BM, BN, BKC, RK>(g, j)) return;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m0 = 16 * FM * (wave & 1), n0 = 16 * FN * (wave >> 1);
  const int nk = (j.K + BK - 1) / BK;
  Loads<T, BM, !RK, TINY> la(j.A, RK ? j.m : 0, g.lda, j.rows_a, j.K, tid);
  Loads<T, BN, BKC, TINY> lb(j.B, BKC ? 0 : j.n, g.ldb, j.rows_b, j.K, tid);
  i32x4 va[AHEAD][HA], vb[AHEAD][HB];
  uint32_t oa[PA::NV], ob[PB::NV];
  PA::lane_offsets(m0, lane, oa);
  PB::lane_offsets(n0, lane, ob);
  f32x4 acc[FM][FN], sum[FOLD ? FM : 1][FOLD ? FN : 1];
#pragma unroll
  for (int a = 0; a < FM; ++a)
#pragma unroll
    for (int b = 0; b < FN; ++b) {
      acc[a][b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      if constexpr (FOLD) sum[a][b] = acc[a][b];
    }
  const int span = chain_length(j.K, ES) / BK;
  int chain = span;
  auto k_tile = [&](int kt, int set) __attribute__((always_inline)) {
    char* st = lds[kt & 1];
    la.put(st, kt, va[set]);
    lb.put(st + PA::BYTES, kt, vb[set]);
    // one barrier per k-tile: stage t's readers are past it before t + 2 is stored
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    la.load(min(kt + AHEAD, nk - 1), va[set]);  // past the end again the last, unused
    lb.load(min(kt + AHEAD, nk - 1), vb[set]);
    const char *qa[PA::NV], *qb[PB::NV];
#pragma unroll
    for (int i = 0; i < PA::NV; ++i) qa[i] = st + oa[i];
#pragma unroll
    for (int i = 0; i < PB::NV; ++i) qb[i] = st + PA::BYTES + ob[i];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      i32x4 fa[FM], fb[FN];
#pragma unroll
      for (int a = 0; a < FM; ++a) fa[a] = PA::frag(qa, a, h);
#pragma unroll
      for (int b = 0; b < FN; ++b) fb[b] = PB::frag(qb, b, h);
      if constexpr (F32) {  // four products per sum: the sums in turn
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int b = 0; b < FN; ++b)
#pragma unroll
            for (int a = 0; a < FM; ++a)
              acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(f32x4, fb[b])[e], __builtin_bit_cast(f32x4, fa[a])[e],
                                                               acc[a][b], 0, 0, 0);
      } else {
#pragma unroll
        for (int b = 0; b < FN; ++b)
#pragma unroll
          for (int a = 0; a < FM; ++a) mma_tile<T>(acc[a][b], fb[b], fa[a]);
      }
    }
    if constexpr (FOLD) {
      if (--chain == 0) {
#pragma unroll
        for (int a = 0; a < FM; ++a)
#pragma unroll
          for (int b = 0; b < FN; ++b) {
            sum[a][b] += acc[a][b];
            acc[a][b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
          }
        chain = span;
      }
    }
  };
  if (nk > 0) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      la.load(min(i, nk - 1), va[i]);
      lb.load(min(i, nk - 1), vb[i]);
    }
    int kt = 0;
    for (; kt + 1 < nk; kt += 2) {
      k_tile(kt, 0);
      k_tile(kt + 1, 1);
    }
    if (kt < nk) k_tile(kt, 0);
  }
  if constexpr (FOLD) {
#pragma unroll
    for (int a = 0; a < FM; ++a)
#pragma unroll
      for (int b = 0; b < FN; ++b) acc[a][b] += sum[a][b];
  }
  static_assert(4 * kStoreLds<FN> <= sizeof(lds));
  char* own = lds[0] + wave * kStoreLds<FN>;
  __syncthreads();  // the other waves' reads
  if (g.out32)
    store_wave<FM, FN, float>(g, j, acc, m0, n0, lane, own);
  else
    store_wave<FM, FN, T>(g, j, acc, m0, n0, lane, own);
}

static const char* const kGemm = "trnblas_hip_grouped_gemm";
static const char* const kRankK = "trnblas_hip_grouped_rank_k";

// Bound on the row tiles of `rows` rows in `groups` groups and the two gaps.
static int64_t row_tiles(int64_t rows, int64_t groups, int bm) { return rows / bm + std::min(groups + 2, rows); }

static int grid_of(int64_t tiles, const char* what, unsigned* grid) {
  TRNBLAS_CHECK_ARG(tiles < ((int64_t)1 << 31) - 4096, "%s: too many tiles", what);
  *grid = (unsigned)tiles;
  return TRNBLAS_OK;
}

template <typename T, bool BKC, bool RK>
static int run_any(GroupedArgs g, hipStream_t s) {
  constexpr int BM = 32 * any_fm<T, RK>;
  const char* what = RK ? kRankK : kGemm;
  g.tiles_m = (g.M + BM - 1) / BM;
  g.tiles_n = (g.N + 63) / 64;
  unsigned grid;
  const int64_t rows = RK ? (int64_t)g.groups * g.tiles_m : row_tiles(g.rows, g.groups, BM);
  if (int rc = grid_of(rows * g.tiles_n, what, &grid)) return rc;
  // whole rounds of the XCDs, so that each one's last tile is reached
  grid = (grid + kNumXcd - 1) / kNumXcd * kNumXcd;
  constexpr int EV = 16 / sizeof(T);
  const bool tiny = (RK ? g.M : g.K) < EV || (BKC ? g.K : g.N) < EV;
  auto kernel = tiny ? grouped_any_kernel<T, BKC, RK, true> : grouped_any_kernel<T, BKC, RK, false>;
  if constexpr (sizeof(T) == 2) {
    if (needs_chains<T>(g, RK ? g.rows : g.K)) {
      kernel = grouped_any_kernel<T, BKC, RK, false, true>;
      if constexpr (!BKC) {  // a K-contiguous B has long rows then
        if (tiny) kernel = grouped_any_kernel<T, BKC, RK, true, true>;
      }
    }
  }
  hipLaunchKernelGGL(kernel, dim3(grid), dim3(256), 0, s, g);
  return check_launch(what);
}

// Operands that LDS DMA reads in place: see ring.hpp. Whole groups of 16 bytes
// lie inside the operands, or (g.padded) are zeros past their ends. Its 32-bit
// offsets reach over one panel of a K-contiguous operand and one k-tile of the
// other kind.
template <typename T>
static bool dma_ready(const GroupedArgs& g, bool bkc, bool rk) {
  const int64_t es = sizeof(T), far = INT32_MAX - 1024;
  auto whole = [&](const void* p, int64_t ld, int64_t st, int64_t ext) {
    return (uintptr_t)p % 16 == 0 && ld * es % 16 == 0 && st * es % 16 == 0 && (g.padded || ext * es % 16 == 0);
  };
  const int64_t ra = rk ? 128 / es : 256, rb = bkc ? 256 : 128 / es;
  return whole(g.A, g.lda, 0, rk ? g.M : g.K) && whole(g.B, g.ldb, g.sB, bkc ? g.K : g.N) && (!rk || g.rows < far) &&
         ra * g.lda * es < far && rb * g.ldb * es < far;
}

template <typename T, int FM, int FN, bool BKC, bool RK>
static int run_ring(GroupedArgs g, hipStream_t s) {
  constexpr int BM = 32 * FM, BN = 32 * FN;
  const char* what = RK ? kRankK : kGemm;
  g.tiles_m = (g.M + BM - 1) / BM;
  g.tiles_n = (g.N + BN - 1) / BN;
  unsigned grid;
  const int64_t rows = RK ? (int64_t)g.groups * g.tiles_m : row_tiles(g.rows, g.groups, BM);
  if (int rc = grid_of(ring_grid<FM, FN>(g, rows * g.tiles_n), what, &grid)) return rc;
  auto kernel = ring_kernel<T, FM, FN, BKC, RK>;
  if constexpr (sizeof(T) == 2) {
    if (needs_chains<T>(g, RK ? g.rows : g.K)) kernel = ring_kernel<T, FM, FN, BKC, RK, true>;
  }
  hipLaunchKernelGGL(kernel, dim3(grid), dim3(256), 0, s, g, MxScales{});
  return check_launch(what);
}

template <typename T, int MF, int NF, int KS, bool BKC>
static int run_rows(GroupedArgs g, hipStream_t s) {
  constexpr int BN = 128 * NF / KS;
  g.tiles_n = (g.N + BN - 1) / BN;
  unsigned grid;
  if (int rc = grid_of(row_tiles(g.rows, g.groups, 16 * MF) * g.tiles_n, kGemm, &grid)) return rc;
  grid = (grid + kNumXcd - 1) / kNumXcd * kNumXcd;
  auto kernel = rows_kernel<T, MF, NF, KS, BKC>;
  if constexpr (sizeof(T) == 2) {
    if (needs_chains<T>(g, g.K / KS)) kernel = rows_kernel<T, MF, NF, KS, BKC, void, true>;  // a wave's share
  }
  hipLaunchKernelGGL(kernel, dim3(grid), dim3(512), 0, s, g, MxScales{});
  return check_launch(kGemm);
}

// Fewer than eight waves along K: one block of rows, K-contiguous (the plan asks for no other; fp32: not two).
template <typename T, int MF, bool BKC>
static int run_rows_split(int ks, const GroupedArgs& g, hipStream_t s) {
  constexpr int NF = BKC ? 1 : 4;
  if constexpr (MF == 1 && BKC) {
    if (ks == 4) return run_rows<T, MF, NF, 4, BKC>(g, s);
    if constexpr (sizeof(T) == 2) {
      if (ks == 2) return run_rows<T, MF, NF, 2, BKC>(g, s);
    }
    if (ks == 1) return run_rows<T, MF, NF, 1, BKC>(g, s);
  }
  return run_rows<T, MF, NF, 8, BKC>(g, s);
}

// ring: index of kRing16. fp32 takes the 64 x 128 tiles: three workgroups per CU hide
// its longer MFMAs' steps best (8 groups of 128 rows, 2048 x 4096: 217 us, 220 on 128 x
// 128).
template <typename T, bool BKC, bool RK>
static int run_ring_choice(int ring, const GroupedArgs& g, hipStream_t s) {
  if constexpr (sizeof(T) == 2) {
    if (ring == 0) return run_ring<T, 8, 8, BKC, RK>(g, s);
    if (ring == 1) return run_ring<T, 4, 4, BKC, RK>(g, s);
  }
  return run_ring<T, 2, 4, BKC, RK>(g, s);
}

template <typename T, bool BKC>
static int run_grouped(const GroupedArgs& g, hipStream_t s) {
  if (!dma_ready<T>(g, BKC, false)) return run_any<T, BKC, false>(g, s);
  const GroupedChoice c = choose_gemm(sizeof(T), g.rows, g.groups, g.N, g.K, BKC);
  if constexpr (sizeof(T) == 2) {
    if (c.ring < 0 && c.mf == 2) return run_rows_split<T, 2, BKC>(c.ks, g, s);
  } else {
    if (c.ring == kAnyTiles) return run_any<T, BKC, false>(g, s);
  }
  if (c.ring < 0) return run_rows_split<T, 1, BKC>(c.ks, g, s);
  return run_ring_choice<T, BKC, false>(c.ring, g, s);
}

template <typename T>
int grouped_gemm_run(const GroupedArgs& g, bool bkc, hipStream_t s) {
  return bkc ? run_grouped<T, true>(g, s) : run_grouped<T, false>(g, s);
}

template <typename T>
int grouped_rank_k_run(const GroupedArgs& g, hipStream_t s) {
  if (!dma_ready<T>(g, false, true)) return run_any<T, false, true>(g, s);
  return run_ring_choice<T, false, true>(choose_rank_k(sizeof(T), g.groups, g.rows, g.M, g.N), g, s);
}

}  // namespace trnblas
