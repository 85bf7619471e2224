// Products over ragged groups of rows (rows sorted by expert), fp32 / bf16 /
// fp16 on MFMA with fp32 sums:
//  * grouped_gemm:   D[r] = alpha A[r] op(B[g]) + beta C[r] for the rows r of
//    group g (D[r] = beta C[r] for rows of no group);
//  * grouped_rank_k: D[g] = alpha A_g^T B_g + beta C[g], A_g and B_g the rows of
//    group g (the gradient of the former to B).
// The group boundaries are read on the device: nothing waits for the host.
#include <algorithm>

#include "gemm.hpp"
#include "grouped.hpp"

namespace trnblas {

// The tile of a workgroup: where its operand panels start, how many rows of
// each are inside, the k range, and where the output goes.
struct TileJob {
  const char *A, *B;  // panel corners at k = 0
  int rows_a, rows_b, K;
  int64_t m;  // first output row
  int n;      // first output column
  const void* C;
  void* D;
};

// RK: ragged k (grouped_rank_k), else ragged rows.
template <typename T, int BM, int BN, bool BKC, bool RK>
__device__ __forceinline__ bool tile_job(const GroupedArgs& g, TileJob& j) {
  const int64_t es = sizeof(T), eo = g.out32 ? 4 : es;
  if constexpr (RK) {
    const int t = xcd_remap(blockIdx.x, gridDim.x);
    const int per = g.tiles_m * g.tiles_n, grp = t / per;
    int tm, tn;
    grouped_tile(t - grp * per, g.tiles_m, g.tiles_n, 8, tm, tn);
    const int start = boundary(g, grp + 1), end = max(boundary(g, grp + 2), start);
    j.m = tm * BM;
    j.n = tn * BN;
    j.K = end - start;
    j.A = static_cast<const char*>(g.A) + (start * g.lda + j.m) * es;
    j.B = static_cast<const char*>(g.B) + (start * g.ldb + j.n) * es;
    j.rows_a = min(BM, g.M - (int)j.m);
    j.C = static_cast<const char*>(g.C) + (g.C ? grp * g.sC * eo : 0);
    j.D = static_cast<char*>(g.D) + grp * g.sD * eo;
  } else {
    Segment s;
    if (!ragged_tile<BM>(g, blockIdx.x, 8, s)) return false;
    const bool of_group = s.group >= 0 && s.group < g.groups;
    j.m = s.row;
    j.n = s.tn * BN;
    j.K = of_group ? g.K : 0;
    j.A = static_cast<const char*>(g.A) + s.row * g.lda * es;
    j.B = static_cast<const char*>(g.B) + (of_group ? s.group * g.sB + (BKC ? j.n * g.ldb : j.n) : 0) * es;
    j.rows_a = min(BM, s.end - s.row);
    j.C = g.C;
    j.D = g.D;
  }
  j.rows_b = min(BN, g.N - j.n);
  return true;
}

// The 16-byte group of an operand at (row, k): `n` of its EV values are inside.
typedef i32x4 __attribute__((aligned(2))) i32x4_at2;
typedef i32x4 __attribute__((aligned(4))) i32x4_at4;

template <typename T>
__device__ __forceinline__ i32x4 load_any(const char* p, int n) {
  constexpr int EV = 16 / sizeof(T);
  using loose = std::conditional_t<sizeof(T) == 2, i32x4_at2, i32x4_at4>;
  if (n >= EV) return *reinterpret_cast<const loose*>(p);
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

template <int FM, int FN, typename O>
__device__ __forceinline__ void store_wave(const GroupedArgs& g, const TileJob& j, const f32x4 (&acc)[FM][FN], int m0,
                                           int n0, int lane) {
#pragma unroll
  for (int a = 0; a < FM; ++a) {
    const int m = m0 + 16 * a + (lane & 15);
    if (m < j.rows_a) {
#pragma unroll
      for (int b = 0; b < FN; ++b)
        store_quad<O>(g, static_cast<const O*>(j.C), static_cast<O*>(j.D), j.m + m, j.n + n0 + 16 * b + 4 * (lane >> 4), acc[a][b]);
    }
  }
}

// Operands of any alignment and any strides: the panels go through registers.
// 256 threads on a 64 x 64 tile, each wave 32 x 32; the loads of k-tile t + 1 are
// in flight behind the MFMAs of t. fp32 sums restart every chain_length(K)
// values of k (gemm.hpp).
template <typename T, bool BKC, bool RK>
__global__ __launch_bounds__(256) void grouped_any_kernel(GroupedArgs g) {
  constexpr int BM = 64, BN = 64, FM = 2, FN = 2;
  using PA = Panel<T, BM, !RK>;
  using PB = Panel<T, BN, BKC>;
  constexpr int BK = PA::BK, EV = PA::EV, ES = sizeof(T);
  constexpr bool FOLD = std::is_same_v<T, float>;
  __shared__ __attribute__((aligned(16))) char lds[2][PA::BYTES + PB::BYTES];
  TileJob j;
  if (!tile_job<T, BM, BN, BKC, RK>(g, j)) return;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m0 = 32 * (wave & 1), n0 = 32 * (wave >> 1);
  int ra, ka, rb, kb;
  PA::where(tid, ra, ka);
  PB::where(tid, rb, kb);
  const char* pa = j.A + (RK ? (int64_t)ka * g.lda + ra : (int64_t)ra * g.lda + ka) * ES;
  const char* pb = j.B + (BKC ? (int64_t)rb * g.ldb + kb : (int64_t)kb * g.ldb + rb) * ES;
  const int64_t step_a = (RK ? BK * g.lda : BK) * ES, step_b = (BKC ? BK : BK * g.ldb) * ES;
  const int nk = (j.K + BK - 1) / BK;
  i32x4 va, vb;
  auto load = [&](int kt) __attribute__((always_inline)) {
    const int left = j.K - kt * BK;
    va = load_any<T>(pa + kt * step_a, RK ? (ka < left ? j.rows_a - ra : 0) : (ra < j.rows_a ? left - ka : 0));
    vb = load_any<T>(pb + kt * step_b, BKC ? (rb < j.rows_b ? left - kb : 0) : (kb < left ? j.rows_b - rb : 0));
  };
  f32x4 acc[FM][FN], sum[FM][FN];
#pragma unroll
  for (int a = 0; a < FM; ++a)
#pragma unroll
    for (int b = 0; b < FN; ++b) acc[a][b] = sum[a][b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  const int span = chain_length(j.K, ES) / BK;
  int chain = span;
  if (nk > 0) load(0);
  for (int kt = 0; kt < nk; ++kt) {
    char* st = lds[kt & 1];
    *reinterpret_cast<i32x4*>(st + 16 * tid) = va;
    *reinterpret_cast<i32x4*>(st + PA::BYTES + 16 * tid) = vb;
    // one barrier per k-tile: stage t's readers are past it before t + 2 is stored
    __syncthreads();
    if (kt + 1 < nk) load(kt + 1);
    i32x4 fa[FM], fb[FN];
#pragma unroll
    for (int a = 0; a < FM; ++a) fa[a] = PA::frag(st, m0 + 16 * a, lane);
#pragma unroll
    for (int b = 0; b < FN; ++b) fb[b] = PB::frag(st + PA::BYTES, n0 + 16 * b, lane);
#pragma unroll
    for (int b = 0; b < FN; ++b)
#pragma unroll
      for (int a = 0; a < FM; ++a) mma_tile<T>(acc[a][b], fb[b], fa[a]);
    if (FOLD && --chain == 0) {
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
  if (FOLD) {
#pragma unroll
    for (int a = 0; a < FM; ++a)
#pragma unroll
      for (int b = 0; b < FN; ++b) acc[a][b] += sum[a][b];
  }
  if (g.out32)
    store_wave<FM, FN, float>(g, j, acc, m0, n0, lane);
  else
    store_wave<FM, FN, T>(g, j, acc, m0, n0, lane);
}

static const char* kGemm = "trnblas_hip_grouped_gemm";
static const char* kRankK = "trnblas_hip_grouped_rank_k";

// Bound on the row tiles of `rows` rows in `groups` groups and the two gaps.
static int64_t row_tiles(int64_t rows, int64_t groups, int bm) { return rows / bm + std::min(groups + 2, rows); }

static int grid_of(int64_t tiles, const char* what, unsigned* grid) {
  TRNBLAS_CHECK_ARG(tiles < (int64_t)1 << 31, "%s: too many tiles", what);
  *grid = (unsigned)tiles;
  return TRNBLAS_OK;
}

template <typename T, bool BKC, bool RK>
static int run_any(GroupedArgs g, hipStream_t s) {
  const char* what = RK ? kRankK : kGemm;
  g.tiles_m = (g.M + 63) / 64;
  g.tiles_n = (g.N + 63) / 64;
  unsigned grid;
  const int64_t rows = RK ? (int64_t)g.groups * g.tiles_m : row_tiles(g.rows, g.groups, 64);
  if (int rc = grid_of(rows * g.tiles_n, what, &grid)) return rc;
  // whole rounds of the XCDs: a grid that is a bound on the tiles reaches the last one of each
  if (!RK) grid = (grid + kNumXcd - 1) / kNumXcd * kNumXcd;
  hipLaunchKernelGGL((grouped_any_kernel<T, BKC, RK>), dim3(grid), dim3(256), 0, s, g);
  return check_launch(what);
}

template <typename T>
static int run_gemm(const GroupedArgs& g, bool bkc, hipStream_t s) {
  return bkc ? run_any<T, true, false>(g, s) : run_any<T, false, false>(g, s);
}

template <typename T>
static int run_rank_k(const GroupedArgs& g, hipStream_t s) {
  return run_any<T, false, true>(g, s);
}

static bool quads(const GroupedArgs& g, int dtype) {
  const int64_t eo = g.out32 || dtype == TRNBLAS_F32 ? 4 : 2;
  auto ok = [&](const void* p, int64_t ld, int64_t st) {
    return (uintptr_t)p % (4 * eo) == 0 && ld % 4 == 0 && st % 4 == 0;
  };
  return ok(g.D, g.ldd, g.sD) && (g.C == nullptr || ok(g.C, g.ldc, g.sC));
}

// checks and fields that both entry points share
static int common_args(const char* what, GroupedArgs& g, int dtype, int out_f32, int64_t groups, int64_t rows, double alpha,
                       double beta, const void* offsets, int offsets64, const void* C) {
  TRNBLAS_CHECK_ARG(dtype == TRNBLAS_F32 || dtype == TRNBLAS_BF16 || dtype == TRNBLAS_F16, "%s: bad dtype %d", what, dtype);
  TRNBLAS_CHECK_ARG(groups >= 0 && groups < (1 << 24) && rows >= 0 && rows < INT32_MAX - 1024,
                    "%s: bad sizes (groups %lld, rows %lld)", what, (long long)groups, (long long)rows);
  TRNBLAS_CHECK_ARG(offsets != nullptr && (uintptr_t)offsets % (offsets64 ? 8 : 4) == 0, "%s: offsets missing or misaligned", what);
  TRNBLAS_CHECK_ARG(beta == 0.0 || C != nullptr, "%s: beta != 0 without C", what);
  g.offsets = offsets;
  g.offsets64 = offsets64 != 0;
  g.groups = (int)groups;
  g.rows = (int)rows;
  g.alpha = (float)alpha;
  g.beta = (float)beta;
  g.out32 = out_f32 != 0 || dtype == TRNBLAS_F32;
  return TRNBLAS_OK;
}

}  // namespace trnblas

using namespace trnblas;

extern "C" int trnblas_hip_grouped_gemm(int dtype, int out_f32, int transB, int64_t groups, int64_t rows, int64_t N, int64_t K,
                                        double alpha, const void* A, int64_t lda, const void* B, int64_t ldb, int64_t strideB,
                                        const void* offsets, int offsets64, double beta, const void* C, int64_t ldc, void* D,
                                        int64_t ldd, void* stream) {
  GroupedArgs g{};
  if (int rc = common_args(kGemm, g, dtype, out_f32, groups, rows, alpha, beta, offsets, offsets64, C)) return rc;
  TRNBLAS_CHECK_ARG(N >= 0 && N < INT32_MAX - 1024 && K >= 0 && K < INT32_MAX - 1024, "%s: bad sizes (N %lld, K %lld)", kGemm,
                    (long long)N, (long long)K);
  TRNBLAS_CHECK_ARG(lda >= K && ldb >= (transB ? K : N) && ldd >= N && (beta == 0.0 || ldc >= N) && strideB >= 0,
                    "%s: bad leading dimension", kGemm);
  if (rows == 0 || N == 0) return TRNBLAS_OK;
  TRNBLAS_CHECK_ARG(D != nullptr && ((A != nullptr && B != nullptr) || K == 0 || groups == 0), "%s: null operand", kGemm);
  g.A = A, g.lda = lda;
  g.B = B, g.ldb = ldb, g.sB = strideB;
  g.C = beta != 0.0 ? C : nullptr, g.ldc = ldc;
  g.D = D, g.ldd = ldd;
  g.N = (int)N, g.K = (int)K;
  g.vec4 = quads(g, dtype);
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case TRNBLAS_F32: return run_gemm<float>(g, transB != 0, s);
    case TRNBLAS_BF16: return run_gemm<__bf16>(g, transB != 0, s);
    default: return run_gemm<_Float16>(g, transB != 0, s);
  }
}

extern "C" int trnblas_hip_grouped_rank_k(int dtype, int out_f32, int64_t groups, int64_t rows, int64_t M, int64_t N, double alpha,
                                          const void* A, int64_t lda, const void* B, int64_t ldb, const void* offsets,
                                          int offsets64, double beta, const void* C, int64_t ldc, int64_t strideC, void* D,
                                          int64_t ldd, int64_t strideD, void* stream) {
  GroupedArgs g{};
  if (int rc = common_args(kRankK, g, dtype, out_f32, groups, rows, alpha, beta, offsets, offsets64, C)) return rc;
  TRNBLAS_CHECK_ARG(M >= 0 && M < INT32_MAX - 1024 && N >= 0 && N < INT32_MAX - 1024, "%s: bad sizes (M %lld, N %lld)", kRankK,
                    (long long)M, (long long)N);
  TRNBLAS_CHECK_ARG(lda >= M && ldb >= N && ldd >= N && (beta == 0.0 || ldc >= N) && strideC >= 0 && strideD >= 0,
                    "%s: bad leading dimension", kRankK);
  if (groups == 0 || M == 0 || N == 0) return TRNBLAS_OK;
  TRNBLAS_CHECK_ARG(D != nullptr && ((A != nullptr && B != nullptr) || rows == 0), "%s: null operand", kRankK);
  g.A = A, g.lda = lda;
  g.B = B, g.ldb = ldb;
  g.C = beta != 0.0 ? C : nullptr, g.ldc = ldc, g.sC = strideC;
  g.D = D, g.ldd = ldd, g.sD = strideD;
  g.M = (int)M, g.N = (int)N;
  g.vec4 = quads(g, dtype);
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case TRNBLAS_F32: return run_rank_k<float>(g, s);
    case TRNBLAS_BF16: return run_rank_k<__bf16>(g, s);
    default: return run_rank_k<_Float16>(g, s);
  }
}
