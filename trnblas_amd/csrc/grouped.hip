// Products over ragged groups of rows (rows sorted by expert), fp32 / bf16 /
// fp16 on MFMA with fp32 sums:
//  * grouped_gemm:   D[r] = alpha A[r] op(B[g]) + beta C[r] for the rows r of
//    group g (D[r] = beta C[r] for rows of no group);
//  * grouped_rank_k: D[g] = alpha A_g^T B_g + beta C[g], A_g and B_g the rows of
//    group g (the gradient of the former to B).
// The group boundaries are read on the device: nothing waits for the host.
#include <algorithm>
#include <cstring>

#include "grouped.hpp"
#include "grouped_plan.hpp"

namespace trnblas {

static const char* kGemm = "trnblas_hip_grouped_gemm";
static const char* kRankK = "trnblas_hip_grouped_rank_k";

static bool quads(const GroupedArgs& g, int dtype) {
  const int64_t eo = g.out32 || dtype == TRNBLAS_F32 ? 4 : 2;
  auto ok = [&](const void* p, int64_t ld, int64_t st) {
    return (uintptr_t)p % (4 * eo) == 0 && ld % 4 == 0 && st % 4 == 0;
  };
  return ok(g.D, g.ldd, g.sD) && (g.C == nullptr || ok(g.C, g.ldc, g.sC));
}

// checks and fields that both entry points share
static int common_args(const char* what, GroupedArgs& g, int dtype, int out_f32, int64_t groups, int64_t rows, double alpha,
                       double beta, const void* offsets, int offsets64, const void* C, int padded) {
  TRNBLAS_CHECK_ARG(dtype == TRNBLAS_F32 || dtype == TRNBLAS_BF16 || dtype == TRNBLAS_F16, "%s: bad dtype %d", what, dtype);
  TRNBLAS_CHECK_ARG(groups >= 0 && groups < (1 << 24) && rows >= 0 && rows < INT32_MAX - 1024,
                    "%s: bad sizes (groups %lld, rows %lld)", what, (long long)groups, (long long)rows);
  TRNBLAS_CHECK_ARG(offsets != nullptr ? (uintptr_t)offsets % (offsets64 ? 8 : 4) == 0 : groups == 1,
                    "%s: offsets missing or misaligned", what);
  TRNBLAS_CHECK_ARG(beta == 0.0 || C != nullptr, "%s: beta != 0 without C", what);
  g.padded = padded != 0;
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
                                        int64_t ldd, int padded, void* stream) {
  GroupedArgs g{};
  if (int rc = common_args(kGemm, g, dtype, out_f32, groups, rows, alpha, beta, offsets, offsets64, C, padded)) return rc;
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
    case TRNBLAS_F32: return grouped_gemm_run<float>(g, transB != 0, s);
    case TRNBLAS_BF16: return grouped_gemm_run<__bf16>(g, transB != 0, s);
    default: return grouped_gemm_run<_Float16>(g, transB != 0, s);
  }
}

extern "C" int trnblas_hip_grouped_rank_k(int dtype, int out_f32, int64_t groups, int64_t rows, int64_t M, int64_t N, double alpha,
                                          const void* A, int64_t lda, const void* B, int64_t ldb, const void* offsets,
                                          int offsets64, double beta, const void* C, int64_t ldc, int64_t strideC, void* D,
                                          int64_t ldd, int64_t strideD, int padded, void* stream) {
  GroupedArgs g{};
  if (int rc = common_args(kRankK, g, dtype, out_f32, groups, rows, alpha, beta, offsets, offsets64, C, padded)) return rc;
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
    case TRNBLAS_F32: return grouped_rank_k_run<float>(g, s);
    case TRNBLAS_BF16: return grouped_rank_k_run<__bf16>(g, s);
    default: return grouped_rank_k_run<_Float16>(g, s);
  }
}

static GroupedChoice gemm_choice(int op, int64_t es, int transB, int64_t groups, int64_t rows, int64_t N, int64_t K) {
  return op == 2 ? choose_mx(rows, groups, N, K) : choose_gemm((int)es, rows, groups, N, K, transB != 0);
}

extern "C" int trnblas_hip_grouped_rows_plan(int op, int dtype, int transB, int64_t groups, int64_t rows, int64_t N, int64_t K,
                                             int32_t plan[3]) {
  TRNBLAS_CHECK_ARG(plan != nullptr && op != 1, "trnblas_hip_grouped_rows_plan: bad arguments");
  const char* name = trnblas_hip_grouped_plan(op, dtype, transB, groups, rows, 0, N, K);
  TRNBLAS_CHECK_ARG(name != nullptr, "trnblas_hip_grouped_rows_plan: bad arguments");
  plan[0] = plan[1] = plan[2] = 0;
  if (strcmp(name, "rows_kernel") != 0) return TRNBLAS_OK;
  const GroupedChoice c = gemm_choice(op, dtype == TRNBLAS_F32 ? 4 : 2, transB, groups, rows, N, K);
  plan[0] = c.mf, plan[1] = c.ks;
  plan[2] = op == 2 && quantised_in_place(c, rows, K);
  return TRNBLAS_OK;
}

extern "C" const char* trnblas_hip_grouped_plan(int op, int dtype, int transB, int64_t groups, int64_t rows, int64_t M, int64_t N,
                                                int64_t K) {
  static const char* const kRingNames[] = {"ring_kernel 256 x 256", "ring_kernel 128 x 128", "ring_kernel 64 x 128"};
  const int64_t es = dtype == TRNBLAS_F32 ? 4 : 2, first = op == 1 ? M : K, second = op == 1 || !transB ? N : K;
  if (op < 0 || op > 2 || dtype < 0 || dtype > 2 || groups < 1 || rows < 1 || M < 0 || N < 1 || K < 0) {
    set_error("trnblas_hip_grouped_plan: bad arguments");
    return nullptr;
  }
  if (op < 2 && (first * es % 16 != 0 || second * es % 16 != 0)) return "grouped_any_kernel";
  const int ring = op == 1 ? choose_rank_k((int)es, groups, rows, M, N) : gemm_choice(op, es, transB, groups, rows, N, K).ring;
  return ring < 0 ? "rows_kernel" : ring == kAnyTiles ? "grouped_any_kernel" : kRingNames[ring];
}
