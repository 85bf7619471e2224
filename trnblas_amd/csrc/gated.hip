// Gated projections H = act(A G) * (A U), [G | U] one matrix of 2 N columns: the C entry of the
// products (ring.hpp, rows.hpp) and the elementwise kernels beside them.
#include "gate.hpp"
#include "grouped.hpp"
#include "grouped_plan.hpp"

namespace trnblas {

static const char* const kGated = "trnblas_hip_gated_gemm";
static const char* const kGate = "trnblas_hip_gate";
static const char* const kGateBackward = "trnblas_hip_gate_backward";

struct GateArgs {
  const void* P;  // rows x 2 n: gates, then ups; fp32 (backward)
  int64_t ldp;
  const void* dH;  // backward
  int64_t ldg;
  void* D;  // H, or dP (backward)
  int64_t ldd;
  void* S;  // P in D's type, or null (forward)
  int64_t lds;
  int64_t rows;
  int n, act;
  int vec;  // whole groups of V values, every row's start aligned to them
};

// V values from p, as floats.
template <int V, typename T>
__device__ __forceinline__ void load_values(const T* p, float (&v)[V]) {
  typedef T tv __attribute__((ext_vector_type(V)));
  const tv w = *reinterpret_cast<const tv*>(p);
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = (float)w[i];
}
template <int V, typename T>
__device__ __forceinline__ void store_values(T* p, const float (&v)[V]) {
  typedef T tv __attribute__((ext_vector_type(V)));
  tv w;
#pragma unroll
  for (int i = 0; i < V; ++i) w[i] = (T)v[i];
  *reinterpret_cast<tv*>(p) = w;
}

// One thread takes V values of a row: 64 x 4 threads, columns by rows. Rows that start anywhere, or end inside eight
// values: one each, side by side (301 x 771 fp32: 3.0 us, with eight each 6.3).
constexpr int kGateV = 8;

template <typename T, typename O, int V>
__global__ __launch_bounds__(256) void gate_kernel(GateArgs g) {
  const int c = V * (blockIdx.x * 64 + threadIdx.x);
  if (c >= g.n) return;
  for (int64_t r = blockIdx.y * 4 + threadIdx.y; r < g.rows; r += 4 * gridDim.y) {
    const T* p = static_cast<const T*>(g.P) + r * g.ldp + c;
    float a[V], u[V], h[V];
    load_values<V>(p, a);
    load_values<V>(p + g.n, u);
#pragma unroll
    for (int i = 0; i < V; ++i) h[i] = gate(g.act, a[i]) * u[i];
    store_values<V>(static_cast<O*>(g.D) + r * g.ldd + c, h);
    if (g.S) {
      O* s = static_cast<O*>(g.S) + r * g.lds + c;
      store_values<V>(s, a);
      store_values<V>(s + g.n, u);
    }
  }
}

// dG = dH * U * act'(G), dU = dH * act(G), rounded once, to dH's type. The sums P = [G | U] are fp32: in fp16 a gate or an
// up past 65504 would be infinite where H and both gradients are not, and sums rounded to bf16 put the gradients
// 0.0030 of their norm from the 64-bit ones (0.0023). Four values a thread, 16 bytes of P: 8192 x 4096 bf16 88 us, 470 MB at
// 5.3 TB/s; eight 104.
template <typename T, int V>
__global__ __launch_bounds__(256) void gate_backward_kernel(GateArgs g) {
  const int c = V * (blockIdx.x * 64 + threadIdx.x);
  if (c >= g.n) return;
  for (int64_t r = blockIdx.y * 4 + threadIdx.y; r < g.rows; r += 4 * gridDim.y) {
    const float* p = static_cast<const float*>(g.P) + r * g.ldp + c;
    float a[V], u[V], d[V];
    load_values<V>(p, a);
    load_values<V>(p + g.n, u);
    load_values<V>(static_cast<const T*>(g.dH) + r * g.ldg + c, d);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float y, slope;
      gate_slope(g.act, a[i], y, slope);
      a[i] = d[i] * u[i] * slope;
      u[i] = d[i] * y;
    }
    T* o = static_cast<T*>(g.D) + r * g.ldd + c;
    store_values<V>(o, a);
    store_values<V>(o + g.n, u);
  }
}

static dim3 gate_grid(const GateArgs& g, int values) {
  const int64_t rows = (g.rows + 3) / 4;
  const int columns = 64 * (g.vec ? values : 1);
  return dim3((unsigned)((g.n + columns - 1) / columns), (unsigned)(rows < 32768 ? rows : 32768));
}

template <typename T, typename O>
static void launch_gate(const GateArgs& g, hipStream_t s) {
  if (g.vec)
    hipLaunchKernelGGL((gate_kernel<T, O, kGateV>), gate_grid(g, kGateV), dim3(64, 4), 0, s, g);
  else
    hipLaunchKernelGGL((gate_kernel<T, O, 1>), gate_grid(g, 1), dim3(64, 4), 0, s, g);
}

template <typename T>
static void launch_gate_backward(const GateArgs& g, hipStream_t s) {
  if (g.vec)
    hipLaunchKernelGGL((gate_backward_kernel<T, 4>), gate_grid(g, 4), dim3(64, 4), 0, s, g);
  else
    hipLaunchKernelGGL((gate_backward_kernel<T, 1>), gate_grid(g, 1), dim3(64, 4), 0, s, g);
}

static bool whole(const void* p, int64_t ld, int64_t n, int es) {
  const int v = kGateV * es < 16 ? kGateV * es : 16;
  return p == nullptr || ((uintptr_t)p % v == 0 && ld * es % v == 0 && n * es % v == 0);
}

static int check_gate(const char* what, int act, int dtype, int64_t rows, int64_t N) {
  TRNBLAS_CHECK_ARG(act >= TRNBLAS_ACT_SILU && act <= TRNBLAS_ACT_SIGMOID, "%s: bad activation %d", what, act);
  TRNBLAS_CHECK_ARG(dtype == TRNBLAS_F32 || dtype == TRNBLAS_BF16 || dtype == TRNBLAS_F16, "%s: bad dtype %d", what, dtype);
  TRNBLAS_CHECK_ARG(rows >= 0 && rows < INT32_MAX - 1024 && N >= 0 && N < (INT32_MAX >> 1) - 1024, "%s: bad sizes (rows %lld, N %lld)",
                    what, (long long)rows, (long long)N);
  return TRNBLAS_OK;
}

}  // namespace trnblas

using namespace trnblas;

extern "C" int trnblas_hip_gate(int act, int dtype, int out_dtype, int64_t rows, int64_t N, const void* P, int64_t ldp, void* H,
                                int64_t ldh, void* S, int64_t lds, void* stream) {
  if (int rc = check_gate(kGate, act, dtype, rows, N)) return rc;
  TRNBLAS_CHECK_ARG(out_dtype == dtype || (dtype == TRNBLAS_F32 && (out_dtype == TRNBLAS_BF16 || out_dtype == TRNBLAS_F16)),
                    "%s: bad result dtype %d", kGate, out_dtype);
  TRNBLAS_CHECK_ARG(ldp >= 2 * N && ldh >= N && (S == nullptr || lds >= 2 * N), "%s: bad leading dimension", kGate);
  if (rows == 0 || N == 0) return TRNBLAS_OK;
  TRNBLAS_CHECK_ARG(P != nullptr && H != nullptr, "%s: null operand", kGate);
  const int es = dtype == TRNBLAS_F32 ? 4 : 2, eo = out_dtype == TRNBLAS_F32 ? 4 : 2;
  GateArgs g{};
  g.P = P, g.ldp = ldp, g.D = H, g.ldd = ldh, g.S = S, g.lds = lds;
  g.rows = rows, g.n = (int)N, g.act = act;
  g.vec = N % kGateV == 0 && whole(P, ldp, N, es) && whole(H, ldh, N, eo) && whole(S, lds, N, eo);
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype == TRNBLAS_F32 ? 3 + out_dtype : dtype) {
    case TRNBLAS_BF16: launch_gate<__bf16, __bf16>(g, s); break;
    case TRNBLAS_F16: launch_gate<_Float16, _Float16>(g, s); break;
    case 3 + TRNBLAS_BF16: launch_gate<float, __bf16>(g, s); break;
    case 3 + TRNBLAS_F16: launch_gate<float, _Float16>(g, s); break;
    default: launch_gate<float, float>(g, s); break;
  }
  return check_launch(kGate);
}

extern "C" int trnblas_hip_gate_backward(int act, int dtype, int64_t rows, int64_t N, const float* P, int64_t ldp, const void* dH,
                                         int64_t ldg, void* dP, int64_t ldd, void* stream) {
  if (int rc = check_gate(kGateBackward, act, dtype, rows, N)) return rc;
  TRNBLAS_CHECK_ARG(ldp >= 2 * N && ldg >= N && ldd >= 2 * N, "%s: bad leading dimension", kGateBackward);
  if (rows == 0 || N == 0) return TRNBLAS_OK;
  TRNBLAS_CHECK_ARG(P != nullptr && dH != nullptr && dP != nullptr, "%s: null operand", kGateBackward);
  const int es = dtype == TRNBLAS_F32 ? 4 : 2;
  GateArgs g{};
  g.P = P, g.ldp = ldp, g.dH = dH, g.ldg = ldg, g.D = dP, g.ldd = ldd;
  g.rows = rows, g.n = (int)N, g.act = act;
  g.vec = N % kGateV == 0 && whole(P, ldp, N, 4) && whole(dH, ldg, N, es) && whole(dP, ldd, N, es);
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case TRNBLAS_F32: launch_gate_backward<float>(g, s); break;
    case TRNBLAS_BF16: launch_gate_backward<__bf16>(g, s); break;
    default: launch_gate_backward<_Float16>(g, s); break;
  }
  return check_launch(kGateBackward);
}

extern "C" int trnblas_hip_gated_gemm(int act, int dtype, int transB, int64_t groups, int64_t rows, int64_t N, int64_t K,
                                      const void* A, int64_t lda, const void* B, int64_t ldb, int64_t strideB, int64_t strideU,
                                      const void* offsets, int offsets64, void* H, int64_t ldh, float* P, int64_t ldp, int padded,
                                      void* stream) {
  if (int rc = check_gate(kGated, act, dtype, rows, N)) return rc;
  TRNBLAS_CHECK_ARG(groups >= 0 && groups < (1 << 24) && K >= 0 && K < INT32_MAX - 1024, "%s: bad sizes (groups %lld, K %lld)", kGated,
                    (long long)groups, (long long)K);
  TRNBLAS_CHECK_ARG(offsets != nullptr ? (uintptr_t)offsets % (offsets64 ? 8 : 4) == 0 : groups == 1,
                    "%s: offsets missing or misaligned", kGated);
  TRNBLAS_CHECK_ARG(lda >= K && ldb >= (transB ? K : N) && strideB >= 0 && strideU >= 0 && ldh >= N && (P == nullptr || ldp >= 2 * N),
                    "%s: bad leading dimension", kGated);
  if (rows == 0 || N == 0) return TRNBLAS_OK;
  TRNBLAS_CHECK_ARG(H != nullptr && ((A != nullptr && B != nullptr) || K == 0 || groups == 0), "%s: null operand", kGated);
  GroupedArgs g{};
  g.A = A, g.lda = lda;
  g.B = B, g.ldb = ldb, g.sB = strideB, g.sU = strideU;
  g.D = H, g.ldd = ldh;
  g.P = P, g.ldp = ldp;
  g.offsets = offsets, g.offsets64 = offsets64 != 0;
  g.groups = (int)groups, g.rows = (int)rows, g.N = (int)N, g.K = (int)K;
  g.alpha = 1.0f;
  g.act = act;
  g.out32 = dtype == TRNBLAS_F32;
  g.padded = padded != 0;
  const int64_t eo = g.out32 ? 4 : 2;
  g.vec4 = (uintptr_t)H % (4 * eo) == 0 && ldh % 4 == 0 &&
           (P == nullptr || ((uintptr_t)P % 16 == 0 && ldp % 4 == 0 && N % 4 == 0));
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case TRNBLAS_F32: return gated_gemm_run<float>(g, transB != 0, s);
    case TRNBLAS_BF16: return gated_gemm_run<__bf16>(g, transB != 0, s);
    default: return gated_gemm_run<_Float16>(g, transB != 0, s);
  }
}

extern "C" const char* trnblas_hip_gated_plan(int dtype, int transB, int64_t groups, int64_t rows, int64_t N, int64_t K) {
  static const char* const kRing[] = {"gated_ring_kernel 256 x 128", "gated_ring_kernel 128 x 64", "gated_ring_kernel 64 x 64"};
  static const char* const kRows[] = {"rows_kernel 16 1", "rows_kernel 16 2", "rows_kernel 16 4", "rows_kernel 16 8", "rows_kernel 32 8"};
  if (dtype < 0 || dtype > 2 || groups < 1 || rows < 1 || N < 1 || K < 0) {
    set_error("trnblas_hip_gated_plan: bad arguments");
    return nullptr;
  }
  const GroupedChoice c = choose_gated(dtype == TRNBLAS_F32 ? 4 : 2, rows, groups, N, K, transB != 0);
  if (c.ring >= 0) return kRing[c.ring];
  return kRows[c.mf == 2 ? 4 : c.ks == 8 ? 3 : c.ks / 2];
}
