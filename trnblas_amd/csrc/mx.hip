// Microscaled 4-bit floats: quantisation, its reverse, and products of such
// operands (one matrix, or one per ragged group of rows).
//
// A value is an e2m1 code (0, .5, 1, 1.5, 2, 3, 4, 6 and a sign) times 2^e, one
// e per 32 values along K, stored as the byte e + 127; byte 255 makes its 32
// values NaN. Layout of a matrix of R rows by K:
//  * codes: row-major, two per byte (the even one low), rows of Kp / 2 bytes, Kp
//    = K rounded up to 32 (the last block filled with zeros);
//  * scales: as v_mfma_scale_f32_16x16x128_f8f6f4 takes them. A chunk of 256
//    bytes serves 16 rows by 512 values of K: byte 64 (b % 4) + 4 r + b / 4 is row r,
//    block b of its 16. Lane l of an MFMA holds row l % 16 and block l / 16 of
//    four, so one dword per lane holds its scales of four MFMAs along K, and the
//    64 lanes read 256 bytes in a row.
#include <algorithm>

#include "grouped_plan.hpp"
#include "ring.hpp"
#include "rows.hpp"

namespace trnblas {

static const char* kQuantize = "trnblas_hip_mx_quantize";
static const char* kDequantize = "trnblas_hip_mx_dequantize";
static const char* kMxGemm = "trnblas_hip_mx_gemm";

struct QuantArgs {
  const void* X;
  int64_t sr, sk, sx;  // strides of rows, K and batch, in elements
  int R, K;
  int chunks;    // of scales along K
  int row_bytes;  // of codes
  uint8_t* codes;
  uint8_t* scales;
  int vec;  // 16-byte loads (K-contiguous: every row starts on 16 bytes)
};

// Rows by K, 16 rows x 512 values per workgroup of 256 threads: a wave takes
// four rows, a lane eight values of each, four lanes a block. Bound by memory: 8192 x
// 8192 bf16 28 us, fp32 49 us (6.1 and 6.2 TB/s).
template <typename T>
__global__ __launch_bounds__(256) void mx_quantize_kernel(QuantArgs g) {
  __shared__ uint32_t sc[kChunk / 4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int block = blockIdx.x / g.chunks, chunk = blockIdx.x - block * g.chunks, r0 = block * 16;
  const int k = chunk * 512 + 8 * lane;
  const T* X = static_cast<const T*>(g.X) + blockIdx.y * g.sx;
  float v[4][8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = r0 + 4 * wave + i;
    const int left = r < g.R ? g.K - k : 0;
    const T* p = X + r * g.sr + k * g.sk;
    if (g.vec && left >= 8) {
      union {
        i32x4 w[sizeof(T) / 2];
        T e[8];
      } u;
#pragma unroll
      for (int h = 0; h < (int)sizeof(T) / 2; ++h) u.w[h] = reinterpret_cast<const i32x4*>(p)[h];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] = (float)u.e[e];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] = e < left ? (float)p[e * g.sk] : 0.0f;
    }
  }
  uint8_t* codes = g.codes + (int64_t)blockIdx.y * g.R * g.row_bytes;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int rr = 4 * wave + i;
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, __builtin_bit_cast(uint32_t, v[i][e]) & 0x7fffffffu);
    top = max(top, (uint32_t)__shfl_xor((int)top, 1));
    top = max(top, (uint32_t)__shfl_xor((int)top, 2));
    const uint32_t byte = scale_byte(top);
    const uint32_t c = byte == 255 ? 0u : codes8(v[i], inverse_scale(byte));
    const int off = k >> 1;
    if (r0 + rr < g.R && off < g.row_bytes) *reinterpret_cast<uint32_t*>(codes + (int64_t)(r0 + rr) * g.row_bytes + off) = c;
    const int b = lane >> 2;
    if ((lane & 3) == 0) reinterpret_cast<uint8_t*>(sc)[64 * (b & 3) + 4 * rr + (b >> 2)] = (uint8_t)byte;
  }
  __syncthreads();
  if (tid < kChunk / 4) {
    uint8_t* scales = g.scales + ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * kChunk;
    reinterpret_cast<uint32_t*>(scales)[tid] = sc[tid];
  }
}

// K by rows (a row's values are sk apart, rows next to each other): 64 rows x 128
// values per workgroup, a wave one block of 32 of each row, a lane one row, so
// that its loads are 64 neighbouring values; the codes go out through LDS, 64 bytes
// per row. Bound by memory: 8192 x 8192 bf16 28 us (6.1 TB/s).
template <typename T>
__global__ __launch_bounds__(256) void mx_quantize_columns_kernel(QuantArgs g) {
  __shared__ __attribute__((aligned(16))) char sc[64 * 80];  // 16 bytes between rows
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int tiles_k = g.chunks * 4;
  const int tr = blockIdx.x / tiles_k, tk = blockIdx.x - tr * tiles_k;
  const int r = tr * 64 + lane, b = tk * 4 + wave, k = 32 * b;
  const int left = r < g.R ? g.K - k : 0;
  const T* p = static_cast<const T*>(g.X) + blockIdx.y * g.sx + r * g.sr + k * g.sk;
  float v[4][8];
  if (left >= 32) {
#pragma unroll
    for (int e = 0; e < 32; ++e) v[e / 8][e % 8] = (float)p[e * g.sk];
  } else {
#pragma unroll
    for (int e = 0; e < 32; ++e) v[e / 8][e % 8] = e < left ? (float)p[e * g.sk] : 0.0f;
  }
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 32; ++e) top = max(top, __builtin_bit_cast(uint32_t, v[e / 8][e % 8]) & 0x7fffffffu);
  const uint32_t byte = scale_byte(top);
  i32x4 c = {0, 0, 0, 0};
  if (byte != 255) {
#pragma unroll
    for (int q = 0; q < 4; ++q) c[q] = (int)codes8(v[q], inverse_scale(byte));
  }
  *reinterpret_cast<i32x4*>(sc + 80 * lane + 16 * wave) = c;
  const int row_blocks = (g.R + 15) / 16;
  if (r < 16 * row_blocks) {
    uint8_t* scales = g.scales + (((int64_t)blockIdx.y * row_blocks + (r >> 4)) * g.chunks + (b >> 4)) * kChunk;
    scales[64 * (b & 3) + 4 * (r & 15) + ((b >> 2) & 3)] = (uint8_t)byte;
  }
  __syncthreads();
  const int row = tr * 64 + threadIdx.x / 4, off = 64 * tk + 16 * (threadIdx.x & 3);
  if (row < g.R && off < g.row_bytes)
    *reinterpret_cast<i32x4*>(g.codes + ((int64_t)blockIdx.y * g.R + row) * g.row_bytes + off) =
        *reinterpret_cast<const i32x4*>(sc + 80 * (threadIdx.x / 4) + 16 * (threadIdx.x & 3));
}

struct DequantArgs {
  const uint8_t* codes;
  const uint8_t* scales;
  int R, K, chunks, row_bytes;
  void* D;
  int64_t ldd, sD;
  int vec;
};

template <typename T>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(DequantArgs g) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int block = blockIdx.x / g.chunks, chunk = blockIdx.x - block * g.chunks, r0 = block * 16;
  const uint8_t* codes = g.codes + (int64_t)blockIdx.y * g.R * g.row_bytes;
  const uint8_t* scales = g.scales + ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * kChunk;
  constexpr int V = 16 / sizeof(T);  // values of a lane's 16-byte store, neighbours of the next lane's
#pragma unroll
  for (int i = 0; i < 4 * 8 / V; ++i) {
    const int rr = 4 * wave + i / (8 / V), r = r0 + rr;
    const int kk = V * (64 * (i % (8 / V)) + lane), k = chunk * 512 + kk, b = kk >> 5;
    const int left = r < g.R ? g.K - k : 0;
    if (left <= 0) continue;
    const uint8_t* p = codes + (int64_t)r * g.row_bytes + (k >> 1);
    const uint32_t c = V == 8 ? *reinterpret_cast<const uint32_t*>(p) : *reinterpret_cast<const uint16_t*>(p);
    const uint32_t byte = scales[64 * (b & 3) + 4 * rr + (b >> 2)];
    const float s = byte == 255 ? __builtin_nanf("") : __builtin_bit_cast(float, byte ? byte << 23 : 0x00400000u);
    T o[V];
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    each<V / 2>([&](auto uc) __attribute__((always_inline)) {
      constexpr int u = decltype(uc)::value;
      const f32x2 x = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, u);
      o[2 * u] = (T)(x[0] * s);
      o[2 * u + 1] = (T)(x[1] * s);
    });
    T* d = static_cast<T*>(g.D) + blockIdx.y * g.sD + r * g.ldd + k;
    if (g.vec && left >= V) {
      *reinterpret_cast<i32x4*>(d) = *reinterpret_cast<const i32x4*>(o);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (e < left) d[e] = o[e];
    }
  }
}

// Bound on the tiles of bm rows (see ragged_tile).
static int64_t mx_tiles(const GroupedArgs& g, int bm) {
  return (g.rows / bm + std::min<int64_t>(g.groups + 2, g.rows)) * g.tiles_n;
}

static int mx_grid(int64_t tiles, unsigned* grid) {
  TRNBLAS_CHECK_ARG(tiles < ((int64_t)1 << 31) - 4096, "%s: too many tiles", kMxGemm);
  *grid = (unsigned)((tiles + kNumXcd - 1) / kNumXcd * kNumXcd);
  return TRNBLAS_OK;
}

template <int FM, int FN>
static int run_ring(GroupedArgs g, const MxScales& x, hipStream_t s) {
  constexpr int BM = 32 * FM, BN = 32 * FN;
  g.tiles_n = (g.N + BN - 1) / BN;
  unsigned grid;
  if (int rc = mx_grid(ring_grid<FM, FN>(g, mx_tiles(g, BM)), &grid)) return rc;
  hipLaunchKernelGGL((ring_kernel<fp4x2, FM, FN, true, false>), dim3(grid), dim3(256), 0, s, g, x);
  return check_launch(kMxGemm);
}

template <int MF, int KS, typename X>
static int run_rows(GroupedArgs g, const MxScales& x, hipStream_t s) {
  constexpr int BN = 128 / KS;
  g.tiles_n = (g.N + BN - 1) / BN;
  unsigned grid;
  if (int rc = mx_grid(mx_tiles(g, 16 * MF), &grid)) return rc;
  hipLaunchKernelGGL((rows_kernel<fp4x2, MF, 1, KS, true, X>), dim3(grid), dim3(512), 0, s, g, x);
  return check_launch(kMxGemm);
}

template <int MF, typename X = void>
static int run_rows_split(int ks, const GroupedArgs& g, const MxScales& x, hipStream_t s) {
  return ks == 8   ? run_rows<MF, 8, X>(g, x, s)
         : ks == 4 ? run_rows<MF, 4, X>(g, x, s)
         : ks == 2 ? run_rows<MF, 2, X>(g, x, s)
                   : run_rows<MF, 1, X>(g, x, s);
}

static int run_mx(const GroupedChoice& c, const GroupedArgs& g, const MxScales& x, hipStream_t s) {
  switch (c.ring) {
    case 0: return run_ring<8, 8>(g, x, s);
    case 1: return run_ring<4, 4>(g, x, s);
    case 2: return run_ring<2, 4>(g, x, s);
    default: return c.mf == 1 ? run_rows_split<1>(c.ks, g, x, s) : run_rows_split<2>(c.ks, g, x, s);
  }
}

static int check_layout(const char* what, int64_t R, int64_t K, int64_t batch) {
  TRNBLAS_CHECK_ARG(R >= 0 && R < INT32_MAX - 1024 && K >= 0 && K < INT32_MAX - 1024 && batch >= 0 && batch < 65536,
                    "%s: bad sizes (rows %lld, K %lld, batch %lld)", what, (long long)R, (long long)K, (long long)batch);
  return TRNBLAS_OK;
}

// Workgroups of 16 rows by 512 values per matrix, the chunks of a row block in a
// row; the matrix is the grid's y.
static int chunk_grid(const char* what, int64_t R, int64_t K, int64_t batch, dim3* grid) {
  const int64_t n = (R + 15) / 16 * ((K + 511) / 512);
  TRNBLAS_CHECK_ARG(n < (int64_t)1 << 31, "%s: matrix too large (%lld x %lld)", what, (long long)R, (long long)K);
  *grid = dim3((unsigned)n, (unsigned)batch);
  return TRNBLAS_OK;
}

}  // namespace trnblas

using namespace trnblas;

extern "C" int trnblas_hip_mx_quantize(int dtype, int64_t R, int64_t K, const void* X, int64_t sr, int64_t sk, int64_t sx,
                                       void* codes, void* scales, int64_t batch, void* stream) {
  TRNBLAS_CHECK_ARG(dtype == TRNBLAS_F32 || dtype == TRNBLAS_BF16 || dtype == TRNBLAS_F16, "%s: bad dtype %d", kQuantize, dtype);
  if (int rc = check_layout(kQuantize, R, K, batch)) return rc;
  TRNBLAS_CHECK_ARG(sr >= 0 && sk >= 0 && sx >= 0, "%s: negative stride", kQuantize);
  if (R == 0 || K == 0 || batch == 0) return TRNBLAS_OK;
  TRNBLAS_CHECK_ARG(X != nullptr && codes != nullptr && scales != nullptr, "%s: null operand", kQuantize);
  TRNBLAS_CHECK_ARG((uintptr_t)codes % 16 == 0 && (uintptr_t)scales % 16 == 0, "%s: codes and scales must be 16-byte aligned", kQuantize);
  dim3 grid;
  if (int rc = chunk_grid(kQuantize, R, K, batch, &grid)) return rc;
  const int es = dtype == TRNBLAS_F32 ? 4 : 2;
  QuantArgs g{};
  g.X = X, g.sr = sr, g.sk = sk, g.sx = sx;
  g.R = (int)R, g.K = (int)K;
  g.chunks = (int)((K + 511) / 512);
  g.row_bytes = (int)((K + 31) / 32 * 16);
  g.codes = static_cast<uint8_t*>(codes);
  g.scales = static_cast<uint8_t*>(scales);
  g.vec = sk == 1 && (uintptr_t)X % 16 == 0 && sr * es % 16 == 0 && sx * es % 16 == 0;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (sr == 1 && sk > 1 && R >= 16) {
    const int64_t tiles = (R + 63) / 64 * 4 * g.chunks;
    TRNBLAS_CHECK_ARG(tiles < (int64_t)1 << 31, "%s: matrix too large (%lld x %lld)", kQuantize, (long long)R, (long long)K);
    const dim3 by_columns((unsigned)tiles, (unsigned)batch);
    switch (dtype) {
      case TRNBLAS_F32: hipLaunchKernelGGL(mx_quantize_columns_kernel<float>, by_columns, dim3(256), 0, s, g); break;
      case TRNBLAS_BF16: hipLaunchKernelGGL(mx_quantize_columns_kernel<__bf16>, by_columns, dim3(256), 0, s, g); break;
      default: hipLaunchKernelGGL(mx_quantize_columns_kernel<_Float16>, by_columns, dim3(256), 0, s, g); break;
    }
    return check_launch(kQuantize);
  }
  switch (dtype) {
    case TRNBLAS_F32: hipLaunchKernelGGL(mx_quantize_kernel<float>, grid, dim3(256), 0, s, g); break;
    case TRNBLAS_BF16: hipLaunchKernelGGL(mx_quantize_kernel<__bf16>, grid, dim3(256), 0, s, g); break;
    default: hipLaunchKernelGGL(mx_quantize_kernel<_Float16>, grid, dim3(256), 0, s, g); break;
  }
  return check_launch(kQuantize);
}

extern "C" int trnblas_hip_mx_dequantize(int dtype, int64_t R, int64_t K, const void* codes, const void* scales, void* D,
                                         int64_t ldd, int64_t strideD, int64_t batch, void* stream) {
  TRNBLAS_CHECK_ARG(dtype == TRNBLAS_F32 || dtype == TRNBLAS_BF16 || dtype == TRNBLAS_F16, "%s: bad dtype %d", kDequantize, dtype);
  if (int rc = check_layout(kDequantize, R, K, batch)) return rc;
  TRNBLAS_CHECK_ARG(ldd >= K && strideD >= 0, "%s: bad leading dimension", kDequantize);
  if (R == 0 || K == 0 || batch == 0) return TRNBLAS_OK;
  TRNBLAS_CHECK_ARG(D != nullptr && codes != nullptr && scales != nullptr, "%s: null operand", kDequantize);
  TRNBLAS_CHECK_ARG((uintptr_t)codes % 16 == 0 && (uintptr_t)scales % 16 == 0, "%s: codes and scales must be 16-byte aligned", kDequantize);
  dim3 grid;
  if (int rc = chunk_grid(kDequantize, R, K, batch, &grid)) return rc;
  const int es = dtype == TRNBLAS_F32 ? 4 : 2;
  DequantArgs g{};
  g.codes = static_cast<const uint8_t*>(codes);
  g.scales = static_cast<const uint8_t*>(scales);
  g.R = (int)R, g.K = (int)K;
  g.chunks = (int)((K + 511) / 512);
  g.row_bytes = (int)((K + 31) / 32 * 16);
  g.D = D, g.ldd = ldd, g.sD = strideD;
  g.vec = (uintptr_t)D % 16 == 0 && ldd * es % 16 == 0 && strideD * es % 16 == 0;
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case TRNBLAS_F32: hipLaunchKernelGGL(mx_dequantize_kernel<float>, grid, dim3(256), 0, s, g); break;
    case TRNBLAS_BF16: hipLaunchKernelGGL(mx_dequantize_kernel<__bf16>, grid, dim3(256), 0, s, g); break;
    default: hipLaunchKernelGGL(mx_dequantize_kernel<_Float16>, grid, dim3(256), 0, s, g); break;
  }
  return check_launch(kDequantize);
}

// The checks and arguments that both products share; K in values.
static int mx_args(GroupedArgs& g, MxScales& x, int out_dtype, int64_t groups, int64_t rows, int64_t N, int64_t K, double alpha,
                   const void* B, const void* B_scales, const void* offsets, int offsets64, double beta, const void* C, int64_t ldc,
                   void* D, int64_t ldd) {
  TRNBLAS_CHECK_ARG(out_dtype == TRNBLAS_F32 || out_dtype == TRNBLAS_BF16 || out_dtype == TRNBLAS_F16, "%s: bad dtype %d", kMxGemm, out_dtype);
  // K: a panel's codes and a tile's scales lie within 32-bit offsets
  TRNBLAS_CHECK_ARG(groups >= 0 && groups < (1 << 24) && rows >= 0 && rows < INT32_MAX - 1024 && N >= 0 &&
                        N < INT32_MAX - 1024 && K >= 0 && K < 8 << 20,
                    "%s: bad sizes (groups %lld, rows %lld, N %lld, K %lld)", kMxGemm, (long long)groups, (long long)rows,
                    (long long)N, (long long)K);
  TRNBLAS_CHECK_ARG(offsets != nullptr ? (uintptr_t)offsets % (offsets64 ? 8 : 4) == 0 : groups == 1,
                    "%s: offsets missing or misaligned", kMxGemm);
  TRNBLAS_CHECK_ARG(beta == 0.0 || C != nullptr, "%s: beta != 0 without C", kMxGemm);
  TRNBLAS_CHECK_ARG(ldd >= N && (beta == 0.0 || ldc >= N), "%s: bad leading dimension", kMxGemm);
  if (rows == 0 || N == 0) return TRNBLAS_OK;
  TRNBLAS_CHECK_ARG(D != nullptr && (K == 0 || groups == 0 || (B && B_scales)), "%s: null operand", kMxGemm);
  TRNBLAS_CHECK_ARG((uintptr_t)B % 16 == 0 && (uintptr_t)B_scales % 16 == 0, "%s: codes and scales must be 16-byte aligned", kMxGemm);
  g.B = B;
  g.lda = g.ldb = (K + 31) / 32 * 16;
  g.sB = N * g.ldb;
  x.b = static_cast<const uint8_t*>(B_scales);
  x.chunks = (int)((K + 511) / 512);
  x.b_step = (N + 15) / 16 * x.chunks * kChunk;
  g.offsets = offsets;
  g.offsets64 = offsets64 != 0;
  g.groups = (int)groups, g.rows = (int)rows, g.N = (int)N, g.K = (int)g.lda;  // bytes of codes along K
  g.alpha = (float)alpha, g.beta = (float)beta;
  g.C = beta != 0.0 ? C : nullptr, g.ldc = ldc;
  g.D = D, g.ldd = ldd;
  g.out32 = out_dtype == TRNBLAS_F32, g.out_f16 = out_dtype == TRNBLAS_F16;
  const int eo = g.out32 ? 4 : 2;
  g.vec4 = (uintptr_t)D % (4 * eo) == 0 && ldd % 4 == 0 && (g.C == nullptr || ((uintptr_t)C % (4 * eo) == 0 && ldc % 4 == 0));
  return TRNBLAS_OK;
}

static size_t codes_bytes(int64_t rows, int64_t K) { return (size_t)(rows * ((K + 31) / 32 * 16)); }
static size_t scales_bytes(int64_t rows, int64_t K) { return (size_t)((rows + 15) / 16 * ((K + 511) / 512) * kChunk); }

extern "C" int trnblas_hip_mx_gemm(int out_dtype, int64_t groups, int64_t rows, int64_t N, int64_t K, double alpha,
                                   const void* A, const void* A_scales, const void* B, const void* B_scales,
                                   const void* offsets, int offsets64, double beta, const void* C, int64_t ldc, void* D,
                                   int64_t ldd, void* stream) {
  GroupedArgs g{};
  MxScales x{};
  if (int rc = mx_args(g, x, out_dtype, groups, rows, N, K, alpha, B, B_scales, offsets, offsets64, beta, C, ldc, D, ldd)) return rc;
  if (rows == 0 || N == 0) return TRNBLAS_OK;
  TRNBLAS_CHECK_ARG(K == 0 || groups == 0 || (A && A_scales), "%s: null operand", kMxGemm);
  TRNBLAS_CHECK_ARG((uintptr_t)A % 16 == 0 && (uintptr_t)A_scales % 16 == 0, "%s: codes and scales must be 16-byte aligned", kMxGemm);
  g.A = A;
  x.a = static_cast<const uint8_t*>(A_scales);
  return run_mx(choose_mx(rows, groups, N, K), g, x, static_cast<hipStream_t>(stream));
}

extern "C" size_t trnblas_hip_mx_gemm_from_workspace(int64_t rows, int64_t K) {
  if (rows <= 0 || K <= 0) return 0;
  return (codes_bytes(rows, K) + 255) / 256 * 256 + scales_bytes(rows, K);
}

extern "C" int trnblas_hip_mx_gemm_from(int dtype, int out_dtype, int64_t groups, int64_t rows, int64_t N, int64_t K, double alpha,
                                        const void* A, int64_t sr, int64_t sk, const void* B, const void* B_scales,
                                        const void* offsets, int offsets64, double beta, const void* C, int64_t ldc, void* D,
                                        int64_t ldd, void* workspace, size_t workspace_bytes, void* stream) {
  GroupedArgs g{};
  MxScales x{};
  TRNBLAS_CHECK_ARG(dtype == TRNBLAS_F32 || dtype == TRNBLAS_BF16 || dtype == TRNBLAS_F16, "%s: bad dtype %d", kMxGemm, dtype);
  TRNBLAS_CHECK_ARG(sr >= 0 && sk >= 0, "%s: negative stride", kMxGemm);
  if (int rc = mx_args(g, x, out_dtype, groups, rows, N, K, alpha, B, B_scales, offsets, offsets64, beta, C, ldc, D, ldd)) return rc;
  if (rows == 0 || N == 0) return TRNBLAS_OK;
  TRNBLAS_CHECK_ARG(K == 0 || groups == 0 || A, "%s: null operand", kMxGemm);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const GroupedChoice c = choose_mx(rows, groups, N, K);
  if (sk == 1 && quantised_in_place(c, rows, K)) {
    const int es = dtype == TRNBLAS_F32 ? 4 : 2;
    x.x = A, x.ldx = sr, x.kx = (int)K;
    x.vec = (uintptr_t)A % 16 == 0 && (sr * es % 16 == 0 || rows == 1);
    switch (dtype) {
      case TRNBLAS_F32: return run_rows_split<1, float>(c.ks, g, x, s);
      case TRNBLAS_BF16: return run_rows_split<1, __bf16>(c.ks, g, x, s);
      default: return run_rows_split<1, _Float16>(c.ks, g, x, s);
    }
  }
  if (K > 0 && groups > 0) {
    const size_t need = trnblas_hip_mx_gemm_from_workspace(rows, K);
    if (workspace == nullptr || workspace_bytes < need || (uintptr_t)workspace % 16 != 0) {
      set_error("%s: workspace of %zu bytes, 16-byte aligned, needed (got %zu)", kMxGemm, need, workspace_bytes);
      return TRNBLAS_E_WORKSPACE;
    }
    uint8_t* codes = static_cast<uint8_t*>(workspace);
    uint8_t* scales = codes + (codes_bytes(rows, K) + 255) / 256 * 256;
    if (int rc = trnblas_hip_mx_quantize(dtype, rows, K, A, sr, sk, 0, codes, scales, 1, stream)) return rc;
    g.A = codes;
    x.a = scales;
  }
  return run_mx(c, g, x, s);
}
