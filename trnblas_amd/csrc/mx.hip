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

#include "grouped.hpp"

namespace trnblas {

typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int kChunk = 256;  // bytes of scales per 16 rows x 512 values

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

// Scale byte of a block whose largest magnitude has these bits (as fp32):
// floor(log2) - 2 so that it lands in [4, 8), not below 2^-127; infinities and
// NaN give 255.
__device__ __forceinline__ uint32_t scale_byte(uint32_t top) {
  const uint32_t e = top >> 23;
  return e == 255 ? 255u : e > 2 ? e - 2 : 0u;
}
// 2^-(byte - 127)
__device__ __forceinline__ float inverse_scale(uint32_t byte) { return __builtin_bit_cast(float, (254u - byte) << 23); }

// Eight values times inv (exact but for results far below 0.25) to eight
// codes: the conversion rounds to nearest even and saturates at 6.
__device__ __forceinline__ uint32_t codes8(const float (&v)[8], float inv) {
  uint32_t c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0] * inv, v[1] * inv, 1.0f, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2] * inv, v[3] * inv, 1.0f, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4] * inv, v[5] * inv, 1.0f, 2);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6] * inv, v[7] * inv, 1.0f, 3);
  return c;
}

// Rows by K, 16 rows x 512 values per workgroup of 256 threads: a wave takes
// four rows, a lane eight values of each, four lanes a block.
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
  const int k = chunk * 512 + 8 * lane, b = lane >> 2;
  const uint8_t* codes = g.codes + (int64_t)blockIdx.y * g.R * g.row_bytes;
  const uint8_t* scales = g.scales + ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * kChunk;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int rr = 4 * wave + i, r = r0 + rr;
    const int left = r < g.R ? g.K - k : 0;
    if (left <= 0) continue;
    const uint32_t c = *reinterpret_cast<const uint32_t*>(codes + (int64_t)r * g.row_bytes + (k >> 1));
    const uint32_t byte = scales[64 * (b & 3) + 4 * rr + (b >> 2)];
    const float s = byte == 255 ? __builtin_nanf("") : __builtin_bit_cast(float, byte ? byte << 23 : 0x00400000u);
    T o[8];
    typedef float f32x2 __attribute__((ext_vector_type(2)));
#define TRNBLAS_PAIR(i)                                                        \
  {                                                                            \
    const f32x2 x = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, i);      \
    o[2 * i] = (T)(x[0] * s);                                                  \
    o[2 * i + 1] = (T)(x[1] * s);                                              \
  }
    TRNBLAS_PAIR(0)
    TRNBLAS_PAIR(1)
    TRNBLAS_PAIR(2)
    TRNBLAS_PAIR(3)
#undef TRNBLAS_PAIR
    T* d = static_cast<T*>(g.D) + blockIdx.y * g.sD + r * g.ldd + k;
    if (g.vec && left >= 8) {
#pragma unroll
      for (int h = 0; h < (int)sizeof(T) / 2; ++h) reinterpret_cast<i32x4*>(d)[h] = reinterpret_cast<const i32x4*>(o)[h];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < left) d[e] = o[e];
    }
  }
}

// acc += (16 rows n) x (16 rows m) over 128 values of K; byte J of each scale
// dword. Lane l holds column m = l % 16 and rows n = 4 (l / 16) + r.
template <int J>
__device__ __forceinline__ void mma_mx(f32x4& acc, const i32x4& n, const i32x4& m, int sn, int sm) {
  const i32x8 a = {n[0], n[1], n[2], n[3], 0, 0, 0, 0}, b = {m[0], m[1], m[2], m[3], 0, 0, 0, 0};
  acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 4, 4, J, sn, J, sm);
}

struct MxArgs {
  GroupedArgs g;  // A, B: codes; lda, ldb: bytes per row; sB: bytes per matrix
  const uint8_t* sa;
  const uint8_t* sb;
  int chunks;       // of scales along K, the same for A and B
  int64_t sb_step;  // bytes of scales per matrix of B
};

// 64 x 64 tiles, each wave 32 x 32, its fragments straight from memory.
template <typename O>
__global__ __launch_bounds__(256) void mx_any_kernel(MxArgs x) {
  const GroupedArgs& g = x.g;
  Segment s;
  if (!ragged_tile<64>(g, blockIdx.x, 8, s)) return;
  const bool of_group = s.group >= 0 && s.group < g.groups;
  const int lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m0 = s.row + 32 * (wave & 1), n0 = s.tn * 64 + 32 * (wave >> 1);
  const int nk = of_group ? (int)((g.lda + 63) / 64) : 0;  // 64-byte k-tiles
  const uint8_t *pa[2], *pb[2];
  const uint32_t *qa[2], *qb[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    // rows past the segment or the matrix repeat its last one: not stored
    const int64_t m = min(m0 + 16 * i + li, s.end - 1), n = min(n0 + 16 * i + li, g.N - 1);
    pa[i] = static_cast<const uint8_t*>(g.A) + m * g.lda + 16 * lg;
    pb[i] = static_cast<const uint8_t*>(g.B) + s.group * g.sB + n * g.ldb + 16 * lg;
    qa[i] = reinterpret_cast<const uint32_t*>(x.sa + (m >> 4) * x.chunks * kChunk + 64 * lg + 4 * (m & 15));
    qb[i] = reinterpret_cast<const uint32_t*>(x.sb + s.group * x.sb_step + (n >> 4) * x.chunks * kChunk + 64 * lg + 4 * (n & 15));
  }
  f32x4 acc[2][2];
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int b = 0; b < 2; ++b) acc[a][b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  auto tile = [&](int kt, auto j, const int (&sa)[2], const int (&sb)[2]) __attribute__((always_inline)) {
    if (kt >= nk) return;
    i32x4 fa[2], fb[2];
    const bool in = 64 * kt + 16 * lg < (int)g.lda;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      fa[i] = fb[i] = i32x4{0, 0, 0, 0};
      if (in) {
        fa[i] = *reinterpret_cast<const i32x4*>(pa[i] + 64 * kt);
        fb[i] = *reinterpret_cast<const i32x4*>(pb[i] + 64 * kt);
      }
    }
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int a = 0; a < 2; ++a) mma_mx<decltype(j)::value>(acc[a][b], fb[b], fa[a], sb[b], sa[a]);
  };
  for (int c = 0; 4 * c < nk; ++c) {
    int sa[2], sb[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      sa[i] = qa[i][c * (kChunk / 4)];
      sb[i] = qb[i][c * (kChunk / 4)];
    }
    tile(4 * c, std::integral_constant<int, 0>{}, sa, sb);
    tile(4 * c + 1, std::integral_constant<int, 1>{}, sa, sb);
    tile(4 * c + 2, std::integral_constant<int, 2>{}, sa, sb);
    tile(4 * c + 3, std::integral_constant<int, 3>{}, sa, sb);
  }
#pragma unroll
  for (int a = 0; a < 2; ++a) {
    const int m = m0 + 16 * a + li;
    if (m < s.end) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
        store_quad<O>(g, static_cast<const O*>(g.C), static_cast<O*>(g.D), m, n0 + 16 * b + 4 * lg, acc[a][b]);
    }
  }
}

template <typename O>
static int run_mx(MxArgs x, hipStream_t s) {
  GroupedArgs& g = x.g;
  g.tiles_n = (g.N + 63) / 64;
  const int64_t tiles = (g.rows / 64 + std::min<int64_t>(g.groups + 2, g.rows)) * g.tiles_n;
  TRNBLAS_CHECK_ARG(tiles < ((int64_t)1 << 31) - 8, "%s: too many tiles", kMxGemm);
  const unsigned grid = (unsigned)((tiles + kNumXcd - 1) / kNumXcd * kNumXcd);
  hipLaunchKernelGGL(mx_any_kernel<O>, dim3(grid), dim3(256), 0, s, x);
  return check_launch(kMxGemm);
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

extern "C" int trnblas_hip_mx_gemm(int out_dtype, int64_t groups, int64_t rows, int64_t N, int64_t K, double alpha,
                                   const void* A, const void* A_scales, const void* B, const void* B_scales,
                                   const void* offsets, int offsets64, double beta, const void* C, int64_t ldc, void* D,
                                   int64_t ldd, void* stream) {
  TRNBLAS_CHECK_ARG(out_dtype == TRNBLAS_F32 || out_dtype == TRNBLAS_BF16 || out_dtype == TRNBLAS_F16, "%s: bad dtype %d", kMxGemm, out_dtype);
  TRNBLAS_CHECK_ARG(groups >= 0 && groups < (1 << 24) && rows >= 0 && rows < INT32_MAX - 1024 && N >= 0 &&
                        N < INT32_MAX - 1024 && K >= 0 && K < INT32_MAX - 1024,
                    "%s: bad sizes (groups %lld, rows %lld, N %lld, K %lld)", kMxGemm, (long long)groups, (long long)rows,
                    (long long)N, (long long)K);
  TRNBLAS_CHECK_ARG(offsets != nullptr ? (uintptr_t)offsets % (offsets64 ? 8 : 4) == 0 : groups == 1,
                    "%s: offsets missing or misaligned", kMxGemm);
  TRNBLAS_CHECK_ARG(beta == 0.0 || C != nullptr, "%s: beta != 0 without C", kMxGemm);
  TRNBLAS_CHECK_ARG(ldd >= N && (beta == 0.0 || ldc >= N), "%s: bad leading dimension", kMxGemm);
  if (rows == 0 || N == 0) return TRNBLAS_OK;
  TRNBLAS_CHECK_ARG(D != nullptr && (K == 0 || groups == 0 || (A && A_scales && B && B_scales)), "%s: null operand", kMxGemm);
  for (const void* p : {A, A_scales, B, B_scales})
    TRNBLAS_CHECK_ARG((uintptr_t)p % 16 == 0, "%s: codes and scales must be 16-byte aligned", kMxGemm);
  MxArgs x{};
  GroupedArgs& g = x.g;
  g.A = A, g.B = B;
  g.lda = g.ldb = (K + 31) / 32 * 16;
  g.sB = N * g.ldb;
  x.sa = static_cast<const uint8_t*>(A_scales);
  x.sb = static_cast<const uint8_t*>(B_scales);
  x.chunks = (int)((K + 511) / 512);
  x.sb_step = (N + 15) / 16 * x.chunks * kChunk;
  g.offsets = offsets;
  g.offsets64 = offsets64 != 0;
  g.groups = (int)groups, g.rows = (int)rows, g.N = (int)N, g.K = (int)K;
  g.alpha = (float)alpha, g.beta = (float)beta;
  g.C = beta != 0.0 ? C : nullptr, g.ldc = ldc;
  g.D = D, g.ldd = ldd;
  const int eo = out_dtype == TRNBLAS_F32 ? 4 : 2;
  g.vec4 = (uintptr_t)D % (4 * eo) == 0 && ldd % 4 == 0 && (g.C == nullptr || ((uintptr_t)C % (4 * eo) == 0 && ldc % 4 == 0));
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (out_dtype) {
    case TRNBLAS_F32: return run_mx<float>(x, s);
    case TRNBLAS_BF16: return run_mx<__bf16>(x, s);
    default: return run_mx<_Float16>(x, s);
  }
}
