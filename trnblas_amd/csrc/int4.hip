// 4-bit integer weights with scales of groups (int4.hpp): quantisation, its reverse, and
// the C entry of their products.
#include <algorithm>

#include "int4.hpp"

namespace trnblas {

static const char* const kQuantize = "trnblas_hip_int4_quantize";
static const char* const kDequantize = "trnblas_hip_int4_dequantize";
static const char* const kGemm = kInt4Gemm;

struct Int4QuantArgs {
  const void* X;
  int64_t sr, sk, sx;  // strides of rows, K and batch, in elements
  int R, K, chunks, steps;
  uint8_t* codes;
  uint16_t* scales;
  uint8_t* zeros;  // or null: symmetric
  int scale_f16;
  int vec;  // K-contiguous, every row starts on 16 bytes
};

// What a group's values become. A scale that is not finite (an infinity or a NaN among the
// values, or a range past the scale's type) is a NaN, and with it the whole group.
struct Int4Group {
  uint16_t bits;
  float s, z;
};

__device__ __forceinline__ uint16_t int4_scale_bits(float s, int f16) {
  return f16 ? __builtin_bit_cast(uint16_t, (_Float16)s) : __builtin_bit_cast(uint16_t, (__bf16)s);
}

// lo, hi: the least and largest value, and zero; top: bits of the largest magnitude.
template <bool ZEROS>
__device__ __forceinline__ Int4Group int4_group(float lo, float hi, uint32_t top, int f16) {
  Int4Group q;
  q.bits = int4_scale_bits(ZEROS ? (hi - lo) / 15.0f : __builtin_bit_cast(float, top) / 7.0f, f16);
  q.s = int4_scale(q.bits, f16);
  if (top >= 0x7f800000u || !(__builtin_fabsf(q.s) <= 3.4028235e38f)) {
    q.bits = int4_scale_bits(__builtin_nanf(""), f16);
    q.s = 0.0f;  // codes of zero
  }
  q.z = ZEROS ? (q.s > 0.0f ? fminf(fmaxf(rintf(-lo / q.s), 0.0f), 15.0f) : 0.0f) : 8.0f;
  return q;
}

// Eight values as nibbles q - 8. round(x / s) is taken from the product with the reciprocal of s: |x / s| < 23 (15
// times what rounding the scale takes away, a third of it at most), so that the product is within 2^-18 of
// the quotient, and adding 1.5 * 2^23 rounds it to a whole number, whose low bits are the code's.
// Values of 16 bits: a quotient of two numbers of 11 bits is halfway between two whole numbers or 2^-13 from that at
// least. In steps of 2^-13 or 2^-14, where 1024 is added, the product of a quotient halfway is exactly that, and another's
// on its side. Values of 32 bits: where the product is within 2^-16 of halfway, they are divided, as where the scale has
// no reciprocal.
template <bool NARROW, bool ZEROS>
__device__ __forceinline__ uint32_t int4_dword(const float (&x)[8], const Int4Group& q) {
  constexpr float kWhole = 0x1.8p23f;
  const float inverse = __builtin_amdgcn_rcpf(q.s), lo = kWhole - q.z, hi = kWhole + 15.0f - q.z;
  float v[8], off = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if constexpr (NARROW) {
      v[e] = __builtin_fmaf(x[e], inverse, 1024.0f) + (kWhole - 1024.0f);
    } else {
      v[e] = __builtin_fmaf(x[e], inverse, kWhole);
      off = fmaxf(off, __builtin_fabsf(__builtin_fmaf(x[e], inverse, kWhole - v[e])));
    }
  }
  if (off > 0.5f - 0x1p-16f || q.s < 0x1p-120f || q.s > 0x1p120f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = kWhole + (q.s > 0.0f ? rintf(x[e] / q.s) : 0.0f);
  }
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int e = 2 * (i & 3) + i / 4;  // the nibbles from the lowest
    const float c = __builtin_amdgcn_fmed3f(v[e], lo, hi) + (ZEROS ? q.z - 8.0f : 0.0f);
    w = __builtin_amdgcn_alignbit(__builtin_bit_cast(uint32_t, c), w, 4);
  }
  return w;
}

// The least, the largest and the largest magnitude of values: of 16 bits in pairs, as whole numbers in their order.
template <typename T, bool ZEROS>
struct Int4Range;

template <bool ZEROS>
struct Int4Range<float, ZEROS> {
  float lo = 0.0f, hi = 0.0f;
  uint32_t top = 0;
  __device__ __forceinline__ void take(const float (&x)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (ZEROS) lo = fminf(lo, x[e]), hi = fmaxf(hi, x[e]);
      top = max(top, __builtin_bit_cast(uint32_t, x[e]) & 0x7fffffffu);
    }
  }
  __device__ __forceinline__ void join(int lanes) {
    if constexpr (ZEROS) lo = fminf(lo, __shfl_xor(lo, lanes)), hi = fmaxf(hi, __shfl_xor(hi, lanes));
    top = max(top, (uint32_t)__shfl_xor((int)top, lanes));
  }
  __device__ __forceinline__ Int4Group group(int f16) const { return int4_group<ZEROS>(lo, hi, top, f16); }
};

template <typename T, bool ZEROS>
struct Int4Range {
  using i16x2 = __attribute__((ext_vector_type(2))) int16_t;
  i16x2 lo = 0, hi = 0;  // symmetric: hi alone, of magnitudes
  __device__ __forceinline__ void take(const T (&x)[8]) {
    i16x2 v[4];
    __builtin_memcpy(v, x, 16);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (ZEROS) {
        v[e] ^= (v[e] >> 15) & 0x7fff;
        lo = __builtin_elementwise_min(lo, v[e]);
      } else {
        v[e] &= 0x7fff;
      }
      hi = __builtin_elementwise_max(hi, v[e]);
    }
  }
  __device__ __forceinline__ void join(int lanes) {
    if constexpr (ZEROS) lo = __builtin_elementwise_min(lo, __builtin_bit_cast(i16x2, __shfl_xor(__builtin_bit_cast(int, lo), lanes)));
    hi = __builtin_elementwise_max(hi, __builtin_bit_cast(i16x2, __shfl_xor(__builtin_bit_cast(int, hi), lanes)));
  }
  __device__ __forceinline__ Int4Group group(int f16) const {
    const int16_t l = min(lo.x, lo.y), h = max(hi.x, hi.y);
    const float least = (float)__builtin_bit_cast(T, (int16_t)(l ^ (l >> 15 & 0x7fff))), most = (float)__builtin_bit_cast(T, h);
    // (a NaN's bits are past an infinity's on its side)
    const uint32_t top = max(__builtin_bit_cast(uint32_t, least) & 0x7fffffffu, __builtin_bit_cast(uint32_t, most));
    return int4_group<ZEROS>(least, most, top, f16);
  }
};

// 16 rows x 128 values per wave, four waves per workgroup: lane 16 p + r takes row r, k = 32 h + 8 p .. + 7
// for h = 0 .. 3, which are its 16 bytes of codes; a group's values lie in the four lanes of a row.
// 8192 x 8192 bf16 in groups of 128: 34 us, 168 MB at 4.9 TB/s. With a division for each value, extremes as floats and a scale
// for each h it was 63 us, bound by the vector unit. A transposed 487 x 1283 fp32: 5.5 us, 6.8 with loads behind branches.
template <typename T, int STEPS, bool ZEROS>
__global__ __launch_bounds__(256) void int4_quantize_kernel(Int4QuantArgs g) {
  const int lane = threadIdx.x & 63, r = lane & 15, p = lane >> 4;
  const int blocks = (g.R + 15) / 16;
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (item >= (int64_t)blocks * g.chunks) return;
  const int block = (int)(item / g.chunks), chunk = (int)(item - (int64_t)block * g.chunks);
  const int row = 16 * block + r;
  T v[4][8];
  if (g.vec && (chunk + 1) * 128 <= g.K && row < g.R) {
    const T* x = static_cast<const T*>(g.X) + blockIdx.y * g.sx + row * g.sr + 128 * chunk + 8 * p;
#pragma unroll
    for (int h = 0; h < 4; ++h)
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
        const i32x4 w = *reinterpret_cast<const i32x4*>(x + 32 * h + 16 / sizeof(T) * i);
        __builtin_memcpy(&v[h][16 / sizeof(T) * i], &w, 16);
      }
  } else {
    // values past the matrix: its last one instead, then zero, so that no load waits for a branch
    const T* x = static_cast<const T*>(g.X) + blockIdx.y * g.sx + (row < g.R ? row : g.R - 1) * g.sr;
#pragma unroll
    for (int h = 0; h < 4; ++h)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[h][e] = x[min(128 * chunk + 32 * h + 8 * p + e, g.K - 1) * g.sk];
#pragma unroll
    for (int h = 0; h < 4; ++h)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (row >= g.R || 128 * chunk + 32 * h + 8 * p + e >= g.K) v[h][e] = (T)0.0f;
  }
  const int64_t at = ((blockIdx.y * (int64_t)blocks + block) * g.chunks + chunk);
  i32x4 w;
#pragma unroll
  for (int h = 0; h < 4; h += STEPS) {
    Int4Range<T, ZEROS> range;
#pragma unroll
    for (int i = 0; i < STEPS; ++i) range.take(v[h + i]);
    range.join(16), range.join(32);
    const Int4Group q = range.group(g.scale_f16);
#pragma unroll
    for (int i = h; i < h + STEPS; ++i) {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = (float)v[i][e];
      w[i] = (int)int4_dword<sizeof(T) == 2, ZEROS>(x, q);
      const int left = row < g.R ? g.K - (128 * chunk + 32 * i + 8 * p) : 0;
      if (left < 8) {
        uint32_t keep = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) keep |= (e < left ? 15u : 0u) << 4 * (e / 2 + 4 * (e & 1));
        w[i] &= (int)keep;
      }
    }
    if (p == 0) {
      const int64_t to = (at * 16 + r) * (4 / STEPS) + h / STEPS;
      const bool inside = row < g.R && 128 * chunk + 32 * h < g.K;
      g.scales[to] = inside ? q.bits : 0;
      if constexpr (ZEROS) g.zeros[to] = inside ? (uint8_t)q.z : 0;
    }
  }
  *reinterpret_cast<i32x4*>(g.codes + at * kInt4Chunk + 16 * lane) = w;
}

template <typename T, int STEPS>
static void launch_quantize(const Int4QuantArgs& g, dim3 grid, hipStream_t s) {
  if (g.zeros != nullptr)
    hipLaunchKernelGGL((int4_quantize_kernel<T, STEPS, true>), grid, dim3(256), 0, s, g);
  else
    hipLaunchKernelGGL((int4_quantize_kernel<T, STEPS, false>), grid, dim3(256), 0, s, g);
}

template <typename T>
static void launch_quantize(const Int4QuantArgs& g, dim3 grid, hipStream_t s) {
  switch (g.steps) {
    case 1: return launch_quantize<T, 1>(g, grid, s);
    case 2: return launch_quantize<T, 2>(g, grid, s);
    default: return launch_quantize<T, 4>(g, grid, s);
  }
}

struct Int4DequantArgs {
  const uint8_t* codes;
  const uint16_t* scales;
  const uint8_t* zeros;
  int R, K, chunks, steps, scale_f16;
  void* D;
  int64_t ldd, sD;
  int vec;
};

template <typename T>
__global__ __launch_bounds__(256) void int4_dequantize_kernel(Int4DequantArgs g) {
  const int lane = threadIdx.x & 63, r = lane & 15, p = lane >> 4;
  const int blocks = (g.R + 15) / 16;
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (item >= (int64_t)blocks * g.chunks) return;
  const int block = (int)(item / g.chunks), chunk = (int)(item - (int64_t)block * g.chunks);
  const int row = 16 * block + r;
  const i32x4 w =
      *reinterpret_cast<const i32x4*>(g.codes + ((blockIdx.y * (int64_t)blocks + block) * g.chunks + chunk) * kInt4Chunk + 16 * lane);
  T* D = static_cast<T*>(g.D) + blockIdx.y * g.sD + row * g.ldd;
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    const int64_t at = (((blockIdx.y * (int64_t)blocks + block) * g.chunks + chunk) * 16 + r) * (4 / g.steps) + h / g.steps;
    const float s = int4_scale(g.scales[at], g.scale_f16), z = g.zeros ? (float)g.zeros[at] : 8.0f;
    const int k = 128 * chunk + 32 * h + 8 * p, left = row < g.R ? g.K - k : 0;
    union {
      T e[8];
      i32x4 v[sizeof(T) / 2];
    } o;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t c = ((uint32_t)w[h] >> 4 * (e / 2 + 4 * (e & 1)) & 15u) ^ 8u;
      o.e[e] = (T)(((float)c - z) * s);
    }
    if (g.vec && left >= 8) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<i32x4*>(D + k)[i] = o.v[i];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < left) D[k + e] = o.e[e];
    }
  }
}

// Rows as the products' kernels read them: `kp` values each, zeros past K, of bf16 or fp16; fp32 as three bf16
// pieces whose sum it is (each takes the value's next eight bits, by truncation; an infinity or a NaN
// stands in the first alone).
struct Int4RowsArgs {
  const void* A;
  int64_t sr, sk;
  int64_t rows;
  int K, kp;
  void* D;
  int64_t step;  // from one piece to the next
};

template <typename T>
__global__ __launch_bounds__(256) void int4_rows_of_kernel(Int4RowsArgs g) {
  const int per = g.kp / 8;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t r = i / per;
  if (r >= g.rows) return;
  const int k = 8 * (int)(i - r * per);
  const T* a = static_cast<const T*>(g.A) + r * g.sr + k * g.sk;
  T v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = k + e < g.K ? a[e * g.sk] : (T)0.0f;
  uint16_t* d = static_cast<uint16_t*>(g.D) + r * g.kp + k;
  if constexpr (sizeof(T) == 2) {
    *reinterpret_cast<i32x4*>(d) = *reinterpret_cast<const i32x4*>(v);
  } else {
    uint16_t o[3][8] __attribute__((aligned(16)));
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t bits = __builtin_bit_cast(uint32_t, v[e]);
      const bool finite = (bits & 0x7f800000u) != 0x7f800000u;
      const float mid = v[e] - __builtin_bit_cast(float, bits & 0xffff0000u);
      const uint32_t m = __builtin_bit_cast(uint32_t, mid);
      const float low = mid - __builtin_bit_cast(float, m & 0xffff0000u);
      // a NaN whose payload lies in the low half stays one
      o[0][e] = (uint16_t)(bits >> 16 | (!finite && (bits & 0x007fffffu) ? 0x40u : 0u));
      o[1][e] = finite ? (uint16_t)(m >> 16) : 0;
      o[2][e] = finite ? (uint16_t)(__builtin_bit_cast(uint32_t, low) >> 16) : 0;
    }
#pragma unroll
    for (int p = 0; p < 3; ++p) *reinterpret_cast<i32x4*>(d + p * g.step) = *reinterpret_cast<const i32x4*>(o[p]);
  }
}

// The parts' sums of int4_tile_kernel to results, four columns per thread, in the order of the parts.
template <bool GATED>
__global__ __launch_bounds__(256) void int4_join_kernel(GroupedArgs g, Int4Args q) {
  const int quads = (g.N + 3) / 4;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, m = i / quads;
  if (m >= g.rows) return;
  const int n = 4 * (int)(i - m * quads);
  const int64_t step = g.rows * q.ldp;
  const float* p = q.partial + m * q.ldp + n;
  f32x4 v = *reinterpret_cast<const f32x4*>(p), w = v;
  if constexpr (GATED) w = *reinterpret_cast<const f32x4*>(p + g.N);
  for (int part = 1; part < q.splits; ++part) {
    p += step;
    v += *reinterpret_cast<const f32x4*>(p);
    if constexpr (GATED) w += *reinterpret_cast<const f32x4*>(p + g.N);
  }
  int4_store<GATED>(g, m, n, v, w);
}

static int check_int4(const char* what, int64_t R, int64_t K, int64_t group, int scale_dtype, int64_t batch) {
  TRNBLAS_CHECK_ARG(R >= 0 && R < INT32_MAX - 1024 && K >= 0 && K < INT32_MAX - 1024 && batch >= 0 && batch < 65536,
                    "%s: bad sizes (rows %lld, K %lld, batch %lld)", what, (long long)R, (long long)K, (long long)batch);
  TRNBLAS_CHECK_ARG(group == 32 || group == 64 || group == 128, "%s: bad group %lld (32, 64 or 128)", what, (long long)group);
  TRNBLAS_CHECK_ARG(scale_dtype == TRNBLAS_BF16 || scale_dtype == TRNBLAS_F16, "%s: bad scale dtype %d", what, scale_dtype);
  return TRNBLAS_OK;
}

static int check_int4_buffers(const char* what, const void* codes, const void* scales, const void* zeros) {
  TRNBLAS_CHECK_ARG((uintptr_t)codes % 16 == 0 && (uintptr_t)scales % 16 == 0 && (uintptr_t)zeros % 16 == 0,
                    "%s: codes, scales and zeros must be 16-byte aligned", what);
  return TRNBLAS_OK;
}

// Four chunks per workgroup; the matrix is the grid's y.
static int int4_chunk_grid(const char* what, int64_t R, int64_t K, int64_t batch, dim3* grid) {
  const int64_t n = ((R + 15) / 16 * ((K + 127) / 128) + 3) / 4;
  TRNBLAS_CHECK_ARG(n < (int64_t)1 << 31, "%s: matrix too large (%lld x %lld)", what, (long long)R, (long long)K);
  *grid = dim3((unsigned)n, (unsigned)batch);
  return TRNBLAS_OK;
}

}  // namespace trnblas

using namespace trnblas;

extern "C" int trnblas_hip_int4_quantize(int dtype, int scale_dtype, int64_t R, int64_t K, int64_t group, const void* X, int64_t sr,
                                         int64_t sk, int64_t sx, void* codes, void* scales, void* zeros, int64_t batch,
                                         void* stream) {
  TRNBLAS_CHECK_ARG(dtype == TRNBLAS_F32 || dtype == TRNBLAS_BF16 || dtype == TRNBLAS_F16, "%s: bad dtype %d", kQuantize, dtype);
  if (int rc = check_int4(kQuantize, R, K, group, scale_dtype, batch)) return rc;
  TRNBLAS_CHECK_ARG(sr >= 0 && sk >= 0 && sx >= 0, "%s: negative stride", kQuantize);
  if (R == 0 || K == 0 || batch == 0) return TRNBLAS_OK;
  TRNBLAS_CHECK_ARG(X != nullptr && codes != nullptr && scales != nullptr, "%s: null operand", kQuantize);
  if (int rc = check_int4_buffers(kQuantize, codes, scales, zeros)) return rc;
  dim3 grid;
  if (int rc = int4_chunk_grid(kQuantize, R, K, batch, &grid)) return rc;
  const int es = dtype == TRNBLAS_F32 ? 4 : 2;
  Int4QuantArgs g{};
  g.X = X, g.sr = sr, g.sk = sk, g.sx = sx;
  g.R = (int)R, g.K = (int)K, g.chunks = (int)((K + 127) / 128), g.steps = (int)(group / 32);
  g.codes = static_cast<uint8_t*>(codes), g.scales = static_cast<uint16_t*>(scales), g.zeros = static_cast<uint8_t*>(zeros);
  g.scale_f16 = scale_dtype == TRNBLAS_F16;
  g.vec = sk == 1 && (uintptr_t)X % 16 == 0 && sr * es % 16 == 0 && sx * es % 16 == 0;
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case TRNBLAS_F32: launch_quantize<float>(g, grid, s); break;
    case TRNBLAS_BF16: launch_quantize<__bf16>(g, grid, s); break;
    default: launch_quantize<_Float16>(g, grid, s); break;
  }
  return check_launch(kQuantize);
}

extern "C" int trnblas_hip_int4_dequantize(int dtype, int scale_dtype, int64_t R, int64_t K, int64_t group, const void* codes,
                                           const void* scales, const void* zeros, void* D, int64_t ldd, int64_t strideD,
                                           int64_t batch, void* stream) {
  TRNBLAS_CHECK_ARG(dtype == TRNBLAS_F32 || dtype == TRNBLAS_BF16 || dtype == TRNBLAS_F16, "%s: bad dtype %d", kDequantize, dtype);
  if (int rc = check_int4(kDequantize, R, K, group, scale_dtype, batch)) return rc;
  TRNBLAS_CHECK_ARG(ldd >= K && strideD >= 0, "%s: bad leading dimension", kDequantize);
  if (R == 0 || K == 0 || batch == 0) return TRNBLAS_OK;
  TRNBLAS_CHECK_ARG(D != nullptr && codes != nullptr && scales != nullptr, "%s: null operand", kDequantize);
  if (int rc = check_int4_buffers(kDequantize, codes, scales, zeros)) return rc;
  dim3 grid;
  if (int rc = int4_chunk_grid(kDequantize, R, K, batch, &grid)) return rc;
  const int es = dtype == TRNBLAS_F32 ? 4 : 2;
  Int4DequantArgs g{};
  g.codes = static_cast<const uint8_t*>(codes), g.scales = static_cast<const uint16_t*>(scales);
  g.zeros = static_cast<const uint8_t*>(zeros);
  g.R = (int)R, g.K = (int)K, g.chunks = (int)((K + 127) / 128), g.steps = (int)(group / 32);
  g.scale_f16 = scale_dtype == TRNBLAS_F16;
  g.D = D, g.ldd = ldd, g.sD = strideD;
  g.vec = (uintptr_t)D % 16 == 0 && ldd * es % 16 == 0 && strideD * es % 16 == 0;
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case TRNBLAS_F32: hipLaunchKernelGGL(int4_dequantize_kernel<float>, grid, dim3(256), 0, s, g); break;
    case TRNBLAS_BF16: hipLaunchKernelGGL(int4_dequantize_kernel<__bf16>, grid, dim3(256), 0, s, g); break;
    default: hipLaunchKernelGGL(int4_dequantize_kernel<_Float16>, grid, dim3(256), 0, s, g); break;
  }
  return check_launch(kDequantize);
}

constexpr int64_t kInt4Far = (int64_t)1 << 22;  // elements between rows that are read in place

static int64_t up128(int64_t k) { return (k + 127) / 128 * 128; }

// Rows as the kernels read them, and the parts' sums behind them.
static size_t rows_bytes(int dtype, int64_t rows, int64_t K) { return (size_t)(rows * up128(K)) * 2 * (dtype == TRNBLAS_F32 ? 3 : 1); }
static int64_t partial_ld(bool gated, int64_t N) { return ((gated ? 2 * N : N) + 3) / 4 * 4; }

extern "C" size_t trnblas_hip_int4_gemm_workspace(int dtype, int gated, int64_t groups, int64_t rows, int64_t N, int64_t K,
                                                  int64_t group) {
  if (rows <= 0 || K <= 0 || N <= 0 || groups <= 0) return 0;
  const Int4Choice c = choose_int4(rows, groups, N, K, (int)(group / 32), dtype == TRNBLAS_F32 ? 3 : 1, gated != 0);
  return rows_bytes(dtype, rows, K) + (c.splits > 1 ? (size_t)c.splits * rows * partial_ld(gated != 0, N) * 4 : 0);
}

extern "C" int trnblas_hip_int4_gemm(int dtype, int out_dtype, int gated, int act, int64_t groups, int64_t rows, int64_t N, int64_t K,
                                     int64_t group, double alpha, const void* A, int64_t sr, int64_t sk, const void* codes,
                                     const void* scales, const void* zeros, int scale_dtype, const void* offsets, int offsets64,
                                     double beta, const void* C, int64_t ldc, void* D, int64_t ldd, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  TRNBLAS_CHECK_ARG(dtype == TRNBLAS_F32 || dtype == TRNBLAS_BF16 || dtype == TRNBLAS_F16, "%s: bad dtype %d", kGemm, dtype);
  TRNBLAS_CHECK_ARG(out_dtype == TRNBLAS_F32 || out_dtype == TRNBLAS_BF16 || out_dtype == TRNBLAS_F16, "%s: bad result dtype %d",
                    kGemm, out_dtype);
  TRNBLAS_CHECK_ARG(!gated || (act >= TRNBLAS_ACT_SILU && act <= TRNBLAS_ACT_SIGMOID && alpha == 1.0 && beta == 0.0),
                    "%s: bad activation %d (and alpha 1, beta 0 with one)", kGemm, act);
  if (int rc = check_int4(kGemm, N, K, group, scale_dtype, 0)) return rc;
  // K: a tile's rows, and two row blocks' codes, lie within 32-bit offsets
  TRNBLAS_CHECK_ARG(groups >= 0 && groups < (1 << 24) && rows >= 0 && rows < INT32_MAX - 1024 && N < (INT32_MAX >> 1) - 1024 &&
                        K <= kInt4Far,
                    "%s: bad sizes (groups %lld, rows %lld, N %lld, K %lld)", kGemm, (long long)groups, (long long)rows, (long long)N,
                    (long long)K);
  TRNBLAS_CHECK_ARG(offsets != nullptr ? (uintptr_t)offsets % (offsets64 ? 8 : 4) == 0 : groups == 1,
                    "%s: offsets missing or misaligned", kGemm);
  TRNBLAS_CHECK_ARG(beta == 0.0 || C != nullptr, "%s: beta != 0 without C", kGemm);
  TRNBLAS_CHECK_ARG(sr >= 0 && sk >= 0, "%s: negative stride", kGemm);
  TRNBLAS_CHECK_ARG(ldd >= N && (beta == 0.0 || ldc >= N), "%s: bad leading dimension", kGemm);
  if (rows == 0 || N == 0) return TRNBLAS_OK;
  const bool sums = K > 0 && groups > 0;
  TRNBLAS_CHECK_ARG(D != nullptr && (!sums || (A && codes && scales)), "%s: null operand", kGemm);
  if (int rc = check_int4_buffers(kGemm, codes, scales, zeros)) return rc;
  hipStream_t s = static_cast<hipStream_t>(stream);
  GroupedArgs g{};
  Int4Args q{};
  g.A = A, g.lda = sr;
  g.K = (int)K;
  // (rows far apart: a tile's lie within 32-bit offsets)
  Int4Choice c = choose_int4(rows, groups, N, K, (int)(group / 32), dtype == TRNBLAS_F32 ? 3 : 1, gated != 0);
  const bool lay = sums && (dtype == TRNBLAS_F32 || sk != 1 || K % 8 != 0 || (uintptr_t)A % 16 != 0 || (rows > 1 && (sr % 8 != 0 || sr > kInt4Far)));
  if (!sums || c.tile == 0) c.splits = 1;
  if (lay || c.splits > 1) {
    const size_t need = (lay ? rows_bytes(dtype, rows, K) : 0) + (c.splits > 1 ? (size_t)c.splits * rows * partial_ld(gated != 0, N) * 4 : 0);
    if (workspace == nullptr || workspace_bytes < need || (uintptr_t)workspace % 16 != 0) {
      set_error("%s: workspace of %zu bytes, 16-byte aligned, needed (got %zu)", kGemm, need, workspace_bytes);
      return TRNBLAS_E_WORKSPACE;
    }
  }
  if (lay) {
    Int4RowsArgs r{A, sr, sk, rows, (int)K, (int)up128(K), workspace, rows * up128(K)};
    const int64_t grid = (rows * (r.kp / 8) + 255) / 256;
    TRNBLAS_CHECK_ARG(grid < (int64_t)1 << 31, "%s: too many rows", kGemm);
    switch (dtype) {
      case TRNBLAS_F32: hipLaunchKernelGGL(int4_rows_of_kernel<float>, dim3((unsigned)grid), dim3(256), 0, s, r); break;
      case TRNBLAS_BF16: hipLaunchKernelGGL(int4_rows_of_kernel<__bf16>, dim3((unsigned)grid), dim3(256), 0, s, r); break;
      default: hipLaunchKernelGGL(int4_rows_of_kernel<_Float16>, dim3((unsigned)grid), dim3(256), 0, s, r); break;
    }
    if (int rc = check_launch(kGemm)) return rc;
    g.A = workspace, g.lda = r.kp, q.a_step = r.step;
    g.K = r.kp;
  }
  const int64_t matrix_rows = gated ? 2 * N : N;
  q.codes = static_cast<const uint8_t*>(codes), q.scales = static_cast<const uint16_t*>(scales);
  q.zeros = static_cast<const uint8_t*>(zeros);
  q.chunks = (int)((K + 127) / 128), q.steps = (int)(group / 32), q.scale_f16 = scale_dtype == TRNBLAS_F16;
  q.codes_step = (matrix_rows + 15) / 16 * q.chunks * kInt4Chunk;
  q.groups_step = (matrix_rows + 15) / 16 * q.chunks * (4 / q.steps) * 16;
  g.offsets = offsets, g.offsets64 = offsets64 != 0;
  g.groups = (int)groups, g.rows = (int)rows, g.N = (int)N;
  g.alpha = (float)alpha, g.beta = (float)beta;
  g.C = beta != 0.0 ? C : nullptr, g.ldc = ldc;
  g.D = D, g.ldd = ldd;
  g.act = act;
  g.out32 = out_dtype == TRNBLAS_F32, g.out_f16 = out_dtype == TRNBLAS_F16;
  const int eo = g.out32 ? 4 : 2;
  g.vec4 = (uintptr_t)D % (4 * eo) == 0 && ldd % 4 == 0 && (g.C == nullptr || ((uintptr_t)C % (4 * eo) == 0 && ldc % 4 == 0));
  q.splits = c.splits;
  q.ldp = partial_ld(gated != 0, N);
  q.partial = reinterpret_cast<float*>(static_cast<char*>(workspace) + (lay ? rows_bytes(dtype, rows, K) : 0));
  const int pieces = dtype == TRNBLAS_F32 ? 3 : 1;
  if (c.tile == 0)
    return dtype == TRNBLAS_F16 ? int4_gemm_run<_Float16>(g, q, 1, gated != 0, s) : int4_gemm_run<__bf16>(g, q, pieces, gated != 0, s);
  if (int rc = dtype == TRNBLAS_F16 ? int4_tile_run<_Float16>(g, q, 1, gated != 0, c.tile, s)
                                    : int4_tile_run<__bf16>(g, q, pieces, gated != 0, c.tile, s))
    return rc;
  if (q.splits > 1) {
    const int64_t grid = (rows * ((N + 3) / 4) + 255) / 256;
    TRNBLAS_CHECK_ARG(grid < (int64_t)1 << 31, "%s: too many rows", kGemm);
    if (gated)
      hipLaunchKernelGGL(int4_join_kernel<true>, dim3((unsigned)grid), dim3(256), 0, s, g, q);
    else
      hipLaunchKernelGGL(int4_join_kernel<false>, dim3((unsigned)grid), dim3(256), 0, s, g, q);
    return check_launch(kGemm);
  }
  return TRNBLAS_OK;
}

extern "C" int trnblas_hip_int4_plan(int dtype, int gated, int64_t groups, int64_t rows, int64_t N, int64_t K, int64_t group,
                                     int32_t plan[5]) {
  TRNBLAS_CHECK_ARG(plan != nullptr && dtype >= 0 && dtype <= 2 && groups >= 1 && rows >= 1 && N >= 1 && K >= 1 &&
                        (group == 32 || group == 64 || group == 128),
                    "trnblas_hip_int4_plan: bad arguments");
  const Int4Choice c = choose_int4(rows, groups, N, K, (int)(group / 32), dtype == TRNBLAS_F32 ? 3 : 1, gated != 0);
  const bool few = c.tile == 0;
  plan[0] = c.tile, plan[1] = c.splits, plan[2] = few ? c.mf : 0, plan[3] = few ? c.nf : 0, plan[4] = few ? c.ks : 0;
  return TRNBLAS_OK;
}
