// 4-bit integer weights with scales of groups along K: their layout and the step
// from codes to matrix-instruction operands.
//
// A weight is (q - z) s: q of 4 bits, a scale s (bf16 or fp16) and a zero point z (a byte; 8
// where a matrix has none) for each 32, 64 or 128 values along K of a row. A matrix of R rows by K:
//  * codes: 1 KiB per 16 rows x 128 values, chunks along K back to back. The 16 bytes at
//    16 (16 p + r), p = 0 .. 3, are of row r; dword h of them holds k = 32 h + 8 p + e, e = 0 .. 7: what lane 16
//    p + r of a 16 x 16 x 32 matrix instruction takes in step h. Nibble e / 2 of it (e even) or 4 + e / 2
//    (odd) is q - 8 as a signed number. Values outside the matrix are zero.
//  * scales, zero points: per 16 rows x 128 values the rows' one after the other, 4, 2 or 1 each, so that a
//    lane loads those of its row and chunk at once. Those outside the matrix are zero.
#pragma once

#include <algorithm>

#include "gate.hpp"
#include "gemm.hpp"
#include "grouped.hpp"
#include "grouped_plan.hpp"
#include "ring.hpp"

namespace trnblas {

struct Int4Args {
  const uint8_t* codes;
  const uint16_t* scales;
  const uint8_t* zeros;  // or null
  int chunks;            // along K
  int steps;             // of 32 values per group: 1, 2 or 4
  int scale_f16;
  int64_t codes_step, groups_step;  // from one matrix of a stack to the next: bytes of codes; scales
  int64_t a_step;                   // elements from one piece of A to the next (fp32)
  int splits;                       // parts of K (int4_tile_kernel)
  float* partial;                   // their sums, rows of ldp values
  int64_t ldp;
};

constexpr int kInt4Chunk = 1024;  // bytes of codes

// A buffer at a (uniform) address; reads at or past kRecords bytes from it give zeros with no memory access.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_at(const void* p) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(uniform(static_cast<const char*>(p))), 0, kRecords, 0x00020000);
}

__device__ __forceinline__ float int4_scale(uint16_t bits, int f16) {
  return f16 ? (float)__builtin_bit_cast(_Float16, bits) : __builtin_bit_cast(float, (uint32_t)bits << 16);
}

// The eight values of a dword of codes as an MFMA operand, exact: fp16 q - z by setting them
// into the mantissa of 1024 (1024 + q - (1024 + z)); bf16 (q - z) / 16 by the hardware's
// conversion of signed nibbles to sixteenths. zc: fp16 -(1024 + z) twice, bf16 (8 - z) / 16 (ZERO only).
template <typename T, bool ZERO>
__device__ __forceinline__ i32x4 int4_values(uint32_t w, uint32_t zc) {
  i32x4 v;
  if constexpr (std::is_same_v<T, _Float16>) {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v[i] = __builtin_bit_cast(
          int, __builtin_bit_cast(f16x2, ((w >> 4 * i) & 0x000f000fu) ^ 0x64086408u) + __builtin_bit_cast(f16x2, zc));
  } else {
    // by asm: the compiler shifts bytes down that the instruction can pick, and waits between each conversion
    // and what takes it (17 instructions and 8 waits for eight values; 13)
    float f[8];
    asm("v_lshrrev_b32 %8, 4, %9\n\t"
        "v_cvt_off_f32_i4 %0, %9\n\t"
        "v_cvt_off_f32_i4_sdwa %1, %9 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_2\n\t"
        "v_cvt_off_f32_i4_sdwa %4, %9 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_1\n\t"
        "v_cvt_off_f32_i4_sdwa %5, %9 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_3\n\t"
        "v_cvt_off_f32_i4 %2, %8\n\t"
        "v_cvt_off_f32_i4_sdwa %3, %8 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_2\n\t"
        "v_cvt_off_f32_i4_sdwa %6, %8 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_1\n\t"
        "v_cvt_off_f32_i4_sdwa %7, %8 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_3"
        : "=&v"(f[0]), "=&v"(f[1]), "=&v"(f[2]), "=&v"(f[3]), "=&v"(f[4]), "=&v"(f[5]), "=&v"(f[6]), "=&v"(f[7]), "=&v"(v[0])
        : "v"(w));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (ZERO) f[2 * i] += __builtin_bit_cast(float, zc), f[2 * i + 1] += __builtin_bit_cast(float, zc);
      v[i] = (int)__builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, f[2 * i + 1]), __builtin_bit_cast(uint32_t, f[2 * i]), 0x07060302u);
    }
  }
  return v;
}

// The constant that int4_values takes for a zero point, and the factor that its sums miss.
template <typename T>
__device__ __forceinline__ uint32_t int4_zero(uint32_t z) {
  if constexpr (std::is_same_v<T, _Float16>) {
    const uint32_t h = __builtin_bit_cast(uint16_t, (_Float16)(-1024.0f - (float)z));
    return h << 16 | h;
  } else {
    return __builtin_bit_cast(uint32_t, 0.5f - 0.0625f * (float)z);
  }
}
template <typename T>
constexpr float kInt4Unit = std::is_same_v<T, _Float16> ? 1.0f : 16.0f;

// acc += (16 rows m) x (16 columns n) over 32 values of k: lane l holds column n = l % 16, rows m = 4 (l / 16) + r.
template <typename T>
__device__ __forceinline__ f32x4 int4_mma(const i32x4& m, const i32x4& n, const f32x4& acc) {
  if constexpr (std::is_same_v<T, _Float16>)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, m), __builtin_bit_cast(f16x8, n), acc, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, m), __builtin_bit_cast(bf16x8, n), acc, 0, 0, 0);
}

// D[m][n .. n + 3] of a product's sums, or of gates and ups.
template <bool GATED>
__device__ __forceinline__ void int4_store(const GroupedArgs& g, int64_t m, int n, f32x4 v, const f32x4& ups) {
  if constexpr (GATED) {
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] = gate(g.act, v[u]) * ups[u];
  }
  if (g.out32)
    store_quad<float>(g, static_cast<const float*>(g.C), static_cast<float*>(g.D), m, n, v);
  else if (g.out_f16)
    store_quad<_Float16>(g, static_cast<const _Float16*>(g.C), static_cast<_Float16*>(g.D), m, n, v);
  else
    store_quad<__bf16>(g, static_cast<const __bf16*>(g.C), static_cast<__bf16*>(g.D), m, n, v);
}

static const char* const kInt4Gemm = "trnblas_hip_int4_gemm";

// Bound on the tiles of bm rows (see ragged_tile), in whole rounds of the XCDs.
static int int4_grid(const GroupedArgs& g, int bm, unsigned* grid) {
  const int64_t tiles = (g.rows / bm + std::min<int64_t>(g.groups + 2, g.rows)) * g.tiles_n;
  TRNBLAS_CHECK_ARG(tiles < ((int64_t)1 << 31) - 4096, "%s: too many tiles", kInt4Gemm);
  *grid = (unsigned)((tiles + kNumXcd - 1) / kNumXcd * kNumXcd);
  return TRNBLAS_OK;
}

// The launches for operands as the kernels read them (rows 16-byte aligned, K a multiple of 8): T
// fp16 or bf16, `pieces` 1, or 3 bf16 pieces of fp32 rows. int4_f16.hip, int4_bf16.hip.
template <typename T>
int int4_gemm_run(const GroupedArgs& g, const Int4Args& q, int pieces, bool gated, hipStream_t s);
// The tile kernel; `rows` of a tile 64 or 128. int4_tile_f16.hip, int4_tile_bf16.hip.
template <typename T>
int int4_tile_run(const GroupedArgs& g, const Int4Args& q, int pieces, bool gated, int rows, hipStream_t s);

}  // namespace trnblas
