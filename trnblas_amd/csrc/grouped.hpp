// What the grouped products share: the argument block, the map from
// workgroups to tiles of ragged groups, LDS panels with their fragment reads,
// and the epilogue.
#pragma once

#include <type_traits>

#include "common.hpp"

namespace trnblas {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

struct GroupedArgs {
  const void* A;
  int64_t lda;
  const void* B;
  int64_t ldb, sB;
  const void* C;
  int64_t ldc, sC;
  void* D;
  int64_t ldd, sD;
  const void* offsets;  // device int32 or int64 [groups + 1], or null: one group of all rows
  int offsets64;
  int groups, rows;  // rows of the ragged operand(s)
  int M, N, K;       // ragged rows: M unused; ragged k: K unused
  int tiles_m, tiles_n;
  float alpha, beta;
  int out32;  // D and C are fp32 whatever the operands are
  int vec4;   // D and C take 4-element accesses (aligned, ld % 4 == 0)
};

// Boundaries of the row segments: 0, offsets[0 .. groups], rows. Segment 0
// (rows before the first group) and segment groups + 1 (rows after the last)
// belong to no group; segment i is group i - 1. Every boundary is clamped to
// [0, rows], so no offset can lead outside the operands.
__device__ __forceinline__ int boundary(const GroupedArgs& g, int i) {
  if (i <= 0) return 0;
  if (i > g.groups + 1) return g.rows;
  if (g.offsets == nullptr) return i == 1 ? 0 : g.rows;
  if (g.offsets64) {
    const int64_t o = static_cast<const int64_t*>(g.offsets)[i - 1];
    return o < 0 ? 0 : o > g.rows ? g.rows : (int)o;
  }
  const int o = static_cast<const int32_t*>(g.offsets)[i - 1];
  return min(max(o, 0), g.rows);
}

struct Segment {
  int group;       // -1 or groups: rows of no group
  int start, end;  // its rows
  int row;         // first row of this tile
  int tn;          // column tile
};

// Inclusive sum over the lanes of the wave.
__device__ __forceinline__ int wave_scan(int v, int lane) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int o = __shfl_up(v, d);
    if (lane >= d) v += o;
  }
  return v;
}

// Tile of workgroup `bid` among ragged rows cut into tiles of BM rows per
// segment and g.tiles_n column tiles; false when there is none left. The
// number of tiles is known on the device only: the grid is a bound, and each
// wave counts the tiles of 64 segments at a time (one load and a scan).
// Workgroups go to the XCDs round-robin: each XCD walks one contiguous range
// of the tiles that are really there, in bands of `band` row tiles by columns.
template <int BM>
__device__ __forceinline__ bool ragged_tile(const GroupedArgs& g, int bid, int band, Segment& s) {
  const int lane = threadIdx.x & 63;
  const int nseg = g.groups + 2;
  int total = 0, st = 0, en = 0, incl = 0;
  for (int base = 0; base < nseg; base += 64) {
    const int i = base + lane;
    st = boundary(g, i);
    en = max(boundary(g, i + 1), st);
    incl = wave_scan(i < nseg ? (en - st + BM - 1) / BM : 0, lane);
    total += __builtin_amdgcn_readlane(incl, 63);
  }
  const int ntile = total * g.tiles_n;
  const int q = ntile / kNumXcd, r = ntile % kNumXcd;
  const int x = bid % kNumXcd, i = bid / kNumXcd;
  if (i >= q + (x < r)) return false;
  const int t = x * q + min(x, r) + i;
  int tm, tn;
  grouped_tile(t, total, g.tiles_n, band, tm, tn);
  s.tn = tn;
  if (nseg > 64) {  // walk the segments again up to the one that holds tm
    int before = 0;
    for (int base = 0;; base += 64) {
      const int j = base + lane;
      st = boundary(g, j);
      en = max(boundary(g, j + 1), st);
      incl = wave_scan(j < nseg ? (en - st + BM - 1) / BM : 0, lane);
      const int sum = __builtin_amdgcn_readlane(incl, 63);
      if (tm < before + sum || base + 64 >= nseg) {
        tm -= before;
        s.group = base - 1;
        break;
      }
      before += sum;
    }
  } else {
    s.group = -1;
  }
  const uint64_t past = __ballot(incl > tm);
  if (past == 0) return false;
  const int l = __builtin_ctzll(past);
  s.group += l;
  s.start = __builtin_amdgcn_readlane(st, l);
  s.end = __builtin_amdgcn_readlane(en, l);
  const int first = l ? __builtin_amdgcn_readlane(incl, l - 1) : 0;
  s.row = s.start + (tm - first) * BM;
  return true;
}

// ds_read_b64_tr_b16: in each group of 16 lanes every lane loads 8 bytes (four
// 16-bit values) at its own address, and lane i receives, for j = 0 .. 3, value
// i % 4 of the 8 bytes loaded by lane 4 j + i / 4 of its group.
__device__ __forceinline__ s16x4 lds_transpose(const void* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(const_cast<void*>(p)));
}

// LDS panel of ROWS rows (of M or N) by one k-tile of 64 bytes per row.
// KC: the operand's rows are K-contiguous; row r takes 64 bytes, its 16-byte
// group q in slot q ^ ((r / 4) % 4), so that the 16 lanes of a quarter wave,
// which read the same group of 16 rows, cover all banks. Otherwise rows of k
// with ROWS values each; 16-byte group q of row k sits in slot q ^ swz(k): the
// transposing reads of 16 lanes take four rows of k at the same columns (16-bit
// types), the four quarters of a wave rows k, k + 4, k + 8, k + 12 (fp32).
template <typename T, int ROWS, bool KC>
struct Panel {
  static constexpr int ES = sizeof(T), EV = 16 / ES, BK = 64 / ES, BYTES = ROWS * 64;
  static constexpr int GPR = ROWS / EV;  // groups per row of k
  static __device__ __forceinline__ int swz(int k) {
    if constexpr (ES == 4) return 4 * ((k >> 2) & 3);
    return ROWS >= 128 ? 4 * (k & 3) : 4 * ((k >> 1) & 1);
  }
  // which values 16-byte group `i` of the panel (in LDS order) holds
  static __device__ __forceinline__ void where(int i, int& row, int& k) {
    if constexpr (KC) {
      row = i >> 2;
      k = EV * ((i & 3) ^ ((row >> 2) & 3));
    } else {
      k = i / GPR;
      row = EV * ((i % GPR) ^ swz(k));
    }
  }
  // MFMA operand of rows row0 .. row0 + 15: lane l holds row l % 16, 16 bytes
  // of k from group l / 16.
  static __device__ __forceinline__ i32x4 frag(const char* p, int row0, int lane) {
    const int li = lane & 15, lg = lane >> 4;
    if constexpr (KC) {
      const int r = row0 + li;
      return *reinterpret_cast<const i32x4*>(p + r * 64 + 16 * (lg ^ ((r >> 2) & 3)));
    } else if constexpr (ES == 4) {
      const int c = row0 + li;
      i32x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        v[e] = *reinterpret_cast<const int*>(p + (4 * lg + e) * (ROWS * 4) + 16 * ((c >> 2) ^ (4 * lg)) + 4 * (c & 3));
      return v;
    } else {
      const int k = 8 * lg + (li >> 2), c = row0 + 4 * (li & 3);
      const char* s = p + k * (ROWS * 2) + 16 * ((c >> 3) ^ swz(k)) + 2 * (c & 4);
      union {
        s16x4 h[2];
        i32x4 v;
      } u;
      u.h[0] = lds_transpose(s);
      u.h[1] = lds_transpose(s + 4 * (ROWS * 2));
      return u.v;
    }
  }
};

// acc += one k-tile of (rows n of b) x (rows m of a): lane l holds column
// m = l % 16 and rows n = 4 (l / 16) + r, so four consecutive n of one m.
template <typename T>
__device__ __forceinline__ void mma_tile(f32x4& acc, const i32x4& b, const i32x4& a) {
  if constexpr (std::is_same_v<T, float>) {
    const f32x4 x = __builtin_bit_cast(f32x4, b), y = __builtin_bit_cast(f32x4, a);
#pragma unroll
    for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], y[e], acc, 0, 0, 0);
  } else if constexpr (std::is_same_v<T, __bf16>) {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, b), __builtin_bit_cast(bf16x8, a), acc, 0, 0, 0);
  } else {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, b), __builtin_bit_cast(f16x8, a), acc, 0, 0, 0);
  }
}

// D[m][n .. n + 3] = alpha acc + beta C in the type O (m inside the output;
// columns past N are not touched; C not read when beta == 0).
template <typename O>
__device__ __forceinline__ void store_quad(const GroupedArgs& g, const O* C, O* D, int64_t m, int n, const f32x4& acc) {
  typedef O o4 __attribute__((ext_vector_type(4)));
  const int left = g.N - n;
  if (left <= 0) return;
  float v[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) v[u] = g.alpha * acc[u];
  O* d = D + m * g.ldd + n;
  const O* c = C + m * g.ldc + n;
  if (g.vec4 && left >= 4) {
    if (g.beta != 0.0f) {
      const o4 w = *reinterpret_cast<const o4*>(c);
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = __builtin_fmaf(g.beta, (float)w[u], v[u]);
    }
    *reinterpret_cast<o4*>(d) = o4{(O)v[0], (O)v[1], (O)v[2], (O)v[3]};
  } else {
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (u < left) {
        if (g.beta != 0.0f) v[u] = __builtin_fmaf(g.beta, (float)c[u], v[u]);
        d[u] = (O)v[u];
      }
  }
}

}  // namespace trnblas
