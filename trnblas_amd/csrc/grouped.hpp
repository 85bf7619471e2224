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
  int slots;  // workgroups that run at a time (tiles of one workgroup per CU)
  float alpha, beta;
  int out_f16;  // D and C are fp16 (products of 4-bit floats; else bf16 or fp32)
  int out32;  // D and C are fp32 whatever the operands are
  int padded; // operands end in zeros up to 16 bytes (host only)
  int vec4;   // D and C take 4-element accesses (aligned, ld % 4 == 0)
};

// An fp32 result of 16-bit operands is summed in chains of at most so many values of k. One chain
// is a random walk of its roundings: the largest error of same-sign products over |A||B| was
// 7.3e-7 after 1024 values, 1.4e-6 after 4096, 2.2e-6 after 8192 and 8.7e-6 after 131072 (bf16 and
// fp16 alike); chains leave 1.4e-6 at 4096 and less from there on. (A 16-bit result is
// rounded to 2^-9 or 2^-12 at its end: one chain.) The kernels that restart their sums are CHAINS
// ones, launched where k is longer: a second set of sums in every one would cost the
// others' occupancy (rows_kernel of two blocks 126 registers, 135 with them: one workgroup
// per CU instead of two).
constexpr int kChain16 = 4096;

// Whether such a product (k: its rows where these are ragged) needs them.
template <typename T>
inline bool needs_chains(const GroupedArgs& g, int64_t k) {
  return sizeof(T) == 2 && g.out32 && k > kChain16;
}

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
  int quarter;     // of the tile, or -1
};

// Tiles that SPLIT (see tile_of) leaves whole.
__device__ __forceinline__ int whole_tiles(const GroupedArgs& g, int tiles) {
  const int whole = tiles / g.slots * g.slots;
  return 4 * (tiles - whole) > 3 * g.slots ? tiles : whole;
}

// Tile of workgroup `bid` among `tiles`; false when there is none left. Workgroups
// go to the XCDs round-robin: each XCD walks one contiguous range of the tiles.
// SPLIT (one workgroup per CU, g.slots of them): tiles that would not fill a last
// round are cut into quarters, one workgroup each, unless they fill three quarters
// of it: a quarter takes about a third of a tile's time.
template <bool SPLIT>
__device__ __forceinline__ bool tile_of(const GroupedArgs& g, int bid, int tiles, int& tile, int& quarter) {
  auto range = [](int b, int n, int& t) __attribute__((always_inline)) {
    const int q = n / kNumXcd, r = n % kNumXcd, x = b % kNumXcd, i = b / kNumXcd;
    t = x * q + min(x, r) + i;
    return i < q + (x < r);
  };
  quarter = -1;
  if constexpr (!SPLIT) return range(bid, tiles, tile);
  const int whole = whole_tiles(g, tiles), cut = tiles - whole;
  const int first = (whole + kNumXcd - 1) / kNumXcd * kNumXcd;  // workgroups up to here take whole tiles
  if (bid < first) return range(bid, whole, tile);
  if (!range(bid - first, 4 * cut, tile)) return false;
  quarter = tile & 3;
  tile = whole + (tile >> 2);
  return true;
}

// Inclusive sum over the lanes of the wave, by DPP: lanes 1, 2, 4 and 8 back in
// each row of 16, then the rows' last lanes broadcast to the rows after them.
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
  return v;
}

// tile_of among ragged rows cut into tiles of BM rows per segment and g.tiles_n
// column tiles, walked in bands of `band` row tiles by columns. The number of
// tiles is known on the device only: the grid is a bound, and each wave counts the
// tiles of 64 segments at a time (one load and a scan).
template <int BM, bool SPLIT = false>
__device__ __forceinline__ bool ragged_tile(const GroupedArgs& g, int bid, int band, Segment& s) {
  const int lane = threadIdx.x & 63;
  const int nseg = g.groups + 2;
  int total = 0, st = 0, en = 0, incl = 0;
  for (int base = 0; base < nseg; base += 64) {
    const int i = base + lane;
    st = boundary(g, i);
    en = max(boundary(g, i + 1), st);
    incl = wave_scan(i < nseg ? (en - st + BM - 1) / BM : 0);
    total += __builtin_amdgcn_readlane(incl, 63);
  }
  int t, tm, tn;
  if (!tile_of<SPLIT>(g, bid, total * g.tiles_n, t, s.quarter)) return false;
  grouped_tile(t, total, g.tiles_n, band, tm, tn);
  s.tn = tn;
  if (nseg > 64) {  // walk the segments again up to the one that holds tm
    int before = 0;
    for (int base = 0;; base += 64) {
      const int j = base + lane;
      st = boundary(g, j);
      en = max(boundary(g, j + 1), st);
      incl = wave_scan(j < nseg ? (en - st + BM - 1) / BM : 0);
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

// LDS panel of ROWS rows (of M or N) by one k-tile of 128 bytes per row, two
// MFMA steps of 64 bytes.
// KC: the operand's rows are K-contiguous; row r takes 128 bytes, its 16-byte
// group q in slot q ^ ((r / 2) % 8). A 16-byte LDS read serves lanes 0-3, 12-15 and
// 20-27 together, then 4-11, 16-19 and 28-31 (and the same of the upper half):
// each such set then covers all banks. (64 bytes per row and k-tile cost 10 %:
// the L2 serves 128-byte lines.) Otherwise rows of k with ROWS values each; 16-byte
// group q of row k sits in slot q ^ swz(k): the transposing reads of 32 lanes take
// rows k .. k + 3 and k + 8 .. k + 11 at the same columns (16-bit types), the four
// quarters of a wave rows k, k + 4, k + 8, k + 12 (fp32).
template <typename T, int ROWS, bool KC>
struct Panel {
  static constexpr int ES = sizeof(T), EV = 16 / ES, BK = 128 / ES, BYTES = ROWS * 128;
  static constexpr int GPR = ROWS / EV;  // groups per row of k
  static __device__ __forceinline__ int swz(int k) {
    if constexpr (ES == 4) return 4 * ((k >> 2) & 3);
    return (ROWS >= 128 ? 4 * (k & 3) : 4 * ((k >> 1) & 1)) + 2 * ((k >> 3) & 1);
  }
  // which values 16-byte group `i` of the panel (in LDS order) holds
  static __device__ __forceinline__ void where(int i, int& row, int& k) {
    if constexpr (KC) {
      row = i >> 3;
      k = EV * ((i & 7) ^ ((row >> 1) & 7));
    } else {
      k = i / GPR;
      row = EV * ((i % GPR) ^ swz(k));
    }
  }
  // MFMA operand i of a wave whose rows start at row0 (a multiple of 64, or of
  // 32 with fewer than five operands), step s: rows row0 + 16 i .. + 15, lane l with
  // row l % 16 and 16 bytes of k from group 4 s + l / 16. The swizzles make its LDS
  // offset a constant plus one of NV offsets of the lane.
  static constexpr int NV = KC ? 2 : ES == 4 ? 4 : 8;
  static __device__ __forceinline__ void lane_offsets(int row0, int lane, uint32_t (&v)[NV]) {
    const int li = lane & 15, lg = lane >> 4;
    if constexpr (KC) {
#pragma unroll
      for (int s = 0; s < 2; ++s) v[s] = (row0 + li) * 128 + 16 * ((4 * s + lg) ^ (li >> 1));
    } else if constexpr (ES == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        v[i] = 4 * lg * (ROWS * 4) + 16 * (((row0 >> 2) + 4 * i + (li >> 2)) ^ (4 * lg)) + 4 * (li & 3);
    } else {
      const int k = 8 * lg + (li >> 2);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        v[i] = k * (ROWS * 2) + 16 * (((row0 >> 3) + 2 * i + ((li & 3) >> 1)) ^ swz(k)) + 8 * (li & 1);
    }
  }
  // p: the panel plus lane_offsets'
  static __device__ __forceinline__ i32x4 frag(const char* const (&p)[NV], int i, int s) {
    if constexpr (KC) {
      return *reinterpret_cast<const i32x4*>(p[s] + 2048 * i);
    } else if constexpr (ES == 4) {
      i32x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        v[e] = *reinterpret_cast<const int*>(p[i & 3] + (16 * s + e) * (ROWS * 4) + 256 * (i >> 2));
      return v;
    } else {
      const char* q = p[i & 7] + 256 * (i >> 3) + 32 * s * (ROWS * 2);
      union {
        s16x4 h[2];
        i32x4 v;
      } u;
      u.h[0] = lds_transpose(q);
      u.h[1] = lds_transpose(q + 4 * (ROWS * 2));
      return u.v;
    }
  }
};

// acc += one MFMA step of (rows n of b) x (rows m of a): lane l holds column
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

// The tile of a workgroup: where its operand panels start, how many rows of
// each are inside, the k range, and where the output goes.
struct TileJob {
  const char *A, *B;  // panel corners at k = 0
  int rows_a, rows_b, K;
  int group, quarter;
  int64_t m;  // first output row
  int n;      // first output column
  const void* C;
  void* D;
};

// The group that has the nth most rows, of at most 64.
__device__ __forceinline__ int by_rows(const GroupedArgs& g, int nth) {
  const int lane = threadIdx.x & 63;
  const int rows = lane < g.groups ? max(boundary(g, lane + 2) - boundary(g, lane + 1), 0) : -1;
  int before = 0;
  for (int j = 0; j < g.groups; ++j) {
    const int other = __builtin_amdgcn_readlane(rows, j);
    before += other > rows || (other == rows && j < lane);
  }
  return __builtin_ctzll(__ballot(before == nth));
}

// RK: ragged k (grouped_rank_k), else ragged rows.
template <typename T, int BM, int BN, bool BKC, bool RK, bool SPLIT = false>
__device__ __forceinline__ bool tile_job(const GroupedArgs& g, TileJob& j) {
  const int64_t es = sizeof(T), eo = g.out32 ? 4 : es;
  if constexpr (RK) {
    const int per = g.tiles_m * g.tiles_n;
    int t, tm, tn;
    if (!tile_of<SPLIT>(g, blockIdx.x, g.groups * per, t, j.quarter)) return false;
    // The groups' numbers of rows differ: each XCD takes an eighth of every group's
    // tiles (32768 rows in 8 groups, 4096 x 2048: 490 us with one range of tiles per XCD,
    // 440 now), on 256 x 256 tiles the longest first, so that the last round is short
    // (418; 24 groups, 2048 x 1024, added to fp32: 150 and 137).
    int grp = t / per, in = t - grp * per;
    const int tiles = g.groups * per, whole = SPLIT ? whole_tiles(g, tiles) : tiles;
    if (per % kNumXcd == 0 && whole % kNumXcd == 0) {
      const int first = t < whole ? 0 : whole, each = ((t < whole ? whole : tiles) - first) / kNumXcd, share = per / kNumXcd;
      const int x = (t - first) / each, i = first / kNumXcd + (t - first) - x * each;
      grp = i / share;
      in = x * share + i - grp * share;
      if (SPLIT && g.groups <= 64) grp = by_rows(g, grp);
    }
    grouped_tile(in, g.tiles_m, g.tiles_n, 8, tm, tn);
    const int start = boundary(g, grp + 1), end = max(boundary(g, grp + 2), start);
    j.group = grp;
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
    if (!ragged_tile<BM, SPLIT>(g, blockIdx.x, 8, s)) return false;
    j.quarter = s.quarter;
    const bool of_group = s.group >= 0 && s.group < g.groups;
    j.group = s.group;
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
  if constexpr (SPLIT) {
    if (j.quarter >= 0) {
      const int m = BM / 2 * (j.quarter & 1), n = BN / 2 * (j.quarter >> 1);
      j.rows_a = min(BM / 2, j.rows_a - m);
      j.rows_b = min(BN / 2, j.rows_b - n);
      if (j.rows_a <= 0 || j.rows_b <= 0) return false;
      j.m += m, j.n += n;
      j.A += (RK ? m : m * g.lda) * es;
      j.B += (BKC ? n * g.ldb : n) * es;
    }
  }
  return true;
}

// The outputs of a wave: blocks of 16 x 16 from row m0, column n0 of the tile.
// Whole quads (aligned, N a multiple of 4): all of C's quads of a block row are
// under way before the first is used, the next row's behind this row's stores (one
// quad at a time, each waiting for its C, the accumulated fp32 gradients of 24 groups
// took 186 us). Quads outside repeat the last one inside. Rows that start anywhere:
// a block row goes through LDS (kStoreLds bytes of the wave's own, no longer used by
// others), so that neighbouring lanes store neighbouring values (four separate
// stores of each lane's quad: 16383 x 4095 bf16 took 120 us longer).
template <int FN>
constexpr int kStoreLds = 16 * (16 * FN + 4) * 4;
template <int FM, int FN, typename O>
__device__ __forceinline__ void store_wave(const GroupedArgs& g, const TileJob& j, const f32x4 (&acc)[FM][FN], int m0,
                                           int n0, int lane, char* lds) {
  typedef O o4 __attribute__((ext_vector_type(4)));
  const O* C = static_cast<const O*>(j.C);
  O* D = static_cast<O*>(j.D);
  const int li = lane & 15, n = j.n + n0 + 4 * (lane >> 4);
  // the sum of a block, read here: the compiler would scale all of them before the branches
  auto take = [&](int a, int b) __attribute__((always_inline)) {
    f32x4 v = acc[a][b];
    asm volatile("" : "+v"(v));
    return v;
  };
  if (g.vec4 && (g.N & 3) == 0) {
    auto store = [&](int a, auto value) __attribute__((always_inline)) {
      const int m = m0 + 16 * a + li;
      O* d = D + (j.m + m) * g.ldd + n;
#pragma unroll
      for (int b = 0; b < FN; ++b) {
        const f32x4 v = value(a, b);
        if (m < j.rows_a && n + 16 * b < g.N) *reinterpret_cast<o4*>(d + 16 * b) = o4{(O)v[0], (O)v[1], (O)v[2], (O)v[3]};
      }
      __builtin_amdgcn_sched_barrier(0);  // a row's registers at a time
    };
    // 16-bit rows that start on 16 bytes: lanes 16 apart exchange halves of two
    // blocks, so that a lane stores 16 bytes and a row 64 at a time (8 and 32: 8192 x
    // 2048 x 8192 237 us, now 223; 8191 x 2056 x 4104 of 4-bit values 88, now 82)
    if constexpr (sizeof(O) == 2) {
      if (g.beta == 0.0f && (((uint64_t)D / 2 | (uint64_t)g.ldd | (uint64_t)g.N) & 7) == 0) {
        typedef int i32x2 __attribute__((ext_vector_type(2)));
        auto pack = [&](int a, int b) __attribute__((always_inline)) {
          const f32x4 v = take(a, b) * g.alpha;
          return __builtin_bit_cast(i32x2, o4{(O)v[0], (O)v[1], (O)v[2], (O)v[3]});
        };
        const int lg = lane >> 4, col = j.n + n0 + 16 * (lg & 1) + 8 * (lg >> 1);
#pragma unroll
        for (int a = 0; a < FM; ++a) {
          const int m = m0 + 16 * a + li;
          O* d = D + (j.m + m) * g.ldd + col;
#pragma unroll
          for (int b = 0; b < FN; b += 2) {
            const i32x2 x = pack(a, b), y = pack(a, b + 1);
            const auto p = __builtin_amdgcn_permlane16_swap(x[0], y[0], false, false);
            const auto q = __builtin_amdgcn_permlane16_swap(x[1], y[1], false, false);
            if (m < j.rows_a && col + 16 * b < g.N)
              *reinterpret_cast<i32x4*>(d + 16 * b) = i32x4{(int)p[0], (int)q[0], (int)p[1], (int)q[1]};
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        return;
      }
    }
    if (g.beta == 0.0f) {
#pragma unroll
      for (int a = 0; a < FM; ++a) store(a, [&](int p, int b) __attribute__((always_inline)) { return take(p, b) * g.alpha; });
    } else {
      o4 c[2][FN];
      auto load = [&](int a) __attribute__((always_inline)) {
        const O* p = C + (j.m + min(m0 + 16 * a + li, j.rows_a - 1)) * g.ldc;
#pragma unroll
        for (int b = 0; b < FN; ++b) c[a & 1][b] = *reinterpret_cast<const o4*>(p + min(n + 16 * b, g.N - 4));
      };
      load(0);
#pragma unroll
      for (int a = 0; a < FM; ++a) {
        if (a + 1 < FM) load(a + 1);
        store(a, [&](int p, int b) __attribute__((always_inline)) {
          f32x4 v = take(p, b);
#pragma unroll
          for (int u = 0; u < 4; ++u) v[u] = __builtin_fmaf(g.beta, (float)c[p & 1][b][u], g.alpha * v[u]);
          return v;
        });
      }
    }
    return;
  }
  constexpr int W = 16 * FN, LD = W + 4;
  float* buf = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int a = 0; a < FM; ++a) {
#pragma unroll
    for (int b = 0; b < FN; ++b) *reinterpret_cast<f32x4*>(buf + li * LD + 16 * b + 4 * (lane >> 4)) = take(a, b) * g.alpha;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int h = 0; h < W / 4; ++h) {
      const int e = 64 * h + lane, r = e / W, c = e % W, m = m0 + 16 * a + r, col = j.n + n0 + c;
      float v = buf[r * LD + c];
      if (m < j.rows_a && col < g.N) {
        if (g.beta != 0.0f) v = __builtin_fmaf(g.beta, (float)C[(j.m + m) * g.ldc + col], v);
        D[(j.m + m) * g.ldd + col] = (O)v;
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
}

// The launches for one element type (grouped_run.hpp); bkc: B's columns are
// K-contiguous.
template <typename T>
int grouped_gemm_run(const GroupedArgs& g, bool bkc, hipStream_t s);
template <typename T>
int grouped_rank_k_run(const GroupedArgs& g, hipStream_t s);

}  // namespace trnblas
