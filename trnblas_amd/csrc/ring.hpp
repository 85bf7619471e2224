// The grouped products' main kernel: operands that LDS DMA can read in place
// (16-byte aligned bases, leading dimensions, strides and contiguous extents),
// k-tiles of 128 bytes per row in two LDS stages.
#pragma once

#include "gemm.hpp"
#include "grouped.hpp"
#include "grouped_plan.hpp"

namespace trnblas {

// Codes of microscaled 4-bit floats, two per byte: an operand type of one byte
// whose "values" along k are bytes.
struct fp4x2 {
  uint8_t v;
};

typedef int i32x8 __attribute__((ext_vector_type(8)));

// f(0) .. f(N - 1), each with its number as a constant.
template <int N, int I = 0, typename F>
__device__ __forceinline__ void each(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    each<N, I + 1>(f);
  }
}

constexpr int kChunk = 256;  // bytes of scales per 16 rows x 512 values (mx.hip)

struct MxScales {
  const uint8_t* a;
  const uint8_t* b;
  const void* x;    // rows_kernel: A before quantisation, kx values per row,
  int64_t ldx;      // leading dimension ldx
  int kx;
  int vec;          // its rows start on 16 bytes
  int chunks;       // along K, the same for A and B
  int64_t b_step;   // bytes per matrix of B
};

// Offset of a pointer into LDS.
__device__ __forceinline__ uint32_t lds_offset(const void* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p;
}

// A buffer resource at a (uniform) address: reads at or past `records` bytes from
// it give zeros with no memory access.
constexpr int kRecords = 0x7ffffff0;
constexpr uint32_t kPastEnd = 0x80000000u;  // an offset past any resource's records

__device__ __forceinline__ i32x4 dma_rsrc(const void* base, int records) {
  const uint64_t b = (uint64_t)base;
  i32x4 r;
  r[0] = __builtin_amdgcn_readfirstlane((int)(uint32_t)b);
  r[1] = __builtin_amdgcn_readfirstlane((int)((uint32_t)(b >> 32) & 0xffffu));
  r[2] = __builtin_amdgcn_readfirstlane(records);
  r[3] = 0x00020000;
  return r;
}

// One LDS DMA of the wave: lane l's 16 bytes at offset voff of the resource land
// at LDS offset lds + AT + 16 l. Inline asm for the reason given at
// lds_dma16_asm; three instructions, so that they fit between two MFMAs.
template <int AT>
__device__ __forceinline__ void lds_dma(const i32x4& rsrc, uint32_t lds, uint32_t voff) {
  asm volatile("s_add_u32 m0, %0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(voff), "s"(rsrc), "n"(AT)
               : "memory", "m0", "scc");
}

// acc += (rows n) x (rows m) over one k-tile of a 16 x 16 block; fp4x2: with byte
// BYTE of each scale dword. Lane l holds column m = l % 16 and rows n = 4 (l
// / 16) + r. Inline asm with the sum in accumulation registers: left to choose,
// the compiler moves the 64 blocks of a wave through four of them. Volatile, so
// that the LDS reads and DMAs written between MFMAs stay there. The hazards that
// the compiler cannot see: a block's next MFMA comes at least FM FN - 1 MFMAs
// later, the epilogue waits (settle), and no vector instruction writes an operand
// within two wait states: operands and scales are as LDS reads leave them, the
// scale's byte is the instruction's to pick, and a step begins with the wait.
template <typename T, int BYTE>
__device__ __forceinline__ void mma_block(f32x4& acc, const i32x4& n, const i32x4& m, int sn, int sm) {
  if constexpr (std::is_same_v<T, fp4x2>)
    asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[%5,%5,0] op_sel_hi:[%6,%6,0] cbsz:4 blgp:4"
                 : "+a"(acc)
                 : "v"(n), "v"(m), "v"(sn), "v"(sm), "n"(BYTE & 1), "n"(BYTE >> 1));
  else if constexpr (std::is_same_v<T, __bf16>)
    asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(acc) : "v"(n), "v"(m));
  else if constexpr (std::is_same_v<T, _Float16>)
    asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(acc) : "v"(n), "v"(m));
  else
    mma_tile<T>(acc, n, m);
}
// The wait states between the last mma_block and the first read of a sum: no
// use of the sums comes before the statement that takes them here.
template <int FM, int FN>
__device__ __forceinline__ void settle(f32x4 (&acc)[FM][FN]) {
  asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
#pragma unroll
  for (int a = 0; a < FM; ++a)
#pragma unroll
    for (int b = 0; b < FN; ++b) asm volatile("" : "+a"(acc[a][b]));
}

// The LDS DMA of one operand's panel: a wave moves NB blocks of 1 KiB per
// k-tile. Per lane and block it keeps the offset of its 16-byte group from the
// panel's corner at the current k-tile; groups of rows outside the tile, those past
// K in the last k-tile, and whole k-tiles after it read zeros.
template <typename T, int ROWS, bool KC, int WAVES>
struct PanelDma {
  using P = Panel<T, ROWS, KC>;
  static constexpr int NB = P::BYTES / 1024 / WAVES;
  static_assert(NB >= 1, "a block for every wave");
  const char* base;  // of the next k-tile to move
  int64_t step;      // bytes per k-tile
  uint32_t off[NB];
  __device__ __forceinline__ void init(const char* corner, int64_t ld, int rows, int wave, int lane) {
    base = corner;
    step = KC ? 128 : (int64_t)P::BK * ld * P::ES;
#pragma unroll
    for (int u = 0; u < NB; ++u) {
      int r, k;
      P::where((NB * wave + u) * 64 + lane, r, k);
      off[u] = r < rows ? (uint32_t)((KC ? r * ld + k : k * ld + r) * P::ES) : kPastEnd;
    }
  }
  // before the last k-tile, of `left` < BK values of k
  __device__ __forceinline__ void last(int left, int wave, int lane) {
#pragma unroll
    for (int u = 0; u < NB; ++u) {
      int r, k;
      P::where((NB * wave + u) * 64 + lane, r, k);
      if (k >= left) off[u] = kPastEnd;
    }
  }
};

// 2 x 2 waves, each FM x FN MFMA blocks of 16 x 16: a tile of BM x BN = 32 FM x 32 FN
// outputs, in k-tiles of 128 bytes per row, two MFMA steps, and two LDS stages.
// While the MFMAs of a step run the wave reads the fragments of the next step into
// its other register set: those of step 1 in the first half of step 0, those of
// the next k-tile in the second half of step 1. In the middle of step 0 a barrier
// tells that every wave has read k-tile t; the DMAs of k-tile t + 2 into its stage
// follow, over the rest of the k-tile. In the middle of step 1 one tells that
// k-tile t + 1, sent out a k-tile before, has landed (vmcnt leaves out the DMAs of t +
// 2). Reads and DMAs are spread between the MFMAs: a wave has its SIMD to itself,
// and whatever does not fit between two MFMAs (16 cycles) idles the matrix unit.
//
// Measured, 256 x 256 tiles: bf16 8192^3 K-contiguous 715 us (1.54 PFLOP/s), 32768 rows
// in 16 groups by 4096^2 868-905 (1.2-1.27); 4-bit 8192 x 8192 x 32768 5.1 PFLOP/s. The
// MFMAs alone run at 2.4 PFLOP/s (4-bit 8.8): with the reads and DMAs between them
// they take 80 % of the cycles, at the clock that the power limit leaves. A tile costs
// 10 us besides its k-tiles, most of it the stores of all CUs at once (8192 x 2048 x
// 8192 223 us, 194 without stores); starting the CUs at different times gained nothing.
// One barrier per k-tile instead of two: column-contiguous operands 1.11 PFLOP/s against 1.18.
//
// Scales (fp4x2): a dword per row and block-of-four serves four steps. They come
// by DMA too, whole chunks, two groups of four steps ahead, into a ring of two: a group
// is in registers before its slot is filled again.
// The rows of a tile start anywhere in a chunk, so A's take one chunk more.
// The sizes of a tile's LDS.
template <typename T, int FM, int FN>
struct RingLds {
  static constexpr int BM = 32 * FM, BN = 32 * FN, NS = 2, STAGE = 128 * (BM + BN);
  static constexpr int SA = BM / 64 + 1, SB = BN / 64;  // scale DMAs of a group: four chunks each
  static constexpr int SGROUP = std::is_same_v<T, fp4x2> ? 1024 * (SA + SB) : 0, SRING = 2;
  static constexpr int BYTES = NS * STAGE + SRING * SGROUP;
};

// Whether the plan's entry is of these tiles, and as many of its workgroups fit into a CU's LDS.
template <typename T, int FM, int FN>
constexpr bool fits(const RingCost& c) {
  return c.fm == FM && c.fn == FN && c.per_cu * RingLds<T, FM, FN>::BYTES <= 160 << 10;
}
static_assert(fits<__bf16, 8, 8>(kRing16[0]) && fits<__bf16, 4, 4>(kRing16[1]) && fits<__bf16, 2, 4>(kRing16[2]), "16-bit plan");
static_assert(fits<fp4x2, 8, 8>(kRing4[0]) && fits<fp4x2, 4, 4>(kRing4[1]) && fits<fp4x2, 2, 4>(kRing4[2]), "4-bit plan");

// The lane's number; ANEW: counted where it is asked for (kernels of chains: 256 x 256 tiles can
// keep neither it nor the addresses made of it from one chain to the next).
template <bool ANEW>
__device__ __forceinline__ int lane_of() {
  int lane = threadIdx.x & 63;
  if constexpr (ANEW) asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(lane));
  return lane;
}

template <typename T, int FM, int FN, bool BKC, bool RK, bool CHAINS>
__device__ __forceinline__ void ring_tile(const GroupedArgs& g, const MxScales& x, const TileJob& j, int wave, char* lds) {
  constexpr bool MX = std::is_same_v<T, fp4x2>, FOLD = std::is_same_v<T, float>;
  using L = RingLds<T, FM, FN>;
  constexpr int WAVES = 4, BM = L::BM, BN = L::BN, NS = L::NS, SA = L::SA, SB = L::SB, SGROUP = L::SGROUP, SRING = L::SRING;
  using DA = PanelDma<T, BM, !RK, WAVES>;
  using DB = PanelDma<T, BN, BKC, WAVES>;
  using PA = typename DA::P;
  using PB = typename DB::P;
  constexpr int STAGE = L::STAGE;
  constexpr int ND = DA::NB + DB::NB;  // DMAs per wave and k-tile, besides scales
  static_assert(STAGE == PA::BYTES + PB::BYTES && SA + SB <= 16, "one scale DMA per wave and step");
  const int lane = lane_of<CHAINS>();
  const int m0 = (wave & 1) * (16 * FM), n0 = (wave >> 1) * (16 * FN);
  const int nk = (j.K + PA::BK - 1) / PA::BK;
  const uint32_t lds0 = lds_offset(lds);
  DA da;
  DB db;
  da.init(j.A, g.lda, j.rows_a, wave, lane);
  db.init(j.B, g.ldb, j.rows_b, wave, lane);
  i32x4 ra, rb;
  uint32_t sta, stb;  // LDS offsets of the wave's blocks in the stage that takes the DMA
  // k-tile kt is the next to move, into stage kt % NS
  auto dma_turn = [&](int kt) __attribute__((always_inline)) {
    const int left = j.K - kt * PA::BK;
    if (left > 0 && left < PA::BK) {
      da.last(left, wave, CHAINS ? lane_of<CHAINS>() : lane);
      db.last(left, wave, CHAINS ? lane_of<CHAINS>() : lane);
    }
    const uint32_t st = lds0 + (uint32_t)kt % NS * STAGE;
    sta = st + DA::NB * 1024 * wave;
    stb = st + PA::BYTES + DB::NB * 1024 * wave;
    ra = dma_rsrc(da.base, left > 0 ? kRecords : 0);
    rb = dma_rsrc(db.base, left > 0 ? kRecords : 0);
    da.base += da.step;
    db.base += db.step;
  };
  auto dma = [&](auto uc) __attribute__((always_inline)) {
    constexpr int u = decltype(uc)::value;
    if constexpr (u < DA::NB)
      lds_dma<1024 * u>(ra, sta, da.off[u]);
    else if constexpr (u < ND)
      lds_dma<1024 * (u - DA::NB)>(rb, stb, db.off[u - DA::NB]);
  };

  // DMA i of a scale group: chunks 4 i .. 4 i + 3 of A's rows, then of B's. In
  // the loop wave w sends DMAs 8 (t % 2) + w and + 4 in k-tile t.
  [[maybe_unused]] uint32_t soff = 0;
  [[maybe_unused]] const uint8_t *sa = nullptr, *sb = nullptr;
  if constexpr (MX) {
    sa = x.a + (j.m >> 4) * x.chunks * kChunk;
    sb = x.b + j.group * x.b_step + (int64_t)(j.n >> 4) * x.chunks * kChunk;
    soff = (uint32_t)(lane >> 4) * x.chunks * kChunk + 16 * (lane & 15);
  }
  auto scale_dma = [&](int grp, int i) __attribute__((always_inline)) {
    if constexpr (MX) {
      const bool of_a = i < SA;
      const int c0 = 4 * (of_a ? i : i - SA);  // first chunk row
      // chunk rows of the tile; the last one of a matrix may be short of rows, never of bytes
      const int have = of_a ? ((int)(j.m & 15) + j.rows_a + 15) >> 4 : (j.rows_b + 15) >> 4;
      const uint32_t off = soff + (uint32_t)c0 * x.chunks * kChunk + (uint32_t)grp * kChunk;
      lds_dma<0>(dma_rsrc(of_a ? sa : sb, grp < x.chunks ? kRecords : 0),
                 lds0 + NS * STAGE + (uint32_t)grp % SRING * SGROUP + 1024 * i, c0 + (lane >> 4) < have ? off : kPastEnd);
    }
  };

  f32x4 acc[FM][FN];
  [[maybe_unused]] f32x4 sum[FOLD ? FM : 1][FOLD ? FN : 1];
#pragma unroll
  for (int a = 0; a < FM; ++a)
#pragma unroll
    for (int b = 0; b < FN; ++b) {
      acc[a][b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      if constexpr (FOLD) sum[a][b] = acc[a][b];
    }
  [[maybe_unused]] int qa[FM], qb[FN];
  auto read_scales = [&](int grp) __attribute__((always_inline)) {
    if constexpr (MX) {
      const char* p = lds + NS * STAGE + (uint32_t)grp % SRING * SGROUP + 64 * (lane >> 4);
      const int r = (int)(j.m & 15) + (lane & 15);
      const char* pa = p + (r >> 4) * kChunk + 4 * (r & 15) + m0 / 16 * kChunk;
      const char* pb = p + SA * 1024 + 4 * (lane & 15) + n0 / 16 * kChunk;
#pragma unroll
      for (int a = 0; a < FM; ++a) qa[a] = *reinterpret_cast<const int*>(pa + a * kChunk);
#pragma unroll
      for (int b = 0; b < FN; ++b) qb[b] = *reinterpret_cast<const int*>(pb + b * kChunk);
    }
  };
  i32x4 fa[2][FM], fb[2][FN];
  const char *pa[PA::NV], *pb[PB::NV];
  {
    uint32_t oa[PA::NV], ob[PB::NV];
    PA::lane_offsets(m0, lane, oa);
    PB::lane_offsets(n0, lane, ob);
#pragma unroll
    for (int i = 0; i < PA::NV; ++i) pa[i] = lds + oa[i];
#pragma unroll
    for (int i = 0; i < PB::NV; ++i) pb[i] = lds + PA::BYTES + ob[i];
  }
  // the reads go on to the stage of k-tile kt
  auto read_from = [&](int kt) __attribute__((always_inline)) {
    const int d = kt & 1 ? STAGE : -STAGE;
#pragma unroll
    for (int i = 0; i < PA::NV; ++i) pa[i] += d;
#pragma unroll
    for (int i = 0; i < PB::NV; ++i) pb[i] += d;
  };
  auto read = [&](int i, int set) __attribute__((always_inline)) {
    if (i < FN)
      fb[set][i] = PB::frag(pb, i, set);
    else if (i < FN + FM)
      fa[set][i - FN] = PA::frag(pa, i - FN, set);
  };
  [[maybe_unused]] int span = 0, chain = 0;
  // step s of k-tile kt (an odd one: ODD; fp4x2 only): the MFMAs of register set s, reads of the other set
  auto step = [&](int kt, auto oddc, auto sc) __attribute__((always_inline)) {
    constexpr int s = decltype(sc)::value, ODD = decltype(oddc)::value;
    constexpr int MM = FM * FN, HALF = MM / 2;
    constexpr int R0 = s ? HALF : 0, RW = MM * 3 / 8;           // MFMAs behind which the reads go
    constexpr int DW = MM * 5 / 4;                              // and the DMAs, from HALF of step 0
    constexpr int SENT = (MM * ND + DW - 1) / DW;               // DMAs sent when step 1 waits
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): this step's fragments
    asm volatile("s_nop 1");             // registers that the compiler moved where paths meet
    each<MM>([&](auto ic) __attribute__((always_inline)) {
      constexpr int i = decltype(ic)::value, a = i % FM, b = i / FM, t = s * MM + i - HALF;
      if constexpr (i == HALF) {
        if constexpr (s == 0) {
          __builtin_amdgcn_s_waitcnt(0xc07f);
          asm volatile("s_barrier" ::: "memory");
          dma_turn(kt + 2);
        } else {
          asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(SENT) : "memory");
          read_from(kt + 1);
        }
      }
      mma_block<T, 2 * ODD + s>(acc[a][b], fb[s][b], fa[s][a], MX ? qb[b] : 0, MX ? qa[a] : 0);
      each<ND>([&](auto uc) __attribute__((always_inline)) {
        if constexpr (t >= 0 && decltype(uc)::value * DW / ND == t) dma(uc);
      });
#pragma unroll
      for (int r = 0; r < FM + FN; ++r)
        if (R0 + r * RW / (FM + FN) == i) read(r, s ^ 1);
    });
    if constexpr (MX && s == 1) {
      const int i = 8 * ODD + wave;
      if (i < SA + SB) scale_dma((kt >> 1) + 2, i);
      if (i + 4 < SA + SB) scale_dma((kt >> 1) + 2, i + 4);
      if constexpr (ODD) read_scales((kt >> 1) + 1);
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
    if constexpr (MX) {
#pragma unroll
      for (int grp = 0; grp < 2; ++grp)
#pragma unroll
        for (int i = 0; i < SA + SB; i += 4)
          if (i + wave < SA + SB) scale_dma(grp, i + wave);
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      dma_turn(t);
      each<ND>(dma);
    }
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(ND) : "memory");
    read_scales(0);
#pragma unroll
    for (int i = 0; i < FN + FM; ++i) read(i, 0);
    if constexpr (FOLD) chain = span = 2 * chain_length(j.K, 4) / PA::BK;
    constexpr std::integral_constant<int, 0> zero{};
    constexpr std::integral_constant<int, 1> one{};
    if constexpr (MX) {
      // two k-tiles at a time: the four bytes of a scale dword
      for (int kt = 0; kt < nk; kt += 2) {
        step(kt, zero, zero);
        step(kt, zero, one);
        if (kt + 1 < nk) {
          step(kt + 1, one, zero);
          step(kt + 1, one, one);
        }
      }
    } else {
      for (int kt = 0; kt < nk; ++kt) {
        step(kt, zero, zero);
        step(kt, zero, one);
      }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no DMA into the LDS of the next workgroup
    if constexpr (!FOLD) settle(acc);
  }
  if constexpr (FOLD) {
#pragma unroll
    for (int a = 0; a < FM; ++a)
#pragma unroll
      for (int b = 0; b < FN; ++b) acc[a][b] += sum[a][b];
  }
  using O = std::conditional_t<MX, __bf16, T>;
  static_assert(4 * kStoreLds<FN> <= L::BYTES);
  char* own = lds + wave * kStoreLds<FN>;
  if (!(g.vec4 && (g.N & 3) == 0)) __syncthreads();  // the other waves' reads
  if (CHAINS || g.out32)
    store_wave<FM, FN, float>(g, j, acc, m0, n0, CHAINS ? lane_of<CHAINS>() : lane, own);
  else if (MX && g.out_f16)
    store_wave<FM, FN, _Float16>(g, j, acc, m0, n0, lane, own);
  else
    store_wave<FM, FN, O>(g, j, acc, m0, n0, lane, own);
}

// An address that all lanes have, as a scalar.
__device__ __forceinline__ const char* uniform(const char* p) {
  const uint64_t a = (uint64_t)p;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)a), hi = __builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32));
  return reinterpret_cast<const char*>((uint64_t)hi << 32 | lo);
}

// CHAINS (see kChain16): 256 x 256 tiles have no registers for a second set of sums, so each
// chain after the first takes its sum from D. 32768 rows in 2 groups by 4096 x 2048 take 455 us with
// these round trips, 396 as one chain; where no group has a second chain the kernel costs 3 %.
template <typename T, int FM, int FN, bool BKC, bool RK, bool CHAINS>
__device__ __forceinline__ void ring_chains(GroupedArgs g, const MxScales& x, TileJob j, int wave, char* lds) {
  if constexpr (!CHAINS) {
    ring_tile<T, FM, FN, BKC, RK, false>(g, x, j, wave, lds);
  } else {
    // what the loop carries, in scalar registers
    j.A = uniform(j.A), j.B = uniform(j.B), j.D = const_cast<char*>(uniform(static_cast<char*>(j.D)));
    j.C = uniform(static_cast<const char*>(j.C));
    for (int left = __builtin_amdgcn_readfirstlane(j.K);;) {
      j.K = min(left, kChain16);
      ring_tile<T, FM, FN, BKC, RK, true>(g, x, j, wave, lds);
      left -= j.K;
      if (left <= 0) return;
      j.A += j.K * (RK ? g.lda : 1) * (int64_t)sizeof(T);
      j.B += j.K * (BKC ? 1 : g.ldb) * (int64_t)sizeof(T);
      j.C = j.D, g.ldc = g.ldd, g.beta = 1.0f;  // each lane reads what it wrote
      __syncthreads();  // the other waves' LDS reads, before the next chain's DMAs
    }
  }
}

template <typename T, int FM, int FN, bool BKC, bool RK, bool CHAINS = false>
__global__ __launch_bounds__(256, FM * FN <= 16 ? 2 : 1) void ring_kernel(GroupedArgs g, MxScales x) {
  constexpr bool SPLIT = FM * FN == 64;  // one workgroup per CU: see tile_of
  __shared__ __attribute__((aligned(16))) char lds[RingLds<T, FM, FN>::BYTES];
  TileJob j;
  if (!tile_job<T, 32 * FM, 32 * FN, BKC, RK, SPLIT>(g, j)) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if constexpr (SPLIT) {
    if (j.quarter >= 0) {
      ring_chains<T, FM / 2, FN / 2, BKC, RK, CHAINS>(g, x, j, wave, lds);
      return;
    }
  }
  ring_chains<T, FM, FN, BKC, RK, CHAINS>(g, x, j, wave, lds);
}

// Workgroups of such a launch over `tiles` tiles (or at most so many), SPLIT's
// quarters included.
template <int FM, int FN>
static int64_t ring_grid(GroupedArgs& g, int64_t tiles) {
  g.slots = device_cus();
  return (tiles + (FM * FN == 64 ? 9 * g.slots / 4 + 2 * kNumXcd : 0) + kNumXcd - 1) / kNumXcd * kNumXcd;
}

}  // namespace trnblas
