// MXFP4 products of more than a few rows: tiles in LDS, the matrix cores fed from there.
//
// A K slice is 256 numbers: one 128-byte line of every row of A and B.  Lines are copied global ->
// LDS directly (global_load_lds, 16 bytes per lane, no registers in between) into two slots each;
// the 16-byte chunk c of row r lands at chunk position c ^ ((r >> 1) & 7), which makes the
// operand reads (ds_read_b128: 16 rows, one chunk each) free of bank conflicts.  Lane group g of a
// wavefront takes chunks 2g and 2g + 1 of a line, i.e. blocks 2g and 2g + 1 of the slice, in its
// two steps of 128.
//
// A slice is four phases: the lower half of a wave's m tiles with the first and the second step,
// then the upper half with both.  Operands are read one phase ahead, so the lower half of the A
// slot and all of the B slot are free after the first phase and are refilled from the second on,
// the upper half of A from the fourth: a line has a slice and a half to arrive, and a barrier
// every two phases says both that what comes next has landed and that what goes next has been
// read.  The refills walk ahead of the products across tile boundaries, so nothing drains between
// the tiles of a workgroup; only the output passes in between, through a staging area of its own,
// as whole lines.  Every operand read and every load sits behind a matrix instruction (pinned with
// scheduling barriers), as in matmul_dma_kernel.h.
//
// Rows past the end of A or B repeat the last row, chunks past the end of a row the last chunk; the
// scales that go with such a chunk are 2^-127 on both sides, whose products vanish in float32.
//
// The scales are laid out beforehand (mxfp4_arrange_scales, into the workspace) so that the two
// bytes a lane needs of each of four 16-row tiles are adjacent: a wave reads its 128 x 8 scales of
// a slice with two 8-byte LDS reads, and they come into LDS with two small loads per wave.  Read as
// they are stored it would take twelve 2-byte reads.
#include <type_traits>

#include "mxfp4_mfma.h"

namespace afir {

namespace {

template <int N>
__device__ __forceinline__ void wait_vmcnt() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
template <int OFF>
__device__ __forceinline__ void read16(uint32_t addr, u32x4 &dst) {
  asm volatile("ds_read_b128 %0, %1 offset:%2" : "=&v"(dst) : "v"(addr), "n"(OFF) : "memory");
}
template <int OFF>
__device__ __forceinline__ void read8(uint32_t addr, u32x2 &dst) {
  asm volatile("ds_read_b64 %0, %1 offset:%2" : "=&v"(dst) : "v"(addr), "n"(OFF) : "memory");
}
template <int I, int N, typename F>
__device__ __forceinline__ void static_for(F &&f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    static_for<I + 1, N>(f);
  }
}
// registers that reads in flight were given, handed back as fresh values after the wait
template <typename T, int N>
__device__ __forceinline__ void settle(T (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(v[i]));
}

// item R of N goes behind matrix instruction place(R, N, NM) of NM
constexpr int place(int r, int n, int nm) { return n <= nm ? r : r * nm / n; }

constexpr int kSliceBytes = 128;          // of a row: 256 codes, 8 blocks
constexpr int kSliceBlocks = 8;
constexpr int kUnitRows = 64;             // rows whose scales of a slice are one piece of 512 bytes
constexpr int kUnitBytes = kUnitRows * kSliceBlocks;
constexpr int kUnitPad = 4;               // units are allotted in fours: the rows of the largest tile

inline int64_t scale_units(int64_t rows) {
  return (rows + kUnitRows * kUnitPad - 1) / (kUnitRows * kUnitPad) * kUnitPad;
}
inline int64_t slices_of(int64_t kb) { return (kb + kSliceBlocks - 1) / kSliceBlocks; }

// scales [rows][kb] -> [slice][unit][lane][4 tiles][2]: lane l = 16 g + r holds, of row 16 i + r of the
// unit, blocks 2g and 2g + 1 of the slice.  A's units first, then B's.  A workgroup turns a unit's rows
// of 16 slices (128 bytes each) in LDS, so that both sides move whole lines.
constexpr int kTurnSlices = 16, kTurnPitch = kTurnSlices * kSliceBlocks + 4;
typedef u32x4 u32x4_any __attribute__((aligned(1)));
__global__ __launch_bounds__(256) void mxfp4_arrange_scales(MxOperands p, int units_a, int units_b, int slices,
                                                            int turns, unsigned char *__restrict__ out) {
  __shared__ __align__(16) unsigned char tile[kUnitRows * kTurnPitch];
  const int64_t total = (int64_t)(units_a + units_b) * turns;
  for (int64_t item = blockIdx.x; item < total; item += gridDim.x) {
    const int unit_all = (int)(item / turns), s0 = (int)(item % turns) * kTurnSlices;
    const bool is_a = unit_all < units_a;
    const int unit = is_a ? unit_all : unit_all - units_a, units = is_a ? units_a : units_b, rows = is_a ? p.m : p.n;
    const uint8_t *const s = is_a ? p.a_scales : p.b_scales;
    for (int i = threadIdx.x; i < kUnitRows * 8; i += 256) {
      const int r = i >> 3, at = (i & 7) * 16, block = s0 * kSliceBlocks + at;
      const int row = unit * kUnitRows + r < rows ? unit * kUnitRows + r : rows - 1;
      const uint8_t *const q = s + (int64_t)row * p.kb + block;
      uint32_t w[4] = {0, 0, 0, 0};   // past the end: 2^-127
      if (block + 16 <= p.kb) {
        const u32x4 v = *reinterpret_cast<const u32x4_any *>(q);
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (block + e < p.kb) w[e / 4] |= (uint32_t)q[e] << (8 * (e & 3));
      }
      uint32_t *const to = reinterpret_cast<uint32_t *>(tile + r * kTurnPitch + at);
#pragma unroll
      for (int e = 0; e < 4; ++e) to[e] = w[e];
    }
    __syncthreads();
    u32x2 *const to = reinterpret_cast<u32x2 *>(out + (is_a ? 0 : (int64_t)units_a * slices * kUnitBytes));
    for (int i = threadIdx.x; i < kTurnSlices * 64; i += 256) {
      const int lane = i & 63, ds = i >> 6, slice = s0 + ds;
      if (slice < slices) {
        const unsigned char *const from = tile + (lane & 15) * kTurnPitch + ds * kSliceBlocks + 2 * (lane >> 4);
        uint32_t w[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) w[t] = *reinterpret_cast<const uint16_t *>(from + t * 16 * kTurnPitch);
        to[((int64_t)slice * units + unit) * 64 + lane] = u32x2{w[0] | (w[1] << 16), w[2] | (w[3] << 16)};
      }
    }
    __syncthreads();
  }
}

__device__ __forceinline__ void map_tile(int p, int tiles_m, int tiles_n, int &tm, int &tn) {
  // tiles of one XCD (workgroup i runs on XCD i % 8) form patches of four tile rows
  const int ntiles = tiles_m * tiles_n;
  int q = p;
  if (ntiles % kNumXCD == 0) q = (p % kNumXCD) * (ntiles / kNumXCD) + p / kNumXCD;
  constexpr int kGroupM = 4;
  const int per_group = kGroupM * tiles_n;
  const int group = q / per_group, within = q % per_group, first_m = group * kGroupM;
  const int gsize = tiles_m - first_m < kGroupM ? tiles_m - first_m : kGroupM;
  tm = first_m + within % gsize;
  tn = within / gsize;
}

// WM x WN wavefronts, each TM x TN tiles of 16 x 16.
template <int WM, int WN, int TM, int TN>
struct Tile {
  static constexpr int kWaves = WM * WN, kBM = WM * TM * 16, kBN = WN * TN * 16;
  static constexpr int kSlotA = kBM * kSliceBytes, kSlotB = kBN * kSliceBytes;
  static constexpr int kScaleA = kBM * kSliceBlocks, kScaleB = kBN * kSliceBlocks;
  static constexpr int kOffB = 2 * kSlotA, kOffScaleA = kOffB + 2 * kSlotB, kOffScaleB = kOffScaleA + 2 * kScaleA;
  static constexpr int kOffStage = kOffScaleB + 2 * kScaleB;
  static constexpr int kStageBytes = 16 * 128;   // per wave: 16 rows of one 128-byte line
  static constexpr int kLds = kOffStage + kWaves * kStageBytes;
  static constexpr int kHalf = TM / 2;
  // direct-to-LDS loads of a wave per slice: regions of 1 KiB (8 rows) of half of A and of B,
  // and 256 bytes of each operand's scales
  static constexpr int kRegA = kBM / 2 / 8 / kWaves, kRegB = kBN / 8 / kWaves;
  static constexpr int kLoadsEarly = kRegA + kRegB + 2, kLoads = kLoadsEarly + kRegA;
  static_assert(TM % 8 == 0 || TM == 4, "A scales are read for four tiles at a time");
  static_assert(TN == 4, "B scales are read for four tiles at a time");
  static_assert(kRegA * kWaves * 16 == kBM && kRegB * kWaves * 8 == kBN, "whole regions per wave");
  static_assert(kScaleA == kWaves * 256 && kScaleB <= kWaves * 256, "one 4-byte load per lane");
};

template <int WM, int WN, int TM, int TN, int KIND>
__global__ __launch_bounds__(WM *WN * 64) void mxfp4_matmul_tiles(MxOperands p, const unsigned char *__restrict__ scales,
                                                                  int units_a, int units_b, int slices, int tiles_m,
                                                                  int tiles_n) {
  using T = Tile<WM, WN, TM, TN>;
  constexpr int kHalf = T::kHalf, NM = kHalf * TN;   // matrix instructions of a phase
  __shared__ __align__(1024) unsigned char smem[T::kLds];
  const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char *)smem;
  const int t = threadIdx.x, lane = t & 63, li = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6), wm = wave / WN, wn = wave % WN;
  const uint32_t pitch = (uint32_t)p.kb * kMxBlockBytes;
  const int total_tiles = tiles_m * tiles_n;

  // ---- operand reads: lane l reads row l % 16 of a tile, chunk 2 (l / 16) + step ----
  const uint32_t swz = (uint32_t)((li >> 1) & 7);
  const uint32_t rd_a0 = (uint32_t)((wm * TM * 16 + li) * kSliceBytes) + ((2 * g) ^ swz) * 16;   // step 1: ^ 16
  const uint32_t rd_b0 = (uint32_t)(T::kOffB + (wn * TN * 16 + li) * kSliceBytes) + ((2 * g) ^ swz) * 16;
  const uint32_t rd_sa = (uint32_t)(T::kOffScaleA + wm * (TM / 4) * kUnitBytes + lane * 8);
  const uint32_t rd_sb = (uint32_t)(T::kOffScaleB + wn * (TN / 4) * kUnitBytes + lane * 8);

  // ---- the cursor: tile and slice whose lines are requested next ----
  // A load's source is a wave-uniform base (the tile's first row) plus a per-lane offset: the row's,
  // kept per region, and the column's, kept per parity of the region (the swizzle repeats every 16 rows).
  int cur_tile = blockIdx.x, cur_left = 0, cur_slice = 0, cur_slot = 0;
  const unsigned char *base_a = nullptr, *base_b = nullptr;
  const unsigned char *scale_a = nullptr, *scale_b = nullptr;
  uint32_t row_a[2 * T::kRegA], row_b[T::kRegB], col[2];
  int tile_sa = 0, tile_sb = 0;   // the tile's first units
  // region q of a half of A: rows of the half's m tiles, one wave row after the other
  auto region_row_a = [&](int half, int q) {
    const int region = wave * T::kRegA + q;                     // of the half's regions
    constexpr int per_wm = kHalf * 2;                           // regions of a wave row's half
    return (region / per_wm) * TM * 16 + half * kHalf * 16 + (region % per_wm) * 8;
  };
  auto set_col = [&]() {
#pragma unroll
    for (int par = 0; par < 2; ++par) {
      const uint32_t c = (uint32_t)((lane & 7) ^ ((par * 4 + (lane >> 4)) & 7));
      const uint32_t at = (uint32_t)cur_slice * kSliceBytes + c * 16;
      col[par] = at < pitch ? at : pitch - 16;
    }
    scale_a = scales + ((int64_t)cur_slice * units_a + tile_sa) * kUnitBytes + wave * 256;
    scale_b = scales + ((int64_t)units_a * slices + (int64_t)cur_slice * units_b + tile_sb) * kUnitBytes + wave * 256;
  };
  auto begin_cursor = [&]() {
    int tm, tn;
    map_tile(cur_tile, tiles_m, tiles_n, tm, tn);
    const int m0 = tm * T::kBM, n0 = tn * T::kBN;
    base_a = p.a + (int64_t)m0 * pitch;
    base_b = p.b + (int64_t)n0 * pitch;
    tile_sa = m0 / kUnitRows;
    tile_sb = n0 / kUnitRows;
    const int last_m = p.m - 1 - m0, last_n = p.n - 1 - n0;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int q = 0; q < T::kRegA; ++q) {
        const int r = region_row_a(h, q) + (lane >> 3);
        row_a[h * T::kRegA + q] = (uint32_t)(r < last_m ? r : last_m) * pitch;
      }
#pragma unroll
    for (int q = 0; q < T::kRegB; ++q) {
      const int r = (wave * T::kRegB + q) * 8 + (lane >> 3);
      row_b[q] = (uint32_t)(r < last_n ? r : last_n) * pitch;
    }
    // tiles start their walk over K at different slices: the row pitch is often a power of two, and
    // without it all workgroups would ask the same few channels for the same lines at the same time
    cur_slice = (int)((unsigned)(tm + tn) % (unsigned)slices);
    cur_left = slices;
    set_col();
  };
  auto next_slice = [&]() {
    cur_slot ^= 1;
    --cur_left;
    cur_slice = cur_slice + 1 == slices ? 0 : cur_slice + 1;
    set_col();
  };
  auto next_tile = [&]() {   // when no slice of the tile is left
    // past the last tile the cursor walks that tile again: what it requests then is not read, and
    // the slices need no other form for the end
    if (cur_tile + (int)gridDim.x < total_tiles) cur_tile += gridDim.x;
    begin_cursor();
  };
  auto dma16 = [&](const unsigned char *base, uint32_t offset, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(offset), "s"(base) : "memory");
  };
  auto dma4 = [&](const unsigned char *base, uint32_t offset, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(to), "v"(offset), "s"(base) : "memory");
  };
  auto load_a = [&](auto half_tag, auto q_tag) {
    constexpr int h = decltype(half_tag)::value, q = decltype(q_tag)::value;
    const int row = region_row_a(h, q);
    dma16(base_a, row_a[h * T::kRegA + q] + ((row >> 3) & 1 ? col[1] : col[0]),
          lds + (uint32_t)(cur_slot * T::kSlotA + row * kSliceBytes));
  };
  // loads 0 .. kLoadsEarly - 1 of a slice: the lower half of A, B, the scales
  auto load_early = [&](auto x_tag) {
    constexpr int X = decltype(x_tag)::value;
    if constexpr (X < T::kRegA) {
      load_a(std::integral_constant<int, 0>{}, x_tag);
    } else if constexpr (X < T::kRegA + T::kRegB) {
      constexpr int q = X - T::kRegA;
      const int region = wave * T::kRegB + q;
      dma16(base_b, row_b[q] + (region & 1 ? col[1] : col[0]),
            lds + (uint32_t)(T::kOffB + cur_slot * T::kSlotB + region * 1024));
    } else if constexpr (X == T::kRegA + T::kRegB) {
      dma4(scale_a, (uint32_t)(lane * 4),
           lds + (uint32_t)(T::kOffScaleA + cur_slot * T::kScaleA + wave * 256));
    } else {
      dma4(scale_b, (uint32_t)(lane * 4),
           lds + (uint32_t)(T::kOffScaleB + cur_slot * T::kScaleB + wave * 256));
    }
  };
  if (cur_tile >= total_tiles) return;
  // the first two slices
  begin_cursor();
  static_for<0, T::kLoadsEarly>([&](auto x) { load_early(x); });
  static_for<0, T::kRegA>([&](auto q) { load_a(std::integral_constant<int, 1>{}, q); });
  next_slice();
  if (cur_left == 0) next_tile();
  static_for<0, T::kLoadsEarly>([&](auto x) { load_early(x); });

  u32x4 a0[kHalf], a1[kHalf], b0[TN], b1[TN];
  u32x2 sa[TM / 4], sb[1], sa_next[TM / 4], sb_next[1];
  int slot = 0;

  // the reads of a phase, in the order the next phase uses them
  auto read_a = [&](auto half_tag, uint32_t addr, u32x4(&dst)[kHalf], auto i_tag) {
    constexpr int h = decltype(half_tag)::value, i = decltype(i_tag)::value;
    read16<(h * kHalf + i) * 16 * kSliceBytes>(addr, dst[i]);
  };
  auto read_b = [&](uint32_t addr, u32x4(&dst)[TN], auto j_tag) {
    constexpr int j = decltype(j_tag)::value;
    read16<j * 16 * kSliceBytes>(addr, dst[j]);
  };
  constexpr int kNextReads = kHalf + TN + TM / 4 + 1;
  auto read_next = [&](uint32_t aa, uint32_t ba, uint32_t ssa, uint32_t ssb, auto r_tag) {
    constexpr int R = decltype(r_tag)::value;
    if constexpr (R < TM / 4) read8<R * kUnitBytes>(ssa, sa_next[R]);
    else if constexpr (R == TM / 4) read8<0>(ssb, sb_next[0]);
    else if constexpr (R == TM / 4 + 1) read_b(ba, b0, std::integral_constant<int, 0>{});
    else if constexpr (R < TM / 4 + 2 + kHalf) read_a(std::integral_constant<int, 0>{}, aa, a0, std::integral_constant<int, R - TM / 4 - 2>{});
    else read_b(ba, b0, std::integral_constant<int, R - TM / 4 - 1 - kHalf>{});
  };
  auto pin = [] { __builtin_amdgcn_sched_barrier(0); };

  // what the last phase of a slice does for the first one: lines landed, everyone agrees, reads
  wait_vmcnt<T::kLoads>();
  __builtin_amdgcn_s_barrier();
  static_for<0, T::kRegA>([&](auto q) { load_a(std::integral_constant<int, 1>{}, q); });
  next_slice();
  if (cur_left == 0) next_tile();
  static_for<0, kNextReads>([&](auto r) { read_next(lds + rd_a0, lds + rd_b0, lds + rd_sa, lds + rd_sb, r); });
  wait_lds();
  settle(a0);
  settle(b0);
  settle(sa_next);
  settle(sb_next);
#pragma unroll
  for (int i = 0; i < TM / 4; ++i) sa[i] = sa_next[i];
  sb[0] = sb_next[0];

  f32x4 acc[TM][TN];
  // matrix instruction X of a phase: n tile X / kHalf, m tile (half) kHalf + X % kHalf, step S
  auto mfma = [&](auto half_tag, auto step_tag, auto x_tag, const u32x4(&a)[kHalf], const u32x4(&b)[TN]) {
    constexpr int h = decltype(half_tag)::value, S = decltype(step_tag)::value, X = decltype(x_tag)::value;
    constexpr int j = X / kHalf, i = X % kHalf, it = h * kHalf + i;
    const uint32_t wa = (it & 2) ? sa[it / 4].y : sa[it / 4].x, wb = (j & 2) ? sb[0].y : sb[0].x;
    acc[it][j] = mfma_fp4<(j & 1) * 2 + S, (it & 1) * 2 + S>(b[j], a[i], acc[it][j], wb, wa);
  };
  using C0 = std::integral_constant<int, 0>;
  using C1 = std::integral_constant<int, 1>;

  for (int tile = blockIdx.x; tile < total_tiles; tile += gridDim.x) {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    // Slices up to the one after which the cursor goes to its next tile, that, and the others: the loop over
    // slices has no branch in it, behind which the compiler would gather the matrix instructions.
    for (int todo = slices; todo > 0;) {
     const int run = cur_left < todo ? cur_left : todo;
     todo -= run;
     for (int s = 0; s < run; ++s) {
      const uint32_t at_a = lds + (uint32_t)(slot * T::kSlotA) + rd_a0, at_b = lds + (uint32_t)(slot * T::kSlotB) + rd_b0;
      // ---- phase 0: lower half, step 0; reads for phase 1
      pin();
      static_for<0, NM>([&](auto x) {
        constexpr int X = decltype(x)::value;
        mfma(C0{}, C0{}, x, a0, b0);
        pin();
        static_for<0, kHalf + TN>([&](auto r) {
          constexpr int R = decltype(r)::value;
          if constexpr (place(R, kHalf + TN, NM) == X) {
            if constexpr (R == 0) read_b(at_b ^ 16u, b1, C0{});
            else if constexpr (R <= kHalf) read_a(C0{}, at_a ^ 16u, a1, std::integral_constant<int, R - 1>{});
            else read_b(at_b ^ 16u, b1, std::integral_constant<int, R - kHalf>{});
          }
        });
        pin();
      });
      wait_lds();
      settle(a1);
      settle(b1);
      pin();
      // ---- phase 1: lower half, step 1.  The upper half of A has landed; the slot's lower half and B are read
      static_for<0, NM>([&](auto x) {
        constexpr int X = decltype(x)::value;
        mfma(C0{}, C1{}, x, a1, b1);
        pin();
        if constexpr (X == 0) {
          wait_vmcnt<T::kLoads>();   // younger than this slice's late loads: all of the next slice's
          __builtin_amdgcn_s_barrier();
          pin();
        }
        constexpr int N = kHalf + T::kLoadsEarly;
        static_for<0, N>([&](auto r) {
          constexpr int R = decltype(r)::value;
          if constexpr (place(R, N, NM) == X) {
            if constexpr (R < kHalf) read_a(C1{}, at_a, a0, std::integral_constant<int, R>{});
            else load_early(std::integral_constant<int, R - kHalf>{});
          }
        });
        pin();
      });
      wait_lds();
      settle(a0);
      pin();
      // ---- phase 2: upper half, step 0; reads for phase 3
      static_for<0, NM>([&](auto x) {
        constexpr int X = decltype(x)::value;
        mfma(C1{}, C0{}, x, a0, b0);
        pin();
        if constexpr (X < kHalf) read_a(C1{}, at_a ^ 16u, a1, x);
        pin();
      });
      wait_lds();
      settle(a1);
      pin();
      // ---- phase 3: upper half, step 1.  The next slice's lower half, B and scales have landed
      slot ^= 1;
      const uint32_t na = lds + (uint32_t)(slot * T::kSlotA) + rd_a0, nb = lds + (uint32_t)(slot * T::kSlotB) + rd_b0;
      const uint32_t nsa = lds + (uint32_t)(slot * T::kScaleA) + rd_sa, nsb = lds + (uint32_t)(slot * T::kScaleB) + rd_sb;
      static_for<0, NM>([&](auto x) {
        constexpr int X = decltype(x)::value;
        mfma(C1{}, C1{}, x, a1, b1);
        pin();
        if constexpr (X == 0) {
          wait_vmcnt<T::kLoads>();   // younger than the next slice's early loads: its late ones, the early ones behind them
          __builtin_amdgcn_s_barrier();
          pin();
        }
        constexpr int N = kNextReads + T::kRegA;
        static_for<0, N>([&](auto r) {
          constexpr int R = decltype(r)::value;
          if constexpr (place(R, N, NM) == X) {
            if constexpr (R < kNextReads) read_next(na, nb, nsa, nsb, r);
            else load_a(C1{}, std::integral_constant<int, R - kNextReads>{});
          }
        });
        pin();
      });
      wait_lds();
      settle(a0);
      settle(b0);
      settle(sa_next);
      settle(sb_next);
#pragma unroll
      for (int i = 0; i < TM / 4; ++i) sa[i] = sa_next[i];
      sb[0] = sb_next[0];
      pin();
      next_slice();
     }
     if (cur_left == 0) next_tile();
    }

    // ---- the tile's output: bias, slope, rounding; through the wave's staging rows as whole lines ----
    int tm, tn;
    map_tile(tile, tiles_m, tiles_n, tm, tn);
    const int m0 = tm * T::kBM + wm * TM * 16, n0 = tn * T::kBN + wn * TN * 16;
    constexpr int kSize = KIND == kElemF32 ? 4 : 2;
    constexpr int kJ = kSize == 4 ? 2 : 4;          // n tiles of a staged line
    unsigned char *const stage = smem + T::kOffStage + wave * T::kStageBytes;
    // the lane number again, opaque to the compiler, so that what follows is computed here and not
    // kept through the slices
    int lane_e;
    asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(lane_e));
    const int lie = lane_e & 15, ge = lane_e >> 4;
    float bias[TN][4];
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int n = n0 + j * 16 + 4 * ge + e;
        bias[j][e] = p.bias && n < p.n ? Elem<KIND>::load(p.bias, n) : -0.f;   // -0: the identity of the add
      }
    static_for<0, TM>([&](auto i_tag) {
      constexpr int i = decltype(i_tag)::value;
      static_for<0, TN / kJ>([&](auto jh_tag) {
        constexpr int jh = decltype(jh_tag)::value;
        static_for<0, kJ>([&](auto jj_tag) {
          constexpr int jj = decltype(jj_tag)::value, j = jh * kJ + jj;
          float v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            v[e] = acc[i][j][e] + bias[j][e];
            v[e] = fmaxf(v[e], v[e] * p.alpha);
          }
          // row lie of the staged 16, bytes (jj * 16 + 4 ge) * kSize of its line
          if constexpr (kSize == 4) {
            const int chunk = (jj * 4 + ge) ^ (lie & 7);
            *reinterpret_cast<f32x4 *>(stage + lie * 128 + chunk * 16) = f32x4{v[0], v[1], v[2], v[3]};
          } else {
            uint32_t w[2];
            Elem<KIND>::pack(v, w);
            const int chunk = (jj * 2 + (ge >> 1)) ^ (lie & 7);
            *reinterpret_cast<u32x2 *>(stage + lie * 128 + chunk * 16 + (ge & 1) * 8) = u32x2{w[0], w[1]};
          }
        });
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int r = q * 8 + (lane_e >> 3), c = lane_e & 7;
          const u32x4 line = *reinterpret_cast<const u32x4 *>(stage + r * 128 + ((c ^ (r & 7)) * 16));
          const int m = m0 + i * 16 + r, n = n0 + jh * kJ * 16 + c * (16 / kSize);
          if (m < p.m && n < p.n) {
            typedef typename Elem<KIND>::type E;
            E *const o = static_cast<E *>(p.out) + (int64_t)m * p.n + n;
            if (n + 16 / kSize <= p.n) {
              __builtin_nontemporal_store(line, reinterpret_cast<u32x4_u *>(o));
            } else {
              const uint32_t w[4] = {line.x, line.y, line.z, line.w};
#pragma unroll
              for (int e = 0; e < 16 / kSize - 1; ++e)
                if (n + e < p.n) {
                  if constexpr (kSize == 4) o[e] = __uint_as_float(w[e]);
                  else o[e] = (uint16_t)(w[e / 2] >> (16 * (e & 1)));
                }
            }
          }
        }
      });
    });
  }
  wait_vmcnt<0>();   // the cursor's last requests still write this workgroup's LDS
}

template <int WM, int WN, int TM, int TN, int KIND>
LaunchStatus tiles_launch(const MxOperands &p, const unsigned char *scales, int units_a, int units_b, int slices,
                          int per_cu, uint32_t block_dim, hipStream_t stream) {
  using T = Tile<WM, WN, TM, TN>;
  const int tiles_m = (p.m + T::kBM - 1) / T::kBM, tiles_n = (p.n + T::kBN - 1) / T::kBN;
  int64_t blocks = (int64_t)tiles_m * tiles_n;
  if (blocks > 0x7fffffff) return invalid("mxfp4_matmul: too many output tiles");
  const int64_t most = (int64_t)device_cus() * per_cu;
  if (blocks > most) blocks = most;
  if (block_dim) blocks = block_dim;
  AFIR_LAUNCH("mxfp4_matmul_tiles", (mxfp4_matmul_tiles<WM, WN, TM, TN, KIND>), dim3((unsigned)blocks),
              dim3(T::kWaves * 64), 0, stream, p, scales, units_a, units_b, slices, tiles_m, tiles_n);
  return after_launch();
}

template <int KIND>
LaunchStatus tiles(const MxOperands &p, void *workspace, uint32_t block_dim, hipStream_t stream) {
  const int slices = (int)slices_of(p.kb), units_a = (int)scale_units(p.m), units_b = (int)scale_units(p.n);
  const int turns = (slices + kTurnSlices - 1) / kTurnSlices;
  const int64_t items = (int64_t)(units_a + units_b) * turns, most = (int64_t)1 << 20;
  AFIR_LAUNCH("mxfp4_arrange_scales", mxfp4_arrange_scales, dim3((unsigned)(items < most ? items : most)), dim3(256), 0,
              stream, p, units_a, units_b, slices, turns, static_cast<unsigned char *>(workspace));
  const LaunchStatus st = after_launch();
  if (st.code) return st;
  const unsigned char *const scales = static_cast<const unsigned char *>(workspace);
  const int64_t large = (int64_t)((p.m + 255) / 256) * ((p.n + 255) / 256);
  if (large >= device_cus())
    return tiles_launch<2, 4, 8, 4, KIND>(p, scales, units_a, units_b, slices, 1, block_dim, stream);
  return tiles_launch<2, 2, 4, 4, KIND>(p, scales, units_a, units_b, slices, 2, block_dim, stream);
}

}  // namespace

bool mxfp4_dma_supported(const MxOperands &p) {
  // the offset of a lane's line from its tile's first row has 32 bits
  return p.m > 64 && p.kb > 0 && (int64_t)p.kb * kMxBlockBytes * 256 < (int64_t)1 << 32;
}

size_t mxfp4_dma_workspace(int64_t m, int64_t kb, int64_t n) {
  return (size_t)((scale_units(m) + scale_units(n)) * slices_of(kb) * kUnitBytes);
}

LaunchStatus launch_mxfp4_dma(const MxOperands &p, int elem_kind, void *workspace, uint32_t block_dim, hipStream_t stream) {
  switch (elem_kind) {
    case kElemF32: return tiles<kElemF32>(p, workspace, block_dim, stream);
    case kElemF16: return tiles<kElemF16>(p, workspace, block_dim, stream);
    default: return tiles<kElemBF16>(p, workspace, block_dim, stream);
  }
}

}  // namespace afir
