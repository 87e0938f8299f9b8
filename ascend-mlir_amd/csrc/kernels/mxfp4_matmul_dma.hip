// MXFP4 products of more than a few rows: tiles in LDS, the matrix cores fed from there.
//
// A K slice is 256 numbers: one 128-byte line of every row of A and B.  Lines are copied global ->
// LDS directly (global_load_lds, 16 bytes per lane, no registers in between) into two slots each;
// the 16-byte chunk c of row r lands at chunk position c ^ ((r >> 1) & 7).  Lane group g of a
// wavefront takes chunks g and 4 + g of a line, i.e. blocks g and 4 + g of the slice, in its two
// steps of 128: with that the operand reads (ds_read_b128) are free of bank conflicts, with 2g and
// 2g + 1 half of the LDS cycles were conflicts.
//
// A slice is four phases: the lower half of a wave's m tiles with the first and the second step,
// then the upper half with both.  Operands are read one phase ahead, so the lower half of the A
// slot and all of the B slot are free after the first phase and are refilled from the second on,
// the upper half of A from the fourth: a line has a slice and a half to arrive, and a barrier
// every two phases says both that what comes next has landed and that what goes next has been
// read.  The refills walk ahead of the products across tile boundaries, so nothing drains between
// the tiles of a workgroup; only the output passes in between.  Every operand read and every load sits behind a matrix instruction (pinned with
// scheduling barriers), as in matmul_dma_kernel.h.
//
// Rows past the end of A or B repeat the last row.  A last slice that is not whole starts early, so
// that it ends with the row; the scales that go with the blocks it repeats are 2^-127 on both sides,
// and their products vanish in float32.
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
// The lane number, opaque to the compiler: what is computed from it is computed where it stands, once
// per tile, and not kept in registers (or scratch memory, whose accesses would wait for every load in
// flight) through the slices.
__device__ __forceinline__ int lane_here() {
  int lane;
  asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(lane));
  return lane;
}
// lanes 16 .. 31 and 48 .. 63 of `a` and lanes 0 .. 15 and 32 .. 47 of `b` change places
__device__ __forceinline__ u32x2 swap_odd_even(uint32_t a, uint32_t b) {
  const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
  return u32x2{(uint32_t)r[0], (uint32_t)r[1]};
}
// of every 16 lanes: x in lanes 0 .. 7, y of those lanes in lanes 8 .. 15
__device__ __forceinline__ uint32_t exchange_high(uint32_t x, uint32_t y) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)y, 0x128, 0xf, 0xc, false);   // row_ror:8, lanes 8 .. 15
}
// ... x of lanes 8 .. 15 in lanes 0 .. 7, y in lanes 8 .. 15
__device__ __forceinline__ uint32_t exchange_low(uint32_t x, uint32_t y) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)y, (int)x, 0x128, 0xf, 0x3, false);   // row_ror:8, lanes 0 .. 7
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

// item R of N goes behind matrix instruction place(R, N, NM) of NM; reads (the first `reads`) one after
// the other, loads two instructions apart where there is room
constexpr int place(int r, int n, int nm, int reads) {
  return n > nm ? r * nm / n : r < reads || reads + 2 * (n - reads) > nm ? r : reads + 2 * (r - reads);
}

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
// unit, blocks g and 4 + g of the slice.  A's units first, then B's.  A workgroup turns a unit's rows
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
      const int lane = i & 63, ds = i >> 6, slice = s0 + ds, g = lane >> 4;
      if (slice < slices) {
        // a last slice that starts `early` blocks early: those get 2^-127
        const int early = (slice + 1) * kSliceBlocks > p.kb ? (slice + 1) * kSliceBlocks - p.kb : 0;
        const unsigned char *const from = tile + (lane & 15) * kTurnPitch + ds * kSliceBlocks + g - early;
        uint32_t w[4];
#pragma unroll
        for (int t = 0; t < 4; ++t)
          w[t] = (g >= early ? (uint32_t)from[t * 16 * kTurnPitch] : 0u) |
                 (g + 4 >= early ? (uint32_t)from[t * 16 * kTurnPitch + 4] << 8 : 0u);
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
  static constexpr int kScaleA = kBM * kSliceBlocks, kScale = kScaleA + kBN * kSliceBlocks;   // A's units, then B's
  static constexpr int kOffB = 2 * kSlotA, kOffScale = kOffB + 2 * kSlotB;
  static constexpr int kLds = kOffScale + 2 * kScale;
  static constexpr int kHalf = TM / 2;
  // direct-to-LDS loads of a wave per slice: regions of 1 KiB (8 rows) of half of A and of B, and the
  // wave's share of the scales, one load of 16 bytes per lane or two of 4
  static constexpr int kRegA = kBM / 2 / 8 / kWaves, kRegB = kBN / 8 / kWaves;
  static constexpr int kScaleShare = kScale / kWaves, kScaleLoads = kScaleShare == 1024 ? 1 : 2;
  static constexpr int kLoadsEarly = kRegA + kRegB + kScaleLoads, kLoads = kLoadsEarly + kRegA;
  static_assert(TM % 4 == 0 && TN % 4 == 0, "scales are read for four tiles at a time");
  static_assert(kRegA * kWaves * 16 == kBM && kRegB * kWaves * 8 == kBN, "whole regions per wave");
  static_assert(kScaleShare == 1024 || kScaleShare == 512, "one 16-byte load per lane or two of 4");
  static_assert(kScaleA % kScaleShare == 0, "a wave's share is of one operand");
};

template <int WM, int WN, int TM, int TN, int KIND>
__global__ __launch_bounds__(WM *WN * 64, 2) void mxfp4_matmul_tiles(MxOperands p, const unsigned char *__restrict__ scales,
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

  // ---- operand reads: lane l reads row l % 16 of a tile, chunk l / 16 + 4 step ----
  const uint32_t swz = (uint32_t)((li >> 1) & 7);
  const uint32_t rd_a0 = (uint32_t)((wm * TM * 16 + li) * kSliceBytes) + (g ^ swz) * 16;   // step 1: ^ 64
  const uint32_t rd_b0 = (uint32_t)(T::kOffB + (wn * TN * 16 + li) * kSliceBytes) + (g ^ swz) * 16;
  const uint32_t rd_sa = (uint32_t)(T::kOffScale + wm * (TM / 4) * kUnitBytes + lane * 8);
  const uint32_t rd_sb = (uint32_t)(T::kOffScale + T::kScaleA + wn * (TN / 4) * kUnitBytes + lane * 8);

  // ---- the cursor: tile and slice whose lines are requested next ----
  // A load's source is a wave-uniform base (the tile's first row at the slice's first column) plus a
  // per-lane offset (row and chunk) that is kept per region.
  int cur_tile = blockIdx.x, cur_slice = 0, cur_slot = 0;
  const unsigned char *base_a = nullptr, *base_b = nullptr, *base_s = nullptr;   // of the tile
  const unsigned char *at_a = nullptr, *at_b = nullptr, *at_s = nullptr;         // ... at the slice
  const bool scales_of_a = wave * T::kScaleShare < T::kScaleA;
  const int64_t scale_step = (int64_t)(scales_of_a ? units_a : units_b) * kUnitBytes;
  uint32_t off_a[2 * T::kRegA], off_b[T::kRegB];
  // region q of a half of A: rows of the half's m tiles, one wave row after the other
  auto region_row_a = [&](int half, int q) {
    const int region = wave * T::kRegA + q;                     // of the half's regions
    constexpr int per_wm = kHalf * 2;                           // regions of a wave row's half
    return (region / per_wm) * TM * 16 + half * kHalf * 16 + (region % per_wm) * 8;
  };
  // the offset of this lane's 16 bytes: row and chunk of the region that starts at `row` of the tile
  auto lane_offset = [&](int lane_c, int row, int last) {
    const int r = row + (lane_c >> 3), chunk = (lane_c & 7) ^ ((r >> 1) & 7);
    return (uint32_t)(r < last ? r : last) * pitch + (uint32_t)(chunk * 16);
  };
  auto set_slice = [&]() {
    // the last slice of a row that is no whole number of them starts early enough to end with the row;
    // the blocks it has in common with the one before it come with scales that take them out
    const uint32_t at = (uint32_t)cur_slice * kSliceBytes;
    const uint32_t column = at < pitch - kSliceBytes ? at : pitch - kSliceBytes;
    at_a = base_a + column;
    at_b = base_b + column;
    at_s = base_s + (int64_t)cur_slice * scale_step;
  };
  auto begin_cursor = [&]() {
    int tm, tn;
    map_tile(cur_tile, tiles_m, tiles_n, tm, tn);
    const int m0 = tm * T::kBM, n0 = tn * T::kBN;
    base_a = p.a + (int64_t)m0 * pitch;
    base_b = p.b + (int64_t)n0 * pitch;
    base_s = scales + (scales_of_a ? (int64_t)m0 * kSliceBlocks + wave * T::kScaleShare
                                   : ((int64_t)units_a * slices * kUnitRows + n0) * kSliceBlocks +
                                         (wave * T::kScaleShare - T::kScaleA));
    const int lane_c = lane_here();
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int q = 0; q < T::kRegA; ++q) off_a[h * T::kRegA + q] = lane_offset(lane_c, region_row_a(h, q), p.m - 1 - m0);
#pragma unroll
    for (int q = 0; q < T::kRegB; ++q) off_b[q] = lane_offset(lane_c, (wave * T::kRegB + q) * 8, p.n - 1 - n0);
    // all tiles walk K from its start: workgroups of one XCD that share rows then ask for the same lines
    // at about the same time.  (Starting each tile at another slice, to spread the requests over the
    // memory channels, measured 4 % slower at 8192^3.)
    cur_slice = 0;
    set_slice();
  };
  auto next_slice = [&]() {
    cur_slot ^= 1;
    ++cur_slice;
    set_slice();
  };
  auto next_tile = [&]() {   // when cur_slice has come to the end
    // past the last tile the cursor walks that tile again: what it requests then is not read, and
    // the slices need no other form for the end
    if (cur_tile + (int)gridDim.x < total_tiles) cur_tile += gridDim.x;
    begin_cursor();
  };
  // 16 (4) bytes per lane, one after the other from `to` + OFF
  auto dma16 = [&](const unsigned char *base, uint32_t offset, uint32_t to, auto off_tag) {
    asm volatile("s_add_u32 m0, %0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 ::"s"(to), "v"(offset), "s"(base), "n"(decltype(off_tag)::value) : "memory", "scc");
  };
  auto dma4 = [&](const unsigned char *base, uint32_t offset, uint32_t to, auto off_tag) {
    asm volatile("s_add_u32 m0, %0, %3\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2"
                 ::"s"(to), "v"(offset), "s"(base), "n"(decltype(off_tag)::value) : "memory", "scc");
  };
  // LDS addresses of this wave's first region of each half of A, of B and of its scales, in slot 0
  constexpr int kRun = kHalf * 2;   // regions of a half that follow one another
  static_assert(kRun % T::kRegA == 0, "a wave's regions of a half are adjacent");
  const uint32_t to_a = lds + (uint32_t)(region_row_a(0, 0) * kSliceBytes);
  const uint32_t to_b = lds + (uint32_t)(T::kOffB + wave * T::kRegB * 1024);
  const uint32_t to_s = lds + (uint32_t)(T::kOffScale + wave * T::kScaleShare);
  auto load_a = [&](auto half_tag, auto q_tag) {
    constexpr int h = decltype(half_tag)::value, q = decltype(q_tag)::value;
    dma16(at_a, off_a[h * T::kRegA + q], to_a + (uint32_t)(cur_slot * T::kSlotA),
          std::integral_constant<int, h * kHalf * 16 * kSliceBytes + q * 1024>{});
  };
  // loads 0 .. kLoadsEarly - 1 of a slice: the lower half of A, B, the scales
  auto load_early = [&](auto x_tag) {
    constexpr int X = decltype(x_tag)::value;
    if constexpr (X < T::kRegA) {
      load_a(std::integral_constant<int, 0>{}, x_tag);
    } else if constexpr (X < T::kRegA + T::kRegB) {
      constexpr int q = X - T::kRegA;
      dma16(at_b, off_b[q], to_b + (uint32_t)(cur_slot * T::kSlotB), std::integral_constant<int, q * 1024>{});
    } else if constexpr (T::kScaleLoads == 1) {
      dma16(at_s, (uint32_t)(lane * 16), to_s + (uint32_t)(cur_slot * T::kScale), std::integral_constant<int, 0>{});
    } else {
      constexpr int part = X - T::kRegA - T::kRegB;
      dma4(at_s, (uint32_t)(lane * 4 + part * 256), to_s + (uint32_t)(cur_slot * T::kScale),
           std::integral_constant<int, part * 256>{});
    }
  };

  if (cur_tile >= total_tiles) return;
  // the first two slices
  begin_cursor();
  static_for<0, T::kLoadsEarly>([&](auto x) { load_early(x); });
  static_for<0, T::kRegA>([&](auto q) { load_a(std::integral_constant<int, 1>{}, q); });
  next_slice();
  if (cur_slice == slices) next_tile();
  static_for<0, T::kLoadsEarly>([&](auto x) { load_early(x); });

  u32x4 a0[kHalf], a1[kHalf], b0[TN], b1[TN];
  u32x2 sa[TM / 4], sb[TN / 4], sa_next[TM / 4], sb_next[TN / 4];
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
  constexpr int kScaleReads = TM / 4 + TN / 4, kNextReads = kHalf + TN + kScaleReads;
  auto read_next = [&](uint32_t aa, uint32_t ba, uint32_t ssa, uint32_t ssb, auto r_tag) {
    constexpr int R = decltype(r_tag)::value;
    if constexpr (R < TM / 4) read8<R * kUnitBytes>(ssa, sa_next[R]);
    else if constexpr (R < kScaleReads) read8<(R - TM / 4) * kUnitBytes>(ssb, sb_next[R - TM / 4]);
    else if constexpr (R == kScaleReads) read_b(ba, b0, std::integral_constant<int, 0>{});
    else if constexpr (R <= kScaleReads + kHalf) read_a(std::integral_constant<int, 0>{}, aa, a0, std::integral_constant<int, R - kScaleReads - 1>{});
    else read_b(ba, b0, std::integral_constant<int, R - kScaleReads - kHalf>{});
  };
  auto pin = [] { __builtin_amdgcn_sched_barrier(0); };

  // what the last phase of a slice does for the first one: lines landed, everyone agrees, reads
  wait_vmcnt<T::kLoads>();
  __builtin_amdgcn_s_barrier();
  static_for<0, T::kRegA>([&](auto q) { load_a(std::integral_constant<int, 1>{}, q); });
  next_slice();
  if (cur_slice == slices) next_tile();
  static_for<0, kNextReads>([&](auto r) { read_next(lds + rd_a0, lds + rd_b0, lds + rd_sa, lds + rd_sb, r); });
  wait_lds();
  settle(a0);
  settle(b0);
  settle(sa_next);
  settle(sb_next);
#pragma unroll
  for (int i = 0; i < TM / 4; ++i) sa[i] = sa_next[i];
#pragma unroll
  for (int j = 0; j < TN / 4; ++j) sb[j] = sb_next[j];

  f32x4 acc[TM][TN];
  // matrix instruction X of a phase: n tile X / kHalf, m tile (half) kHalf + X % kHalf, step S
  auto mfma = [&](auto half_tag, auto step_tag, auto x_tag, const u32x4(&a)[kHalf], const u32x4(&b)[TN]) {
    constexpr int h = decltype(half_tag)::value, S = decltype(step_tag)::value, X = decltype(x_tag)::value;
    constexpr int j = X / kHalf, i = X % kHalf, it = h * kHalf + i;
    const uint32_t wa = (it & 2) ? sa[it / 4].y : sa[it / 4].x, wb = (j & 2) ? sb[j / 4].y : sb[j / 4].x;
    acc[it][j] = mfma_fp4<(j & 1) * 2 + S, (it & 1) * 2 + S>(b[j], a[i], acc[it][j], wb, wa);
  };
  using C0 = std::integral_constant<int, 0>;
  using C1 = std::integral_constant<int, 1>;

  constexpr int kSize = KIND == kElemF32 ? 4 : 2;
  // The bias of a lane's columns (four adjacent ones of n tile j), as stored; -0 where there is none (the
  // identity of the add).  It comes through the scalar cache: a vector load would have to wait for every
  // line that was requested before it.
  auto bias_of = [&](int n0, auto j_tag, uint32_t(&w)[kSize]) {
    constexpr int j = decltype(j_tag)::value, kWords = 16 * kSize / 4;
    const int ge = lane_here() >> 4;
#pragma unroll
    for (int e = 0; e < kSize; ++e) w[e] = kSize == 4 ? 0x80000000u : 0x80008000u;
    if (!p.bias) return;
    if (n0 + TN * 16 <= p.n && (reinterpret_cast<uintptr_t>(p.bias) & 3u) == 0) {
      typedef const __attribute__((address_space(4))) uint32_t *ScalarWords;
      const ScalarWords q = (ScalarWords)(reinterpret_cast<uintptr_t>(p.bias) + (uintptr_t)(n0 + j * 16) * kSize);
#pragma unroll
      for (int e = 0; e < kSize; ++e) {
        const uint32_t low = (ge & 1) ? q[kWords / 4 + e] : q[e];
        const uint32_t high = (ge & 1) ? q[3 * kWords / 4 + e] : q[kWords / 2 + e];
        w[e] = (ge & 2) ? high : low;
      }
    } else {
      const int n = n0 + j * 16 + 4 * ge;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < p.n) {
          if constexpr (kSize == 4) {
            w[e] = static_cast<const uint32_t *>(p.bias)[n + e];
          } else {
            const uint32_t one = static_cast<const uint16_t *>(p.bias)[n + e];
            w[e / 2] = e & 1 ? (w[e / 2] & 0xffffu) | one << 16 : (w[e / 2] & 0xffff0000u) | one;
          }
        }
    }
  };

  for (int tile = blockIdx.x; tile < total_tiles; tile += gridDim.x) {
    int tm, tn;
    map_tile(tile, tiles_m, tiles_n, tm, tn);
    const int m0 = tm * T::kBM + wm * TM * 16, n0 = tn * T::kBN + wn * TN * 16;   // the wave's part of the tile
    static_for<0, TN>([&](auto j_tag) {   // the sums start from the bias
      constexpr int j = decltype(j_tag)::value;
      uint32_t w[kSize];
      float b[4];
      bias_of(n0, j_tag, w);
      Elem<KIND>::unpack(w, b);
#pragma unroll
      for (int i = 0; i < TM; ++i) acc[i][j] = f32x4{b[0], b[1], b[2], b[3]};
    });
    // One slice, in which no branch may stand: behind one the compiler would gather the matrix instructions.
    auto slice = [&]() {
      const uint32_t here_a = lds + (uint32_t)(slot * T::kSlotA) + rd_a0, here_b = lds + (uint32_t)(slot * T::kSlotB) + rd_b0;
      // ---- phase 0: lower half, step 0; reads for phase 1
      pin();
      static_for<0, NM>([&](auto x) {
        constexpr int X = decltype(x)::value;
        mfma(C0{}, C0{}, x, a0, b0);
        pin();
        static_for<0, kHalf + TN>([&](auto r) {
          constexpr int R = decltype(r)::value;
          if constexpr (place(R, kHalf + TN, NM, kHalf + TN) == X) {
            if constexpr (R == 0) read_b(here_b ^ 64u, b1, C0{});
            else if constexpr (R <= kHalf) read_a(C0{}, here_a ^ 64u, a1, std::integral_constant<int, R - 1>{});
            else read_b(here_b ^ 64u, b1, std::integral_constant<int, R - kHalf>{});
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
          if constexpr (place(R, N, NM, kHalf) == X) {
            if constexpr (R < kHalf) read_a(C1{}, here_a, a0, std::integral_constant<int, R>{});
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
        if constexpr (X < kHalf) read_a(C1{}, here_a ^ 64u, a1, x);
        pin();
      });
      wait_lds();
      settle(a1);
      pin();
      // ---- phase 3: upper half, step 1.  The next slice's lower half, B and scales have landed
      slot ^= 1;
      const uint32_t na = lds + (uint32_t)(slot * T::kSlotA) + rd_a0, nb = lds + (uint32_t)(slot * T::kSlotB) + rd_b0;
      const uint32_t nsa = lds + (uint32_t)(slot * T::kScale) + rd_sa, nsb = lds + (uint32_t)(slot * T::kScale) + rd_sb;
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
          if constexpr (place(R, N, NM, kNextReads) == X) {
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
#pragma unroll
      for (int j = 0; j < TN / 4; ++j) sb[j] = sb_next[j];
      pin();
      next_slice();
    };
    // slices up to the one after which the cursor goes to its next tile, and from there on
    int todo = slices;
    while (todo > 0) {
      const int run = slices - cur_slice < todo ? slices - cur_slice : todo;
      todo -= run;
      for (int s = 0; s < run; ++s) slice();
      if (cur_slice == slices) next_tile();
    }

    // ---- the tile's output: slope, rounding, stores ----
    // A lane holds four adjacent columns (4 ge ..) of row lie of every 16 x 16 tile: 16 bytes in 32 bits.
    // In 16 bits two n tiles first exchange halves between lanes 16 apart, after which a lane has eight
    // adjacent columns of one of them.  Either way four lanes hold 64 adjacent bytes of a row, and two
    // such sets are 128: they exchange rows 8 to 15 of the first for rows 0 to 7 of the second, so that a
    // store writes eight whole lines.  (With 64 bytes of sixteen rows per store the kernel took 15 % longer.)
    //
    // Tiles that lie inside the output as a whole (kInside) store without any test.
    const int lane_e = lane_here(), lie = lane_e & 15, ge = lane_e >> 4;
    typedef typename Elem<KIND>::type E;
    auto outputs = [&](auto slope_tag, auto inside_tag) {
      constexpr bool kSlope = decltype(slope_tag)::value, kInside = decltype(inside_tag)::value;
      E *row = static_cast<E *>(p.out) + (int64_t)m0 * p.n + n0;   // wave-uniform
      constexpr int kSide = 64 / kSize;                            // columns of 64 bytes
      const int lane_col = (lie >> 3) * kSide + (kSize == 4 ? 4 * ge : (ge & 1) * 16 + (ge >> 1) * 8);
      const uint32_t lane_at = (uint32_t)((lie & 7) * p.n + lane_col);
      auto packed = [&](const f32x4 &c, uint32_t(&w)[kSize]) {
        float v[4] = {c[0], c[1], c[2], c[3]};
        if constexpr (kSlope) {
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = fmaxf(v[e], v[e] * p.alpha);
        }
        Elem<KIND>::pack(v, w);
      };
      // 16 bytes at row m0 + r + lie % 8, column n0 + at + the lane's; `row` points to row m0 + r
      auto store = [&](int r, int at, u32x4 w) {
        E *const o = row + at + lane_at;
        if constexpr (kInside) {
          __builtin_nontemporal_store(w, reinterpret_cast<u32x4_u *>(o));
        } else {
          const int n = n0 + at + lane_col;
          if (m0 + r + (lie & 7) >= p.m || n >= p.n) return;
          if (n + 16 / kSize <= p.n) {
            __builtin_nontemporal_store(w, reinterpret_cast<u32x4_u *>(o));
          } else {
            const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int e = 0; e < 16 / kSize - 1; ++e)
              if (n + e < p.n) {
                if constexpr (kSize == 4) o[e] = __uint_as_float(v[e]);
                else o[e] = (uint16_t)(v[e / 2] >> (16 * (e & 1)));
              }
          }
        }
      };
      // `sets` of two times 64 bytes of a row: X and Y
      auto both = [&](int r, int at, u32x4 x, u32x4 y) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t first = exchange_high(x[e], y[e]), second = exchange_low(x[e], y[e]);
          x[e] = first;
          y[e] = second;
        }
        store(r, at, x);
        row += (int64_t)8 * p.n;
        store(r + 8, at, y);
        row -= (int64_t)8 * p.n;
      };
      static_for<0, TM>([&](auto i_tag) {
        constexpr int i = decltype(i_tag)::value;
        if constexpr (kSize == 4) {
          static_for<0, TN / 2>([&](auto j_tag) {
            constexpr int j = 2 * decltype(j_tag)::value;
            uint32_t w0[4], w1[4];
            packed(acc[i][j], w0);
            packed(acc[i][j + 1], w1);
            both(i * 16, j * 16, u32x4{w0[0], w0[1], w0[2], w0[3]}, u32x4{w1[0], w1[1], w1[2], w1[3]});
          });
        } else {
          static_for<0, TN / 4>([&](auto j_tag) {
            constexpr int j = 4 * decltype(j_tag)::value;
            u32x4 set[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t w0[2], w1[2];
              packed(acc[i][j + 2 * h], w0);
              packed(acc[i][j + 2 * h + 1], w1);
              // rows of 16 lanes: the odd ones of the first change places with the even ones of the second
              const u32x2 x = swap_odd_even(w0[0], w1[0]), y = swap_odd_even(w0[1], w1[1]);
              set[h] = u32x4{x.x, y.x, x.y, y.y};
            }
            both(i * 16, j * 16, set[0], set[1]);
          });
        }
        row += (int64_t)16 * p.n;
      });
    };
    const bool inside = m0 + TM * 16 <= p.m && n0 + TN * 16 <= p.n;   // of the wave's rows and columns
    if (!inside) outputs(std::true_type{}, std::false_type{});
    else if (p.alpha != 1.f) outputs(std::true_type{}, std::true_type{});
    else outputs(std::false_type{}, std::true_type{});
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
  return p.m > 64 && p.kb >= kSliceBlocks && (int64_t)p.kb * kMxBlockBytes * 256 < (int64_t)1 << 32;
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
