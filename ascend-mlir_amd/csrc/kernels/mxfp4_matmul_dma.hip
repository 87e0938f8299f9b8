// MXFP4 products of more output tiles than compute units: tiles in LDS, the matrix cores fed from there.
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
// the tiles of a workgroup; only the output passes in between.  Every operand read and every load sits
// behind a matrix instruction (pinned with scheduling barriers), as in matmul_dma_kernel.h.
//
// 8192 x 8192 x 8192 into bfloat16: 232 us, 4.7 PFLOP/s, 6 us of it the arranging of the scales.  With
// operands that are all alike it is 176 us (6.2 PFLOP/s): what bounds random ones is the power that the
// matrix cores draw (fed from registers alone they reach 7.4 PFLOP/s, 9.6 with constant operands).
//
// Rows past the end of A or B repeat the last row.  A last slice that is not whole starts early, so
// that it ends with the row; the scales that go with the blocks it repeats are 2^-127 on both sides,
// and their products vanish in float32.
//
// The scales are laid out beforehand (mxfp4_arrange_scales, into the workspace) so that the two
// bytes a lane needs of each of four 16-row tiles are adjacent: a wave reads its 128 x 8 scales of
// a slice with two 8-byte LDS reads, and they come into LDS with two small loads per wave.  Read as
// they are stored it would take twelve 2-byte reads.
#include "mxfp4_mfma.h"

namespace afir {

namespace {

// item R of N goes behind matrix instruction place(R, N, NM) of NM; reads (the first `reads`) one after
// the other, loads two instructions apart where there is room
constexpr int place(int r, int n, int nm, int reads) {
  return n > nm ? r * nm / n : r < reads || reads + 2 * (n - reads) > nm ? r : reads + 2 * (r - reads);
}

constexpr int kUnitRows = 64;             // rows whose scales of a slice are one piece of 512 bytes
constexpr int kUnitBytes = kUnitRows * kMxSliceBlocks;
constexpr int kUnitPad = 4;               // units are allotted in fours: the rows of the largest tile

inline int64_t scale_units(int64_t rows) {
  return (rows + kUnitRows * kUnitPad - 1) / (kUnitRows * kUnitPad) * kUnitPad;
}
inline int64_t slices_of(int64_t kb) { return (kb + kMxSliceBlocks - 1) / kMxSliceBlocks; }

// scales [rows][kb] -> [slice][unit][lane][4 tiles][2]: lane l = 16 g + r holds, of row 16 i + r of the
// unit, blocks g and 4 + g of the slice.  A's units first, then B's.  A workgroup turns a unit's rows
// of 16 slices (128 bytes each) in LDS, so that both sides move whole lines.
constexpr int kTurnSlices = 16, kTurnPitch = kTurnSlices * kMxSliceBlocks + 4;
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
      const int r = i >> 3, at = (i & 7) * 16, block = s0 * kMxSliceBlocks + at;
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
        const int early = (slice + 1) * kMxSliceBlocks > p.kb ? (slice + 1) * kMxSliceBlocks - p.kb : 0;
        const unsigned char *const from = tile + (lane & 15) * kTurnPitch + ds * kMxSliceBlocks + g - early;
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

// WM x WN wavefronts, each TM x TN tiles of 16 x 16.
template <int WM, int WN, int TM, int TN>
struct Tile {
  static constexpr int kWaves = WM * WN, kBM = WM * TM * 16, kBN = WN * TN * 16;
  static constexpr int kSlotA = kBM * kMxSliceBytes, kSlotB = kBN * kMxSliceBytes;
  static constexpr int kScaleA = kBM * kMxSliceBlocks, kScale = kScaleA + kBN * kMxSliceBlocks;   // A's units, then B's
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
  const uint32_t rd_a0 = (uint32_t)((wm * TM * 16 + li) * kMxSliceBytes) + (g ^ swz) * 16;   // step 1: ^ 64
  const uint32_t rd_b0 = (uint32_t)(T::kOffB + (wn * TN * 16 + li) * kMxSliceBytes) + (g ^ swz) * 16;
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
    const uint32_t at = (uint32_t)cur_slice * kMxSliceBytes;
    const uint32_t column = at < pitch - kMxSliceBytes ? at : pitch - kMxSliceBytes;
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
    base_s = scales + (scales_of_a ? (int64_t)m0 * kMxSliceBlocks + wave * T::kScaleShare
                                   : ((int64_t)units_a * slices * kUnitRows + n0) * kMxSliceBlocks +
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
  // LDS addresses of this wave's first region of each half of A, of B and of its scales, in slot 0
  constexpr int kRun = kHalf * 2;   // regions of a half that follow one another
  static_assert(kRun % T::kRegA == 0, "a wave's regions of a half are adjacent");
  const uint32_t to_a = lds + (uint32_t)(region_row_a(0, 0) * kMxSliceBytes);
  const uint32_t to_b = lds + (uint32_t)(T::kOffB + wave * T::kRegB * 1024);
  const uint32_t to_s = lds + (uint32_t)(T::kOffScale + wave * T::kScaleShare);
  auto load_a = [&](auto half_tag, auto q_tag) {
    constexpr int h = decltype(half_tag)::value, q = decltype(q_tag)::value;
    to_lds16<h * kHalf * 16 * kMxSliceBytes + q * 1024>(at_a, off_a[h * T::kRegA + q], to_a + (uint32_t)(cur_slot * T::kSlotA));
  };
  // loads 0 .. kLoadsEarly - 1 of a slice: the lower half of A, B, the scales
  auto load_early = [&](auto x_tag) {
    constexpr int X = decltype(x_tag)::value;
    if constexpr (X < T::kRegA) {
      load_a(std::integral_constant<int, 0>{}, x_tag);
    } else if constexpr (X < T::kRegA + T::kRegB) {
      constexpr int q = X - T::kRegA;
      to_lds16<q * 1024>(at_b, off_b[q], to_b + (uint32_t)(cur_slot * T::kSlotB));
    } else if constexpr (T::kScaleLoads == 1) {
      to_lds16<0>(at_s, (uint32_t)(lane * 16), to_s + (uint32_t)(cur_slot * T::kScale));
    } else {
      constexpr int part = X - T::kRegA - T::kRegB;
      to_lds4<part * 256>(at_s, (uint32_t)(lane * 4 + part * 256), to_s + (uint32_t)(cur_slot * T::kScale));
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
    read16<(h * kHalf + i) * 16 * kMxSliceBytes>(addr, dst[i]);
  };
  auto read_b = [&](uint32_t addr, u32x4(&dst)[TN], auto j_tag) {
    constexpr int j = decltype(j_tag)::value;
    read16<j * 16 * kMxSliceBytes>(addr, dst[j]);
  };
  constexpr int kScaleReads = TM / 4 + TN / 4, kNextReads = kHalf + TN + kScaleReads;
  auto read_next = [&](uint32_t aa, uint32_t ba, uint32_t ssa, uint32_t ssb, auto r_tag) {
    constexpr int R = decltype(r_tag)::value;
    if constexpr (R < TM / 4) read8<R * kUnitBytes>(ssa, sa_next[R]);
    else if constexpr (R < kScaleReads) read8<(R - TM / 4) * kUnitBytes>(ssb, sb_next[R - TM / 4]);
    else if constexpr (R == kScaleReads) read_b(ba, b0, std::integral_constant<int, 0>{});
    else if constexpr (R <= kScaleReads + kHalf)
      read_a(std::integral_constant<int, 0>{}, aa, a0, std::integral_constant<int, R - kScaleReads - 1>{});
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

  for (int tile = blockIdx.x; tile < total_tiles; tile += gridDim.x) {
    int tm, tn;
    map_tile(tile, tiles_m, tiles_n, tm, tn);
    const int m0 = tm * T::kBM + wm * TM * 16, n0 = tn * T::kBN + wn * TN * 16;   // the wave's part of the tile
    start_from_bias<KIND>(p, n0, acc);
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

    store_outputs<KIND>(p, m0, n0, acc);
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
  // 256 x 256 tiles once there is one for every compute unit (with 128 x 128 ones instead: 2048 x 8192 x 8192, 256 tiles,
  // 67 us against 79; 5120 x 5120 x 4096, 400 tiles, 61 against 70; 8192^3 236 against 296), below that 128 x 128 (1024 x
  // 8192 x 8192, 128 large tiles, 44 against 47).  The rule does not count rounds: 192 large tiles would take 55 us against
  // 62 (1536 x 8192 x 8192), while a second round of few large tiles costs more than small ones (4352 x 4352 x 4096, 289
  // tiles, 60 against 53; 4096 x 5120 x 5120, 320 tiles, 71 against 65).
  const int64_t large = (int64_t)((p.m + 255) / 256) * ((p.n + 255) / 256);
  if (large >= device_cus())
    return tiles_launch<2, 4, 8, 4, KIND>(p, scales, units_a, units_b, slices, 1, block_dim, stream);
  return tiles_launch<2, 2, 4, 4, KIND>(p, scales, units_a, units_b, slices, 2, block_dim, stream);
}

}  // namespace

bool mxfp4_dma_supported(const MxOperands &p) {
  // the offset of a lane's line from its tile's first row has 32 bits
  return p.m > 64 && p.kb >= kMxSliceBlocks && p.n <= kMxMaxColumns && (int64_t)p.kb * kMxBlockBytes * 256 < (int64_t)1 << 32;
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
