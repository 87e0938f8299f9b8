// MXFP4 products whose output has about as many tiles as the chip has compute units, or fewer: one
// workgroup per tile, and the tile's size chosen to fill the chip.
//
// A slice of K is 256 numbers, one 128-byte line of every row of the tile's A and B.  The slices pass
// through a ring of slots in LDS, filled by direct-to-LDS loads.  Per slice there is one wait for the
// loads and one barrier, behind which the slot that everyone has left is filled again; a slice is
// multiplied out of registers while the next one is read from LDS.  Chunks are placed and chosen as in
// mxfp4_matmul_dma.hip (chunk c of row r at c ^ ((r >> 1) & 7); lane group g takes blocks g and 4 + g).
//
// The scales of 32 slices (or of fewer, rounded up to a power of two) come first, whole 16-byte pieces
// swizzled by the row, so that the reads of sixteen rows' eight bytes meet no bank twice.  (Eight bytes a
// row with every slice took half as many instructions again as the slice itself.)  A last slice that is
// not whole starts early, so that it ends with the row; the blocks that it repeats get the scale 2^-127 on
// both sides, and their products vanish in float32.
//
// How deep the ring is (3, 4 or 8 slots) measured the same.  What a slice costs is its issue, LDS and
// barrier time: requesting the next lines between the products took 512 x 8192 x 8192 from 28.3 to 26.1 us;
// the smaller tiles hide it in the other workgroups of their compute unit.  Measured: 48 x 8200 x 4096 8.7 us,
// 128 x 8192 x 8192 14.6, 256 x 8192 x 8192 19.6, 1003 x 2056 x 1376 10.1 (11.1 into float32), 1024 x 4096 x 4096 17.
#include "mxfp4_mfma.h"

namespace afir {

namespace {

constexpr int kScaleRow = 256, kScaleSlices = kScaleRow / kMxSliceBlocks;   // bytes and slices of a row held in LDS
typedef u32x4 u32x4_any __attribute__((aligned(1)));
typedef u32x2 u32x2_any __attribute__((aligned(1)));

template <int WM, int WN, int TM, int TN, int SLOTS>
struct Ring {
  static constexpr int kWaves = WM * WN, kBM = WM * TM * 16, kBN = WN * TN * 16;
  static constexpr int kRows = kBM + kBN;                       // A's rows, then B's
  static constexpr int kSlot = kRows * kMxSliceBytes;
  static constexpr int kOffScale = SLOTS * kSlot, kLds = kOffScale + kRows * kScaleRow;
  // loads of a wave per slice: regions of 1 KiB (8 rows) of A and of B
  static constexpr int kRegA = kBM / 8 / kWaves, kRegB = kBN / 8 / kWaves, kLoads = kRegA + kRegB;
  static_assert(kRegA * 8 * kWaves == kBM && kRegB * 8 * kWaves == kBN, "whole regions per wave");
  static_assert(kLds <= 160 * 1024 && kLoads * (SLOTS - 1) <= 63, "fits the LDS and the load counter");
};

enum ScaleRows { kPieces, kWords, kBytes };   // what the scale rows are whole numbers of

template <int WM, int WN, int TM, int TN, int SLOTS, int KIND>
__global__ __launch_bounds__(WM *WN * 64, (Ring<WM, WN, TM, TN, SLOTS>::kLds > 80 * 1024 ? 1 : 2)) void
mxfp4_matmul_ring(MxOperands p, int slices, ScaleRows how, int tiles_m, int tiles_n) {
  using T = Ring<WM, WN, TM, TN, SLOTS>;
  __shared__ __align__(1024) unsigned char smem[T::kLds];
  const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char *)smem;
  const int t = threadIdx.x, lane = t & 63, li = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6), wm = wave / WN, wn = wave % WN;
  const uint32_t pitch = (uint32_t)p.kb * kMxBlockBytes;

  for (int tile = blockIdx.x; tile < tiles_m * tiles_n; tile += gridDim.x) {
    int tm, tn;
    map_tile(tile, tiles_m, tiles_n, tm, tn);
    const int m0 = tm * T::kBM, n0 = tn * T::kBN;

    // ---- sources: a wave-uniform base that follows the slices, a per-lane offset per region ----
    // (rows past the end of A or B repeat the last one)
    const unsigned char *const base_a = p.a + (int64_t)m0 * pitch, *const base_b = p.b + (int64_t)n0 * pitch;
    uint32_t off_a[T::kRegA], off_b[T::kRegB];
    auto lane_offset = [&](int row, int last) {
      const int r = row + (lane >> 3), chunk = (lane & 7) ^ ((r >> 1) & 7);
      return (uint32_t)(r < last ? r : last) * pitch + (uint32_t)(chunk * 16);
    };
#pragma unroll
    for (int q = 0; q < T::kRegA; ++q) off_a[q] = lane_offset((wave * T::kRegA + q) * 8, p.m - 1 - m0);
#pragma unroll
    for (int q = 0; q < T::kRegB; ++q) off_b[q] = lane_offset((wave * T::kRegB + q) * 8, p.n - 1 - n0);
    const uint32_t to_a = lds + (uint32_t)(wave * T::kRegA * 1024);
    const uint32_t to_b = lds + (uint32_t)(T::kBM * kMxSliceBytes + wave * T::kRegB * 1024);
    auto load_region = [&](int block, int slot, auto q_tag) {   // one of the wave's of a slice, block its first
      constexpr int q = decltype(q_tag)::value;
      const int64_t at = (int64_t)block * kMxBlockBytes;
      if constexpr (q < T::kRegA) to_lds16<q * 1024>(base_a + at, off_a[q], to_a + (uint32_t)(slot * T::kSlot));
      else to_lds16<(q - T::kRegA) * 1024>(base_b + at, off_b[q - T::kRegA], to_b + (uint32_t)(slot * T::kSlot));
    };
    auto first_block = [&](int slice) {
      return (slice + 1) * kMxSliceBlocks <= p.kb ? slice * kMxSliceBlocks : p.kb - kMxSliceBlocks;
    };
    auto load_slice = [&](int slice, int slot) {
      static_for<0, T::kLoads>([&](auto q) { load_region(first_block(slice), slot, q); });
    };
    // The scales of slices first .. first + count - 1 of all of the tile's rows.  Rows of whole 16-byte pieces
    // (K a multiple of 512) or words (of 128) go to LDS directly, beside the first slices; others through
    // registers, 1 to 3 us at the start of a tile.
    auto scale_row = [&](int r) {
      const bool of_a = r < T::kBM;
      const int row = of_a ? m0 + r : n0 + r - T::kBM, rows = of_a ? p.m : p.n;
      return (of_a ? p.a_scales : p.b_scales) + (int64_t)(row < rows ? row : rows - 1) * p.kb;
    };
    // A row takes 2^row_log bytes of LDS, a power of two of pieces.  Piece c of row r is at c ^ (r >> (4 - piece_log)):
    // rows that share banks differ in it.
    const int held = slices < kScaleSlices ? slices : kScaleSlices;
    const int piece_log = 31 - __builtin_clz((unsigned)((held + 1) / 2 * 2 - 1)), row_log = piece_log + 4;
    const int piece_mask = (1 << piece_log) - 1;
    auto place_of = [&](int r, int c) { return ((r >> (4 - piece_log)) ^ c) & piece_mask; };   // and back
    auto load_scales = [&](int first) {
      const int block0 = first * kMxSliceBlocks;
      const uint32_t to = lds + (uint32_t)T::kOffScale;
      const int per_load = how == kPieces ? 6 - piece_log : 4 - piece_log;   // log2 of the rows of one load
      for (int i = wave; i << per_load < T::kRows; i += T::kWaves) {   // (rows past the last repeat it)
        if (how == kPieces) {
          const int r = (i << per_load) + (lane >> piece_log), at = block0 + (place_of(r, lane) << 4);
          to_lds16_at(scale_row(r) + (at <= p.kb - 16 ? at : p.kb - 16), to + (uint32_t)(i * 1024));
        } else {
          const int r = (i << per_load) + (lane >> (piece_log + 2));
          const int at = block0 + (place_of(r, lane >> 2) << 4) + (lane & 3) * 4;
          to_lds4_at(scale_row(r) + (at <= p.kb - 4 ? at : p.kb - 4), to + (uint32_t)(i * 256));
        }
      }
    };
    auto piece_of = [&](int r, int c) { return T::kOffScale + (r << row_log) + (place_of(r, c) << 4); };
    // a last slice of four blocks (rows of whole words) has them in its first word: they belong in the second
    auto shift_last = [&](int s) {
      for (int r = t; r < T::kRows; r += T::kWaves * 64) {
        u32x2 *const q = reinterpret_cast<u32x2 *>(smem + piece_of(r, s >> 1) + ((s & 1) << 3));
        *q = u32x2{0u, q->x};
      }
    };
    auto stage_scales = [&](int first, int count) {
      const int pieces = (count + 1) / 2;   // of 16 bytes: two slices
      for (int i = t; i < T::kRows * pieces; i += T::kWaves * 64) {
        const int r = i / pieces, c = i % pieces, block = (first + 2 * c) * kMxSliceBlocks;
        const uint8_t *const q = scale_row(r);
        u32x4 w = {0, 0, 0, 0};
        if (block + 16 <= p.kb) {
          w = *reinterpret_cast<const u32x4_any *>(q + block);
        } else {
          // the last piece: a slice is whole, or starts early, or is not there
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int b = block + h * kMxSliceBlocks, early = b + kMxSliceBlocks - p.kb;
            if (early >= kMxSliceBlocks) continue;
            const u32x2 v = *reinterpret_cast<const u32x2_any *>(q + (early > 0 ? p.kb - kMxSliceBlocks : b));
            uint64_t both = (uint64_t)v.y << 32 | v.x;
            if (early > 0) both = both >> (8 * early) << (8 * early);
            w[2 * h] = (uint32_t)both;
            w[2 * h + 1] = (uint32_t)(both >> 32);
          }
        }
        *reinterpret_cast<u32x4 *>(smem + piece_of(r, c)) = w;
      }
    };

    // ---- operand reads ----
    const uint32_t swz = (uint32_t)((li >> 1) & 7), chunk = (g ^ swz) * 16;   // second step: chunk ^ 64
    const uint32_t rd_a = (uint32_t)((wm * TM * 16 + li) * kMxSliceBytes) + chunk;
    const uint32_t rd_b = (uint32_t)((T::kBM + wn * TN * 16 + li) * kMxSliceBytes) + chunk;
    const uint32_t rd_sa = (uint32_t)(T::kOffScale + ((wm * TM * 16 + li) << row_log));
    const uint32_t rd_sb = (uint32_t)(T::kOffScale + ((T::kBM + wn * TN * 16 + li) << row_log));
    const int shift = 8 * g;

    f32x4 acc[TM][TN];
    start_from_bias<KIND>(p, n0 + wn * TN * 16, acc);

    // Slice s is multiplied out of registers while slice s + 1 is read from LDS into others, so the slot of
    // slice s is free by then.
    struct Operands {
      u32x4 a[2][TM], b[2][TN];
      u32x2 sa[TM], sb[TN];
    };
    struct Places {
      uint32_t a, b, sa, sb;
    };
    auto places = [&](int slot, int s) {   // of slice s of those whose scales are in LDS
      const uint32_t piece = (uint32_t)((place_of(li, s >> 1) << 4) | ((s & 1) << 3)), at = lds + (uint32_t)(slot * T::kSlot);
      return Places{at + rd_a, at + rd_b, lds + rd_sa + piece, lds + rd_sb + piece};
    };
    // one of a slice's reads: first the scales, then the first and the second step's codes
    auto read_one = [&](Operands &o, const Places &at, auto r_tag) {
      constexpr int r = decltype(r_tag)::value, c = (r - TM - TN) % (TM + TN), step = (r - TM - TN) / (TM + TN);
      if constexpr (r < TM) read8<0>(at.sa + (uint32_t)(r * 16 << row_log), o.sa[r]);
      else if constexpr (r < TM + TN) read8<0>(at.sb + (uint32_t)((r - TM) * 16 << row_log), o.sb[r - TM]);
      else if constexpr (c < TM) read16<c * 16 * kMxSliceBytes>(at.a ^ (step * 64u), o.a[step][c]);
      else read16<(c - TM) * 16 * kMxSliceBytes>(at.b ^ (step * 64u), o.b[step][c - TM]);
    };
    constexpr int kReads = 3 * (TM + TN);
    auto read = [&](Operands &o, int slot, int s) {
      const Places at = places(slot, s);
      static_for<0, kReads>([&](auto r) { read_one(o, at, r); });
    };
    auto arrived = [&](Operands &o) {
      wait_lds();
      settle(o.a[0]);
      settle(o.a[1]);
      settle(o.b[0]);
      settle(o.b[1]);
      settle(o.sa);
      settle(o.sb);
    };
    auto multiply = [&](const Operands &o, auto step_tag) {
      constexpr int S = decltype(step_tag)::value;
      uint32_t sa[TM], sb[TN];
#pragma unroll
      for (int i = 0; i < TM; ++i) sa[i] = o.sa[i][S] >> shift;
#pragma unroll
      for (int j = 0; j < TN; ++j) sb[j] = o.sb[j][S] >> shift;
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int i = 0; i < TM; ++i) acc[i][j] = mfma_fp4<0, 0>(o.b[S][j], o.a[S][i], acc[i][j], sb[j], sa[i]);
    };
    using First = std::integral_constant<int, 0>;
    using Second = std::integral_constant<int, 1>;
    auto run = [&](int first, int count) {   // slices first .. first + count - 1, whose scales are in LDS
      int slot = 0;   // of the slice being multiplied
      // A slice that another one follows.  STEADY: SLOTS slices follow, the last of which is requested now.
      auto slice = [&](int s, Operands &here, Operands &next, auto steady_tag) {
        constexpr bool STEADY = decltype(steady_tag)::value;
        // slice s + 1 has landed, the ones after it may be under way
        if (STEADY || s + SLOTS <= count) wait_vmcnt<T::kLoads *(SLOTS - 2)>();
        else wait_vmcnt<0>();
        __builtin_amdgcn_s_barrier();   // ... everyone's part of it, and everyone has read slice s
        const int free = slot;
        if (!STEADY && s + SLOTS < count) load_slice(first + s + SLOTS, free);
        slot = slot + 1 == SLOTS ? 0 : slot + 1;
        // (requested and awaited in one straight run of instructions: where paths meet the compiler may
        // copy registers, and must not find any whose reads are under way)
        const Places at = places(slot, s + 1);
        const int block = first_block(first + s + SLOTS);
        uint32_t sa[2][TM], sb[2][TN];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int i = 0; i < TM; ++i) sa[h][i] = here.sa[i][h] >> shift;
#pragma unroll
          for (int j = 0; j < TN; ++j) sb[h][j] = here.sb[j][h] >> shift;
        }
        // the reads over the first 3/4 of the products; the loads over all of them, where no other workgroup
        // on the compute unit fills the time that their issue takes
        static_for<0, 2 * TN>([&](auto x_tag) {
          constexpr int x = decltype(x_tag)::value, h = x / TN, j = x % TN;
          constexpr int parts = 2 * TN * 3 / 4, load_parts = T::kLds > 80 * 1024 ? 2 * TN : 1;
          if constexpr (x < parts)
            static_for<kReads * x / parts, kReads *(x + 1) / parts>([&](auto r) { read_one(next, at, r); });
          if constexpr (STEADY && x < load_parts)
            static_for<T::kLoads * x / load_parts, T::kLoads *(x + 1) / load_parts>([&](auto q) { load_region(block, free, q); });
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int i = 0; i < TM; ++i) acc[i][j] = mfma_fp4<0, 0>(here.b[h][j], here.a[h][i], acc[i][j], sb[h][j], sa[h][i]);
          __builtin_amdgcn_sched_barrier(0);
        });
        arrived(next);
      };
      auto last_slice = [&](Operands &here) {
        multiply(here, First{});
        multiply(here, Second{});
      };
      if (how != kBytes) load_scales(first);
      else stage_scales(first, count);
      for (int s = 0; s < SLOTS && s < count; ++s) load_slice(first + s, s);
      // the scales and slice 0 have landed
      if (count >= SLOTS) wait_vmcnt<T::kLoads *(SLOTS - 1)>();
      else wait_vmcnt<0>();
      __syncthreads();
      if (how != kBytes && first + count == slices && slices * kMxSliceBlocks != p.kb) {
        shift_last(count - 1);
        __syncthreads();
      }
      Operands even, odd;
      read(even, 0, 0);
      arrived(even);
      int s = 0;
      for (; s + 1 + SLOTS < count; s += 2) {
        slice(s, even, odd, std::true_type{});
        slice(s + 1, odd, even, std::true_type{});
      }
      for (; s + 2 < count; s += 2) {
        slice(s, even, odd, std::false_type{});
        slice(s + 1, odd, even, std::false_type{});
      }
      if (s + 1 < count) {
        slice(s, even, odd, std::false_type{});
        last_slice(odd);
      } else {
        last_slice(even);
      }
    };
    for (int first = 0; first < slices; first += kScaleSlices) {
      run(first, slices - first < kScaleSlices ? slices - first : kScaleSlices);
      __builtin_amdgcn_s_barrier();   // everyone has read the ring and the scales before they are filled again
    }
    store_outputs<KIND>(p, m0 + wm * TM * 16, n0 + wn * TN * 16, acc);
  }
}

template <int WM, int WN, int TM, int TN, int SLOTS, int KIND>
LaunchStatus ring_launch(const MxOperands &p, uint32_t block_dim, hipStream_t stream) {
  using T = Ring<WM, WN, TM, TN, SLOTS>;
  const int tiles_m = (p.m + T::kBM - 1) / T::kBM, tiles_n = (p.n + T::kBN - 1) / T::kBN;
  const int64_t blocks = (int64_t)tiles_m * tiles_n;
  if (blocks > 0x7fffffff) return invalid("mxfp4_matmul: too many output tiles");
  const uintptr_t starts = reinterpret_cast<uintptr_t>(p.a_scales) | reinterpret_cast<uintptr_t>(p.b_scales);
  const ScaleRows how = (starts | (uintptr_t)p.kb) % 16 == 0 ? kPieces : (starts | (uintptr_t)p.kb) % 4 == 0 ? kWords : kBytes;
  AFIR_LAUNCH("mxfp4_matmul_ring", (mxfp4_matmul_ring<WM, WN, TM, TN, SLOTS, KIND>),
              dim3(block_dim ? block_dim : (unsigned)blocks), dim3(T::kWaves * 64), 0, stream, p, (p.kb + kMxSliceBlocks - 1) / kMxSliceBlocks, how, tiles_m, tiles_n);
  return after_launch();
}

// The tile is the one that takes the fullest compute unit the shortest time.  What a slice of one tile
// costs there, alone and beside others, in units of 10 ns as measured at K = 4096 and 8192:
struct TileCost {
  int rows, columns, alone, beside;
  int of(int64_t m, int64_t n, int64_t cus) const {
    const int64_t tiles = ((m + rows - 1) / rows) * ((n + columns - 1) / columns), fullest = (tiles + cus - 1) / cus;
    const int64_t cost = fullest * beside;
    return (int)(cost < alone ? alone : cost > 1 << 30 ? 1 << 30 : cost);
  }
};
constexpr TileCost kTiles[] = {{128, 128, 75, 75}, {128, 64, 53, 53}, {64, 64, 38, 35}, {32, 32, 31, 14}};

template <int KIND>
LaunchStatus ring(const MxOperands &p, uint32_t block_dim, hipStream_t stream) {
  const int64_t cus = device_cus();
  int best = 3;
  for (int i = 2; i >= 0; --i) {
    // (with half of the tile's rows past the end the time is that of reading B, which a tile's costs do not show)
    if (p.m > kTiles[i].rows / 2 && kTiles[i].of(p.m, p.n, cus) <= kTiles[best].of(p.m, p.n, cus)) best = i;
  }
  switch (best) {
    case 0: return ring_launch<2, 2, 4, 4, 3, KIND>(p, block_dim, stream);
    case 1: return ring_launch<2, 2, 4, 2, 3, KIND>(p, block_dim, stream);
    case 2: return ring_launch<2, 2, 2, 2, 3, KIND>(p, block_dim, stream);
    default: return ring_launch<2, 1, 1, 2, 3, KIND>(p, block_dim, stream);
  }
}

}  // namespace

bool mxfp4_ring_supported(const MxOperands &p) {
  // a whole slice, 32-bit offsets within a tile
  return p.kb >= kMxSliceBlocks && p.n <= kMxMaxColumns && (int64_t)p.kb * kMxBlockBytes * 128 < (int64_t)1 << 32;
}

LaunchStatus launch_mxfp4_ring(const MxOperands &p, int elem_kind, uint32_t block_dim, hipStream_t stream) {
  switch (elem_kind) {
    case kElemF32: return ring<kElemF32>(p, block_dim, stream);
    case kElemF16: return ring<kElemF16>(p, block_dim, stream);
    default: return ring<kElemBF16>(p, block_dim, stream);
  }
}

}  // namespace afir
