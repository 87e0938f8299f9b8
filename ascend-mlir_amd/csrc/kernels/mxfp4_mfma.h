// The scaled fp4 matrix instruction and the operands of an MXFP4 product, shared by its kernels.
//
// v_mfma_scale_f32_16x16x128_f8f6f4 multiplies 16 x 128 by 128 x 16 codes and applies the block
// scales: lane l holds row l % 16, the 32 codes (16 bytes) of one block, and that block's scale
// byte; the four lanes of a row hold four different blocks.  Which four is free as long as both
// operands agree, since a sum over blocks has no order that matters.  Products of two codes are
// multiples of 1/4 up to 36, and the instruction adds them in float32.  B is the row operand, so a
// lane's four accumulators are four consecutive columns of one output row.
#pragma once

#include <type_traits>

#include "kernels.h"
#include "mxfp4.h"

namespace afir {

typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int kMxSliceBytes = 128, kMxSliceBlocks = 8;   // of a row: 256 numbers, one line of codes
constexpr int kMxMaxColumns = 1 << 26;                   // of an output whose rows are addressed with 32-bit offsets
constexpr int kFp4 = 4;   // the format number of e2m1 in the instruction's two format fields

// scale byte BA of `sa` and BB of `sb` go with these 16 bytes
template <int BB, int BA>
__device__ __forceinline__ f32x4 mfma_fp4(u32x4 b, u32x4 a, f32x4 c, uint32_t sb, uint32_t sa) {
  const i32x8 b8 = {(int)b.x, (int)b.y, (int)b.z, (int)b.w, 0, 0, 0, 0};
  const i32x8 a8 = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b8, a8, c, kFp4, kFp4, BB, (int)sb, BA, (int)sa);
}

struct MxOperands {
  const unsigned char *a, *b;         // codes, kb * 16 bytes a row
  const uint8_t *a_scales, *b_scales; // kb bytes a row
  const void *bias;                   // of the output's type, or null
  void *out;
  int m, n, kb;
  float alpha;
};

// ---- direct-to-LDS loads, LDS reads and their waits ----
// The loads and the reads that have to overlap them are issued from inline asm, with explicit waits:
// the compiler would wait for every load in flight before any LDS read that might alias one.

template <int N>
__device__ __forceinline__ void wait_vmcnt() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void wait_lds() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
}
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

// 16 (4) bytes per lane from base + offset, one after the other from LDS address `to` + OFF
template <int OFF>
__device__ __forceinline__ void to_lds16(const unsigned char *base, uint32_t offset, uint32_t to) {
  asm volatile("s_add_u32 m0, %0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               ::"s"(to), "v"(offset), "s"(base), "n"(OFF) : "memory", "scc");
}
// 16 (4) bytes per lane from an address of its own
__device__ __forceinline__ void to_lds4_at(const unsigned char *from, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(to), "v"(from) : "memory");
}
__device__ __forceinline__ void to_lds16_at(const unsigned char *from, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(from) : "memory");
}
template <int OFF>
__device__ __forceinline__ void to_lds4(const unsigned char *base, uint32_t offset, uint32_t to) {
  asm volatile("s_add_u32 m0, %0, %3\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2"
               ::"s"(to), "v"(offset), "s"(base), "n"(OFF) : "memory", "scc");
}

// ---- the two ends of a wave's sums: TM x TN tiles from row m0, column n0 of the output ----

// The sums start from the bias of their columns (four adjacent ones of each n tile), or from -0, the
// identity of the add.  It comes through the scalar cache: a vector load would have to wait for every
// line that was requested before it.
template <int KIND, int TM, int TN>
__device__ __forceinline__ void start_from_bias(const MxOperands &p, int n0, f32x4 (&acc)[TM][TN]) {
  constexpr int kSize = KIND == kElemF32 ? 4 : 2, kWords = 16 * kSize / 4;
  const int ge = lane_here() >> 4;
  static_for<0, TN>([&](auto j_tag) {
    constexpr int j = decltype(j_tag)::value;
    uint32_t w[kSize];
#pragma unroll
    for (int e = 0; e < kSize; ++e) w[e] = kSize == 4 ? 0x80000000u : 0x80008000u;
    if (p.bias && n0 + TN * 16 <= p.n && (reinterpret_cast<uintptr_t>(p.bias) & 3u) == 0) {
      typedef const __attribute__((address_space(4))) uint32_t *ScalarWords;
      const ScalarWords q = (ScalarWords)(reinterpret_cast<uintptr_t>(p.bias) + (uintptr_t)(n0 + j * 16) * kSize);
#pragma unroll
      for (int e = 0; e < kSize; ++e) {
        const uint32_t low = (ge & 1) ? q[kWords / 4 + e] : q[e];
        const uint32_t high = (ge & 1) ? q[3 * kWords / 4 + e] : q[kWords / 2 + e];
        w[e] = (ge & 2) ? high : low;
      }
    } else if (p.bias) {
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
    float b[4];
    Elem<KIND>::unpack(w, b);
#pragma unroll
    for (int i = 0; i < TM; ++i) acc[i][j] = f32x4{b[0], b[1], b[2], b[3]};
  });
}

// Slope, rounding, stores.  A lane holds four adjacent columns (4 ge ..) of row lie of every 16 x 16
// tile: 16 bytes in 32 bits.  In 16 bits two n tiles first exchange halves between lanes 16 apart,
// after which a lane has eight adjacent columns of one of them.  Either way four lanes hold 64 adjacent
// bytes of a row, and two such sets are 128: they exchange rows 8 to 15 of the first for rows 0 to 7 of
// the second, so that a store writes eight whole lines.  (With 64 bytes of sixteen rows per store an
// 8192^3 product took 4 % longer.)  Parts that lie inside the output as a whole store without any test.
template <int KIND, int TM, int TN>
__device__ __forceinline__ void store_outputs(const MxOperands &p, int m0, int n0, const f32x4 (&acc)[TM][TN]) {
  constexpr int kSize = KIND == kElemF32 ? 4 : 2;
  constexpr int kSide = 64 / kSize;                            // columns of 64 bytes
  constexpr bool kLines = TN * 16 * kSize >= 128;              // the wave's columns fill a line
  static_assert(TN * 16 * kSize % (kLines ? 128 : 64) == 0, "whole sets of 64 bytes, pairs of them in lines");
  typedef typename Elem<KIND>::type E;
  const int lane = lane_here(), lie = lane & 15, ge = lane >> 4;
  const int lane_col = (kLines ? (lie >> 3) * kSide : 0) + (kSize == 4 ? 4 * ge : (ge & 1) * 16 + (ge >> 1) * 8);
  const int lane_row = kLines ? lie & 7 : lie;
  // Rows of whole lines are streamed past the L2 (8192 x 8192 x 64: 38 us against 49); in others neighbouring
  // tiles share lines, which the L2 puts together (8000 x 8100 x 1000: 64 us against 80).
  const bool streams = ((reinterpret_cast<uintptr_t>(p.out) | (uintptr_t)p.n * kSize) & 127u) == 0;
  auto outputs = [&](auto slope_tag, auto inside_tag, auto streams_tag) {
    constexpr bool kSlope = decltype(slope_tag)::value, kInside = decltype(inside_tag)::value;
    constexpr bool kStreams = decltype(streams_tag)::value;
    E *row = static_cast<E *>(p.out) + (int64_t)m0 * p.n + n0;   // wave-uniform
    const uint32_t lane_at = (uint32_t)(lane_row * p.n + lane_col);
    auto packed = [&](const f32x4 &c, uint32_t(&w)[kSize]) {
      float v[4] = {c[0], c[1], c[2], c[3]};
      if constexpr (kSlope) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = fmaxf(v[e], v[e] * p.alpha);
      }
      Elem<KIND>::pack(v, w);
    };
    // 16 bytes at row m0 + r + the lane's, column n0 + at + the lane's; `row` points to row m0 + r
    auto put = [&](E *o, u32x4 w) {
      if constexpr (kStreams) __builtin_nontemporal_store(w, reinterpret_cast<u32x4_u *>(o));
      else *reinterpret_cast<u32x4_u *>(o) = w;
    };
    auto store = [&](int r, int at, u32x4 w) {
      E *const o = row + at + lane_at;
      if constexpr (kInside) {
        put(o, w);
      } else {
        const int n = n0 + at + lane_col;
        if (m0 + r + lane_row >= p.m || n >= p.n) return;
        if (n + 16 / kSize <= p.n) {
          put(o, w);
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
    // two sets of 64 bytes of a row
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
      // set `s` of the row: n tile s, or tiles 2s and 2s + 1 in 16 bits
      auto set = [&](auto s_tag) {
        constexpr int s = decltype(s_tag)::value;
        if constexpr (kSize == 4) {
          uint32_t w[4];
          packed(acc[i][s], w);
          return u32x4{w[0], w[1], w[2], w[3]};
        } else {
          uint32_t w0[2], w1[2];
          packed(acc[i][2 * s], w0);
          packed(acc[i][2 * s + 1], w1);
          // rows of 16 lanes: the odd ones of the first change places with the even ones of the second
          const u32x2 x = swap_odd_even(w0[0], w1[0]), y = swap_odd_even(w0[1], w1[1]);
          return u32x4{x.x, y.x, x.y, y.y};
        }
      };
      constexpr int kSets = TN * 16 * kSize / 64;
      if constexpr (kLines) {
        static_for<0, kSets / 2>([&](auto h_tag) {
          constexpr int s = 2 * decltype(h_tag)::value;
          both(i * 16, s * kSide, set(std::integral_constant<int, s>{}), set(std::integral_constant<int, s + 1>{}));
        });
      } else {
        store(i * 16, 0, set(std::integral_constant<int, 0>{}));
      }
      row += (int64_t)16 * p.n;
    });
  };
  const bool inside = m0 + TM * 16 <= p.m && n0 + TN * 16 <= p.n;
  if (!inside) outputs(std::true_type{}, std::false_type{}, std::false_type{});
  else if (!streams) outputs(std::true_type{}, std::true_type{}, std::false_type{});
  else if (p.alpha != 1.f) outputs(std::true_type{}, std::true_type{}, std::true_type{});
  else outputs(std::false_type{}, std::true_type{}, std::true_type{});
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

// One workgroup per tile (mxfp4_matmul_ring.hip).
bool mxfp4_ring_supported(const MxOperands &p);
LaunchStatus launch_mxfp4_ring(const MxOperands &p, int elem_kind, uint32_t block_dim, hipStream_t stream);
// Tiled kernels for products of more than a few rows (mxfp4_matmul_dma.hip).
bool mxfp4_dma_supported(const MxOperands &p);
size_t mxfp4_dma_workspace(int64_t m, int64_t kb, int64_t n);
LaunchStatus launch_mxfp4_dma(const MxOperands &p, int elem_kind, void *workspace, uint32_t block_dim, hipStream_t stream);

}  // namespace afir
