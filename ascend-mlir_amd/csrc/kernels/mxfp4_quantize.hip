// Quantisation to MXFP4 (mxfp4.h) along the rows of a matrix or down its columns.
//
// Memory-bound: every number is read once and leaves as half a byte, plus one scale byte per 32,
// plus, on request, the number its code stands for.  The largest magnitude of a block is taken on
// the bit patterns (for non-negative floats their order is the order of the values, and infinities
// and NaNs come out on top), so there is no rounding anywhere but in the conversion itself and the
// results do not depend on which lane does what.
#include "kernels.h"
#include "mxfp4.h"

namespace afir {

namespace {

constexpr int kThreads = 256;

// n / d for 32-bit n by one high multiply (d >= 1, fixed per launch): the divisor's reciprocal,
// rounded up, with the 33rd bit folded into the add.
struct FastDivisor {
  uint32_t d, m, shift;
};
inline FastDivisor fast_divisor(uint32_t d) {
  uint32_t s = 0;
  while (s < 32 && ((uint64_t)1 << s) < d) ++s;
  const uint64_t m = (((uint64_t)1 << 32) * (((uint64_t)1 << s) - d)) / d + 1;
  return FastDivisor{d, (uint32_t)m, s};
}
__device__ __forceinline__ uint32_t fast_divide(uint32_t n, const FastDivisor &f) {
  if (f.shift == 0) return n;
  const uint32_t t = __umulhi(f.m, n);
  return (t + ((n - t) >> 1)) >> (f.shift - 1);
}

// The largest of four neighbouring lanes' values (lanes 4i .. 4i + 3).
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, true);   // quad_perm [1,0,3,2]
  v = v > o ? v : o;
  o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, true);            // quad_perm [2,3,0,1]
  return v > o ? v : o;
}

// Blocks along the rows.  Four lanes share a block, eight numbers each: 16-byte loads for the
// 16-bit types, a scale from two steps across the quad.  The (row, quad) pairs are dealt out flat,
// so rows of any length fill the wavefronts; a lane asks for kUnroll groups before it uses the
// first.  `groups` is a row's lanes, four to a block; numbers past the row's end count as zeros.
// bf16 8192 x 8192 with values: 48.5 us (6.3 TB/s), 51.4 with values stored by way of the L2; without values 29
// (5.9 TB/s).  float32, whose lanes take two pieces 32 bytes apart: 107 (5.4 TB/s), without values 54.
template <int KIND, bool VALUES>
__global__ __launch_bounds__(kThreads) void mxfp4_quantize_rows(const void *__restrict__ x, int64_t ld,
                                                                uint32_t *__restrict__ codes,
                                                                uint8_t *__restrict__ scales, void *__restrict__ values,
                                                                int64_t k, FastDivisor groups, uint32_t total,
                                                                int unroll_blocks) {
  constexpr int kUnroll = 4;
  constexpr int kWords = 32 / Elem<KIND>::kPer16;   // 32-bit words of eight numbers
  typedef typename Elem<KIND>::type T;
  for (int block = blockIdx.x; block < unroll_blocks; block += gridDim.x) {
    const uint32_t first = (uint32_t)block * (kThreads * kUnroll) + threadIdx.x;
    uint32_t w[kUnroll][kWords];
    int64_t row[kUnroll];
    int64_t at[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const uint32_t i = first + u * kThreads;
      const uint32_t r = fast_divide(i, groups);
      row[u] = r;
      at[u] = (int64_t)(i - r * groups.d) * 8;
#pragma unroll
      for (int q = 0; q < kWords; ++q) w[u][q] = 0;
      if (i < total) {
        const T *p = static_cast<const T *>(x) + row[u] * ld + at[u];
        if (at[u] + 8 <= k) {
          if constexpr (kWords == 4) {
            const u32x4 v = *reinterpret_cast<const u32x4_u *>(p);
            w[u][0] = v.x; w[u][1] = v.y; w[u][2] = v.z; w[u][3] = v.w;
          } else {
            const u32x4 v = *reinterpret_cast<const u32x4_u *>(p), z = *reinterpret_cast<const u32x4_u *>(p + 4);
            w[u][0] = v.x; w[u][1] = v.y; w[u][2] = v.z; w[u][3] = v.w;
            w[u][kWords - 4] = z.x; w[u][kWords - 3] = z.y; w[u][kWords - 2] = z.z; w[u][kWords - 1] = z.w;
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (at[u] + e < k) {
              if constexpr (kWords == 4) w[u][e / 2] |= (uint32_t)p[e] << (16 * (e & 1));
              else w[u][e] = __float_as_uint(p[e]);
            }
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const uint32_t i = first + u * kThreads;
      float v[8];
      Elem<KIND>::unpack(w[u], v);
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t b = __float_as_uint(v[e]) & 0x7fffffffu;
        top = b > top ? b : top;
      }
      top = quad_max(top);   // (a quad's lanes are four groups of one block: all in range or none)
      const uint32_t byte = mx_scale_byte(top);
      const float scale = mx_scale_value(byte);
      const uint32_t code = byte == 255u ? 0u : mx_encode8(v, scale);
      if (i < total) {
        // row r's codes follow row r - 1's: group i of the launch is word i
        codes[i] = code;
        if ((i & 3u) == 0) scales[i >> 2] = (uint8_t)byte;
        if constexpr (VALUES) {
          float back[8];
          mx_decode8(code, scale, back);
          if (byte == 255u) {
#pragma unroll
            for (int e = 0; e < 8; ++e) back[e] = __uint_as_float(0x7fc00000u);
          }
          T *p = static_cast<T *>(values) + row[u] * k + at[u];
          if (at[u] + 8 <= k) {
            uint32_t o[kWords];
            Elem<KIND>::pack(back, o);
            __builtin_nontemporal_store(u32x4{o[0], o[1], o[2], o[3]}, reinterpret_cast<u32x4_u *>(p));
            if constexpr (kWords == 8)
              __builtin_nontemporal_store(u32x4{o[kWords - 4], o[kWords - 3], o[kWords - 2], o[kWords - 1]},
                                          reinterpret_cast<u32x4_u *>(p + 4));
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (at[u] + e < k) Elem<KIND>::store(p, e, back[e]);
          }
        }
      }
    }
  }
}

// Blocks down the columns of x [K, R], codes and scales laid out as for the rows of its transpose.
// A workgroup takes 256 rows of 64 lanes' columns; a wavefront takes 32 of the rows, one block of
// every column, and a lane holds the block of its own one or two columns (4 bytes of a row) in
// registers: 32 loads in flight, each a contiguous piece of a row, and no exchange between lanes.
// The eight blocks of a column meet in LDS and leave as whole 128-byte lines of its code row.  Rows that
// are no whole number of lines share lines between neighbouring tiles, which therefore belong to one XCD,
// whose L2 puts them together: float32 [8192, 4099] with values 54 us against 72 with neighbours on
// different XCDs (and 71 with stores that bypass the L2); 63 us (4.5 TB/s) where the output is not in the
// last-level cache from the call before.  bf16 [8192, 8192]: 66 us (4.6 TB/s), without values 43.
constexpr int kColWaves = 8;
template <int KIND, bool VALUES>
__global__ __launch_bounds__(kColWaves * 64) void mxfp4_quantize_cols(const void *__restrict__ x, int64_t ld,
                                                                      unsigned char *__restrict__ codes,
                                                                      uint8_t *__restrict__ scales,
                                                                      void *__restrict__ values, int64_t k, int64_t r,
                                                                      int64_t kb, int tiles_r, int64_t tiles) {
  constexpr int VC = Elem<KIND>::kPer16 / 4;   // columns of a lane
  constexpr int kCols = 64 * VC;
  typedef typename Elem<KIND>::type T;
  __shared__ __align__(16) u32x4 code_tile[kCols * kColWaves];
  __shared__ __align__(8) uint8_t scale_tile[kCols * kColWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // workgroup i runs on XCD i % 8, and an XCD takes tiles that follow one another
  const int64_t per_xcd = (tiles + kNumXCD - 1) / kNumXCD;
  for (int64_t q = blockIdx.x; q < per_xcd * kNumXCD; q += gridDim.x) {
    const int64_t tile = q % kNumXCD * per_xcd + q / kNumXCD;
    if (tile >= tiles) continue;
    const int64_t c0 = (tile % tiles_r) * kCols, b0 = (tile / tiles_r) * kColWaves;
    const int64_t c = c0 + lane * VC, k0 = (b0 + wave) * kMxBlock;
    uint32_t w[kMxBlock];
    const T *p = static_cast<const T *>(x) + k0 * ld + c;
#pragma unroll
    for (int i = 0; i < kMxBlock; ++i) {
      w[i] = 0;
      if (k0 + i < k) {
        if (c + VC <= r) w[i] = *reinterpret_cast<const u32_u *>(p + (int64_t)i * ld);
        else if (VC == 2 && c < r) w[i] = reinterpret_cast<const uint16_t *>(p + (int64_t)i * ld)[0];
      }
    }
    uint32_t top[VC];
#pragma unroll
    for (int h = 0; h < VC; ++h) top[h] = 0;
#pragma unroll
    for (int i = 0; i < kMxBlock; ++i) {
      float v[VC];
      const uint32_t one[1] = {w[i]};
      Elem<KIND>::unpack(one, v);
#pragma unroll
      for (int h = 0; h < VC; ++h) {
        const uint32_t b = __float_as_uint(v[h]) & 0x7fffffffu;
        top[h] = b > top[h] ? b : top[h];
      }
    }
    uint32_t code[VC][4];
    float scale[VC];
    uint32_t byte[VC];
#pragma unroll
    for (int h = 0; h < VC; ++h) {
      byte[h] = mx_scale_byte(top[h]);
      scale[h] = mx_scale_value(byte[h]);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float both[VC];
          const uint32_t one[1] = {w[8 * q + e]};
          Elem<KIND>::unpack(one, both);
          v[e] = both[h];
        }
        code[h][q] = byte[h] == 255u ? 0u : mx_encode8(v, scale[h]);
      }
      const int col = lane * VC + h;
      code_tile[col * kColWaves + (wave ^ (col & 7))] = u32x4{code[h][0], code[h][1], code[h][2], code[h][3]};
      scale_tile[col * kColWaves + wave] = (uint8_t)byte[h];
    }
    if constexpr (VALUES) {
      T *o = static_cast<T *>(values) + k0 * r + c;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float back[VC][8];
#pragma unroll
        for (int h = 0; h < VC; ++h) {
          mx_decode8(code[h][q], scale[h], back[h]);
          if (byte[h] == 255u) {
#pragma unroll
            for (int e = 0; e < 8; ++e) back[h][e] = __uint_as_float(0x7fc00000u);
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int i = 8 * q + e;
          if (k0 + i < k) {
            float v[VC];
            uint32_t one[1];
#pragma unroll
            for (int h = 0; h < VC; ++h) v[h] = back[h][e];
            Elem<KIND>::pack(v, one);
            if (c + VC <= r) *reinterpret_cast<u32_u *>(o + (int64_t)i * r) = one[0];
            else if (VC == 2 && c < r) reinterpret_cast<uint16_t *>(o + (int64_t)i * r)[0] = (uint16_t)one[0];
          }
        }
      }
    }
    __syncthreads();
    const int nb = kb - b0 < kColWaves ? (int)(kb - b0) : kColWaves;
#pragma unroll
    for (int j = 0; j < VC; ++j) {
      const int item = j * (kColWaves * 64) + threadIdx.x, col = item >> 3, chunk = item & 7;
      if (c0 + col < r && chunk < nb) {
        *reinterpret_cast<u32x4 *>(codes + ((c0 + col) * kb + b0 + chunk) * kMxBlockBytes) =
            code_tile[col * kColWaves + (chunk ^ (col & 7))];
        scales[(c0 + col) * kb + b0 + chunk] = scale_tile[col * kColWaves + chunk];
      }
    }
    __syncthreads();
  }
}

template <int KIND, bool VALUES>
LaunchStatus quantize_rows(const void *x, int64_t ld, void *codes, void *scales, void *values, int64_t rows, int64_t k,
                           uint32_t block_dim, hipStream_t stream) {
  const int64_t kb = (k + kMxBlock - 1) / kMxBlock, groups = kb * 4;
  constexpr int64_t kPerBlock = kThreads * 4;
  // a launch indexes its groups with 32 bits; longer matrices go out in pieces of rows
  const int64_t most = ((int64_t)1 << 31) / groups;
  const int64_t size = KIND == kElemF32 ? 4 : 2;
  for (int64_t r0 = 0; r0 < rows; r0 += most) {
    const int64_t n = rows - r0 < most ? rows - r0 : most;
    const int64_t total = n * groups, blocks = (total + kPerBlock - 1) / kPerBlock;
    const int64_t grid = block_dim ? block_dim : blocks;
    AFIR_LAUNCH("mxfp4_quantize_rows", (mxfp4_quantize_rows<KIND, VALUES>), dim3((unsigned)grid), dim3(kThreads), 0, stream,
                static_cast<const char *>(x) + r0 * ld * size, ld,
                reinterpret_cast<uint32_t *>(static_cast<char *>(codes) + r0 * kb * kMxBlockBytes),
                static_cast<uint8_t *>(scales) + r0 * kb,
                VALUES ? static_cast<void *>(static_cast<char *>(values) + r0 * k * size) : nullptr, k,
                fast_divisor((uint32_t)groups), (uint32_t)total, (int)blocks);
    const LaunchStatus st = after_launch();
    if (st.code) return st;
  }
  return ok_status();
}

template <int KIND, bool VALUES>
LaunchStatus quantize_cols(const void *x, int64_t ld, void *codes, void *scales, void *values, int64_t r, int64_t k,
                           uint32_t block_dim, hipStream_t stream) {
  constexpr int kCols = 64 * (Elem<KIND>::kPer16 / 4);
  const int64_t kb = (k + kMxBlock - 1) / kMxBlock;
  const int64_t tiles_r = (r + kCols - 1) / kCols, tiles = tiles_r * ((kb + kColWaves - 1) / kColWaves);
  const int64_t places = (tiles + kNumXCD - 1) / kNumXCD * kNumXCD;
  int64_t grid = places < (int64_t)1 << 20 ? places : (int64_t)1 << 20;
  if (block_dim) grid = block_dim;
  AFIR_LAUNCH("mxfp4_quantize_cols", (mxfp4_quantize_cols<KIND, VALUES>), dim3((unsigned)grid), dim3(kColWaves * 64), 0,
              stream, x, ld, static_cast<unsigned char *>(codes), static_cast<uint8_t *>(scales), values, k, r, kb,
              (int)tiles_r, tiles);
  return after_launch();
}

template <int KIND>
LaunchStatus quantize(const void *x, int64_t ld, void *codes, void *scales, void *values, int64_t r, int64_t k,
                      bool columns, uint32_t block_dim, hipStream_t stream) {
  if (columns)
    return values ? quantize_cols<KIND, true>(x, ld, codes, scales, values, r, k, block_dim, stream)
                  : quantize_cols<KIND, false>(x, ld, codes, scales, values, r, k, block_dim, stream);
  return values ? quantize_rows<KIND, true>(x, ld, codes, scales, values, r, k, block_dim, stream)
                : quantize_rows<KIND, false>(x, ld, codes, scales, values, r, k, block_dim, stream);
}

}  // namespace

LaunchStatus launch_mxfp4_quantize(const void *x, int64_t ld, void *codes, void *scales, void *values, int64_t r,
                                   int64_t k, bool columns, int elem_kind, uint32_t block_dim, hipStream_t stream) {
  if (r < 0 || k < 0) return invalid("mxfp4_quantize: negative extent");
  if (r == 0 || k == 0) return ok_status();
  if (!x || !codes || !scales) return invalid("mxfp4_quantize: null tensor pointer");
  if (r > (int64_t)1 << 31 || k > (int64_t)1 << 31) return invalid("mxfp4_quantize: extent above 2^31");
  if (ld < (columns ? r : k)) return invalid("mxfp4_quantize: row stride below the row's length");
  if (ld > ((int64_t)1 << 46) / (columns ? k : r)) return invalid("mxfp4_quantize: row stride out of range");
  if (elem_kind < kElemF32 || elem_kind > kElemBF16) return invalid("mxfp4_quantize: elem_type must be 0, 1 or 2");
  const uintptr_t elem = elem_kind == kElemF32 ? 4 : 2;
  if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(values)) % elem)
    return invalid("mxfp4_quantize: tensor off its element's alignment");
  if (!aligned16(codes)) return invalid("mxfp4_quantize: codes must start on a 16-byte boundary");
  switch (elem_kind) {
    case kElemF32: return quantize<kElemF32>(x, ld, codes, scales, values, r, k, columns, block_dim, stream);
    case kElemF16: return quantize<kElemF16>(x, ld, codes, scales, values, r, k, columns, block_dim, stream);
    default: return quantize<kElemBF16>(x, ld, codes, scales, values, r, k, columns, block_dim, stream);
  }
}

}  // namespace afir
