// out = leakyrelu(A B^T + bias) with A [M, K] and B [N, K] in MXFP4 (mxfp4.h) along K.
// Products of few rows; the dispatch of all of them.
#include "mxfp4_mfma.h"

namespace afir {

namespace {

typedef uint32_t u32_any __attribute__((aligned(1)));
constexpr int64_t kMaxExtent = 0x7ffffe00;   // extents and what a tile rounds them up to are 32-bit

template <int KIND>
__device__ __forceinline__ void finish_one(const MxOperands &p, int m, int n, float v) {
  if (p.bias) v += Elem<KIND>::load(p.bias, n);
  v = fmaxf(v, v * p.alpha);
  Elem<KIND>::store(p.out, (int64_t)m * p.n + n, v);
}

// Few rows of A (MT tiles of 16): the time is that of reading B.  A workgroup owns 16 * NT
// columns and its eight wavefronts deal the blocks of K out among themselves, 16 blocks at a time:
// lane group g of a wavefront takes blocks 4g .. 4g + 3, so a row's scales are one 32-bit load and
// its codes four 16-byte loads.  Everything of a step is requested before the first product.  The
// eight partial sums meet in LDS and are added in a fixed order.
constexpr int kRowsWaves = 8;
template <int MT, int NT, int KIND>
__global__ __launch_bounds__(kRowsWaves * 64) void mxfp4_matmul_rows(MxOperands p, int tiles_n, int chunks_m,
                                                                     int blocks) {
  constexpr int kCols = 16 * NT, kRows = 16 * MT;
  __shared__ f32x4 part[kRowsWaves][kRows * kCols / 4];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, li = lane & 15, g = lane >> 4;
  const int64_t pitch = (int64_t)p.kb * kMxBlockBytes;
  for (int block = blockIdx.x; block < blocks; block += gridDim.x) {
    // chunks of A that share columns follow one another on one XCD, whose L2 then holds the columns' B
    const int xcd = block % kNumXCD, idx = block / kNumXCD;
    const int tile_n = (idx / chunks_m) * kNumXCD + xcd, m0 = (idx % chunks_m) * kRows;
    if (tile_n >= tiles_n) continue;
    const int n0 = tile_n * kCols;
    // rows past the end repeat the last one; what they give is not stored
    int64_t row_a[MT], row_b[NT];
#pragma unroll
    for (int i = 0; i < MT; ++i) row_a[i] = m0 + i * 16 + li < p.m ? m0 + i * 16 + li : p.m - 1;
#pragma unroll
    for (int j = 0; j < NT; ++j) row_b[j] = n0 + j * 16 + li < p.n ? n0 + j * 16 + li : p.n - 1;
    f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int step = wave; step * 16 < p.kb; step += kRowsWaves) {
      const int k0 = step * 16 + 4 * g;
      u32x4 a[MT][4], b[NT][4];
      uint32_t sa[MT], sb[NT];
      if (step * 16 + 16 <= p.kb) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const u32x4 *q = reinterpret_cast<const u32x4 *>(p.b + row_b[j] * pitch) + k0;
#pragma unroll
          for (int c = 0; c < 4; ++c) b[j][c] = q[c];
          sb[j] = *reinterpret_cast<const u32_any *>(p.b_scales + row_b[j] * p.kb + k0);
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          const u32x4 *q = reinterpret_cast<const u32x4 *>(p.a + row_a[i] * pitch) + k0;
#pragma unroll
          for (int c = 0; c < 4; ++c) a[i][c] = q[c];
          sa[i] = *reinterpret_cast<const u32_any *>(p.a_scales + row_a[i] * p.kb + k0);
        }
      } else {   // the blocks past the end: zeros, at scale 1
        auto fetch = [&](const unsigned char *codes, const uint8_t *scales, int64_t row, u32x4 (&w)[4], uint32_t &s) {
          s = 0;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const bool in = k0 + c < p.kb;
            w[c] = in ? reinterpret_cast<const u32x4 *>(codes + row * pitch)[k0 + c] : u32x4{0, 0, 0, 0};
            s |= (in ? (uint32_t)scales[row * p.kb + k0 + c] : 127u) << (8 * c);
          }
        };
#pragma unroll
        for (int j = 0; j < NT; ++j) fetch(p.b, p.b_scales, row_b[j], b[j], sb[j]);
#pragma unroll
        for (int i = 0; i < MT; ++i) fetch(p.a, p.a_scales, row_a[i], a[i], sa[i]);
      }
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          acc[i][j] = mfma_fp4<0, 0>(b[j][0], a[i][0], acc[i][j], sb[j], sa[i]);
          acc[i][j] = mfma_fp4<1, 1>(b[j][1], a[i][1], acc[i][j], sb[j], sa[i]);
          acc[i][j] = mfma_fp4<2, 2>(b[j][2], a[i][2], acc[i][j], sb[j], sa[i]);
          acc[i][j] = mfma_fp4<3, 3>(b[j][3], a[i][3], acc[i][j], sb[j], sa[i]);
        }
    }
    // part[wave]: row-major [kRows][kCols]; lane: row i * 16 + li, columns j * 16 + 4 g ..
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) part[wave][((i * 16 + li) * kCols + j * 16 + 4 * g) / 4] = acc[i][j];
    __syncthreads();
    for (int e = t; e < kRows * kCols; e += kRowsWaves * 64) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < kRowsWaves; ++w) v += reinterpret_cast<const float *>(part[w])[e];
      const int m = m0 + e / kCols, n = n0 + e % kCols;
      if (m < p.m && n < p.n) finish_one<KIND>(p, m, n, v);
    }
    __syncthreads();
  }
}

template <int MT, int NT, int KIND>
LaunchStatus rows_launch(const MxOperands &p, uint32_t block_dim, hipStream_t stream) {
  const int tiles_n = (p.n + 16 * NT - 1) / (16 * NT), chunks_m = (p.m + 16 * MT - 1) / (16 * MT);
  const int64_t blocks = (int64_t)((tiles_n + kNumXCD - 1) / kNumXCD) * kNumXCD * chunks_m;
  if (blocks > 0x7fffffff) return invalid("mxfp4_matmul: too many output tiles");
  AFIR_LAUNCH("mxfp4_matmul_rows", (mxfp4_matmul_rows<MT, NT, KIND>), dim3(block_dim ? block_dim : (unsigned)blocks),
              dim3(kRowsWaves * 64), 0, stream, p, tiles_n, chunks_m, (int)blocks);
  return after_launch();
}

template <int KIND>
LaunchStatus matmul(const MxOperands &p, void *workspace, uint32_t block_dim, hipStream_t stream) {
  if (workspace && mxfp4_dma_supported(p)) return launch_mxfp4_dma(p, KIND, workspace, block_dim, stream);
  if (p.m <= 16) return rows_launch<1, 2, KIND>(p, block_dim, stream);
  if (p.m <= 32) return rows_launch<2, 2, KIND>(p, block_dim, stream);
  return rows_launch<4, 2, KIND>(p, block_dim, stream);
}

}  // namespace

size_t mxfp4_matmul_workspace(int64_t m, int64_t k, int64_t n) {
  if (m <= 0 || n <= 0 || k <= 0 || m > kMaxExtent || n > kMaxExtent || k > kMaxExtent) return 0;
  const int kb = (int)((k + kMxBlock - 1) / kMxBlock);
  MxOperands p{};
  p.m = (int)m;
  p.n = (int)n;
  p.kb = kb;
  return mxfp4_dma_supported(p) ? mxfp4_dma_workspace(m, kb, n) : 0;
}

LaunchStatus launch_mxfp4_matmul(const void *a, const void *a_scales, const void *b, const void *b_scales,
                                 const void *bias, void *out, int64_t m, int64_t k, int64_t n, float alpha,
                                 int elem_kind, void *workspace, uint32_t block_dim, hipStream_t stream) {
  if (m < 0 || k < 0 || n < 0) return invalid("mxfp4_matmul_add_leakyrelu: negative extent");
  if (m == 0 || n == 0) return ok_status();
  if (m > kMaxExtent || n > kMaxExtent || k > kMaxExtent) return invalid("mxfp4_matmul_add_leakyrelu: extent above 2^31");
  if (!out || (k > 0 && (!a || !a_scales || !b || !b_scales)))
    return invalid("mxfp4_matmul_add_leakyrelu: null tensor pointer");
  if (elem_kind < kElemF32 || elem_kind > kElemBF16)
    return invalid("mxfp4_matmul_add_leakyrelu: elem_type must be 0, 1 or 2");
  const uintptr_t elem = elem_kind == kElemF32 ? 4 : 2;
  if ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(bias)) % elem)
    return invalid("mxfp4_matmul_add_leakyrelu: tensor off its element's alignment");
  if (!aligned16(workspace)) return invalid("mxfp4_matmul_add_leakyrelu: workspace off a 16-byte boundary");
  if (!aligned16(a) || !aligned16(b))
    return invalid("mxfp4_matmul_add_leakyrelu: codes must start on a 16-byte boundary");
  const MxOperands p{static_cast<const unsigned char *>(a), static_cast<const unsigned char *>(b),
                     static_cast<const uint8_t *>(a_scales), static_cast<const uint8_t *>(b_scales), bias, out,
                     (int)m, (int)n, (int)((k + kMxBlock - 1) / kMxBlock), alpha};
  switch (elem_kind) {
    case kElemF32: return matmul<kElemF32>(p, workspace, block_dim, stream);
    case kElemF16: return matmul<kElemF16>(p, workspace, block_dim, stream);
    default: return matmul<kElemBF16>(p, workspace, block_dim, stream);
  }
}

}  // namespace afir
