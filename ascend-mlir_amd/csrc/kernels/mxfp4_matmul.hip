// out = leakyrelu(A B^T + bias) with A [M, K] and B [N, K] in MXFP4 (mxfp4.h) along K.
// Products of few rows; the dispatch of all of them.
#include "mxfp4_mfma.h"

namespace afir {

namespace {

typedef u32x4 u32x4_any __attribute__((aligned(1)));
constexpr int64_t kMaxExtent = 0x7ffffe00;   // extents and what a tile rounds them up to are 32-bit

template <int KIND>
__device__ __forceinline__ void finish_one(const MxOperands &p, int m, int n, float v) {
  if (p.bias) v += Elem<KIND>::load(p.bias, n);
  v = fmaxf(v, v * p.alpha);
  Elem<KIND>::store(p.out, (int64_t)m * p.n + n, v);
}

// Up to 16 rows of A: the time is that of reading B.  A workgroup owns 16 * NT columns and its eight
// wavefronts deal the blocks of K out among themselves, 16 blocks (256 bytes of a row) at a step.  Of a
// step, lane group g of a wavefront takes blocks g, 4 + g, 8 + g and 12 + g: each of the four loads then
// covers 64 adjacent bytes of each of the 16 rows, a quarter of the segments that four adjacent blocks per
// lane would touch.  The row's sixteen scales come as one 16-byte load and are shifted to the lane's byte.
// Everything of a step is requested before the first product; two workgroups on a compute unit cover the
// rest (requesting the next step ahead as well gained nothing: 9.3 against 9.0 us for one row at
// 8192 x 8192).  The eight partial sums meet in LDS and are added in a fixed order.
// One row: 9.0 us at 8192 x 8192 (4.0 TB/s; the bytes alone take 7.3 as a large copy moves them), 3.8 at
// 4096 x 4096; 16 rows at 8192 x 8192 9.7.
constexpr int kRowsWaves = 8;

// 16 rows' codes and scales of one step
struct RowsPiece {
  u32x4 w[4], s;
  // all 16 blocks of the step are there
  __device__ __forceinline__ void load(const unsigned char *codes, const uint8_t *scales, int64_t row, int kb, int step, int g) {
    const u32x4 *const q = reinterpret_cast<const u32x4 *>(codes + row * kb * kMxBlockBytes) + step * 16 + g;
#pragma unroll
    for (int c = 0; c < 4; ++c) w[c] = q[4 * c];
    s = *reinterpret_cast<const u32x4_any *>(scales + row * kb + step * 16);
  }
  // the blocks past the end: zeros, at scale 1
  __device__ __forceinline__ void load_tail(const unsigned char *codes, const uint8_t *scales, int64_t row, int kb, int step,
                                            int g) {
    uint32_t v[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int block = step * 16 + 4 * c + g;
      w[c] = block < kb ? reinterpret_cast<const u32x4 *>(codes + row * kb * kMxBlockBytes)[block] : u32x4{0, 0, 0, 0};
      v[c] = (block < kb ? (uint32_t)scales[row * kb + block] : 127u) << (8 * g);
    }
    s = u32x4{v[0], v[1], v[2], v[3]};
  }
};

template <int NT, int KIND>
__global__ __launch_bounds__(kRowsWaves * 64, 4) void mxfp4_matmul_rows(MxOperands p, int tiles_n, int chunks_m,
                                                                        int blocks) {
  constexpr int kCols = 16 * NT, kRows = 16;
  __shared__ f32x4 part[kRowsWaves][kRows * kCols / 4];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, li = lane & 15, g = lane >> 4;
  const int shift = 8 * g;
  for (int block = blockIdx.x; block < blocks; block += gridDim.x) {
    // chunks of A that share columns follow one another on one XCD, whose L2 then holds the columns' B
    const int xcd = block % kNumXCD, idx = block / kNumXCD;
    const int tile_n = (idx / chunks_m) * kNumXCD + xcd, m0 = (idx % chunks_m) * kRows;
    if (tile_n >= tiles_n) continue;
    const int n0 = tile_n * kCols;
    // rows past the end repeat the last one; what they give is not stored
    const int64_t row_a = m0 + li < p.m ? m0 + li : p.m - 1;
    int64_t row_b[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) row_b[j] = n0 + j * 16 + li < p.n ? n0 + j * 16 + li : p.n - 1;
    f32x4 acc[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    RowsPiece a, b[NT];
    auto multiply = [&]() {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const uint32_t sa = a.s[c] >> shift;
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[j] = mfma_fp4<0, 0>(b[j].w[c], a.w[c], acc[j], b[j].s[c] >> shift, sa);
      }
    };
    const int whole = p.kb / 16;   // steps of 16 blocks
    int step = wave;
    for (; step < whole; step += kRowsWaves) {
#pragma unroll
      for (int j = 0; j < NT; ++j) b[j].load(p.b, p.b_scales, row_b[j], p.kb, step, g);
      a.load(p.a, p.a_scales, row_a, p.kb, step, g);
      multiply();
    }
    if (step == whole && whole * 16 < p.kb) {
#pragma unroll
      for (int j = 0; j < NT; ++j) b[j].load_tail(p.b, p.b_scales, row_b[j], p.kb, step, g);
      a.load_tail(p.a, p.a_scales, row_a, p.kb, step, g);
      multiply();
    }
    // part[wave]: row-major [kRows][kCols]; lane: row li, columns j * 16 + 4 g ..
#pragma unroll
    for (int j = 0; j < NT; ++j) part[wave][(li * kCols + j * 16 + 4 * g) / 4] = acc[j];
    __syncthreads();
    for (int e = t; e < kRows * kCols; e += kRowsWaves * 64) {
      const int m = m0 + e / kCols, n = n0 + e % kCols;
      if (m < p.m && n < p.n) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < kRowsWaves; ++w) v += reinterpret_cast<const float *>(part[w])[e];
        finish_one<KIND>(p, m, n, v);
      }
    }
    __syncthreads();
  }
}

template <int NT, int KIND>
LaunchStatus rows_launch(const MxOperands &p, uint32_t block_dim, hipStream_t stream) {
  const int tiles_n = (p.n + 16 * NT - 1) / (16 * NT), chunks_m = (p.m + 15) / 16;
  const int64_t blocks = (int64_t)((tiles_n + kNumXCD - 1) / kNumXCD) * kNumXCD * chunks_m;
  // (a launch holds less than 2^32 threads, 2^23 workgroups of these; beyond the bound they take several places)
  constexpr int64_t kMost = (int64_t)1 << 20;
  if (blocks > 0x7fffffff - kMost) return invalid("mxfp4_matmul: too many output tiles");
  const int64_t grid = block_dim ? block_dim : blocks < kMost ? blocks : kMost;
  AFIR_LAUNCH("mxfp4_matmul_rows", (mxfp4_matmul_rows<NT, KIND>), dim3((unsigned)grid), dim3(kRowsWaves * 64), 0, stream, p,
              tiles_n, chunks_m, (int)blocks);
  return after_launch();
}

// K below 256 (or out of the other kernels' range): a wavefront takes the blocks of its TM * 16 rows of A and
// TN * 16 of B straight into registers, a slice of eight at a time.  Such a product is bound by its output:
// 8192 x 8192 x 64 into bfloat16 38 us (3.5 TB/s of output), 4096 x 4096 x 128 12.7 (102 on the kernel above).
template <int TM, int TN, int KIND>
__global__ __launch_bounds__(256) void mxfp4_matmul_direct(MxOperands p, int tiles_m, int tiles_n) {
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, li = lane & 15, g = lane >> 4;
  for (int tile = blockIdx.x; tile < tiles_m * tiles_n; tile += gridDim.x) {
    int tm, tn;
    map_tile(tile, tiles_m, tiles_n, tm, tn);
    const int m0 = (tm * 2 + wave / 2) * TM * 16, n0 = (tn * 2 + wave % 2) * TN * 16;
    f32x4 acc[TM][TN];
    start_from_bias<KIND>(p, n0, acc);
    // rows past the end repeat the last one; blocks past it are zeros at scale 1
    auto load = [&](const unsigned char *codes, const uint8_t *scales, int64_t row, int block, u32x4 &w, uint32_t &s) {
      const bool there = block < p.kb;
      const int64_t at = row * p.kb + block;
      w = there ? *reinterpret_cast<const u32x4 *>(codes + at * kMxBlockBytes) : u32x4{0, 0, 0, 0};
      s = there ? scales[at] : 127u;
    };
    for (int block = g; block - g < p.kb; block += kMxSliceBlocks) {
      u32x4 a[2][TM], b[2][TN];
      uint32_t sa[2][TM], sb[2][TN];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          const int row = n0 + j * 16 + li;
          load(p.b, p.b_scales, row < p.n ? row : p.n - 1, block + 4 * h, b[h][j], sb[h][j]);
        }
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          const int row = m0 + i * 16 + li;
          load(p.a, p.a_scales, row < p.m ? row : p.m - 1, block + 4 * h, a[h][i], sa[h][i]);
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
          for (int i = 0; i < TM; ++i) acc[i][j] = mfma_fp4<0, 0>(b[h][j], a[h][i], acc[i][j], sb[h][j], sa[h][i]);
    }
    store_outputs<KIND>(p, m0, n0, acc);
  }
}

template <int TM, int TN, int KIND>
LaunchStatus direct_launch(const MxOperands &p, uint32_t block_dim, hipStream_t stream) {
  const int tiles_m = (p.m + 32 * TM - 1) / (32 * TM), tiles_n = (p.n + 32 * TN - 1) / (32 * TN);
  const int64_t blocks = (int64_t)tiles_m * tiles_n;
  if (blocks > 0x7fffffff) return invalid("mxfp4_matmul: too many output tiles");
  AFIR_LAUNCH("mxfp4_matmul_direct", (mxfp4_matmul_direct<TM, TN, KIND>), dim3(block_dim ? block_dim : (unsigned)blocks),
              dim3(256), 0, stream, p, tiles_m, tiles_n);
  return after_launch();
}

// A tile per workgroup up to 64 rows (8.7 us against 15.8 on the kernel of few rows at 48 x 8200 x 4096), and while
// each compute unit gets at most one of 128 x 128 (512 x 8192 x 8192: 27 us, 28 on tiles in turn); beyond that
// tiles in turn (1024 x 8192 x 8192: 45 us against 55).
bool one_tile_each(const MxOperands &p) {
  return p.m > 16 && mxfp4_ring_supported(p) &&
         (p.m <= 64 || (int64_t)((p.m + 127) / 128) * ((p.n + 127) / 128) <= device_cus());
}

template <int KIND>
LaunchStatus matmul(const MxOperands &p, void *workspace, uint32_t block_dim, hipStream_t stream) {
  // Up to 16 rows; 16 columns a workgroup where that gives no compute unit a second one (4096 x 4096, one row:
  // 3.8 us against 4.8 with 32; 8192 x 8192, 16 rows: 11.8 against 9.6).
  if (p.m <= 16 && p.n <= 16 * device_cus()) return rows_launch<1, KIND>(p, block_dim, stream);
  if (p.m <= 16) return rows_launch<2, KIND>(p, block_dim, stream);
  if (one_tile_each(p)) return launch_mxfp4_ring(p, KIND, block_dim, stream);
  if (workspace && mxfp4_dma_supported(p)) return launch_mxfp4_dma(p, KIND, workspace, block_dim, stream);
  if (mxfp4_ring_supported(p)) return launch_mxfp4_ring(p, KIND, block_dim, stream);
  if (p.n > kMxMaxColumns) return rows_launch<2, KIND>(p, block_dim, stream);
  // (tiles of 64 x 64 while 128 x 128 ones would not fill the chip twice: 100 x 100 x 100 3.3 us against 5.9, but
  // 4096 x 4096 x 224 16.6 against 13.8)
  if ((int64_t)((p.m + 127) / 128) * ((p.n + 127) / 128) >= 2 * device_cus())
    return direct_launch<4, 4, KIND>(p, block_dim, stream);
  return direct_launch<2, 2, KIND>(p, block_dim, stream);
}

}  // namespace

size_t mxfp4_matmul_workspace(int64_t m, int64_t k, int64_t n) {
  if (m <= 0 || n <= 0 || k <= 0 || m > kMaxExtent || n > kMaxExtent || k > kMaxExtent) return 0;
  const int kb = (int)((k + kMxBlock - 1) / kMxBlock);
  MxOperands p{};
  p.m = (int)m;
  p.n = (int)n;
  p.kb = kb;
  return mxfp4_dma_supported(p) && !one_tile_each(p) ? mxfp4_dma_workspace(m, kb, n) : 0;
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
