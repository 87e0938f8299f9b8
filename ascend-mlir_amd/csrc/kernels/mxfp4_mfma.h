// The scaled fp4 matrix instruction and the operands of an MXFP4 product, shared by its kernels.
//
// v_mfma_scale_f32_16x16x128_f8f6f4 multiplies 16 x 128 by 128 x 16 codes and applies the block
// scales: lane l holds row l % 16, the 32 codes (16 bytes) of one block, and that block's scale
// byte; the four lanes of a row hold four different blocks.  Which four is free as long as both
// operands agree, since a sum over blocks has no order that matters.  Products of two codes are
// multiples of 1/4 up to 36, and the instruction adds them in float32.  B is the row operand, so a
// lane's four accumulators are four consecutive columns of one output row.
#pragma once

#include "kernels.h"
#include "mxfp4.h"

namespace afir {

typedef int i32x8 __attribute__((ext_vector_type(8)));

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

// Tiled kernels for products of more than a few rows (mxfp4_matmul_dma.hip).
bool mxfp4_dma_supported(const MxOperands &p);
size_t mxfp4_dma_workspace(int64_t m, int64_t kb, int64_t n);
LaunchStatus launch_mxfp4_dma(const MxOperands &p, int elem_kind, void *workspace, uint32_t block_dim, hipStream_t stream);

}  // namespace afir
