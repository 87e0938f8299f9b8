// The norms before and after a residual block, fused with the gate and the residual sum:
//
//   y = s * x + gate * (f * rstd(f)) * post_weight        rstd(v) = 1 / sqrt(mean(v^2) + eps)
//   h = y * rstd(y) * pre_weight                           (y unrounded)
//
// f is what the block gave, h what the next one takes, x and y the residual stream.  Without f, y
// is x itself (the norm ahead of the first block); without pre_weight there is no h.  A gate row
// serves rows_per_gate rows: 1 for a gate per element, a sequence's length for a modulated block, M
// for one learned row.
//
// Memory-bound: forward reads x and f and writes y and h, backward reads the gradients of y and h,
// y and f, and writes the gradients of x and f.  A row stays in registers from its load to its
// store: the two row sums (forward) and the two rounds of row sums (backward) are the only
// exchange between lanes.  All arithmetic is float32, each result rounded once as it is stored.
//
// bf16 8192 x 4096, a gate per 2048 rows: forward 46 us (5.8 TB/s), backward 87 and 8 for the join of the
// column sums (4.6 TB/s; some 350 vector instructions a row and wavefront keep the vector units half busy).
// float32 4096 x 4096: 45 and 88 us.  Rows above 8192 (16-bit types; 4096 x 16384): forward 107 us (5.0 TB/s), backward
// 359 (2.2 TB/s): two and four pieces a lane spill registers there.  Short rows leave lanes idle: a row has at least a
// wavefront (bf16 8192 x 256, three rows to a gate: 10 and 26 us).
#include <utility>

#include "kernels.h"
#include "mxfp4.h"

namespace afir {

namespace {

typedef f32x4 f32x4_u __attribute__((aligned(4)));

// What a lane holds of a row: ITEMS 16-byte pieces, lanes adjacent.
template <int KIND, int ITEMS>
struct Piece {
  uint32_t w[ITEMS][4];
};

// Row pieces of a lane; numbers past the row's end are zeros and add nothing to any sum.  (A
// 16-byte access needs the alignment of an element only, see mxfp4.h.)
template <int KIND, int LANES, int ITEMS>
__device__ __forceinline__ void load_row(const void *base, int64_t offset, int lane, uint32_t n, Piece<KIND, ITEMS> &p) {
  constexpr int V = Elem<KIND>::kPer16;
  typedef typename Elem<KIND>::type T;
  const T *row = static_cast<const T *>(base) + offset;
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const uint32_t e = (uint32_t)(lane + i * LANES) * V;   // (32-bit: the row's start stays a scalar)
    p.w[i][0] = p.w[i][1] = p.w[i][2] = p.w[i][3] = 0;
    if (e + V <= n) {
      const u32x4 v = *reinterpret_cast<const u32x4_u *>(row + e);
      p.w[i][0] = v.x; p.w[i][1] = v.y; p.w[i][2] = v.z; p.w[i][3] = v.w;
    } else {
#pragma unroll
      for (int j = 0; j < V - 1; ++j)
        if (e + j < n) {
          if constexpr (V == 8) p.w[i][j / 2] |= (uint32_t)row[e + j] << (16 * (j & 1));
          else p.w[i][j] = __float_as_uint(row[e + j]);
        }
    }
  }
}
template <int KIND, int LANES>
__device__ __forceinline__ void store_item(void *base, int64_t offset, uint32_t e, uint32_t n,
                                           const float (&v)[Elem<KIND>::kPer16]) {
  constexpr int V = Elem<KIND>::kPer16;
  typedef typename Elem<KIND>::type T;
  T *row = static_cast<T *>(base) + offset;
  if (e + V <= n) {
    uint32_t w[4];
    Elem<KIND>::pack(v, w);
    *reinterpret_cast<u32x4_u *>(row + e) = u32x4{w[0], w[1], w[2], w[3]};
  } else {
#pragma unroll
    for (int j = 0; j < V - 1; ++j)
      if (e + j < n) Elem<KIND>::store(row, e + j, v[j]);
  }
}

// Sums over the WAVES wavefronts of a row, in a fixed order.  Calls alternate between two slots
// (`turn`), so the barrier of a call also separates the reads of the call before it from the writes
// of the call after it, which go to the same slot.
template <int WAVES, int COUNT>
__device__ __forceinline__ void row_sums(float (&v)[COUNT], float *lds, int &turn, int wave) {
#pragma unroll
  for (int c = 0; c < COUNT; ++c) v[c] = wave_sum(v[c]);
  if constexpr (WAVES > 1) {
    f32x4 *const part = reinterpret_cast<f32x4 *>(lds) + turn * WAVES;
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) {
      f32x4 mine = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < COUNT; ++c) mine[c] = v[c];
      part[wave] = mine;
    }
    __syncthreads();
    // every 16 lanes take the WAVES sums, one each, and add them across (as wave_sum does within a row of 16)
    const int from = threadIdx.x & 15;
    const f32x4 one = from < WAVES ? part[from] : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < COUNT; ++c) {
      v[c] = dpp_add<0xB1>(one[c]);
      v[c] = dpp_add<0x4E>(v[c]);
      v[c] = dpp_add<0x141>(v[c]);
      v[c] = dpp_add<0x140>(v[c]);
    }
  }
}

// (at most 2^31 rows, and the launch holds rows_per_gate to them: a 64-bit division is some 100 instructions)
__device__ __forceinline__ int64_t gate_row(int64_t row, int64_t rows_per_gate) {
  return (uint32_t)row / (uint32_t)rows_per_gate;
}

__device__ __forceinline__ float rstd_of(float sum_of_squares, float inv_n, float eps) {
  return 1.0f / sqrtf(sum_of_squares * inv_n + eps);
}

// forward: rows of one wavefront, which need no barrier, are four to a workgroup
constexpr int threads_of(int waves) { return waves == 1 ? 256 : waves * 64; }

template <int KIND, int WAVES, int ITEMS>
__global__ __launch_bounds__(threads_of(WAVES)) void norm_gate_forward(NormGateArgs p) {
  constexpr int V = Elem<KIND>::kPer16, kLanes = WAVES * 64, kRowsHere = threads_of(WAVES) / kLanes;
  __shared__ __align__(16) float lds[2 * WAVES * 4];
  const int lane = threadIdx.x % kLanes, wave = lane >> 6;
  const uint32_t n = (uint32_t)p.n;
  Piece<KIND, ITEMS> post, pre;
  if (p.f) load_row<KIND, kLanes, ITEMS>(p.post_weight, 0, lane, n, post);
  if (p.h) load_row<KIND, kLanes, ITEMS>(p.pre_weight, 0, lane, n, pre);
  const int64_t stride = (int64_t)gridDim.x * kRowsHere;
  int64_t row = (int64_t)blockIdx.x * kRowsHere + threadIdx.x / kLanes;
  int turn = 0;
  Piece<KIND, ITEMS> x, f, gate;
  auto fetch = [&](int64_t r) {
    load_row<KIND, kLanes, ITEMS>(p.x, r * p.ld_x, lane, n, x);
    if (p.f) {
      load_row<KIND, kLanes, ITEMS>(p.f, r * p.ld_f, lane, n, f);
      if (p.gate) load_row<KIND, kLanes, ITEMS>(p.gate, gate_row(r, p.rows_per_gate) * p.ld_gate, lane, n, gate);
    }
  };
  if (row < p.m) fetch(row);
  for (; row < p.m; row += stride) {
    float y[ITEMS][V];
    if (p.f) {
      float sum[1] = {0.f};
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        float v[V];
        Elem<KIND>::unpack(f.w[i], v);
#pragma unroll
        for (int j = 0; j < V; ++j) sum[0] += v[j] * v[j];
      }
      row_sums<WAVES>(sum, lds, turn, wave);
      const float rf = rstd_of(sum[0], p.inv_n, p.eps);
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        float vx[V], vf[V], vg[V], vw[V];
        Elem<KIND>::unpack(x.w[i], vx);
        Elem<KIND>::unpack(f.w[i], vf);
        Elem<KIND>::unpack(post.w[i], vw);
        if (p.gate) Elem<KIND>::unpack(gate.w[i], vg);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float b = vf[j] * rf * vw[j];
          y[i][j] = p.residual_scale * vx[j] + (p.gate ? vg[j] * b : b);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) Elem<KIND>::unpack(x.w[i], y[i]);
    }
    if (row + stride < p.m) fetch(row + stride);
    if (p.y)
#pragma unroll
      for (int i = 0; i < ITEMS; ++i)
        store_item<KIND, kLanes>(p.y, row * p.ld_y, (uint32_t)(lane + i * kLanes) * V, n, y[i]);
    if (p.h) {
      float sum[1] = {0.f};
#pragma unroll
      for (int i = 0; i < ITEMS; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) sum[0] += y[i][j] * y[i][j];
      row_sums<WAVES>(sum, lds, turn, wave);
      const float ry = rstd_of(sum[0], p.inv_n, p.eps);
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        float vw[V], o[V];
        Elem<KIND>::unpack(pre.w[i], vw);
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = y[i][j] * ry * vw[j];
        store_item<KIND, kLanes>(p.h, row * p.ld_h, (uint32_t)(lane + i * kLanes) * V, n, o);
      }
    }
  }
}

template <int KIND, int WAVES, int ITEMS>
LaunchStatus forward_launch(const NormGateArgs &p, uint32_t block_dim, hipStream_t stream) {
  constexpr int kRowsHere = threads_of(WAVES) / (WAVES * 64);
  int64_t blocks = (p.m + kRowsHere - 1) / kRowsHere;
  const int64_t most = (int64_t)device_cus() * 8;
  if (blocks > most) blocks = most;
  if (block_dim) blocks = block_dim;
  AFIR_LAUNCH("norm_gate_forward", (norm_gate_forward<KIND, WAVES, ITEMS>), dim3((unsigned)blocks),
              dim3(threads_of(WAVES)), 0, stream, p);
  return after_launch();
}

template <int KIND>
LaunchStatus forward(const NormGateArgs &p, uint32_t block_dim, hipStream_t stream) {
  const int64_t pieces = (p.n + Elem<KIND>::kPer16 - 1) / Elem<KIND>::kPer16;
  if (pieces <= 64) return forward_launch<KIND, 1, 1>(p, block_dim, stream);
  if (pieces <= 128) return forward_launch<KIND, 2, 1>(p, block_dim, stream);
  if (pieces <= 256) return forward_launch<KIND, 4, 1>(p, block_dim, stream);
  if (pieces <= 512) return forward_launch<KIND, 8, 1>(p, block_dim, stream);
  if (pieces <= 1024) return forward_launch<KIND, 16, 1>(p, block_dim, stream);
  if constexpr (kNormMaxColumns / Elem<KIND>::kPer16 > 2048)
    if (pieces > 2048) return forward_launch<KIND, 16, 4>(p, block_dim, stream);
  return forward_launch<KIND, 16, 2>(p, block_dim, stream);
}

// ---- backward ----
//
// With yn = y rstd(y), fn = f rstd(f) and a = dh * pre_weight:
//   t  = dy + rstd(y) (a - yn mean(a yn))            the gradient of the unscaled sum
//   dx = s t          b = t gate post_weight
//   df = rstd(f) (b - fn mean(b fn))
//   dpost_weight = sum over rows of t gate fn         dpre_weight = sum over rows of dh yn
//   dgate = post_weight * sum over the gate row's rows of t fn
// mean(a yn) and both rstd need one round of row sums, mean(b fn) a second one; nothing is kept
// from the forward pass but y.
//
// The column sums: the wavefronts of a row walk a stretch of rows and keep their share of its columns
// in registers.  A workgroup has eight wavefronts where a row has fewer, adds its stretches' sums in LDS
// and writes one row of float32 partial sums, which a second kernel adds; all in a fixed order.  A
// stretch never straddles two gate rows unless it covers each of them whole, so either the gate is
// one row throughout a workgroup (kOneGate: the partial sum is that of t fn, which serves dgate and,
// weighted with the gate, dpost_weight), or dgate's rows are finished within the stretch.
// (bf16 8192 x 32: 20 us; with a partial row per stretch 48, most of it their sum.)
constexpr int groups_of(int waves) { return waves < 8 ? 8 / waves : 1; }   // stretches of a workgroup
struct Stretches {       // stretch i: rows from (i / per_span) * span + (i % per_span) * rows
  uint32_t span;         // rows of one gate row, or of several whole ones
  uint32_t per_span, rows, count;   // (per_span and count: whole workgroups of stretches)
  bool one_gate;
};

inline Stretches plan_stretches(int64_t m, int64_t rows_per_gate, bool gate, int64_t stretches, int groups) {
  const int64_t rows = (m + stretches - 1) / stretches, per_gate = gate && rows_per_gate < m ? rows_per_gate : m;
  // Whole gate rows, as many as fit; or one longer than `rows`, where splitting it over a workgroup's stretches
  // would leave many of them idle (bf16 8192 x 256, 3 rows to a gate: 27 us against 75; 16 rows: 68 against 24).
  const bool whole = gate && per_gate <= rows * (groups + 1) / 2;
  const int64_t span = whole && per_gate < rows ? rows / per_gate * per_gate : per_gate;
  int64_t per_span = whole ? 1 : (per_gate + rows - 1) / rows, count = (m + span - 1) / span;
  Stretches s;
  s.one_gate = !whole || per_gate == m;
  if (s.one_gate) per_span = (per_span + groups - 1) / groups * groups;
  count = (count * per_span + groups - 1) / groups * groups;
  s.span = (uint32_t)span;
  s.per_span = (uint32_t)per_span;
  s.rows = (uint32_t)((span + per_span - 1) / per_span);
  s.count = (uint32_t)count;
  return s;
}

template <int V>
__device__ __forceinline__ void store_sums(float *row, uint32_t e, uint32_t n, const float (&v)[V]) {
  if (e + V <= n) {
#pragma unroll
    for (int j = 0; j < V; j += 4) *reinterpret_cast<f32x4_u *>(row + e + j) = f32x4{v[j], v[j + 1], v[j + 2], v[j + 3]};
  } else {
#pragma unroll
    for (int j = 0; j < V - 1; ++j)
      if (e + j < n) row[e + j] = v[j];
  }
}

template <int KIND, int WAVES, int ITEMS, bool kOneGate>
__global__ __launch_bounds__(WAVES * groups_of(WAVES) * 64, 4) void norm_gate_backward(NormGateGradArgs p, Stretches s) {
  constexpr int V = Elem<KIND>::kPer16, kLanes = WAVES * 64;
  constexpr int kGroups = groups_of(WAVES);
  constexpr bool kAhead = ITEMS == 1;
  // rows of several wavefronts meet at barriers, so stretches of one workgroup take the same number of steps
  constexpr bool kMayIdle = kGroups > 1 && WAVES > 1;
  __shared__ __align__(16) float sums_lds[kGroups][2 * WAVES * 4];
  __shared__ f32x4 joined[kGroups > 1 ? kGroups - 1 : 1][kGroups > 1 ? V / 4 : 1][kLanes];
  const int lane = threadIdx.x % kLanes, wave = lane >> 6;
  const int group = kGroups == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / kLanes);   // (a scalar, like its rows)
  float *const lds = sums_lds[group];
  const uint32_t n = (uint32_t)p.n;
  Piece<KIND, ITEMS> post, pre;
  if (!kOneGate && p.f) load_row<KIND, kLanes, ITEMS>(p.post_weight, 0, lane, n, post);
  if (p.dh) load_row<KIND, kLanes, ITEMS>(p.pre_weight, 0, lane, n, pre);
  int turn = 0;
  for (uint32_t place = blockIdx.x; place < s.count / kGroups; place += gridDim.x) {
    const uint32_t stretch = place * kGroups + group;
    const int64_t first = (int64_t)(stretch / s.per_span) * s.span, r0 = first + (int64_t)(stretch % s.per_span) * s.rows;
    int64_t r1 = r0 + s.rows < first + s.span ? r0 + s.rows : first + s.span;
    r1 = r1 < p.m ? r1 : p.m;
    float acc_post[ITEMS][V], acc_pre[ITEMS][V], acc_gate[kOneGate ? 1 : ITEMS][V];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        acc_post[i][j] = acc_pre[i][j] = 0.f;
        if constexpr (!kOneGate) acc_gate[i][j] = 0.f;
      }
    Piece<KIND, ITEMS> dy, dh, y, f, gate;
    if constexpr (kMayIdle) dy = dh = y = f = gate = Piece<KIND, ITEMS>{};
    auto fetch = [&](int64_t r) {
      if (p.dy) load_row<KIND, kLanes, ITEMS>(p.dy, r * p.ld_dy, lane, n, dy);
      if (p.dh) {
        load_row<KIND, kLanes, ITEMS>(p.dh, r * p.ld_dh, lane, n, dh);
        load_row<KIND, kLanes, ITEMS>(p.y, r * p.ld_y, lane, n, y);
      }
      if (p.f) {
        load_row<KIND, kLanes, ITEMS>(p.f, r * p.ld_f, lane, n, f);
        if (!kOneGate && p.gate) load_row<KIND, kLanes, ITEMS>(p.gate, gate_row(r, p.rows_per_gate) * p.ld_gate, lane, n, gate);
      }
    };
    if (r0 < r1) {
      if (kOneGate && p.f) load_row<KIND, kLanes, ITEMS>(p.post_weight, 0, lane, n, post);
      if (kOneGate && p.f && p.gate)
        load_row<KIND, kLanes, ITEMS>(p.gate, gate_row(first, p.rows_per_gate) * p.ld_gate, lane, n, gate);
      fetch(r0);
    }
    // gate post_weight: held through the stretch where it is one row and there are registers for it
    constexpr bool kHeld = kOneGate && ITEMS == 1;
    float held[V];
    auto weights = [&](int i, const Piece<KIND, ITEMS> &gate_now, float (&w)[V]) {
      float vg[V];
      Elem<KIND>::unpack(post.w[i], w);
      if (!p.gate) return;
      Elem<KIND>::unpack(gate_now.w[i], vg);
#pragma unroll
      for (int j = 0; j < V; ++j) w[j] *= vg[j];
    };
    if (kHeld && p.f && r0 < r1) weights(0, gate, held);
    auto weight_row = [&](int i, const Piece<KIND, ITEMS> &gate_now, float (&w)[V]) {
      if constexpr (kHeld) {
#pragma unroll
        for (int j = 0; j < V; ++j) w[j] = held[j];
      } else {
        weights(i, gate_now, w);
      }
    };
    auto unpack_a = [&](int i, float (&v)[V]) {   // a = dh pre_weight
      float vw[V];
      Elem<KIND>::unpack(dh.w[i], v);
      Elem<KIND>::unpack(pre.w[i], vw);
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] *= vw[j];
    };
    const int64_t end = kMayIdle ? r0 + s.rows : r1;
    for (int64_t row = r0; row < end; ++row) {
      const bool active = !kMayIdle || row < r1;
      float sums[3] = {0.f, 0.f, 0.f};   // y^2, a y, f^2
      float a[V], t[ITEMS][V];   // (a stays where there are registers, or is formed anew)
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        if (p.dh) {
          float vy[V];
          Elem<KIND>::unpack(y.w[i], vy);
          unpack_a(i, a);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            sums[0] += vy[j] * vy[j];
            sums[1] += a[j] * vy[j];
          }
        }
        if (p.f) {
          float vf[V];
          Elem<KIND>::unpack(f.w[i], vf);
#pragma unroll
          for (int j = 0; j < V; ++j) sums[2] += vf[j] * vf[j];
        }
      }
      row_sums<WAVES>(sums, lds, turn, wave);
      const float ry = rstd_of(sums[0], p.inv_n, p.eps), rf = rstd_of(sums[2], p.inv_n, p.eps);
      const float my = ry * sums[1] * p.inv_n;   // mean(a yn)
      float dot[1] = {0.f};                      // b f
      if (active) {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
          if (p.dy) Elem<KIND>::unpack(dy.w[i], t[i]);
          else
#pragma unroll
            for (int j = 0; j < V; ++j) t[i][j] = 0.f;
          if (p.dh) {
            float vy[V], vd[V];
            Elem<KIND>::unpack(y.w[i], vy);
            Elem<KIND>::unpack(dh.w[i], vd);
            if (ITEMS > 1 || !kOneGate) unpack_a(i, a);
#pragma unroll
            for (int j = 0; j < V; ++j) {
              const float yn = vy[j] * ry;
              t[i][j] += ry * (a[j] - yn * my);
              acc_pre[i][j] += vd[j] * yn;
            }
          }
          if (p.f) {
            float vf[V], vg[V], vw[V];
            Elem<KIND>::unpack(f.w[i], vf);
            weight_row(i, gate, vw);
            if (!kOneGate && p.gate) Elem<KIND>::unpack(gate.w[i], vg);
#pragma unroll
            for (int j = 0; j < V; ++j) {
              const float tf = t[i][j] * (vf[j] * rf);
              dot[0] += t[i][j] * vw[j] * vf[j];
              if constexpr (kOneGate) {
                acc_post[i][j] += tf;
              } else {
                acc_post[i][j] += p.gate ? vg[j] * tf : tf;
                acc_gate[i][j] += tf;
              }
            }
          }
        }
      }
      // the next row is requested here, ahead of this row's stores and second round of sums; rows of
      // several pieces per lane have no registers for two rows and request theirs when they are done
      const Piece<KIND, ITEMS> f_here = f, gate_here = gate;
      if (kAhead && row + 1 < r1) fetch(row + 1);
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        float o[V];
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = p.residual_scale * t[i][j];
        if (active) store_item<KIND, kLanes>(p.dx, row * p.ld_dx, (uint32_t)(lane + i * kLanes) * V, n, o);
      }
      if (p.f) {
        row_sums<WAVES>(dot, lds, turn, wave);
        const float mf = rf * dot[0] * p.inv_n;   // mean(b fn)
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
          float o[V], vf[V], vw[V];
          Elem<KIND>::unpack(f_here.w[i], vf);
          weight_row(i, gate_here, vw);
#pragma unroll
          for (int j = 0; j < V; ++j) o[j] = rf * (t[i][j] * vw[j] - vf[j] * rf * mf);
          if (active) store_item<KIND, kLanes>(p.df, row * p.ld_df, (uint32_t)(lane + i * kLanes) * V, n, o);
        }
        if constexpr (!kOneGate) {
          if (active && ((uint32_t)(row + 1) % (uint32_t)p.rows_per_gate == 0 || row + 1 == p.m)) {
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
              float o[V], vw[V];
              Elem<KIND>::unpack(post.w[i], vw);
#pragma unroll
              for (int j = 0; j < V; ++j) {
                o[j] = acc_gate[i][j] * vw[j];
                acc_gate[i][j] = 0.f;
              }
              store_item<KIND, kLanes>(p.dgate, gate_row(row, p.rows_per_gate) * p.n, (uint32_t)(lane + i * kLanes) * V, n, o);
            }
          }
        }
      }
      if (!kAhead && row + 1 < r1) fetch(row + 1);
    }
    if constexpr (kGroups > 1) {
      auto join = [&](float (&acc)[V]) {
        __syncthreads();
        if (group > 0)
#pragma unroll
          for (int j = 0; j < V; j += 4) joined[group - 1][j / 4][lane] = f32x4{acc[j], acc[j + 1], acc[j + 2], acc[j + 3]};
        __syncthreads();
        if (group == 0)
#pragma unroll
          for (int other = 0; other < kGroups - 1; ++other)
#pragma unroll
            for (int j = 0; j < V; ++j) acc[j] += joined[other][j / 4][lane][j % 4];
      };
      if (p.f) join(acc_post[0]);
      if (p.dh) join(acc_pre[0]);
    }
    float *const part_post = p.partial + (int64_t)place * p.n;
    float *const part_pre = p.partial + ((int64_t)(s.count / kGroups) + place) * p.n;
    if (group == 0)
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        const uint32_t e = (uint32_t)(lane + i * kLanes) * V;
        if (p.f) store_sums(part_post, e, n, acc_post[i]);
        if (p.dh) store_sums(part_pre, e, n, acc_pre[i]);
      }
  }
}

// Adds the partial rows: blockIdx.y 0 gives dpre_weight, 1 dpost_weight, 2 + g gate row g (kOneGate
// launches with a gate).  32 columns per workgroup, a line of a partial row, four to a lane; 64 groups of
// lanes share the rows, eight rows in flight each.  Their sums are added in a fixed order: the groups of a
// wavefront across its lanes, the wavefronts through LDS.
constexpr int kJoinColumns = 32, kJoinLanes = kJoinColumns / 4, kJoinGroups = 64, kJoinWaves = kJoinGroups * kJoinLanes / 64;
template <int KIND>
__global__ __launch_bounds__(kJoinWaves * 64) void norm_gate_join(NormGateGradArgs p, Stretches s, int64_t column_tiles) {
  __shared__ f32x4 lds[kJoinWaves][kJoinLanes];
  const int four = threadIdx.x % kJoinLanes, group = threadIdx.x / kJoinLanes;
  const int what = blockIdx.y;
  if ((what == 0 && !p.dh) || (what == 1 && !p.f)) return;
  const float *const part = p.partial + (what == 0 ? (int64_t)s.count * p.n : 0);
  const uint32_t first = what < 2 ? 0 : (what - 2) * s.per_span, last = what < 2 ? s.count : first + s.per_span;
  const bool weighted = what == 1 && s.one_gate && p.gate;
  for (int64_t tile = blockIdx.x; tile < column_tiles; tile += gridDim.x) {
    const int64_t e0 = tile * kJoinColumns + four * 4;
    const int here = p.n - e0 < 4 ? (p.n > e0 ? (int)(p.n - e0) : 0) : 4;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    auto add = [&](uint32_t r, auto weighted_tag) {
      f32x4 x = {0.f, 0.f, 0.f, 0.f}, w = {1.f, 1.f, 1.f, 1.f};
      if (here == 4) {
        x = *reinterpret_cast<const f32x4_u *>(part + (int64_t)r * p.n + e0);
      } else {
#pragma unroll
        for (int j = 0; j < 3; ++j)
          if (j < here) x[j] = part[(int64_t)r * p.n + e0 + j];
      }
      if constexpr (decltype(weighted_tag)::value) {
        const int64_t at = (int64_t)(r / s.per_span) * p.ld_gate + e0;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (j < here) w[j] = Elem<KIND>::load(p.gate, at + j);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] += x[j] * w[j];
    };
    if (weighted) {
#pragma unroll 4
      for (uint32_t r = first + group; r < last; r += kJoinGroups) add(r, std::true_type{});
    } else {
#pragma unroll 8
      for (uint32_t r = first + group; r < last; r += kJoinGroups) add(r, std::false_type{});
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      // lanes 8, 16 and 32 apart hold the same columns
      v[j] += __shfl_xor(v[j], 8);
      v[j] += __shfl_xor(v[j], 16);
      v[j] += __shfl_xor(v[j], 32);
    }
    if ((threadIdx.x & 63) < kJoinLanes) lds[threadIdx.x >> 6][four] = v;
    __syncthreads();
    const int64_t e = tile * kJoinColumns + threadIdx.x;
    if (threadIdx.x < kJoinColumns && e < p.n) {
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < kJoinWaves; ++w) sum += reinterpret_cast<const float *>(lds[w])[threadIdx.x];
      if (what == 0) Elem<KIND>::store(p.dpre_weight, e, sum);
      else if (what == 1) Elem<KIND>::store(p.dpost_weight, e, sum);
      else Elem<KIND>::store(p.dgate, (what - 2) * p.n + e, sum * Elem<KIND>::load(p.post_weight, e));
    }
    __syncthreads();
  }
}

// Wavefronts a row of the backward pass is spread over, and 16-byte pieces per lane.
struct RowShape {
  int waves, items;
};
inline RowShape backward_shape(int64_t n, int elem_kind) {
  const int64_t pieces = elem_kind == kElemF32 ? (n + 3) / 4 : (n + 7) / 8;
  for (int waves = 1; waves <= 16; waves *= 2)
    if (pieces <= 64 * waves) return {waves, 1};
  return {16, pieces <= 2048 ? 2 : 4};
}
inline Stretches backward_stretches(int64_t m, int64_t n, int64_t rows_per_gate, bool gate, int elem_kind) {
  const int waves = backward_shape(n, elem_kind).waves;
  return plan_stretches(m, rows_per_gate, gate, (int64_t)device_cus() * (waves <= 8 ? 16 / waves : 1), groups_of(waves));
}

template <int KIND, int WAVES, int ITEMS>
LaunchStatus backward_launch(const NormGateGradArgs &p, const Stretches &s, uint32_t block_dim, hipStream_t stream) {
  constexpr int kGroups = groups_of(WAVES);
  const int64_t most = (int64_t)1 << 20, all = s.count / kGroups, blocks = block_dim ? block_dim : all < most ? all : most;
  if (s.one_gate)
    AFIR_LAUNCH("norm_gate_backward", (norm_gate_backward<KIND, WAVES, ITEMS, true>), dim3((unsigned)blocks),
                dim3(WAVES * kGroups * 64), 0, stream, p, s);
  else
    AFIR_LAUNCH("norm_gate_backward", (norm_gate_backward<KIND, WAVES, ITEMS, false>), dim3((unsigned)blocks),
                dim3(WAVES * kGroups * 64), 0, stream, p, s);
  const LaunchStatus st = after_launch();
  if (st.code) return st;
  const int64_t column_tiles = (p.n + kJoinColumns - 1) / kJoinColumns;
  Stretches partial = s;   // in rows of partial sums
  partial.count /= kGroups;
  if (s.one_gate) partial.per_span /= kGroups;
  const int64_t gates = s.one_gate && p.f && p.gate ? (p.m + p.rows_per_gate - 1) / p.rows_per_gate : 0;
  AFIR_LAUNCH("norm_gate_join", (norm_gate_join<KIND>), dim3((unsigned)column_tiles, (unsigned)(2 + gates)),
              dim3(kJoinWaves * 64), 0, stream, p, partial, column_tiles);
  return after_launch();
}

template <int KIND>
LaunchStatus backward(const NormGateGradArgs &p, uint32_t block_dim, hipStream_t stream) {
  const Stretches s = backward_stretches(p.m, p.n, p.rows_per_gate, p.f && p.gate, KIND);
  const RowShape shape = backward_shape(p.n, KIND);
  if constexpr (kNormMaxColumns / Elem<KIND>::kPer16 > 2048)
    if (shape.items == 4) return backward_launch<KIND, 16, 4>(p, s, block_dim, stream);
  if (shape.items == 2) return backward_launch<KIND, 16, 2>(p, s, block_dim, stream);
  switch (shape.waves) {
    case 1: return backward_launch<KIND, 1, 1>(p, s, block_dim, stream);
    case 2: return backward_launch<KIND, 2, 1>(p, s, block_dim, stream);
    case 4: return backward_launch<KIND, 4, 1>(p, s, block_dim, stream);
    case 8: return backward_launch<KIND, 8, 1>(p, s, block_dim, stream);
    default: return backward_launch<KIND, 16, 1>(p, s, block_dim, stream);
  }
}

// Whether two results of m rows of n numbers share one: rows of one stride by what the starts are apart,
// modulo the stride; rows of different strides as soon as the stretches of memory that they span do.
bool results_overlap(const void *a, int64_t ld_a, const void *b, int64_t ld_b, int64_t m, int64_t n, int64_t size) {
  if (reinterpret_cast<uintptr_t>(a) > reinterpret_cast<uintptr_t>(b)) {
    std::swap(a, b);
    std::swap(ld_a, ld_b);
  }
  const uint64_t apart = (reinterpret_cast<uintptr_t>(b) - reinterpret_cast<uintptr_t>(a)) / (uint64_t)size;
  if (apart >= (uint64_t)((m - 1) * ld_a + n)) return false;
  if (ld_a != ld_b) return true;
  const int64_t rows = (int64_t)apart / ld_a, within = (int64_t)apart % ld_a;   // b starts in row `rows` of a, or behind it
  return within < n || (within > ld_a - n && rows + 1 < m);
}

}  // namespace

LaunchStatus launch_norm_gate_residual(const NormGateArgs &args, int elem_kind, uint32_t block_dim, hipStream_t stream) {
  NormGateArgs p = args;
  if (p.m < 0 || p.n < 0) return invalid("norm_gate_residual: negative extent");
  if (p.m == 0 || p.n == 0) return ok_status();
  if (elem_kind < kElemF32 || elem_kind > kElemBF16) return invalid("norm_gate_residual: elem_type must be 0, 1 or 2");
  if (p.m > 0x7fffffff || p.n > kNormMaxColumns)
    return invalid("norm_gate_residual: more than 2^31 rows or rows of more than 16384 numbers");
  if (!p.x) return invalid("norm_gate_residual: null tensor pointer");
  if (!p.f && !p.h) return invalid("norm_gate_residual: neither a block output nor a norm of the sum is asked for");
  if (p.f && (!p.post_weight || !p.y)) return invalid("norm_gate_residual: f needs post_weight and y");
  if (!p.f && (p.y || p.gate)) return invalid("norm_gate_residual: without f there is no y and no gate");
  if (p.h && !p.pre_weight) return invalid("norm_gate_residual: h needs pre_weight");
  if (p.rows_per_gate < 1) return invalid("norm_gate_residual: rows_per_gate must be positive");
  if (!(p.eps >= 0.f)) return invalid("norm_gate_residual: eps must not be negative");
  const int64_t most = ((int64_t)1 << 46) / p.m;
  for (int64_t ld : {p.ld_x, p.f ? p.ld_f : p.n, p.gate ? p.ld_gate : p.n, p.y ? p.ld_y : p.n, p.h ? p.ld_h : p.n})
    if (ld < p.n || ld > most) return invalid("norm_gate_residual: row stride below the row's length or out of range");
  const uintptr_t elem = elem_kind == kElemF32 ? 4 : 2;
  for (const void *q : {p.x, p.f, p.gate, p.post_weight, p.pre_weight, (const void *)p.y, (const void *)p.h})
    if (reinterpret_cast<uintptr_t>(q) % elem) return invalid("norm_gate_residual: tensor off its element's alignment");
  if (p.y && p.h && results_overlap(p.y, p.ld_y, p.h, p.ld_h, p.m, p.n, elem))
    return invalid("norm_gate_residual: y and h are two results and must not overlap");
  p.inv_n = (float)(1.0 / (double)p.n);
  if (p.rows_per_gate > p.m) p.rows_per_gate = p.m;
  switch (elem_kind) {
    case kElemF32: return forward<kElemF32>(p, block_dim, stream);
    case kElemF16: return forward<kElemF16>(p, block_dim, stream);
    default: return forward<kElemBF16>(p, block_dim, stream);
  }
}

size_t norm_gate_backward_workspace(int64_t m, int64_t n, int64_t rows_per_gate, bool gate, int elem_kind) {
  if (m <= 0 || n <= 0 || rows_per_gate < 1) return 0;
  return (size_t)(backward_stretches(m, n, rows_per_gate, gate, elem_kind).count /
                  groups_of(backward_shape(n, elem_kind).waves)) * (size_t)n * 2 * sizeof(float);
}

LaunchStatus launch_norm_gate_residual_backward(const NormGateGradArgs &args, int elem_kind, uint32_t block_dim,
                                                hipStream_t stream) {
  NormGateGradArgs p = args;
  if (p.m < 0 || p.n < 0) return invalid("norm_gate_residual_backward: negative extent");
  if (elem_kind < kElemF32 || elem_kind > kElemBF16)
    return invalid("norm_gate_residual_backward: elem_type must be 0, 1 or 2");
  if (p.m == 0 || p.n == 0) return invalid("norm_gate_residual_backward: empty tensors have no gradients to write");
  if (p.m > 0x7fffffff || p.n > kNormMaxColumns)
    return invalid("norm_gate_residual_backward: more than 2^31 rows or rows of more than 16384 numbers");
  if (!p.f && !p.dh) return invalid("norm_gate_residual_backward: neither a block output nor a norm of the sum is given");
  if (!p.dx || (!p.dy && !p.dh)) return invalid("norm_gate_residual_backward: null tensor pointer");
  if (p.dh && (!p.y || !p.pre_weight || !p.dpre_weight))
    return invalid("norm_gate_residual_backward: dh needs y, pre_weight and dpre_weight");
  if (p.f && (!p.post_weight || !p.df || !p.dpost_weight))
    return invalid("norm_gate_residual_backward: f needs post_weight, df and dpost_weight");
  if (!p.f && p.gate) return invalid("norm_gate_residual_backward: without f there is no gate");
  if (!p.gate != !p.dgate) return invalid("norm_gate_residual_backward: gate and dgate go together");
  if (!p.partial) return invalid("norm_gate_residual_backward: null workspace");
  if (p.rows_per_gate < 1) return invalid("norm_gate_residual_backward: rows_per_gate must be positive");
  if (!(p.eps >= 0.f)) return invalid("norm_gate_residual_backward: eps must not be negative");
  const int64_t most = ((int64_t)1 << 46) / p.m;
  for (int64_t ld : {p.dy ? p.ld_dy : p.n, p.dh ? p.ld_dh : p.n, p.dh ? p.ld_y : p.n, p.f ? p.ld_f : p.n,
                     p.gate ? p.ld_gate : p.n, p.ld_dx, p.f ? p.ld_df : p.n})
    if (ld < p.n || ld > most)
      return invalid("norm_gate_residual_backward: row stride below the row's length or out of range");
  const uintptr_t elem = elem_kind == kElemF32 ? 4 : 2;
  for (const void *q : {p.dy, p.dh, p.y, p.f, p.gate, p.post_weight, p.pre_weight, (const void *)p.dx, (const void *)p.df,
                        (const void *)p.dpost_weight, (const void *)p.dgate, (const void *)p.dpre_weight})
    if (reinterpret_cast<uintptr_t>(q) % elem)
      return invalid("norm_gate_residual_backward: tensor off its element's alignment");
  if (reinterpret_cast<uintptr_t>(p.partial) % 4) return invalid("norm_gate_residual_backward: workspace off a 4-byte boundary");
  if (p.f && results_overlap(p.dx, p.ld_dx, p.df, p.ld_df, p.m, p.n, elem))
    return invalid("norm_gate_residual_backward: dx and df are two results and must not overlap");
  p.inv_n = (float)(1.0 / (double)p.n);
  if (p.rows_per_gate > p.m) p.rows_per_gate = p.m;
  switch (elem_kind) {
    case kElemF32: return backward<kElemF32>(p, block_dim, stream);
    case kElemF16: return backward<kElemF16>(p, block_dim, stream);
    default: return backward<kElemBF16>(p, block_dim, stream);
  }
}

}  // namespace afir
