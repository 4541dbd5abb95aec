// residual_norm.hip -- the norms after a block and before the next one, with
// the block's gate and residual scale, and their gradients.
//
//   xhat = x r1,  r1 = (mean x^2 + eps)^-1/2      the block's output x, by row
//   y = residual + scale gate w1 xhat              the residual stream
//   h = w2 yhat,  yhat = y r2,  r2 = (mean y^2 + eps)^-1/2
//
//   b = w2 dh,  e = dy + r2 (b - yhat mean(b yhat))     the residual's gradient
//   a = scale gate w1 e,  dx = r1 (a - xhat mean(a xhat))
//   dw2 = sum dh yhat;  with a gate by column c = sum e xhat, dw1 = scale gate c,
//   dgate = scale w1 c;  with a gate by element c = sum e gate xhat, dw1 = scale c,
//   dgate = scale e w1 xhat.  Sums over the rows.
//
// Without the norm after the block xhat = x, r1 = 1 and dx = a.
// Memory bounds both directions: a row of each input is read once and stays in
// the registers of its lanes until its outputs are written; y goes into the
// second norm in 32 bits, before its rounding.
#include <algorithm>

#include "norm.hpp"

namespace sporder_hip {

namespace {

struct BlockArgs {
  int64_t rows, dim, x_stride, res_stride, gate_stride, y_stride, h_stride;
  const void *x, *residual, *gate, *gate_vector, *w1, *w2;
  void *y, *h;
  float *post_rstd, *rstd;
  float scale, eps;
  int vector_type;
  bool post;
};

struct BlockGradArgs {
  int64_t rows, dim, dy_stride, dh_stride, x_stride, y_stride, gate_stride;
  int64_t dx_stride, dres_stride, dgate_stride;
  const void *dy, *dh, *x, *y, *gate, *gate_vector, *w1, *w2;
  const float *post_rstd, *rstd;
  void *dx, *dres, *dgate;
  float *partial; // [grid][2][dim] sums c and dw2, or null
  float scale;
  int vector_type;
  bool post;
};

// scale w1 gate of a lane's columns.
template <bool LOOSE, int VEC, int L, int C, typename A>
__device__ __forceinline__ void load_gain(const A &a, int lane, float (&out)[C][VEC]) {
  float gate[C][VEC];
  load_vector<LOOSE, VEC, L>(a.w1, a.vector_type, a.dim, 1.0f, lane, out);
  load_vector<LOOSE, VEC, L>(a.gate_vector, a.vector_type, a.dim, 1.0f, lane, gate);
#pragma unroll
  for (int c = 0; c < C; ++c) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) out[c][i] *= a.scale * gate[c][i];
  }
}

// A row's words from an optional tensor.
template <bool LOOSE, int VEC, int L, int C, typename T>
__device__ __forceinline__ void fetch_row(const void *base, int64_t row, int64_t stride, int64_t dim,
                                          bool live, int lane, Words<T, VEC> (&out)[C]) {
  const T *const p = static_cast<const T *>(base) + row * stride;
#pragma unroll
  for (int c = 0; c < C; ++c)
    out[c] = fetch_words<LOOSE, false, VEC>(p, (c * L + lane) * VEC, dim, live && base);
}

template <int VEC, int C, typename T>
__device__ __forceinline__ void to_floats(const Words<T, VEC> (&w)[C], float (&out)[C][VEC]) {
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const auto q = __builtin_bit_cast(Pack<T, VEC>, w[c]);
#pragma unroll
    for (int i = 0; i < VEC; ++i) out[c][i] = static_cast<float>(q.v[i]);
  }
}

template <bool LOOSE, int VEC, int L, int C, typename T>
__device__ __forceinline__ void put_row(T *p, int64_t dim, int lane, const float (&v)[C][VEC]) {
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int col = (c * L + lane) * VEC;
    if (col < dim) put<LOOSE, VEC>(p + col, dim - col, v[c]);
  }
}

// A row per L lanes, held in registers between its read and both outputs' writes: 16,384
// rows of 4,096 bfloat16 with a residual in 99 us (5.4 TB/s), by torch operations 1,242.
// Loose accesses of 16-bit elements: 97,560 rows of 1,025 in 258 us (3.1 TB/s) where 1,024 take 149,
// with 85 million turns of the first-level caches for 13 million; rows of 100 and 101 in 278 and
// 311, the address units busy 89 % of the time.
template <typename T, bool LOOSE, int VEC, int L, int C>
__global__ void __launch_bounds__(norm_block(L)) block_norm_kernel(BlockArgs a) {
  constexpr int kGroups = norm_block(L) / L;
  __shared__ float shared[2][1][norm_block(L) / kWave];
  RowSum<L, 1> row_sum{shared};
  const int lane = threadIdx.x % L, group = threadIdx.x / L;
  const float dim = static_cast<float>(a.dim);

  float gain[C][VEC], w2[C][VEC];
  load_gain<LOOSE, VEC, L>(a, lane, gain);
  load_vector<LOOSE, VEC, L>(a.w2, a.vector_type, a.dim, 1.0f, lane, w2);

  for (int64_t first = static_cast<int64_t>(blockIdx.x) * kGroups; first < a.rows;
       first += static_cast<int64_t>(gridDim.x) * kGroups) {
    const int64_t row = first + group;
    const bool live = row < a.rows;
    Words<T, VEC> raw_x[C], raw_r[C], raw_g[C];
    fetch_row<LOOSE, VEC, L>(a.x, row, a.x_stride, a.dim, live, lane, raw_x);
    fetch_row<LOOSE, VEC, L>(a.residual, row, a.res_stride, a.dim, live, lane, raw_r);
    if (a.gate) fetch_row<LOOSE, VEC, L>(a.gate, row, a.gate_stride, a.dim, live, lane, raw_g);
    float v[C][VEC], r[C][VEC];
    to_floats<VEC>(raw_x, v);
    float s[1] = {0.0f};
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) s[0] += v[c][i] * v[c][i];
    }
    float r1 = 1.0f;
    if (a.post) {
      row_sum(s);
      r1 = 1.0f / sqrtf(s[0] / dim + a.eps);
    }
    if (a.gate) {
      float g[C][VEC];
      to_floats<VEC>(raw_g, g);
#pragma unroll
      for (int c = 0; c < C; ++c) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[c][i] *= g[c][i];
      }
    }
    to_floats<VEC>(raw_r, r);
    s[0] = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        v[c][i] = r[c][i] + v[c][i] * r1 * gain[c][i];
        // Past the row's end an infinite r1 would make 0 a NaN.
        s[0] += (c * L + lane) * VEC + (LOOSE ? i : 0) < a.dim ? v[c][i] * v[c][i] : 0.0f;
      }
    }
    row_sum(s);
    const float r2 = 1.0f / sqrtf(s[0] / dim + a.eps);
    if (!live) continue;
    put_row<LOOSE, VEC, L>(static_cast<T *>(a.y) + row * a.y_stride, a.dim, lane, v);
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[c][i] *= r2 * w2[c][i];
    }
    put_row<LOOSE, VEC, L>(static_cast<T *>(a.h) + row * a.h_stride, a.dim, lane, v);
    if (lane == 0) {
      a.post_rstd[row] = r1;
      a.rstd[row] = r2;
    }
  }
}

__device__ __forceinline__ float element_of(const void *p, int type, int64_t i) {
  float v = 1.0f;
  if (p) with_type(p, type, [&](auto *q) { v = static_cast<float>(q[i]); });
  return v;
}

// Rows that no workgroup's registers hold: three passes over each, by elements (2,000
// rows of 40,000 floats in 655 us, 2.0 TB/s, bfloat16 720, 0.9).
template <typename T> __global__ void __launch_bounds__(1024) block_norm_long_kernel(BlockArgs a) {
  __shared__ float shared[2][1][1024 / kWave];
  RowSum<1024, 1> row_sum{shared};
  const float dim = static_cast<float>(a.dim);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *const x = static_cast<const T *>(a.x) + row * a.x_stride;
    const T *const res = static_cast<const T *>(a.residual) + row * a.res_stride;
    const T *const gate = static_cast<const T *>(a.gate) + row * a.gate_stride;
    T *const y = static_cast<T *>(a.y) + row * a.y_stride, *const h = static_cast<T *>(a.h) + row * a.h_stride;
    float s[1] = {0.0f};
    float r1 = 1.0f;
    if (a.post) {
      for (int64_t i = threadIdx.x; i < a.dim; i += 1024) s[0] += static_cast<float>(x[i]) * static_cast<float>(x[i]);
      row_sum(s);
      r1 = 1.0f / sqrtf(s[0] / dim + a.eps);
    }
    auto value = [&](int64_t i) {
      float v = static_cast<float>(x[i]);
      if (a.gate) v *= static_cast<float>(gate[i]);
      const float gain = element_of(a.w1, a.vector_type, i) *
                         (a.scale * element_of(a.gate_vector, a.vector_type, i));
      return (a.residual ? static_cast<float>(res[i]) : 0.0f) + v * r1 * gain;
    };
    s[0] = 0.0f;
    for (int64_t i = threadIdx.x; i < a.dim; i += 1024) {
      const float v = value(i);
      s[0] += v * v;
    }
    row_sum(s);
    const float r2 = 1.0f / sqrtf(s[0] / dim + a.eps);
    for (int64_t i = threadIdx.x; i < a.dim; i += 1024) {
      const float v = value(i);
      y[i] = static_cast<T>(v);
      h[i] = static_cast<T>(v * r2 * element_of(a.w2, a.vector_type, i));
    }
    if (threadIdx.x == 0) {
      a.post_rstd[row] = r1;
      a.rstd[row] = r2;
    }
  }
}

// 2,449,029 rows of 128 floats in 1,472 us (5.1 TB/s), 16,384 of 4,096 bfloat16 with a gate by
// row in 211 (5.1 TB/s); rows of 16-bit elements of odd length, whose accesses are loose, 1.8 to
// 3.4 TB/s (such an access takes the caches six times as many turns; below).
// The gradients by element, and the workgroup's sums over its rows by column,
// kept in registers and written as one row of partial sums at the end.  No
// atomics: the order of every sum is fixed by the grid.
template <typename T, bool LOOSE, int VEC, int L, int C>
__global__ void __launch_bounds__(norm_block(L)) block_norm_grad_kernel(BlockGradArgs a) {
  constexpr int kGroups = norm_block(L) / L;
  constexpr int kSpan = L * C * VEC; // columns that a group holds
  constexpr int kBlockWaves = norm_block(L) / kWave;
  constexpr int kRowWaves = L > kWave ? L / kWave : 1;
  constexpr int kSlots = kBlockWaves / kRowWaves;
  __shared__ float shared[2][1][kBlockWaves];
  __shared__ float joined[L < 256 ? kSlots : 1][L < 256 ? kSpan : 1];
  RowSum<L, 1> row_sum{shared};
  const int lane = threadIdx.x % L, group = threadIdx.x / L;
  const float dim = static_cast<float>(a.dim);

  float gain[C][VEC], w2[C][VEC], c1[C][VEC] = {}, c2[C][VEC] = {};
  load_gain<LOOSE, VEC, L>(a, lane, gain);
  load_vector<LOOSE, VEC, L>(a.w2, a.vector_type, a.dim, 1.0f, lane, w2);

  for (int64_t first = static_cast<int64_t>(blockIdx.x) * kGroups; first < a.rows;
       first += static_cast<int64_t>(gridDim.x) * kGroups) {
    const int64_t row = first + group;
    const bool live = row < a.rows;
    Words<T, VEC> raw_y[C], raw_dh[C], raw_dy[C], raw_x[C], raw_g[C];
    const float r1 = live ? a.post_rstd[row] : 0.0f, r2 = live ? a.rstd[row] : 0.0f;
    fetch_row<LOOSE, VEC, L>(a.y, row, a.y_stride, a.dim, live, lane, raw_y);
    fetch_row<LOOSE, VEC, L>(a.dh, row, a.dh_stride, a.dim, live, lane, raw_dh);
    fetch_row<LOOSE, VEC, L>(a.dy, row, a.dy_stride, a.dim, live, lane, raw_dy);
    fetch_row<LOOSE, VEC, L>(a.x, row, a.x_stride, a.dim, live, lane, raw_x);
    if (a.gate) fetch_row<LOOSE, VEC, L>(a.gate, row, a.gate_stride, a.dim, live, lane, raw_g);
    float b[C][VEC], u[C][VEC], e[C][VEC];
    to_floats<VEC>(raw_y, u);
    to_floats<VEC>(raw_dh, b);
    float s[1] = {0.0f};
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const bool inside = (c * L + lane) * VEC + (LOOSE ? i : 0) < a.dim;
        u[c][i] *= inside ? r2 : 0.0f; // 0 times an infinite r2 is no 0
        c2[c][i] += b[c][i] * u[c][i];
        b[c][i] *= w2[c][i];
        s[0] += b[c][i] * u[c][i];
      }
    }
    row_sum(s);
    const float m1 = s[0] / dim;
    to_floats<VEC>(raw_dy, e);
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) e[c][i] += (b[c][i] - u[c][i] * m1) * r2;
    }
    if (live)
      put_row<LOOSE, VEC, L>(static_cast<T *>(a.dres) + row * a.dres_stride, a.dim, lane, e);
    to_floats<VEC>(raw_x, u);
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        u[c][i] *= (c * L + lane) * VEC + (LOOSE ? i : 0) < a.dim ? r1 : 0.0f;
    }
    if (a.gate) {
      float g[C][VEC];
#pragma unroll
      for (int c = 0; c < C; ++c) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) g[c][i] = e[c][i] * gain[c][i] * u[c][i];
      }
      if (live)
        put_row<LOOSE, VEC, L>(static_cast<T *>(a.dgate) + row * a.dgate_stride, a.dim, lane, g);
      to_floats<VEC>(raw_g, g);
#pragma unroll
      for (int c = 0; c < C; ++c) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) e[c][i] *= g[c][i];
      }
    }
    s[0] = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        c1[c][i] += e[c][i] * u[c][i];
        e[c][i] *= gain[c][i];
        s[0] += e[c][i] * u[c][i];
      }
    }
    float m2 = 0.0f;
    if (a.post) {
      row_sum(s);
      m2 = s[0] / dim;
    }
    if (!live) continue;
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) e[c][i] = (e[c][i] - u[c][i] * m2) * r1;
    }
    put_row<LOOSE, VEC, L>(static_cast<T *>(a.dx) + row * a.dx_stride, a.dim, lane, e);
  }

  if (!a.partial) return;
  float *const out = a.partial + static_cast<int64_t>(blockIdx.x) * 2 * a.dim;
  if constexpr (L >= 256) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const int64_t col = (c * L + lane) * VEC + i;
        if (col < a.dim) {
          out[col] = c1[c][i];
          out[a.dim + col] = c2[c][i];
        }
      }
    }
  } else {
    // Groups of a wave by lane exchange, then the waves through LDS.
    const int slot = threadIdx.x / kWave / kRowWaves;
#pragma unroll
    for (int what = 0; what < 2; ++what) {
      if (what) __syncthreads();
#pragma unroll
      for (int c = 0; c < C; ++c) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          float v = what ? c2[c][i] : c1[c][i];
#pragma unroll
          for (int j = L; j < kWave; j <<= 1) v += lane_xor_f32(v, j);
          if (L >= kWave || threadIdx.x % kWave < L) joined[slot][(c * L + lane) * VEC + i] = v;
        }
      }
      __syncthreads();
      for (int col = threadIdx.x; col < kSpan; col += norm_block(L)) {
        if (col >= a.dim) continue;
        float v = 0.0f;
#pragma unroll
        for (int k = 0; k < kSlots; ++k) v += joined[k][col];
        out[what * a.dim + col] = v;
      }
    }
  }
}

// Rows whose column sums and weights would not fit the registers besides: 1,024 lanes of
// 16 elements, tensor after tensor, the weights read for each row (L2 holds them) and
// the column sums in LDS.  3,900 rows of 16,384 bfloat16 with a gate by row in 230 us (4.5 TB/s;
// by three passes 1,417), floats 402 (5.1 TB/s).
constexpr int kWideLanes = 1024, kWideDim = kWideLanes * 16;
template <typename T, bool LOOSE, int VEC>
__global__ void __launch_bounds__(kWideLanes) block_norm_grad_wide_kernel(BlockGradArgs a) {
  constexpr int L = kWideLanes, C = 16 / VEC;
  __shared__ float shared[2][1][L / kWave];
  __shared__ __attribute__((aligned(16))) float sums[2][kWideDim];
  RowSum<L, 1> row_sum{shared};
  const int lane = threadIdx.x;
  const float dim = static_cast<float>(a.dim);
#pragma unroll
  for (int c = 0; c < C; ++c) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) sums[0][(c * L + lane) * VEC + i] = sums[1][(c * L + lane) * VEC + i] = 0.0f;
  }
  auto add = [&](int which, const float (&v)[C][VEC], const float (&w)[C][VEC]) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) sums[which][(c * L + lane) * VEC + i] += v[c][i] * w[c][i];
    }
  };
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const float r1 = a.post_rstd[row], r2 = a.rstd[row];
    int place = lane;
    asm volatile("" : "+v"(place)); // else the weights' addresses fill the registers before the loop
    Words<T, VEC> raw[C], raw_two[C];
    float b[C][VEC], u[C][VEC], w[C][VEC];
    fetch_row<LOOSE, VEC, L>(a.y, row, a.y_stride, a.dim, true, lane, raw);
    fetch_row<LOOSE, VEC, L>(a.dh, row, a.dh_stride, a.dim, true, lane, raw_two);
    load_vector<LOOSE, VEC, L>(a.w2, a.vector_type, a.dim, 1.0f, place, w);
    to_floats<VEC>(raw, u);
    to_floats<VEC>(raw_two, b);
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        u[c][i] *= (c * L + lane) * VEC + (LOOSE ? i : 0) < a.dim ? r2 : 0.0f;
    }
    add(1, b, u);
    float s[1] = {0.0f};
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        b[c][i] *= w[c][i];
        s[0] += b[c][i] * u[c][i];
      }
    }
    fetch_row<LOOSE, VEC, L>(a.dy, row, a.dy_stride, a.dim, true, lane, raw);
    fetch_row<LOOSE, VEC, L>(a.x, row, a.x_stride, a.dim, true, lane, raw_two);
    row_sum(s);
    const float m1 = s[0] / dim;
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) b[c][i] = (b[c][i] - u[c][i] * m1) * r2;
    }
    to_floats<VEC>(raw, u);
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) b[c][i] += u[c][i];
    }
    put_row<LOOSE, VEC, L>(static_cast<T *>(a.dres) + row * a.dres_stride, a.dim, lane, b);
    fetch_row<LOOSE, VEC, L>(a.gate, row, a.gate_stride, a.dim, true, lane, raw);
    load_gain<LOOSE, VEC, L>(a, place, w);
    to_floats<VEC>(raw_two, u);
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        u[c][i] *= (c * L + lane) * VEC + (LOOSE ? i : 0) < a.dim ? r1 : 0.0f;
    }
    if (a.gate) {
      T *const dgate = static_cast<T *>(a.dgate) + row * a.dgate_stride;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int col = (c * L + lane) * VEC;
        const auto gate = __builtin_bit_cast(Pack<T, VEC>, raw[c]);
        float g[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          g[i] = b[c][i] * w[c][i] * u[c][i];
          b[c][i] *= static_cast<float>(gate.v[i]);
        }
        if (col < a.dim) put<LOOSE, VEC>(dgate + col, a.dim - col, g);
      }
    }
    add(0, b, u);
    s[0] = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        b[c][i] *= w[c][i];
        s[0] += b[c][i] * u[c][i];
      }
    }
    float m2 = 0.0f;
    if (a.post) {
      row_sum(s);
      m2 = s[0] / dim;
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) b[c][i] = (b[c][i] - u[c][i] * m2) * r1;
    }
    put_row<LOOSE, VEC, L>(static_cast<T *>(a.dx) + row * a.dx_stride, a.dim, lane, b);
  }
  if (!a.partial) return;
  float *const out = a.partial + static_cast<int64_t>(blockIdx.x) * 2 * a.dim;
  __syncthreads();
  for (int64_t i = lane; i < a.dim; i += L) {
    out[i] = sums[0][i];
    out[a.dim + i] = sums[1][i];
  }
}

// Rows that no workgroup's registers hold: three passes over each, by elements;
// the column sums stay in the workgroup's partial row (2,000 rows of 20,000 floats in 592 us,
// 1.6 TB/s, bfloat16 757, 0.6).
template <typename T>
__global__ void __launch_bounds__(1024) block_norm_grad_long_kernel(BlockGradArgs a) {
  __shared__ float shared[2][1][1024 / kWave];
  RowSum<1024, 1> row_sum{shared};
  const float dim = static_cast<float>(a.dim);
  float *const out = a.partial ? a.partial + static_cast<int64_t>(blockIdx.x) * 2 * a.dim : nullptr;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *const dy = static_cast<const T *>(a.dy) + row * a.dy_stride;
    const T *const dh = static_cast<const T *>(a.dh) + row * a.dh_stride;
    const T *const x = static_cast<const T *>(a.x) + row * a.x_stride;
    const T *const y = static_cast<const T *>(a.y) + row * a.y_stride;
    const T *const gate = static_cast<const T *>(a.gate) + row * a.gate_stride;
    T *const dx = static_cast<T *>(a.dx) + row * a.dx_stride;
    T *const dres = static_cast<T *>(a.dres) + row * a.dres_stride;
    T *const dgate = static_cast<T *>(a.dgate) + row * a.dgate_stride;
    const float r1 = a.post_rstd[row], r2 = a.rstd[row];
    const bool again = row != blockIdx.x;
    float s[1] = {0.0f};
    for (int64_t i = threadIdx.x; i < a.dim; i += 1024) {
      const float d = a.dh ? static_cast<float>(dh[i]) : 0.0f, u = static_cast<float>(y[i]) * r2;
      s[0] += d * element_of(a.w2, a.vector_type, i) * u;
      if (out) out[a.dim + i] = (again ? out[a.dim + i] : 0.0f) + d * u;
    }
    row_sum(s);
    const float m1 = s[0] / dim;
    auto stream_grad = [&](int64_t i) {
      const float d = a.dh ? static_cast<float>(dh[i]) : 0.0f, u = static_cast<float>(y[i]) * r2;
      return (a.dy ? static_cast<float>(dy[i]) : 0.0f) +
             (d * element_of(a.w2, a.vector_type, i) - u * m1) * r2;
    };
    auto gain = [&](int64_t i) {
      return element_of(a.w1, a.vector_type, i) *
             (a.scale * element_of(a.gate_vector, a.vector_type, i));
    };
    s[0] = 0.0f;
    for (int64_t i = threadIdx.x; i < a.dim; i += 1024) {
      const float e = stream_grad(i), u = static_cast<float>(x[i]) * r1;
      const float t = a.gate ? e * static_cast<float>(gate[i]) : e;
      s[0] += t * gain(i) * u;
      if (out) out[i] = (again ? out[i] : 0.0f) + t * u;
    }
    row_sum(s);
    const float m2 = a.post ? s[0] / dim : 0.0f;
    for (int64_t i = threadIdx.x; i < a.dim; i += 1024) {
      const float e = stream_grad(i), u = static_cast<float>(x[i]) * r1, k = gain(i);
      dres[i] = static_cast<T>(e);
      if (a.gate) dgate[i] = static_cast<T>(e * k * u);
      const float t = a.gate ? e * static_cast<float>(gate[i]) : e;
      dx[i] = static_cast<T>((t * k - u * m2) * r1);
    }
  }
}

// Column sums of the partial rows and what they make: 64 columns per workgroup,
// 16 threads per column over interleaved rows, added up in LDS.
constexpr int kSumRows = 16;
struct BlockSumArgs {
  const float *partial;
  int64_t count, dim;
  const void *gate_vector, *w1;
  void *dgate, *dw1, *dw2;
  float scale;
  int vector_type;
};

__global__ void __launch_bounds__(kWave *kSumRows) block_norm_sum_kernel(BlockSumArgs a) {
  __shared__ float part[kSumRows][kWave];
  const int x = threadIdx.x % kWave, y = threadIdx.x / kWave;
  const int64_t col = static_cast<int64_t>(blockIdx.x) * kWave + x; // of 2 dim
  float v = 0.0f;
  if (col < 2 * a.dim) {
#pragma unroll 8
    for (int64_t r = y; r < a.count; r += kSumRows) v += a.partial[r * 2 * a.dim + col];
  }
  part[y][x] = v;
  __syncthreads();
  if (y != 0 || col >= 2 * a.dim) return;
  v = 0.0f;
#pragma unroll
  for (int k = 0; k < kSumRows; ++k) v += part[k][x];
  if (col >= a.dim) {
    if (a.dw2) store_typed(a.dw2, a.vector_type, col - a.dim, v);
    return;
  }
  if (a.dw1)
    store_typed(a.dw1, a.vector_type, col,
                v * (a.scale * element_of(a.gate_vector, a.vector_type, col)));
  if (a.dgate)
    store_typed(a.dgate, a.vector_type, col, v * (a.scale * element_of(a.w1, a.vector_type, col)));
}

// Zero rows have zero sums.
__global__ void block_norm_zero_kernel(BlockSumArgs a) {
  const int64_t i = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x;
  if (i >= a.dim) return;
  if (a.dw1) store_typed(a.dw1, a.vector_type, i, 0.0f);
  if (a.dw2) store_typed(a.dw2, a.vector_type, i, 0.0f);
  if (a.dgate) store_typed(a.dgate, a.vector_type, i, 0.0f);
}

constexpr int64_t kMostGroups = 256 * 8;
constexpr int64_t kBlockMostDim = 512 * 32;     // forward, in registers
constexpr int64_t kBlockGradMostDim = 512 * 16; // backward

// f with a row's lanes and the elements of each, as types.
template <typename F> int32_t forward_lanes(int64_t dim, F &&f) {
  if (dim <= 16) return f(Const<2>{}, Const<8>{});
  if (dim <= 32) return f(Const<4>{}, Const<8>{});
  if (dim <= 64) return f(Const<8>{}, Const<8>{});
  if (dim <= 128) return f(Const<16>{}, Const<8>{});
  if (dim <= 256) return f(Const<32>{}, Const<8>{});
  if (dim <= 512) return f(Const<64>{}, Const<8>{});
  if (dim <= 1024) return f(Const<64>{}, Const<16>{});
  if (dim <= 2048) return f(Const<128>{}, Const<16>{});
  if (dim <= 4096) return f(Const<256>{}, Const<16>{});
  if (dim <= 8192) return f(Const<512>{}, Const<16>{});
  return f(Const<512>{}, Const<32>{});
}

template <typename F> int32_t backward_lanes(int64_t dim, F &&f) {
  if (dim <= 16) return f(Const<2>{}, Const<8>{});
  if (dim <= 32) return f(Const<4>{}, Const<8>{});
  if (dim <= 64) return f(Const<8>{}, Const<8>{});
  if (dim <= 128) return f(Const<16>{}, Const<8>{});
  if (dim <= 256) return f(Const<32>{}, Const<8>{});
  if (dim <= 512) return f(Const<64>{}, Const<8>{});
  if (dim <= 1024) return f(Const<128>{}, Const<8>{});
  if (dim <= 2048) return f(Const<256>{}, Const<8>{});
  if (dim <= 4096) return f(Const<512>{}, Const<8>{});
  return f(Const<512>{}, Const<16>{});
}

// Rows at a time of a workgroup of the gradient, by backward_lanes.
int64_t grad_groups(int64_t dim) {
  int lanes = 2;
  while (lanes < 512 && lanes * 8 < dim) lanes *= 2;
  return norm_block(lanes) / lanes;
}

// Workgroups of the gradient, each with a partial row of 2 dim floats: at most enough to fill
// the card, few enough that the partial rows stay small beside the rows themselves (eight
// turns of rows for each), but no fewer than the CUs while each has two turns.
int64_t grad_blocks(int64_t rows, int64_t dim) {
  const int64_t most = dim > 4096 ? 512 : 1024, turns = ceil_div64(rows, grad_groups(dim));
  return std::min(most, std::max(ceil_div64(turns, 8), std::min<int64_t>(256, ceil_div64(turns, 2))));
}

template <typename T> int32_t block_typed(const BlockArgs &a, void *stream) {
  if (a.dim > kBlockMostDim)
    return launch(block_norm_long_kernel<T>, dim3(std::min(a.rows, kMostGroups)), dim3(1024), stream, a);
  constexpr int kVec = 16 / sizeof(T);
  const bool whole = row_vec(sizeof(T), a.dim, {a.x_stride, a.res_stride, a.gate_stride, a.y_stride, a.h_stride},
                             {a.x, a.residual, a.gate, a.gate_vector, a.w1, a.w2, a.y, a.h}) == kVec;
  return forward_lanes(a.dim, [&](auto lanes, auto elements) {
    constexpr int L = decltype(lanes)::value, E = decltype(elements)::value;
    const dim3 grid(std::min(ceil_div64(a.rows, norm_block(L) / L), kMostGroups));
    return whole ? launch(block_norm_kernel<T, false, kVec, L, E / kVec>, grid, dim3(norm_block(L)), stream, a)
                 : launch(block_norm_kernel<T, true, kVec, L, E / kVec>, grid, dim3(norm_block(L)), stream, a);
  });
}

template <typename T> int32_t block_grad_typed(const BlockGradArgs &a, int64_t blocks, void *stream) {
  if (a.dim > kWideDim) return launch(block_norm_grad_long_kernel<T>, dim3(blocks), dim3(1024), stream, a);
  constexpr int kVec = 16 / sizeof(T);
  const bool whole = row_vec(sizeof(T), a.dim,
                             {a.dy_stride, a.dh_stride, a.x_stride, a.y_stride, a.gate_stride, a.dx_stride,
                              a.dres_stride, a.dgate_stride},
                             {a.dy, a.dh, a.x, a.y, a.gate, a.gate_vector, a.w1, a.w2, a.dx, a.dres,
                              a.dgate}) == kVec;
  if (a.dim > kBlockGradMostDim)
    return whole ? launch(block_norm_grad_wide_kernel<T, false, kVec>, dim3(blocks), dim3(kWideLanes), stream, a)
                 : launch(block_norm_grad_wide_kernel<T, true, kVec>, dim3(blocks), dim3(kWideLanes), stream, a);
  return backward_lanes(a.dim, [&](auto lanes, auto elements) {
    constexpr int L = decltype(lanes)::value, E = decltype(elements)::value;
    return whole ? launch(block_norm_grad_kernel<T, false, kVec, L, E / kVec>, dim3(blocks),
                          dim3(norm_block(L)), stream, a)
                 : launch(block_norm_grad_kernel<T, true, kVec, L, E / kVec>, dim3(blocks),
                          dim3(norm_block(L)), stream, a);
  });
}

} // namespace

} // namespace sporder_hip

using namespace sporder_hip;

extern "C" {

int32_t sporder_residual_norm(void *stream, int32_t type, int32_t vector_type, int64_t rows,
                              int64_t dim, int64_t x_stride, const void *d_x,
                              int64_t residual_stride, const void *d_residual,
                              int32_t gate_by_row, int64_t gate_stride, const void *d_gate,
                              const void *d_post_weight, const void *d_weight, float scale,
                              float eps, int32_t post_norm, int64_t y_stride, void *d_y,
                              int64_t h_stride, void *d_h, float *d_post_rstd, float *d_rstd) {
  if (!type_known(type) || !type_known(vector_type) || rows < 0 || dim < 1 || dim > kMostDim ||
      x_stride < 0 || residual_stride < 0 || gate_stride < 0 || y_stride < 0 || h_stride < 0 ||
      (rows > 1 && (y_stride < dim || h_stride < dim)) || !(eps >= 0.0f) ||
      (!post_norm && d_post_weight))
    return SPORDER_BAD_ARGUMENT;
  if (rows == 0) return SPORDER_OK;
  if (!d_x || !d_y || !d_h || !d_post_rstd || !d_rstd) return SPORDER_BAD_ARGUMENT;
  const bool by_row = gate_by_row && d_gate;
  const BlockArgs a{rows, dim, x_stride, d_residual ? residual_stride : 0, by_row ? gate_stride : 0,
                    y_stride, h_stride, d_x, d_residual, by_row ? d_gate : nullptr,
                    by_row ? nullptr : d_gate, d_post_weight, d_weight, d_y, d_h, d_post_rstd,
                    d_rstd, scale, eps, vector_type, post_norm != 0};
  if (type == SPORDER_TYPE_BF16) return block_typed<bf16_t>(a, stream);
  if (type == SPORDER_TYPE_F16) return block_typed<f16_t>(a, stream);
  return block_typed<float>(a, stream);
}

size_t sporder_residual_norm_grad_work_bytes(int64_t rows, int64_t dim) {
  if (rows < 1 || dim < 1 || dim > kMostDim) return 0;
  return static_cast<size_t>(grad_blocks(rows, dim)) * 2 * dim * sizeof(float);
}

int32_t sporder_residual_norm_grad(void *stream, int32_t type, int32_t vector_type, int64_t rows,
                                   int64_t dim, int64_t dy_stride, const void *d_dy,
                                   int64_t dh_stride, const void *d_dh, int64_t x_stride,
                                   const void *d_x, int64_t y_stride, const void *d_y,
                                   const float *d_post_rstd, const float *d_rstd,
                                   int32_t gate_by_row, int64_t gate_stride, const void *d_gate,
                                   const void *d_post_weight, const void *d_weight, float scale,
                                   int32_t post_norm, int64_t dx_stride, void *d_dx,
                                   int64_t dresidual_stride, void *d_dresidual,
                                   int64_t dgate_stride, void *d_dgate, void *d_dpost_weight,
                                   void *d_dweight, void *d_work, size_t work_bytes) {
  if (!type_known(type) || !type_known(vector_type) || rows < 0 || dim < 1 || dim > kMostDim ||
      dy_stride < 0 || dh_stride < 0 || x_stride < 0 || y_stride < 0 || gate_stride < 0 ||
      dx_stride < 0 || dresidual_stride < 0 || dgate_stride < 0 ||
      (rows > 1 && (dx_stride < dim || dresidual_stride < dim)) ||
      (!post_norm && (d_post_weight || d_dpost_weight)))
    return SPORDER_BAD_ARGUMENT;
  const bool by_row = gate_by_row && d_gate;
  if (!d_gate && d_dgate) return SPORDER_BAD_ARGUMENT;
  void *const dgate_vector = by_row ? nullptr : d_dgate;
  const bool columns = dgate_vector || d_dpost_weight || d_dweight;
  BlockSumArgs sums{nullptr, 0, dim, by_row ? nullptr : d_gate, d_post_weight, dgate_vector,
                    d_dpost_weight, d_dweight, scale, vector_type};
  if (rows == 0) {
    if (!columns) return SPORDER_OK;
    return launch(block_norm_zero_kernel, dim3(ceil_div64(dim, 256)), dim3(256), stream, sums);
  }
  if (!d_x || !d_y || !d_post_rstd || !d_rstd || !d_dx || !d_dresidual ||
      (by_row && (!d_dgate || (rows > 1 && dgate_stride < dim))))
    return SPORDER_BAD_ARGUMENT;
  const int64_t blocks = grad_blocks(rows, dim);
  if (columns && (!d_work || !aligned_to(d_work, 256) ||
                  work_bytes < sporder_residual_norm_grad_work_bytes(rows, dim)))
    return SPORDER_BAD_ARGUMENT;
  const BlockGradArgs a{rows, dim, d_dy ? dy_stride : 0, d_dh ? dh_stride : 0, x_stride, y_stride,
                        by_row ? gate_stride : 0, dx_stride, dresidual_stride,
                        by_row ? dgate_stride : 0, d_dy, d_dh, d_x, d_y,
                        by_row ? d_gate : nullptr, by_row ? nullptr : d_gate, d_post_weight,
                        d_weight, d_post_rstd, d_rstd, d_dx, d_dresidual,
                        by_row ? d_dgate : nullptr, columns ? static_cast<float *>(d_work) : nullptr,
                        scale, vector_type, post_norm != 0};
  const int32_t rc = type == SPORDER_TYPE_BF16  ? block_grad_typed<bf16_t>(a, blocks, stream)
                     : type == SPORDER_TYPE_F16 ? block_grad_typed<f16_t>(a, blocks, stream)
                                                : block_grad_typed<float>(a, blocks, stream);
  if (rc != SPORDER_OK || !columns) return rc;
  sums.partial = a.partial;
  sums.count = blocks;
  return launch(block_norm_sum_kernel, dim3(ceil_div64(2 * dim, kWave)), dim3(kWave * kSumRows),
                stream, sums);
}

} // extern "C"
