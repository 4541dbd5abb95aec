// layer_norm.hip -- layer norm and its gradients.
//
//   mean = sum x / D,  var = sum (x - mean)^2 / D,  rstd = (var + eps)^-1/2
//   h = (x - mean) rstd,  y = w h + b
//   g = w dy,  dx = rstd (g - sum g / D - h sum (g h) / D)
//   dw = sum over rows of dy h,  db = sum over rows of dy
//
// A row is held in the registers of L lanes, C vectors of VEC elements each,
// so it is read once: the variance is the mean square of the centred row, not
// a difference of sums that cancels.  HBM bounds both directions (a row is
// read and written once, ~8 and ~14 operations per element).  L is the
// smallest group that holds the row at 16 elements per lane (rows of up to
// 1024 elements: part of a wave, several rows per wave; longer ones several
// waves); rows past what 512 lanes hold (32768 elements forward, 16384
// backward) are read more than once.
#include <algorithm>

#include "dense.hpp"

namespace sporder_hip {

namespace {

struct NormArgs {
  int64_t rows, dim, x_stride, y_stride;
  const void *x, *weight, *bias;
  void *y;
  float *mean, *rstd;
  float eps;
  int weight_type;
};

struct NormGradArgs {
  int64_t rows, dim, dy_stride, x_stride, dx_stride;
  const void *dy, *x, *weight;
  const float *mean, *rstd;
  void *dx;
  float *partial; // [grid][2][dim] sums of dy h and dy, or null
  int weight_type;
};

// Sums of N values over the L lanes that hold a row, in each of them.  Past a
// wave the waves' sums meet in `shared`; calls alternate between its halves
// (`turn`), so that one barrier per call is enough: a wave writes a half again
// only after the barrier of the call between.
constexpr int norm_block(int lanes) { return lanes > 256 ? lanes : 256; }

template <int L, int N> struct RowSum {
  static constexpr int kWaves = L > kWave ? L / kWave : 1; // of a row
  static constexpr int kBlockWaves = norm_block(L) / kWave;
  float (*shared)[N][kBlockWaves];
  int turn = 0;

  __device__ __forceinline__ void operator()(float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = group_sum<(L < kWave ? L : kWave)>(v[i]);
    if constexpr (L > kWave) {
      const int wave = threadIdx.x / kWave;
      if (threadIdx.x % kWave == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) shared[turn][i][wave] = v[i];
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float *const row = shared[turn][i] + wave / kWaves * kWaves;
        float s = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) s += row[w];
        v[i] = s;
      }
      turn ^= 1;
    }
  }
};

// A lane's part of weight or bias, or `value` where there is none.
template <int VEC, int L, int C>
__device__ __forceinline__ void load_vector(const void *p, int type, int64_t dim, float value,
                                            int lane, float (&out)[C][VEC]) {
#pragma unroll
  for (int c = 0; c < C; ++c) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) out[c][i] = value;
  }
  if (!p) return;
  with_type(p, type, [&](auto *w) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int col = (c * L + lane) * VEC;
      if (col < dim) load_f32<VEC>(w + col, out[c]);
    }
  });
}

template <typename T, int VEC, int L, int C>
__global__ void __launch_bounds__(norm_block(L)) layer_norm_kernel(NormArgs a) {
  constexpr int kGroups = norm_block(L) / L;
  __shared__ float shared[2][1][norm_block(L) / kWave];
  RowSum<L, 1> row_sum{shared};
  const int lane = threadIdx.x % L, group = threadIdx.x / L;
  const float dim = static_cast<float>(a.dim);

  float w[C][VEC], b[C][VEC];
  load_vector<VEC, L>(a.weight, a.weight_type, a.dim, 1.0f, lane, w);
  load_vector<VEC, L>(a.bias, a.weight_type, a.dim, 0.0f, lane, b);

  for (int64_t first = static_cast<int64_t>(blockIdx.x) * kGroups; first < a.rows;
       first += static_cast<int64_t>(gridDim.x) * kGroups) {
    const int64_t row = first + group;
    const bool live = row < a.rows;
    const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
    float v[C][VEC];
    float s[1] = {0.0f};
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int col = (c * L + lane) * VEC;
      if (live && col < a.dim) {
        load_f32<VEC>(x + col, v[c]);
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[c][i] = 0.0f;
      }
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) s[0] += v[c][i];
    }
    row_sum(s);
    const float mean = s[0] / dim;
    s[0] = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const bool in = (c * L + lane) * VEC < a.dim;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        v[c][i] -= mean;
        s[0] += in ? v[c][i] * v[c][i] : 0.0f;
      }
    }
    row_sum(s);
    const float rstd = 1.0f / sqrtf(s[0] / dim + a.eps);
    if (!live) continue;
    T *y = static_cast<T *>(a.y) + row * a.y_stride;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int col = (c * L + lane) * VEC;
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[c][i] = v[c][i] * rstd * w[c][i] + b[c][i];
      if (col < a.dim) store_f32<VEC>(y + col, v[c]);
    }
    if (lane == 0) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
  }
}

// Rows that no workgroup's registers hold: three passes over each.
template <typename T> __global__ void __launch_bounds__(1024) layer_norm_long_kernel(NormArgs a) {
  __shared__ float shared[2][1][1024 / kWave];
  RowSum<1024, 1> row_sum{shared};
  const float dim = static_cast<float>(a.dim);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
    T *y = static_cast<T *>(a.y) + row * a.y_stride;
    float s[1] = {0.0f};
    for (int64_t i = threadIdx.x; i < a.dim; i += 1024) s[0] += static_cast<float>(x[i]);
    row_sum(s);
    const float mean = s[0] / dim;
    s[0] = 0.0f;
    for (int64_t i = threadIdx.x; i < a.dim; i += 1024) {
      const float d = static_cast<float>(x[i]) - mean;
      s[0] += d * d;
    }
    row_sum(s);
    const float rstd = 1.0f / sqrtf(s[0] / dim + a.eps);
    for (int64_t i = threadIdx.x; i < a.dim; i += 1024) {
      float w = 1.0f, b = 0.0f;
      if (a.weight) with_type(a.weight, a.weight_type, [&](auto *p) { w = static_cast<float>(p[i]); });
      if (a.bias) with_type(a.bias, a.weight_type, [&](auto *p) { b = static_cast<float>(p[i]); });
      y[i] = static_cast<T>((static_cast<float>(x[i]) - mean) * rstd * w + b);
    }
    if (threadIdx.x == 0) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
  }
}

// dx, and the workgroup's sums of dy h and dy by column: each lane keeps its
// columns' sums in registers over all the rows that it takes, the groups of a
// workgroup are added up at the end and the workgroup writes one row of
// partial sums.  No atomics: the order of every sum is fixed by the grid.
template <typename T, int VEC, int L, int C>
__global__ void __launch_bounds__(norm_block(L)) layer_norm_grad_kernel(NormGradArgs a) {
  constexpr int kGroups = norm_block(L) / L;
  constexpr int kSpan = L * C * VEC; // columns that a group holds
  constexpr int kBlockWaves = norm_block(L) / kWave;
  constexpr int kRowWaves = L > kWave ? L / kWave : 1;
  constexpr int kSlots = kBlockWaves / kRowWaves; // waves, or groups of waves, of whole rows
  __shared__ float shared[2][2][kBlockWaves];
  __shared__ float joined[L < 256 ? kSlots : 1][L < 256 ? kSpan : 1];
  RowSum<L, 2> row_sum{shared};
  const int lane = threadIdx.x % L, group = threadIdx.x / L;
  const float dim = static_cast<float>(a.dim);

  float w[C][VEC], dw[C][VEC] = {}, db[C][VEC] = {};
  load_vector<VEC, L>(a.weight, a.weight_type, a.dim, 1.0f, lane, w);

  for (int64_t first = static_cast<int64_t>(blockIdx.x) * kGroups; first < a.rows;
       first += static_cast<int64_t>(gridDim.x) * kGroups) {
    const int64_t row = first + group;
    const bool live = row < a.rows;
    const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
    const T *dy = static_cast<const T *>(a.dy) + row * a.dy_stride;
    const float mean = live ? a.mean[row] : 0.0f, rstd = live ? a.rstd[row] : 0.0f;
    float h[C][VEC], g[C][VEC];
    float s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int col = (c * L + lane) * VEC;
      if (live && col < a.dim) {
        load_f32<VEC>(x + col, h[c]);
        load_f32<VEC>(dy + col, g[c]);
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) h[c][i] = mean, g[c][i] = 0.0f;
      }
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        h[c][i] = (h[c][i] - mean) * rstd;
        dw[c][i] += g[c][i] * h[c][i];
        db[c][i] += g[c][i];
        g[c][i] *= w[c][i];
        s[0] += g[c][i];
        s[1] += g[c][i] * h[c][i];
      }
    }
    row_sum(s);
    const float m1 = s[0] / dim, m2 = s[1] / dim;
    if (!live) continue;
    T *dx = static_cast<T *>(a.dx) + row * a.dx_stride;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int col = (c * L + lane) * VEC;
#pragma unroll
      for (int i = 0; i < VEC; ++i) g[c][i] = (g[c][i] - m1 - h[c][i] * m2) * rstd;
      if (col < a.dim) store_f32<VEC>(dx + col, g[c]);
    }
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
          out[col] = dw[c][i];
          out[a.dim + col] = db[c][i];
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
          float v = what ? db[c][i] : dw[c][i];
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

// Rows that no workgroup's registers hold: two passes over each, the column
// sums kept in the workgroup's partial row (each thread its own columns).
template <typename T>
__global__ void __launch_bounds__(1024) layer_norm_grad_long_kernel(NormGradArgs a) {
  __shared__ float shared[2][2][1024 / kWave];
  RowSum<1024, 2> row_sum{shared};
  const float dim = static_cast<float>(a.dim);
  float *const out = a.partial ? a.partial + static_cast<int64_t>(blockIdx.x) * 2 * a.dim : nullptr;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
    const T *dy = static_cast<const T *>(a.dy) + row * a.dy_stride;
    T *dx = static_cast<T *>(a.dx) + row * a.dx_stride;
    const float mean = a.mean[row], rstd = a.rstd[row];
    float s[2] = {0.0f, 0.0f};
    for (int64_t i = threadIdx.x; i < a.dim; i += 1024) {
      float w = 1.0f;
      if (a.weight) with_type(a.weight, a.weight_type, [&](auto *p) { w = static_cast<float>(p[i]); });
      const float h = (static_cast<float>(x[i]) - mean) * rstd, d = static_cast<float>(dy[i]);
      s[0] += d * w;
      s[1] += d * w * h;
      if (out) {
        const bool again = row != blockIdx.x;
        out[i] = (again ? out[i] : 0.0f) + d * h;
        out[a.dim + i] = (again ? out[a.dim + i] : 0.0f) + d;
      }
    }
    row_sum(s);
    const float m1 = s[0] / dim, m2 = s[1] / dim;
    for (int64_t i = threadIdx.x; i < a.dim; i += 1024) {
      float w = 1.0f;
      if (a.weight) with_type(a.weight, a.weight_type, [&](auto *p) { w = static_cast<float>(p[i]); });
      const float h = (static_cast<float>(x[i]) - mean) * rstd, d = static_cast<float>(dy[i]);
      dx[i] = static_cast<T>((d * w - m1 - h * m2) * rstd);
    }
  }
}

// Column sums of the partial rows: 64 columns per workgroup, 16 threads per
// column over interleaved rows, added up in LDS.
constexpr int kSumRows = 16;
__global__ void __launch_bounds__(kWave *kSumRows)
    norm_column_sum_kernel(const float *partial, int64_t count, int64_t dim, void *dweight,
                           void *dbias, int weight_type) {
  __shared__ float part[kSumRows][kWave];
  const int x = threadIdx.x % kWave, y = threadIdx.x / kWave;
  const int64_t col = static_cast<int64_t>(blockIdx.x) * kWave + x; // of 2 dim
  float v = 0.0f;
  if (col < 2 * dim) {
#pragma unroll 8
    for (int64_t r = y; r < count; r += kSumRows) v += partial[r * 2 * dim + col];
  }
  part[y][x] = v;
  __syncthreads();
  if (y != 0 || col >= 2 * dim) return;
  v = 0.0f;
#pragma unroll
  for (int k = 0; k < kSumRows; ++k) v += part[k][x];
  void *const to = col < dim ? dweight : dbias;
  if (to) store_typed(to, weight_type, col < dim ? col : col - dim, v);
}

// Rows of no elements to sum: the gradients of zero rows are zero.
__global__ void norm_zero_kernel(int64_t dim, void *dweight, void *dbias, int weight_type) {
  const int64_t i = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x;
  if (i >= dim) return;
  if (dweight) store_typed(dweight, weight_type, i, 0.0f);
  if (dbias) store_typed(dbias, weight_type, i, 0.0f);
}

constexpr int64_t kMaxNormBlocks = 256 * 8;
constexpr int64_t kNormMostDim = 512 * 64;     // forward, in registers
constexpr int64_t kNormGradMostDim = 512 * 32; // backward: dw and db are held too

template <typename T, int VEC, int L, int E> int32_t run_norm(const NormArgs &a, void *stream) {
  constexpr int kGroups = norm_block(L) / L;
  const int64_t blocks = std::min(ceil_div64(a.rows, kGroups), kMaxNormBlocks);
  return launch(layer_norm_kernel<T, VEC, L, E / VEC>, dim3(blocks), dim3(norm_block(L)), stream,
                a);
}

template <typename T, int VEC> int32_t pick_norm(const NormArgs &a, void *stream) {
  const int64_t d = a.dim;
  if constexpr (VEC == 1) { // single elements: whole waves on a row, for contiguous accesses
    if (d <= 32) return run_norm<T, 1, 32, 1>(a, stream);
    if (d <= 128) return run_norm<T, 1, 64, 2>(a, stream);
    if (d <= 256) return run_norm<T, 1, 64, 4>(a, stream);
    if (d <= 512) return run_norm<T, 1, 64, 8>(a, stream);
  } else {
    if (d <= 64) return run_norm<T, VEC, 8, 8>(a, stream);
    if (d <= 128) return run_norm<T, VEC, 8, 16>(a, stream);
    if (d <= 256) return run_norm<T, VEC, 16, 16>(a, stream);
    if (d <= 512) return run_norm<T, VEC, 32, 16>(a, stream);
  }
  if (d <= 1024) return run_norm<T, VEC, 64, 16>(a, stream);
  if (d <= 2048) return run_norm<T, VEC, 128, 16>(a, stream);
  if (d <= 4096) return run_norm<T, VEC, 256, 16>(a, stream);
  if (d <= 8192) return run_norm<T, VEC, 512, 16>(a, stream);
  if (d <= 16384) return run_norm<T, VEC, 512, 32>(a, stream);
  return run_norm<T, VEC, 512, 64>(a, stream);
}

template <typename T, int VEC, int L, int E>
int32_t run_norm_grad(const NormGradArgs &a, int64_t blocks, void *stream) {
  return launch(layer_norm_grad_kernel<T, VEC, L, E / VEC>, dim3(blocks), dim3(norm_block(L)),
                stream, a);
}

template <typename T, int VEC>
int32_t pick_norm_grad(const NormGradArgs &a, int64_t blocks, void *stream) {
  const int64_t d = a.dim;
  if constexpr (VEC == 1) {
    if (d <= 32) return run_norm_grad<T, 1, 32, 1>(a, blocks, stream);
    if (d <= 128) return run_norm_grad<T, 1, 64, 2>(a, blocks, stream);
    if (d <= 256) return run_norm_grad<T, 1, 64, 4>(a, blocks, stream);
    if (d <= 512) return run_norm_grad<T, 1, 64, 8>(a, blocks, stream);
  } else {
    if (d <= 64) return run_norm_grad<T, VEC, 8, 8>(a, blocks, stream);
    if (d <= 128) return run_norm_grad<T, VEC, 8, 16>(a, blocks, stream);
    if (d <= 256) return run_norm_grad<T, VEC, 16, 16>(a, blocks, stream);
    if (d <= 512) return run_norm_grad<T, VEC, 32, 16>(a, blocks, stream);
  }
  if (d <= 1024) return run_norm_grad<T, VEC, 64, 16>(a, blocks, stream);
  if (d <= 2048) return run_norm_grad<T, VEC, 128, 16>(a, blocks, stream);
  if (d <= 4096) return run_norm_grad<T, VEC, 256, 16>(a, blocks, stream);
  if (d <= 8192) return run_norm_grad<T, VEC, 512, 16>(a, blocks, stream);
  return run_norm_grad<T, VEC, 512, 32>(a, blocks, stream);
}

template <typename T> int32_t norm_typed(const NormArgs &a, void *stream) {
  if (a.dim > kNormMostDim)
    return launch(layer_norm_long_kernel<T>, dim3(std::min(a.rows, kMaxNormBlocks)), dim3(1024),
                  stream, a);
  const int vec = row_vec(sizeof(T), a.dim, {a.x_stride, a.y_stride},
                          {a.x, a.y, a.weight, a.bias});
  if constexpr (sizeof(T) == 2) {
    if (vec == 8) return pick_norm<T, 8>(a, stream);
  }
  if (vec == 4) return pick_norm<T, 4>(a, stream);
  return pick_norm<T, 1>(a, stream);
}

template <typename T>
int32_t norm_grad_typed(const NormGradArgs &a, int64_t blocks, void *stream) {
  if (a.dim > kNormGradMostDim)
    return launch(layer_norm_grad_long_kernel<T>, dim3(blocks), dim3(1024), stream, a);
  const int vec = row_vec(sizeof(T), a.dim, {a.x_stride, a.dy_stride, a.dx_stride},
                          {a.x, a.dy, a.dx, a.weight});
  if constexpr (sizeof(T) == 2) {
    if (vec == 8) return pick_norm_grad<T, 8>(a, blocks, stream);
  }
  if (vec == 4) return pick_norm_grad<T, 4>(a, blocks, stream);
  return pick_norm_grad<T, 1>(a, blocks, stream);
}

// Workgroups of the gradient, each with a partial row of 2 dim floats: enough
// to fill the card, and few enough that the partial rows stay small beside
// the rows themselves (at least 8 rows per workgroup).
int64_t norm_grad_blocks(int64_t rows, int64_t dim) {
  int lanes = 8;
  while (lanes < 512 && lanes * 16 < dim) lanes *= 2;
  const int64_t groups = norm_block(lanes) / lanes;
  const int64_t most = std::max<int64_t>(256, kMaxNormBlocks * 256 / norm_block(lanes) / 2);
  return std::max<int64_t>(1, std::min(ceil_div64(rows, 8 * groups), most));
}

} // namespace

} // namespace sporder_hip

using namespace sporder_hip;

extern "C" {

int32_t sporder_layer_norm(void *stream, int32_t type, int32_t weight_type, int64_t rows,
                           int64_t dim, int64_t x_stride, const void *d_x, const void *d_weight,
                           const void *d_bias, float eps, int64_t y_stride, void *d_y,
                           float *d_mean, float *d_rstd) {
  if (!type_known(type) || !type_known(weight_type) || rows < 0 || dim < 1 || dim > kMostDim ||
      x_stride < 0 ||
      y_stride < 0 || (rows > 1 && y_stride < dim) || !(eps >= 0.0f))
    return SPORDER_BAD_ARGUMENT;
  if (rows == 0) return SPORDER_OK;
  if (!d_x || !d_y || !d_mean || !d_rstd) return SPORDER_BAD_ARGUMENT;
  const NormArgs a{rows, dim,    x_stride, y_stride, d_x, d_weight,
                   d_bias, d_y, d_mean,   d_rstd,   eps, weight_type};
  if (type == SPORDER_TYPE_BF16) return norm_typed<bf16_t>(a, stream);
  if (type == SPORDER_TYPE_F16) return norm_typed<f16_t>(a, stream);
  return norm_typed<float>(a, stream);
}

size_t sporder_layer_norm_grad_work_bytes(int64_t rows, int64_t dim) {
  if (rows < 1 || dim < 1 || dim > kMostDim) return 0;
  return static_cast<size_t>(norm_grad_blocks(rows, dim)) * 2 * dim * sizeof(float);
}

int32_t sporder_layer_norm_grad(void *stream, int32_t type, int32_t weight_type, int64_t rows,
                                int64_t dim, int64_t dy_stride, const void *d_dy,
                                int64_t x_stride, const void *d_x, const float *d_mean,
                                const float *d_rstd, const void *d_weight, int64_t dx_stride,
                                void *d_dx, void *d_dweight, void *d_dbias, void *d_work,
                                size_t work_bytes) {
  if (!type_known(type) || !type_known(weight_type) || rows < 0 || dim < 1 || dim > kMostDim ||
      x_stride < 0 ||
      dy_stride < 0 || dx_stride < 0 || (rows > 1 && dx_stride < dim))
    return SPORDER_BAD_ARGUMENT;
  const bool columns = d_dweight || d_dbias;
  if (rows == 0) {
    if (!columns) return SPORDER_OK;
    return launch(norm_zero_kernel, dim3(ceil_div64(dim, 256)), dim3(256), stream, dim, d_dweight,
                  d_dbias, weight_type);
  }
  if (!d_dy || !d_x || !d_mean || !d_rstd || !d_dx) return SPORDER_BAD_ARGUMENT;
  const int64_t blocks = norm_grad_blocks(rows, dim);
  if (columns &&
      (!d_work || !aligned_to(d_work, 4) || work_bytes < sporder_layer_norm_grad_work_bytes(rows, dim)))
    return SPORDER_BAD_ARGUMENT;
  float *const partial = columns ? static_cast<float *>(d_work) : nullptr;
  const NormGradArgs a{rows, dim,      dy_stride, x_stride, dx_stride, d_dy,
                       d_x,  d_weight, d_mean,    d_rstd,   d_dx,      partial, weight_type};
  int32_t rc = type == SPORDER_TYPE_BF16  ? norm_grad_typed<bf16_t>(a, blocks, stream)
               : type == SPORDER_TYPE_F16 ? norm_grad_typed<f16_t>(a, blocks, stream)
                                          : norm_grad_typed<float>(a, blocks, stream);
  if (rc != SPORDER_OK || !columns) return rc;
  return launch(norm_column_sum_kernel, dim3(ceil_div64(2 * dim, kWave)), dim3(kWave * kSumRows),
                stream, partial, blocks, dim, d_dweight, d_dbias, weight_type);
}

} // extern "C"
