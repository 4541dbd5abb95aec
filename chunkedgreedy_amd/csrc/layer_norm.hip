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
template <bool LOOSE, int VEC, int L, int C>
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
      if (col >= dim) continue;
      const auto q = fetch<LOOSE, VEC>(w + col, dim - col);
#pragma unroll
      for (int i = 0; i < VEC; ++i) out[c][i] = static_cast<float>(q.v[i]);
    }
  });
}

// A row stays in the registers of its L lanes from its one read to its one
// write; the variance is a second sum over the registers, so that a large mean
// cancels nothing.  Bound by memory: 2.4 million rows of 128 floats in 485 us,
// 2.53 GB at 5.2 TB/s; 64 rows of 512 16-bit elements take 3.6 us.
template <typename T, bool LOOSE, int VEC, int L, int C>
__global__ void __launch_bounds__(norm_block(L)) layer_norm_kernel(NormArgs a) {
  constexpr int kGroups = norm_block(L) / L;
  // 100 million elements in rows of 101 143 us, 159 without; of 8195 205, 146.
  constexpr bool kClamp = LOOSE && sizeof(T) == 2 && L < 512;
  __shared__ float shared[2][1][norm_block(L) / kWave];
  RowSum<L, 1> row_sum{shared};
  const int lane = threadIdx.x % L, group = threadIdx.x / L;
  const float dim = static_cast<float>(a.dim);

  float w[C][VEC], b[C][VEC];
  load_vector<LOOSE, VEC, L>(a.weight, a.weight_type, a.dim, 1.0f, lane, w);
  load_vector<LOOSE, VEC, L>(a.bias, a.weight_type, a.dim, 0.0f, lane, b);

  for (int64_t first = static_cast<int64_t>(blockIdx.x) * kGroups; first < a.rows;
       first += static_cast<int64_t>(gridDim.x) * kGroups) {
    const int64_t row = first + group;
    const bool live = row < a.rows;
    const T *const x = static_cast<const T *>(a.x) + (kClamp && !live ? first : row) * a.x_stride;
    Words<T, VEC> raw[C];
    float v[C][VEC];
    float s[1] = {0.0f};
#pragma unroll
    for (int c = 0; c < C; ++c) {
      raw[c] = fetch_words<LOOSE, kClamp, VEC>(x, (c * L + lane) * VEC, a.dim, live);
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const auto q = elements<kClamp, VEC, T>(raw[c], (c * L + lane) * VEC, a.dim, live);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        v[c][i] = static_cast<float>(q.v[i]);
        s[0] += v[c][i];
      }
    }
    row_sum(s);
    const float mean = s[0] / dim;
    s[0] = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        v[c][i] -= mean;
        s[0] += (c * L + lane) * VEC + (LOOSE ? i : 0) < a.dim ? v[c][i] * v[c][i] : 0.0f;
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
      if (col < a.dim) put<LOOSE, VEC>(y + col, a.dim - col, v[c]);
    }
    if (lane == 0) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
  }
}

// Rows that no workgroup's registers hold: three passes over each, by elements.
// Bound by the passes' latency: 100 million elements in rows of 40,000 take 270
// us with 16 bits (1.5 TB/s), 315 with 32 (2.5 TB/s).
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
// partial sums.  No atomics: the order of every sum is fixed by the grid.  The
// next row is on its way while a row is worked on, where registers allow.
// Bound by memory: 16,384 rows of 4096 16-bit elements in 90 us, 403 MB and 34
// of partial rows at 4.9 TB/s; 1,000,003 of 100 floats in 239 us, 5.0 TB/s.
template <typename T, bool LOOSE, int VEC, int L, int C>
__global__ void __launch_bounds__(norm_block(L)) layer_norm_grad_kernel(NormGradArgs a) {
  constexpr int kGroups = norm_block(L) / L;
  constexpr bool kClamp = LOOSE && sizeof(T) == 2; // rows of 101 170 us, 208 without
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
  load_vector<LOOSE, VEC, L>(a.weight, a.weight_type, a.dim, 1.0f, lane, w);

  Words<T, VEC> next_x[C], next_dy[C];
  float next_mean = 0.0f, next_rstd = 0.0f;
  auto fetch_next = [&](int64_t row) {
    const bool live = row < a.rows;
    const int64_t from = kClamp && !live ? a.rows - 1 : row;
    const T *const x = static_cast<const T *>(a.x) + from * a.x_stride;
    const T *const dy = static_cast<const T *>(a.dy) + from * a.dy_stride;
    auto part = [&](const T *p, int c) {
      return fetch_words<LOOSE, kClamp, VEC>(p, (c * L + lane) * VEC, a.dim, live);
    };
    auto stats = [&]() {
      next_mean = live ? a.mean[row] : 0.0f;
      next_rstd = live ? a.rstd[row] : 0.0f;
    };
    // The order of the loads.  16-bit rows at whole accesses, and any at 8 bytes
    // an access, are faster alternating between x and dy (100 million elements
    // in rows of 300: 127 us, 196 one row after the other; of 64: 120, 128);
    // wider rows of floats that end inside a line one after the other (in rows
    // of 100: 241 us, 332 alternating), and so rows that are fetched ahead.
    if constexpr ((sizeof(T) == 2 && !LOOSE && L < 512) || VEC * sizeof(T) == 8) {
      stats();
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int col = (c * L + lane) * VEC;
        next_x[c] = next_dy[c] = Words<T, VEC>{};
        if (kClamp || (live && col < a.dim)) { // one branch for both loads
          next_x[c] = part(x, c);
          next_dy[c] = part(dy, c);
        }
      }
    } else {
#pragma unroll
      for (int c = 0; c < C; ++c) next_x[c] = part(x, c);
#pragma unroll
      for (int c = 0; c < C; ++c) next_dy[c] = part(dy, c);
      stats();
    }
  };
  // Measured with rows of 8192 16-bit elements: 144 us for 100 million, 176
  // without; shorter rows have more waves to hide behind and lose 6 to 12 %,
  // and 32 elements per lane would spill.
  constexpr bool kAhead = L == 512 && C * VEC <= 16;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kGroups;
  if (kAhead) fetch_next(static_cast<int64_t>(blockIdx.x) * kGroups + group);
  for (int64_t first = static_cast<int64_t>(blockIdx.x) * kGroups; first < a.rows; first += stride) {
    const int64_t row = first + group;
    if (!kAhead) fetch_next(row);
    const float mean = next_mean, rstd = next_rstd;
    float h[C][VEC], g[C][VEC];
    float s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int col = (c * L + lane) * VEC;
      const auto x = elements<kClamp, VEC, T>(next_x[c], col, a.dim, row < a.rows);
      const auto dy = elements<kClamp, VEC, T>(next_dy[c], col, a.dim, row < a.rows);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        h[c][i] = static_cast<float>(x.v[i]);
        g[c][i] = static_cast<float>(dy.v[i]);
      }
    }
    if (kAhead) fetch_next(row + stride);
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int col = (c * L + lane) * VEC;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        // Past the row's end h is 0: -mean rstd may pass 32 bits where no h of
        // the row does, and a dy of 0 times infinity is not 0.
        h[c][i] = (h[c][i] - mean) * (col + (LOOSE ? i : 0) < a.dim ? rstd : 0.0f);
        dw[c][i] += g[c][i] * h[c][i];
        db[c][i] += g[c][i];
        g[c][i] *= w[c][i];
        s[0] += g[c][i];
        s[1] += g[c][i] * h[c][i];
      }
    }
    row_sum(s);
    const float m1 = s[0] / dim, m2 = s[1] / dim;
    if (row >= a.rows) continue;
    T *dx = static_cast<T *>(a.dx) + row * a.dx_stride;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int col = (c * L + lane) * VEC;
#pragma unroll
      for (int i = 0; i < VEC; ++i) g[c][i] = (g[c][i] - m1 - h[c][i] * m2) * rstd;
      if (col < a.dim) put<LOOSE, VEC>(dx + col, a.dim - col, g[c]);
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
// sums kept in the workgroup's partial row (each thread its own columns):
// 100 million elements in rows of 24,001 take 560 us with 16 bits and 710 with
// 32, of 100,001 1,312 and 1,745: the partial row is read and written for each,
// and 1,000 rows are 125 workgroups, half a card, of 8 rows in turn.
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
// column over interleaved rows, added up in LDS: 6 us for 1,024 rows of 8,192.
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

// f with a row's lanes and the elements of each, as types: the smallest group
// that holds the row at 8 elements per lane up to 64, at 16 past them, and
// past 8192 a workgroup of 512 with as many as `most` elements need.
template <int N> using Const = std::integral_constant<int, N>;
template <int MOST, typename F> int32_t with_lanes(int64_t dim, F &&f) {
  if (dim <= 16) return f(Const<2>{}, Const<8>{});
  if (dim <= 32) return f(Const<4>{}, Const<8>{});
  if (dim <= 64) return f(Const<8>{}, Const<8>{});
  if (dim <= 128) return f(Const<8>{}, Const<16>{});
  if (dim <= 256) return f(Const<16>{}, Const<16>{});
  if (dim <= 512) return f(Const<32>{}, Const<16>{});
  if (dim <= 1024) return f(Const<64>{}, Const<16>{});
  if (dim <= 2048) return f(Const<128>{}, Const<16>{});
  if (dim <= 4096) return f(Const<256>{}, Const<16>{});
  if (dim <= 8192) return f(Const<512>{}, Const<16>{});
  if (MOST == 32 || dim <= 16384) return f(Const<512>{}, Const<32>{});
  return f(Const<512>{}, Const<MOST>{});
}

// Rows at a time of a workgroup of the gradient, by with_lanes.  Rows of 65 to
// 512 elements read one at a time (with_waves) are fewer at a time than this,
// 4, so that their workgroups take more turns than the grid is made for.
int64_t norm_groups(int64_t dim) {
  int lanes = dim <= 16 ? 2 : dim <= 32 ? 4 : 8;
  while (lanes < 512 && lanes * 16 < dim) lanes *= 2;
  return norm_block(lanes) / lanes;
}

// The same for accesses of a few bytes: whole waves on a row, for contiguous
// accesses.
template <int MOST, typename F> int32_t with_waves(int64_t dim, F &&f) {
  if (dim <= 128) return f(Const<64>{}, Const<2>{});
  if (dim <= 256) return f(Const<64>{}, Const<4>{});
  if (dim <= 512) return f(Const<64>{}, Const<8>{});
  return with_lanes<MOST>(dim, f);
}

// Rows of 32-bit elements that no vector fits are read by elements where a wave
// has many of a row side by side, by vectors at any alignment where it has few
// and where a lane would hold many elements apart (100 million elements, by
// elements and by vectors: rows of 101 forward 224 and 284 us, backward 288 and
// 339; of 24001 forward 488 and 280; of 12003 backward 371 and 314).  Rows of
// 16-bit elements are always read by vectors; the gradient takes 4 elements at
// a time up to 4096 (rows of 259: 168 us, 214 with 8) and 8 past it.
constexpr bool norm_loose(int64_t dim) { return dim <= 64 || dim > 16384; }
constexpr bool norm_grad_loose(int64_t dim) { return dim <= 64 || dim > 8192; }
constexpr int norm_grad_loose_vec(int64_t dim) { return dim <= 4096 ? 4 : 8; }

// Kernels are built for what the rules above pick at some dim that their lanes
// and elements hold.
template <typename T, bool LOOSE, int VEC> int32_t norm_lanes(const NormArgs &a, void *stream) {
  auto go = [&](auto lanes, auto elements) {
    constexpr int L = decltype(lanes)::value, E = decltype(elements)::value;
    if constexpr (sizeof(T) == 4 && (LOOSE || VEC == 1) && norm_loose(L * E) != LOOSE) {
      return static_cast<int32_t>(SPORDER_BAD_ARGUMENT); // not reached
    } else {
      const int64_t blocks = std::min(ceil_div64(a.rows, norm_block(L) / L), kMaxNormBlocks);
      return launch(layer_norm_kernel<T, LOOSE, VEC, L, E / VEC>, dim3(blocks), dim3(norm_block(L)),
                    stream, a);
    }
  };
  if constexpr (VEC >= 4)
    return with_lanes<64>(a.dim, go);
  else
    return with_waves<64>(a.dim, go);
}

template <typename T, bool LOOSE, int VEC>
int32_t norm_grad_lanes(const NormGradArgs &a, int64_t blocks, void *stream) {
  auto go = [&](auto lanes, auto elements) {
    constexpr int L = decltype(lanes)::value, E = decltype(elements)::value;
    if constexpr ((sizeof(T) == 4 && (LOOSE || VEC == 1) && norm_grad_loose(L * E) != LOOSE) ||
                  (sizeof(T) == 2 && LOOSE && norm_grad_loose_vec(L * E) != VEC)) {
      return static_cast<int32_t>(SPORDER_BAD_ARGUMENT); // not reached
    } else {
      return launch(layer_norm_grad_kernel<T, LOOSE, VEC, L, E / VEC>, dim3(blocks),
                    dim3(norm_block(L)), stream, a);
    }
  };
  if constexpr (VEC >= 4)
    return with_lanes<32>(a.dim, go);
  else
    return with_waves<32>(a.dim, go);
}

template <typename T> int32_t norm_typed(const NormArgs &a, void *stream) {
  if (a.dim > kNormMostDim)
    return launch(layer_norm_long_kernel<T>, dim3(std::min(a.rows, kMaxNormBlocks)), dim3(1024),
                  stream, a);
  const int vec = row_vec(sizeof(T), a.dim, {a.x_stride, a.y_stride}, {a.x, a.y, a.weight, a.bias});
  if constexpr (sizeof(T) == 2) {
    if (vec == 8) return norm_lanes<T, false, 8>(a, stream);
    if (vec == 4) return norm_lanes<T, false, 4>(a, stream);
    return norm_lanes<T, true, 8>(a, stream);
  } else {
    if (vec == 4) return norm_lanes<T, false, 4>(a, stream);
    return norm_loose(a.dim) ? norm_lanes<T, true, 4>(a, stream) : norm_lanes<T, false, 1>(a, stream);
  }
}

template <typename T>
int32_t norm_grad_typed(const NormGradArgs &a, int64_t blocks, void *stream) {
  if (a.dim > kNormGradMostDim)
    return launch(layer_norm_grad_long_kernel<T>, dim3(blocks), dim3(1024), stream, a);
  const int vec = row_vec(sizeof(T), a.dim, {a.x_stride, a.dy_stride, a.dx_stride},
                          {a.x, a.dy, a.dx, a.weight});
  if constexpr (sizeof(T) == 2) {
    if (vec == 8) return norm_grad_lanes<T, false, 8>(a, blocks, stream);
    if (vec == 4) return norm_grad_lanes<T, false, 4>(a, blocks, stream);
    return norm_grad_loose_vec(a.dim) == 4 ? norm_grad_lanes<T, true, 4>(a, blocks, stream)
                                           : norm_grad_lanes<T, true, 8>(a, blocks, stream);
  } else {
    if (vec == 4) return norm_grad_lanes<T, false, 4>(a, blocks, stream);
    return norm_grad_loose(a.dim) ? norm_grad_lanes<T, true, 4>(a, blocks, stream)
                                  : norm_grad_lanes<T, false, 1>(a, blocks, stream);
  }
}

// Workgroups of the gradient, each with a partial row of 2 dim floats: at most
// enough to fill the card, and few enough that the partial rows stay small
// beside the rows themselves (8 turns of rows per workgroup, so that few rows
// leave CUs without work).
int64_t norm_grad_blocks(int64_t rows, int64_t dim) {
  const int64_t most = dim > 4096 ? 512 : 1024;
  return std::max<int64_t>(1, std::min(ceil_div64(rows, 8 * norm_groups(dim)), most));
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
      (!d_work || !aligned_to(d_work, 256) || work_bytes < sporder_layer_norm_grad_work_bytes(rows, dim)))
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
