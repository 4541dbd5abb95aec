// cross_entropy_few.hip -- linear cross entropy where all classes' weights fit a
// workgroup's LDS (a graph's node classes): one pass over the rows each way.
//
// A workgroup keeps w in LDS and takes tiles of rows.  The products are 32-bit ones
// (16 x 16 x 4 per matrix instruction) whatever the type, so nothing is rounded on
// the way:
//   z^T = w x^T      classes down (a lane's registers), rows across (lanes)
//   dx^T = w^T g^T   features down, rows across
//   dw = g^T x       classes down, features across, in registers over all tiles
// A matrix instruction's four steps along the sum may be any four: lane group q
// takes elements 4 q .. 4 q + 3 of 16 (one LDS access for four instructions where
// they lie side by side), and in the last two products rows r + 4 q, which
// with rows 4 floats longer than a multiple of 16 lie in different banks.
#include <algorithm>

#include "cross_entropy.hpp"

namespace sporder_hip {

namespace {

using f32x4 = float __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr int kLds = 160 * 1024;

struct FewArgs {
  CeCall c;
  int64_t tiles;
  double *sums;   // [grid][2], forward
  float *dw_part; // [grid][VB * 16][dim_pad], backward
  float *db_part; // [grid][VB * 16]
};

__device__ __forceinline__ f32x4 mfma_16x16(float a, float b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// Four elements of a row from `col` on as floats, zeros past its end.
template <typename T>
__device__ __forceinline__ f32x4 four(const T *row, int col, int dim) {
  f32x4 v = {};
  if (col < dim) {
    const auto q = fetch<true, 4>(row + col, dim - col);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = static_cast<float>(q.v[e]);
  }
  return v;
}

// w and the bias (-inf past the classes) to LDS, rows of `stride` floats.
template <typename T, int VB, int DB>
__device__ __forceinline__ void hold_weights(const CeCall &c, float *w, float *bias, int stride) {
  const int part = threadIdx.x % 16 * 4;
  for (int v = threadIdx.x / 16; v < VB * 16; v += kThreads / 16) {
    const T *const row = static_cast<const T *>(c.w) + v * c.w_stride;
#pragma unroll
    for (int k = 0; k < DB; ++k)
      if (k * 64 + part < stride - 4)
        *reinterpret_cast<f32x4 *>(w + v * stride + k * 64 + part) =
            v < c.classes ? four<T>(row, k * 64 + part, static_cast<int>(c.dim)) : f32x4{};
  }
  for (int v = threadIdx.x; v < VB * 16; v += kThreads) {
    float b = v < c.classes ? 0.0f : -INFINITY;
    if (c.bias && v < c.classes) with_type(c.bias, c.bias_type, [&](auto *p) { b = static_cast<float>(p[v]); });
    bias[v] = b;
  }
}

// A tile's rows on their way: 16 threads a row, zeros for rows that count nothing.
template <typename T, int TB, int DB>
__device__ __forceinline__ void fetch_tile(const CeCall &c, int64_t first, f32x4 (&v)[TB][DB]) {
  const int part = threadIdx.x % 16 * 4;
#pragma unroll
  for (int i = 0; i < TB; ++i) {
    const int64_t row = first + i * 16 + threadIdx.x / 16;
    const bool on = row < c.rows && counted(c, target_of(c, row));
    const T *const x = static_cast<const T *>(c.x) + row * c.x_stride;
#pragma unroll
    for (int k = 0; k < DB; ++k)
      v[i][k] = on ? four<T>(x, k * 64 + part, static_cast<int>(c.dim)) : f32x4{};
  }
}

template <int TB, int DB>
__device__ __forceinline__ void put_tile(float *x, int stride, const f32x4 (&v)[TB][DB]) {
  const int part = threadIdx.x % 16 * 4;
#pragma unroll
  for (int i = 0; i < TB; ++i) {
#pragma unroll
    for (int k = 0; k < DB; ++k)
      if (k * 64 + part < stride - 4)
        *reinterpret_cast<f32x4 *>(x + (i * 16 + threadIdx.x / 16) * stride + k * 64 + part) = v[i][k];
  }
}

// z of 16 rows (of x, from `rows` on) and every STEP-th block of 16 classes.
template <int BLOCKS, int STEP>
__device__ __forceinline__ void logits(const float *w, const float *rows, int stride, f32x4 (&z)[BLOCKS]) {
  const int lane = lane_id(), at = lane % 16 * stride + lane / 16 * 4;
  for (int k = 0; k < stride - 4; k += 16) {
    const f32x4 b = *reinterpret_cast<const f32x4 *>(rows + at + k);
#pragma unroll
    for (int v = 0; v < BLOCKS; ++v) {
      const f32x4 a = *reinterpret_cast<const f32x4 *>(w + v * STEP * 16 * stride + at + k);
#pragma unroll
      for (int e = 0; e < 4; ++e) z[v] = mfma_16x16(a[e], b[e], z[v]);
    }
  }
}

// ---- forward: 64 rows a tile, 16 a wave ------------------------------------------------

template <typename T, int VB, int DB>
__global__ void __launch_bounds__(kThreads) few_loss_kernel(FewArgs a) {
  extern __shared__ __attribute__((aligned(16))) float lds[];
  const CeCall &c = a.c;
  const int stride = static_cast<int>(ceil_div64(c.dim, 16)) * 16 + 4;
  float *const w = lds, *const x = w + VB * 16 * stride, *const bias = x + 64 * stride;
  const int lane = lane_id(), wave = threadIdx.x / kWave;
  hold_weights<T, VB, DB>(c, w, bias, stride);
  double sum = 0.0, n = 0.0;
  f32x4 next[4][DB];
  fetch_tile<T>(c, blockIdx.x * int64_t(64), next);
  for (int64_t tile = blockIdx.x; tile < a.tiles; tile += gridDim.x) {
    __syncthreads(); // the tile before is done with
    put_tile(x, stride, next);
    __syncthreads();
    fetch_tile<T>(c, (tile + gridDim.x) * 64, next);
    f32x4 z[VB] = {};
    logits<VB, 1>(w, x + wave * 16 * stride, stride, z);
    const int64_t row = tile * 64 + wave * 16 + lane % 16;
    const int64_t target = row < c.rows ? target_of(c, row) : c.ignore;
    const int at = counted(c, target) ? static_cast<int>(target) : -1;
    float most = -INFINITY, hit = 0.0f;
#pragma unroll
    for (int v = 0; v < VB; ++v) {
      const f32x4 b = *reinterpret_cast<const f32x4 *>(bias + v * 16 + lane / 16 * 4);
      z[v] += b;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        most = fmaxf(most, z[v][e]);
        hit += v * 16 + lane / 16 * 4 + e == at ? z[v][e] : 0.0f;
      }
    }
    most = fmaxf(most, lane_xor_f32(most, 16));
    most = fmaxf(most, lane_xor_f32(most, 32));
    const float base = most == -INFINITY ? 0.0f : most;
    float total = 0.0f;
#pragma unroll
    for (int v = 0; v < VB; ++v) {
#pragma unroll
      for (int e = 0; e < 4; ++e) total += exp_of(z[v][e] - base);
    }
    total += lane_xor_f32(total, 16);
    hit += lane_xor_f32(hit, 16);
    total += lane_xor_f32(total, 32);
    hit += lane_xor_f32(hit, 32);
    if (lane < 16 && row < c.rows) {
      float lse = base + logf(total), loss = lse - hit;
      if (!counted(c, target)) loss = lse = target == c.ignore ? 0.0f : NAN;
      c.lse[row] = lse;
      c.loss[row] = loss;
      sum += loss;
      n += target == c.ignore ? 0.0 : 1.0;
    }
  }
  __shared__ double part[2][4];
  const double v = block_sums(sum, n, part);
  if (threadIdx.x >= 2) return;
  if (gridDim.x == 1)
    c.sums[threadIdx.x] = static_cast<float>(v);
  else
    a.sums[2 * blockIdx.x + threadIdx.x] = v;
}

__global__ void __launch_bounds__(kThreads) few_total_kernel(FewArgs a, int blocks) {
  __shared__ double part[2][4];
  double s = 0.0, n = 0.0;
  for (int i = threadIdx.x; i < blocks; i += kThreads) {
    s += a.sums[2 * i];
    n += a.sums[2 * i + 1];
  }
  const double v = block_sums(s, n, part);
  if (threadIdx.x < 2) a.c.sums[threadIdx.x] = static_cast<float>(v);
}

// ---- backward: TB * 16 rows a tile -----------------------------------------------------

template <typename T, int VB, int DB, int TB>
__global__ void __launch_bounds__(kThreads) few_grad_kernel(FewArgs a) {
  extern __shared__ __attribute__((aligned(16))) float lds[];
  constexpr int kRows = TB * 16, kSplit = 4 / TB; // waves that share a block of rows
  constexpr int kMine = (VB + kSplit - 1) / kSplit;
  constexpr int kG = VB * 16 + 4; // floats of a row of g
  const CeCall &c = a.c;
  const int dim16 = static_cast<int>(ceil_div64(c.dim, 16)), stride = dim16 * 16 + 4;
  float *const w = lds, *const x = w + VB * 16 * stride, *const g = x + kRows * stride;
  float *const bias = g + kRows * kG;
  const int lane = lane_id(), wave = threadIdx.x / kWave, q = lane / 16, l = lane % 16;
  const int tb = wave % TB, part = wave / TB;
  hold_weights<T, VB, DB>(c, w, bias, stride);
  f32x4 dw[VB][DB] = {};
  float db[VB] = {};
  f32x4 next[TB][DB];
  fetch_tile<T>(c, blockIdx.x * int64_t(kRows), next);
  for (int64_t tile = blockIdx.x; tile < a.tiles; tile += gridDim.x) {
    __syncthreads();
    put_tile(x, stride, next);
    __syncthreads();
    fetch_tile<T>(c, (tile + gridDim.x) * kRows, next);

    // g of this wave's rows and classes.
    const int64_t row = tile * kRows + tb * 16 + l;
    const int64_t target = row < c.rows ? target_of(c, row) : -1;
    const bool on = row < c.rows && counted(c, target);
    const int at = on ? static_cast<int>(target) : -1;
    const float lse = on ? c.given_lse[row] : 0.0f;
    const float s = on ? c.grad[row * c.grad_stride] : 0.0f;
    f32x4 z[kMine] = {};
    // With an odd number of blocks the last wave multiplies some of x for its last one
    // (x lies behind w) and leaves it.
    logits<kMine, kSplit>(w + part * 16 * stride, x + tb * 16 * stride, stride, z);
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int v = (i * kSplit + part) * 16 + q * 4;
      if (v >= VB * 16) continue;
      const f32x4 b = *reinterpret_cast<const f32x4 *>(bias + v);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p = exp_of(z[i][e] + b[e] - lse) - (v + e == at ? 1.0f : 0.0f);
        z[i][e] = on ? p * s : 0.0f;
      }
      *reinterpret_cast<f32x4 *>(g + (tb * 16 + l) * kG + v) = z[i];
    }
    __syncthreads();

    // dx: this wave's rows and every kSplit-th block of features.
    for (int j = part; j < dim16; j += kSplit) {
      f32x4 d = {};
#pragma unroll
      for (int v = 0; v < VB; ++v) {
        const f32x4 gv = *reinterpret_cast<const f32x4 *>(g + (tb * 16 + l) * kG + v * 16 + q * 4);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          d = mfma_16x16(w[(v * 16 + q * 4 + e) * stride + j * 16 + l], gv[e], d);
      }
      const int col = j * 16 + q * 4;
      if (row < c.rows && col < c.dim) {
        const float out[4] = {d[0], d[1], d[2], d[3]};
        put<true, 4>(static_cast<T *>(c.dx) + row * c.dx_stride + col, c.dim - col, out);
      }
    }
    // dw: all classes and every fourth block of features.
#pragma unroll
    for (int t = 0; t < TB; ++t) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = t * 16 + q * 4 + e;
        float gv[VB];
#pragma unroll
        for (int v = 0; v < VB; ++v) {
          gv[v] = g[r * kG + v * 16 + l];
          db[v] += gv[v];
        }
#pragma unroll
        for (int k = 0; k < DB; ++k) {
          if (k * 4 + wave >= dim16) continue;
          const float xv = x[r * stride + (k * 4 + wave) * 16 + l];
#pragma unroll
          for (int v = 0; v < VB; ++v) dw[v][k] = mfma_16x16(gv[v], xv, dw[v][k]);
        }
      }
    }
  }
  float *const out = a.dw_part + blockIdx.x * int64_t(VB * 16) * (dim16 * 16);
#pragma unroll
  for (int v = 0; v < VB; ++v) {
#pragma unroll
    for (int k = 0; k < DB; ++k) {
      if (k * 4 + wave >= dim16) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        out[(v * 16 + q * 4 + e) * (dim16 * 16) + (k * 4 + wave) * 16 + l] = dw[v][k][e];
    }
    db[v] += lane_xor_f32(db[v], 16);
    db[v] += lane_xor_f32(db[v], 32);
    if (wave == 0 && q == 0) a.db_part[blockIdx.x * int64_t(VB * 16) + v * 16 + l] = db[v];
  }
}

// The workgroups' sums of dw and db: 64 elements per workgroup, 16 threads each.
__global__ void __launch_bounds__(1024)
    few_sum_kernel(FewArgs a, int64_t blocks, int64_t classes_pad, int64_t dim_pad) {
  __shared__ float part[16][kWave];
  const int x = threadIdx.x % kWave, y = threadIdx.x / kWave;
  const int64_t i = blockIdx.x * int64_t(kWave) + x, all = classes_pad * dim_pad;
  float s = 0.0f;
  if (i < all) {
#pragma unroll 8
    for (int64_t b = y; b < blocks; b += 16) s += a.dw_part[b * all + i];
  } else if (i < all + classes_pad) {
#pragma unroll 8
    for (int64_t b = y; b < blocks; b += 16) s += a.db_part[b * classes_pad + i - all];
  }
  part[y][x] = s;
  __syncthreads();
  if (y != 0) return;
  s = 0.0f;
#pragma unroll
  for (int k = 0; k < 16; ++k) s += part[k][x];
  if (i < all) {
    const int64_t v = i / dim_pad, j = i % dim_pad;
    if (v < a.c.classes && j < a.c.dim) store_typed(a.c.dw, a.c.dw_type, v * a.c.dw_stride + j, s);
  } else if (a.c.db && i - all < a.c.classes) {
    store_typed(a.c.db, a.c.bias_type, i - all, s);
  }
}

// ---- host --------------------------------------------------------------------------------

constexpr int kBlocks[] = {1, 2, 3, 4, 6, 8, 12}; // of 16 classes that kernels are built for
int class_blocks(int64_t classes) {
  for (int b : kBlocks)
    if (classes <= b * 16) return b;
  return 0;
}
// Blocks of 64 features.
int feature_blocks(int64_t dim) { return dim <= 64 ? 1 : dim <= 128 ? 2 : dim <= 256 ? 4 : dim <= 512 ? 8 : 0; }

int64_t floats_of(int64_t dim, int blocks, int rows, bool backward) {
  const int64_t stride = ceil_div64(dim, 16) * 16 + 4;
  return (blocks * 16 + rows) * stride + (backward ? rows * (blocks * 16 + 4) : 0) + blocks * 16;
}
bool fits(int64_t dim, int blocks, int rows, bool backward) {
  return floats_of(dim, blocks, rows, backward) * 4 + 256 <= kLds;
}
// 64 rows a tile where they fit LDS and, beside dw, the registers.
constexpr bool whole_tile(int vb, int db) { return vb * db < 24 && db < 8; }
int tile_rows(int64_t dim, int64_t classes) {
  const int b = class_blocks(classes);
  return whole_tile(b, feature_blocks(dim)) && fits(dim, b, 64, true) ? 64 : 32;
}

// Workgroups: two per CU where their LDS allows it.
int64_t grid_of(int64_t rows, int64_t dim, int64_t classes, bool backward) {
  const int tile = backward ? tile_rows(dim, classes) : 64;
  const int64_t each = floats_of(dim, class_blocks(classes), tile, backward) * 4 + 256;
  return std::min(ceil_div64(rows, tile), 256 * std::min<int64_t>(kLds / each, 2));
}

template <typename F> int32_t with_blocks(int64_t dim, int64_t classes, F &&f) {
  auto classes_of = [&](auto db) {
    constexpr int DB = decltype(db)::value;
    const int b = class_blocks(classes);
    auto at = [&](auto vb) {
      if constexpr (decltype(vb)::value * DB <= 24)
        return f(vb, db);
      else
        return static_cast<int32_t>(SPORDER_BAD_ARGUMENT); // not reached
    };
    switch (b) {
    case 1: return at(std::integral_constant<int, 1>{});
    case 2: return at(std::integral_constant<int, 2>{});
    case 3: return at(std::integral_constant<int, 3>{});
    case 4: return at(std::integral_constant<int, 4>{});
    case 6: return at(std::integral_constant<int, 6>{});
    case 8: return at(std::integral_constant<int, 8>{});
    default: return at(std::integral_constant<int, 12>{});
    }
  };
  switch (feature_blocks(dim)) {
  case 1: return classes_of(std::integral_constant<int, 1>{});
  case 2: return classes_of(std::integral_constant<int, 2>{});
  case 4: return classes_of(std::integral_constant<int, 4>{});
  default: return classes_of(std::integral_constant<int, 8>{});
  }
}

// LDS past 64 KB has to be asked for.
template <typename... P, typename... A>
int32_t launch_lds(void (*kernel)(P...), int64_t grid, int64_t lds, void *stream, A... args) {
  if (lds > 65536 && hipFuncSetAttribute(reinterpret_cast<const void *>(kernel),
                                         hipFuncAttributeMaxDynamicSharedMemorySize,
                                         static_cast<int>(lds)) != hipSuccess) {
    (void)hipGetLastError();
    return SPORDER_LAUNCH_FAILED;
  }
  std::tuple<P...> held(static_cast<P>(args)...);
  const hipError_t err = std::apply(
      [&](P &...p) {
        void *list[] = {static_cast<void *>(&p)...};
        return hipLaunchKernel(reinterpret_cast<const void *>(kernel), dim3(grid), dim3(kThreads), list,
                               lds, static_cast<hipStream_t>(stream));
      },
      held);
  if (err == hipSuccess) return SPORDER_OK;
  (void)hipGetLastError();
  return SPORDER_LAUNCH_FAILED;
}

struct FewLayout {
  size_t sums, dw, db, bytes;
  int64_t grid;
};
FewLayout few_layout(int64_t rows, int64_t dim, int64_t classes, bool backward) {
  FewLayout l{};
  l.grid = grid_of(rows, dim, classes, backward);
  const int64_t pad = class_blocks(classes) * 16;
  size_t at = 0;
  auto take = [&](int64_t bytes) {
    const size_t here = at;
    at += Workspace::align(bytes);
    return here;
  };
  if (!backward) {
    l.sums = take(l.grid * 16);
  } else {
    l.dw = take(l.grid * pad * ceil_div64(dim, 16) * 16 * 4);
    l.db = take(l.grid * pad * 4);
  }
  l.bytes = at;
  return l;
}

template <typename T> int32_t few_loss(const FewArgs &a, int64_t grid, void *stream) {
  return with_blocks(a.c.dim, a.c.classes, [&](auto vb, auto db) {
    constexpr int VB = decltype(vb)::value, DB = decltype(db)::value;
    return launch_lds(few_loss_kernel<T, VB, DB>, grid, floats_of(a.c.dim, VB, 64, false) * 4, stream, a);
  });
}

template <typename T> int32_t few_grad(const FewArgs &a, int64_t grid, void *stream) {
  const int rows = tile_rows(a.c.dim, a.c.classes);
  return with_blocks(a.c.dim, a.c.classes, [&](auto vb, auto db) {
    constexpr int VB = decltype(vb)::value, DB = decltype(db)::value;
    const int64_t lds = floats_of(a.c.dim, VB, rows, true) * 4;
    if constexpr (whole_tile(VB, DB)) {
      if (rows == 64) return launch_lds(few_grad_kernel<T, VB, DB, 4>, grid, lds, stream, a);
    }
    return launch_lds(few_grad_kernel<T, VB, DB, 2>, grid, lds, stream, a);
  });
}

} // namespace

bool few_takes(int64_t dim, int64_t classes, bool backward) {
  const int b = class_blocks(classes), f = feature_blocks(dim);
  return b && f && b * f <= 24 && fits(dim, b, backward ? 32 : 64, backward);
}

size_t few_work_bytes(int64_t rows, int64_t dim, int64_t classes, bool backward) {
  return few_layout(rows, dim, classes, backward).bytes;
}

int32_t few_forward(const CeCall &c, void *work, void *stream) {
  const FewLayout l = few_layout(c.rows, c.dim, c.classes, false);
  FewArgs a{c, ceil_div64(c.rows, 64), reinterpret_cast<double *>(static_cast<char *>(work) + l.sums), nullptr,
            nullptr};
  const int32_t rc = c.type == SPORDER_TYPE_BF16  ? few_loss<bf16_t>(a, l.grid, stream)
                     : c.type == SPORDER_TYPE_F16 ? few_loss<f16_t>(a, l.grid, stream)
                                                  : few_loss<float>(a, l.grid, stream);
  if (rc != SPORDER_OK || l.grid == 1) return rc;
  return launch(few_total_kernel, dim3(1), dim3(kThreads), stream, a, static_cast<int>(l.grid));
}

int32_t few_backward(const CeCall &c, void *work, void *stream) {
  const FewLayout l = few_layout(c.rows, c.dim, c.classes, true);
  char *const base = static_cast<char *>(work);
  FewArgs a{c, ceil_div64(c.rows, tile_rows(c.dim, c.classes)), nullptr,
            reinterpret_cast<float *>(base + l.dw), reinterpret_cast<float *>(base + l.db)};
  const int32_t rc = c.type == SPORDER_TYPE_BF16  ? few_grad<bf16_t>(a, l.grid, stream)
                     : c.type == SPORDER_TYPE_F16 ? few_grad<f16_t>(a, l.grid, stream)
                                                  : few_grad<float>(a, l.grid, stream);
  if (rc != SPORDER_OK) return rc;
  const int64_t pad = class_blocks(c.classes) * 16, dim_pad = ceil_div64(c.dim, 16) * 16;
  return launch(few_sum_kernel, dim3(ceil_div64(pad * dim_pad + pad, kWave)), dim3(1024), stream, a, l.grid, pad,
                dim_pad);
}

} // namespace sporder_hip
