// cross_entropy_narrow.hip -- linear cross entropy of a few rows over many classes.
//
// With up to 64 rows w's traffic is all there is: each kernel reads it (or writes dw)
// once, as it lies, and multiplies in 32 bits, 32 x 32 x 2 a matrix instruction, so that
// nothing is packed, transposed or rounded first.
//   z = w x^T       a workgroup per 32 classes, its waves share the features
//   dx^T = w^T g^T  128 features a wave, the classes in parts, joined after
//   dw = g^T x      32 classes a wave, 128 features at a time
// A matrix instruction's lanes take row (or column) l % 32 and the sum's element l / 32;
// which elements those are is free as long as both operands agree, and so is the order of
// rows.  So a lane's eight neighbouring elements serve eight instructions, and where
// features lie across lanes, four neighbouring ones serve four blocks of 32.
// Not at memory's rate: one row over 50,000 x 4,096 floats in 240 us (3.4 TB/s; a copy reaches 5.7),
// for an access of a wave takes 64 bytes of 32 rows of w each, two to four accesses ahead; from some
// 32 rows on, and in 16-bit types from the first, the 32-bit products take as long (64 rows over
// 30,000 x 4,096 floats 298 us, of which the products are worth 102; one row over 50,000 x 4,096
// bfloat16 with its gradients 479 us, its bytes 144).
#include <algorithm>

#include "cross_entropy.hpp"
#include "mfma_product.hpp"

namespace sporder_hip {

namespace {

constexpr int kBlock = 32; // classes of a workgroup
constexpr int kWaves = 4, kThreads = kWaves * kWave;

struct NarrowArgs {
  CeCall c;
  float2 *partial;  // [class blocks][row blocks * 32]
  float *hit;       // [row blocks * 32]
  float *g;         // [class blocks * 32][row blocks * 32]
  float *dx_part;   // [splits][row blocks * 32][dim_pad]
  int64_t blocks, dim_pad, splits;
};

__device__ __forceinline__ f32x16 mfma_floats(float a, float b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0);
}

// A row's class, -1 where it counts nothing, -2 where it is no class.
__device__ __forceinline__ int class_at(const CeCall &c, int64_t row) {
  if (row >= c.rows) return -1;
  const int64_t t = target_of(c, row);
  return t == c.ignore ? -1 : t >= 0 && t < c.classes ? static_cast<int>(t) : -2;
}

// Bit t: whether row t counts.
__device__ __forceinline__ uint64_t rows_counted(const CeCall &c) {
  return __ballot(class_at(c, lane_id()) >= 0);
}

template <typename T, int TB, bool BACKWARD>
__global__ void __launch_bounds__(kThreads) narrow_logit_kernel(NarrowArgs a) {
  __shared__ float sums[kWaves - 1][TB][16][kWave];
  const CeCall &c = a.c;
  const int lane = lane_id(), l = lane % 32, h = lane / 32;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t v0 = xcd_block() * kBlock;
  const T *const w = static_cast<const T *>(c.w) + min(v0 + l, c.classes - 1) * c.w_stride;
  const T *x[TB];
#pragma unroll
  for (int t = 0; t < TB; ++t)
    x[t] = static_cast<const T *>(c.x) + min(static_cast<int64_t>(t * 32 + l), c.rows - 1) * c.x_stride;
  f32x16 acc[TB] = {};
  auto multiply = [&](const Pack<T, 8> &wv, const Pack<T, 8> (&xv)[TB]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
#pragma unroll
      for (int t = 0; t < TB; ++t)
        acc[t] = mfma_floats(static_cast<float>(wv.v[e]), static_cast<float>(xv[t].v[e]), acc[t]);
    }
  };
  // Groups of 16 features, eight of each a lane's; a wave takes every fourth.
  const int groups = static_cast<int>(c.dim / 16), col = h * 8;
  constexpr int kAhead = sizeof(T) == 2 ? 4 : 2;
  int k = wave;
  for (; k + (kAhead - 1) * kWaves < groups; k += kAhead * kWaves) {
    Pack<T, 8> wv[kAhead], xv[kAhead][TB];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int64_t at = (k + i * kWaves) * 16 + col;
      wv[i] = fetch<true, 8>(w + at, 8);
#pragma unroll
      for (int t = 0; t < TB; ++t) xv[i][t] = fetch<true, 8>(x[t] + at, 8);
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) multiply(wv[i], xv[i]);
  }
  for (; k * 16 < c.dim; k += kWaves) {
    const int64_t at = k * 16 + col;
    Pack<T, 8> wv{}, xv[TB] = {};
    if (at < c.dim) {
      wv = fetch<true, 8>(w + at, c.dim - at);
#pragma unroll
      for (int t = 0; t < TB; ++t) xv[t] = fetch<true, 8>(x[t] + at, c.dim - at);
    }
    multiply(wv, xv);
  }
  if (wave > 0) {
#pragma unroll
    for (int t = 0; t < TB; ++t) {
#pragma unroll
      for (int r = 0; r < 16; ++r) sums[wave - 1][t][r][lane] = acc[t][r];
    }
  }
  __syncthreads();
  if (wave > 0) return;
  float db[16] = {};
#pragma unroll
  for (int t = 0; t < TB; ++t) {
    const int64_t row = t * 32 + l;
    const int at = class_at(c, row);
    float z[16], most = -INFINITY;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      z[r] = (acc[t][r] + sums[0][t][r][lane]) + (sums[1][t][r][lane] + sums[2][t][r][lane]);
      const int64_t v = v0 + result_row(r);
      if (c.bias && v < c.classes) with_type(c.bias, c.bias_type, [&](auto *p) { z[r] += static_cast<float>(p[v]); });
      if (v >= c.classes) z[r] = -INFINITY;
      most = fmaxf(most, z[r]);
    }
    if constexpr (!BACKWARD) {
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (v0 + result_row(r) == at) a.hit[row] = z[r];
      most = fmaxf(most, lane_xor_f32(most, 32));
      const float base = most == -INFINITY ? 0.0f : most;
      float sum = 0.0f;
#pragma unroll
      for (int r = 0; r < 16; ++r) sum += exp_of(z[r] - base);
      sum += lane_xor_f32(sum, 32);
      if (h == 0) a.partial[v0 / kBlock * (TB * 32) + row] = make_float2(most, sum);
    } else {
      const int64_t in = min(row, c.rows - 1);
      const float lse = c.given_lse[in], miss = miss_of(c, fetch_loss(c, in)), scale = c.grad[in * c.grad_stride];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int64_t v = v0 + result_row(r);
        const float p = less_target(exp_of(z[r] - lse), v == at, miss);
        const float g = at >= 0 ? p * scale : 0.0f;
        a.g[v * (TB * 32) + row] = g;
        db[r] += g;
      }
    }
  }
  if constexpr (BACKWARD) {
    if (!c.db) return;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float v = group_sum<32>(db[r]);
      const int64_t at = v0 + result_row(r);
      if (l == 0 && at < c.classes) store_typed(c.db, c.bias_type, at, v);
    }
  }
}

// A row per workgroup: joins its pieces.  The last sums are the first workgroup's alone,
// of one row each in order: another launch for them.
__global__ void __launch_bounds__(256) narrow_join_kernel(NarrowArgs a, int rows_pad) {
  __shared__ float2 part[4];
  const CeCall &c = a.c;
  const int64_t row = blockIdx.x;
  float most = -INFINITY, sum = 0.0f;
#pragma unroll 4
  for (int64_t b = threadIdx.x; b < a.blocks; b += 256) {
    const float2 p = a.partial[b * rows_pad + row];
    const float m = fmaxf(most, p.x), base = m == -INFINITY ? 0.0f : m;
    sum = sum * exp_of(most - base) + p.y * exp_of(p.x - base);
    most = m;
  }
  auto join = [&](float m2, float s2) {
    const float m = fmaxf(most, m2), base = m == -INFINITY ? 0.0f : m;
    sum = sum * exp_of(most - base) + s2 * exp_of(m2 - base);
    most = m;
  };
#pragma unroll
  for (int j = 1; j < kWave; j <<= 1) join(__shfl_xor(most, j), __shfl_xor(sum, j));
  if (lane_id() == 0) part[threadIdx.x / kWave] = make_float2(most, sum);
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int k = 1; k < 4; ++k) join(part[k].x, part[k].y);
  const int at = class_at(c, row);
  const float base = most == -INFINITY ? 0.0f : most;
  c.lse[row] = at >= 0 ? base + logf(sum) : at == -1 ? 0.0f : NAN;
  c.loss[row] = at >= 0 ? loss_of(base, sum, a.hit[row]) : at == -1 ? 0.0f : NAN;
}

__global__ void __launch_bounds__(kWave) narrow_sums_kernel(NarrowArgs a) {
  const CeCall &c = a.c;
  const int64_t row = threadIdx.x;
  double s = 0.0, n = 0.0;
  if (row < c.rows) {
    s = c.loss[row];
    n = target_of(c, row) == c.ignore ? 0.0 : 1.0;
  }
#pragma unroll
  for (int j = 1; j < kWave; j <<= 1) {
    s += __shfl_xor(s, j);
    n += __shfl_xor(n, j);
  }
  if (row < 2) c.sums[row] = static_cast<float>(row ? n : s);
}

template <typename T, int TB>
__global__ void __launch_bounds__(kThreads) narrow_dx_kernel(NarrowArgs a) {
  const CeCall &c = a.c;
  const int lane = lane_id(), l = lane % 32, h = lane / 32;
  const int64_t j0 = (blockIdx.x * int64_t(kWaves) + threadIdx.x / kWave) * 128;
  if (j0 >= c.dim) return;
  // Whole blocks of 32 classes: g is there for all of them (zero past the classes).
  const int64_t each = ceil_div64(a.blocks, a.splits) * kBlock;
  const int64_t first = blockIdx.y * each, last = min(first + each, a.blocks * kBlock);
  const T *const w = static_cast<const T *>(c.w);
  const int dim = static_cast<int>(c.dim), col = static_cast<int>(j0) + 4 * l;
  f32x16 acc[4][TB] = {};
  constexpr int kAhead = 8;
  for (int64_t v0 = first; v0 < last; v0 += 2 * kAhead) {
    Words<T, 4> wv[kAhead];
    float gv[kAhead][TB];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int64_t v = v0 + 2 * i + h;
      wv[i] = four<T>(w + min(v, c.classes - 1) * c.w_stride, col, dim);
#pragma unroll
      for (int t = 0; t < TB; ++t) gv[i][t] = a.g[v * (TB * 32) + t * 32 + l];
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      f32x4 f = floats<T>(wv[i], col, dim);
      if (v0 + 2 * i + h >= c.classes) f = f32x4{}; // the last row again: it may be infinite
#pragma unroll
      for (int e = 0; e < 4; ++e) {
#pragma unroll
        for (int t = 0; t < TB; ++t) acc[e][t] = mfma_floats(f[e], gv[i][t], acc[e][t]);
      }
    }
  }
  // Row m of block e is feature 4 m + e.
#pragma unroll
  for (int t = 0; t < TB; ++t) {
    float *const out = a.dx_part + (blockIdx.y * int64_t(TB * 32) + t * 32 + l) * a.dim_pad + j0;
#pragma unroll
    for (int r = 0; r < 16; ++r)
      *reinterpret_cast<float4 *>(out + 4 * result_row(r)) =
          make_float4(acc[0][t][r], acc[1][t][r], acc[2][t][r], acc[3][t][r]);
  }
}

template <typename T>
__global__ void __launch_bounds__(256) narrow_finish_kernel(NarrowArgs a, int rows_pad) {
  const CeCall &c = a.c;
  const int64_t row = blockIdx.y, j = (blockIdx.x * int64_t(256) + threadIdx.x) * 4;
  if (j >= c.dim) return;
  const bool on = class_at(c, row) >= 0;
  float v[4] = {};
  if (on) {
#pragma unroll 4
    for (int64_t s = 0; s < a.splits; ++s) {
      const float4 p = *reinterpret_cast<const float4 *>(a.dx_part + (s * rows_pad + row) * a.dim_pad + j);
      v[0] += p.x, v[1] += p.y, v[2] += p.z, v[3] += p.w;
    }
  }
  put<true, 4>(static_cast<T *>(c.dx) + row * c.dx_stride + j, c.dim - j, v);
}

template <typename T, typename O, int TB>
__global__ void __launch_bounds__(kThreads) narrow_dw_kernel(NarrowArgs a) {
  const CeCall &c = a.c;
  const int lane = lane_id(), l = lane % 32, h = lane / 32;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t v0 = xcd_block() * kBlock;
  const uint64_t on = rows_counted(c);
  float gv[16 * TB]; // of class l, rows 2 s + h
#pragma unroll
  for (int s = 0; s < 16 * TB; ++s) gv[s] = a.g[(v0 + l) * (TB * 32) + 2 * s + h];
  for (int64_t j0 = wave * 128; j0 < c.dim; j0 += kWaves * 128) {
    f32x16 acc[4] = {};
    const int dim = static_cast<int>(c.dim), col = static_cast<int>(j0) + 4 * l;
    constexpr int kAhead = 8;
#pragma unroll
    for (int s0 = 0; s0 < 16 * TB; s0 += kAhead) {
      if (2 * s0 >= c.rows) continue;
      Words<T, 4> xv[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int64_t row = min(static_cast<int64_t>(2 * (s0 + i) + h), c.rows - 1);
        xv[i] = four<T>(static_cast<const T *>(c.x) + row * c.x_stride, col, dim);
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        f32x4 f = floats<T>(xv[i], col, dim);
        if (!(on >> (2 * (s0 + i) + h) & 1)) f = f32x4{}; // a row that counts nothing may hold anything
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] = mfma_floats(gv[s0 + i], f[e], acc[e]);
      }
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int64_t v = v0 + result_row(r), j = j0 + 4 * l;
      const float out[4] = {acc[0][r], acc[1][r], acc[2][r], acc[3][r]};
      if (v < c.classes && j < c.dim) put<true, 4>(static_cast<O *>(c.dw) + v * c.dw_stride + j, c.dim - j, out);
    }
  }
}

// ---- host --------------------------------------------------------------------------------

int row_blocks(int64_t rows) { return rows <= 32 ? 1 : 2; }

// Parts of the classes in dx's sum: some 2,048 waves, of 64 classes at least.
int64_t dx_splits(int64_t dim, int64_t classes) {
  const int64_t across = ceil_div64(dim, 128);
  return std::clamp<int64_t>(2048 / across, 1, std::max<int64_t>(1, classes / 64));
}

NarrowArgs narrow_layout(const CeCall &c, bool backward, void *work, size_t &bytes) {
  NarrowArgs a{};
  a.c = c;
  a.blocks = ceil_div64(c.classes, kBlock);
  a.dim_pad = ceil_div64(c.dim, 128) * 128;
  a.splits = dx_splits(c.dim, c.classes);
  const int64_t rows = row_blocks(c.rows) * 32;
  size_t at = 0;
  auto take = [&](auto *&q, int64_t count) {
    using P = std::remove_reference_t<decltype(*q)>;
    q = reinterpret_cast<P *>(static_cast<char *>(work) + at);
    at += Workspace::align(static_cast<size_t>(count) * sizeof(P));
  };
  if (backward) {
    take(a.g, a.blocks * kBlock * rows);
    take(a.dx_part, a.splits * rows * a.dim_pad);
  } else {
    take(a.partial, a.blocks * rows);
    take(a.hit, rows);
  }
  bytes = at;
  return a;
}

template <typename T, int TB> int32_t narrow_loss(const NarrowArgs &a, void *stream) {
  int32_t rc = launch(narrow_logit_kernel<T, TB, false>, dim3(a.blocks), dim3(kThreads), stream, a);
  if (rc == SPORDER_OK) rc = launch(narrow_join_kernel, dim3(a.c.rows), dim3(256), stream, a, TB * 32);
  if (rc == SPORDER_OK) rc = launch(narrow_sums_kernel, dim3(1), dim3(kWave), stream, a);
  return rc;
}

template <typename T, int TB> int32_t narrow_grad(const NarrowArgs &a, void *stream) {
  int32_t rc = launch(narrow_logit_kernel<T, TB, true>, dim3(a.blocks), dim3(kThreads), stream, a);
  if (rc != SPORDER_OK) return rc;
  rc = launch(narrow_dx_kernel<T, TB>, dim3(ceil_div64(a.c.dim, kWaves * 128), a.splits), dim3(kThreads), stream, a);
  if (rc != SPORDER_OK) return rc;
  rc = launch(narrow_finish_kernel<T>, dim3(ceil_div64(a.c.dim, 1024), a.c.rows), dim3(256), stream, a, TB * 32);
  if (rc != SPORDER_OK) return rc;
  if constexpr (sizeof(T) == 2) {
    if (a.c.dw_type != SPORDER_TYPE_F32)
      return launch(narrow_dw_kernel<T, T, TB>, dim3(a.blocks), dim3(kThreads), stream, a);
  }
  return launch(narrow_dw_kernel<T, float, TB>, dim3(a.blocks), dim3(kThreads), stream, a);
}

template <typename T> int32_t narrow_typed(const NarrowArgs &a, bool backward, void *stream) {
  if (row_blocks(a.c.rows) == 1)
    return backward ? narrow_grad<T, 1>(a, stream) : narrow_loss<T, 1>(a, stream);
  return backward ? narrow_grad<T, 2>(a, stream) : narrow_loss<T, 2>(a, stream);
}

} // namespace

// Measured both ways.  32-bit types: 50,000 x 4,096, one row 243 us and the tiles 648 (with the
// gradients 668 and 1,646), 30,000 x 4,096, 64 rows 302 and 449 (791 and 1,153).  16-bit
// types, whose w the tiles read as it is: forward 164 and 106 us for one row of the first, 156
// and 65 for 64, but 35 and 37 for up to 32 rows of 16,000 x 2,048 and 24 and 28 of 1,000 x 512
// (three launches instead of five); with the gradients 491 and 812, 16 rows of 50,000 x 2,048
// 268 and 443, but 64 rows 627 and 380.
bool narrow_takes(int type, int64_t rows, int64_t dim, int64_t classes, bool backward) {
  if (dim < 8) return false;
  if (type == SPORDER_TYPE_F32) return rows <= 64;
  return rows <= 32 && (backward || classes * dim <= int64_t(1) << 25);
}

size_t narrow_work_bytes(int64_t rows, int64_t dim, int64_t classes, bool backward) {
  CeCall c{};
  c.rows = rows, c.dim = dim, c.classes = classes;
  size_t bytes = 0;
  narrow_layout(c, backward, nullptr, bytes);
  return bytes;
}

int32_t narrow_run(const CeCall &c, bool backward, void *work, void *stream) {
  size_t bytes = 0;
  const NarrowArgs a = narrow_layout(c, backward, work, bytes);
  if (c.type == SPORDER_TYPE_BF16) return narrow_typed<bf16_t>(a, backward, stream);
  if (c.type == SPORDER_TYPE_F16) return narrow_typed<f16_t>(a, backward, stream);
  return narrow_typed<float>(a, backward, stream);
}

} // namespace sporder_hip
