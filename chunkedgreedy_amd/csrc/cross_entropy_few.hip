// cross_entropy_few.hip -- linear cross entropy where all classes' weights fit a
// workgroup's LDS (a graph's node classes): one pass over the rows each way.
//
// A workgroup keeps w in LDS and takes 16 or 32 rows at a time:
//   z^T = w x^T      classes down (a lane's registers), rows across (lanes)
//   dx^T = w^T g^T   features down, rows across
//   dw = g^T x       classes down, features across, in registers over all tiles
// Three kernels: the loss, whose rows never see LDS; the gradients where a wave's own tile
// fits LDS besides w; and the gradients with tiles shared by the workgroup, in 32-bit
// products (16 x 16 x 4 per matrix instruction) whatever the type.
// A matrix instruction's four steps along the sum may be any four: there lane group q
// takes elements 4 q .. 4 q + 3 of 16 (one LDS access for four instructions where
// they lie side by side), and in the last two products rows r + 4 q, which
// with rows 4 floats longer than a multiple of 16 lie in different banks.
#include <algorithm>

#include "cross_entropy.hpp"
#include "mfma_product.hpp"

namespace sporder_hip {

namespace {

constexpr int kLossThreads = 256, kGradThreads = 512;
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

// Floats of a row of x or w in LDS: whole blocks of 64 features, so that rows' places are
// constants (a stride known at run time cost 36 registers of addresses).
constexpr int few_stride(int feature_blocks) { return feature_blocks * 64 + 4; }

// w and the bias (-inf past the classes) to LDS.
template <typename T, int VB, int DB, int THREADS>
__device__ __forceinline__ void hold_weights(const CeCall &c, float *w, float *bias) {
  constexpr int stride = few_stride(DB);
  const int part = threadIdx.x % 16 * 4, dim = static_cast<int>(c.dim);
  for (int v = threadIdx.x / 16; v < VB * 16; v += THREADS / 16) {
    const T *const row = static_cast<const T *>(c.w) + v * c.w_stride;
#pragma unroll
    for (int k = 0; k < DB; ++k)
      *reinterpret_cast<f32x4 *>(w + v * stride + k * 64 + part) =
          v < c.classes ? floats<T>(four<T>(row, k * 64 + part, dim), k * 64 + part, dim) : f32x4{};
  }
  for (int v = threadIdx.x; v < VB * 16; v += THREADS) {
    float b = v < c.classes ? 0.0f : -INFINITY;
    if (c.bias && v < c.classes) with_type(c.bias, c.bias_type, [&](auto *p) { b = static_cast<float>(p[v]); });
    bias[v] = b;
  }
}

// The targets of the rows that a thread fetches of a tile: 16 threads a row, STEP rows
// at a time.
template <int STEP, int N>
__device__ __forceinline__ void fetch_targets(const CeCall &c, int64_t first, RawTarget (&t)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) t[i] = fetch_target(c, first + i * STEP + threadIdx.x / 16);
}
template <int STEP, int N>
__device__ __forceinline__ void classes_of(const CeCall &c, int64_t first, const RawTarget (&t)[N], int (&k)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) k[i] = class_of(c, first + i * STEP + threadIdx.x / 16, t[i]);
}

// The rows' words on their way.  Rows that count nothing are read as the first one, which
// the caches hold: a branch around the loads would make each wait for its target.
template <typename T, int STEP, int N, int DB>
__device__ __forceinline__ void fetch_tile(const CeCall &c, int64_t first, const int (&t)[N],
                                           Words<T, 4> (&v)[N][DB]) {
  const int part = threadIdx.x % 16 * 4;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int64_t row = t[i] >= 0 ? first + i * STEP + threadIdx.x / 16 : 0;
    const T *const x = static_cast<const T *>(c.x) + row * c.x_stride;
#pragma unroll
    for (int k = 0; k < DB; ++k) v[i][k] = four<T>(x, k * 64 + part, static_cast<int>(c.dim));
  }
}

// And in LDS, zeros for those that count nothing and past their ends.
template <typename T, int STEP, int N, int DB>
__device__ __forceinline__ void put_tile(const CeCall &c, float *x, const int (&t)[N],
                                         const Words<T, 4> (&v)[N][DB]) {
  const int part = threadIdx.x % 16 * 4;
#pragma unroll
  for (int i = 0; i < N; ++i) {
#pragma unroll
    for (int k = 0; k < DB; ++k) {
      const int col = k * 64 + part;
      *reinterpret_cast<f32x4 *>(x + (i * STEP + threadIdx.x / 16) * few_stride(DB) + col) =
          t[i] >= 0 ? floats<T>(v[i][k], col, static_cast<int>(c.dim)) : f32x4{};
    }
  }
}

// z of 16 rows (of x, from `rows` on) and every STEP-th block of 16 classes, `blocks` of
// them.
template <int BLOCKS, int STEP, int DB>
__device__ __forceinline__ void logits(const float *w, const float *rows, int dim16, int blocks,
                                       f32x4 (&z)[BLOCKS]) {
  constexpr int stride = few_stride(DB);
  const int lane = lane_id(), at = lane % 16 * stride + lane / 16 * 4;
  for (int k = 0; k < dim16; ++k) {
    const f32x4 b = *reinterpret_cast<const f32x4 *>(rows + at + k * 16);
#pragma unroll
    for (int v = 0; v < BLOCKS; ++v) {
      if (v >= blocks) continue;
      const f32x4 a = *reinterpret_cast<const f32x4 *>(w + v * STEP * 16 * stride + at + k * 16);
#pragma unroll
      for (int e = 0; e < 4; ++e) z[v] = mfma_16x16(a[e], b[e], z[v]);
    }
  }
}

// ---- forward: rows straight from memory, 16 a wave ----------------------------------------

// A lane's eight neighbouring features of a row are what a matrix instruction takes, so x
// goes from memory to registers and to the products, and only w is in LDS: 16-bit types as
// they are, 32-bit ones as two 16-bit halves of their row's unit, three products for each
// (22 bits).  An access that would pass the row's end is the row's last one, and w's copy in
// LDS has those features there, each once, and zeros: nothing of x is moved or masked.
// 2,449,029 rows of 128, 47 classes in 280 to 306 us (4.2 to 4.5 TB/s; 32-bit products from
// tiles in LDS took 482), bfloat16 140 (4.8 TB/s; 430); 580,000 rows of 500, 80 classes, bfloat16
// 130 us (tiles of any number of classes: 464).  What keeps it from a copy's rate are the address
// units, busy 81 % of the time (bfloat16 77 %): an access of a wave lies in 16 rows.
template <typename T> struct LossType {
  using U = T;
  static constexpr int kPlanes = 1;
};
template <> struct LossType<float> {
  using U = f16_t;
  static constexpr int kPlanes = 2;
};

__device__ __forceinline__ f32x4 mfma_sixteen(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma_sixteen(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ void split_eight(const float (&v)[8], f16x8 &hi, f16x8 &lo) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const f16_t h = static_cast<f16_t>(v[e]);
    hi[e] = h;
    lo[e] = static_cast<f16_t>(v[e] - static_cast<float>(h));
  }
}

template <typename T> constexpr int loss_lds(int class_blocks, int feature_blocks) {
  return class_blocks * 16 * ((feature_blocks * 64 + 8) * 2 * LossType<T>::kPlanes + 8);
}
// Workgroups on a CU that registers allow.
template <typename T> constexpr int loss_groups(int class_blocks, int feature_blocks) {
  const int bytes = feature_blocks * sizeof(T);
  return bytes <= 8 && class_blocks <= 6 && class_blocks * bytes <= 32 ? 2 : 1;
}

template <typename T, int VB, int DB>
__global__ void __launch_bounds__(kGradThreads, 2 * loss_groups<T>(VB, DB)) few_loss_kernel(FewArgs a) {
  extern __shared__ __attribute__((aligned(16))) float lds[];
  using U = typename LossType<T>::U;
  using U8 = U __attribute__((ext_vector_type(8)));
  constexpr int kPlanes = LossType<T>::kPlanes, kVec = 16 / sizeof(T), kV = VB * 16, kW = DB * 64 + 8;
  constexpr int kParts = 8 / kVec; // accesses for eight features
  constexpr bool kAhead = DB * sizeof(T) <= 16; // the next row's words have room in registers
  const CeCall &c = a.c;
  const int dim = static_cast<int>(c.dim), tid = threadIdx.x, lane = lane_id(), q = lane / 16, l = lane % 16;
  float *const w_unit = lds, *const bias = lds + kV;
  U *const w = reinterpret_cast<U *>(lds + 2 * kV); // hi, then lo

  // w by accesses as x's, 16 threads a row.
  const int part = tid % 16 * 4, inside = part % kVec;
  for (int v = tid / 16; v < kV; v += kGradThreads / 16) {
    const T *const row = static_cast<const T *>(c.w) + min(static_cast<int64_t>(v), c.classes - 1) * c.w_stride;
    f32x4 f[DB];
    float most = 0.0f;
#pragma unroll
    for (int k = 0; k < DB; ++k) {
      const int start = k * 64 + part - inside, from = min(start, dim - kVec) + inside;
      const auto p = __builtin_bit_cast(Pack<T, 4>, *reinterpret_cast<const LoosePack<T, 4> *>(row + from));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f[k][e] = v < c.classes && from + e >= start ? static_cast<float>(p.v[e]) : 0.0f;
        most = fmaxf(most, fabsf(f[k][e]));
      }
    }
    float scale = 1.0f;
    if constexpr (kPlanes == 2) {
      const float u = unit_of(group_max<16>(most));
      scale = unit_inverse(u);
      if (part == 0) w_unit[v] = u;
    }
#pragma unroll
    for (int k = 0; k < DB; ++k) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float s = f[k][e] * scale;
        const U h = static_cast<U>(s);
        w[v * kW + k * 64 + part + e] = h;
        if constexpr (kPlanes == 2) w[(kV + v) * kW + k * 64 + part + e] = static_cast<U>(s - static_cast<float>(h));
      }
    }
  }
  for (int v = tid; v < kV; v += kGradThreads) {
    float b = v < c.classes ? 0.0f : -INFINITY;
    if (c.bias && v < c.classes) with_type(c.bias, c.bias_type, [&](auto *p) { b = static_cast<float>(p[v]); });
    bias[v] = b;
  }
  __syncthreads();

  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int64_t step = gridDim.x * int64_t(kGradThreads / kWave * 16);
  const int64_t first = (blockIdx.x * int64_t(kGradThreads / kWave) + wave) * 16;
  int next_at;
  RawTarget next_target;
  Words<T, kVec> next[DB * 2][kParts];
  // Rows that count nothing are read as the first one, which the caches hold.
  auto fetch_row = [&](int64_t r) {
    next_at = class_of(c, r, next_target);
    const T *const x = static_cast<const T *>(c.x) + (next_at >= 0 ? r : 0) * c.x_stride;
#pragma unroll
    for (int k = 0; k < DB * 2; ++k) {
#pragma unroll
      for (int i = 0; i < kParts; ++i)
        next[k][i] = __builtin_bit_cast(Words<T, kVec>, *reinterpret_cast<const LoosePack<T, kVec> *>(
                                                            x + min(k * 32 + q * 8 + i * kVec, dim - kVec)));
    }
  };
  next_target = fetch_target(c, first + l);
  if constexpr (kAhead) {
    fetch_row(first + l);
    __builtin_amdgcn_sched_barrier(0); // loads in the loop's order, so that it waits for no later ones
    next_target = fetch_target(c, first + l + step);
  }
  double sum = 0.0, n = 0.0;
  for (int64_t r0 = first; r0 < c.rows; r0 += step) {
    const int64_t row = r0 + l;
    if constexpr (!kAhead) {
      fetch_row(row);
      next_target = fetch_target(c, row + step);
    }
    Words<T, kVec> x[DB * 2][kParts];
#pragma unroll
    for (int k = 0; k < DB * 2; ++k) {
#pragma unroll
      for (int i = 0; i < kParts; ++i) x[k][i] = next[k][i];
    }
    const int at = next_at;
    if constexpr (kAhead) {
      fetch_row(row + step);
      next_target = fetch_target(c, row + 2 * step);
    }
    float unit = 1.0f, inverse = 1.0f;
    if constexpr (kPlanes == 2) {
      float most = 0.0f;
#pragma unroll
      for (int k = 0; k < DB * 2; ++k) {
#pragma unroll
        for (int i = 0; i < kParts; ++i) {
          const auto p = __builtin_bit_cast(Pack<T, kVec>, x[k][i]);
#pragma unroll
          for (int e = 0; e < kVec; ++e) most = fmaxf(most, fabsf(static_cast<float>(p.v[e])));
        }
      }
      most = fmaxf(most, lane_xor_f32(most, 16));
      most = fmaxf(most, lane_xor_f32(most, 32));
      unit = unit_of(most);
      inverse = unit_inverse(unit);
    }
    // Places in LDS that the compiler can't tell from the last row's, or it would keep all of
    // w in registers.
    uint32_t w_at = l * kW + q * 8, four_at = q * 4;
    asm volatile("" : "+v"(w_at), "+v"(four_at));
    f32x4 z[VB] = {};
#pragma unroll
    for (int k = 0; k < DB * 2; ++k) {
      U8 hi, lo;
      if constexpr (kPlanes == 2) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const auto p = __builtin_bit_cast(Pack<T, kVec>, x[k][i]);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[i * 4 + e] = p.v[e] * inverse;
        }
        split_eight(v, hi, lo);
      } else {
        hi = __builtin_bit_cast(U8, x[k][0]);
      }
#pragma unroll
      for (int b = 0; b < VB; ++b) {
        const U *const from = w + w_at + b * 16 * kW + k * 32;
        const U8 wh = *reinterpret_cast<const U8 *>(from);
        z[b] = mfma_sixteen(wh, hi, z[b]);
        if constexpr (kPlanes == 2) {
          z[b] = mfma_sixteen(wh, lo, z[b]);
          z[b] = mfma_sixteen(*reinterpret_cast<const U8 *>(from + kV * kW), hi, z[b]);
        }
      }
    }
    float most = -INFINITY, hit = 0.0f;
    const int mine = at - static_cast<int>(four_at);
#pragma unroll
    for (int v = 0; v < VB; ++v) {
      const f32x4 b = *reinterpret_cast<const f32x4 *>(bias + four_at + v * 16);
      if constexpr (kPlanes == 2) {
        const f32x4 u = *reinterpret_cast<const f32x4 *>(w_unit + four_at + v * 16);
#pragma unroll
        for (int e = 0; e < 4; ++e) z[v][e] = z[v][e] * unit * u[e];
      }
      z[v] += b;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        most = fmaxf(most, z[v][e]);
        hit += v * 16 + e == mine ? z[v][e] : 0.0f;
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
    if (lane < 16 && at > -3) {
      float lse = base + logf(total), loss = loss_of(base, total, hit);
      if (at < 0) loss = lse = at == -1 ? 0.0f : NAN;
      c.lse[row] = lse;
      c.loss[row] = loss;
      sum += loss;
      n += at == -1 ? 0.0 : 1.0;
    }
  }
  __shared__ double parts[2][kGradThreads / kWave];
  const double v = block_sums(sum, n, parts);
  if (tid >= 2) return;
  if (gridDim.x == 1)
    c.sums[tid] = static_cast<float>(v);
  else
    a.sums[2 * blockIdx.x + tid] = v;
}

__global__ void __launch_bounds__(kLossThreads) few_total_kernel(FewArgs a, int blocks) {
  __shared__ double part[2][4];
  double s = 0.0, n = 0.0;
  for (int i = threadIdx.x; i < blocks; i += kLossThreads) {
    s += a.sums[2 * i];
    n += a.sums[2 * i + 1];
  }
  const double v = block_sums(s, n, part);
  if (threadIdx.x < 2) a.c.sums[threadIdx.x] = static_cast<float>(v);
}

// ---- backward: 32 rows a tile, eight waves -----------------------------------------------

constexpr int kRows = 32, kSplit = 4; // waves that share a block of 16 rows

// dx of a tile goes out a tile later, by whole rows through LDS.  (Stored from the
// accumulators, 64 bytes of 16 rows at a time, it took a third of the kernel's time; stored at
// the tile's end, the next tile's loads waited for it.)
template <typename T, int VB, int DB>
__global__ void __launch_bounds__(kGradThreads, VB * ((DB + 1) / 2) <= 4 && DB < 8 ? 4 : 2) few_grad_kernel(FewArgs a) {
  extern __shared__ __attribute__((aligned(16))) float lds[];
  constexpr int kMine = (VB + kSplit - 1) / kSplit;
  constexpr int kG = VB * 16 + 4;  // floats of a row of g
  constexpr int kD = (DB + 1) / 2; // blocks of 128 features
  constexpr int stride = few_stride(DB);
  const CeCall &c = a.c;
  const int dim16 = static_cast<int>(ceil_div64(c.dim, 16));
  float *const w = lds, *const x = w + VB * 16 * stride, *const dx = x + kRows * stride;
  float *const g = dx + kRows * stride, *const bias = g + kRows * kG;
  const int lane = lane_id(), q = lane / 16, l = lane % 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int tb = wave % 2, part = wave / 2;
  hold_weights<T, VB, DB, kGradThreads>(c, w, bias);
  f32x4 dw[VB][kD] = {};
  float db[VB] = {};
  const int64_t step = gridDim.x * int64_t(kRows), first = blockIdx.x * int64_t(kRows);
  int target[1];            // of the rows on their way
  RawTarget next_target[1]; // of those after them
  Words<T, 4> next[1][DB];
  fetch_targets<32>(c, first, next_target);
  classes_of<32>(c, first, next_target, target);
  fetch_tile<T, 32>(c, first, target, next);
  __builtin_amdgcn_sched_barrier(0); // loads in the loop's order, so that it waits for no later ones
  fetch_targets<32>(c, first + step, next_target);
  // This lane's row: its class, scale and lse, a tile ahead too.
  RawTarget next_class;
  float next_lse, next_loss, next_scale;
  auto fetch_row = [&](int64_t r) {
    next_class = fetch_target(c, r);
    const int64_t in = min(r, c.rows - 1);
    next_lse = c.given_lse[in];
    next_loss = fetch_loss(c, in);
    next_scale = c.grad[in * c.grad_stride];
  };
  fetch_row(first + tb * 16 + l);
  auto put_dx = [&](int64_t tile) {
    const int64_t r = tile * kRows + threadIdx.x / 16;
    if (r >= c.rows) return;
    T *const out = static_cast<T *>(c.dx) + r * c.dx_stride;
#pragma unroll
    for (int k = 0; k < DB; ++k) {
      const int col = k * 64 + threadIdx.x % 16 * 4;
      if (col >= c.dim) continue;
      const f32x4 f = *reinterpret_cast<const f32x4 *>(dx + threadIdx.x / 16 * stride + col);
      const float v[4] = {f[0], f[1], f[2], f[3]};
      put<true, 4>(out + col, c.dim - col, v);
    }
  };
  int64_t tile = blockIdx.x;
  for (; tile < a.tiles; tile += gridDim.x) {
    __syncthreads(); // x is read no more, the last tile's dx is there
    put_tile<T, 32>(c, x, target, next);
    __syncthreads();
    classes_of<32>(c, tile * kRows + step, next_target, target);
    fetch_tile<T, 32>(c, tile * kRows + step, target, next);
    fetch_targets<32>(c, tile * kRows + 2 * step, next_target);
    const int64_t row = tile * kRows + tb * 16 + l; // made anew: registers are short
    const int at = class_of(c, row, next_class);
    const float lse = at >= 0 ? next_lse : 0.0f, miss = miss_of(c, next_loss), s = next_scale;
    fetch_row(row + step);
    if (tile != blockIdx.x) put_dx(tile - gridDim.x);

    // g of this wave's rows and classes.
    f32x4 z[kMine] = {};
    logits<kMine, kSplit, DB>(w + part * 16 * stride, x + tb * 16 * stride, dim16,
                              (VB - part + kSplit - 1) / kSplit, z);
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int v = (i * kSplit + part) * 16 + q * 4;
      if (v >= VB * 16) continue;
      const f32x4 b = *reinterpret_cast<const f32x4 *>(bias + v);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p = less_target(exp_of(z[i][e] + b[e] - lse), v + e == at, miss);
        z[i][e] = at >= 0 ? p * s : 0.0f;
      }
      *reinterpret_cast<f32x4 *>(g + (tb * 16 + l) * kG + v) = z[i];
    }
    __syncthreads();

    // dx: this wave's rows and every kSplit-th block of features.
#pragma unroll 1
    for (int j = part; j < dim16; j += kSplit) {
      f32x4 d = {};
#pragma unroll
      for (int v = 0; v < VB; ++v) {
        const f32x4 gv = *reinterpret_cast<const f32x4 *>(g + (tb * 16 + l) * kG + v * 16 + q * 4);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          d = mfma_16x16(w[(v * 16 + q * 4 + e) * stride + j * 16 + l], gv[e], d);
      }
      if (at < 0) d = f32x4{}; // g is 0, but w may hold anything
      *reinterpret_cast<f32x4 *>(dx + (tb * 16 + l) * stride + j * 16 + q * 4) = d;
    }
    // dw: all classes and every eighth block of features.
#pragma unroll 1
    for (int t = 0; t < kRows / 16; ++t) {
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
        for (int k = 0; k < kD; ++k) {
          if (k * 8 + wave >= dim16) continue;
          const float xv = x[r * stride + (k * 8 + wave) * 16 + l];
#pragma unroll
          for (int v = 0; v < VB; ++v) dw[v][k] = mfma_16x16(gv[v], xv, dw[v][k]);
        }
      }
    }
  }
  __syncthreads();
  put_dx(tile - gridDim.x);
  float *const out = a.dw_part + blockIdx.x * int64_t(VB * 16) * (dim16 * 16);
#pragma unroll
  for (int v = 0; v < VB; ++v) {
#pragma unroll
    for (int k = 0; k < kD; ++k) {
      if (k * 8 + wave >= dim16) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        out[(v * 16 + q * 4 + e) * (dim16 * 16) + (k * 8 + wave) * 16 + l] = dw[v][k][e];
    }
    db[v] += lane_xor_f32(db[v], 16);
    db[v] += lane_xor_f32(db[v], 32);
    if (wave == 0 && q == 0) a.db_part[blockIdx.x * int64_t(VB * 16) + v * 16 + l] = db[v];
  }
}

// ---- backward, a wave to itself: 16 rows a tile -------------------------------------------

// Where w is small enough for LDS to hold besides it a tile for each of eight waves,
// every wave takes tiles of its own and keeps a dw of its own, so that nothing waits at
// barriers and one wave's loads and stores run beside another's products (rows of 128, 47
// classes: with tiles shared by eight waves the products' 750 us and memory's 420 came one
// after the other).  z and dx are products of 16-bit halves here, three for each (22 bits,
// in units of x's and w's rows and w's columns, as in the tiled form), at a fifth of the
// 32-bit products' time; dw, which sums over rows of any scale, stays with those.  Rows are
// of whole accesses of four elements, and dx's at such addresses.
template <int VB, int DB> struct WaveShape {
  static constexpr int kV = VB * 16, kV32 = (VB + 1) / 2 * 32, kD = DB * 64;
  static constexpr int kW = kD + 8, kT = kV32 + 8;   // halves of a row of w and of w^T
  static constexpr int kX = kD + 4, kG = kV + 4;     // floats of a row of x and g
  static constexpr int kWaves = kGradThreads / kWave;
  static constexpr int kTile = 16 * (kX + kG) + 16;  // floats of a wave
  static constexpr int kHalves = 2 * (kV * kW + kD * kT);
  static constexpr int kFloats = kHalves / 2 + 2 * kV + kD + kWaves * kTile;
  static constexpr int kJoin = kV * kX + kV;         // dw and db of the workgroup, over it all
  static constexpr bool kFits = VB * DB <= 6 && VB < 6 && kFloats * 4 <= kLds && kJoin <= kFloats;
};

template <typename T, int VB, int DB>
__global__ void __launch_bounds__(kGradThreads, 2) few_grad_wave_kernel(FewArgs a) {
  extern __shared__ __attribute__((aligned(16))) float lds[];
  using S = WaveShape<VB, DB>;
  const CeCall &c = a.c;
  const int dim = static_cast<int>(c.dim), dim16 = (dim + 15) / 16;
  f16_t *const w = reinterpret_cast<f16_t *>(lds), *const wt = w + 2 * S::kV * S::kW; // hi, then lo
  float *const w_unit = lds + S::kHalves / 2, *const bias = w_unit + S::kV, *const t_unit = bias + S::kV;
  const int tid = threadIdx.x, lane = lane_id(), q = lane / 16, l = lane % 16;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  float *const x = t_unit + S::kD + wave * S::kTile, *const g = x + 16 * S::kX, *const x_unit = g + 16 * S::kG;

  // w's rows in their units, 16 threads a row.
  const int part = tid % 16 * 4;
  for (int v = tid / 16; v < S::kV; v += kGradThreads / 16) {
    const T *const row = static_cast<const T *>(c.w) + min(static_cast<int64_t>(v), c.classes - 1) * c.w_stride;
    f32x4 f[DB];
    float most = 0.0f;
#pragma unroll
    for (int k = 0; k < DB; ++k) {
      f[k] = floats<T>(four<T>(row, k * 64 + part, dim), k * 64 + part, dim);
#pragma unroll
      for (int e = 0; e < 4; ++e) most = fmaxf(most, fabsf(f[k][e]));
    }
    const float u = unit_of(group_max<16>(most)), scale = unit_inverse(u);
    if (part == 0) w_unit[v] = u;
#pragma unroll
    for (int k = 0; k < DB; ++k) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float s = v < c.classes ? f[k][e] * scale : 0.0f;
        const f16_t h = static_cast<f16_t>(s);
        w[v * S::kW + k * 64 + part + e] = h;
        w[(S::kV + v) * S::kW + k * 64 + part + e] = static_cast<f16_t>(s - static_cast<float>(h));
      }
    }
  }
  // w's columns in theirs: of 32 classes 16 (e / 4) + 4 q + e % 4 is a lane group's half e.
  for (int j = tid; j < S::kD; j += kGradThreads) {
    const T *const col = static_cast<const T *>(c.w) + min(j, dim - 1);
    float most = 0.0f;
    for (int v = 0; v < static_cast<int>(c.classes); ++v) most = fmaxf(most, fabsf(static_cast<float>(col[v * c.w_stride])));
    const float u = unit_of(most), scale = unit_inverse(u);
    t_unit[j] = u;
    for (int i = 0; i < S::kV32; ++i) {
      const int v = i / 32 * 32 + i % 8 / 4 * 16 + i % 32 / 8 * 4 + i % 4;
      const float s = v < c.classes && j < dim ? static_cast<float>(col[v * c.w_stride]) * scale : 0.0f;
      const f16_t h = static_cast<f16_t>(s);
      wt[j * S::kT + i] = h;
      wt[(S::kD + j) * S::kT + i] = static_cast<f16_t>(s - static_cast<float>(h));
    }
  }
  for (int v = tid; v < S::kV; v += kGradThreads) {
    float b = v < c.classes ? 0.0f : -INFINITY;
    if (c.bias && v < c.classes) with_type(c.bias, c.bias_type, [&](auto *p) { b = static_cast<float>(p[v]); });
    bias[v] = b;
  }
  __syncthreads();

  f32x4 dw[VB][DB * 4] = {};
  float db[VB] = {};
  const int64_t step = gridDim.x * int64_t(S::kWaves * 16), first = (blockIdx.x * int64_t(S::kWaves) + wave) * 16;
  // Rows on their way: 16 lanes a row, four at a time.
  int target[4];
  RawTarget next_target[4];
  Words<T, 4> next[4][DB];
  auto targets_from = [&](int64_t r) {
#pragma unroll
    for (int i = 0; i < 4; ++i) next_target[i] = fetch_target(c, r + i * 4 + q);
  };
  // A tile's rows from a base that the wave shares, in bytes: registers are short.
  const uint32_t x_step = static_cast<uint32_t>(c.x_stride * sizeof(T));
  const uint32_t dx_step = static_cast<uint32_t>(c.dx_stride * sizeof(T));
  auto rows_from = [&](int64_t r) {
    const char *const base = static_cast<const char *>(c.x) + min(r, c.rows - 1) * (c.x_stride * sizeof(T));
    uint32_t mine = q * x_step;
    asm volatile("" : "+v"(mine)); // as below
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      target[i] = class_of(c, r + i * 4 + q, next_target[i]);
      const uint32_t row = target[i] >= 0 ? mine + i * 4 * x_step : 0;
#pragma unroll
      for (int k = 0; k < DB; ++k) {
        const uint32_t col = static_cast<uint32_t>(min(k * 64 + l * 4, dim - 4) * sizeof(T));
        next[i][k] = __builtin_bit_cast(Words<T, 4>, *reinterpret_cast<const LoosePack<T, 4> *>(base + (row + col)));
      }
    }
  };
  RawTarget next_class;
  float next_lse, next_loss, next_scale;
  auto fetch_row = [&](int64_t r) {
    next_class = fetch_target(c, r);
    const int64_t in = min(r, c.rows - 1);
    next_lse = c.given_lse[in];
    next_loss = fetch_loss(c, in);
    next_scale = c.grad[in * c.grad_stride];
  };
  targets_from(first);
  rows_from(first);
  __builtin_amdgcn_sched_barrier(0); // loads in the loop's order, so that it waits for no later ones
  targets_from(first + step);
  fetch_row(first + l);

  for (int64_t r0 = first; r0 < c.rows; r0 += step) {
    wave_lds_order(); // the last tile's rows are out
    const bool every = __all(min(min(target[0], target[1]), min(target[2], target[3])) >= 0);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float most = 0.0f;
#pragma unroll
      for (int k = 0; k < DB; ++k) {
        const auto p = __builtin_bit_cast(Pack<T, 4>, next[i][k]);
        f32x4 f;
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = static_cast<float>(p.v[e]);
        if (k == DB - 1 && k * 64 + l * 4 >= dim) f = f32x4{};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (!every) f[e] = target[i] >= 0 ? f[e] : 0.0f;
          most = fmaxf(most, fabsf(f[e]));
        }
        *reinterpret_cast<f32x4 *>(x + (i * 4 + q) * S::kX + k * 64 + l * 4) = f;
      }
      most = group_max<16>(most);
      if (l == 0) x_unit[i * 4 + q] = unit_of(most);
    }
    wave_lds_order();
    rows_from(r0 + step);
    targets_from(r0 + 2 * step);
    const int at = class_of(c, r0 + l, next_class);
    const float lse = at >= 0 ? next_lse : 0.0f, miss = miss_of(c, next_loss), scale = next_scale;
    fetch_row(r0 + step + l);

    // z, and g of them.
    const float unit = x_unit[l], inverse = unit_inverse(unit);
    f32x4 z[VB] = {};
#pragma unroll
    for (int k = 0; k < DB * 2; ++k) {
      const f32x4 one = *reinterpret_cast<const f32x4 *>(x + l * S::kX + k * 32 + q * 8);
      const f32x4 two = *reinterpret_cast<const f32x4 *>(x + l * S::kX + k * 32 + q * 8 + 4);
      float v[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] = one[e] * inverse;
        v[4 + e] = two[e] * inverse;
      }
      f16x8 hi, lo;
      split_eight(v, hi, lo);
      f16x8 wh[VB], wl[VB];
#pragma unroll
      for (int b = 0; b < VB; ++b) {
        const f16_t *const from = w + (b * 16 + l) * S::kW + k * 32 + q * 8;
        wh[b] = *reinterpret_cast<const f16x8 *>(from);
        wl[b] = *reinterpret_cast<const f16x8 *>(from + S::kV * S::kW);
      }
#pragma unroll
      for (int b = 0; b < VB; ++b) z[b] = mfma_sixteen(wl[b], hi, z[b]);
#pragma unroll
      for (int b = 0; b < VB; ++b) z[b] = mfma_sixteen(wh[b], lo, z[b]);
#pragma unroll
      for (int b = 0; b < VB; ++b) z[b] = mfma_sixteen(wh[b], hi, z[b]);
    }
    f16x8 gh[S::kV32 / 32], gl[S::kV32 / 32];
#pragma unroll
    for (int b = 0; b < VB; ++b) {
      const int v = b * 16 + q * 4;
      const f32x4 add = *reinterpret_cast<const f32x4 *>(bias + v), u = *reinterpret_cast<const f32x4 *>(w_unit + v);
      f32x4 out;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p = less_target(exp_of(z[b][e] * (unit * u[e]) + add[e] - lse), v + e == at, miss);
        const float held = at >= 0 ? p : 0.0f, much = held * 8192.0f;
        out[e] = at >= 0 ? held * scale : 0.0f;
        const f16_t h = static_cast<f16_t>(much);
        gh[b / 2][b % 2 * 4 + e] = h;
        gl[b / 2][b % 2 * 4 + e] = static_cast<f16_t>(much - static_cast<float>(h));
      }
      *reinterpret_cast<f32x4 *>(g + l * S::kG + v) = out;
    }
    if constexpr (VB % 2 == 1) { // no classes there
#pragma unroll
      for (int e = 4; e < 8; ++e) gh[VB / 2][e] = gl[VB / 2][e] = static_cast<f16_t>(0.0f);
    }

    wave_lds_order();
    // dw.
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float gv[VB];
#pragma unroll
      for (int b = 0; b < VB; ++b) {
        gv[b] = g[(q * 4 + e) * S::kG + b * 16 + l];
        db[b] += gv[b];
      }
#pragma unroll
      for (int j = 0; j < DB * 4; ++j) {
        const float xv = x[(q * 4 + e) * S::kX + j * 16 + l];
#pragma unroll
        for (int b = 0; b < VB; ++b) dw[b][j] = mfma_16x16(gv[b], xv, dw[b][j]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    // dx.
    const float down = scale * (1.0f / 8192.0f);
    const bool all_count = __all(at >= 0); // else rows of zeros, whatever w and the scale hold
    constexpr int kSide = 2; // side by side: one after another would wait for its sum
    f32x4 d[DB * 4] = {};
#pragma unroll
    for (int j0 = 0; j0 < DB * 4; j0 += kSide) {
#pragma unroll
      for (int b = 0; b < S::kV32 / 32; ++b) {
        f16x8 th[kSide], tl[kSide];
#pragma unroll
        for (int j = 0; j < kSide; ++j) {
          const f16_t *const from = wt + ((j0 + j) * 16 + l) * S::kT + b * 32 + q * 8;
          th[j] = *reinterpret_cast<const f16x8 *>(from);
          tl[j] = *reinterpret_cast<const f16x8 *>(from + S::kD * S::kT);
        }
#pragma unroll
        for (int j = 0; j < kSide; ++j) d[j0 + j] = mfma_sixteen(tl[j], gh[b], d[j0 + j]);
#pragma unroll
        for (int j = 0; j < kSide; ++j) d[j0 + j] = mfma_sixteen(th[j], gl[b], d[j0 + j]);
#pragma unroll
        for (int j = 0; j < kSide; ++j) d[j0 + j] = mfma_sixteen(th[j], gh[b], d[j0 + j]);
        __builtin_amdgcn_sched_barrier(0); // the next ones' operands would not fit the registers
      }
    }
    // dx in place of x, and out by whole rows.
    wave_lds_order();
#pragma unroll
    for (int j = 0; j < DB * 4; ++j) {
      const f32x4 u = *reinterpret_cast<const f32x4 *>(t_unit + j * 16 + q * 4);
      d[j] = d[j] * u * down;
      if (!all_count) d[j] = at >= 0 ? d[j] : f32x4{};
      *reinterpret_cast<f32x4 *>(x + l * S::kX + j * 16 + q * 4) = d[j];
    }
    wave_lds_order();
    char *const to = static_cast<char *>(c.dx) + r0 * (c.dx_stride * sizeof(T));
    uint32_t place = q * dx_step + l * static_cast<uint32_t>(4 * sizeof(T));
    asm volatile("" : "+v"(place)); // else eight places are made before the loop, as 64-bit addresses
    const int left = static_cast<int>(min(c.rows - r0, int64_t(16)));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i * 4 + q >= left) continue;
#pragma unroll
      for (int k = 0; k < DB; ++k) {
        const f32x4 f = *reinterpret_cast<const f32x4 *>(x + (i * 4 + q) * S::kX + k * 64 + l * 4);
        const float v[4] = {f[0], f[1], f[2], f[3]};
        if (k < DB - 1 || k * 64 + l * 4 < dim)
          store_f32<4>(reinterpret_cast<T *>(to + (place + i * 4 * dx_step)) + k * 64, v);
      }
    }
  }

  // The waves' sums, one after another.
  float *const join = lds, *const join_db = lds + S::kV * S::kX;
  for (int turn = 0; turn < S::kWaves; ++turn) {
    __syncthreads();
    if (wave != turn) continue;
#pragma unroll
    for (int b = 0; b < VB; ++b) {
#pragma unroll
      for (int j = 0; j < DB * 4; ++j) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float &to = join[(b * 16 + q * 4 + e) * S::kX + j * 16 + l];
          to = (turn ? to : 0.0f) + dw[b][j][e];
        }
      }
      db[b] += lane_xor_f32(db[b], 16);
      db[b] += lane_xor_f32(db[b], 32);
      if (q == 0) join_db[b * 16 + l] = (turn ? join_db[b * 16 + l] : 0.0f) + db[b];
    }
  }
  __syncthreads();
  float *const out = a.dw_part + blockIdx.x * int64_t(S::kV) * (dim16 * 16);
  for (int i = tid; i < S::kV * dim16 * 16; i += kGradThreads)
    out[i] = join[i / (dim16 * 16) * S::kX + i % (dim16 * 16)];
  if (tid < S::kV) a.db_part[blockIdx.x * int64_t(S::kV) + tid] = join_db[tid];
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
int feature_blocks(int64_t dim) {
  for (int b : {1, 2, 3, 4, 6, 8})
    if (dim <= b * 64) return b;
  return 0;
}

// Blocks of classes times blocks of features that kernels are built for: what LDS holds of w
// in 32 bits, or in 16.
constexpr int kMostBlocks = 24, kMostHalves = 48;

// Backward, with tiles shared by the workgroup.
int64_t floats_of(int64_t dim, int blocks) {
  const int64_t stride = few_stride(feature_blocks(dim));
  return (blocks * 16 + 2 * kRows) * stride + kRows * (blocks * 16 + 4) + blocks * 16;
}
int64_t lds_of(int64_t dim, int64_t classes) { return floats_of(dim, class_blocks(classes)) * 4 + 256; }

template <int MOST, typename F> int32_t with_blocks(int64_t dim, int64_t classes, F &&f);

// The LDS of the backward pass that gives each wave tiles of its own, 0 where it doesn't fit.
int64_t wave_lds(int64_t dim, int64_t classes) {
  int64_t bytes = 0;
  if (dim % 4 != 0) return bytes;
  with_blocks<kMostBlocks>(dim, classes, [&](auto vb, auto db) {
    using S = WaveShape<decltype(vb)::value, decltype(db)::value>;
    if constexpr (S::kFits) bytes = S::kFloats * 4;
    return static_cast<int32_t>(SPORDER_OK);
  });
  return bytes;
}

// Whether a call takes that.
template <typename T> bool by_waves(const CeCall &c) {
  constexpr int64_t kFar = int64_t(1) << 24; // sixteen rows apart in 32 bits
  return wave_lds(c.dim, c.classes) && (c.dx_stride % 4 == 0 || c.rows == 1) && aligned_to(c.dx, 4 * sizeof(T)) &&
         c.x_stride < kFar && c.dx_stride < kFar;
}
bool by_waves(const CeCall &c) { return c.type == SPORDER_TYPE_F32 ? by_waves<float>(c) : by_waves<f16_t>(c); }

// Workgroups: as many per CU as fit, up to two.
int64_t grid_of(int64_t rows, int64_t dim, int64_t classes) {
  return std::min(ceil_div64(rows, kRows), 256 * std::min<int64_t>(kLds / lds_of(dim, classes), 2));
}

// f with the class and feature blocks, as types.
template <int MOST, typename F> int32_t with_blocks(int64_t dim, int64_t classes, F &&f) {
  auto classes_of = [&](auto db) {
    constexpr int DB = decltype(db)::value;
    const int b = class_blocks(classes);
    auto at = [&](auto vb) {
      if constexpr (decltype(vb)::value * DB <= MOST)
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
  case 3: return classes_of(std::integral_constant<int, 3>{});
  case 4: return classes_of(std::integral_constant<int, 4>{});
  case 6: return classes_of(std::integral_constant<int, 6>{});
  default: return classes_of(std::integral_constant<int, 8>{});
  }
}

// LDS past 64 KB has to be asked for.
template <typename... P, typename... A>
int32_t launch_lds(void (*kernel)(P...), int64_t grid, int threads, int64_t lds, void *stream, A... args) {
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
        return hipLaunchKernel(reinterpret_cast<const void *>(kernel), dim3(grid), dim3(threads), list,
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
  if (backward) l.grid = grid_of(rows, dim, classes); // at least what either backward pass takes
  const int64_t pad = class_blocks(classes) * 16;
  size_t at = 0;
  auto take = [&](int64_t bytes) {
    const size_t here = at;
    at += Workspace::align(bytes);
    return here;
  };
  if (!backward) {
    l.sums = take(2 * 256 * 16);
  } else {
    l.dw = take(l.grid * pad * ceil_div64(dim, 16) * 16 * 4);
    l.db = take(l.grid * pad * 4);
  }
  l.bytes = at;
  return l;
}

template <typename T> int32_t few_loss(const FewArgs &a, void *stream) {
  int64_t grid = 0;
  constexpr int kMost = sizeof(T) == 2 ? kMostHalves : kMostBlocks;
  const int32_t rc = with_blocks<kMost>(a.c.dim, a.c.classes, [&](auto vb, auto db) {
    constexpr int VB = decltype(vb)::value, DB = decltype(db)::value;
    constexpr int lds = loss_lds<T>(VB, DB);
    static_assert(lds + 256 <= kLds);
    grid = std::min<int64_t>(ceil_div64(a.c.rows, kGradThreads / 4),
                             256 * std::min(kLds / (lds + 256), loss_groups<T>(VB, DB)));
    return launch_lds(few_loss_kernel<T, VB, DB>, grid, kGradThreads, lds, stream, a);
  });
  if (rc != SPORDER_OK || grid == 1) return rc;
  return launch(few_total_kernel, dim3(1), dim3(kLossThreads), stream, a, static_cast<int>(grid));
}

template <typename T> int32_t few_grad(const FewArgs &a, int64_t grid, void *stream) {
  return with_blocks<kMostBlocks>(a.c.dim, a.c.classes, [&](auto vb, auto db) {
    constexpr int VB = decltype(vb)::value, DB = decltype(db)::value;
    using S = WaveShape<VB, DB>;
    if constexpr (S::kFits) {
      if (by_waves(a.c))
        return launch_lds(few_grad_wave_kernel<T, VB, DB>, grid, kGradThreads, S::kFloats * 4, stream, a);
    }
    return launch_lds(few_grad_kernel<T, VB, DB>, grid, kGradThreads, floats_of(a.c.dim, VB) * 4, stream, a);
  });
}

} // namespace

bool few_takes(int type, int64_t dim, int64_t classes, bool backward) {
  const int blocks = class_blocks(classes) * feature_blocks(dim);
  const int most = type != SPORDER_TYPE_F32 && !backward ? kMostHalves : kMostBlocks;
  return dim >= 8 && blocks && blocks <= most && (!backward || lds_of(dim, classes) <= kLds);
}

size_t few_work_bytes(int64_t rows, int64_t dim, int64_t classes, bool backward) {
  return few_layout(rows, dim, classes, backward).bytes;
}

int32_t few_forward(const CeCall &c, void *work, void *stream) {
  const FewLayout l = few_layout(c.rows, c.dim, c.classes, false);
  FewArgs a{c, 0, reinterpret_cast<double *>(static_cast<char *>(work) + l.sums), nullptr,
            nullptr};
  return c.type == SPORDER_TYPE_BF16  ? few_loss<bf16_t>(a, stream)
         : c.type == SPORDER_TYPE_F16 ? few_loss<f16_t>(a, stream)
                                      : few_loss<float>(a, stream);
}

int32_t few_backward(const CeCall &c, void *work, void *stream) {
  const FewLayout l = few_layout(c.rows, c.dim, c.classes, true);
  char *const base = static_cast<char *>(work);
  const int64_t grid = by_waves(c) ? std::min<int64_t>(ceil_div64(c.rows, 16 * 8), 256) : l.grid;
  FewArgs a{c, ceil_div64(c.rows, kRows), nullptr,
            reinterpret_cast<float *>(base + l.dw), reinterpret_cast<float *>(base + l.db)};
  const int32_t rc = c.type == SPORDER_TYPE_BF16  ? few_grad<bf16_t>(a, grid, stream)
                     : c.type == SPORDER_TYPE_F16 ? few_grad<f16_t>(a, grid, stream)
                                                  : few_grad<float>(a, grid, stream);
  if (rc != SPORDER_OK) return rc;
  const int64_t pad = class_blocks(c.classes) * 16, dim_pad = ceil_div64(c.dim, 16) * 16;
  return launch(few_sum_kernel, dim3(ceil_div64(pad * dim_pad + pad, kWave)), dim3(1024), stream, a, grid, pad,
                dim_pad);
}

} // namespace sporder_hip
