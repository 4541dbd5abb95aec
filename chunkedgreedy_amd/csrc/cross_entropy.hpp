// cross_entropy.hpp -- the three forms of the linear cross entropy: tiles of
// 16-bit products over any number of classes (cross_entropy.hip), one pass over
// the rows where the classes' weights fit a workgroup's LDS
// (cross_entropy_few.hip), and 32-bit products straight from memory for a few rows
// (cross_entropy_narrow.hip).
#pragma once

#include "dense.hpp"

namespace sporder_hip {

// What a call passes, for either form.
struct CeCall {
  int64_t rows, dim, classes;
  int64_t x_stride, w_stride; // elements
  const void *x, *w, *bias, *targets;
  int64_t ignore;
  int type, bias_type, target_bits;
  // forward
  float *loss, *lse, *sums;
  // backward
  const float *grad, *given_lse, *given_loss; // the loss may be null
  int64_t grad_stride;
  void *dx, *dw, *db;
  int64_t dx_stride, dw_stride;
  int dw_type;
};

__device__ __forceinline__ int64_t target_of(const CeCall &a, int64_t row) {
  return a.target_bits == 64 ? static_cast<const int64_t *>(a.targets)[row]
                             : static_cast<const int32_t *>(a.targets)[row];
}
__device__ __forceinline__ bool counted(const CeCall &a, int64_t target) {
  return target != a.ignore && target >= 0 && target < a.classes;
}

// A row's target as it lies in memory, loaded some time before it is looked at: without a
// branch (past the rows the last one's), for a branch's end would wait for it and for
// every load before it.
struct RawTarget {
  int32_t low, high;
};
__device__ __forceinline__ RawTarget fetch_target(const CeCall &c, int64_t row) {
  const int words = c.target_bits / 32;
  const int32_t *const p = static_cast<const int32_t *>(c.targets) + min(row, c.rows - 1) * words;
  return {p[0], p[words - 1]};
}

// As a class, -1 where it counts nothing, -2 where it is no class, -3 past the rows.
__device__ __forceinline__ int class_of(const CeCall &c, int64_t row, const RawTarget &raw) {
  const int high = c.target_bits == 64 ? raw.high : raw.low >> 31;
  const bool ignored = raw.low == static_cast<int>(c.ignore) && high == static_cast<int>(c.ignore >> 32);
  const bool in = high == 0 && static_cast<uint32_t>(raw.low) < static_cast<uint32_t>(c.classes);
  const int k = ignored ? -1 : in ? raw.low : -2;
  return row < c.rows ? k : -3;
}

constexpr float kLog2e = 1.44269504088896340736f;
__device__ __forceinline__ float exp_of(float v) { return __builtin_amdgcn_exp2f(v * kLog2e); }

// A row's loss from its largest logit, the sum of exponentials beside it and the target's
// logit.  From lse, where the logit is added to the sum's logarithm, a sure row's loss would
// have half a step of lse's (60 beside a rival 12 below: 6.1e-6 would come out as 7.6e-6).
__device__ __forceinline__ float loss_of(float base, float sum, float hit) {
  return (base - hit) + logf(sum);
}

// Backward, the target's exp(z - lse) - 1 = e^-loss - 1: made of the loss where it is given,
// else 1 (no such value) and the caller makes it of lse, whose half step is all that a sure
// row's has left.
// Below 1/2 by the series of (1 - e^-x) / x to x^8 (what follows is below 2^-30 of it), above
// it nothing cancels.  (The library's expm1f needs more registers than few_grad_kernel has.)
__device__ __forceinline__ float miss_of(const CeCall &c, float loss) {
  float p = 1.0f / 362880.0f;
  p = 1.0f / 40320.0f - loss * p;
  p = 1.0f / 5040.0f - loss * p;
  p = 1.0f / 720.0f - loss * p;
  p = 1.0f / 120.0f - loss * p;
  p = 1.0f / 24.0f - loss * p;
  p = 1.0f / 6.0f - loss * p;
  p = 0.5f - loss * p;
  p = 1.0f - loss * p;
  const float miss = loss < 0.5f ? -loss * p : exp_of(-loss) - 1.0f;
  return c.given_loss ? miss : 1.0f;
}
// exp(z - lse) - [target] of a class.
__device__ __forceinline__ float less_target(float p, bool is_target, float miss) {
  const float t = miss <= 0.0f ? miss : p - 1.0f;
  return is_target ? t : p;
}
// A row's given loss, or something to load in its place: without a branch.
__device__ __forceinline__ float fetch_loss(const CeCall &c, int64_t row) {
  return (c.given_loss ? c.given_loss : c.given_lse)[row];
}

// Sums of two values over a workgroup of WAVES waves, in 64 bits and a fixed order, in its
// first two threads (the first value in thread 0).
template <int WAVES>
__device__ __forceinline__ double block_sums(double s, double n, double (&part)[2][WAVES]) {
#pragma unroll
  for (int j = 1; j < kWave; j <<= 1) {
    s += __shfl_xor(s, j);
    n += __shfl_xor(n, j);
  }
  if (lane_id() == 0) {
    part[0][threadIdx.x / kWave] = s;
    part[1][threadIdx.x / kWave] = n;
  }
  __syncthreads();
  double all = 0.0;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) all += part[threadIdx.x & 1][i];
  return all;
}

using f32x4 = float __attribute__((ext_vector_type(4)));

// Four elements of a row from `col` on, or its last four where it ends before (a row has
// four at least).
template <typename T> __device__ __forceinline__ Words<T, 4> four(const T *row, int col, int dim) {
  return __builtin_bit_cast(Words<T, 4>, *reinterpret_cast<const LoosePack<T, 4> *>(row + min(col, dim - 4)));
}

// As floats, zeros past the row's end.
template <typename T> __device__ __forceinline__ f32x4 floats(const Words<T, 4> &words, int col, int dim) {
  const auto q = __builtin_bit_cast(Pack<T, 4>, words);
  f32x4 v;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = static_cast<float>(q.v[e]);
  if (dim % 4 != 0) { // move the row's last elements to their places
    const int past = col + 4 - dim;
    if (past > 0)
      v = past == 1   ? f32x4{v[1], v[2], v[3], 0.0f}
          : past == 2 ? f32x4{v[2], v[3], 0.0f, 0.0f}
          : past == 3 ? f32x4{v[3], 0.0f, 0.0f, 0.0f}
                      : f32x4{};
  } else if (col >= dim) {
    v = f32x4{};
  }
  return v;
}

// The one-pass form.
bool few_takes(int type, int64_t dim, int64_t classes, bool backward);
size_t few_work_bytes(int64_t rows, int64_t dim, int64_t classes, bool backward);
int32_t few_forward(const CeCall &a, void *work, void *stream);
int32_t few_backward(const CeCall &a, void *work, void *stream);

// The form of few rows.
bool narrow_takes(int type, int64_t rows, int64_t dim, int64_t classes, bool backward);
size_t narrow_work_bytes(int64_t rows, int64_t dim, int64_t classes, bool backward);
int32_t narrow_run(const CeCall &a, bool backward, void *work, void *stream);

} // namespace sporder_hip
