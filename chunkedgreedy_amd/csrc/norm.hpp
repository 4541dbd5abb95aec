// norm.hpp -- pieces shared by the norms (layer_norm.hip, residual_norm.hip),
// whose rows are held in the registers of L lanes: sums over those lanes, and a
// lane's part of a vector of weights.
#pragma once

#include "dense.hpp"

namespace sporder_hip {

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

// A lane's part of a vector of weights, or `value` where there is none.
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

template <int N> using Const = std::integral_constant<int, N>;

} // namespace sporder_hip
