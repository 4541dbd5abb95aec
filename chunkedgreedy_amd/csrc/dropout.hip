// dropout.hip -- dropout from a counter, its mask never stored.
//
//   out_i = residual_i + (u_i >= t ? x_i / (1 - p) : 0),   t = round(p 2^32)
//
// u_i are the 32 random bits of element i (counted along the rows), so the
// gradient is the same call on the gradient: the mask is made again.  A
// Philox4x32-10 block gives 8 elements 16 bits each: element i has half i % 2
// of word (i % 8) / 2 of the block with counter (i / 8, offset) under the key
// `seed`, as the high half of u_i.  Its low half is the same half of the block
// with counter (i / 8, offset + 2^63), which matters only where the high half
// equals t's: a wave makes that block where one of its elements ties (512 in
// 65,536), so p keeps 32 bits at the price of 16.
//
// Bound by memory: 2,449,029 x 128 floats in 427 us (5.9 TB/s), 16,384 x 4,096 bfloat16
// with a residual in 71 us (5.7 TB/s).
#include <algorithm>
#include <cmath>

#include "dense.hpp"
#include "philox.hpp"

namespace sporder_hip {

namespace {

struct DropoutArgs {
  int64_t rows, dim, x_stride, r_stride, out_stride;
  const void *x, *residual;
  void *out;
  uint64_t seed, offset;
  const uint64_t *state; // more seed and offset, or null
  uint32_t high, low;    // of t; 65536 and 0 where nothing is kept
  float scale;
  bool stream;
};

struct Key {
  uint2 seed, offset;
};

__device__ __forceinline__ Key dropout_key(const DropoutArgs &a) {
  uint64_t seed = a.seed, offset = a.offset;
  if (a.state) {
    seed += a.state[0];
    offset += a.state[1];
  }
  offset &= ~uint64_t(0) >> 1;
  return {make_uint2(static_cast<uint32_t>(seed), static_cast<uint32_t>(seed >> 32)),
          make_uint2(static_cast<uint32_t>(offset), static_cast<uint32_t>(offset >> 32))};
}

// Bit e: whether element e of a block of 8 is kept.
__device__ __forceinline__ uint32_t keep_bits(const DropoutArgs &a, const Key &k, uint64_t block) {
  const uint32_t b0 = static_cast<uint32_t>(block), b1 = static_cast<uint32_t>(block >> 32);
  const uint4 r = philox4x32_10(make_uint4(b0, b1, k.offset.x, k.offset.y), k.seed);
  const uint32_t word[4] = {r.x, r.y, r.z, r.w};
  uint32_t above = 0, tie = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t half = e & 1 ? word[e / 2] >> 16 : word[e / 2] & 0xFFFFu;
    above |= half > a.high ? 1u << e : 0u;
    tie |= half == a.high ? 1u << e : 0u;
  }
  if (a.low == 0) return above | tie;
  if (tie) {
    const uint4 s = philox4x32_10(make_uint4(b0, b1, k.offset.x, k.offset.y | 1u << 31), k.seed);
    const uint32_t low[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t half = e & 1 ? low[e / 2] >> 16 : low[e / 2] & 0xFFFFu;
      if (half >= a.low) above |= tie & 1u << e;
    }
  }
  return above;
}

// Rows without gaps are one row of n elements.  A lane makes the bits of one
// block and takes accesses of 16 bytes side by side with its neighbours': of 16
// bits an element they are the lane's own block, of 32 bits half of another
// lane's, whose bits it fetches.
template <typename T, bool LOOSE, int ITEMS>
__global__ void __launch_bounds__(256) dropout_flat_kernel(DropoutArgs a, int64_t n) {
  constexpr int kVec = 16 / sizeof(T), kParts = 8 / kVec;
  const Key key = dropout_key(a);
  const int lane = lane_id();
  const T *const x = static_cast<const T *>(a.x), *const res = static_cast<const T *>(a.residual);
  T *const out = static_cast<T *>(a.out);
  constexpr int kTurn = ITEMS * kWave; // blocks of 8 elements of a wave
  for (int64_t first = (blockIdx.x * int64_t(256 / kWave) + threadIdx.x / kWave) * kTurn;
       first * 8 < n; first += gridDim.x * int64_t(256 / kWave) * kTurn) {
    Pack<T, kVec> v[ITEMS][kParts], r[ITEMS][kParts];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
#pragma unroll
      for (int p = 0; p < kParts; ++p) {
        const int64_t at = (first + i * kWave) * 8 + (p * kWave + lane) * kVec;
        if (at < n) {
          v[i][p] = fetch<LOOSE, kVec>(x + at, n - at);
          if (res) r[i][p] = fetch<LOOSE, kVec>(res + at, n - at);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const uint32_t mine = keep_bits(a, key, first + i * kWave + lane);
#pragma unroll
      for (int p = 0; p < kParts; ++p) {
        uint32_t bits = mine;
        if constexpr (kParts > 1) {
          static_assert(kParts == 2);
          bits = __shfl(mine, p * (kWave / 2) + lane / 2) >> lane % 2 * kVec;
        }
        const int64_t at = (first + i * kWave) * 8 + (p * kWave + lane) * kVec;
        if (at >= n) continue;
        float o[kVec];
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          o[e] = bits >> e & 1 ? static_cast<float>(v[i][p].v[e]) * a.scale : 0.0f;
          if (res) o[e] += static_cast<float>(r[i][p].v[e]);
        }
        if constexpr (LOOSE)
          put<true, kVec>(out + at, n - at, o);
        else
          put_f32<kVec>(a.stream, out + at, o);
      }
    }
  }
}

// Rows with gaps: a block of 8 elements per lane, by one access where they lie
// in one row (1,000,003 rows of 128 floats 5.2 TB/s; of 99, where blocks end inside rows, 3.4 to
// 3.7; bfloat16 4.5 and 2.6).  Rows of 128 bfloat16 are bound by the generator (the vector units are
// busy 90 % of the time, of 99 73 %), rows of 99 floats by the address units (81 %).
template <typename T> __global__ void __launch_bounds__(256) dropout_rows_kernel(DropoutArgs a) {
  const Key key = dropout_key(a);
  const int64_t n = a.rows * a.dim;
  for (int64_t block = blockIdx.x * int64_t(256) + threadIdx.x; block * 8 < n;
       block += gridDim.x * int64_t(256)) {
    const uint32_t bits = keep_bits(a, key, block);
    int64_t row = block * 8 / a.dim, col = block * 8 - row * a.dim;
    const int64_t left = min(n - block * 8, int64_t(8));
    const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
    const T *res = static_cast<const T *>(a.residual) + (a.residual ? row * a.r_stride : 0);
    T *out = static_cast<T *>(a.out) + row * a.out_stride;
    if (col + 8 <= a.dim) {
      const Pack<T, 8> v = fetch<true, 8>(x + col, 8);
      float o[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = bits >> e & 1 ? static_cast<float>(v.v[e]) * a.scale : 0.0f;
      if (a.residual) {
        const Pack<T, 8> r = fetch<true, 8>(res + col, 8);
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] += static_cast<float>(r.v[e]);
      }
      put<true, 8>(out + col, 8, o);
      continue;
    }
    for (int e = 0; e < left; ++e) {
      float o = bits >> e & 1 ? static_cast<float>(x[col]) * a.scale : 0.0f;
      if (a.residual) o += static_cast<float>(res[col]);
      out[col] = static_cast<T>(o);
      if (++col == a.dim) {
        col = 0;
        x += a.x_stride;
        res += a.residual ? a.r_stride : 0;
        out += a.out_stride;
      }
    }
  }
}

constexpr int64_t kMostElements = int64_t(1) << 60;
constexpr int64_t kMostGroups = int64_t(1) << 22;
constexpr int64_t kManyBlocks = 1 << 20; // blocks of 8 from which a lane takes several

template <typename T> int32_t dropout_typed(DropoutArgs a, void *stream) {
  const int64_t n = a.rows * a.dim, blocks = ceil_div64(n, 8);
  const bool flat = a.rows == 1 || (a.x_stride == a.dim && a.out_stride == a.dim &&
                                    (!a.residual || a.r_stride == a.dim));
  if (!flat)
    return launch(dropout_rows_kernel<T>, dim3(std::min(ceil_div64(blocks, 256), kMostGroups)), dim3(256),
                  stream, a);
  a.stream = n * static_cast<int64_t>(sizeof(T)) >= kStreamBytes;
  const bool loose = n % 8 != 0 || !aligned_to(a.x, 16) || !aligned_to(a.out, 16) ||
                     !aligned_to(a.residual, 16);
  auto go = [&](auto kernel, int items) {
    return launch(kernel, dim3(std::min(ceil_div64(blocks, 256 * items), kMostGroups)), dim3(256),
                  stream, a, n);
  };
  if (blocks < kManyBlocks)
    return loose ? go(dropout_flat_kernel<T, true, 1>, 1) : go(dropout_flat_kernel<T, false, 1>, 1);
  return loose ? go(dropout_flat_kernel<T, true, 2>, 2) : go(dropout_flat_kernel<T, false, 2>, 2);
}

} // namespace

} // namespace sporder_hip

using namespace sporder_hip;

extern "C" {

int32_t sporder_dropout(void *stream, int32_t type, int64_t rows, int64_t dim, int64_t x_stride,
                        const void *d_x, int64_t residual_stride, const void *d_residual, double p,
                        uint64_t seed, uint64_t offset, const uint64_t *d_state, int64_t out_stride,
                        void *d_out) {
  if (!type_known(type) || rows < 0 || dim < 1 || rows > kMostElements / dim || x_stride < 0 ||
      residual_stride < 0 || out_stride < 0 || (rows > 1 && out_stride < dim) || !(p >= 0.0) ||
      !(p <= 1.0) || offset >> 63)
    return SPORDER_BAD_ARGUMENT;
  if (rows == 0) return SPORDER_OK;
  if (!d_x || !d_out || !aligned_to(d_state, 8)) return SPORDER_BAD_ARGUMENT;
  const double t = std::nearbyint(p * 4294967296.0);
  const uint64_t bits = static_cast<uint64_t>(t);
  const DropoutArgs a{rows,
                      dim,
                      x_stride,
                      residual_stride,
                      out_stride,
                      d_x,
                      d_residual,
                      d_out,
                      seed,
                      offset,
                      d_state,
                      static_cast<uint32_t>(bits >> 16),
                      static_cast<uint32_t>(bits & 0xFFFFu),
                      p < 1.0 ? static_cast<float>(1.0 / (1.0 - p)) : 0.0f,
                      false};
  if (type == SPORDER_TYPE_BF16) return dropout_typed<bf16_t>(a, stream);
  if (type == SPORDER_TYPE_F16) return dropout_typed<f16_t>(a, stream);
  return dropout_typed<float>(a, stream);
}

} // extern "C"
