// mfma_product.hpp -- C = A B^T of 16-bit operands whose rows lie along the sum,
// a tile of C per workgroup, left in the accumulators for the caller's epilogue.
//
// An operand row is cut into stages of 64 elements (128 bytes).  Both operands'
// rows of a stage go straight from memory to LDS (no registers between), one
// stage ahead of the products; a wave fetches eight rows an access.  LDS keeps
// a row's eight 16-byte parts in the order part ^ (row % 8), so that the eight
// rows that a matrix instruction's lanes read side by side lie in eight
// different bank groups.
//
// Operands of 32-bit values are two planes of 16-bit halves, x = hi + lo of 22
// bits; the product is hi hi + hi lo + lo hi, each a pass of the same loop.
#pragma once

#include "dense.hpp"

namespace sporder_hip {

using f32x16 = float __attribute__((ext_vector_type(16)));
using bf16x8 = bf16_t __attribute__((ext_vector_type(8)));
using f16x8 = f16_t __attribute__((ext_vector_type(8)));

constexpr int kStageBytes = 128; // of an operand row
constexpr int kStageK = 64;

__device__ __forceinline__ f32x16 mfma_32x32(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma_32x32(f16x8 a, f16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// Row of a 32 x 32 result that a lane's register r holds; its column is lane % 32.
__device__ __forceinline__ int result_row(int r) { return 8 * (r / 4) + 4 * (lane_id() / 32) + r % 4; }

__device__ __forceinline__ uint32_t lds_address(const void *p) {
  return static_cast<uint32_t>(
      reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) void *)p));
}

// 16 bytes per lane from base + offset to LDS, lane after lane from `lds` on.
// The caller waits (vmcnt) before a barrier that comes before any read of them.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm" // M0 is named for the reader
__device__ __forceinline__ void fetch_to_lds(const char *base, uint32_t offset, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               :
               : "s"(lds), "v"(offset), "s"(base)
               : "m0");
}
#pragma clang diagnostic pop

// Everything fetched has arrived, and every wave is done with what it read.
__device__ __forceinline__ void stage_barrier() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// WM x WN waves of MB x NB blocks of 32 x 32 each.
template <int WM_, int WN_, int MB_, int NB_> struct TileShape {
  static constexpr int WM = WM_, WN = WN_, MB = MB_, NB = NB_;
  static constexpr int kM = WM * MB * 32, kN = WN * NB * 32;
  static constexpr int kWaves = WM * WN, kThreads = kWaves * kWave;
  static constexpr int kFetchA = kM / 8 / kWaves, kFetchB = kN / 8 / kWaves; // of a wave, a stage
  static constexpr int kStage = (kM + kN) * kStageBytes;
  static_assert(kFetchA * kWaves * 8 == kM && kFetchB * kWaves * 8 == kN);
};

// Byte offsets of the parts that this lane fetches, from each fetched row's.
template <int WAVES, int COUNT, typename F>
__device__ __forceinline__ void fetch_offsets(int wave, uint32_t (&out)[COUNT], F &&row_offset) {
  const int lane = lane_id();
#pragma unroll
  for (int i = 0; i < COUNT; ++i)
    out[i] = row_offset((wave * COUNT + i) * 8 + lane / 8) + (lane % 8 ^ lane / 8) * 16;
}

template <typename U> struct HalfVector;
template <> struct HalfVector<bf16_t> { using type = bf16x8; };
template <> struct HalfVector<f16_t> { using type = f16x8; };

// acc += A B^T over `stages` stages (of each plane).  `lds` holds two stages.
// Ends with a barrier: the caller may use LDS again.
template <typename U, int PLANES, typename S>
__device__ __forceinline__ void tile_product(char *lds, int wave, const char *a, int64_t a_plane,
                                             const uint32_t (&a_off)[S::kFetchA], const char *b,
                                             int64_t b_plane, const uint32_t (&b_off)[S::kFetchB],
                                             int stages, f32x16 (&acc)[S::MB][S::NB]) {
  using Vec = typename HalfVector<U>::type;
  const int lane = lane_id();
  const uint32_t to = lds_address(lds);
  const int wm = wave / S::WN, wn = wave % S::WN;
  const int total = PLANES == 2 ? 3 * stages : stages;
  auto issue = [&](int s) {
    const char *pa = a, *pb = b;
    if constexpr (PLANES == 2) { // hi hi, hi lo, lo hi
      const int part = s % 3;
      pa += (s / 3) * kStageBytes + (part == 2 ? a_plane : 0);
      pb += (s / 3) * kStageBytes + (part == 1 ? b_plane : 0);
    } else {
      pa += int64_t(s) * kStageBytes;
      pb += int64_t(s) * kStageBytes;
    }
    const uint32_t half = to + (s & 1) * S::kStage;
#pragma unroll
    for (int i = 0; i < S::kFetchA; ++i)
      fetch_to_lds(pa, a_off[i], half + (wave * S::kFetchA + i) * 1024);
#pragma unroll
    for (int i = 0; i < S::kFetchB; ++i)
      fetch_to_lds(pb, b_off[i], half + S::kM * kStageBytes + (wave * S::kFetchB + i) * 1024);
  };
  if (total > 0) issue(0);
  for (int s = 0; s < total; ++s) {
    stage_barrier();
    if (s + 1 < total) issue(s + 1);
    const char *const pa = lds + (s & 1) * S::kStage + wm * S::MB * 32 * kStageBytes;
    const char *const pb = lds + (s & 1) * S::kStage + (S::kM + wn * S::NB * 32) * kStageBytes;
#pragma unroll
    for (int k = 0; k < kStageK / 16; ++k) {
      const int at = lane % 32 * kStageBytes + ((2 * k + lane / 32) ^ lane % 8) * 16;
      Vec va[S::MB], vb[S::NB];
#pragma unroll
      for (int j = 0; j < S::NB; ++j)
        vb[j] = *reinterpret_cast<const Vec *>(pb + j * 32 * kStageBytes + at);
#pragma unroll
      for (int i = 0; i < S::MB; ++i)
        va[i] = *reinterpret_cast<const Vec *>(pa + i * 32 * kStageBytes + at);
#pragma unroll
      for (int i = 0; i < S::MB; ++i) {
#pragma unroll
        for (int j = 0; j < S::NB; ++j) acc[i][j] = mfma_32x32(va[i], vb[j], acc[i][j]);
      }
    }
  }
  stage_barrier();
}

// The same for short sums: LDS as a ring of four slots of 32 elements, three of them on
// their way or read from, so that a sum begins with three fetches in flight and its
// matrix instructions go on over the barriers: the first half of a slot's operands is
// read before the barrier that ends the slot before.  2,048 elements of 256 x 256 tiles:
// 1.09 PFLOP/s, 0.98 with two stages; 7,424 elements 0.92, 0.95 with two stages.
template <typename U, int PLANES, typename S>
__device__ __forceinline__ void ring_product(char *lds, int wave, const char *a, int64_t a_plane,
                                             const uint32_t (&a_off)[S::kM / 16 / S::kWaves], const char *b,
                                             int64_t b_plane, const uint32_t (&b_off)[S::kN / 16 / S::kWaves],
                                             int stages, f32x16 (&acc)[S::MB][S::NB]) {
  using Vec = typename HalfVector<U>::type;
  constexpr int kFetchA = S::kM / 16 / S::kWaves, kFetchB = S::kN / 16 / S::kWaves; // 16 rows each
  constexpr int kRing = 4, kHalf = kStageBytes / 2, kSlot = (S::kM + S::kN) * kHalf;
  static_assert(kFetchA + kFetchB == 4); // the waits below leave the last two slots' fetches
  const int lane = lane_id(), wm = wave / S::WN, wn = wave % S::WN, row = lane % 32;
  const uint32_t to = lds_address(lds);
  const int slots = 2 * (PLANES == 2 ? 3 * stages : stages);
  auto issue = [&](int s, int slot) {
    int64_t at = int64_t(s) * kHalf;
    const char *pa = a, *pb = b;
    if constexpr (PLANES == 2) { // hi hi, hi lo, lo hi
      const int part = s % 3;
      at = int64_t(s / 3) * kHalf;
      pa += part == 2 ? a_plane : 0;
      pb += part == 1 ? b_plane : 0;
    }
    const uint32_t base = to + slot * kSlot;
#pragma unroll
    for (int i = 0; i < kFetchA; ++i) fetch_to_lds(pa + at, a_off[i], base + (wave * kFetchA + i) * 1024);
#pragma unroll
    for (int i = 0; i < kFetchB; ++i)
      fetch_to_lds(pb + at, b_off[i], base + S::kM * kHalf + (wave * kFetchB + i) * 1024);
  };
  Vec va[2][S::MB], vb[2][S::NB];
  auto load = [&](int slot, int k) {
    const char *const p = lds + slot * kSlot + row * kHalf + ((2 * k + lane / 32) ^ (row / 2 % 4)) * 16;
#pragma unroll
    for (int j = 0; j < S::NB; ++j)
      vb[k][j] = *reinterpret_cast<const Vec *>(p + (S::kM + (wn * S::NB + j) * 32) * kHalf);
#pragma unroll
    for (int i = 0; i < S::MB; ++i)
      va[k][i] = *reinterpret_cast<const Vec *>(p + (wm * S::MB + i) * 32 * kHalf);
  };
  auto multiply = [&](int k) {
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int i = 0; i < S::MB; ++i) {
#pragma unroll
      for (int j = 0; j < S::NB; ++j) acc[i][j] = mfma_32x32(va[k][i], vb[k][j], acc[i][j]);
    }
    __builtin_amdgcn_s_setprio(0);
  };
  // The slot after the one in use has arrived for every wave, and every wave's reads
  // of the one before are done.
  auto next_slot = [&] {
    asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
#pragma unroll
  for (int s = 0; s < kRing - 1; ++s) issue(min(s, slots - 1), s);
  next_slot();
  load(0, 0);
  for (int s = 0; s < slots; ++s) {
    issue(min(s + kRing - 1, slots - 1), (s + kRing - 1) % kRing); // past the end the last one again
    load(s % kRing, 1);
    multiply(0);
    next_slot();
    load((s + 1) % kRing, 0);
    multiply(1);
  }
  stage_barrier();
}

// Offsets for ring_product: sixteen rows an access, a row's four parts in the order
// part ^ (row / 2 % 4).
template <int COUNT, typename F>
__device__ __forceinline__ void ring_offsets(int wave, uint32_t (&out)[COUNT], F &&row_offset) {
  const int lane = lane_id();
#pragma unroll
  for (int i = 0; i < COUNT; ++i)
    out[i] = row_offset((wave * COUNT + i) * 16 + lane / 4) + (lane % 4 ^ lane / 8 % 4) * 16;
}

// Tile t of `down` x `across`, `group` rows of tiles at a time and down each
// column of them, so that neighbouring tiles share operands on both sides.
__device__ __forceinline__ void place_tile(int64_t t, int64_t down, int64_t across, int group,
                                           int64_t &ti, int64_t &tj) {
  const int64_t g = t / (group * across), first = g * group;
  const int64_t rows = min(int64_t(group), down - first), left = t - g * group * across;
  ti = first + left % rows;
  tj = left / rows;
}

// The unit of a row of 32-bit values at most `bound` in magnitude, a power of
// two with 2^14 <= bound / unit < 2^15 (2^-114 at least), and its inverse.
__device__ __forceinline__ float unit_of(float bound) {
  return __builtin_bit_cast(float, (max(__builtin_bit_cast(uint32_t, bound) >> 23, 27u) - 14) << 23);
}
__device__ __forceinline__ float unit_inverse(float u) {
  return __builtin_bit_cast(float, (254u << 23) - __builtin_bit_cast(uint32_t, u));
}

} // namespace sporder_hip
