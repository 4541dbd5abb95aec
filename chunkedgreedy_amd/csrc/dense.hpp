// dense.hpp -- pieces shared by the training operators (layer_norm.hip,
// embedding.hip, newton_schulz.hip, dropout.hip, residual_norm.hip,
// cross_entropy*.hip): element types, vector access, sums over
// lane groups and the status codes of their C entries.
//
// These entries differ from the rest of the library: they run on the caller's
// stream, return before the work is done, take their scratch from the caller
// and report errors by a return code, because a training step makes them
// many times between two products and reads their results on the same stream.
#pragma once

#include <initializer_list>
#include <tuple>
#include <type_traits>

#include "common.hpp"

namespace sporder_hip {

using bf16_t = __bf16;
using f16_t = _Float16;

template <typename T, int VEC> struct alignas(sizeof(T) * VEC < 16 ? sizeof(T) * VEC : 16) Pack {
  T v[VEC];
};

template <int VEC, typename T>
__device__ __forceinline__ void load_f32(const T *p, float (&out)[VEC]) {
  const Pack<T, VEC> q = *reinterpret_cast<const Pack<T, VEC> *>(p);
#pragma unroll
  for (int i = 0; i < VEC; ++i) out[i] = static_cast<float>(q.v[i]);
}

template <int VEC, typename T>
__device__ __forceinline__ void store_f32(T *p, const float (&in)[VEC]) {
  Pack<T, VEC> q;
#pragma unroll
  for (int i = 0; i < VEC; ++i) q.v[i] = static_cast<T>(in[i]);
  *reinterpret_cast<Pack<T, VEC> *>(p) = q;
}

// The same for rows of any length and alignment: whole vectors at an address
// aligned to elements only (the memory pipe takes them), and the end of the
// row, whose length from p on is `left`, by elements.
template <typename T, int VEC> struct __attribute__((packed, aligned(sizeof(T)))) LoosePack {
  T v[VEC];
};

template <bool LOOSE, int VEC, typename T>
__device__ __forceinline__ Pack<T, VEC> fetch(const T *p, int64_t left) {
  Pack<T, VEC> q;
  if constexpr (!LOOSE) {
    q = *reinterpret_cast<const Pack<T, VEC> *>(p);
  } else if (left >= VEC) {
    const LoosePack<T, VEC> r = *reinterpret_cast<const LoosePack<T, VEC> *>(p);
#pragma unroll
    for (int i = 0; i < VEC; ++i) q.v[i] = r.v[i];
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) q.v[i] = i < left ? p[i] : static_cast<T>(0.0f);
  }
  return q;
}

// A row's VEC elements from `col` on in two halves, for rows of which many
// accesses are to be on their way at once: the words, then the elements, zeros
// past the row's end and where the row is not `live`.  Elements converted
// between accesses would make each wait for the one before.  A loose row that
// holds a vector can be read by vectors alone (CLAMP), the last one ending with
// the row and moved into place afterwards: `row` is then a row's address whether
// it is live or not.
template <typename T, int VEC> struct Words {
  uint32_t v[VEC * sizeof(T) / 4];
};

template <bool LOOSE, bool CLAMP, int VEC, typename T>
__device__ __forceinline__ Words<T, VEC> fetch_words(const T *row, int col, int64_t dim, bool live) {
  if constexpr (CLAMP) {
    if (dim >= VEC)
      return __builtin_bit_cast(Words<T, VEC>,
                                *reinterpret_cast<const LoosePack<T, VEC> *>(
                                    row + min(col, static_cast<int>(dim) - VEC)));
  }
  return live && col < dim ? __builtin_bit_cast(Words<T, VEC>, fetch<LOOSE, VEC>(row + col, dim - col))
                           : Words<T, VEC>{};
}

template <bool CLAMP, int VEC, typename T>
__device__ __forceinline__ Pack<T, VEC> elements(Words<T, VEC> w, int col, int64_t dim, bool live) {
  if constexpr (CLAMP) {
    using Bits = std::conditional_t<sizeof(w) == 16, unsigned __int128, uint64_t>;
    const int past = live ? col + VEC - static_cast<int>(dim) : VEC;
    if (dim >= VEC && past > 0)
      w = past < VEC ? __builtin_bit_cast(Words<T, VEC>, __builtin_bit_cast(Bits, w) >> past * 8 * sizeof(T))
                     : Words<T, VEC>{};
  }
  return __builtin_bit_cast(Pack<T, VEC>, w);
}

template <bool LOOSE, int VEC, typename T>
__device__ __forceinline__ void put(T *p, int64_t left, const float (&in)[VEC]) {
  if constexpr (!LOOSE) {
    store_f32<VEC>(p, in);
  } else if (left >= VEC) {
    LoosePack<T, VEC> q;
#pragma unroll
    for (int i = 0; i < VEC; ++i) q.v[i] = static_cast<T>(in[i]);
    *reinterpret_cast<LoosePack<T, VEC> *>(p) = q;
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (i < left) p[i] = static_cast<T>(in[i]);
  }
}

// The same past the caches, for output too large to be found there by its
// reader: it leaves them to what the kernel still reads.
template <int VEC, typename T>
__device__ __forceinline__ void stream_f32(T *p, const float (&in)[VEC]) {
  using words = uint32_t __attribute__((ext_vector_type(4)));
  Pack<T, VEC> q;
#pragma unroll
  for (int i = 0; i < VEC; ++i) q.v[i] = static_cast<T>(in[i]);
  if constexpr (sizeof(q) % 16 == 0) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(q) / 16); ++i)
      __builtin_nontemporal_store(reinterpret_cast<const words *>(&q)[i],
                                  reinterpret_cast<words *>(p) + i);
  } else if constexpr (sizeof(q) == 8) {
    __builtin_nontemporal_store(__builtin_bit_cast(uint64_t, q), reinterpret_cast<uint64_t *>(p));
  } else {
    static_assert(VEC == 1);
    __builtin_nontemporal_store(q.v[0], p);
  }
}

// Output from which on stores go past the caches (the last level holds 256 MB,
// and what was read is in it too).
constexpr int64_t kStreamBytes = int64_t(64) << 20;

template <int VEC, typename T>
__device__ __forceinline__ void put_f32(bool stream, T *p, const float (&in)[VEC]) {
  if (stream)
    stream_f32<VEC>(p, in);
  else
    store_f32<VEC>(p, in);
}

// Calls f with a pointer of the type known at run time.  The branch goes
// around whole loops: one around each access would make them wait for one
// another.
template <typename F> __device__ __forceinline__ void with_type(const void *p, int type, F &&f) {
  if (type == SPORDER_TYPE_BF16)
    f(static_cast<const bf16_t *>(p));
  else if (type == SPORDER_TYPE_F16)
    f(static_cast<const f16_t *>(p));
  else
    f(static_cast<const float *>(p));
}
__device__ __forceinline__ void store_typed(void *p, int type, int64_t i, float v) {
  if (type == SPORDER_TYPE_BF16)
    static_cast<bf16_t *>(p)[i] = static_cast<bf16_t>(v);
  else if (type == SPORDER_TYPE_F16)
    static_cast<f16_t *>(p)[i] = static_cast<f16_t>(v);
  else
    static_cast<float *>(p)[i] = v;
}

// Sum over aligned groups of L lanes (a power of two up to 64), in every lane.
template <int L> __device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int j = 1; j < L; j <<= 1) v += lane_xor_f32(v, j);
  return v;
}

// The largest of theirs (of NaN and a number, the number).
template <int L> __device__ __forceinline__ float group_max(float v) {
#pragma unroll
  for (int j = 1; j < L; j <<= 1) v = fmaxf(v, lane_xor_f32(v, j));
  return v;
}

constexpr bool type_known(int32_t t) { return t >= SPORDER_TYPE_F32 && t <= SPORDER_TYPE_F16; }
constexpr int type_bytes(int32_t t) { return t == SPORDER_TYPE_F32 ? 4 : 2; }

// Queues a kernel and tells its own status: hipGetLastError would also report
// an error that some earlier call of the caller's left behind.
template <typename... P, typename... A>
inline int32_t launch(void (*kernel)(P...), dim3 grid, dim3 block, void *stream, A... args) {
  std::tuple<P...> held(static_cast<P>(args)...);
  const hipError_t err = std::apply(
      [&](P &...a) {
        void *list[] = {static_cast<void *>(&a)...};
        return hipLaunchKernel(reinterpret_cast<const void *>(kernel), grid, block, list, 0,
                               static_cast<hipStream_t>(stream));
      },
      held);
  if (err == hipSuccess) return SPORDER_OK;
  (void)hipGetLastError(); // reported here, so not left for the caller's next check
  return SPORDER_LAUNCH_FAILED;
}

inline bool aligned_to(const void *p, size_t bytes) {
  return reinterpret_cast<uintptr_t>(p) % bytes == 0;
}

constexpr int64_t kMostDim = int64_t(1) << 23; // elements of a row

// Elements per access of rows of `bytes_each` bytes an element: 16 bytes, or 4
// elements, where the length, the strides and the bases (16-byte aligned)
// allow it, else one element.
inline int row_vec(int bytes_each, int64_t dim, std::initializer_list<int64_t> strides,
                   std::initializer_list<const void *> bases) {
  for (int vec : {16 / bytes_each, 4}) {
    bool ok = dim % vec == 0;
    for (int64_t s : strides) ok = ok && s % vec == 0;
    for (const void *p : bases) ok = ok && aligned_to(p, 16);
    if (ok) return vec;
  }
  return 1;
}

} // namespace sporder_hip
