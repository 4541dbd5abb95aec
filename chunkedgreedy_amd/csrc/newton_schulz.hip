// newton_schulz.hip -- orthogonalising a matrix by Newton-Schulz products.
//
//   X = G / (|G|_F + eps),  then `steps` times:
//   A = X X^T,  B = b A + c A A,  X <- a X + B X        (m <= n; else of G^T)
//
// Each singular value s of G / |G| becomes p(p(...p(s))), p(s) = a s + b s^3 +
// c s^5, and the singular vectors stay.
//
// Products.  The matrix units multiply 32-bit floats at a sixteenth of the rate of
// 16-bit ones, so every operand x is kept as two 16-bit halves of x 2^11:
// hi = fl16(x 2^11) and lo = fl16(x 2^11 - hi), together 22 bits and a sign,
// and a product is hi hi + hi lo + lo hi with 32-bit accumulation: three
// matrix products, and lo lo (2^-22 of the result) left out.  All values are
// at most 31 in magnitude (singular values start at most 1 and the entry
// refuses coefficients that take X's, A's or B's past 31), so hi does not
// overflow, and lo keeps absolute steps of 2^-35 where the largest singular
// value starts at most 1.
//
// Layout.  Operands are stored as the matrix units read them: blocks of 32
// rows by 16 columns, each 64 lanes of 8 halves (lane l holds row l % 32,
// columns 8 (l / 32) to + 7), hi block then lo block.  A tile's blocks are
// then contiguous in memory and in LDS, and every access is 16 bytes per
// lane in lane order.  All products are rows times rows (P Q^T), X is kept in
// both orders, and A and B are symmetric: their tiles on and above the diagonal
// are computed and written twice.  Rows and columns are padded with zeros,
// which stay zero.
#include <algorithm>
#include <cmath>

#include "dense.hpp"

namespace sporder_hip {

namespace {

using f16x8 = f16_t __attribute__((ext_vector_type(8)));
using f32x16 = float __attribute__((ext_vector_type(16)));

constexpr float kScale = 2048.0f; // of the stored halves
constexpr double kMostValue = 31.0;
constexpr int kBlock = 256;
constexpr int kPad = 128; // rows and columns are padded to multiples of it
constexpr int kStageRow = 36; // words per row of a wave's transposing buffer

struct OrthoArgs {
  const void *g;
  void *out;
  int64_t batch, m, n;          // of X: m <= n
  int64_t g_batch, g_stride;    // of g, in elements
  int mp, np;                   // padded
  int tall;                     // X = G^T
  int type;
  double eps;
  float a, b, c;
  double *partial;              // [batch][kNormBlocks]
  uint4 *x, *xt, *xt_next, *gram, *poly; // packed operands, one after another per matrix
};

// uint4 units of a packed operand of `rows` by `cols` (both padded).
__host__ __device__ constexpr int64_t packed_units(int64_t rows, int64_t cols) {
  return rows * cols / 4; // two halves of 2 bytes each: 4 bytes per element
}

// One wave's 32 x 32 block with row i0 and column j0: lane l holds column
// l % 32, rows 8 q + 4 (l / 32) + e in v[4 q + e], scaled.
// by_col receives the block with columns as operand rows, by_row (if not
// null) with its own; k_col and k_row are their numbers of 16-column blocks.
__device__ __forceinline__ void split_halves(float v, uint32_t &hi, uint32_t &lo) {
  const f16_t h = static_cast<f16_t>(v);
  const f16_t l = static_cast<f16_t>(v - static_cast<float>(h));
  hi = __builtin_bit_cast(uint16_t, h);
  lo = __builtin_bit_cast(uint16_t, l);
}

__device__ __forceinline__ uint2 *col_place(uint4 *p, int k_blocks, int i0, int j0, int q,
                                            int plane, int lane) {
  const int64_t block = static_cast<int64_t>(j0 / 32) * k_blocks + i0 / 16 + q / 2;
  uint4 *const unit = p + (block * 2 + plane) * kWave + lane % 32 + 32 * (q % 2);
  return reinterpret_cast<uint2 *>(unit) + lane / 32;
}

__device__ __forceinline__ void store_block(const float (&v)[16], uint4 *by_col, int k_col,
                                            uint4 *by_row, int k_row, int i0, int j0,
                                            uint32_t *stage) {
  const int lane = lane_id();
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      split_halves(v[4 * q + e], hi[e], lo[e]);
      if (by_row) stage[(8 * q + 4 * (lane / 32) + e) * kStageRow + lane % 32] = hi[e] | lo[e] << 16;
    }
    *col_place(by_col, k_col, i0, j0, q, 0, lane) =
        make_uint2(hi[0] | hi[1] << 16, hi[2] | hi[3] << 16);
    *col_place(by_col, k_col, i0, j0, q, 1, lane) =
        make_uint2(lo[0] | lo[1] << 16, lo[2] | lo[3] << 16);
  }
  if (!by_row) return;
  wave_lds_order();
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const int row = lane % 32, part = lane / 32 + 2 * s; // 8 columns from 8 part
    const uint4 *const from = reinterpret_cast<const uint4 *>(stage + row * kStageRow + 8 * part);
    const uint4 p = from[0], q = from[1];
    uint4 hi, lo;
    hi.x = (p.x & 0xffff) | p.y << 16, lo.x = p.x >> 16 | (p.y & 0xffff0000u);
    hi.y = (p.z & 0xffff) | p.w << 16, lo.y = p.z >> 16 | (p.w & 0xffff0000u);
    hi.z = (q.x & 0xffff) | q.y << 16, lo.z = q.x >> 16 | (q.y & 0xffff0000u);
    hi.w = (q.z & 0xffff) | q.w << 16, lo.w = q.z >> 16 | (q.w & 0xffff0000u);
    const int64_t block = static_cast<int64_t>(i0 / 32) * k_row + j0 / 16 + part / 2;
    uint4 *const unit = by_row + block * 2 * kWave + row + 32 * (part % 2);
    unit[0] = hi;
    unit[kWave] = lo;
  }
  wave_lds_order();
}

// The values (scaled) that store_block put into by_col.
__device__ __forceinline__ void load_block(const uint4 *by_col, int k_col, int i0, int j0,
                                           float (&v)[16]) {
  const int lane = lane_id();
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const uint2 h = *col_place(const_cast<uint4 *>(by_col), k_col, i0, j0, q, 0, lane);
    const uint2 l = *col_place(const_cast<uint4 *>(by_col), k_col, i0, j0, q, 1, lane);
    const uint32_t hs[4] = {h.x & 0xffff, h.x >> 16, h.y & 0xffff, h.y >> 16};
    const uint32_t ls[4] = {l.x & 0xffff, l.x >> 16, l.y & 0xffff, l.y >> 16};
#pragma unroll
    for (int e = 0; e < 4; ++e)
      v[4 * q + e] =
          static_cast<float>(__builtin_bit_cast(f16_t, static_cast<uint16_t>(hs[e]))) +
          static_cast<float>(__builtin_bit_cast(f16_t, static_cast<uint16_t>(ls[e])));
  }
}

// ---- norm and packing ------------------------------------------------------------

constexpr int kNormBlocks = 256; // partial sums per matrix

// Sums of squares in 64 bits: no overflow or underflow at any finite input.
__global__ void __launch_bounds__(kBlock) ortho_norm_kernel(OrthoArgs a) {
  const int64_t z = blockIdx.y, rows = a.tall ? a.n : a.m, cols = a.tall ? a.m : a.n;
  double s = 0.0;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const int64_t base = z * a.g_batch + r * a.g_stride;
    for (int64_t c = threadIdx.x; c < cols; c += kBlock) {
      const double v = load_typed(a.g, a.type, base + c);
      s += v * v;
    }
  }
  __shared__ double part[kBlock];
  part[threadIdx.x] = s;
  __syncthreads();
  for (int k = kBlock / 2; k > 0; k /= 2) {
    if (threadIdx.x < k) part[threadIdx.x] += part[threadIdx.x + k];
    __syncthreads();
  }
  if (threadIdx.x == 0) a.partial[z * kNormBlocks + blockIdx.x] = part[0];
}

// Packs X = G / (|G| + eps), 64 x 64 per workgroup, a 32 x 32 block per wave.
__global__ void __launch_bounds__(kBlock) ortho_pack_kernel(OrthoArgs a, int norm_blocks) {
  __shared__ double part[kBlock];
  __shared__ __attribute__((aligned(16))) uint32_t stage[4][32 * kStageRow];
  const int64_t z = blockIdx.y;
  part[threadIdx.x] =
      static_cast<int>(threadIdx.x) < norm_blocks ? a.partial[z * kNormBlocks + threadIdx.x] : 0.0;
  __syncthreads();
  for (int k = kBlock / 2; k > 0; k /= 2) {
    if (threadIdx.x < k) part[threadIdx.x] += part[threadIdx.x + k];
    __syncthreads();
  }
  const double scale = static_cast<double>(kScale) / (sqrt(part[0]) + a.eps);
  const int wave = threadIdx.x / kWave, lane = lane_id();
  const int across = a.np / 64;
  const int i0 = blockIdx.x / across * 64 + wave / 2 * 32;
  const int j0 = blockIdx.x % across * 64 + wave % 2 * 32;
  const int j = j0 + lane % 32;
  float v[16];
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int i = i0 + 8 * (r / 4) + 4 * (lane / 32) + r % 4;
    v[r] = 0.0f;
    if (i < a.m && j < a.n) {
      const int64_t at = a.tall ? j * a.g_stride + i : i * a.g_stride + j;
      v[r] = static_cast<float>(load_typed(a.g, a.type, z * a.g_batch + at) * scale);
    }
  }
  const int64_t units = packed_units(a.mp, a.np);
  store_block(v, a.xt + z * units, a.mp / 16, a.x + z * units, a.np / 16, i0, j0, stage[wave]);
}

// ---- products ----------------------------------------------------------------------

enum Product { kGram, kPoly, kUpdate, kLast };

// C = P Q^T of packed operands, one TILE x TILE tile per workgroup of 2 x 2
// waves, 32 columns of both operands per stage: loaded to registers while the
// stage before is multiplied, then stored to the other half of LDS.
//   kGram:   P = Q = X;          writes A = C
//   kPoly:   P = Q = A;          writes B = b A + c C
//   kUpdate: P = B, Q = X^T;     writes X = a X + C in both orders
//   kLast:   the same to out, rounded to its type
template <int WHAT, int TILE>
__global__ void __launch_bounds__(kBlock) ortho_product_kernel(OrthoArgs a) {
  constexpr int kRows = TILE / 32;     // blocks of 32 rows of each operand
  constexpr int kSide = kRows / 2;     // of a wave
  constexpr int kStage = 4 * kWave;    // units of 32 rows and 32 columns: 2 blocks, hi and lo
  __shared__ __attribute__((aligned(16))) uint4 lds[2][2][kRows * kStage];
  constexpr bool kSymmetric = WHAT == kGram || WHAT == kPoly;

  const int64_t z = blockIdx.y;
  const int64_t xu = packed_units(a.mp, a.np), mu = packed_units(a.mp, a.mp);
  const uint4 *const p = WHAT == kGram ? a.x + z * xu : WHAT == kPoly ? a.gram + z * mu : a.poly + z * mu;
  const uint4 *const q = kSymmetric ? p : a.xt + z * xu;
  const int k_blocks = (WHAT == kGram ? a.np : a.mp) / 16; // both operands'
  const int tiles_n = (kSymmetric ? a.mp : a.np) / TILE;

  int ti, tj;
  if (kSymmetric) { // row ti of the triangle holds tiles_n - ti tiles
    const int t = blockIdx.x;
    ti = static_cast<int>((2 * tiles_n + 1 - sqrtf(static_cast<float>((2 * tiles_n + 1) * (2 * tiles_n + 1) - 8 * t))) / 2);
    while (ti > 0 && ti * tiles_n - ti * (ti - 1) / 2 > t) --ti;
    while ((ti + 1) * tiles_n - (ti + 1) * ti / 2 <= t) ++ti;
    tj = ti + t - (ti * tiles_n - ti * (ti - 1) / 2);
  } else {
    ti = blockIdx.x / tiles_n;
    tj = blockIdx.x % tiles_n;
  }

  const int tid = threadIdx.x, lane = lane_id(), wave = tid / kWave;
  const int wy = wave / 2, wx = wave % 2;
  const int64_t step = static_cast<int64_t>(k_blocks) * 2 * kWave; // units of 32 operand rows
  const uint4 *const pt = p + ti * kRows * step + tid;
  const uint4 *const qt = q + tj * kRows * step + tid;

  f32x16 acc[kSide][kSide];
#pragma unroll
  for (int i = 0; i < kSide; ++i) {
#pragma unroll
    for (int j = 0; j < kSide; ++j) {
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
    }
  }

  using u32x4 = uint32_t __attribute__((ext_vector_type(4)));
  u32x4 next[2][kRows];
  auto fetch = [&](int stage) {
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      next[0][r] = *reinterpret_cast<const u32x4 *>(pt + r * step + stage * kStage);
      next[1][r] = *reinterpret_cast<const u32x4 *>(qt + r * step + stage * kStage);
    }
  };
  auto put = [&](int half) {
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      *reinterpret_cast<u32x4 *>(&lds[half][0][r * kStage + tid]) = next[0][r];
      *reinterpret_cast<u32x4 *>(&lds[half][1][r * kStage + tid]) = next[1][r];
    }
  };
  const int stages = k_blocks / 2;
  fetch(0);
  put(0);
  __syncthreads();
  for (int s = 0; s < stages; ++s) {
    if (s + 1 < stages) fetch(s + 1);
    const uint4 *const lp = lds[s & 1][0], *const lq = lds[s & 1][1];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      f16x8 ph[kSide], pl[kSide], qh[kSide], ql[kSide];
#pragma unroll
      for (int i = 0; i < kSide; ++i) {
        const uint4 *const u = lp + (wy * kSide + i) * kStage + k * 2 * kWave + lane;
        ph[i] = __builtin_bit_cast(f16x8, u[0]);
        pl[i] = __builtin_bit_cast(f16x8, u[kWave]);
        const uint4 *const w = lq + (wx * kSide + i) * kStage + k * 2 * kWave + lane;
        qh[i] = __builtin_bit_cast(f16x8, w[0]);
        ql[i] = __builtin_bit_cast(f16x8, w[kWave]);
      }
#pragma unroll
      for (int i = 0; i < kSide; ++i) {
#pragma unroll
        for (int j = 0; j < kSide; ++j) {
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(pl[i], qh[j], acc[i][j], 0, 0, 0);
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ph[i], ql[j], acc[i][j], 0, 0, 0);
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ph[i], qh[j], acc[i][j], 0, 0, 0);
        }
      }
    }
    if (s + 1 < stages) put((s + 1) & 1);
    __syncthreads();
  }

  // The accumulators hold products of two scaled values.
  uint32_t *const stage = reinterpret_cast<uint32_t *>(&lds[0][0][0]) + wave * 32 * kStageRow;
#pragma unroll
  for (int bi = 0; bi < kSide; ++bi) {
#pragma unroll
    for (int bj = 0; bj < kSide; ++bj) {
      const int i0 = ti * TILE + (wy * kSide + bi) * 32, j0 = tj * TILE + (wx * kSide + bj) * 32;
      float v[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) v[r] = acc[bi][bj][r] * (1.0f / kScale);
      if constexpr (WHAT == kGram) {
        uint4 *const to = a.gram + z * mu;
        store_block(v, to, a.mp / 16, ti != tj ? to : nullptr, a.mp / 16, i0, j0, stage);
      } else if constexpr (WHAT == kPoly) {
        float old[16];
        load_block(p, a.mp / 16, i0, j0, old);
#pragma unroll
        for (int r = 0; r < 16; ++r) v[r] = a.b * old[r] + a.c * v[r];
        uint4 *const to = a.poly + z * mu;
        store_block(v, to, a.mp / 16, ti != tj ? to : nullptr, a.mp / 16, i0, j0, stage);
      } else {
        float old[16];
        load_block(q, a.mp / 16, i0, j0, old);
#pragma unroll
        for (int r = 0; r < 16; ++r) v[r] = a.a * old[r] + v[r];
        if constexpr (WHAT == kUpdate) {
          store_block(v, a.xt_next + z * xu, a.mp / 16, a.x + z * xu, a.np / 16, i0, j0, stage);
        } else {
          const int64_t j = j0 + lane % 32;
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int64_t i = i0 + 8 * (r / 4) + 4 * (lane / 32) + r % 4;
            if (i < a.m && j < a.n)
              store_typed(a.out, a.type, z * a.m * a.n + (a.tall ? j * a.m + i : i * a.n + j),
                          v[r] * (1.0f / kScale));
          }
        }
      }
    }
  }
}

// ---- host ----------------------------------------------------------------------------

struct OrthoLayout {
  int64_t m, n, mp, np;
  size_t partial, x, xt, xt_next, gram, poly, bytes;
};

OrthoLayout ortho_layout(int64_t batch, int64_t rows, int64_t cols) {
  OrthoLayout l{};
  l.m = std::min(rows, cols), l.n = std::max(rows, cols);
  l.mp = ceil_div64(l.m, kPad) * kPad, l.np = ceil_div64(l.n, kPad) * kPad;
  size_t at = 0;
  auto take = [&](int64_t elems, size_t size) {
    const size_t here = at;
    at += Workspace::align(static_cast<size_t>(batch * elems) * size);
    return here;
  };
  l.partial = take(kNormBlocks, sizeof(double));
  l.x = take(packed_units(l.mp, l.np), sizeof(uint4));
  l.xt = take(packed_units(l.mp, l.np), sizeof(uint4));
  l.xt_next = take(packed_units(l.mp, l.np), sizeof(uint4));
  l.gram = take(packed_units(l.mp, l.mp), sizeof(uint4));
  l.poly = take(packed_units(l.mp, l.mp), sizeof(uint4));
  l.bytes = at;
  return l;
}

constexpr int64_t kMostSide = 1 << 16;
constexpr int64_t kMostBatch = 1 << 15;

bool ortho_sizes(int64_t batch, int64_t rows, int64_t cols) {
  return batch >= 0 && batch <= kMostBatch && rows >= 1 && cols >= 1 && rows <= kMostSide &&
         cols <= kMostSide;
}

// Whether every value of the iteration stays in the halves' range: the largest
// singular value starts at most 1, and after a step is at most the maximum of
// |p| up to the largest before, at its end or where p' = a + 3 b t + 5 c t^2
// (t = s^2) is 0.  A's are its square and B's the maximum of |b t + c t^2|.
bool ortho_bounded(double a, double b, double c, int32_t steps) {
  if (!std::isfinite(a) || !std::isfinite(b) || !std::isfinite(c)) return false;
  double s = 1.0;
  for (int32_t k = 0; k < steps; ++k) {
    const double t = s * s;
    double poly = std::abs(b * t + c * t * t);
    if (c != 0.0 && -b / (2 * c) > 0.0 && -b / (2 * c) < t) poly = std::max(poly, std::abs(b * b / (4 * c)));
    double next = std::abs(s * (a + t * (b + t * c)));
    const double disc = 9 * b * b - 20 * a * c;
    double roots[3] = {-1.0, -1.0, -1.0};
    if (c != 0.0 && disc >= 0.0) {
      roots[0] = (-3 * b + std::sqrt(disc)) / (10 * c);
      roots[1] = (-3 * b - std::sqrt(disc)) / (10 * c);
    }
    if (c == 0.0 && b != 0.0) roots[2] = -a / (3 * b);
    for (double r : roots)
      if (r > 0.0 && r < t) next = std::max(next, std::abs(std::sqrt(r) * (a + r * (b + r * c))));
    if (!(t <= kMostValue && poly <= kMostValue && next <= kMostValue)) return false;
    s = next;
  }
  return true;
}

template <int WHAT> int32_t run_product(const OrthoArgs &a, void *stream) {
  constexpr bool kSymmetric = WHAT == kGram || WHAT == kPoly;
  auto tiles = [&](int64_t tile) {
    const int64_t down = a.mp / tile, across = a.np / tile;
    return kSymmetric ? down * (down + 1) / 2 : down * across;
  };
  return launch(ortho_product_kernel<WHAT, 128>, dim3(tiles(128), a.batch), dim3(kBlock), stream, a);
}

} // namespace

} // namespace sporder_hip

using namespace sporder_hip;

extern "C" {

size_t sporder_newton_schulz_work_bytes(int64_t batch, int64_t rows, int64_t cols) {
  return ortho_sizes(batch, rows, cols) ? ortho_layout(batch, rows, cols).bytes : 0;
}

int32_t sporder_newton_schulz(void *stream, int32_t type, int64_t batch, int64_t rows,
                              int64_t cols, int64_t g_batch_stride, int64_t g_stride,
                              const void *d_g, int32_t steps, double a, double b, double c,
                              double eps, void *d_out, void *d_work, size_t work_bytes) {
  if (!type_known(type) || !ortho_sizes(batch, rows, cols) || g_stride < 0 || g_batch_stride < 0 ||
      steps < 1 || !(eps >= 0.0) || !ortho_bounded(a, b, c, steps))
    return SPORDER_BAD_ARGUMENT;
  if (batch == 0) return SPORDER_OK;
  const OrthoLayout l = ortho_layout(batch, rows, cols);
  if (!d_g || !d_out || !d_work || !aligned_to(d_work, 256) || work_bytes < l.bytes)
    return SPORDER_BAD_ARGUMENT;
  char *const w = static_cast<char *>(d_work);
  OrthoArgs args{d_g,
                 d_out,
                 batch,
                 l.m,
                 l.n,
                 g_batch_stride,
                 g_stride,
                 static_cast<int>(l.mp),
                 static_cast<int>(l.np),
                 rows > cols,
                 type,
                 eps,
                 static_cast<float>(a),
                 static_cast<float>(b),
                 static_cast<float>(c),
                 reinterpret_cast<double *>(w + l.partial),
                 reinterpret_cast<uint4 *>(w + l.x),
                 reinterpret_cast<uint4 *>(w + l.xt),
                 reinterpret_cast<uint4 *>(w + l.xt_next),
                 reinterpret_cast<uint4 *>(w + l.gram),
                 reinterpret_cast<uint4 *>(w + l.poly)};
  const int norm_blocks = static_cast<int>(std::min<int64_t>(rows, kNormBlocks));
  int32_t rc = launch(ortho_norm_kernel, dim3(norm_blocks, batch), dim3(kBlock), stream, args);
  if (rc == SPORDER_OK)
    rc = launch(ortho_pack_kernel, dim3(l.mp / 64 * (l.np / 64), batch), dim3(kBlock), stream, args,
                norm_blocks);
  for (int32_t k = 0; k < steps && rc == SPORDER_OK; ++k) {
    rc = run_product<kGram>(args, stream);
    if (rc == SPORDER_OK) rc = run_product<kPoly>(args, stream);
    if (rc == SPORDER_OK)
      rc = k + 1 < steps ? run_product<kUpdate>(args, stream) : run_product<kLast>(args, stream);
    std::swap(args.xt, args.xt_next);
  }
  return rc;
}

} // extern "C"
