// newton_schulz.hip -- orthogonalising a matrix by Newton-Schulz products.
//
//   X = G / (|G|_F + eps),  then `steps` times:
//   A = X X^T,  B = b A + c A A,  X <- a X + B X        (m <= n; else of G^T)
//
// Each singular value s of G / |G| becomes p(p(...p(s))), p(s) = a s + b s^3 +
// c s^5, and the singular vectors stay.
//
// Products.  The matrix units multiply 32-bit floats at a sixteenth of the rate of
// 16-bit ones, so an operand x is two 16-bit halves, hi = fl16(x / u) and lo =
// fl16(x / u - hi), together 22 bits and a sign, and a product is hi hi + hi lo +
// lo hi with 32-bit accumulation: three matrix products, and lo lo (2^-22 of the
// result) left out.  X itself is held in 32 bits: only B X is made of halves.
//
// Units.  Small singular values grow by |a| a step, and a small row or column
// keeps its own size beside large ones, so steps that are absolute, or relative
// to the whole matrix, would grow into the result.  Every operand row has a unit
// u of its own, a power of two with 2^14 <= bound / u < 2^15 for a bound on the
// row's norm: nothing passes 2^16, and lo is exact down to 2^-39 of the bound.
// With q(t) = a + b t + c t^2 the update is q(A) X = X q(X^T X), so a step
// multiplies the norm of a row or column of X by at most the maximum g of |q(t)|,
// t = s^2, over the singular values s in [0, S] that occur, and leaves it at most
// S; A = X X^T has rows of at most S times X's, B = X (X^T (b + c A)) of at most h
// times, the maximum of |s (b + c s^2)|.  S, g and h follow from the coefficients
// and the number of steps, the first bounds from the largest elements of X's rows
// and columns.
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
using u32x4 = uint32_t __attribute__((ext_vector_type(4)));
using f32x16 = float __attribute__((ext_vector_type(16)));

constexpr double kMostValue = 31.0; // of singular values, A's and B's: past it nothing converges
constexpr int kBlock = 256;
constexpr int kPad = 128; // rows and columns are padded to multiples of it
constexpr int kStageRow = 40; // halves per row of a wave's transposing buffer

struct OrthoArgs {
  const void *g;
  void *out;
  int64_t batch, m, n;          // of X: m <= n
  int64_t g_batch, g_stride;    // of g, in elements
  int mp, np;                   // padded
  int tall;                     // X = G^T
  double eps;
  float a, b, c;
  float root_m, root_n;         // a little more than the roots of m and n
  float most, growth;           // S and g
  float now, next;              // growth of the norms up to this step, and past it
  float gram_unit, poly_unit;   // powers of two, at least S and h: units of A and B beside X's
  int row_strips, col_strips;   // of g, for its norm
  double *partial;              // [batch][kNormBlocks]
  float *row_part, *col_part;   // [batch][col_strips][g's rows], [batch][row_strips][g's columns]
  float *row_bound, *col_bound; // [batch][mp], [batch][np] of the first X
  float4 *state;                // X by blocks of 32 x 32, in the order of a wave's results
  uint4 *x, *xt, *xt_next, *gram, *poly; // packed operands, one after another per matrix
};

// uint4 units of a packed operand of `rows` by `cols` (both padded).
__host__ __device__ constexpr int64_t packed_units(int64_t rows, int64_t cols) {
  return rows * cols / 4; // two halves of 2 bytes each: 4 bytes per element
}

// The unit of a row whose norm is at most `bound`; the least, of bounds up to
// 2^-99, is 2^-114.
__device__ __forceinline__ float unit_above(float bound) {
  return __builtin_bit_cast(float, (max(__builtin_bit_cast(uint32_t, bound) >> 23, 27u) - 14) << 23);
}
// 1 / u for a power of two.
__device__ __forceinline__ float inverse(float u) {
  return __builtin_bit_cast(float, (254u << 23) - __builtin_bit_cast(uint32_t, u));
}
// The bound on a row or column of the first X from its largest element before
// the scaling and its length's root.
__device__ __forceinline__ float first_bound(float most, double scale, float root) {
  return fminf(1.0f, static_cast<float>(most * scale) * root); // NaN: 1
}

// The halves of two values in their units, hi and lo each packed in a word.
__device__ __forceinline__ void split_halves(float x, float y, uint32_t &hi, uint32_t &lo) {
  using f16x2 = f16_t __attribute__((ext_vector_type(2)));
  using f32x2 = float __attribute__((ext_vector_type(2)));
  const f32x2 v = {x, y};
  const f16x2 h = __builtin_convertvector(v, f16x2);
  // As products with -1: one mixed-precision instruction each, and exact.
  const f32x2 rest = {__builtin_fmaf(static_cast<float>(h.x), -1.0f, x),
                      __builtin_fmaf(static_cast<float>(h.y), -1.0f, y)};
  const f16x2 l = __builtin_convertvector(rest, f16x2);
  hi = __builtin_bit_cast(uint32_t, h);
  lo = __builtin_bit_cast(uint32_t, l);
}

// A wave's 32 x 32 block with row i0 and column j0: lane l holds column l % 32,
// rows 8 q + 4 (l / 32) + e in v[4 q + e].
__device__ __forceinline__ int block_row(int r) { return 8 * (r / 4) + 4 * (lane_id() / 32) + r % 4; }

// The units of a lane's rows, from their bounds.
__device__ __forceinline__ void row_units(const float4 (&bounds)[4], float growth, float most,
                                          float (&u)[16]) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    u[4 * q] = unit_above(fminf(most, bounds[q].x * growth));
    u[4 * q + 1] = unit_above(fminf(most, bounds[q].y * growth));
    u[4 * q + 2] = unit_above(fminf(most, bounds[q].z * growth));
    u[4 * q + 3] = unit_above(fminf(most, bounds[q].w * growth));
  }
}

__device__ __forceinline__ uint2 *col_place(uint4 *p, int k_blocks, int i0, int j0, int q,
                                            int plane, int lane) {
  const int64_t block = static_cast<int64_t>(j0 / 32) * k_blocks + i0 / 16 + q / 2;
  uint4 *const unit = p + (block * 2 + plane) * kWave + lane % 32 + 32 * (q % 2);
  return reinterpret_cast<uint2 *>(unit) + lane / 32;
}

// Stores a block, in units of its columns, with columns as operand rows; k_col
// is the operand's number of 16-column blocks.
__device__ __forceinline__ void store_by_col(const float (&v)[16], uint4 *by_col, int k_col, int i0,
                                             int j0) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint2 hi, lo;
    split_halves(v[4 * q], v[4 * q + 1], hi.x, lo.x);
    split_halves(v[4 * q + 2], v[4 * q + 3], hi.y, lo.y);
    *col_place(by_col, k_col, i0, j0, q, 0, lane_id()) = hi;
    *col_place(by_col, k_col, i0, j0, q, 1, lane_id()) = lo;
  }
}

// The same in units of its rows, with its own rows as operand rows: 8
// neighbouring columns of a row take a turn through LDS (`stage`, which may be
// the block's own place in by_row).
__device__ __forceinline__ void store_by_row(const float (&v)[16], uint4 *by_row, int k_row, int i0,
                                             int j0, uint16_t *stage) {
  const int lane = lane_id();
  uint32_t half[2][8];
  u32x4 held[2][2];
#pragma unroll
  for (int r = 0; r < 8; ++r) split_halves(v[2 * r], v[2 * r + 1], half[0][r], half[1][r]);
#pragma unroll
  for (int plane = 0; plane < 2; ++plane) {
    const uint32_t(&h)[8] = half[plane];
    // A word holds rows r and r + 1 of a column; with the neighbouring
    // column's, an even lane makes row r's word of both and an odd one r + 1's.
#pragma unroll
    for (int r = 0; r < 16; r += 2) {
      const uint32_t word = __builtin_amdgcn_perm(lane_xor_u32(h[r / 2], 1), h[r / 2],
                                                  lane & 1 ? 0x03020706 : 0x05040100);
      const int row = block_row(r) + (lane & 1);
      *reinterpret_cast<uint32_t *>(stage + row * kStageRow + (lane % 32 & ~1)) = word;
    }
    wave_lds_order();
#pragma unroll
    for (int s = 0; s < 2; ++s)
      held[plane][s] = *reinterpret_cast<const u32x4 *>(stage + lane % 32 * kStageRow +
                                                        8 * (lane / 32 + 2 * s));
    wave_lds_order();
  }
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const int part = lane / 32 + 2 * s; // 8 columns from 8 part
    const int64_t block = static_cast<int64_t>(i0 / 32) * k_row + j0 / 16 + part / 2;
#pragma unroll
    for (int plane = 0; plane < 2; ++plane)
      *reinterpret_cast<u32x4 *>(by_row + (block * 2 + plane) * kWave + lane % 32 +
                                 32 * (part % 2)) = held[plane][s];
  }
}

// X's block in the state, float4 q of lane l.
__device__ __forceinline__ float4 *state_place(const OrthoArgs &a, int64_t z, int i0, int j0, int q) {
  const int64_t block = static_cast<int64_t>(i0 / 32) * (a.np / 32) + j0 / 32;
  return a.state + z * (static_cast<int64_t>(a.mp) * a.np / 4) + (block * 4 + q) * kWave + lane_id();
}

// What a product's block is combined with, to be fetched early: hi and lo as
// store_by_col put them, or the state, and the bounds of its rows and column.
struct HeldBlock {
  uint4 word[4];
  float4 rows[4];
  float column;
};

// ---- norm and packing ------------------------------------------------------------

constexpr int kNormBlocks = 256; // partial sums per matrix, at most
constexpr int kNormThreads = 512;

constexpr int kStripCols = 512; // columns of a workgroup's strip: 8 per lane
constexpr int kStripRows = 32;  // and its rows, at least

// Sums of squares in 64 bits (no overflow or underflow at any finite input) and
// the largest elements of rows and columns, for a strip of rows and columns per
// workgroup: a row per wave, four of them under way.  4096 x 4096 floats in 18
// us, 3.8 TB/s.
template <typename T, int VEC>
__global__ void __launch_bounds__(kNormThreads) ortho_norm_kernel(OrthoArgs a) {
  constexpr int kParts = kStripCols / kWave / VEC, kWaves = kNormThreads / kWave, kRows = 4;
  const int64_t z = blockIdx.y, rows = a.tall ? a.n : a.m, cols = a.tall ? a.m : a.n;
  const int col_strip = blockIdx.x % a.col_strips, row_strip = blockIdx.x / a.col_strips;
  const int64_t per = ceil_div64(rows, a.row_strips);
  const int64_t first = row_strip * per, last = min(first + per, rows);
  const int64_t col0 = static_cast<int64_t>(col_strip) * kStripCols;
  const int lane = lane_id(), wave = threadIdx.x / kWave;
  const T *const g = static_cast<const T *>(a.g) + z * a.g_batch;
  float *const row_part = a.row_part + (z * a.col_strips + col_strip) * rows;
  float col_most[kParts][VEC] = {};
  double s[kRows] = {};
  for (int64_t row = first + wave; row < last; row += kRows * kWaves) {
    float v[kRows][kParts][VEC];
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
#pragma unroll
      for (int p = 0; p < kParts; ++p) {
        const int64_t col = col0 + (p * kWave + lane) * VEC;
        if (row + u * kWaves < last && col < cols) {
          load_f32<VEC>(g + (row + u * kWaves) * a.g_stride + col, v[u][p]);
        } else {
#pragma unroll
          for (int i = 0; i < VEC; ++i) v[u][p][i] = 0.0f;
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      float most = 0.0f;
#pragma unroll
      for (int p = 0; p < kParts; ++p) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          s[u] += static_cast<double>(v[u][p][i]) * v[u][p][i];
          most = fmaxf(most, fabsf(v[u][p][i]));
          col_most[p][i] = fmaxf(col_most[p][i], fabsf(v[u][p][i]));
        }
      }
      most = group_max<kWave>(most);
      if (lane == 0 && row + u * kWaves < last) row_part[row + u * kWaves] = most;
    }
  }
  __shared__ double part[kNormThreads];
  __shared__ float most[kWaves][kStripCols];
  part[threadIdx.x] = (s[0] + s[1]) + (s[2] + s[3]);
#pragma unroll
  for (int p = 0; p < kParts; ++p) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) most[wave][(p * kWave + lane) * VEC + i] = col_most[p][i];
  }
  __syncthreads();
  static_assert(kNormThreads == kStripCols);
  float m = 0.0f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) m = fmaxf(m, most[w][threadIdx.x]);
  if (col0 + threadIdx.x < cols)
    a.col_part[(z * a.row_strips + row_strip) * cols + col0 + threadIdx.x] = m;
  for (int k = kNormThreads / 2; k > 0; k /= 2) {
    if (threadIdx.x < k) part[threadIdx.x] += part[threadIdx.x + k];
    __syncthreads();
  }
  if (threadIdx.x == 0) a.partial[z * kNormBlocks + blockIdx.x] = part[0];
}

// Packs X = G / (|G| + eps), 64 x 64 per workgroup, a 32 x 32 block per wave,
// after the bounds of the rows and columns that it meets: 4096 x 4096 floats in
// 57 us, 268 MB at 4.7 TB/s.
template <typename T>
__global__ void __launch_bounds__(kBlock, 6) ortho_pack_kernel(OrthoArgs a, int norm_blocks) {
  __shared__ __attribute__((aligned(16))) uint16_t stage[4][32 * kStageRow];
  __shared__ float most[2][128];
  __shared__ __attribute__((aligned(16))) float bound[128]; // 64 rows, then 64 columns
  const int64_t z = blockIdx.y;
  const int tid = threadIdx.x, wave = tid / kWave, lane = lane_id();
  const int across = a.np / 64;
  const int tile_i = blockIdx.x / across * 64, tile_j = blockIdx.x % across * 64;
  const int i0 = tile_i + wave / 2 * 32, j0 = tile_j + wave % 2 * 32;
  const int j = j0 + lane % 32;
  const T *const g = static_cast<const T *>(a.g) + z * a.g_batch;
  float v[16];
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int i = i0 + block_row(r);
    v[r] = 0.0f;
    if (i < a.m && j < a.n)
      v[r] = static_cast<float>(g[a.tall ? j * a.g_stride + i : i * a.g_stride + j]);
  }
  // Two threads for each of the tile's rows and columns.
  const int item = tid % 128;
  const bool column = item >= 64, g_column = column != static_cast<bool>(a.tall);
  const int64_t at = column ? tile_j + item - 64 : tile_i + item, all = column ? a.n : a.m;
  if (at < all) {
    const int strips = g_column ? a.row_strips : a.col_strips;
    const float *const from = (g_column ? a.col_part : a.row_part) + z * strips * all + at;
    float m = 0.0f;
#pragma unroll 8
    for (int k = tid / 128; k < strips; k += 2) m = fmaxf(m, from[k * all]);
    most[tid / 128][item] = m;
  } else {
    most[tid / 128][item] = 0.0f;
  }
  double square = 0.0;
#pragma unroll
  for (int k = 0; k < kNormBlocks / kWave; ++k)
    if (lane + k * kWave < norm_blocks) square += a.partial[z * kNormBlocks + lane + k * kWave];
#pragma unroll
  for (int k = 1; k < kWave; k <<= 1) square += __shfl_xor(square, k);
  const double scale = 1.0 / (sqrt(square) + a.eps);
  __syncthreads();
  if (tid < 128) {
    bound[item] = first_bound(fmaxf(most[0][item], most[1][item]), scale, column ? a.root_m : a.root_n);
    if (!column && tile_j == 0) a.row_bound[z * a.mp + tile_i + item] = bound[item];
    if (column && tile_i == 0) a.col_bound[z * a.np + tile_j + item - 64] = bound[item];
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < 16; ++r) v[r] = static_cast<float>(v[r] * scale);
#pragma unroll
  for (int q = 0; q < 4; ++q)
    *state_place(a, z, i0, j0, q) = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
  const int64_t units = packed_units(a.mp, a.np);
  float u[16], w[16];
  const float col = inverse(unit_above(bound[64 + j0 - tile_j + lane % 32]));
#pragma unroll
  for (int r = 0; r < 16; ++r) w[r] = v[r] * col;
  store_by_col(w, a.xt + z * units, a.mp / 16, i0, j0);
  float4 rows[4];
#pragma unroll
  for (int q = 0; q < 4; ++q)
    rows[q] = *reinterpret_cast<const float4 *>(bound + i0 - tile_i + block_row(4 * q));
  row_units(rows, 1.0f, 1.0f, u);
#pragma unroll
  for (int r = 0; r < 16; ++r) w[r] = v[r] * inverse(u[r]);
  store_by_row(w, a.x + z * units, a.np / 16, i0, j0, stage[wave]);
}

// ---- products ----------------------------------------------------------------------

enum Product { kGram, kPoly, kUpdate, kLast };

// Writes a block of the result.
template <typename T>
__device__ __forceinline__ void write_block(const OrthoArgs &a, int64_t z, int i0, int j0,
                                            const float (&v)[16]) {
  const int64_t j = j0 + lane_id() % 32;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int64_t i = i0 + block_row(r);
    if (i < a.m && j < a.n)
      static_cast<T *>(a.out)[z * a.m * a.n + (a.tall ? j * a.m + i : i * a.n + j)] =
          static_cast<T>(v[r]);
  }
}

// What a product's block (i0, j0) is combined with, where it is.
template <int WHAT>
__device__ __forceinline__ HeldBlock fetch_old(const OrthoArgs &a, int64_t z, int i0, int j0) {
  HeldBlock old{};
  const float *const rows = a.row_bound + z * a.mp;
#pragma unroll
  for (int q = 0; q < 4; ++q) old.rows[q] = *reinterpret_cast<const float4 *>(rows + i0 + block_row(4 * q));
  old.column = (WHAT == kGram || WHAT == kPoly ? rows : a.col_bound + z * a.np)[j0 + lane_id() % 32];
  if constexpr (WHAT == kPoly) {
    uint4 *const from = a.gram + z * packed_units(a.mp, a.mp);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const uint2 hi = *col_place(from, a.mp / 16, i0, j0, q, 0, lane_id());
      const uint2 lo = *col_place(from, a.mp / 16, i0, j0, q, 1, lane_id());
      old.word[q] = make_uint4(hi.x, hi.y, lo.x, lo.y);
    }
  } else if constexpr (WHAT == kUpdate || WHAT == kLast) {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      old.word[q] = *reinterpret_cast<const uint4 *>(state_place(a, z, i0, j0, q));
  }
  return old;
}

// The epilogue of a product for one wave's block: v holds P Q^T in their units,
// so that row i's unit times column j's makes it whole.
template <int WHAT, typename T>
__device__ __forceinline__ void finish_block(const OrthoArgs &a, int64_t z, bool mirror, int i0,
                                             int j0, const float (&v)[16], const HeldBlock &old,
                                             uint16_t *stage) {
  const int64_t xu = packed_units(a.mp, a.np), mu = packed_units(a.mp, a.mp);
  const int km = a.mp / 16, kn = a.np / 16;
  const float uj = unit_above(fminf(a.most, old.column * a.now));
  float u[16], w[16];
  row_units(old.rows, a.now, a.most, u);
  if constexpr (WHAT == kGram || WHAT == kPoly) {
    uint4 *const to = (WHAT == kGram ? a.gram : a.poly) + z * mu;
    if constexpr (WHAT == kGram) { // A = v u uj, and the unit of A's row j is uj gram_unit
      const float scale = 1.0f / a.gram_unit;
#pragma unroll
      for (int r = 0; r < 16; ++r) w[r] = v[r] * (u[r] * scale);
    } else { // A = held uj gram_unit, A A = v u uj gram_unit^2, B's unit uj poly_unit
      using f16x4 = f16_t __attribute__((ext_vector_type(4)));
      const float unit = a.gram_unit / a.poly_unit;
      const float b = a.b * unit, c = a.c * unit * a.gram_unit;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f16x4 hi = __builtin_bit_cast(f16x4, make_uint2(old.word[q].x, old.word[q].y));
        const f16x4 lo = __builtin_bit_cast(f16x4, make_uint2(old.word[q].z, old.word[q].w));
#pragma unroll
        for (int e = 0; e < 4; ++e)
          w[4 * q + e] = b * (static_cast<float>(hi[e]) + static_cast<float>(lo[e])) +
                         c * (v[4 * q + e] * u[4 * q + e]);
      }
    }
    store_by_col(w, to, km, i0, j0);
    if (!mirror) return;
#pragma unroll
    for (int r = 0; r < 16; ++r) w[r] *= uj * inverse(u[r]);
    store_by_row(w, to, km, i0, j0, stage);
  } else {
    float x[16];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const uint32_t held[4] = {old.word[q].x, old.word[q].y, old.word[q].z, old.word[q].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = 4 * q + e;
        x[r] = a.a * __builtin_bit_cast(float, held[e]) + v[r] * (u[r] * a.poly_unit) * uj;
      }
    }
    if constexpr (WHAT == kLast) {
      write_block<T>(a, z, i0, j0, x);
      return;
    }
#pragma unroll
    for (int q = 0; q < 4; ++q)
      *state_place(a, z, i0, j0, q) = make_float4(x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]);
    const float next = inverse(unit_above(fminf(a.most, old.column * a.next)));
#pragma unroll
    for (int r = 0; r < 16; ++r) w[r] = x[r] * next;
    store_by_col(w, a.xt_next + z * xu, km, i0, j0);
    row_units(old.rows, a.next, a.most, u);
#pragma unroll
    for (int r = 0; r < 16; ++r) w[r] = x[r] * inverse(u[r]);
    store_by_row(w, a.x + z * xu, kn, i0, j0, stage);
  }
}

// Tile t of `down` x `across` tiles, `group` rows of tiles at a time and down
// each column of them, so that neighbouring tiles share operands on both
// sides; with `ratio` > 0, of those on and above the diagonal, where row ti
// begins at tile ratio ti.
__device__ __forceinline__ void place_tile(int t, int down, int across, int ratio, int group,
                                           int &ti, int &tj) {
  for (int g = 0;; g += group) {
    const int rows = min(group, down - g), left = across - ratio * g;
    const int corner = ratio ? min(rows * ratio, left) : 0; // columns not all rows reach
    const int cut = ratio * rows * (rows - 1) / 2;
    const int all = rows * left - cut;
    if (t >= all) {
      t -= all;
      continue;
    }
    const int in_corner = rows * corner - cut;
    if (t >= in_corner) {
      t -= in_corner;
      ti = g + t % rows;
      tj = ratio * g + corner + t / rows;
      return;
    }
    for (ti = 0; t >= corner - ratio * ti; ++ti) t -= corner - ratio * ti;
    tj = ratio * (g + ti) + t;
    ti += g;
    return;
  }
}

// C = P Q^T of packed operands, 256 x 128 per workgroup, 64 rows for each of
// four waves, 32 columns of the operands per stage.  A wave reads its own rows
// of P straight into registers, a stage ahead (no other wave of the workgroup
// needs them); Q goes through LDS, which then has 80 KB to move per 1,536
// cycles of products, where two operands in LDS would need twice that and
// would bound the kernel.
//   kGram:   P = Q = X;          writes A = C
//   kPoly:   P = Q = A;          writes B = b A + c C
//   kUpdate: P = B, Q = X^T;     writes X = a X + C in both orders
//   kLast:   the same to out, rounded to its type
// Bound by the matrix units: an update of 4096 x 4096 in 373 to 384 us, 1.07 to
// 1.11 PFLOP/s of 16-bit products, a library's product of that size and type
// 1.15; some 20 us are the 134 MB of X in 32 bits, read and written.
constexpr int kTileRows = 256, kTileCols = 128;

template <int WHAT, typename T>
__global__ void __launch_bounds__(kBlock, 2) ortho_product_kernel(OrthoArgs a) {
  constexpr int kP = 2, kQ = kTileCols / 32; // blocks of 32 rows of P per wave, and of Q
  constexpr int kStage = 4 * kWave;          // units of 32 rows and 32 columns: 2 blocks, hi and lo
  constexpr bool kSymmetric = WHAT == kGram || WHAT == kPoly;
  __shared__ __attribute__((aligned(16))) u32x4 lds[2][kQ * kStage];

  const int64_t z = blockIdx.y;
  const int64_t xu = packed_units(a.mp, a.np), mu = packed_units(a.mp, a.mp);
  const uint4 *const p = WHAT == kGram ? a.x + z * xu : WHAT == kPoly ? a.gram + z * mu : a.poly + z * mu;
  const uint4 *const q = kSymmetric ? p : a.xt + z * xu;
  const int k_blocks = (WHAT == kGram ? a.np : a.mp) / 16; // both operands'
  const int across = (kSymmetric ? a.mp : a.np) / kTileCols;
  const int down = (a.mp + kTileRows - 1) / kTileRows;
  int ti, tj;
  place_tile(static_cast<int>(xcd_block()), down, across, kSymmetric ? 2 : 0, 4, ti, tj);

  const int tid = threadIdx.x, lane = lane_id(), wave = tid / kWave;
  const int64_t step = static_cast<int64_t>(k_blocks) * 2 * kWave; // units of 32 operand rows
  const int rb = ti * (kTileRows / 32) + wave * kP;                // first block of rows
  const bool live = rb * 32 < a.mp; // the last tile may hold 128 rows; mp is a multiple of those
  const u32x4 *const pt = reinterpret_cast<const u32x4 *>(p) + (live ? rb : 0) * step + lane;
  const u32x4 *const qt = reinterpret_cast<const u32x4 *>(q) + tj * kQ * step + tid;

  f32x16 acc[kP][kQ] = {};
  u32x4 pv[2][2][kP][2], qv[kQ]; // P: parity of the stage, block of columns, of rows, hi and lo
  auto fetch_p = [&](u32x4(&v)[2][kP][2], int s) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int i = 0; i < kP; ++i) {
#pragma unroll
        for (int h = 0; h < 2; ++h) v[k][i][h] = pt[i * step + s * kStage + (k * 2 + h) * kWave];
      }
    }
  };
  auto fetch_q = [&](int s) {
#pragma unroll
    for (int r = 0; r < kQ; ++r) qv[r] = qt[r * step + s * kStage];
  };
  auto put_q = [&](int half) {
#pragma unroll
    for (int r = 0; r < kQ; ++r) lds[half][r * kStage + tid] = qv[r];
  };
  auto multiply = [&](const u32x4(&v)[2][kP][2], const u32x4 *lq) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int j = 0; j < kQ; ++j) {
        const f16x8 qh = __builtin_bit_cast(f16x8, lq[j * kStage + k * 2 * kWave + lane]);
        const f16x8 ql = __builtin_bit_cast(f16x8, lq[j * kStage + (k * 2 + 1) * kWave + lane]);
#pragma unroll
        for (int i = 0; i < kP; ++i)
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, v[k][i][1]), qh,
                                                             acc[i][j], 0, 0, 0);
#pragma unroll
        for (int i = 0; i < kP; ++i)
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, v[k][i][0]), ql,
                                                             acc[i][j], 0, 0, 0);
#pragma unroll
        for (int i = 0; i < kP; ++i)
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, v[k][i][0]), qh,
                                                             acc[i][j], 0, 0, 0);
      }
    }
  };

  const int stages = k_blocks / 2; // a multiple of 4
  fetch_q(0);
  fetch_p(pv[0], 0);
  put_q(0);
  __syncthreads();
  for (int s = 0; s < stages; s += 2) {
#pragma unroll
    for (int odd = 0; odd < 2; ++odd) {
      const int next = min(s + odd + 1, stages - 1);
      fetch_q(next);
      fetch_p(pv[odd ^ 1], next);
      multiply(pv[odd], lds[odd]);
      put_q(odd ^ 1);
      __syncthreads();
    }
  }

  uint16_t *const stage = reinterpret_cast<uint16_t *>(&lds[0][0]) + wave * 32 * kStageRow;
  if (!live) return;
#pragma unroll
  for (int i = 0; i < kP; ++i) {
#pragma unroll
    for (int j = 0; j < kQ; ++j) {
      const int i0 = (rb + i) * 32, j0 = tj * kTileCols + j * 32;
      if (kSymmetric && i0 > j0) continue; // the mirror image of another block
      float v[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) v[r] = acc[i][j][r];
      finish_block<WHAT, T>(a, z, i0 != j0, i0, j0, v, fetch_old<WHAT>(a, z, i0, j0), stage);
    }
  }
}

// The same for products of few tiles: 64 x 64 per workgroup, whose four or
// eight waves each take a part of the columns and read their operands straight
// from memory (in the units' own order, so without LDS), four steps ahead; the
// sums meet in LDS, a block of 32 x 32 for each of four waves.  A CU holds
// eight such waves: eight per tile while there is a CU for each tile, else
// four (1024 x 1536 in 1024: 27 us with eight, 21 with four).  Products of 1024 x
// 1024 x 1536 take 13 to 21 us.  An update of them is 384 tiles, one and a half
// turns of the CUs, that read 240 MB out of L2 at 12 TB/s (39 MB past it), with
// the matrix units busy in 28 % of the cycles.
constexpr int kAhead = 4;

// With first >= 0 they are the tiles of ortho_product_kernel from that one on,
// each as eight of these.
template <int WHAT, typename T, int WAVES>
__global__ void __launch_bounds__(WAVES *kWave) ortho_split_kernel(OrthoArgs a, int first_tile) {
  constexpr bool kSymmetric = WHAT == kGram || WHAT == kPoly;
  constexpr int kHalf = WAVES / 2;
  __shared__ float sums[kHalf][4][16][kWave];
  const int64_t z = blockIdx.y;
  const int64_t xu = packed_units(a.mp, a.np), mu = packed_units(a.mp, a.mp);
  const uint4 *const p = WHAT == kGram ? a.x + z * xu : WHAT == kPoly ? a.gram + z * mu : a.poly + z * mu;
  const uint4 *const q = kSymmetric ? p : a.xt + z * xu;
  const int k_blocks = (WHAT == kGram ? a.np : a.mp) / 16;
  const int across = (kSymmetric ? a.mp : a.np) / 64;
  int ti, tj;
  const int t = static_cast<int>(xcd_block());
  if (first_tile >= 0) {
    place_tile(first_tile + t / 8, (a.mp + kTileRows - 1) / kTileRows, across / 2,
               kSymmetric ? 2 : 0, 4, ti, tj);
    ti = ti * 4 + t % 8 / 2;
    tj = tj * 2 + t % 2;
    if (ti * 64 >= a.mp || (kSymmetric && ti > tj)) return;
  } else {
    place_tile(t, a.mp / 64, across, kSymmetric ? 1 : 0, kSymmetric ? 4 : 8, ti, tj);
  }
  const int wave = threadIdx.x / kWave, lane = lane_id();
  const int64_t step = static_cast<int64_t>(k_blocks) * 2 * kWave;
  const int mine = k_blocks / WAVES; // padded columns: a multiple of 8 blocks
  const int64_t first = static_cast<int64_t>(wave * mine) * 2 * kWave + lane;
  const uint4 *const pt = p + ti * 2 * step + first;
  const uint4 *const qt = q + tj * 2 * step + first;

  const int i0 = ti * 64 + wave % 4 / 2 * 32, j0 = tj * 64 + wave % 2 * 32; // finished by this wave
  HeldBlock old;
  if (wave < 4) old = fetch_old<WHAT>(a, z, i0, j0);
  f32x16 acc[2][2] = {};
  u32x4 next[kAhead][2][2][2]; // step, operand, block of 32 rows, hi and lo
  auto fetch = [&](u32x4(&o)[2][2][2], int k) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        o[0][i][h] = *reinterpret_cast<const u32x4 *>(pt + i * step + (k * 2 + h) * kWave);
        o[1][i][h] = *reinterpret_cast<const u32x4 *>(qt + i * step + (k * 2 + h) * kWave);
      }
    }
  };
#pragma unroll
  for (int d = 0; d < kAhead; ++d) fetch(next[d], min(d, mine - 1));
  for (int k0 = 0; k0 < mine; k0 += kAhead) {
#pragma unroll
    for (int d = 0; d < kAhead; ++d) {
      if (k0 + d < mine) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const f16x8 ph = __builtin_bit_cast(f16x8, next[d][0][i][0]);
            const f16x8 pl = __builtin_bit_cast(f16x8, next[d][0][i][1]);
            const f16x8 qh = __builtin_bit_cast(f16x8, next[d][1][j][0]);
            const f16x8 ql = __builtin_bit_cast(f16x8, next[d][1][j][1]);
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(pl, qh, acc[i][j], 0, 0, 0);
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ph, ql, acc[i][j], 0, 0, 0);
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ph, qh, acc[i][j], 0, 0, 0);
          }
        }
        fetch(next[d], min(k0 + d + kAhead, mine - 1));
      }
    }
  }
  if (wave >= kHalf) {
#pragma unroll
    for (int b = 0; b < 4; ++b) {
#pragma unroll
      for (int r = 0; r < 16; ++r) sums[wave - kHalf][b][r][lane] = acc[b / 2][b % 2][r];
    }
  }
  __syncthreads();
  if (wave < kHalf) {
#pragma unroll
    for (int b = 0; b < 4; ++b) {
#pragma unroll
      for (int r = 0; r < 16; ++r) sums[wave][b][r][lane] += acc[b / 2][b % 2][r];
    }
  }
  __syncthreads();
  if (wave >= 4) return;
  float v[16];
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    v[r] = sums[0][wave][r][lane] + sums[1][wave][r][lane];
    if constexpr (WAVES == 8) v[r] += sums[2][wave][r][lane] + sums[3][wave][r][lane];
  }
  // Only this wave reads block `wave` of the sums: one of them becomes its stage.
  wave_lds_order();
  uint16_t *const stage = reinterpret_cast<uint16_t *>(&sums[0][wave][0][0]);
  finish_block<WHAT, T>(a, z, ti != tj, i0, j0, v, old, stage);
}

// A whole matrix in one workgroup, X and X^T in LDS (at most 16 blocks of
// 32 x 32, padded to 32): its products take less than a launch each.  Eight
// waves take two neighbouring blocks of the result each; A, then B, takes X's
// place until the new X does.  A and B are computed whole: a wave per two
// blocks is there anyway, and needs no mirrored store.  100 x 128 in 52 us, 19 of
// them the CU's matrix units, the rest 15 products' waits and epilogues.
constexpr int kWholeWaves = 8;
constexpr int kWholeBlocks = 2 * kWholeWaves;
constexpr int kWholeUnits = kWholeBlocks * 32 * 32 / 4;
constexpr int kWholeRows = 128, kWholeSides = kWholeRows + 512; // X's rows, and its columns after them

// Whether every wave has at most one pair of neighbouring blocks of X (and of
// the square A, which is no larger).
constexpr bool ortho_whole(int64_t mp, int64_t np) {
  return mp / 32 * ((np / 32 + 1) / 2) <= kWholeWaves;
}

template <typename T>
__global__ void __launch_bounds__(kWholeWaves *kWave) ortho_whole_kernel(OrthoArgs a, int steps) {
  __shared__ __attribute__((aligned(16))) uint4 x[kWholeUnits], xt[kWholeUnits];
  __shared__ double part[kWholeWaves];
  __shared__ __attribute__((aligned(16))) float bound[kWholeSides], unit[2][kWholeSides];
  const int64_t z = blockIdx.x;
  const int wave = threadIdx.x / kWave, lane = lane_id();
  const int mb = a.mp / 32, nb = a.np / 32; // blocks down and across
  const int km = 2 * mb, kn = 2 * nb;       // blocks of 16 columns
  // Blocks (bi, bj) and (bi, bj + 1) of X, and of A and B.
  const int pairs_x = (nb + 1) / 2, pairs_a = (mb + 1) / 2;
  const int xi = wave / pairs_x, xj = wave % pairs_x * 2;
  const int ai = wave / pairs_a, aj = wave % pairs_a * 2;
  const int blocks_x = xi < mb ? min(2, nb - xj) : 0, blocks_a = ai < mb ? min(2, mb - aj) : 0;

  const T *const g = static_cast<const T *>(a.g) + z * a.g_batch;
  float va[2][16], vx[2][16]; // this wave's blocks of A or B, beside X's units, and of X
  double s = 0.0;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int j = (xj + t) * 32 + lane % 32;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int i = xi * 32 + block_row(r);
      vx[t][r] = 0.0f;
      if (t < blocks_x && i < a.m && j < a.n)
        vx[t][r] = static_cast<float>(g[a.tall ? j * a.g_stride + i : i * a.g_stride + j]);
    }
  }
  for (int i = threadIdx.x; i < kWholeSides; i += kWholeWaves * kWave) bound[i] = 0.0f;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      s += static_cast<double>(vx[t][r]) * vx[t][r];
    }
  }
  for (int k = 1; k < kWave; k <<= 1) s += __shfl_xor(s, k);
  if (lane == 0) part[wave] = s;
  __syncthreads();
  s = 0.0;
  for (int w = 0; w < kWholeWaves; ++w) s += part[w];
  const double scale = 1.0 / (sqrt(s) + a.eps);

  // The largest elements of rows and columns, as integers: positive floats order
  // alike, and NaN is past them all.
  auto largest = [&](int at, uint32_t v) { atomicMax(reinterpret_cast<uint32_t *>(bound) + at, v); };
  auto magnitude = [&](int t, int r) { return __builtin_bit_cast(uint32_t, vx[t][r]) & 0x7fffffffu; };
  if (blocks_x) {
    // Rows: each exchange halves the registers, until one row is left per lane.
    uint32_t most[16];
    int row = 0;
#pragma unroll
    for (int r = 0; r < 16; ++r) most[r] = max(magnitude(0, r), magnitude(1, r));
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int half = 8 >> k;
      const bool upper = lane >> k & 1;
      row += upper ? half : 0;
#pragma unroll
      for (int r = 0; r < half; ++r) {
        const uint32_t low = most[r], high = most[r + half];
        most[r] = max(upper ? high : low, lane_xor_u32(upper ? low : high, 1 << k));
      }
    }
    largest(xi * 32 + block_row(row), max(most[0], lane_xor_u32(most[0], 16)));
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      uint32_t column = 0;
#pragma unroll
      for (int r = 0; r < 16; ++r) column = max(column, magnitude(t, r));
      if (t < blocks_x) largest(kWholeRows + (xj + t) * 32 + lane % 32, column);
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kWholeSides; i += kWholeWaves * kWave) {
    bound[i] = first_bound(bound[i], scale, i < kWholeRows ? a.root_n : a.root_m);
    unit[0][i] = unit_above(bound[i]);
  }
  __syncthreads();

  // A block's place in x is its own until the barrier after: its stage.
  auto store_x = [&](int t, const float *units) {
    uint4 *const place = x + (xi * kn + (xj + t) * 2) * 2 * kWave;
    const float column = inverse(units[kWholeRows + (xj + t) * 32 + lane % 32]);
    float w[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) w[r] = vx[t][r] * column;
    store_by_col(w, xt, km, xi * 32, (xj + t) * 32);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float4 u = *reinterpret_cast<const float4 *>(units + xi * 32 + block_row(4 * q));
      w[4 * q] = vx[t][4 * q] * inverse(u.x), w[4 * q + 1] = vx[t][4 * q + 1] * inverse(u.y);
      w[4 * q + 2] = vx[t][4 * q + 2] * inverse(u.z), w[4 * q + 3] = vx[t][4 * q + 3] * inverse(u.w);
    }
    store_by_row(w, x, kn, xi * 32, (xj + t) * 32, reinterpret_cast<uint16_t *>(place));
  };
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    if (t >= blocks_x) continue;
#pragma unroll
    for (int r = 0; r < 16; ++r) vx[t][r] = static_cast<float>(vx[t][r] * scale);
    store_x(t, unit[0]);
  }
  __syncthreads();

  // acc = blocks (bi, bj) and (bi, bj + more) of P Q^T in their units, operands
  // of k blocks.
  f32x16 acc[2];
  auto product = [&](const uint4 *p, const uint4 *q, int k_blocks, int bi, int bj, int more) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[t][r] = 0.0f;
    }
    const uint4 *const pt = p + bi * k_blocks * 2 * kWave + lane;
    const uint4 *const qt = q + bj * k_blocks * 2 * kWave + lane;
    const uint4 *const rt = qt + more * k_blocks * 2 * kWave;
    for (int k = 0; k < k_blocks * 2 * kWave; k += 4 * kWave) { // an even number of blocks
      f16x8 o[2][3][2]; // block, operand, hi and lo
#pragma unroll
      for (int d = 0; d < 2; ++d) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int at = k + (2 * d + h) * kWave;
          o[d][0][h] = __builtin_bit_cast(f16x8, pt[at]);
          o[d][1][h] = __builtin_bit_cast(f16x8, qt[at]);
          o[d][2][h] = __builtin_bit_cast(f16x8, rt[at]);
        }
      }
#pragma unroll
      for (int d = 0; d < 2; ++d) {
#pragma unroll
        for (int h = 0; h < 3; ++h) { // lo hi, hi lo, hi hi
#pragma unroll
          for (int t = 0; t < 2; ++t)
            acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(o[d][0][h == 0], o[d][1 + t][h == 1],
                                                            acc[t], 0, 0, 0);
        }
      }
    }
  };
  // A or B, whose rows have X's units times `unit`.
  auto store_a = [&](float unit) {
    __syncthreads();
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      if (t >= blocks_a) continue;
      float w[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) w[r] = va[t][r] * (1.0f / unit);
      store_by_col(w, x, km, ai * 32, (aj + t) * 32);
    }
    __syncthreads();
  };

  float growth = 1.0f;
  for (int step = 0; step < steps; ++step) {
    const float *const now = unit[step & 1];
    float *const next = unit[~step & 1];
    growth = fminf(growth * a.growth, 0x1p100f);
    // f(block, register, product times its row's unit) for the products of two
    // blocks; their columns' units are left to f.
    auto each = [&](const float4(&rows)[4], auto &&f) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float u[4] = {rows[q].x, rows[q].y, rows[q].z, rows[q].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) f(t, 4 * q + e, acc[t][4 * q + e] * u[e]);
        }
      }
    };
    auto fetch_units = [&](int row0, float4(&rows)[4]) {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        rows[q] = *reinterpret_cast<const float4 *>(now + row0 + block_row(4 * q));
    };
    float4 units[4];
    if (blocks_a) {
      fetch_units(ai * 32, units);
      product(x, x, kn, ai, aj, blocks_a - 1);
      each(units, [&](int t, int r, float v) { va[t][r] = v; });
    }
    // The next units' place was last read before the step.
    for (int i = threadIdx.x; i < kWholeSides; i += kWholeWaves * kWave)
      next[i] = unit_above(fminf(a.most, bound[i] * growth));
    store_a(a.gram_unit);
    if (blocks_a) {
      product(x, x, km, ai, aj, blocks_a - 1);
      const float c = a.c * a.gram_unit * a.gram_unit;
      each(units, [&](int t, int r, float v) { va[t][r] = a.b * va[t][r] + c * v; });
    }
    store_a(a.poly_unit);
    if (blocks_x) {
      fetch_units(xi * 32, units);
      product(x, xt, km, xi, xj, blocks_x - 1);
      const float *const columns = now + kWholeRows + xj * 32 + lane % 32;
      const float column[2] = {columns[0] * a.poly_unit, columns[(blocks_x - 1) * 32] * a.poly_unit};
      each(units, [&](int t, int r, float v) { vx[t][r] = a.a * vx[t][r] + v * column[t]; });
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      if (t >= blocks_x) continue;
      if (step + 1 < steps)
        store_x(t, next);
      else
        write_block<T>(a, z, xi * 32, (xj + t) * 32, vx[t]);
    }
    __syncthreads();
  }
}

// ---- host ----------------------------------------------------------------------------

struct OrthoLayout {
  int64_t m, n, mp, np;
  bool whole; // one workgroup per matrix, no workspace
  size_t partial, row_part, col_part, row_bound, col_bound, state;
  size_t x, xt, xt_next, gram, poly, bytes;
};

// How the norm's workgroups cut G: strips of kStripCols columns, and of at least
// kStripRows rows, at most kNormBlocks together.
struct OrthoStrips {
  int64_t rows, cols;
};
OrthoStrips ortho_strips(int64_t rows, int64_t cols) {
  const int64_t across = ceil_div64(cols, kStripCols);
  return {std::clamp<int64_t>(ceil_div64(rows, kStripRows), 1, kNormBlocks / across), across};
}

OrthoLayout ortho_layout(int64_t batch, int64_t rows, int64_t cols) {
  OrthoLayout l{};
  l.m = std::min(rows, cols), l.n = std::max(rows, cols);
  l.mp = ceil_div64(l.m, 32) * 32, l.np = ceil_div64(l.n, 32) * 32;
  l.whole = ortho_whole(l.mp, l.np);
  if (l.whole) return l;
  l.mp = ceil_div64(l.m, kPad) * kPad, l.np = ceil_div64(l.n, kPad) * kPad;
  size_t at = 0;
  auto take = [&](int64_t elems, size_t size) {
    const size_t here = at;
    at += Workspace::align(static_cast<size_t>(batch * elems) * size);
    return here;
  };
  l.partial = take(kNormBlocks, sizeof(double));
  // Room for G of either orientation.
  const OrthoStrips wide = ortho_strips(l.m, l.n), tall = ortho_strips(l.n, l.m);
  l.row_part = take(std::max(wide.cols * l.m, tall.cols * l.n), sizeof(float));
  l.col_part = take(std::max(wide.rows * l.n, tall.rows * l.m), sizeof(float));
  l.row_bound = take(l.mp, sizeof(float));
  l.col_bound = take(l.np, sizeof(float));
  l.state = take(l.mp * l.np, sizeof(float));
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

// The maxima over the steps, found from the largest singular value: it starts at
// most 1, and after a step is at most the maximum of |p| up to the largest
// before, at its end or where p' = a + 3 b t + 5 c t^2 (t = s^2) is 0.  A's are
// its square and B's the maximum of |b t + c t^2|.
struct OrthoRange {
  bool bounded; // none passes kMostValue
  double most;  // S: of X's singular values
  double growth, poly; // g and h: maxima of |a + b t + c t^2| and |s (b + c t)| up to S
};
OrthoRange ortho_range(double a, double b, double c, int32_t steps) {
  if (!std::isfinite(a) || !std::isfinite(b) || !std::isfinite(c)) return {};
  double s = 1.0, most = 1.0;
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
    if (!(t <= kMostValue && poly <= kMostValue && next <= kMostValue)) return {};
    s = next;
    most = std::max(most, s);
  }
  OrthoRange range{true, most, std::abs(a), 0.0};
  const double end = most * most;
  for (double t : {end, c != 0.0 ? -b / (2 * c) : -1.0})
    if (t > 0.0 && t <= end) range.growth = std::max(range.growth, std::abs(a + t * (b + t * c)));
  for (double t : {end, c != 0.0 ? -b / (3 * c) : -1.0})
    if (t > 0.0 && t <= end) range.poly = std::max(range.poly, std::sqrt(t) * std::abs(b + t * c));
  return range;
}

constexpr int64_t kCus = 256;     // of an MI355X
constexpr int64_t kFewTiles = 128;
constexpr int64_t kMostOver = 96;

// The least power of two that is not below v, from 2^-60 on.
float power_above(double v) {
  return static_cast<float>(std::exp2(std::ceil(std::log2(std::max(v, 0x1p-60)))));
}

template <typename T> int32_t run_norm(const OrthoArgs &a, int blocks, void *stream) {
  const int64_t cols = a.tall ? a.m : a.n;
  const int vec = row_vec(sizeof(T), cols, {a.g_stride, a.g_batch}, {a.g});
  if (vec > 1) // 4 elements: 16 or 8 bytes
    return launch(ortho_norm_kernel<T, 4>, dim3(blocks, a.batch), dim3(kNormThreads), stream, a);
  return launch(ortho_norm_kernel<T, 1>, dim3(blocks, a.batch), dim3(kNormThreads), stream, a);
}

template <int WHAT, typename T>
int32_t run_split(const OrthoArgs &a, int64_t tiles, int first, void *stream) {
  if (tiles * a.batch <= kCus)
    return launch(ortho_split_kernel<WHAT, T, 8>, dim3(tiles, a.batch), dim3(8 * kWave), stream, a,
                  first);
  return launch(ortho_split_kernel<WHAT, T, 4>, dim3(tiles, a.batch), dim3(4 * kWave), stream, a,
                first);
}

template <int WHAT, typename T = float> int32_t run_product(const OrthoArgs &a, void *stream) {
  constexpr bool kSymmetric = WHAT == kGram || WHAT == kPoly;
  const int64_t down = ceil_div64(a.mp, kTileRows), across = (kSymmetric ? a.mp : a.np) / kTileCols;
  const int64_t tiles = kSymmetric ? down * across - down * (down - 1) : down * across;
  if (tiles * a.batch < kFewTiles) {
    const int64_t m64 = a.mp / 64, n64 = a.np / 64;
    return run_split<WHAT, T>(a, kSymmetric ? m64 * (m64 + 1) / 2 : m64 * n64, -1, stream);
  }
  // A CU's tiles take turns: with few tiles past a multiple of the CUs, some CUs
  // would have one more and the rest would wait, so those few are split.
  const int64_t over = a.batch == 1 && tiles > kCus && tiles % kCus <= kMostOver ? tiles % kCus : 0;
  int32_t rc = launch(ortho_product_kernel<WHAT, T>, dim3(tiles - over, a.batch), dim3(kBlock),
                      stream, a);
  if (rc == SPORDER_OK && over > 0)
    rc = run_split<WHAT, T>(a, 8 * over, static_cast<int>(tiles - over), stream);
  return rc;
}

template <typename T>
int32_t ortho_typed(OrthoArgs a, const OrthoLayout &l, int32_t steps, void *stream) {
  if (l.whole)
    return launch(ortho_whole_kernel<T>, dim3(a.batch), dim3(kWholeWaves * kWave), stream, a, steps);
  const int norm_blocks = a.row_strips * a.col_strips;
  int32_t rc = run_norm<T>(a, norm_blocks, stream);
  if (rc == SPORDER_OK)
    rc = launch(ortho_pack_kernel<T>, dim3(l.mp / 64 * (l.np / 64), a.batch), dim3(kBlock), stream,
                a, norm_blocks);
  for (int32_t k = 0; k < steps && rc == SPORDER_OK; ++k) {
    a.now = k > 0 ? a.next : 1.0f;
    a.next = std::min(a.now * a.growth, 0x1p100f);
    rc = run_product<kGram>(a, stream);
    if (rc == SPORDER_OK) rc = run_product<kPoly>(a, stream);
    if (rc == SPORDER_OK)
      rc = k + 1 < steps ? run_product<kUpdate>(a, stream) : run_product<kLast, T>(a, stream);
    std::swap(a.xt, a.xt_next);
  }
  return rc;
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
      steps < 1 || !(eps >= 0.0))
    return SPORDER_BAD_ARGUMENT;
  const OrthoRange range = ortho_range(a, b, c, steps);
  if (!range.bounded) return SPORDER_BAD_ARGUMENT;
  if (batch == 0) return SPORDER_OK;
  const OrthoLayout l = ortho_layout(batch, rows, cols);
  if (!d_g || !d_out) return SPORDER_BAD_ARGUMENT;
  if (l.bytes > 0 && (!d_work || !aligned_to(d_work, 256) || work_bytes < l.bytes))
    return SPORDER_BAD_ARGUMENT;
  char *const w = static_cast<char *>(d_work);
  const bool tall = rows > cols;
  const OrthoStrips strips = ortho_strips(rows, cols);
  OrthoArgs args{};
  args.g = d_g, args.out = d_out;
  args.batch = batch, args.m = l.m, args.n = l.n;
  args.g_batch = g_batch_stride, args.g_stride = g_stride;
  args.mp = static_cast<int>(l.mp), args.np = static_cast<int>(l.np);
  args.tall = tall, args.eps = eps;
  args.a = static_cast<float>(a), args.b = static_cast<float>(b), args.c = static_cast<float>(c);
  args.root_m = static_cast<float>(std::sqrt(l.m) * 1.001);
  args.root_n = static_cast<float>(std::sqrt(l.n) * 1.001);
  args.most = static_cast<float>(range.most), args.growth = static_cast<float>(range.growth);
  args.gram_unit = power_above(range.most), args.poly_unit = power_above(range.poly);
  args.row_strips = static_cast<int>(strips.rows), args.col_strips = static_cast<int>(strips.cols);
  args.partial = reinterpret_cast<double *>(w + l.partial);
  args.row_part = reinterpret_cast<float *>(w + l.row_part);
  args.col_part = reinterpret_cast<float *>(w + l.col_part);
  args.row_bound = reinterpret_cast<float *>(w + l.row_bound);
  args.col_bound = reinterpret_cast<float *>(w + l.col_bound);
  args.state = reinterpret_cast<float4 *>(w + l.state);
  args.x = reinterpret_cast<uint4 *>(w + l.x);
  args.xt = reinterpret_cast<uint4 *>(w + l.xt);
  args.xt_next = reinterpret_cast<uint4 *>(w + l.xt_next);
  args.gram = reinterpret_cast<uint4 *>(w + l.gram);
  args.poly = reinterpret_cast<uint4 *>(w + l.poly);
  if (type == SPORDER_TYPE_BF16) return ortho_typed<bf16_t>(args, l, steps, stream);
  if (type == SPORDER_TYPE_F16) return ortho_typed<f16_t>(args, l, steps, stream);
  return ortho_typed<float>(args, l, steps, stream);
}

} // extern "C"
