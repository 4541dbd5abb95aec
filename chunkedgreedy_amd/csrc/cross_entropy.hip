// cross_entropy.hip -- softmax cross entropy of linear logits that are never
// kept, and its gradients.
//
//   z[t][v] = x[t] . w[v] + b[v],  lse[t] = log sum_v exp z,  loss = lse - z[t][target]
//   g[t][v] = s[t] (exp(z - lse) - [v = target]),  dx = g w,  dw = g^T x,  db = sum_t g
//
// Rows.  Rows whose target is ignored cost nothing: the others are listed first
// and every product runs over the list.
//
// Forward.  A tile of z stays in the accumulators of its workgroup: each wave
// writes its tokens' largest logit and sum of exponentials over its classes, and
// the target's logit where it meets it; a second kernel joins the pieces.
//
// Backward.  For a piece of the rows and of the classes at a time the logits are made
// again and become g, in 16 bits and in both orders, since both products that follow sum
// along another side of it.  dx is summed over the pieces of the classes in 32 bits and final
// with each piece of the rows; dw is final with each piece of the classes, or, where the
// rows are cut too, summed over their pieces in 32 bits.  What the pieces hold is bounded
// (kPieceBytes each of g in either order and of the rows and classes turned for the
// products), so that beside them the scratch is w packed (where it is not read as it lies)
// and, over cut rows, dw in 32 bits.
//
// Types.  The matrix units take 16 bits.  The logits' operands are x and w themselves
// where those are 16 bits wide.  g is rounded to float16 before its products whatever
// the type (to bfloat16, one term with the target's class would bring an error of up
// to 2^-9 into a whole row: dx and dw 3.1e-3 off instead of 1.7e-3, which is the
// rounding of the results), and so w and x are float16 there, in units of their
// columns, powers of two by the largest element: bfloat16 values are exact down to
// 2^-29 of it, smaller ones within 2^-40 of it.  A token's scale s = m c 2^e enters g as
// m times 2^13, where 1 <= |m c| < 2 and c is the mantissa of the first row's, so that 11 bits
// are kept down to g = 2^-26; c and 2^e go to dx in 32 bits, c to dw so too and 2^e with x's
// rows.  Scales that are alike, of a mean or a sum, have m = 1: most rows' largest g lies just
// below 1, which floats hold to 2^-12, and m times it just above it would be held to 2^-11
// (8,192 rows of 2,048, 50,000 classes, c = 1.11: dx and dw 1.1e-3 from those of g in 32 bits
// with c in g, 8.0e-4 without).
// 32-bit operands are two 16-bit halves (22 bits) in units of their row, a power of two
// by its largest element, and products are three.
#include <algorithm>

#include "cross_entropy.hpp"
#include "mfma_product.hpp"

namespace sporder_hip {

namespace {

constexpr int kShift = 13; // g is held 2^13 times as large
constexpr int kListBlock = 1024; // rows of a block of the list
constexpr int64_t kListDirect = 65536; // rows up to which a block counts those before it

struct CeMeta {
  int32_t count; // rows listed
  int32_t most;  // largest exponent of their scales
};

struct CeArgs : CeCall {
  // scratch
  CeMeta *meta;
  int32_t *counts;       // of the list's blocks, past kListDirect rows
  int32_t *list, *target; // of the listed rows
  int32_t *exponent;
  float *mantissa, *row_lse, *miss; // miss_of
  float *bias32;      // [classes_pad], -inf past the classes
  float *hit;         // the target's logit
  float2 *partial;    // [chunks][rows_pad] largest and sum
  double *sum_parts;
  char *xp, *wp;      // operands of z: packed rows, or x and w themselves
  int64_t xp_stride, wp_stride, xp_plane, wp_plane; // bytes
  bool x_packed;      // by list position
  float *x_unit, *w_unit; // of their rows (32-bit types)
  char *xt, *wt;      // transposed operands, [dim][rows_pad] and [dim][piece]
  float *x_most, *w_most; // [dim]: largest of each column
  float *most_part;       // [strips][dim]
  char *g, *gt;       // [rows_pad][piece] and [piece][rows_pad]
  float *dx_part;     // [splits][rows_pad][dim_pad]
  float *dw_part;     // [splits][piece][dim_pad]
  float *db_part;     // [token chunks][piece]
  float *dw_sum, *db_sum; // of the pieces of the rows so far, [classes][dim_pad] and [classes]; or null
  int64_t rows_pad, dim_pad, classes_pad, chunks, piece;
  // A piece of the rows: the listed ones from `skip` on, at most `rows` of them; list, target,
  // exponent, mantissa, row_lse and miss begin there, rows_pad is the piece's.
  int64_t skip;
  bool last; // of the pieces
};

__device__ __forceinline__ int listed_here(const CeMeta *meta, int64_t skip, int64_t most) {
  return static_cast<int>(min(max(meta->count - skip, int64_t(0)), most));
}
__device__ __forceinline__ int listed_here(const CeArgs &a) { return listed_here(a.meta, a.skip, a.rows); }

// c of the scales.
__device__ __forceinline__ float common_mantissa(const CeArgs &a) {
  const uint32_t bits = __builtin_bit_cast(uint32_t, a.grad[0]), e = bits >> 23 & 255;
  return e == 0 || e == 255 ? 1.0f : __builtin_bit_cast(float, (bits & 0x7FFFFFu) | 127u << 23);
}

// ---- the list of rows, and what else comes first -----------------------------------

__device__ __forceinline__ void prepare(const CeArgs &a, int64_t block) {
  const int64_t i = block * 256 + threadIdx.x;
  if (i < a.classes_pad) {
    float b = -INFINITY;
    if (i < a.classes) {
      b = 0.0f;
      if (a.bias) with_type(a.bias, a.bias_type, [&](auto *p) { b = static_cast<float>(p[i]); });
    }
    a.bias32[i] = b;
  }
  if (a.w_unit && i >= a.classes && i < a.classes_pad) a.w_unit[i] = 1.0f;
}

__global__ void __launch_bounds__(256) ce_prepare_kernel(CeArgs a) {
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.meta = {0, -1000};
  prepare(a, blockIdx.x);
}

__global__ void __launch_bounds__(256) ce_count_kernel(CeArgs a) {
  __shared__ int32_t part[4];
  int n = 0;
#pragma unroll
  for (int k = 0; k < kListBlock / 256; ++k) {
    const int64_t row = blockIdx.x * int64_t(kListBlock) + k * 256 + threadIdx.x;
    n += __popcll(__ballot(row < a.rows && counted(a, target_of(a, row))));
  }
  if (lane_id() == 0) part[threadIdx.x / kWave] = n;
  __syncthreads();
  if (threadIdx.x == 0) a.counts[blockIdx.x] = part[0] + part[1] + part[2] + part[3];
}

// Sum over the workgroup, of one int per wave in `part` (uniform in each wave).
__device__ __forceinline__ int block_total(int mine, int32_t *part) {
  __syncthreads();
  if (lane_id() == 0) part[threadIdx.x / kWave] = mine;
  __syncthreads();
  return part[0] + part[1] + part[2] + part[3];
}

__device__ __forceinline__ int wave_total(int v) {
#pragma unroll
  for (int j = 1; j < kWave; j <<= 1) v += __shfl_xor(v, j);
  return v;
}

// The rows' places in the list: those counted before the block, then before the
// thread in it.  Workgroups past the list's `blocks` prepare.
__global__ void __launch_bounds__(256) ce_list_kernel(CeArgs a, bool backward, int blocks) {
  __shared__ int32_t part[4], placed[kListBlock / 256][4], most;
  if (blockIdx.x >= blocks) return prepare(a, blockIdx.x - blocks);
  const int tid = threadIdx.x, wave = tid / kWave, lane = lane_id();
  const int64_t first = blockIdx.x * int64_t(kListBlock);
  if (tid == 0) most = -1000;
  int before = 0;
  if (a.rows <= kListDirect) {
    constexpr int kAhead = 16;
    for (int64_t row = tid; row < first; row += 256 * kAhead) {
      RawTarget raw[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) raw[k] = fetch_target(a, row + k * 256);
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        before += row + k * 256 < first && class_of(a, row + k * 256, raw[k]) >= 0 ? 1 : 0;
    }
  } else {
#pragma unroll 4
    for (int64_t b = tid; b < blockIdx.x; b += 256) before += a.counts[b];
  }
  before = block_total(wave_total(before), part);
  constexpr int kEach = kListBlock / 256;
  RawTarget raw[kEach];
  int target[kEach];
  float scale[kEach] = {}, row_lse[kEach] = {}, row_loss[kEach] = {};
#pragma unroll
  for (int k = 0; k < kEach; ++k) { // past the rows the last one
    const int64_t row = min(first + k * 256 + tid, a.rows - 1);
    raw[k] = fetch_target(a, row);
    if (backward) {
      scale[k] = a.grad[row * a.grad_stride];
      row_lse[k] = a.given_lse[row];
      row_loss[k] = fetch_loss(a, row);
    }
  }
  uint64_t mask[kEach];
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    target[k] = class_of(a, first + k * 256 + tid, raw[k]);
    mask[k] = __ballot(target[k] >= 0);
    if (lane == 0) placed[k][wave] = __popcll(mask[k]);
  }
  __syncthreads();
  const float common = backward ? common_mantissa(a) : 1.0f;
  int top = -1000;
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int64_t row = first + k * 256 + tid;
    int at = before + __popcll(mask[k] & ((uint64_t(1) << lane) - 1));
    for (int w = 0; w < wave; ++w) at += placed[k][w];
    if (mask[k] >> lane & 1) {
      a.list[at] = static_cast<int32_t>(row);
      a.target[at] = target[k];
      if (backward) {
        // |s| = m c 2^e with 1 <= m c < 2 (a scale below 2^-126 keeps its place in m).
        const int e = max(static_cast<int>(__builtin_bit_cast(uint32_t, scale[k]) >> 23 & 255), 1) - 127;
        a.exponent[at] = e;
        a.mantissa[at] = ldexpf(scale[k], -e) / common;
        a.row_lse[at] = row_lse[k];
        a.miss[at] = miss_of(a, row_loss[k]);
        if (scale[k] != 0.0f) top = max(top, e);
      }
    } else if (row < a.rows && !backward) {
      const float none = target[k] == -1 ? 0.0f : NAN;
      a.loss[row] = none;
      a.lse[row] = none;
    }
    before += placed[k][0] + placed[k][1] + placed[k][2] + placed[k][3];
  }
  if (backward) atomicMax(&most, top);
  __syncthreads();
  if (backward && tid == 0) {
    if (blocks == 1)
      a.meta->most = most;
    else
      atomicMax(&a.meta->most, most);
  }
  if (blockIdx.x != blocks - 1) return;
  if (tid == 0) a.meta->count = before;
  // What the last tile reads past the list.
  const int64_t at = before + tid;
  if (at < a.rows_pad) {
    a.list[at] = 0;
    a.target[at] = -1;
    if (backward) {
      a.exponent[at] = 0;
      a.mantissa[at] = 0.0f;
      a.row_lse[at] = 0.0f;
      a.miss[at] = 1.0f;
    }
  }
}

// ---- packing -------------------------------------------------------------------------

template <typename U> __device__ __forceinline__ void split(float v, U &hi, U &lo) {
  hi = static_cast<U>(v);
  lo = static_cast<U>(v - static_cast<float>(hi));
}

// Rows of x (listed) or of w, which one launch packs: a launch costs some 4 us of a small
// call (64 rows of 276 over 243 classes, gradients: 67 us with a launch each).
struct CeRows {
  const void *src;
  int64_t stride, rows;
  const int32_t *list; // of x, from `skip` on
  int64_t skip;
  char *out;
  int64_t out_stride, plane; // bytes
  float *unit;               // of rows (32-bit types)
  float *most;               // of columns
  int64_t blocks;            // workgroups that take these rows
};

// Zeros up to a multiple of 64 elements: a wave per row, 8 elements a lane (580,000 rows of
// 500 bfloat16 260 us, 4.5 TB/s).
template <typename T, typename U, int PLANES>
__global__ void __launch_bounds__(256)
    ce_pack_rows_kernel(CeRows x, CeRows w, int64_t dim, const CeMeta *meta) {
  const bool first = blockIdx.x < x.blocks;
  const CeRows &a = first ? x : w;
  const int64_t row = (blockIdx.x - (first ? 0 : x.blocks)) * int64_t(4) + threadIdx.x / kWave;
  const int32_t *const list = a.list;
  if (row >= (list ? listed_here(meta, a.skip, a.rows) : a.rows)) return;
  const T *const from = static_cast<const T *>(a.src) + (list ? list[row] : row) * a.stride;
  const int64_t out_stride = a.out_stride, plane = a.plane;
  char *const out = a.out;
  float *const unit = a.unit;
  const int lane = lane_id();
  float scale = 1.0f;
  if constexpr (PLANES == 2) {
    float most = 0.0f;
    for (int64_t c = lane * 4; c < dim; c += kWave * 4) {
      const auto q = fetch<true, 4>(from + c, dim - c);
#pragma unroll
      for (int i = 0; i < 4; ++i) most = fmaxf(most, fabsf(static_cast<float>(q.v[i])));
    }
    const float u = unit_of(group_max<kWave>(most));
    scale = unit_inverse(u);
    if (lane == 0) unit[row] = u;
  }
  const int64_t width = ceil_div64(dim, kStageK) * kStageK;
  for (int64_t c = lane * 8; c < width; c += kWave * 8) {
    Pack<T, 8> q{};
    if (c < dim) q = fetch<true, 8>(from + c, dim - c);
    Pack<U, 8> hi, lo;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (PLANES == 2)
        split(static_cast<float>(q.v[i]) * scale, hi.v[i], lo.v[i]);
      else
        hi.v[i] = static_cast<U>(q.v[i]);
    }
    U *const to = reinterpret_cast<U *>(out + row * out_stride) + c;
    *reinterpret_cast<Pack<U, 8> *>(to) = hi;
    if constexpr (PLANES == 2)
      *reinterpret_cast<Pack<U, 8> *>(reinterpret_cast<char *>(to) + plane) = lo;
  }
}

// COUNT accesses of rows whose places are given, at column `col` or, past the rows' ends, the
// rows' last elements: `at` is where that is.  Without a branch at each, which would make the
// next access wait for it.
template <int VEC, int COUNT, typename T>
__device__ __forceinline__ void fetch_columns(const T *src, const int64_t (&place)[COUNT], int64_t stride,
                                              int64_t dim, int64_t col, int64_t &at, Pack<T, VEC> (&q)[COUNT]) {
  at = dim >= VEC ? min(col, dim - VEC) : col;
  if (dim >= VEC) {
#pragma unroll
    for (int k = 0; k < COUNT; ++k)
      q[k] = __builtin_bit_cast(Pack<T, VEC>,
                                *reinterpret_cast<const LoosePack<T, VEC> *>(src + place[k] * stride + at));
  } else {
#pragma unroll
    for (int k = 0; k < COUNT; ++k) q[k] = fetch<true, VEC>(src + place[k] * stride + at, dim - at);
  }
}
template <int COUNT> __device__ __forceinline__ void listed(const int32_t *list, int64_t (&place)[COUNT]) {
  if (!list) return;
#pragma unroll
  for (int k = 0; k < COUNT; ++k) place[k] = list[place[k]];
}

// The largest element of each column of rows of x (listed) or w: a strip of rows and 64
// accesses' columns per workgroup, then the strips'.  (One atomic maximum per strip and
// column instead: 206 us for 50,000 rows of 2,048 16-bit elements.)  Workgroups past both
// write zeros to dx where rows are not listed, 64 rows a wave.
constexpr int kStrips = 1024; // at most
template <typename T>
__global__ void __launch_bounds__(256)
    ce_column_most_kernel(CeRows ax, CeRows aw, CeArgs c, float *most) {
  constexpr int kVec = 16 / sizeof(T), kAhead = 8;
  __shared__ float part[4][kVec][kWave];
  const bool first = blockIdx.y < ax.blocks;
  const CeRows &a = first ? ax : aw;
  const T *const src = static_cast<const T *>(a.src);
  const int32_t *const list = a.list;
  const int64_t all = list ? listed_here(c) : a.rows, stride = a.stride, dim = c.dim;
  const int x = threadIdx.x % kWave, y = threadIdx.x / kWave;
  if (blockIdx.y >= ax.blocks + aw.blocks) {
    const int64_t before = ax.blocks + aw.blocks;
    for (int64_t r0 = ((blockIdx.y - before) * 4 + y) * kWave; r0 < c.rows; r0 += (gridDim.y - before) * 4 * kWave) {
      uint64_t rest = __ballot(r0 + x < c.rows && !counted(c, target_of(c, min(r0 + x, c.rows - 1))));
      for (; rest; rest &= rest - 1) {
        T *const out = static_cast<T *>(c.dx) + (r0 + __builtin_ctzll(rest)) * c.dx_stride;
#pragma unroll
        for (int k = 0; k < kVec; ++k) {
          const int64_t col = (blockIdx.x * int64_t(kVec) + k) * kWave + x;
          if (col < dim) out[col] = static_cast<T>(0.0f);
        }
      }
    }
    return;
  }
  const int64_t col = (blockIdx.x * int64_t(kWave) + x) * kVec, step = a.blocks * 4;
  float m[kVec] = {};
  int64_t at = col;
  if (col < dim) {
    for (int64_t r0 = (blockIdx.y - (first ? 0 : ax.blocks)) * 4 + y; r0 < all; r0 += step * kAhead) {
      int64_t place[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) place[k] = min(r0 + k * step, all - 1); // the last row again
      listed(list, place);
      Pack<T, kVec> q[kAhead];
      fetch_columns<kVec>(src, place, stride, dim, col, at, q);
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
#pragma unroll
        for (int e = 0; e < kVec; ++e) m[e] = fmaxf(m[e], fabsf(static_cast<float>(q[k].v[e])));
      }
    }
  }
  if (dim >= kVec) at = min(col, dim - kVec); // also where no row was
#pragma unroll
  for (int e = 0; e < kVec; ++e) part[y][e][x] = m[e];
  __syncthreads();
  if (y != 0) return;
#pragma unroll
  for (int e = 0; e < kVec; ++e)
    if (col < dim && at + e < dim)
      most[blockIdx.y * dim + at + e] =
          fmaxf(fmaxf(part[0][e][x], part[1][e][x]), fmaxf(part[2][e][x], part[3][e][x]));
}

// The strips' largest: 64 columns per workgroup, four threads each.
__global__ void __launch_bounds__(256)
    ce_strips_most_kernel(const float *parts, CeRows ax, CeRows aw, int64_t dim) {
  __shared__ float part[4][kWave];
  const int64_t strips = blockIdx.y ? aw.blocks : ax.blocks;
  float *const most = blockIdx.y ? aw.most : ax.most;
  if (blockIdx.y) parts += ax.blocks * dim;
  const int x = threadIdx.x % kWave, y = threadIdx.x / kWave;
  const int64_t col = blockIdx.x * int64_t(kWave) + x;
  float m = 0.0f;
  if (col < dim) {
#pragma unroll 8
    for (int64_t s = y; s < strips; s += 4) m = fmaxf(m, parts[s * dim + col]);
  }
  part[y][x] = m;
  __syncthreads();
  if (y == 0 && col < dim) most[col] = fmaxf(fmaxf(part[0][x], part[1][x]), fmaxf(part[2][x], part[3][x]));
}

// Columns of rows of x (listed) or w as operand rows: out[j][k] of k-th row,
// zeros for k past the rows up to a multiple of 64.  64 x 64 per workgroup,
// turned in LDS (25,000 rows of 2,048 bfloat16 49 us, 4.2 TB/s).  Listed rows come with 2^(their exponent - the largest).
template <typename T, int PLANES>
__global__ void __launch_bounds__(256)
    ce_pack_columns_kernel(CeRows ax, CeRows aw, int64_t dim, const CeMeta *meta, const int32_t *exponent) {
  __shared__ float tile[64][65];
  const bool first = blockIdx.x < ax.blocks;
  const CeRows &a = first ? ax : aw;
  const int32_t *const list = a.list;
  const T *const src = static_cast<const T *>(a.src);
  const float *const most = a.most;
  char *const out = a.out;
  const int64_t stride = a.stride, out_stride = a.out_stride, plane = a.plane;
  const int64_t all = list ? listed_here(meta, a.skip, a.rows) : a.rows;
  const int64_t k0 = (blockIdx.x - (first ? 0 : ax.blocks)) * int64_t(64), j0 = blockIdx.y * int64_t(64);
  if (k0 >= all) return;
  constexpr int kVec = 16 / sizeof(T), kAcross = 64 / kVec, kRound = 256 / kAcross, kRounds = 64 / kRound;
  const int x = threadIdx.x % kAcross * kVec, y = threadIdx.x / kAcross;
  const int top = list ? meta->most : 0;
  const int64_t col = j0 + x;
  Pack<T, kVec> q[kRounds];
  int power[kRounds] = {};
  int64_t place[kRounds], at;
#pragma unroll
  for (int i = 0; i < kRounds; ++i) place[i] = min(k0 + y + i * kRound, all - 1);
  if (list) {
#pragma unroll
    for (int i = 0; i < kRounds; ++i) power[i] = min(exponent[place[i]] - top, 0); // no row has a scale: top is below all
  }
  listed(list, place);
  fetch_columns<kVec>(src, place, stride, dim, min(col, dim - 1), at, q);
  float scale[kVec];
#pragma unroll
  for (int e = 0; e < kVec; ++e) scale[e] = unit_inverse(unit_of(most[min(at + e, dim - 1)]));
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    const int r = y + i * kRound;
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      float v = static_cast<float>(q[i].v[e]) * scale[e];
      if (list) v = ldexpf(v, power[i]);
      const int64_t j = at + e - j0; // an access at the end may begin before the tile
      if (j >= 0 && j < 64) tile[r][j] = k0 + r < all ? v : 0.0f;
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int j = threadIdx.x / 8 + 32 * i, c = threadIdx.x % 8 * 8;
    if (j0 + j >= dim) continue;
    Pack<f16_t, 8> hi, lo;
#pragma unroll
    for (int e = 0; e < 8; ++e) split(tile[c + e][j], hi.v[e], lo.v[e]);
    f16_t *const to = reinterpret_cast<f16_t *>(out + (j0 + j) * out_stride) + k0 + c;
    *reinterpret_cast<Pack<f16_t, 8> *>(to) = hi;
    if constexpr (PLANES == 2)
      *reinterpret_cast<Pack<f16_t, 8> *>(reinterpret_cast<char *>(to) + plane) = lo;
  }
}

// ---- logits ----------------------------------------------------------------------------

using Large = TileShape<2, 4, 4, 2>; // 256 classes x 256 tokens
using Middle = TileShape<2, 2, 2, 2>; // 128 x 128
using Narrow = TileShape<4, 1, 1, 1>; // 128 x 32

template <typename S> constexpr int logit_lds(bool backward) {
  const int a = S::kN * (S::kM * 2 + 16), b = S::kM * (S::kN * 2 + 16), c = 2 * S::kStage;
  return backward ? std::max(std::max(a, b), c) : c;
}

// Where a lane holds row `row` of a wave's MB blocks: i * 16 + r of its register, or -1.
template <int MB> __device__ __forceinline__ int register_of(int row) {
  return row >= 0 && row < MB * 32 && (row >> 2 & 1) == lane_id() / 32
             ? (row >> 5) * 16 + (row >> 3 & 3) * 4 + (row & 3)
             : -1;
}

// z of a tile: classes (from v0 on) down, listed rows across.
template <typename U, int PLANES, typename S>
__device__ __forceinline__ void logit_tile(const CeArgs &a, char *lds, int wave, int64_t m0, int64_t n0,
                                           int64_t v0, int count, f32x16 (&acc)[S::MB][S::NB]) {
  auto a_row = [&](int r) {
    return static_cast<uint32_t>(min(static_cast<int64_t>(r), a.classes - 1 - v0 - m0) * a.wp_stride);
  };
  auto b_row = [&](int r) {
    const int64_t n = min(n0 + r, int64_t(count) - 1);
    return static_cast<uint32_t>((a.x_packed ? n - n0 : a.list[n]) * a.xp_stride);
  };
  const char *const pa = a.wp + (v0 + m0) * a.wp_stride, *const pb = a.xp + (a.x_packed ? n0 * a.xp_stride : 0);
  const int stages = static_cast<int>(ceil_div64(a.dim, kStageK));
  if constexpr (S::kThreads == 512) {
    uint32_t a_off[S::kM / 16 / S::kWaves], b_off[S::kN / 16 / S::kWaves];
    ring_offsets(wave, a_off, a_row);
    ring_offsets(wave, b_off, b_row);
    ring_product<U, PLANES, S>(lds, wave, pa, a.wp_plane, a_off, pb, a.xp_plane, b_off, stages, acc);
  } else {
    uint32_t a_off[S::kFetchA], b_off[S::kFetchB];
    fetch_offsets<S::kWaves>(wave, a_off, a_row);
    fetch_offsets<S::kWaves>(wave, b_off, b_row);
    tile_product<U, PLANES, S>(lds, wave, pa, a.wp_plane, a_off, pb, a.xp_plane, b_off, stages, acc);
  }
  // Units and bias.
  const int lane = lane_id(), wm = wave / S::WN, wn = wave % S::WN;
  float x_unit[S::NB];
  if constexpr (PLANES == 2) {
#pragma unroll
    for (int j = 0; j < S::NB; ++j) x_unit[j] = a.x_unit[n0 + (wn * S::NB + j) * 32 + lane % 32];
  }
#pragma unroll
  for (int i = 0; i < S::MB; ++i) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int64_t m = v0 + m0 + (wm * S::MB + i) * 32 + result_row(4 * q);
      const float4 b = *reinterpret_cast<const float4 *>(a.bias32 + m);
      const float bias[4] = {b.x, b.y, b.z, b.w};
      float unit[4] = {1.0f, 1.0f, 1.0f, 1.0f};
      if constexpr (PLANES == 2) {
        const float4 u = *reinterpret_cast<const float4 *>(a.w_unit + m);
        unit[0] = u.x, unit[1] = u.y, unit[2] = u.z, unit[3] = u.w;
      }
#pragma unroll
      for (int j = 0; j < S::NB; ++j) {
        const float un = PLANES == 2 ? x_unit[j] : 1.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float z = acc[i][j][4 * q + e];
          acc[i][j][4 * q + e] = (PLANES == 2 ? z * unit[e] * un : z) + bias[e];
        }
      }
      __builtin_amdgcn_sched_barrier(0); // all vectors at once would not fit the registers
    }
  }
}

// A tile's share of lse: each wave's largest logits and sums over its classes.  Bound by the
// matrix units: 7,373 rows of 2,048 over 50,000 classes, bfloat16, in 1,343 us (1.12 PFLOP/s; the
// library's product alone 1.15 to 1.25), of which the part that is no product is some 7 %.
template <typename U, int PLANES, typename S>
__global__ void __launch_bounds__(S::kThreads) ce_loss_kernel(CeArgs a) {
  __shared__ __attribute__((aligned(16))) char lds[logit_lds<S>(false)];
  const int count = listed_here(a);
  int64_t ti, tj;
  place_tile(xcd_block(), ceil_div64(a.classes, S::kM), ceil_div64(a.rows, S::kN), 8, ti, tj);
  const int64_t m0 = ti * S::kM, n0 = tj * S::kN;
  if (n0 >= count) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = lane_id();
  const int wm = wave / S::WN, wn = wave % S::WN;
  f32x16 acc[S::MB][S::NB] = {};
  logit_tile<U, PLANES, S>(a, lds, wave, m0, n0, 0, count, acc);
#pragma unroll
  for (int j = 0; j < S::NB; ++j) {
    const int64_t n = n0 + (wn * S::NB + j) * 32 + lane % 32;
    const int met = register_of<S::MB>(n < count ? a.target[n] - static_cast<int>(m0) - wm * S::MB * 32 : -1);
    float most = -INFINITY, hit = 0.0f;
#pragma unroll
    for (int i = 0; i < S::MB; ++i) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        most = fmaxf(most, acc[i][j][r]);
        hit = met == i * 16 + r ? acc[i][j][r] : hit;
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if (met >= 0) a.hit[n] = hit;
    most = fmaxf(most, lane_xor_f32(most, 32));
    const float base = most == -INFINITY ? 0.0f : most;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < S::MB; ++i) {
#pragma unroll
      for (int r = 0; r < 16; ++r) sum += exp_of(acc[i][j][r] - base);
      __builtin_amdgcn_sched_barrier(0);
    }
    sum += lane_xor_f32(sum, 32);
    if (lane < 32 && n < count)
      a.partial[(ti * S::WM + wm) * a.rows_pad + n] = make_float2(most, sum);
  }
}

// Joins the pieces of 16 rows, 16 threads each.
__global__ void __launch_bounds__(256) ce_join_kernel(CeArgs a) {
  __shared__ float2 part[16][17];
  const int x = threadIdx.x % 16, y = threadIdx.x / 16;
  const int64_t n = blockIdx.x * int64_t(16) + x;
  const int count = listed_here(a);
  if (blockIdx.x * int64_t(16) >= count) return;
  float most = -INFINITY, sum = 0.0f;
  if (n < count) {
#pragma unroll 4
    for (int64_t c = y; c < a.chunks; c += 16) {
      const float2 p = a.partial[c * a.rows_pad + n];
      const float m = fmaxf(most, p.x), base = m == -INFINITY ? 0.0f : m;
      sum = sum * exp_of(most - base) + p.y * exp_of(p.x - base);
      most = m;
    }
  }
  part[y][x] = make_float2(most, sum);
  __syncthreads();
  if (y != 0 || n >= count) return;
  for (int k = 1; k < 16; ++k) most = fmaxf(most, part[k][x].x);
  const float base = most == -INFINITY ? 0.0f : most;
  sum = 0.0f;
  for (int k = 0; k < 16; ++k) sum += part[k][x].y * exp_of(part[k][x].x - base);
  a.lse[a.list[n]] = base + logf(sum);
  a.loss[a.list[n]] = loss_of(base, sum, a.hit[n]);
}

// The losses' sum and the number of rows not ignored, in 64 bits and a fixed
// order: workgroup by workgroup, then their parts.
constexpr int64_t kSumRows = 8192; // of a workgroup, or more
constexpr int64_t kSumBlocks = 256;

__global__ void __launch_bounds__(256) ce_sums_kernel(CeArgs a, int64_t per) {
  __shared__ double part[2][4];
  const int64_t first = blockIdx.x * per, last = min(first + per, a.rows);
  double s = 0.0, n = 0.0;
#pragma unroll 4
  for (int64_t row = first + threadIdx.x; row < last; row += 256) {
    s += a.loss[row];
    n += target_of(a, row) != a.ignore ? 1.0 : 0.0;
  }
  const double v = block_sums(s, n, part);
  if (threadIdx.x >= 2) return;
  if (gridDim.x == 1)
    a.sums[threadIdx.x] = static_cast<float>(v);
  else
    a.sum_parts[2 * blockIdx.x + threadIdx.x] = v;
}

__global__ void __launch_bounds__(256) ce_total_kernel(CeArgs a, int blocks) {
  __shared__ double part[2][4];
  double s = 0.0, n = 0.0;
  if (static_cast<int>(threadIdx.x) < blocks) {
    s = a.sum_parts[2 * threadIdx.x];
    n = a.sum_parts[2 * threadIdx.x + 1];
  }
  const double v = block_sums(s, n, part);
  if (threadIdx.x < 2) a.sums[threadIdx.x] = static_cast<float>(v);
}

// ---- gradients ---------------------------------------------------------------------------

// g of a tile in both orders, each turned in LDS and written by whole rows.  Half of the classes
// above in 860 us (0.88 PFLOP/s, and 745 MB written in the two orders: 131 us at a copy's rate that
// no other tile's products cover, for two tiles' accumulators don't fit the registers).
template <typename U, int PLANES, typename S>
__global__ void __launch_bounds__(S::kThreads) ce_g_kernel(CeArgs a, int64_t v0) {
  __shared__ __attribute__((aligned(16))) char lds[logit_lds<S>(true)];
  const int count = listed_here(a);
  int64_t ti, tj;
  place_tile(xcd_block(), ceil_div64(min(a.piece, a.classes - v0), S::kM), ceil_div64(a.rows, S::kN), 8,
             ti, tj);
  const int64_t m0 = ti * S::kM, n0 = tj * S::kN;
  if (n0 >= count) return;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / kWave), lane = lane_id();
  const int wm = wave / S::WN, wn = wave % S::WN;
  f32x16 acc[S::MB][S::NB] = {};
  logit_tile<U, PLANES, S>(a, lds, wave, m0, n0, v0, count, acc);
  const float common = common_mantissa(a);
  float lse[S::NB], miss[S::NB], m[S::NB], grad[S::NB];
  int target[S::NB];
#pragma unroll
  for (int j = 0; j < S::NB; ++j) {
    const int64_t n = n0 + (wn * S::NB + j) * 32 + lane % 32;
    const bool on = n < count;
    target[j] = register_of<S::MB>(on ? a.target[n] - static_cast<int>(v0 + m0) - wm * S::MB * 32 : -1);
    lse[j] = on ? a.row_lse[n] : 0.0f;
    miss[j] = on ? a.miss[n] : 1.0f;
    m[j] = on ? a.mantissa[n] * (1 << kShift) : 0.0f;
    grad[j] = on ? ldexpf(a.mantissa[n] * common, a.exponent[n]) : 0.0f;
  }
#pragma unroll
  for (int i = 0; i < S::MB; ++i) {
    float total[16] = {}; // of the classes over this wave's tokens
#pragma unroll
    for (int j = 0; j < S::NB; ++j) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float g = less_target(exp_of(acc[i][j][r] - lse[j]), target[j] == i * 16 + r, miss[j]);
        g = n0 + (wn * S::NB + j) * 32 + lane % 32 < count ? g : 0.0f; // the product is of another row
        total[r] += g * grad[j];
        acc[i][j][r] = g * m[j];
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if (a.db) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float v = group_sum<32>(total[r]);
        if (lane % 32 == 0)
          a.db_part[(tj * S::WN + wn) * a.piece + m0 + (wm * S::MB + i) * 32 + result_row(r)] = v;
      }
    }
  }
  constexpr int kDown = S::kM * 2 + 16, kAcross = S::kN * 2 + 16; // bytes of a row in LDS
#pragma unroll
  for (int plane = 0; plane < PLANES; ++plane) {
    // A plane's halves of classes 2 r and 2 r + 1 of a token.
    auto half = [&](int i, int j, int r) {
      Pack<f16_t, 2> p;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float v = acc[i][j][2 * r + e];
        p.v[e] = static_cast<f16_t>(v);
        if (plane) p.v[e] = static_cast<f16_t>(v - static_cast<float>(p.v[e]));
      }
      return __builtin_bit_cast(uint32_t, p);
    };
    // Not to keep the halves from one use to the next: with the sums they are more than
    // the registers.
    auto forget = [&] {
      if constexpr (PLANES == 2) {
#pragma unroll
        for (int i = 0; i < S::MB; ++i) {
#pragma unroll
          for (int j = 0; j < S::NB; ++j) asm volatile("" : "+v"(acc[i][j]));
        }
      }
    };
    forget();
    if (plane) __syncthreads();
#pragma unroll
    for (int i = 0; i < S::MB; ++i) {
#pragma unroll
      for (int j = 0; j < S::NB; ++j) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<uint2 *>(lds + ((wn * S::NB + j) * 32 + lane % 32) * kDown +
                                     ((wm * S::MB + i) * 32 + result_row(4 * q)) * 2) =
              make_uint2(half(i, j, 2 * q), half(i, j, 2 * q + 1));
      }
    }
    __syncthreads();
    char *const g = a.g + plane * (a.rows_pad * a.piece * 2) + (n0 * a.piece + m0) * 2;
#pragma unroll 4
    for (int c = tid; c < S::kN * (S::kM / 8); c += S::kThreads) {
      const int row = c / (S::kM / 8), part = c % (S::kM / 8);
      *reinterpret_cast<uint4 *>(g + row * a.piece * 2 + part * 16) =
          *reinterpret_cast<const uint4 *>(lds + row * kDown + part * 16);
    }
    __syncthreads();
    forget();
    // A word holds classes r and r + 1 of a token; with the neighbouring token's,
    // an even lane makes class r's word of both and an odd one r + 1's.
#pragma unroll
    for (int i = 0; i < S::MB; ++i) {
#pragma unroll
      for (int j = 0; j < S::NB; ++j) {
#pragma unroll
        for (int r = 0; r < 16; r += 2) {
          const uint32_t mine = half(i, j, r / 2);
          const uint32_t word = __builtin_amdgcn_perm(lane_xor_u32(mine, 1), mine,
                                                      lane & 1 ? 0x03020706 : 0x05040100);
          const int row = (wm * S::MB + i) * 32 + result_row(r) + (lane & 1);
          *reinterpret_cast<uint32_t *>(lds + row * kAcross +
                                        ((wn * S::NB + j) * 32 + (lane % 32 & ~1)) * 2) = word;
        }
      }
    }
    __syncthreads();
    char *const gt = a.gt + plane * (a.rows_pad * a.piece * 2) + (m0 * a.rows_pad + n0) * 2;
#pragma unroll 4
    for (int c = tid; c < S::kM * (S::kN / 8); c += S::kThreads) {
      const int row = c / (S::kN / 8), part = c % (S::kN / 8);
      *reinterpret_cast<uint4 *>(gt + row * a.rows_pad * 2 + part * 16) =
          *reinterpret_cast<const uint4 *>(lds + row * kAcross + part * 16);
    }
  }
}

// Four neighbouring elements of an output row.
template <typename O>
__device__ __forceinline__ void put_four(O *row, int64_t j, int64_t dim, bool whole, const float (&v)[4]) {
  if (whole && j + 4 <= dim) {
    store_f32<4>(row + j, v);
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (j + e < dim) row[j + e] = static_cast<O>(v[e]);
}

// A product's workgroups in a launch: `tiles` of them for each of `splits` parts of the sum,
// from workgroup `first` (a multiple of the XCDs) on.
struct CeShare {
  int64_t first, tiles;
  int splits;
};

// dx (DX) or the piece's rows of dw: features down, listed rows or classes across, over
// part `split` of the sum.  A sum in one part, over one piece, goes straight to the
// output (`direct`); else to the part's place in 32 bits, added to what is there past the
// first piece (`add`).
template <int PLANES, typename S, typename O, bool DX>
__device__ __forceinline__ void gradient_tile(const CeArgs &a, char *lds, int64_t v0, const CeShare &share,
                                              bool direct, bool add) {
  const int count = listed_here(a);
  const int64_t here = min(a.piece, a.classes - v0), across = DX ? a.rows : here;
  const int64_t at = blockIdx.x - share.first, all = share.tiles * share.splits;
  if (at >= all) return; // between two shares
  const int64_t each_xcd = all / kXcds, more = all % kXcds, xcd = at % kXcds;
  const int64_t t = xcd * each_xcd + min(xcd, more) + at / kXcds; // as xcd_block
  const int split = static_cast<int>(t / share.tiles);
  int64_t ti, tj;
  place_tile(t % share.tiles, ceil_div64(a.dim, S::kM), ceil_div64(across, S::kN), 8, ti, tj);
  const int64_t m0 = ti * S::kM, n0 = tj * S::kN;
  const int64_t limit = DX ? count : here;
  if (n0 >= limit) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = lane_id();
  const int wm = wave / S::WN, wn = wave % S::WN;
  const int64_t stride = (DX ? a.piece : a.rows_pad) * 2;
  uint32_t a_off[S::kFetchA], b_off[S::kFetchB];
  fetch_offsets<S::kWaves>(wave, a_off, [&](int r) {
    return static_cast<uint32_t>(min(static_cast<int64_t>(r), a.dim - 1 - m0) * stride);
  });
  fetch_offsets<S::kWaves>(wave, b_off, [&](int r) {
    return static_cast<uint32_t>(min(static_cast<int64_t>(r), limit - 1 - n0) * stride);
  });
  f32x16 acc[S::MB][S::NB] = {};
  const int64_t stages = ceil_div64(DX ? here : count, kStageK), each = ceil_div64(stages, share.splits);
  const int64_t first = min(split * each, stages), mine = min(each, stages - first);
  tile_product<f16_t, PLANES, S>(lds, wave, (DX ? a.wt : a.xt) + m0 * stride + first * kStageBytes,
                                 a.dim * stride, a_off,
                                 (DX ? a.g : a.gt) + n0 * stride + first * kStageBytes,
                                 a.rows_pad * a.piece * 2, b_off, static_cast<int>(mine), acc);
  O *const out = static_cast<O *>(DX ? a.dx : a.dw);
  const int64_t out_stride = DX ? a.dx_stride : a.dw_stride;
  const bool whole = out_stride % 4 == 0 && reinterpret_cast<uintptr_t>(out) % (4 * sizeof(O)) == 0;
  const float common = common_mantissa(a);
  float *const part = (DX ? a.dx_part : a.dw_part) + split * ((DX ? a.rows_pad : a.piece) * a.dim_pad);
#pragma unroll
  for (int j = 0; j < S::NB; ++j) {
    const int64_t n = n0 + (wn * S::NB + j) * 32 + lane % 32;
    if (n >= limit) continue;
    const int power = (DX ? a.exponent[n] : a.meta->most) - kShift;
    O *const row = out + (DX ? a.list[n] : v0 + n) * out_stride;
#pragma unroll
    for (int i = 0; i < S::MB; ++i) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int64_t m = m0 + (wm * S::MB + i) * 32 + result_row(4 * q);
        if (m >= a.dim) continue;
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = acc[i][j][4 * q + e];
        if (direct) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            v[e] = ldexpf(v[e] * (unit_of((DX ? a.w_most : a.x_most)[min(m + e, a.dim - 1)]) * common), power);
          put_four(row, m, a.dim, whole, v);
          continue;
        }
        float4 *const held = reinterpret_cast<float4 *>(part + n * a.dim_pad + m);
        if (add) {
          const float4 old = *held;
          v[0] += old.x, v[1] += old.y, v[2] += old.z, v[3] += old.w;
        }
        *held = make_float4(v[0], v[1], v[2], v[3]);
      }
    }
  }
}

// Both gradients of a piece in one launch, the longer sums first, so that the last ones
// fill what a launch of their own would leave idle.  That piece in 1,500 to 1,540 us (1.0
// PFLOP/s; a launch each 704 and 831 us: there the tiles fill the card either way; 2,001 rows of
// 1,000 over 20,011 classes in 32 bits gained 1,180 -> 1,080 us of the whole call).
template <int PLANES, typename S, typename T, typename O>
__global__ void __launch_bounds__(S::kThreads)
    ce_gradients_kernel(CeArgs a, int64_t v0, CeShare dx, CeShare dw, bool dx_direct, bool add, bool dw_direct) {
  __shared__ __attribute__((aligned(16))) char lds[2 * S::kStage];
  const bool first_dx = dx.first < dw.first;
  if (first_dx == (blockIdx.x < max(dx.first, dw.first)))
    gradient_tile<PLANES, S, T, true>(a, lds, v0, dx, dx_direct, add);
  else
    gradient_tile<PLANES, S, O, false>(a, lds, v0, dw, dw_direct, false);
}

// The parts' sum, four elements of a row per thread; of dw with what the pieces of the rows
// before gave.
template <typename O, bool DX>
__global__ void __launch_bounds__(256) ce_finish_kernel(CeArgs a, int64_t v0, int splits) {
  const int64_t n = blockIdx.z * int64_t(gridDim.y) + blockIdx.y, m = (blockIdx.x * int64_t(256) + threadIdx.x) * 4;
  const int64_t limit = DX ? listed_here(a) : min(a.piece, a.classes - v0);
  if (n >= limit || m >= a.dim) return;
  const int64_t part = (DX ? a.rows_pad : a.piece) * a.dim_pad;
  const float *const from = (DX ? a.dx_part : a.dw_part) + n * a.dim_pad + m;
  float v[4] = {};
  for (int s = 0; s < splits; ++s) {
    const float4 p = *reinterpret_cast<const float4 *>(from + s * part);
    v[0] += p.x, v[1] += p.y, v[2] += p.z, v[3] += p.w;
  }
  if (!DX && a.dw_sum) {
    float4 *const held = reinterpret_cast<float4 *>(a.dw_sum + (v0 + n) * a.dim_pad + m);
    if (a.skip > 0) {
      const float4 old = *held;
      v[0] += old.x, v[1] += old.y, v[2] += old.z, v[3] += old.w;
    }
    if (!a.last) {
      *held = make_float4(v[0], v[1], v[2], v[3]);
      return;
    }
  }
  const int power = (DX ? a.exponent[n] : a.meta->most) - kShift;
  const float common = common_mantissa(a);
#pragma unroll
  for (int e = 0; e < 4; ++e)
    v[e] = ldexpf(v[e] * (unit_of((DX ? a.w_most : a.x_most)[min(m + e, a.dim - 1)]) * common), power);
  O *const out = static_cast<O *>(DX ? a.dx : a.dw);
  const int64_t stride = DX ? a.dx_stride : a.dw_stride;
  const bool whole = stride % 4 == 0 && reinterpret_cast<uintptr_t>(out) % (4 * sizeof(O)) == 0;
  put_four(out + (DX ? a.list[n] : v0 + n) * stride, m, a.dim, whole, v);
}

// db of a piece: 16 classes per workgroup, 64 threads each.
__global__ void __launch_bounds__(1024) ce_bias_kernel(CeArgs a, int64_t v0, int tile) {
  __shared__ float part[64][17];
  const int x = threadIdx.x % 16, y = threadIdx.x / 16;
  const int64_t v = blockIdx.x * int64_t(16) + x;
  const int64_t chunks = ceil_div64(listed_here(a), tile) * (tile / 64);
  float s = 0.0f;
#pragma unroll 8
  for (int64_t c = y; c < chunks; c += 64) s += a.db_part[c * a.piece + v];
  part[y][x] = s;
  __syncthreads();
  for (int k = 32; k > 0; k /= 2) {
    if (y < k) part[y][x] += part[y + k][x];
    __syncthreads();
  }
  if (y != 0 || v0 + v >= a.classes) return;
  s = part[0][x];
  if (a.db_sum) {
    if (a.skip > 0) s += a.db_sum[v0 + v];
    if (!a.last) {
      a.db_sum[v0 + v] = s;
      return;
    }
  }
  store_typed(a.db, a.bias_type, v0 + v, s);
}

// ---- host --------------------------------------------------------------------------------

constexpr int64_t kPieceBytes = int64_t(512) << 20; // of g in one order, and of operands turned for it
constexpr int64_t kMostRows = (int64_t(1) << 23) - 256;
constexpr int64_t kMostListed = (int64_t(1) << 31) - 1024;
constexpr int64_t kMostClasses = int64_t(1) << 25;
constexpr int64_t kMostLogits = int64_t(1) << 37; // a launch's threads in 32 bits
constexpr int64_t kMostFeatures = 65536;

// How a product is cut: tiles of which shape (0 narrow, 1 middle, 2 large), and the sum
// into how many parts.
struct Cut {
  int shape, splits;
};

struct CePlan {
  bool x_direct, w_direct;
  int planes;
  Cut z, dx, dw;
  int64_t row_piece;
  size_t bytes;
};

bool direct_rows(int type, int64_t dim, int64_t stride, const void *p, int64_t span_rows) {
  return type != SPORDER_TYPE_F32 && dim % kStageK == 0 && stride % 8 == 0 && aligned_to(p, 16) &&
         span_rows * stride * 2 < (int64_t(1) << 32);
}

// A large tile (256 x 256, one to a CU) does four times a middle one's products, and of those
// two run on a CU: 8,192 x 50,000 with sums of 2,048 terms take 1.09 PFLOP/s in large tiles
// and 0.985 in middle ones, half the time of a large tile times their ratio.
constexpr double kMiddleTime = 0.55; // of a middle tile, two at a time, beside a large one's

Cut cut_logits(int64_t classes, int64_t rows) {
  const double large = static_cast<double>(ceil_div64(ceil_div64(classes, 256) * ceil_div64(rows, 256), 256));
  const double middle = static_cast<double>(ceil_div64(ceil_div64(classes, 128) * ceil_div64(rows, 128), 512));
  return {large <= middle * kMiddleTime ? 2 : 1, 1};
}

// The shape of both gradients' tiles and the parts of their sums: least time for all tiles
// over the card, the last ones half idle on average.  A part in 32 bits costs what 900
// elements of the sum do (written and read), and 32-bit sums stay below 65,536 terms.
void cut_gradients(int64_t dim, int64_t rows, int64_t classes, Cut &dx, Cut &dw) {
  double least = -1.0;
  auto parts = [](int64_t length) { return ceil_div64(length, 65536); };
  for (int shape : {1, 2}) {
    const int64_t side = shape == 2 ? 256 : 128;
    const double slots = shape == 2 ? 256 : 512, unit = shape == 2 ? 1.0 : kMiddleTime;
    const int64_t down = ceil_div64(dim, side);
    const int64_t nx = down * ceil_div64(rows, side), nw = down * ceil_div64(classes, side);
    for (int64_t sx = parts(classes); sx <= std::max<int64_t>(parts(classes), std::min<int64_t>(classes / 512, 32)); ++sx) {
      for (int64_t sw = parts(rows); sw <= std::max<int64_t>(parts(rows), std::min<int64_t>(rows / 512, 32)); ++sw) {
        const double x = static_cast<double>(classes) / sx + (sx > 1 ? 900.0 : 0.0) + 200.0;
        const double w = static_cast<double>(rows) / sw + (sw > 1 ? 900.0 : 0.0) + 200.0;
        const double all = x * (nx * sx) + w * (nw * sw);
        const double time = std::max(std::max(x, w), all / slots + 0.5 * std::min(x, w)) * unit;
        if (least < 0.0 || time < least) {
          least = time;
          dx = {shape, static_cast<int>(sx)};
          dw = {shape, static_cast<int>(sw)};
        }
      }
    }
  }
}

CePlan lay_out(CeArgs &a, bool backward, void *work) {
  CePlan p{};
  p.planes = a.type == SPORDER_TYPE_F32 ? 2 : 1;
  p.x_direct = direct_rows(a.type, a.dim, a.x_stride, a.x, a.rows);
  p.w_direct = direct_rows(a.type, a.dim, a.w_stride, a.w, 256);
  const int64_t rows_pad = ceil_div64(a.rows, 256) * 256; // of all rows
  a.rows_pad = rows_pad;
  a.dim_pad = ceil_div64(a.dim, kStageK) * kStageK;
  a.piece = ceil_div64(a.classes, 256) * 256;
  if (backward) { // pieces of one size, of at least 1,024 classes (or all) and as many rows as that leaves
    const int64_t elements = kPieceBytes / (2 * p.planes), fewest = std::min<int64_t>(1024, a.piece);
    auto cut = [](int64_t all, int64_t most) {
      return ceil_div64(ceil_div64(all, ceil_div64(all, most / 256 * 256)), 256) * 256;
    };
    a.rows_pad = cut(a.rows, elements / std::max(fewest, a.dim));
    a.piece = cut(a.classes, std::max(fewest, elements / std::max(a.rows_pad, a.dim)));
  }
  p.row_piece = a.rows_pad;
  const bool cut_rows = p.row_piece < a.rows;
  const int64_t rows_here = std::min(a.rows, p.row_piece);
  a.classes_pad = ceil_div64(a.classes, a.piece) * a.piece;
  p.z = cut_logits(std::min(a.piece, a.classes), rows_here);
  if (!backward && a.rows <= 64 && p.planes == 1) p.z.shape = 0;
  const int down = p.z.shape == 2 ? Large::kM : Middle::kM; // classes of a tile
  a.chunks = ceil_div64(a.classes, down) * (p.z.shape == 0 ? Narrow::WM : 2);
  size_t at = 0;
  auto take = [&](auto *&q, int64_t count) {
    using P = std::remove_reference_t<decltype(*q)>;
    q = reinterpret_cast<P *>(static_cast<char *>(work) + at);
    at += Workspace::align(static_cast<size_t>(count) * sizeof(P));
  };
  take(a.meta, 1);
  if (a.rows > kListDirect) take(a.counts, ceil_div64(a.rows, kListBlock));
  take(a.list, rows_pad);
  take(a.target, rows_pad);
  take(a.bias32, a.classes_pad);
  if (p.planes == 2) {
    take(a.x_unit, a.rows_pad);
    take(a.w_unit, a.classes_pad);
  }
  const int64_t row_bytes = a.dim_pad * 2;
  a.x_packed = !p.x_direct;
  if (p.x_direct) {
    a.xp = static_cast<char *>(const_cast<void *>(a.x));
    a.xp_stride = a.x_stride * 2;
  } else {
    a.xp_stride = row_bytes;
    a.xp_plane = rows_here * row_bytes;
    take(a.xp, a.xp_plane * p.planes);
  }
  if (p.w_direct) {
    a.wp = static_cast<char *>(const_cast<void *>(a.w));
    a.wp_stride = a.w_stride * 2;
  } else {
    a.wp_stride = row_bytes;
    a.wp_plane = a.classes * row_bytes;
    take(a.wp, a.wp_plane * p.planes);
  }
  if (!backward) {
    take(a.hit, a.rows_pad);
    take(a.partial, a.chunks * a.rows_pad);
    take(a.sum_parts, 2 * kSumBlocks);
  } else {
    take(a.exponent, rows_pad);
    take(a.mantissa, rows_pad);
    take(a.row_lse, rows_pad);
    take(a.miss, rows_pad);
    cut_gradients(a.dim, rows_here, std::min(a.piece, a.classes), p.dx, p.dw);
    take(a.x_most, a.dim);
    take(a.w_most, a.dim);
    take(a.most_part, 2 * kStrips * a.dim);
    take(a.xt, a.dim * a.rows_pad * 2 * p.planes);
    take(a.wt, a.dim * a.piece * 2 * p.planes);
    take(a.g, a.rows_pad * a.piece * 2 * p.planes);
    take(a.gt, a.rows_pad * a.piece * 2 * p.planes);
    if (a.piece < a.classes || p.dx.splits > 1) take(a.dx_part, p.dx.splits * a.rows_pad * a.dim_pad);
    if (p.dw.splits > 1 || cut_rows) take(a.dw_part, p.dw.splits * a.piece * a.dim_pad);
    if (a.db) take(a.db_part, a.rows_pad / 64 * a.piece);
    if (cut_rows) {
      take(a.dw_sum, a.classes * a.dim_pad);
      take(a.db_sum, a.classes);
    }
  }
  a.rows_pad = rows_pad;
  a.last = true;
  p.bytes = at;
  return p;
}

// Runs steps until one fails.
struct Steps {
  int32_t rc = SPORDER_OK;
  template <typename F> Steps &operator()(F &&f) {
    if (rc == SPORDER_OK) rc = f();
    return *this;
  }
};

CeRows rows_of_x(const CeArgs &a) {
  CeRows r{};
  r.src = a.x, r.stride = a.x_stride, r.rows = a.rows, r.list = a.list, r.skip = a.skip, r.most = a.x_most;
  return r;
}
CeRows rows_of_w(const CeArgs &a) {
  CeRows r{};
  r.src = a.w, r.stride = a.w_stride, r.rows = a.classes, r.most = a.w_most;
  return r;
}

// A piece of the rows from `skip` on.
CeArgs piece_of(CeArgs a, const CePlan &p, int64_t skip) {
  a.last = skip + p.row_piece >= a.rows;
  a.rows = std::min(p.row_piece, a.rows - skip);
  a.rows_pad = p.row_piece;
  a.skip = skip;
  a.list += skip, a.target += skip, a.exponent += skip, a.mantissa += skip, a.row_lse += skip, a.miss += skip;
  return a;
}

// x's rows (of a piece) and, with the first piece, w's.
template <typename T, typename U, int PLANES> int32_t pack_operands(const CeArgs &a, const CePlan &p, void *stream) {
  CeRows x = rows_of_x(a), w = rows_of_w(a);
  x.out = a.xp, x.out_stride = a.xp_stride, x.plane = a.xp_plane, x.unit = a.x_unit;
  w.out = a.wp, w.out_stride = a.wp_stride, w.plane = a.wp_plane, w.unit = a.w_unit;
  if (!p.x_direct) x.blocks = ceil_div64(a.rows, 4);
  if (!p.w_direct && a.skip == 0) w.blocks = ceil_div64(a.classes, 4);
  if (x.blocks + w.blocks == 0) return SPORDER_OK;
  return launch(ce_pack_rows_kernel<T, U, PLANES>, dim3(x.blocks + w.blocks), dim3(256), stream, x, w, a.dim,
                a.meta);
}

int32_t list_rows(const CeArgs &a, bool backward, void *stream) {
  Steps steps;
  const int64_t blocks = ceil_div64(a.rows, kListBlock), others = ceil_div64(a.classes_pad, 256);
  const bool alone = blocks == 1; // no workgroup needs what another one prepares
  if (!alone) steps([&] { return launch(ce_prepare_kernel, dim3(others), dim3(256), stream, a); });
  if (a.rows > kListDirect)
    steps([&] { return launch(ce_count_kernel, dim3(blocks), dim3(256), stream, a); });
  steps([&] {
    return launch(ce_list_kernel, dim3(blocks + (alone ? others : 0)), dim3(256), stream, a, backward, blocks);
  });
  return steps.rc;
}

template <typename T, typename U, int PLANES> int32_t forward(const CeArgs &a, const CePlan &p, void *stream) {
  Steps steps;
  steps([&] { return list_rows(a, false, stream); });
  steps([&] { return pack_operands<T, U, PLANES>(a, p, stream); });
  auto go = [&](auto shape) {
    using S = decltype(shape);
    return launch(ce_loss_kernel<U, PLANES, S>,
                  dim3(ceil_div64(a.classes, S::kM) * ceil_div64(a.rows, S::kN)), dim3(S::kThreads),
                  stream, a);
  };
  steps([&] {
    if constexpr (PLANES == 1) {
      if (p.z.shape == 0) return go(Narrow{});
    }
    return p.z.shape == 2 ? go(Large{}) : go(Middle{});
  });
  steps([&] { return launch(ce_join_kernel, dim3(ceil_div64(a.rows, 16)), dim3(256), stream, a); });
  const int64_t blocks = std::min(ceil_div64(a.rows, kSumRows), kSumBlocks);
  const int64_t per = ceil_div64(a.rows, blocks);
  steps([&] { return launch(ce_sums_kernel, dim3(blocks), dim3(256), stream, a, per); });
  if (blocks > 1)
    steps([&] { return launch(ce_total_kernel, dim3(1), dim3(256), stream, a, static_cast<int>(blocks)); });
  return steps.rc;
}

template <typename O, bool DX>
int32_t finish(const CeArgs &a, int64_t v0, int64_t rows, int splits, void *stream) {
  const int64_t deep = std::min<int64_t>(rows, 32768);
  return launch(ce_finish_kernel<O, DX>, dim3(ceil_div64(a.dim, 1024), ceil_div64(rows, ceil_div64(rows, deep)), ceil_div64(rows, deep)),
                dim3(256), stream, a, v0, splits);
}

// The gradients of a piece of the rows.
template <typename T, typename U, int PLANES> int32_t backward_piece(const CeArgs &a, const CePlan &p, void *stream) {
  Steps steps;
  steps([&] { return pack_operands<T, U, PLANES>(a, p, stream); });
  CeRows x = rows_of_x(a), w = rows_of_w(a);
  x.out = a.xt, x.out_stride = a.rows_pad * 2, x.plane = a.dim * x.out_stride;
  w.out = a.wt, w.out_stride = a.piece * 2, w.plane = a.dim * w.out_stride;
  x.blocks = ceil_div64(a.rows, 64);
  const bool one_piece = a.piece >= a.classes, dx_direct = one_piece && p.dx.splits == 1;
  const bool dw_direct = p.dw.splits == 1 && !a.dw_sum;
  for (int64_t v0 = 0; v0 < a.classes; v0 += a.piece) {
    const int64_t here = std::min(a.piece, a.classes - v0);
    w.src = static_cast<const T *>(a.w) + v0 * a.w_stride, w.rows = here;
    w.blocks = one_piece && a.skip > 0 ? 0 : ceil_div64(here, 64); // or there from the rows before
    steps([&] {
      return launch(ce_pack_columns_kernel<T, PLANES>, dim3(x.blocks + w.blocks, ceil_div64(a.dim, 64)), dim3(256),
                    stream, x, w, a.dim, a.meta, a.exponent);
    });
    x.blocks = 0; // with the first piece
    auto tiles = [&](auto shape) {
      using S = decltype(shape);
      return launch(ce_g_kernel<U, PLANES, S>, dim3(ceil_div64(here, S::kM) * ceil_div64(a.rows, S::kN)),
                    dim3(S::kThreads), stream, a, v0);
    };
    steps([&] { return p.z.shape == 2 ? tiles(Large{}) : tiles(Middle{}); });
    if (a.db)
      steps([&] {
        return launch(ce_bias_kernel, dim3(a.piece / 16), dim3(1024), stream, a, v0,
                      p.z.shape == 2 ? Large::kN : Middle::kN);
      });
    auto gradients = [&](auto shape, auto kind) {
      using S = decltype(shape);
      using O = decltype(kind);
      const int64_t down = ceil_div64(a.dim, S::kM);
      CeShare dx{0, down * ceil_div64(a.rows, S::kN), p.dx.splits};
      CeShare dw{0, down * ceil_div64(here, S::kN), p.dw.splits};
      const bool dx_first = here / dx.splits >= a.rows / dw.splits;
      CeShare &one = dx_first ? dx : dw, &two = dx_first ? dw : dx;
      two.first = ceil_div64(one.tiles * one.splits, kXcds) * kXcds;
      return launch(ce_gradients_kernel<PLANES, S, T, O>, dim3(two.first + two.tiles * two.splits),
                    dim3(S::kThreads), stream, a, v0, dx, dw, dx_direct, v0 > 0, dw_direct);
    };
    auto finish_dw = [&](auto kind) {
      return finish<decltype(kind), false>(a, v0, here, p.dw.splits, stream);
    };
    const bool wide = sizeof(T) == 2 && a.dw_type == SPORDER_TYPE_F32;
    steps([&] {
      if (wide) return p.dx.shape == 2 ? gradients(Large{}, float{}) : gradients(Middle{}, float{});
      return p.dx.shape == 2 ? gradients(Large{}, T{}) : gradients(Middle{}, T{});
    });
    if (!dw_direct) steps([&] { return wide ? finish_dw(float{}) : finish_dw(T{}); });
  }
  if (!dx_direct) steps([&] { return finish<T, true>(a, 0, a.rows, p.dx.splits, stream); });
  return steps.rc;
}

template <typename T, typename U, int PLANES> int32_t backward(const CeArgs &a, const CePlan &p, void *stream) {
  Steps steps;
  steps([&] { return list_rows(a, true, stream); });
  CeRows x = rows_of_x(a), w = rows_of_w(a);
  const int64_t across = ceil_div64(a.dim, kWave * (16 / sizeof(T)));
  auto strips = [&](int64_t rows) {
    return std::min(ceil_div64(rows, 32), std::min<int64_t>(std::max<int64_t>(1024 / across, 64), kStrips));
  };
  x.blocks = strips(a.rows), w.blocks = strips(a.classes);
  steps([&] {
    const int64_t zeros = std::min<int64_t>(ceil_div64(a.rows, 256), kStrips);
    return launch(ce_column_most_kernel<T>, dim3(across, x.blocks + w.blocks + zeros), dim3(256), stream, x, w, a,
                  a.most_part);
  });
  steps([&] {
    return launch(ce_strips_most_kernel, dim3(ceil_div64(a.dim, kWave), 2), dim3(256), stream, a.most_part, x,
                  w, a.dim);
  });
  for (int64_t skip = 0; skip < a.rows; skip += p.row_piece)
    steps([&] { return backward_piece<T, U, PLANES>(piece_of(a, p, skip), p, stream); });
  return steps.rc;
}

// Rows that a call may have, in both directions alike: a training step is refused by its
// forward call or not at all.  Where the loss takes one pass and the gradients tiles, as many
// as the list's numbers hold.
int64_t most_rows(const CeArgs &a) {
  if (!few_takes(a.type, a.dim, a.classes, false)) return std::min(kMostRows, kMostLogits / a.classes);
  return few_takes(a.type, a.dim, a.classes, true) ? kMostLogits : kMostListed;
}

bool bad_sizes(const CeArgs &a) {
  return !type_known(a.type) || !type_known(a.bias_type) || (a.target_bits != 32 && a.target_bits != 64) ||
         a.rows < 0 || a.dim < 1 || a.dim > kMostFeatures || a.classes < 1 || a.classes > kMostClasses ||
         a.rows > most_rows(a) || a.x_stride < 0 || a.w_stride < 0;
}

template <typename T> __global__ void ce_nothing_kernel(CeArgs a) {
  const int64_t i = blockIdx.x * int64_t(256) + threadIdx.x;
  const int64_t step = gridDim.x * int64_t(256);
  for (int64_t k = i; k < a.classes * a.dim; k += step)
    static_cast<T *>(a.dw)[k / a.dim * a.dw_stride + k % a.dim] = static_cast<T>(0.0f);
  for (int64_t k = i; k < a.classes && a.db; k += step) store_typed(a.db, a.bias_type, k, 0.0f);
}

__global__ void ce_no_rows_kernel(CeArgs a) {
  if (threadIdx.x < 2) a.sums[threadIdx.x] = 0.0f;
}

} // namespace

} // namespace sporder_hip

using namespace sporder_hip;

extern "C" {

size_t sporder_linear_cross_entropy_work_bytes(int32_t type, int64_t rows, int64_t dim, int64_t classes,
                                               int64_t x_stride, const void *d_x,
                                               int64_t weight_stride, const void *d_weight) {
  CeArgs a{};
  a.type = type, a.rows = rows, a.dim = dim, a.classes = classes, a.target_bits = 64;
  a.x_stride = x_stride, a.x = d_x, a.w_stride = weight_stride, a.w = d_weight;
  if (bad_sizes(a) || rows == 0) return 0;
  if (few_takes(type, dim, classes, false)) return few_work_bytes(rows, dim, classes, false);
  if (narrow_takes(type, rows, dim, classes, false)) return narrow_work_bytes(rows, dim, classes, false);
  return lay_out(a, false, nullptr).bytes;
}

int32_t sporder_linear_cross_entropy(void *stream, int32_t type, int64_t rows, int64_t dim,
                                     int64_t classes, int64_t x_stride, const void *d_x,
                                     int64_t weight_stride, const void *d_weight, int32_t bias_type,
                                     const void *d_bias, int32_t target_bits, const void *d_targets,
                                     int64_t ignore_index, float *d_loss, float *d_lse,
                                     float *d_sums, void *d_work, size_t work_bytes) {
  CeArgs a{};
  a.type = type, a.rows = rows, a.dim = dim, a.classes = classes, a.target_bits = target_bits;
  a.x_stride = x_stride, a.x = d_x, a.w_stride = weight_stride, a.w = d_weight;
  a.bias_type = bias_type, a.bias = d_bias, a.targets = d_targets, a.ignore = ignore_index;
  a.loss = d_loss, a.lse = d_lse, a.sums = d_sums;
  if (bad_sizes(a) || !d_sums) return SPORDER_BAD_ARGUMENT;
  if (rows == 0) return launch(ce_no_rows_kernel, dim3(1), dim3(kWave), stream, a);
  if (!d_x || !d_weight || !d_targets || !d_loss || !d_lse || !d_work || !aligned_to(d_work, 256))
    return SPORDER_BAD_ARGUMENT;
  if (few_takes(type, dim, classes, false))
    return work_bytes < few_work_bytes(rows, dim, classes, false) ? SPORDER_BAD_ARGUMENT
                                                                   : few_forward(a, d_work, stream);
  if (narrow_takes(type, rows, dim, classes, false))
    return work_bytes < narrow_work_bytes(rows, dim, classes, false) ? SPORDER_BAD_ARGUMENT
                                                                      : narrow_run(a, false, d_work, stream);
  const CePlan p = lay_out(a, false, d_work);
  if (work_bytes < p.bytes) return SPORDER_BAD_ARGUMENT;
  if (type == SPORDER_TYPE_BF16) return forward<bf16_t, bf16_t, 1>(a, p, stream);
  if (type == SPORDER_TYPE_F16) return forward<f16_t, f16_t, 1>(a, p, stream);
  return forward<float, f16_t, 2>(a, p, stream);
}

size_t sporder_linear_cross_entropy_grad_work_bytes(int32_t type, int64_t rows, int64_t dim,
                                                    int64_t classes, int64_t x_stride,
                                                    const void *d_x, int64_t weight_stride,
                                                    const void *d_weight) {
  CeArgs a{};
  a.type = type, a.rows = rows, a.dim = dim, a.classes = classes, a.target_bits = 64;
  a.x_stride = x_stride, a.x = d_x, a.w_stride = weight_stride, a.w = d_weight;
  a.db = &a; // the scratch of a bias whether there is one or not
  if (bad_sizes(a) || rows == 0) return 0;
  if (few_takes(type, dim, classes, true)) return few_work_bytes(rows, dim, classes, true);
  if (narrow_takes(type, rows, dim, classes, true)) return narrow_work_bytes(rows, dim, classes, true);
  return lay_out(a, true, nullptr).bytes;
}

int32_t sporder_linear_cross_entropy_grad_of_loss(
    void *stream, int32_t type, int64_t rows, int64_t dim, int64_t classes, int64_t grad_stride,
    const float *d_grad, int64_t x_stride, const void *d_x, int64_t weight_stride, const void
    *d_weight, int32_t bias_type, const void *d_bias, int32_t target_bits, const void *d_targets,
    int64_t ignore_index, const float *d_lse, const float *d_loss, int64_t dx_stride, void *d_dx,
    int32_t dweight_type, int64_t dweight_stride, void *d_dweight, void *d_dbias, void *d_work,
    size_t work_bytes) {
  CeArgs a{};
  a.type = type, a.rows = rows, a.dim = dim, a.classes = classes, a.target_bits = target_bits;
  a.x_stride = x_stride, a.x = d_x, a.w_stride = weight_stride, a.w = d_weight;
  a.bias_type = bias_type, a.bias = d_bias, a.targets = d_targets, a.ignore = ignore_index;
  a.grad = d_grad, a.grad_stride = grad_stride, a.given_lse = d_lse, a.given_loss = d_loss;
  a.dx = d_dx, a.dx_stride = dx_stride, a.dw = d_dweight, a.dw_stride = dweight_stride;
  a.dw_type = dweight_type, a.db = d_dbias;
  if (bad_sizes(a) || (dweight_type != type && dweight_type != SPORDER_TYPE_F32) || grad_stride < 0 ||
      dx_stride < 0 || (rows > 1 && dx_stride < dim) || dweight_stride < 0 ||
      (classes > 1 && dweight_stride < dim) || !d_dweight)
    return SPORDER_BAD_ARGUMENT;
  if (rows == 0) {
    const dim3 grid(std::min<int64_t>(ceil_div64(classes * dim, 256), 1 << 16));
    return dweight_type == SPORDER_TYPE_F32 ? launch(ce_nothing_kernel<float>, grid, dim3(256), stream, a)
                                            : launch(ce_nothing_kernel<f16_t>, grid, dim3(256), stream, a);
  }
  if (!d_grad || !d_x || !d_weight || !d_targets || !d_lse || !d_dx || !d_work || !aligned_to(d_work, 256))
    return SPORDER_BAD_ARGUMENT;
  if (few_takes(type, dim, classes, true))
    return work_bytes < few_work_bytes(rows, dim, classes, true) ? SPORDER_BAD_ARGUMENT
                                                                  : few_backward(a, d_work, stream);
  if (narrow_takes(type, rows, dim, classes, true))
    return work_bytes < narrow_work_bytes(rows, dim, classes, true) ? SPORDER_BAD_ARGUMENT
                                                                     : narrow_run(a, true, d_work, stream);
  const CePlan p = lay_out(a, true, d_work);
  if (work_bytes < p.bytes) return SPORDER_BAD_ARGUMENT;
  if (type == SPORDER_TYPE_BF16) return backward<bf16_t, bf16_t, 1>(a, p, stream);
  if (type == SPORDER_TYPE_F16) return backward<f16_t, f16_t, 1>(a, p, stream);
  return backward<float, f16_t, 2>(a, p, stream);
}

int32_t sporder_linear_cross_entropy_grad(void *stream, int32_t type, int64_t rows, int64_t dim,
                                          int64_t classes, int64_t grad_stride, const float *d_grad,
                                          int64_t x_stride, const void *d_x, int64_t weight_stride,
                                          const void *d_weight, int32_t bias_type,
                                          const void *d_bias, int32_t target_bits,
                                          const void *d_targets, int64_t ignore_index,
                                          const float *d_lse, int64_t dx_stride, void *d_dx,
                                          int32_t dweight_type, int64_t dweight_stride,
                                          void *d_dweight, void *d_dbias, void *d_work,
                                          size_t work_bytes) {
  return sporder_linear_cross_entropy_grad_of_loss(
      stream, type, rows, dim, classes, grad_stride, d_grad, x_stride, d_x, weight_stride, d_weight,
      bias_type, d_bias, target_bits, d_targets, ignore_index, d_lse, nullptr, dx_stride, d_dx,
      dweight_type, dweight_stride, d_dweight, d_dbias, d_work, work_bytes);
}

} // extern "C"
