// embedding.hip -- rows of a table by token, and the table's gradient.
//
//   out[t] = scale table[tokens[t]]
//   dtable[v] = scale sum of grad[t] over the t with tokens[t] = v
//
// Both move memory and compute next to nothing.  The gradient is a sum over
// equal tokens in the order of t, in 32 bits, written once for every row of
// the table (zero rows too).  Atomic additions would be one launch, but their
// order, and with it the result, changes from run to run and a common token
// serialises them, so the tokens are sorted instead, as far as the sums need
// it and in two launches:
//
//   1. each tile of 4096 tokens is sorted in LDS (stable), and the table's
//      rows, cut into spans, find where their tokens begin in it.  64
//      neighbours of one token in that order (a common token: a hub, padding
//      that is not left out) become one entry,
//   2. whose sum a wave forms;
//   3. a workgroup per span gathers its entries from every tile, in the
//      tiles' order, which is the order of t, sorts them by row in LDS and
//      adds up and writes each row.
#include <algorithm>

#include "dense.hpp"

namespace sporder_hip {

namespace {

constexpr int64_t kMostBlocks = int64_t(1) << 20; // of a launch whose workgroups take turns

// ---- lookup --------------------------------------------------------------------

__device__ __forceinline__ int64_t token_at(const void *tokens, int wide, int64_t i) {
  return wide ? static_cast<const int64_t *>(tokens)[i] : static_cast<const int32_t *>(tokens)[i];
}

struct LookupArgs {
  const void *table, *tokens;
  void *out;
  int64_t count, rows, dim, table_stride, out_stride;
  float scale;
  int wide;
};

// L lanes per token.  A token outside the table gives a row of NaN (row 0 is
// read in its place), so that a wrong id cannot pass for a vector.
template <typename T, int VEC, int L>
__global__ void __launch_bounds__(256) embedding_kernel(LookupArgs a) {
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * (256 / L) + threadIdx.x / L; t < a.count;
       t += static_cast<int64_t>(gridDim.x) * (256 / L)) {
    const int64_t id = token_at(a.tokens, a.wide, t);
    const bool known = id >= 0 && id < a.rows;
    const T *const from = static_cast<const T *>(a.table) + (known ? id : 0) * a.table_stride;
    T *const to = static_cast<T *>(a.out) + t * a.out_stride;
    const float scale = known ? a.scale : __builtin_nanf("");
#pragma unroll 4
    for (int64_t c = (threadIdx.x % L) * VEC; c < a.dim; c += L * VEC) {
      float v[VEC];
      load_f32<VEC>(from + c, v);
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] *= scale;
      store_f32<VEC>(to + c, v);
    }
  }
}

// ---- gradient ------------------------------------------------------------------

constexpr int kTile = 4096;       // tokens sorted by one workgroup
constexpr int kTileBlock = 1024;
constexpr int kTileWaves = kTileBlock / kWave;
constexpr int kTileRounds = kTile / kTileBlock;
constexpr int kChunk = kWave;     // sorted neighbours that may become one entry
constexpr int kTileChunks = kTile / kChunk;
constexpr uint32_t kSummed = 0x80000000u; // an entry that is a chunk's sum
constexpr int kSpanMost = 256;    // table rows per span
constexpr int kListMost = 4096;   // a span's entries that fit the list in LDS

struct GradArgs {
  const void *grad, *tokens;
  void *out;
  int64_t count, rows, dim, grad_stride, out_stride, padding;
  float scale;
  int wide;
  int key_bits;
  int span;      // table rows per workgroup of the last launch
  int64_t spans; // ceil(rows / span)
  int64_t tiles;
  uint32_t *keys;      // [tiles][kTile] the tiles' entries: row,
  uint32_t *sources;   // and token index, or chunk index | kSummed
  uint16_t *order;     // [tiles][kTile] the sorted order within the tile
  uint64_t *uniform;   // [tiles] chunks that are one entry
  uint16_t *starts;    // [tiles][spans + 1] first entry of each span
  float *sums;         // [tiles * kTileChunks][dim]
};

// Peers of this lane: the lanes whose `bits` low bits of `digit` equal its own.
__device__ __forceinline__ uint64_t match_lanes(uint32_t digit, int bits) {
  uint64_t peers = ~uint64_t(0);
  for (int b = 0; b < bits; ++b) {
    const bool bit = (digit >> b) & 1;
    const uint64_t m = ballot(bit);
    peers &= bit ? m : ~m;
  }
  return peers;
}

// Sorts one tile by row (LSD, 8 bits per pass; each wave ranks its own 256
// consecutive items) and writes its entries and the spans' starts.
__global__ void __launch_bounds__(kTileBlock) embedding_tile_kernel(GradArgs a) {
  constexpr int kDigits = 256;
  __shared__ uint32_t key[2][kTile];
  __shared__ uint16_t idx[2][kTile];
  __shared__ uint16_t cnt[kTileWaves][kDigits];
  __shared__ int wave_total[kTileWaves];
  __shared__ int chunk_size[kTileChunks];
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const uint64_t below = (uint64_t(1) << lane) - 1;
  const int64_t tile = blockIdx.x, base = tile * kTile;

#pragma unroll
  for (int r = 0; r < kTileRounds; ++r) {
    const int i = r * kTileBlock + tid;
    uint32_t k = static_cast<uint32_t>(a.rows); // no row: sorted last, dropped
    if (base + i < a.count) {
      const int64_t t = token_at(a.tokens, a.wide, base + i);
      if (t >= 0 && t < a.rows && t != a.padding) k = static_cast<uint32_t>(t);
    }
    key[0][i] = k;
    idx[0][i] = static_cast<uint16_t>(i);
  }
  __syncthreads();

  int from = 0;
  for (int shift = 0; shift < a.key_bits; shift += 8, from ^= 1) {
    const int bits = min(8, a.key_bits - shift);
    for (int i = tid; i < kTileWaves * kDigits / 2; i += kTileBlock)
      reinterpret_cast<uint32_t *>(cnt)[i] = 0;
    __syncthreads();
    int rank[kTileRounds];
#pragma unroll
    for (int r = 0; r < kTileRounds; ++r) {
      const int i = (wave * kTileRounds + r) * kWave + lane;
      const uint32_t d = (key[from][i] >> shift) & (kDigits - 1);
      const uint64_t peers = match_lanes(d, bits);
      rank[r] = cnt[wave][d] + __popcll(peers & below);
      wave_lds_order();
      if ((peers & below) == 0) cnt[wave][d] = static_cast<uint16_t>(rank[r] + __popcll(peers));
      wave_lds_order();
    }
    __syncthreads();
    // cnt[w][d] becomes the place of wave w's first item of digit d.
    int total = 0;
    if (tid < kDigits) {
#pragma unroll
      for (int w = 0; w < kTileWaves; ++w) {
        const int c = cnt[w][tid];
        cnt[w][tid] = static_cast<uint16_t>(total);
        total += c;
      }
      const int incl = wave_incl_scan(total);
      if (lane == kWave - 1) wave_total[wave] = incl;
      total = incl - total;
    }
    __syncthreads();
    if (tid < kDigits) {
      for (int w = 0; w < wave; ++w) total += wave_total[w];
#pragma unroll
      for (int w = 0; w < kTileWaves; ++w) cnt[w][tid] = static_cast<uint16_t>(cnt[w][tid] + total);
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kTileRounds; ++r) {
      const int i = (wave * kTileRounds + r) * kWave + lane;
      const uint32_t k = key[from][i];
      const int to = cnt[wave][(k >> shift) & (kDigits - 1)] + rank[r];
      key[from ^ 1][to] = k;
      idx[from ^ 1][to] = idx[from][i];
    }
    __syncthreads();
  }

  // Entries: a chunk of one row is one, any other chunk its tokens.
  const uint32_t none = static_cast<uint32_t>(a.rows);
#pragma unroll
  for (int r = 0; r < kTileRounds; ++r) {
    const int chunk = wave * kTileRounds + r;
    const uint32_t k = key[from][chunk * kChunk + lane];
    const bool one = ballot(k == static_cast<uint32_t>(readlane(k, 0))) == ~uint64_t(0);
    const int valid = __popcll(ballot(k != none));
    if (lane == 0) chunk_size[chunk] = one && valid ? -1 : valid;
    a.order[base + chunk * kChunk + lane] = idx[from][chunk * kChunk + lane];
  }
  __syncthreads();
  const int mine = chunk_size[lane]; // kTileChunks = kWave: every wave holds all of them
  const int place = wave_incl_scan(mine < 0 ? 1 : mine) - (mine < 0 ? 1 : mine);
  const int entries = wave_sum(mine < 0 ? 1 : mine);
  const uint64_t uniform = ballot(mine < 0);
  if (tid == 0) a.uniform[tile] = uniform;
  const int to = from ^ 1;
#pragma unroll
  for (int r = 0; r < kTileRounds; ++r) {
    const int chunk = wave * kTileRounds + r;
    const uint32_t k = key[from][chunk * kChunk + lane];
    const uint32_t i = idx[from][chunk * kChunk + lane];
    const int at = readlane(place, chunk);
    const bool one = (uniform >> chunk) & 1;
    if (one ? lane == 0 : k != none) {
      key[to][at + lane] = k;
      a.keys[base + at + lane] = k;
      a.sources[base + at + lane] =
          one ? kSummed | static_cast<uint32_t>(tile * kTileChunks + chunk)
              : static_cast<uint32_t>(base + i);
    }
  }
  __syncthreads();
  for (int64_t s = tid; s <= a.spans; s += kTileBlock) {
    const int64_t row = s * a.span;
    int lo = 0, hi = entries;
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (key[to][mid] < row)
        lo = mid + 1;
      else
        hi = mid;
    }
    a.starts[tile * (a.spans + 1) + s] = static_cast<uint16_t>(lo);
  }
}

// The sums of the chunks that are one entry: a workgroup per chunk and slice
// of columns, four waves over the slice's vectors.
template <typename T, int VEC>
__global__ void __launch_bounds__(256) embedding_chunk_kernel(GradArgs a) {
  const int64_t tile = blockIdx.x / kTileChunks;
  const int chunk = blockIdx.x % kTileChunks;
  if (!((a.uniform[tile] >> chunk) & 1)) return;
  __shared__ uint16_t place[kChunk];
  if (threadIdx.x < kChunk) place[threadIdx.x] = a.order[tile * kTile + chunk * kChunk + threadIdx.x];
  __syncthreads();
  const int64_t c = (static_cast<int64_t>(blockIdx.y) * 256 + threadIdx.x) * VEC;
  if (c >= a.dim) return;
  const T *const grad = static_cast<const T *>(a.grad) + tile * kTile * a.grad_stride + c;
  float acc[VEC] = {};
#pragma unroll 8
  for (int i = 0; i < kChunk; ++i) {
    float v[VEC];
    load_f32<VEC>(grad + place[i] * a.grad_stride, v);
#pragma unroll
    for (int k = 0; k < VEC; ++k) acc[k] += v[k];
  }
  store_f32<VEC>(a.sums + static_cast<int64_t>(blockIdx.x) * a.dim + c, acc);
}

template <typename T, int VEC>
__device__ __forceinline__ void add_entry(const GradArgs &a, uint32_t source, int64_t c,
                                          float (&acc)[VEC]) {
  float v[VEC];
  if (source & kSummed)
    load_f32<VEC>(a.sums + static_cast<int64_t>(source & ~kSummed) * a.dim + c, v);
  else
    load_f32<VEC>(static_cast<const T *>(a.grad) + source * a.grad_stride + c, v);
#pragma unroll
  for (int k = 0; k < VEC; ++k) acc[k] += v[k];
}

// One span of table rows.  L lanes per row.
template <typename T, typename O, int VEC, int L>
__global__ void __launch_bounds__(256) embedding_span_kernel(GradArgs a) {
  constexpr int kGroups = 256 / L;
  __shared__ uint32_t source[kListMost];
  __shared__ uint32_t sorted[kListMost];
  __shared__ uint8_t local[kListMost];
  __shared__ int first[kSpanMost + 1];
  __shared__ int next[kSpanMost];
  __shared__ int wave_total[256 / kWave];
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * a.span;
  const int rows = static_cast<int>(min(static_cast<int64_t>(a.span), a.rows - row0));
  const uint16_t *const starts = a.starts + blockIdx.x;

  // The entries, in the tiles' order.
  for (int i = tid; i < kSpanMost; i += 256) next[i] = 0;
  int total = 0;
  for (int64_t t0 = 0; t0 < a.tiles; t0 += 256) {
    const int64_t tile = t0 + tid;
    int lo = 0, n = 0;
    if (tile < a.tiles) {
      lo = starts[tile * (a.spans + 1)];
      n = starts[tile * (a.spans + 1) + 1] - lo;
    }
    const int incl = wave_incl_scan(n);
    __syncthreads(); // the totals of the round before have been read
    if (lane == kWave - 1) wave_total[wave] = incl;
    __syncthreads();
    int at = total + incl - n;
    for (int w = 0; w < 256 / kWave; ++w) {
      if (w < wave) at += wave_total[w];
      total += wave_total[w];
    }
    for (int i = 0; i < n && at + i < kListMost; ++i) {
      const int64_t e = tile * kTile + lo + i;
      const int r = static_cast<int>(a.keys[e] - row0);
      source[at + i] = a.sources[e];
      local[at + i] = static_cast<uint8_t>(r);
      atomicAdd(&next[r], 1);
    }
  }
  __syncthreads();
  const bool listed = total <= kListMost;

  if (listed) {
    // Stable counting sort by row: one wave places the list 64 at a time.
    if (wave == 0) {
      int carry = 0;
      for (int r = lane; r < kSpanMost; r += kWave) {
        const int n = next[r], incl = wave_incl_scan(n);
        first[r] = carry + incl - n;
        next[r] = carry + incl - n;
        carry += readlane(incl, kWave - 1);
      }
      if (lane == 0) first[kSpanMost] = carry;
      wave_lds_order();
      const uint64_t below = (uint64_t(1) << lane) - 1;
      for (int i0 = 0; i0 < total; i0 += kWave) {
        const bool live = i0 + lane < total;
        const uint32_t r = live ? local[i0 + lane] : 0;
        const uint64_t peers = match_lanes(r, 8) & ballot(live);
        if (live) {
          const int at = next[r] + __popcll(peers & below);
          sorted[at] = source[i0 + lane];
          wave_lds_order();
          if ((peers & below) == 0) next[r] = at + __popcll(peers);
        }
        wave_lds_order();
      }
    }
    __syncthreads();
  }

  const int group = tid / L;
  for (int r = group; r < rows; r += kGroups) {
    O *const out = static_cast<O *>(a.out) + (row0 + r) * a.out_stride;
    for (int64_t c = (tid % L) * VEC; c < a.dim; c += L * VEC) {
      float acc[VEC] = {};
      if (listed) {
        const int end = first[r + 1];
#pragma unroll 4
        for (int e = first[r]; e < end; ++e) add_entry<T, VEC>(a, sorted[e], c, acc);
      } else {
        for (int64_t tile = 0; tile < a.tiles; ++tile) {
          const uint16_t *const s = starts + tile * (a.spans + 1);
          const uint32_t *const keys = a.keys + tile * kTile;
          const uint32_t row = static_cast<uint32_t>(row0 + r);
          int lo = s[0], hi = s[1];
          const int end = hi;
          while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (keys[mid] < row)
              lo = mid + 1;
            else
              hi = mid;
          }
          for (; lo < end && keys[lo] == row; ++lo)
            add_entry<T, VEC>(a, a.sources[tile * kTile + lo], c, acc);
        }
      }
#pragma unroll
      for (int k = 0; k < VEC; ++k) acc[k] *= a.scale;
      store_f32<VEC>(out + c, acc);
    }
  }
}

// ---- host ----------------------------------------------------------------------

template <typename T, int VEC, int L> int32_t run_lookup(const LookupArgs &a, void *stream) {
  return launch(embedding_kernel<T, VEC, L>, dim3(std::min(ceil_div64(a.count, 256 / L), kMostBlocks)),
                dim3(256), stream, a);
}

// Lanes per row: a row of a few vectors leaves the rest of the wave to others.
template <typename T, int VEC> int32_t pick_lookup(const LookupArgs &a, void *stream) {
  const int64_t vecs = ceil_div64(a.dim, VEC);
  if (vecs <= 8) return run_lookup<T, VEC, 8>(a, stream);
  if (vecs <= 32) return run_lookup<T, VEC, 32>(a, stream);
  if (vecs <= 256) return run_lookup<T, VEC, 64>(a, stream);
  return run_lookup<T, VEC, 256>(a, stream);
}

template <typename T> int32_t lookup_typed(const LookupArgs &a, void *stream) {
  const int vec = row_vec(sizeof(T), a.dim, {a.table_stride, a.out_stride}, {a.table, a.out});
  if constexpr (sizeof(T) == 2) {
    if (vec == 8) return pick_lookup<T, 8>(a, stream);
  }
  if (vec == 4) return pick_lookup<T, 4>(a, stream);
  return pick_lookup<T, 1>(a, stream);
}

struct GradLayout {
  int span;
  int64_t spans, tiles;
  size_t keys, sources, order, uniform, starts, sums, bytes;
};

// Table rows per span: enough spans to fill the card several times over, and
// at most kSpanMost rows each.
GradLayout grad_layout(int64_t count, int64_t rows, int64_t dim) {
  GradLayout l{};
  l.span = static_cast<int>(std::clamp<int64_t>(rows / 2048, 1, kSpanMost));
  l.spans = ceil_div64(rows, l.span);
  l.tiles = ceil_div64(count, kTile);
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += Workspace::align(bytes);
    return here;
  };
  l.keys = take(static_cast<size_t>(l.tiles) * kTile * sizeof(uint32_t));
  l.sources = take(static_cast<size_t>(l.tiles) * kTile * sizeof(uint32_t));
  l.order = take(static_cast<size_t>(l.tiles) * kTile * sizeof(uint16_t));
  l.uniform = take(static_cast<size_t>(l.tiles) * sizeof(uint64_t));
  l.starts = take(static_cast<size_t>(l.tiles) * (l.spans + 1) * sizeof(uint16_t));
  l.sums = take(static_cast<size_t>(l.tiles) * kTileChunks * dim * sizeof(float));
  l.bytes = at;
  return l;
}

template <typename T, typename O, int VEC, int L>
int32_t run_span(const GradArgs &a, void *stream) {
  return launch(embedding_span_kernel<T, O, VEC, L>, dim3(a.spans), dim3(256), stream, a);
}

template <typename T, typename O, int VEC>
int32_t grad_vec(const GradArgs &a, void *stream) {
  if (a.tiles > 0) {
    int32_t rc = launch(embedding_tile_kernel, dim3(a.tiles), dim3(kTileBlock), stream, a);
    if (rc != SPORDER_OK) return rc;
    rc = launch(embedding_chunk_kernel<T, VEC>,
                dim3(a.tiles * kTileChunks, ceil_div64(a.dim, 256 * VEC)), dim3(256), stream, a);
    if (rc != SPORDER_OK) return rc;
  }
  const int64_t vecs = ceil_div64(a.dim, VEC);
  if (vecs <= 8) return run_span<T, O, VEC, 8>(a, stream);
  if (vecs <= 32) return run_span<T, O, VEC, 32>(a, stream);
  if (vecs <= 256) return run_span<T, O, VEC, 64>(a, stream);
  return run_span<T, O, VEC, 256>(a, stream);
}

template <typename T, typename O> int32_t grad_typed(const GradArgs &a, void *stream) {
  const int vec = row_vec(sizeof(O), a.dim, {a.grad_stride, a.out_stride}, {a.grad, a.out});
  if constexpr (sizeof(O) == 2) {
    if (vec == 8) return grad_vec<T, O, 8>(a, stream);
  }
  if (vec == 4) return grad_vec<T, O, 4>(a, stream);
  return grad_vec<T, O, 1>(a, stream);
}

// Rows count in 31 bits with one value over (no row); a launch has fewer than
// 2^32 threads, and the chunks' launch takes four per token.
constexpr int64_t kMostRows = (int64_t(1) << 31) - 2;
constexpr int64_t kMostTokens = (int64_t(1) << 30) - kTile;

} // namespace

} // namespace sporder_hip

using namespace sporder_hip;

extern "C" {

int32_t sporder_embedding(void *stream, int32_t type, int64_t rows, int64_t dim,
                          int64_t table_stride, const void *d_table, int64_t count,
                          int32_t token_bits, const void *d_tokens, float scale,
                          int64_t out_stride, void *d_out) {
  if (!type_known(type) || rows < 1 || dim < 1 || dim > kMostDim || count < 0 ||
      table_stride < 0 ||
      (count > 1 && out_stride < dim) || (token_bits != 32 && token_bits != 64))
    return SPORDER_BAD_ARGUMENT;
  if (count == 0) return SPORDER_OK;
  if (!d_table || !d_tokens || !d_out) return SPORDER_BAD_ARGUMENT;
  const LookupArgs a{d_table, d_tokens,     d_out,      count, rows,
                     dim,     table_stride, out_stride, scale, token_bits == 64};
  if (type == SPORDER_TYPE_BF16) return lookup_typed<bf16_t>(a, stream);
  if (type == SPORDER_TYPE_F16) return lookup_typed<f16_t>(a, stream);
  return lookup_typed<float>(a, stream);
}

size_t sporder_embedding_grad_work_bytes(int64_t count, int64_t rows, int64_t dim) {
  if (count < 1 || rows < 1 || dim < 1 || dim > kMostDim) return 0;
  return grad_layout(count, rows, dim).bytes;
}

int32_t sporder_embedding_grad(void *stream, int32_t type, int64_t count, int64_t dim,
                               int64_t grad_stride, const void *d_grad, int32_t token_bits,
                               const void *d_tokens, float scale, int64_t padding_idx,
                               int64_t rows, int32_t out_type, int64_t out_stride, void *d_out,
                               void *d_work, size_t work_bytes) {
  if (!type_known(type) || (out_type != type && out_type != SPORDER_TYPE_F32) || rows < 1 ||
      rows > kMostRows || dim < 1 || dim > kMostDim || count < 0 || count > kMostTokens || grad_stride < 0 ||
      (rows > 1 && out_stride < dim) || (token_bits != 32 && token_bits != 64) || !d_out)
    return SPORDER_BAD_ARGUMENT;
  if (count > 0 && (!d_grad || !d_tokens || !d_work || !aligned_to(d_work, 256) ||
                    work_bytes < sporder_embedding_grad_work_bytes(count, rows, dim)))
    return SPORDER_BAD_ARGUMENT;
  const GradLayout l = grad_layout(count, rows, dim);
  char *const w = static_cast<char *>(d_work);
  const GradArgs a{d_grad,
                   d_tokens,
                   d_out,
                   count,
                   rows,
                   dim,
                   grad_stride,
                   out_stride,
                   padding_idx,
                   scale,
                   token_bits == 64,
                   bits_for(rows),
                   l.span,
                   l.spans,
                   l.tiles,
                   reinterpret_cast<uint32_t *>(w + l.keys),
                   reinterpret_cast<uint32_t *>(w + l.sources),
                   reinterpret_cast<uint16_t *>(w + l.order),
                   reinterpret_cast<uint64_t *>(w + l.uniform),
                   reinterpret_cast<uint16_t *>(w + l.starts),
                   reinterpret_cast<float *>(w + l.sums)};
  if (type == SPORDER_TYPE_F32) return grad_typed<float, float>(a, stream);
  if (type == SPORDER_TYPE_BF16)
    return out_type == type ? grad_typed<bf16_t, bf16_t>(a, stream)
                            : grad_typed<bf16_t, float>(a, stream);
  return out_type == type ? grad_typed<f16_t, f16_t>(a, stream)
                          : grad_typed<f16_t, float>(a, stream);
}

} // extern "C"
