// embedding.hip -- rows of a table by token, and the table's gradient.
//
//   out[t] = scale table[tokens[t]]
//   dtable[v] = scale sum of grad[t] over the t with tokens[t] = v
//
// Both move memory and compute next to nothing.  The gradient is a sum over
// equal tokens in 32 bits, written once for every row of the table (zero rows
// too).  Atomic additions would be one launch, but their order, and with it
// the result, changes from run to run and a common token serialises them, so
// the tokens are sorted instead, as far as the sums need it:
//
//   1. each tile of 4096 tokens is sorted in LDS (stable), and the table's
//      rows, cut into spans, find where their tokens begin in it.  16 to 64
//      neighbours of one token in that order (a common token: a hub) become
//      one entry,
//   2. whose sum a group of lanes forms;
//   3. a workgroup per span gathers its entries from every tile, in the
//      tiles' order, sorts them by row in LDS and adds up and writes each row.
//
// A few tokens need no tiles: each span picks its own from all of them, in
// one launch.
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
constexpr int kChunk = kWave;     // sorted neighbours looked at together
constexpr int kTileChunks = kTile / kChunk;
constexpr int kRun = 16;          // equal tokens of a chunk that become one entry
constexpr int kChunkRuns = kChunk / kRun;
constexpr int kTileRuns = kTileChunks * kChunkRuns;
constexpr uint32_t kSummed = 0x80000000u; // an entry that is a run's sum
constexpr int kSpanMost = 256;    // table rows per span
constexpr int kListMost = 2048;   // a span's entries that fit the list in LDS
constexpr int kAlone = 32;        // entries of a row that one group of lanes adds up

struct GradArgs {
  const void *grad, *tokens;
  void *out;
  int64_t count, rows, dim, grad_stride, out_stride, padding;
  float scale;
  int wide;
  int key_bits;
  int span;      // table rows per workgroup of the last launch
  int64_t spans; // ceil(rows / span)
  int64_t tiles; // 0: spans read the tokens themselves
  uint32_t *keys;      // [tiles][kTile] the tiles' entries: row,
  uint32_t *sources;   // and token index, or run index | kSummed
  uint16_t *order;     // [tiles][kTile] the sorted order within the tile
  uint16_t *runs;      // [tiles][kTileRuns] first place in the chunk and length; 0: none
  uint16_t *starts;    // [tiles][spans + 1] first entry of each span
  float *sums;         // [tiles * kTileRuns][dim]
};

// The table rows of tokens first, first + step, ... before a.count; `rows`
// (none) for padding, ids outside and places past the end.
template <int N>
__device__ __forceinline__ void token_rows(const GradArgs &a, int64_t first, int64_t step,
                                           uint32_t (&row)[N]) {
  int64_t t[N];
  auto load = [&](auto *tokens) {
#pragma unroll
    for (int k = 0; k < N; ++k) t[k] = first + k * step < a.count ? tokens[first + k * step] : -1;
  };
  if (a.wide)
    load(static_cast<const int64_t *>(a.tokens));
  else
    load(static_cast<const int32_t *>(a.tokens));
#pragma unroll
  for (int k = 0; k < N; ++k)
    row[k] = static_cast<uint32_t>(t[k] >= 0 && t[k] < a.rows && t[k] != a.padding ? t[k] : a.rows);
}

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
  __shared__ int chunk_entries[kTileChunks];
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const uint64_t below = (uint64_t(1) << lane) - 1;
  const int64_t tile = blockIdx.x, base = tile * kTile;
  const uint32_t none = static_cast<uint32_t>(a.rows); // sorted last, dropped

  uint32_t row[kTileRounds];
  token_rows(a, base + tid, kTileBlock, row);
#pragma unroll
  for (int r = 0; r < kTileRounds; ++r) {
    const int i = r * kTileBlock + tid;
    key[0][i] = row[r];
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

  // Entries: a run of kRun or more equal rows within a chunk is one, held by
  // the run's first lane; every other token is its own.
  uint64_t held[kTileRounds]; // lanes that hold an entry
  uint64_t heads[kTileRounds]; // of them, those whose entry is a run
#pragma unroll
  for (int r = 0; r < kTileRounds; ++r) {
    const int chunk = wave * kTileRounds + r;
    const uint32_t k = key[from][chunk * kChunk + lane];
    const uint32_t before = __shfl_up(k, 1);
    const uint64_t first = ballot(lane == 0 || k != before); // of each run
    const int begin = 63 - __clzll(first & (below | (uint64_t(1) << lane)));
    const uint64_t above = lane == 63 ? 0 : first >> (lane + 1);
    const int end = above ? lane + 1 + __builtin_ctzll(above) : kChunk;
    const bool run = k != none && end - begin >= kRun;
    heads[r] = ballot(run && lane == begin);
    held[r] = ballot(k != none && (!run || lane == begin));
    if (lane == 0) chunk_entries[chunk] = __popcll(held[r]);
    a.order[base + chunk * kChunk + lane] = idx[from][chunk * kChunk + lane];
    uint16_t *const runs = a.runs + tile * kTileRuns + chunk * kChunkRuns;
    if (run && lane == begin)
      runs[__popcll(heads[r] & below)] = static_cast<uint16_t>(begin << 8 | (end - begin));
    if (lane < kChunkRuns && lane >= __popcll(heads[r])) runs[lane] = 0;
  }
  __syncthreads();
  const int mine = chunk_entries[lane]; // kTileChunks = kWave: every wave holds all of them
  const int place = wave_incl_scan(mine) - mine;
  const int entries = wave_sum(mine);
  const int to = from ^ 1;
#pragma unroll
  for (int r = 0; r < kTileRounds; ++r) {
    const int chunk = wave * kTileRounds + r;
    if ((held[r] >> lane) & 1) {
      const uint32_t k = key[from][chunk * kChunk + lane];
      const int at = readlane(place, chunk) + __popcll(held[r] & below);
      key[to][at] = k;
      a.keys[base + at] = k;
      a.sources[base + at] =
          (heads[r] >> lane) & 1
              ? kSummed | static_cast<uint32_t>(tile * kTileRuns + chunk * kChunkRuns +
                                                __popcll(heads[r] & below))
              : static_cast<uint32_t>(base + idx[from][chunk * kChunk + lane]);
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

// The sums of the runs, L lanes each.
template <typename T, int VEC, int L>
__global__ void __launch_bounds__(256) embedding_run_kernel(GradArgs a) {
  const int64_t run = static_cast<int64_t>(blockIdx.x) * (256 / L) + threadIdx.x / L;
  if (run >= a.tiles * kTileRuns) return;
  const int what = a.runs[run];
  if (what == 0) return;
  const int64_t tile = run / kTileRuns;
  const int n = what & 0xff;
  const uint16_t *const order =
      a.order + tile * kTile + run % kTileRuns / kChunkRuns * kChunk + (what >> 8);
  const T *const grad = static_cast<const T *>(a.grad) + tile * kTile * a.grad_stride;
  for (int64_t c = (threadIdx.x % L) * VEC; c < a.dim; c += L * VEC) {
    float acc[VEC] = {};
#pragma unroll 8
    for (int i = 0; i < n; ++i) {
      float v[VEC];
      load_f32<VEC>(grad + order[i] * a.grad_stride + c, v);
#pragma unroll
      for (int k = 0; k < VEC; ++k) acc[k] += v[k];
    }
    store_f32<VEC>(a.sums + run * a.dim + c, acc);
  }
}

// Adds rows base[at[i] & ~kSummed], i in [i, end), to acc.
template <typename T, int VEC>
__device__ __forceinline__ void add_rows(const T *base, int64_t stride, const uint32_t *at, int i,
                                         int end, float (&acc)[VEC]) {
#pragma unroll 8
  for (; i < end; ++i) {
    float v[VEC];
    load_f32<VEC>(base + (at[i] & ~kSummed) * stride, v);
#pragma unroll
    for (int k = 0; k < VEC; ++k) acc[k] += v[k];
  }
}

// One span of table rows, L lanes per row.  A row's entries are added in two
// loops, the sums and the single tokens, so that several loads of each are
// under way at once; a row of many entries (a hub) is shared by all the
// groups of the workgroup, each a contiguous part, joined through LDS.
template <typename T, typename O, int VEC, int L>
__global__ void __launch_bounds__(256) embedding_span_kernel(GradArgs a) {
  constexpr int kGroups = 256 / L;
  constexpr int kBins = 2 * kSpanMost; // sums of row r, tokens of row r
  __shared__ uint32_t source[kListMost];
  __shared__ uint32_t sorted[kListMost];
  __shared__ uint16_t local[kListMost];
  __shared__ int first[kBins + 1];
  __shared__ int next[kBins];
  __shared__ int wave_total[256 / kWave];
  __shared__ float joined[kGroups][L * VEC];
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const uint64_t below = (uint64_t(1) << lane) - 1;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * a.span;
  const int rows = static_cast<int>(min(static_cast<int64_t>(a.span), a.rows - row0));
  const uint16_t *const starts = a.starts + blockIdx.x;

  // Exclusive prefix of one count per thread; `total` gets their sum.
  auto prefix = [&](int n, int &sum) {
    const int incl = wave_incl_scan(n);
    __syncthreads(); // the totals of the call before have been read
    if (lane == kWave - 1) wave_total[wave] = incl;
    __syncthreads();
    int at = incl - n;
    sum = 0;
#pragma unroll
    for (int w = 0; w < 256 / kWave; ++w) {
      if (w < wave) at += wave_total[w];
      sum += wave_total[w];
    }
    return at;
  };
  auto append = [&](int at, uint32_t row, uint32_t what) {
    if (at >= kListMost) return;
    const int bin = 2 * static_cast<int>(row - row0) + ((what & kSummed) == 0);
    source[at] = what;
    local[at] = static_cast<uint16_t>(bin);
    atomicAdd(&next[bin], 1);
  };

  // The entries, in the tiles' order, or the tokens in theirs.
  next[tid] = next[tid + 256] = 0;
  int total = 0;
  if (a.tiles) {
    for (int64_t t0 = 0; t0 < a.tiles; t0 += 256) {
      const int64_t tile = t0 + tid;
      int lo = 0, n = 0, sum;
      if (tile < a.tiles) {
        lo = starts[tile * (a.spans + 1)];
        n = starts[tile * (a.spans + 1) + 1] - lo;
      }
      const int at = total + prefix(n, sum);
      for (int64_t i = 0, e = tile * kTile + lo; i < n; ++i) append(at + i, a.keys[e + i], a.sources[e + i]);
      total += sum;
    }
  } else {
    constexpr int kEach = kListMost / 256;
    const int64_t t0 = static_cast<int64_t>(tid) * kEach;
    uint32_t row[kEach];
    token_rows(a, t0, 1, row);
    int n = 0;
#pragma unroll
    for (int k = 0; k < kEach; ++k) n += row[k] >= row0 && row[k] < row0 + rows;
    int at = prefix(n, total);
#pragma unroll
    for (int k = 0; k < kEach; ++k)
      if (row[k] >= row0 && row[k] < row0 + rows) append(at++, row[k], static_cast<uint32_t>(t0 + k));
  }
  const bool listed = total <= kListMost;

  if (total == 0) { // rows without a token, the most of a large table
    const int64_t vecs = a.dim / VEC, all = rows * vecs;
    O *const out = static_cast<O *>(a.out) + row0 * a.out_stride;
    float zero[VEC] = {};
    if (a.out_stride == a.dim) {
      for (int64_t i = tid; i < all; i += 256) store_f32<VEC>(out + i * VEC, zero);
    } else {
      for (int64_t i = tid; i < all; i += 256)
        store_f32<VEC>(out + i / vecs * a.out_stride + i % vecs * VEC, zero);
    }
    return;
  }

  if (listed) {
    // Stable counting sort by bin: two bins per thread, then one wave places
    // the list 64 at a time.
    __syncthreads();
    const int n0 = next[2 * tid], n1 = next[2 * tid + 1];
    int sum;
    const int at = prefix(n0 + n1, sum);
    first[2 * tid] = next[2 * tid] = at;
    first[2 * tid + 1] = next[2 * tid + 1] = at + n0;
    if (tid == 255) first[kBins] = sum;
    __syncthreads();
  }
  if (listed && wave == 0) {
    for (int i0 = 0; i0 < total; i0 += kWave) {
      const bool live = i0 + lane < total;
      const uint32_t bin = live ? local[i0 + lane] : 0;
      const uint64_t peers = match_lanes(bin, 9) & ballot(live);
      const int at = next[bin] + __popcll(peers & below);
      wave_lds_order();
      if (live) {
        sorted[at] = source[i0 + lane];
        if ((peers & below) == 0) next[bin] = at + __popcll(peers);
      }
      wave_lds_order();
    }
  }
  __syncthreads();

  const int group = tid / L;
  const T *const grad = static_cast<const T *>(a.grad);
  for (int r = group; listed && r < rows; r += kGroups) {
    const int sums = first[2 * r], singles = first[2 * r + 1], end = first[2 * r + 2];
    if (end - sums > kAlone && kGroups > 1) continue;
    O *const out = static_cast<O *>(a.out) + (row0 + r) * a.out_stride;
    for (int64_t c = (tid % L) * VEC; c < a.dim; c += L * VEC) {
      float acc[VEC] = {};
      add_rows<float, VEC>(a.sums + c, a.dim, sorted, sums, singles, acc);
      add_rows<T, VEC>(grad + c, a.grad_stride, sorted, singles, end, acc);
#pragma unroll
      for (int k = 0; k < VEC; ++k) acc[k] *= a.scale;
      store_f32<VEC>(out + c, acc);
    }
  }
  if (listed && kGroups == 1) return;

  // Rows of many entries; every row where the list was too long for LDS.
  for (int r = 0; r < rows; ++r) {
    const int sums = listed ? first[2 * r] : 0, singles = listed ? first[2 * r + 1] : 0;
    const int end = listed ? first[2 * r + 2] : 0;
    if (listed && end - sums <= kAlone) continue;
    O *const out = static_cast<O *>(a.out) + (row0 + r) * a.out_stride;
    for (int64_t c0 = 0; c0 < a.dim; c0 += L * VEC) {
      const int64_t c = c0 + (tid % L) * VEC;
      float acc[VEC] = {};
      if (c < a.dim) {
        if (listed) {
          const int part = (end - sums + kGroups - 1) / kGroups;
          const int from = min(sums + group * part, end), to = min(from + part, end);
          add_rows<float, VEC>(a.sums + c, a.dim, sorted, from, min(to, singles), acc);
          add_rows<T, VEC>(grad + c, a.grad_stride, sorted, max(from, singles), to, acc);
        } else {
          const int64_t part = ceil_div64(a.tiles, kGroups);
          const int64_t last = min((group + 1) * part, a.tiles);
          const uint32_t row = static_cast<uint32_t>(row0 + r);
          for (int64_t tile = group * part; tile < last; ++tile) {
            const uint32_t *const keys = a.keys + tile * kTile;
            const uint32_t *const sources = a.sources + tile * kTile;
            int lo = starts[tile * (a.spans + 1)];
            const int stop = starts[tile * (a.spans + 1) + 1];
            for (int hi = stop; lo < hi;) {
              const int mid = (lo + hi) / 2;
              if (keys[mid] < row)
                lo = mid + 1;
              else
                hi = mid;
            }
            for (; lo < stop && keys[lo] == row; ++lo) {
              if (sources[lo] & kSummed)
                add_rows<float, VEC>(a.sums + c, a.dim, sources, lo, lo + 1, acc);
              else
                add_rows<T, VEC>(grad + c, a.grad_stride, sources, lo, lo + 1, acc);
            }
          }
        }
      }
      __syncthreads(); // the columns before have been read
#pragma unroll
      for (int k = 0; k < VEC; ++k) joined[group][(tid % L) * VEC + k] = acc[k];
      __syncthreads();
      if (group == 0 && c < a.dim) {
        for (int g = 1; g < kGroups; ++g) {
#pragma unroll
          for (int k = 0; k < VEC; ++k) acc[k] += joined[g][(tid % L) * VEC + k];
        }
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[k] *= a.scale;
        store_f32<VEC>(out + c, acc);
      }
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
  size_t keys, sources, order, runs, starts, sums, bytes;
};

// Table rows per span: enough spans to fill the card several times over, and
// at most kSpanMost rows each.  Up to kListMost tokens fit every span's list
// whole, and need no tiles.
GradLayout grad_layout(int64_t count, int64_t rows, int64_t dim) {
  GradLayout l{};
  l.span = static_cast<int>(std::clamp<int64_t>(rows / 2048, 1, kSpanMost));
  l.spans = ceil_div64(rows, l.span);
  if (count <= kListMost) return l;
  l.tiles = ceil_div64(count, kTile);
  size_t at = 0;
  auto take = [&](size_t elems, size_t size) {
    const size_t here = at;
    at += Workspace::align(elems * size);
    return here;
  };
  const size_t tiles = static_cast<size_t>(l.tiles);
  l.keys = take(tiles * kTile, sizeof(uint32_t));
  l.sources = take(tiles * kTile, sizeof(uint32_t));
  l.order = take(tiles * kTile, sizeof(uint16_t));
  l.runs = take(tiles * kTileRuns, sizeof(uint16_t));
  l.starts = take(tiles * (l.spans + 1), sizeof(uint16_t));
  l.sums = take(tiles * kTileRuns * dim, sizeof(float));
  l.bytes = at;
  return l;
}

template <typename T, typename O, int VEC, int L>
int32_t run_grad(const GradArgs &a, void *stream) {
  if (a.tiles > 0) {
    int32_t rc = launch(embedding_tile_kernel, dim3(a.tiles), dim3(kTileBlock), stream, a);
    if (rc != SPORDER_OK) return rc;
    rc = launch(embedding_run_kernel<T, VEC, L>, dim3(ceil_div64(a.tiles * kTileRuns, 256 / L)),
                dim3(256), stream, a);
    if (rc != SPORDER_OK) return rc;
  }
  return launch(embedding_span_kernel<T, O, VEC, L>, dim3(a.spans), dim3(256), stream, a);
}

template <typename T, typename O, int VEC>
int32_t grad_vec(const GradArgs &a, void *stream) {
  const int64_t vecs = ceil_div64(a.dim, VEC);
  if (vecs <= 8) return run_grad<T, O, VEC, 8>(a, stream);
  if (vecs <= 32) return run_grad<T, O, VEC, 32>(a, stream);
  if (vecs <= 256) return run_grad<T, O, VEC, 64>(a, stream);
  return run_grad<T, O, VEC, 256>(a, stream);
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
// 2^32 threads, and the runs' launch takes up to 16 per token.
constexpr int64_t kMostRows = (int64_t(1) << 31) - 2;
constexpr int64_t kMostTokens = (int64_t(1) << 28) - kTile;

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
  if (count > 0 && (!d_grad || !d_tokens)) return SPORDER_BAD_ARGUMENT;
  const GradLayout l = grad_layout(count, rows, dim);
  if (l.bytes > 0 && (!d_work || !aligned_to(d_work, 256) || work_bytes < l.bytes))
    return SPORDER_BAD_ARGUMENT;
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
                   reinterpret_cast<uint16_t *>(w + l.runs),
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
