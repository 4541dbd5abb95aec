// embedding.hip -- rows of a table by token, and the table's gradient.
//
//   out[t] = scale table[tokens[t]]
//   dtable[v] = scale sum of grad[t] over the t with tokens[t] = v
//
// Both move memory and compute next to nothing.  The gradient is a sum over
// equal tokens in 32 bits, written once for every row of the table (zero rows
// too).  Atomic additions would be one launch, but their order, and with it
// the result, changes from run to run and a common token serialises them, so
// the tokens are sorted instead:
//
//   1. each tile of 1024 or 4096 tokens is sorted in LDS (stable), and the
//      table's rows, cut into spans, find where their tokens begin in it.  16
//      to 64 neighbours of one token in that order (a common token: a hub)
//      become one entry,
//   2. whose sum a workgroup forms; in the same launch a workgroup per span
//      gathers its entries from every tile, in the tiles' order, sorts them by
//      row in LDS and writes them out by row;
//   3. the table is written front to back, every lane a few vectors of a row
//      and their sum (this is where the bytes are); rows that still have many
//      entries are shared by a workgroup for each slice of their columns, in
//      the launch's first workgroups.
//
// Few tokens need no tiles: each span picks its own from all of them and sums
// its rows, in one launch.  A large table of few tokens is zeroed at the speed
// of a fill, then a workgroup per token finds its equals and sums their row.
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
  bool stream;
  int64_t row_block; // tokens per workgroup and turn
};

// The vectors of a.row_block rows lie in a row before the workgroup's lanes,
// kItems of them 256 apart per lane and turn: stores fill whole lines whatever
// the row's length, and a lane has kItems rows under way.  A token outside the
// table gives a row of NaN (row 0 is read in its place), so that a wrong id
// cannot pass for a vector.  Bound by memory: 65,536 rows of 2,048 16-bit
// elements of 50,000 in 60 us, 268 MB written at 4.5 TB/s beside the reads.
constexpr int lookup_items(int vec) { return vec == 1 ? 8 : 4; }

template <typename T, int VEC> __global__ void __launch_bounds__(256) embedding_kernel(LookupArgs a) {
  constexpr int kItems = lookup_items(VEC);
  const uint32_t vecs = static_cast<uint32_t>(a.dim / VEC);
  const T *const table = static_cast<const T *>(a.table);
  for (int64_t t0 = static_cast<int64_t>(blockIdx.x) * a.row_block; t0 < a.count;
       t0 += static_cast<int64_t>(gridDim.x) * a.row_block) {
    const uint32_t rows = static_cast<uint32_t>(min(static_cast<int64_t>(a.row_block), a.count - t0));
    const uint32_t all = rows * vecs; // at most kMostDim, or a few thousand
    T *const out = static_cast<T *>(a.out) + t0 * a.out_stride;
    for (uint32_t q0 = threadIdx.x; q0 < all; q0 += 256 * kItems) {
      uint32_t t[kItems], c[kItems];
      int64_t id[kItems];
#pragma unroll
      for (int u = 0; u < kItems; ++u) {
        const uint32_t q = min(q0 + 256 * u, all - 1);
        t[u] = q / vecs;
        c[u] = (q - t[u] * vecs) * VEC;
      }
      auto fetch = [&](auto *tokens) {
#pragma unroll
        for (int u = 0; u < kItems; ++u) id[u] = tokens[t0 + t[u]];
      };
      if (a.wide)
        fetch(static_cast<const int64_t *>(a.tokens));
      else
        fetch(static_cast<const int32_t *>(a.tokens));
      float v[kItems][VEC];
#pragma unroll
      for (int u = 0; u < kItems; ++u)
        load_f32<VEC>(table + (id[u] >= 0 && id[u] < a.rows ? id[u] : 0) * a.table_stride + c[u], v[u]);
#pragma unroll
      for (int u = 0; u < kItems; ++u) {
        const float scale = id[u] >= 0 && id[u] < a.rows ? a.scale : __builtin_nanf("");
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[u][i] *= scale;
        if (q0 + 256 * u < all) put_f32<VEC>(a.stream, out + t[u] * a.out_stride + c[u], v[u]);
      }
    }
  }
}

// ---- gradient ------------------------------------------------------------------

// Tokens sorted by one workgroup: small tiles sort in half the time, but every
// span has to ask each of them.
constexpr int kSmallTile = 1024, kLargeTile = 4096;
constexpr int kMostSmallTiles = 64;
constexpr int kTileRounds = 4;    // tokens per thread of a tile
constexpr int kChunk = kWave;     // sorted neighbours looked at together
constexpr int kRun = 16;          // equal tokens of a chunk that become one entry
constexpr uint32_t kSummed = 0x80000000u; // an entry that is a run's sum
constexpr int kSpanMost = 256;    // table rows per span
constexpr int kListMost = 2048;   // a span's entries in LDS at a time
// Few tokens need no tiles: every span looks through them by itself, in one
// launch, or a workgroup per token does where the table is large.  They are few
// by their number, by what the spans read of them, and by their elements, which
// one workgroup may have to add up alone (2 MB at most, some 25 us).
constexpr int kFewMost = 8192;
constexpr int64_t kFewReads = int64_t(1) << 24, kFewElements = int64_t(1) << 19;
// In a large table (2 million rows of 60 floats, with a workgroup per token and
// with tiles: 2,048 tokens 94 and 124 us, 8,000 184 and 130).
constexpr int kLargeFewMost = 2048;
constexpr int64_t kTokenSlices = 32; // workgroups of one token's columns, at most
constexpr int64_t kLarge = int64_t(1) << 24; // elements of a large table
constexpr int kSparse = 4;        // turns' worth of rows per workgroup, at most
constexpr int kAlone = 8;         // entries of a row that one lane adds up
constexpr int kHubLists = 16;
constexpr int kHubBlocks = 512;   // workgroups of the last launch for rows of more entries
constexpr int kRowsMost = 1024;   // table rows per workgroup of the last launch

struct GradArgs {
  const void *grad, *tokens;
  void *out;
  int64_t count, rows, dim, grad_stride, out_stride, padding;
  float scale;
  int wide;
  bool stream, large;
  int key_bits;
  int row_block; // table rows per workgroup of the last launch
  int span;      // and of the one before it
  int64_t spans; // ceil(rows / span)
  int tile;      // tokens per tile
  int64_t tiles;
  uint32_t *keys;      // [tiles][tile] the tiles' entries: row,
  uint32_t *sources;   // and token index, or run index | kSummed
  uint16_t *order;     // [tiles][tile] the sorted order within the tile
  uint32_t *runs;      // [tiles][tile / kRun] first place in the tile << 8 | length
  int32_t *run_count;  // [tiles]
  uint16_t *starts;    // [tiles][spans + 1] first entry of each span
  float *sums;         // [tiles * tile / kRun][dim]
  uint32_t *list;      // [count] the entries' sources by row, sums first
  int32_t *row_start;  // [rows + 1] first entry in the list
  // Rows of more than kAlone entries: kHubLists lists, each its length and
  // then the rows (one counter for all would have every span's atomic wait for
  // the others': 37 us of 67 with 4,250 such rows).
  int32_t *hubs;       // [kHubLists][hub_stride]
  int64_t hub_stride;
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
  uint32_t low = ~0u, high = ~0u;
  for (int b = 0; b < bits; ++b) {
    const uint32_t set = static_cast<uint32_t>(static_cast<int32_t>(digit << (31 - b)) >> 31);
    const uint64_t m = ballot(set != 0); // lanes with the bit; peers agree with this lane's
    low &= ~(static_cast<uint32_t>(m) ^ set);
    high &= ~(static_cast<uint32_t>(m >> 32) ^ set);
  }
  return static_cast<uint64_t>(high) << 32 | low;
}

// Sorts one tile by row (LSD, 8 bits per pass; each wave ranks its own 256
// consecutive items) and writes its entries and the spans' starts.  Bound by
// latency, some 3 us for each pass and 5 for the rest: 8 tiles of 1024 in 13
// us, 123 of 4096 in 23.
template <int TILE>
__global__ void __launch_bounds__(TILE / kTileRounds) embedding_tile_kernel(GradArgs a) {
  constexpr int kTile = TILE, kTileBlock = TILE / kTileRounds, kTileWaves = kTileBlock / kWave;
  constexpr int kTileChunks = kTile / kChunk, kTileRuns = kTile / kRun;
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
    // cnt[w][d] becomes the place of wave w's first item of digit d: a prefix
    // over digits, then waves, four waves of a digit per thread.
    constexpr int kPart = kTileWaves * kDigits / kTileBlock;
    const int digit = tid / (kTileWaves / kPart), w0 = tid % (kTileWaves / kPart) * kPart;
    int at[kPart], total = 0;
#pragma unroll
    for (int w = 0; w < kPart; ++w) {
      at[w] = total;
      total += cnt[w0 + w][digit];
    }
    const int incl = wave_incl_scan(total);
    if (lane == kWave - 1) wave_total[wave] = incl;
    __syncthreads();
    int before = lane < wave ? wave_total[lane] : 0; // kTileWaves of them
    before = wave_sum(before) + incl - total;
#pragma unroll
    for (int w = 0; w < kPart; ++w) cnt[w0 + w][digit] = static_cast<uint16_t>(before + at[w]);
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
  int length[kTileRounds];
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
    length[r] = end - begin;
    if (lane == 0) chunk_entries[chunk] = __popcll(held[r]) | __popcll(heads[r]) << 16;
    a.order[base + chunk * kChunk + lane] = idx[from][chunk * kChunk + lane];
  }
  __syncthreads();
  // Entries and runs before each chunk, in the halves of a word: every wave
  // holds all of the chunks, at most one per lane.
  const int mine = lane < kTileChunks ? chunk_entries[lane] : 0;
  const int place = wave_incl_scan(mine) - mine;
  const int all = wave_sum(mine), entries = all & 0xffff;
  if (tid == 0) a.run_count[tile] = all >> 16;
  if (tile == 0 && tid < kHubLists) a.hubs[tid * a.hub_stride] = 0;
  const int to = from ^ 1;
#pragma unroll
  for (int r = 0; r < kTileRounds; ++r) {
    const int chunk = wave * kTileRounds + r;
    if ((held[r] >> lane) & 1) {
      const uint32_t k = key[from][chunk * kChunk + lane];
      const int before = readlane(place, chunk);
      const int at = (before & 0xffff) + __popcll(held[r] & below);
      uint32_t what = static_cast<uint32_t>(base + idx[from][chunk * kChunk + lane]);
      if ((heads[r] >> lane) & 1) {
        const int run = (before >> 16) + __popcll(heads[r] & below);
        a.runs[tile * kTileRuns + run] = static_cast<uint32_t>((chunk * kChunk + lane) << 8 | length[r]);
        what = kSummed | static_cast<uint32_t>(tile * kTileRuns + run);
      }
      key[to][at] = k;
      a.keys[base + at] = k;
      a.sources[base + at] = what;
    }
  }
  __syncthreads();
  // Each thread takes neighbouring spans and searches on from the last start:
  // by doubling steps, then between the last two.
  const int64_t per = ceil_div64(a.spans + 1, kTileBlock);
  const int64_t last = min((tid + 1) * per, a.spans + 1);
  int lo = 0; // entries before it are below the row
  for (int64_t s = tid * per; s < last; ++s) {
    const int64_t row = s * a.span;
    int width = s == tid * per ? kTile : 1, hi;
    while ((hi = lo + width) <= entries && key[to][hi - 1] < row) {
      lo = hi;
      width *= 2;
    }
    hi = min(hi, entries + 1) - 1;
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

// The sum of run blocks: `block` of kRunBlocks(tile) for each tile and slice
// of L VEC columns, L lanes per token, 32 / VEC tokens of a lane under way at
// once.
constexpr int run_blocks(int tile) { return tile / 128; }

template <typename T, int VEC, int L>
__device__ __forceinline__ void sum_runs(const GradArgs &a, float (&joined)[4][L * VEC], int64_t block) {
  constexpr int kGroups = 256 / L, kWaves = 256 / kWave;
  constexpr int kMost = kChunk / kGroups, kEach = kMost > 32 / VEC ? 32 / VEC : kMost > 0 ? kMost : 1;
  const int per_tile = run_blocks(a.tile), slices = static_cast<int>(ceil_div64(a.dim, L * VEC));
  const int64_t tile = block / (per_tile * slices);
  const int within = static_cast<int>(block % (per_tile * slices));
  const int runs = a.run_count[tile], tile_runs = a.tile / kRun;
  const int group = threadIdx.x / L, lane = threadIdx.x % L, wave = threadIdx.x / kWave;
  const int64_t c = (static_cast<int64_t>(within / per_tile) * L + lane) * VEC;
  const T *const grad = static_cast<const T *>(a.grad) + tile * a.tile * a.grad_stride + c;
  for (int run = within % per_tile; run < runs; run += per_tile) {
    const uint32_t what = a.runs[tile * tile_runs + run];
    const int n = what & 0xff;
    const uint16_t *const order = a.order + tile * a.tile + (what >> 8);
    float acc[VEC] = {};
    for (int i0 = group; i0 < n; i0 += kEach * kGroups) {
      int64_t at[kEach];
#pragma unroll
      for (int d = 0; d < kEach; ++d) at[d] = order[min(i0 + d * kGroups, n - 1)] * a.grad_stride;
      float v[kEach][VEC] = {};
#pragma unroll
      for (int d = 0; d < kEach; ++d)
        if (c < a.dim && i0 + d * kGroups < n) load_f32<VEC>(grad + at[d], v[d]);
#pragma unroll
      for (int d = 0; d < kEach; ++d) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[k] += v[d][k];
      }
    }
    __syncthreads(); // the run before has been read
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
#pragma unroll
      for (int j = L; j < kWave; j <<= 1) acc[k] += lane_xor_f32(acc[k], j);
      if (threadIdx.x % kWave < L) joined[wave][lane * VEC + k] = acc[k];
    }
    __syncthreads();
    if (threadIdx.x < L && c < a.dim) {
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        acc[k] = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) acc[k] += joined[w][lane * VEC + k];
      }
      store_f32<VEC>(a.sums + (tile * tile_runs + run) * a.dim + c, acc);
    }
  }
}

// A span's entries in LDS.
constexpr int kBins = 2 * kSpanMost; // sums of row r, tokens of row r
__device__ __forceinline__ int entry_bin(int row, uint32_t what) {
  return 2 * row + ((what & kSummed) == 0);
}
constexpr int kSpanWaves = 256 / kWave;
template <typename SOURCE, int MOST> struct SpanList {
  SOURCE source[MOST];
  uint16_t local[MOST]; // their bins
  int first[kBins + 1];
  int next[kBins];
  int wave_total[kSpanWaves];

  // Exclusive prefix of one count per thread; `sum` gets the total.
  __device__ __forceinline__ int prefix(int n, int &sum) {
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const int incl = wave_incl_scan(n);
    __syncthreads(); // the totals of the call before have been read
    if (lane == kWave - 1) wave_total[wave] = incl;
    __syncthreads();
    int at = incl - n;
    sum = 0;
#pragma unroll
    for (int w = 0; w < kSpanWaves; ++w) {
      if (w < wave) at += wave_total[w];
      sum += wave_total[w];
    }
    return at;
  }

  __device__ __forceinline__ void clear() { next[threadIdx.x] = next[threadIdx.x + 256] = 0; }

  // From counts in next to first places, in next and first.
  __device__ __forceinline__ void open() {
    const int tid = threadIdx.x;
    __syncthreads();
    const int n0 = next[2 * tid], n1 = next[2 * tid + 1];
    int sum;
    const int at = prefix(n0 + n1, sum);
    first[2 * tid] = next[2 * tid] = at;
    first[2 * tid + 1] = next[2 * tid + 1] = at + n0;
    if (tid == 255) first[kBins] = sum;
    __syncthreads();
  }

  // Puts the first n entries of the list to their places, in order: one wave,
  // 64 at a time.
  template <typename PUT> __device__ __forceinline__ void place(int n, PUT &&put) {
    const int lane = threadIdx.x;
    if (lane < kWave) {
      const uint64_t below = (uint64_t(1) << lane) - 1;
      for (int i0 = 0; i0 < n; i0 += kWave) {
        const bool live = i0 + lane < n;
        const uint32_t b = live ? local[i0 + lane] : 0;
        const uint64_t peers = match_lanes(b, 9) & ballot(live);
        const int to = next[b] + __popcll(peers & below);
        wave_lds_order();
        if (live) {
          put(to, static_cast<uint32_t>(source[i0 + lane]));
          if ((peers & below) == 0) next[b] = to + __popcll(peers);
        }
        wave_lds_order();
      }
    }
    __syncthreads();
  }
};

// Step 2: `run_grid` workgroups for the runs, then one per span.  Latency of the
// tiles' starts and of the sort in LDS, and the rows of the runs: 12 us for
// 32,768 tokens of 50,000 rows, 41 us for 500,000 of 2.4 million.
template <typename T, int VEC, int L>
__global__ void __launch_bounds__(256) embedding_span_kernel(GradArgs a, int64_t run_grid) {
  __shared__ union {
    SpanList<uint32_t, kListMost> list;
    float joined[4][L * VEC];
  } shared;
  if (blockIdx.x < run_grid) {
    sum_runs<T, VEC, L>(a, shared.joined, blockIdx.x);
    return;
  }
  auto &list = shared.list;
  const int tid = threadIdx.x;
  const int64_t span = blockIdx.x - run_grid;
  const int64_t row0 = span * a.span;
  const int rows = static_cast<int>(min(static_cast<int64_t>(a.span), a.rows - row0));
  const uint16_t *const starts = a.starts + span;

  // f(tile, first entry in it, number, their place in the tiles' order) for
  // every tile, one per thread; their total and the entries of lower rows.
  int total = 0, before = 0;
  auto each_tile = [&](auto &&f) {
    total = before = 0;
    for (int64_t t0 = 0; t0 < a.tiles; t0 += 256) {
      const int64_t tile = t0 + tid;
      int lo = 0, n = 0, sum;
      if (tile < a.tiles) {
        lo = starts[tile * (a.spans + 1)];
        n = starts[tile * (a.spans + 1) + 1] - lo;
      }
      before += lo;
      const int at = total + list.prefix(n, sum);
      f(tile * a.tile + lo, n, at);
      total += sum;
    }
  };
  auto bin_at = [&](int64_t e) {
    return entry_bin(static_cast<int>(a.keys[e] - row0), a.sources[e]);
  };
  // The entries at places [from, from + kListMost) to the list.
  auto gather = [&](int from, bool count) {
    each_tile([&](int64_t e, int n, int at) {
      const int lo = max(from - at, 0), hi = min(n, from + kListMost - at);
      for (int i = lo; i < hi; ++i) {
        const int b = bin_at(e + i);
        list.source[at + i - from] = a.sources[e + i];
        list.local[at + i - from] = static_cast<uint16_t>(b);
        if (count) atomicAdd(&list.next[b], 1);
      }
    });
  };
  list.clear();
  gather(0, true);
  int base;
  list.prefix(before, base);
  if (span == a.spans - 1 && tid == 0) a.row_start[a.rows] = base + total;
  if (total == 0) {
    if (tid < rows) a.row_start[row0 + tid] = base;
    return;
  }
  const int all = total;
  if (all > kListMost) { // the rest is counted where it lies
    each_tile([&](int64_t e, int n, int at) {
      for (int i = max(kListMost - at, 0); i < n; ++i) atomicAdd(&list.next[bin_at(e + i)], 1);
    });
  }
  list.open();
  if (tid < rows) {
    const int at = list.first[2 * tid], n = list.first[2 * tid + 2] - at;
    a.row_start[row0 + tid] = base + at;
    // Their order changes from run to run; each row's sum does not depend on it.
    int32_t *const hubs = a.hubs + span % kHubLists * a.hub_stride;
    if (n > kAlone) hubs[1 + atomicAdd(hubs, 1)] = static_cast<int32_t>(row0 + tid);
  }
  for (int from = 0; from < all; from += kListMost) {
    if (from > 0) {
      gather(from, false);
      __syncthreads();
    }
    list.place(min(all - from, kListMost), [&](int to, uint32_t what) { a.list[base + to] = what; });
  }
}

// Columns [begin, stop) of a row of many entries, [first, end), by the whole
// workgroup: a contiguous part of the entries per group of `wide` lanes (a
// power of two up to a wave), joined across lanes and then through LDS.
template <typename T, typename O, int VEC, typename ENTRY>
__device__ __forceinline__ void sum_hub(const GradArgs &a, float (&joined)[kSpanWaves][kWave * VEC],
                                        int wide, int64_t row, ENTRY &&entry, int first, int end,
                                        int64_t begin, int64_t stop) {
  const int tid = threadIdx.x, part = tid / wide, column = tid % wide * VEC;
  const int each = (end - first + 256 / wide - 1) / (256 / wide);
  const int from = min(first + part * each, end), to = min(from + each, end);
  for (int64_t c = begin + column; c - column < stop; c += wide * VEC) {
    float acc[VEC] = {};
    if (c < stop) {
      const T *const grad = static_cast<const T *>(a.grad) + c;
      const float *const sums = a.sums + c;
      for (int i = from; i < to; i += 8) {
        uint32_t what[8];
        float v[8][VEC] = {};
        int summed = 0; // sums come first: mostly all or none of the eight
#pragma unroll
        for (int d = 0; d < 8; ++d) what[d] = entry(min(i + d, to - 1));
#pragma unroll
        for (int d = 0; d < 8; ++d) summed += what[d] >> 31;
        if (summed < 8) {
#pragma unroll
          for (int d = 0; d < 8; ++d)
            if (i + d < to && !(what[d] & kSummed))
              load_f32<VEC>(grad + what[d] * a.grad_stride, v[d]);
        }
        if (summed > 0) {
#pragma unroll
          for (int d = 0; d < 8; ++d)
            if (i + d < to && (what[d] & kSummed))
              load_f32<VEC>(sums + (what[d] & ~kSummed) * a.dim, v[d]);
        }
#pragma unroll
        for (int d = 0; d < 8; ++d) {
#pragma unroll
          for (int k = 0; k < VEC; ++k) acc[k] += v[d][k];
        }
      }
    }
    for (int j = wide; j < kWave; j <<= 1) {
#pragma unroll
      for (int k = 0; k < VEC; ++k) acc[k] += __shfl_xor(acc[k], j);
    }
    __syncthreads(); // what was here before has been read
    if (tid % kWave < wide) {
#pragma unroll
      for (int k = 0; k < VEC; ++k) joined[tid / kWave][column + k] = acc[k];
    }
    __syncthreads();
    if (tid < wide && c < stop) {
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        acc[k] = 0.0f;
#pragma unroll
        for (int w = 0; w < kSpanWaves; ++w) acc[k] += joined[w][column + k];
        acc[k] *= a.scale;
      }
      put_f32<VEC>(a.stream, static_cast<O *>(a.out) + row * a.out_stride + c, acc);
    }
  }
}

// Rows of a workgroup with entries that its lanes add up alone.
struct BusyRows {
  uint16_t row[kRowsMost];
  int count;
};

// Rows [row0, row0 + rows), of which r's entries are [first(r), first(r + 1)).
// Empty rows are written first, front to back (with ZERO).  The vectors of the
// rows with few entries then lie in a row before the workgroup's lanes, kItems of them 256
// apart per lane and turn, so that stores fill whole lines and every lane has
// kItems loads under way (with the empty rows among them, most lanes would
// have none); the entries after these are fetched meanwhile.
template <typename T, typename O, int VEC, bool ZERO, typename FIRST, typename ENTRY>
__device__ __forceinline__ void sum_rows(const GradArgs &a, BusyRows &busy, int64_t row0, int rows,
                                         FIRST &&first, ENTRY &&entry) {
  constexpr int kItems = 2;
  const uint32_t vecs = static_cast<uint32_t>(a.dim / VEC);
  O *const out = static_cast<O *>(a.out) + row0 * a.out_stride;
  if (threadIdx.x == 0) busy.count = 0;
  __syncthreads();
  for (int r = threadIdx.x; r < rows; r += 256) {
    const int n = first(r + 1) - first(r);
    if (n > 0 && n <= kAlone) busy.row[atomicAdd(&busy.count, 1)] = static_cast<uint16_t>(r);
  }
  __syncthreads();
  const int count = busy.count;
  if (ZERO && count < rows) {
    float zero[VEC] = {};
    if (vecs >= 256) { // a row per turn or more
      for (int r = 0; r < rows; ++r) {
        if (first(r + 1) != first(r)) continue;
        for (uint32_t c = threadIdx.x; c < vecs; c += 256)
          put_f32<VEC>(a.stream, out + r * a.out_stride + static_cast<int64_t>(c) * VEC, zero);
      }
    } else {
      for (uint32_t q = threadIdx.x; q < rows * vecs; q += 256) {
        const int r = q / vecs;
        if (first(r + 1) == first(r))
          put_f32<VEC>(a.stream, out + r * a.out_stride + static_cast<int64_t>(q - r * vecs) * VEC, zero);
      }
    }
  }
  const uint32_t all = count * vecs; // at most 2^31: kMostDim, kSpanMost
  for (uint32_t q0 = threadIdx.x; q0 < all; q0 += 256 * kItems) {
    float acc[kItems][VEC] = {};
    int left[kItems], longest = 0;
    uint32_t r[kItems], c[kItems], at[kItems], what[kItems];
#pragma unroll
    for (int u = 0; u < kItems; ++u) {
      const uint32_t q = q0 + 256 * u, n = min(q, all - 1) / vecs;
      c[u] = (q - n * vecs) * VEC;
      r[u] = busy.row[n];
      at[u] = first(r[u]);
      left[u] = q < all ? first(r[u] + 1) - at[u] : 0;
      longest = max(longest, left[u]);
    }
#pragma unroll
    for (int u = 0; u < kItems; ++u) what[u] = left[u] > 0 ? entry(at[u]) : 0;
    for (int i = 0; i < longest; ++i) {
      float v[kItems][VEC] = {};
      bool sums = false;
#pragma unroll
      for (int u = 0; u < kItems; ++u) {
        if (i < left[u] && !(what[u] & kSummed))
          load_f32<VEC>(static_cast<const T *>(a.grad) + what[u] * a.grad_stride + c[u], v[u]);
        sums = sums || (i < left[u] && (what[u] & kSummed));
      }
      if (sums) {
#pragma unroll
        for (int u = 0; u < kItems; ++u)
          if (i < left[u] && (what[u] & kSummed))
            load_f32<VEC>(a.sums + (what[u] & ~kSummed) * a.dim + c[u], v[u]);
      }
#pragma unroll
      for (int u = 0; u < kItems; ++u) what[u] = i + 1 < left[u] ? entry(at[u] + i + 1) : 0;
#pragma unroll
      for (int u = 0; u < kItems; ++u) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[u][k] += v[u][k];
      }
    }
#pragma unroll
    for (int u = 0; u < kItems; ++u) {
      if (left[u] == 0) continue;
#pragma unroll
      for (int k = 0; k < VEC; ++k) acc[u][k] *= a.scale;
      put_f32<VEC>(a.stream, out + r[u] * a.out_stride + c[u], acc[u]);
    }
  }
}

__host__ __device__ __forceinline__ int hub_lanes(uint32_t vecs) { return vecs <= 8 ? 8 : vecs <= 32 ? 32 : 64; }

// Step 3: a.row_block rows per workgroup, after kHubBlocks workgroups for the
// hubs, which take longest and so begin first.  Bound by memory: 2.4 million rows
// of 100 floats from 500,000 tokens in 253 us, 1.18 GB at 4.7 TB/s.
template <typename T, typename O, int VEC>
__global__ void __launch_bounds__(256) embedding_row_kernel(GradArgs a) {
  __shared__ float joined[kSpanWaves][kWave * VEC];
  __shared__ int start[kRowsMost + 1];
  __shared__ BusyRows busy;
  auto entry = [&](uint32_t i) { return a.list[i]; };
  if (blockIdx.x < kHubBlocks) {
    const uint32_t vecs = static_cast<uint32_t>(a.dim / VEC);
    const int wide = hub_lanes(vecs), slices = (vecs + wide - 1) / wide;
    const int32_t *const hubs = a.hubs + blockIdx.x % kHubLists * a.hub_stride;
    const int64_t all = static_cast<int64_t>(*hubs) * slices;
    for (int64_t i = blockIdx.x / kHubLists; i < all; i += kHubBlocks / kHubLists) {
      const int64_t row = hubs[1 + i / slices], begin = i % slices * wide * VEC;
      sum_hub<T, O, VEC>(a, joined, wide, row, entry, a.row_start[row], a.row_start[row + 1], begin,
                         min(begin + wide * VEC, a.dim));
    }
    return;
  }
  for (int64_t row0 = static_cast<int64_t>(blockIdx.x - kHubBlocks) * a.row_block; row0 < a.rows;
       row0 += static_cast<int64_t>(gridDim.x - kHubBlocks) * a.row_block) {
    const int rows = static_cast<int>(min(static_cast<int64_t>(a.row_block), a.rows - row0));
    for (int i = threadIdx.x; i <= rows; i += 256) start[i] = a.row_start[row0 + i];
    __syncthreads();
    sum_rows<T, O, VEC, true>(
        a, busy, row0, rows, [&](int r) { return start[r]; }, entry);
    __syncthreads(); // `start` and `busy` have been read
  }
}

// Zeros for `rows` rows of `dim` elements, 4 vectors per thread; a contiguous
// table is one row of any length.  A large table that few tokens touch is
// zeroed by a launch of its own, whose waves end with their stores: 6.8 TB/s,
// where spans that zero themselves reach 5.1 (614 MB: 92 and 125 us).
constexpr int kZeroItems = 4;
template <typename O, int VEC>
__global__ void __launch_bounds__(256) embedding_zero_kernel(O *out, int64_t rows, int64_t dim,
                                                             int64_t stride) {
  const int64_t vecs = dim / VEC, all = rows * vecs;
  const int64_t turn = static_cast<int64_t>(gridDim.x) * 256 * kZeroItems;
  float zero[VEC] = {};
  for (int64_t i0 = static_cast<int64_t>(blockIdx.x) * 256 * kZeroItems + threadIdx.x; i0 < all;
       i0 += turn) {
#pragma unroll
    for (int u = 0; u < kZeroItems; ++u) {
      const int64_t i = i0 + 256 * u;
      if (i < all) store_f32<VEC>(out + (rows == 1 ? i * VEC : i / vecs * stride + i % vecs * VEC), zero);
    }
  }
  const int64_t end = vecs * VEC + threadIdx.x; // of a row that is no whole vectors
  if (rows == 1 && blockIdx.x == 0 && end < dim) out[end] = static_cast<O>(0.0f);
}

// Places in order for the tokens of a workgroup that `here` marks, the k-th 64
// of each wave in here[k]: f(k, place) for each, on its lane.  All threads call
// it; the marks' number.
template <int EACH, typename F>
__device__ __forceinline__ int place_marked(int (&counts)[EACH * kSpanWaves],
                                            const uint64_t (&here)[EACH], F &&f) {
  static_assert(EACH * kSpanWaves <= 2 * kWave);
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
#pragma unroll
  for (int k = 0; k < EACH; ++k)
    if (lane == 0) counts[k * kSpanWaves + wave] = __popcll(here[k]);
  __syncthreads();
  const int c0 = lane < EACH * kSpanWaves ? counts[lane] : 0;
  const int c1 = lane + kWave < EACH * kSpanWaves ? counts[lane + kWave] : 0;
  const int in0 = wave_incl_scan(c0), in1 = wave_incl_scan(c1) + readlane(in0, kWave - 1);
  const uint64_t below = (uint64_t(1) << lane) - 1;
#pragma unroll
  for (int k = 0; k < EACH; ++k) {
    const int c = k * kSpanWaves + wave;
    const int before = c < kWave ? readlane(in0 - c0, c) : readlane(in1 - c1, c - kWave);
    if ((here[k] >> lane) & 1) f(k, before + __popcll(here[k] & below));
  }
  return readlane(in1, kWave - 1);
}

// At most MOST tokens and a table that is not large: a span per workgroup,
// zeroed while the tokens are on their way, and its rows that have some written
// again.  Latency: 1,000 tokens of 20,000 rows of 32 floats in 6 us.
template <typename T, typename O, int VEC, int MOST>
__global__ void __launch_bounds__(256) embedding_few_kernel(GradArgs a) {
  constexpr int kEach = MOST / 256;
  __shared__ SpanList<uint16_t, MOST> list;
  __shared__ uint16_t sorted[MOST]; // token indices by row
  __shared__ BusyRows busy;
  __shared__ float joined[kSpanWaves][kWave * VEC];
  __shared__ int counts[kEach * kSpanWaves];
  const int tid = threadIdx.x;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * a.span;
  const int rows = static_cast<int>(min(static_cast<int64_t>(a.span), a.rows - row0));
  list.clear();
  uint32_t row[kEach];
  token_rows(a, tid, 256, row);
  const int64_t vecs = a.dim / VEC, all = rows * vecs;
  O *const out = static_cast<O *>(a.out) + row0 * a.out_stride;
  float zero[VEC] = {};
  for (int64_t i = tid; i < all; i += 256)
    store_f32<VEC>(out + (a.out_stride == a.dim ? i * VEC
                                                : i / vecs * a.out_stride + i % vecs * VEC),
                   zero);
  uint64_t here[kEach];
#pragma unroll
  for (int k = 0; k < kEach; ++k) here[k] = ballot(row[k] >= row0 && row[k] < row0 + rows);
  const int total = place_marked<kEach>(counts, here, [&](int k, int at) { // after the zeros
    const uint32_t token = static_cast<uint32_t>(k * 256 + tid);
    const int b = entry_bin(static_cast<int>(row[k] - row0), token);
    list.source[at] = static_cast<uint16_t>(token);
    list.local[at] = static_cast<uint16_t>(b);
    atomicAdd(&list.next[b], 1);
  });
  if (total == 0) return;
  list.open();
  list.place(total, [&](int to, uint32_t what) { sorted[to] = static_cast<uint16_t>(what); });
  auto first = [&](int r) { return list.first[2 * r]; };
  auto entry = [&](int i) { return static_cast<uint32_t>(sorted[i]); };
  sum_rows<T, O, VEC, false>(a, busy, row0, rows, first, entry);
  if (total <= kAlone) return;
  const int wide = hub_lanes(static_cast<uint32_t>(vecs));
  for (int r = 0; r < rows; ++r) {
    const int from = first(r), to = first(r + 1);
    if (to - from > kAlone)
      sum_hub<T, O, VEC>(a, joined, wide, row0 + r, entry, from, to, 0, a.dim);
  }
}

// At most MOST tokens and a large table, zeroed before: a workgroup per token
// and slice of the columns, which ends if an earlier token is the same, or else
// lists those that are and sums its slice of their row.  Latency: 145 tokens in
// 5 us, after a zeroing that takes 107 to 123 (767 MB).
template <typename T, typename O, int VEC, int MOST>
__global__ void __launch_bounds__(256) embedding_token_kernel(GradArgs a, int64_t slice) {
  constexpr int kEach = MOST / 256;
  __shared__ uint32_t token_row;
  __shared__ uint16_t same[MOST];
  __shared__ float joined[kSpanWaves][kWave * VEC];
  __shared__ int counts[kEach * kSpanWaves];
  const int tid = threadIdx.x, wave_first = tid / kWave * kWave, t = blockIdx.x;
  uint32_t row[kEach];
  token_rows(a, tid, 256, row);
#pragma unroll
  for (int k = 0; k < kEach; ++k)
    if (k * 256 + tid == t) token_row = row[k];
  __syncthreads();
  const uint32_t mine = token_row;
  if (mine == static_cast<uint32_t>(a.rows)) return;
  uint64_t here[kEach];
  bool before = false;
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    here[k] = ballot(row[k] == mine);
    const int ahead = t - (k * 256 + wave_first); // of these 64, how many come before t
    before = before || (ahead >= kWave ? here[k] != 0
                                       : ahead > 0 && (here[k] & ((uint64_t(1) << ahead) - 1)) != 0);
  }
  if (__syncthreads_or(before)) return;
  const int n = place_marked<kEach>(
      counts, here, [&](int k, int at) { same[at] = static_cast<uint16_t>(k * 256 + tid); });
  __syncthreads();
  const int64_t begin = blockIdx.y * slice;
  sum_hub<T, O, VEC>(
      a, joined, hub_lanes(static_cast<uint32_t>(a.dim / VEC)), mine,
      [&](int i) { return static_cast<uint32_t>(same[i]); }, 0, n, begin, min(begin + slice, a.dim));
}

// ---- host ----------------------------------------------------------------------

// Rows per workgroup: about one turn.
template <typename T, int VEC> int32_t run_lookup(LookupArgs a, void *stream) {
  a.row_block = std::max<int64_t>(1, 256 * lookup_items(VEC) * VEC / a.dim);
  return launch(embedding_kernel<T, VEC>,
                dim3(std::min(ceil_div64(a.count, a.row_block), kMostBlocks)), dim3(256), stream, a);
}

template <typename T> int32_t lookup_typed(const LookupArgs &a, void *stream) {
  const int vec = row_vec(sizeof(T), a.dim, {a.table_stride, a.out_stride}, {a.table, a.out});
  if constexpr (sizeof(T) == 2) {
    if (vec == 8) return run_lookup<T, 8>(a, stream);
  }
  if (vec == 4) return run_lookup<T, 4>(a, stream);
  return run_lookup<T, 1>(a, stream);
}

struct GradLayout {
  bool large;
  int span, tile;
  int64_t spans, tiles;
  size_t keys, sources, order, runs, run_count, starts, sums, list, row_start, hubs, bytes;
  int64_t hub_stride;
};

// Table rows per span: enough spans to fill the card several times over, and
// at most kSpanMost rows each.  Few tokens need no tiles.
GradLayout grad_layout(int64_t count, int64_t rows, int64_t dim) {
  GradLayout l{};
  l.large = rows * dim >= kLarge;
  auto cut = [&](int64_t spans) {
    l.span = static_cast<int>(std::clamp<int64_t>(rows / spans, 1, kSpanMost));
    l.spans = ceil_div64(rows, l.span);
  };
  cut(1024);
  if (count * dim <= kFewElements && (l.large ? count <= kLargeFewMost
                                              : count <= kFewMost && count * l.spans <= kFewReads))
    return l;
  cut(2048);
  l.tile = count <= int64_t(kSmallTile) * kMostSmallTiles ? kSmallTile : kLargeTile;
  l.tiles = ceil_div64(count, l.tile);
  size_t at = 0;
  auto take = [&](size_t elems, size_t size) {
    const size_t here = at;
    at += Workspace::align(elems * size);
    return here;
  };
  const size_t tiles = static_cast<size_t>(l.tiles);
  l.keys = take(tiles * l.tile, sizeof(uint32_t));
  l.sources = take(tiles * l.tile, sizeof(uint32_t));
  l.order = take(tiles * l.tile, sizeof(uint16_t));
  l.runs = take(tiles * l.tile / kRun, sizeof(uint32_t));
  l.run_count = take(tiles, sizeof(int32_t));
  l.starts = take(tiles * (l.spans + 1), sizeof(uint16_t));
  l.sums = take(tiles * l.tile / kRun * dim, sizeof(float));
  l.list = take(count, sizeof(uint32_t));
  l.row_start = take(rows + 1, sizeof(int32_t));
  l.hub_stride = ceil_div64(1 + count / (kAlone + 1), 64) * 64; // lines of their own
  l.hubs = take(kHubLists * l.hub_stride, sizeof(int32_t));
  l.bytes = at;
  return l;
}

template <typename T, int VEC> int32_t run_spans(const GradArgs &a, void *stream) {
  const int64_t vecs = ceil_div64(a.dim, VEC);
  auto go = [&](auto kernel, int lanes) {
    const int64_t run_grid = a.tiles * run_blocks(a.tile) * ceil_div64(vecs, lanes);
    return launch(kernel, dim3(run_grid + a.spans), dim3(256), stream, a, run_grid);
  };
  if (vecs <= 8) return go(embedding_span_kernel<T, VEC, 8>, 8);
  if (vecs <= 32) return go(embedding_span_kernel<T, VEC, 32>, 32);
  return go(embedding_span_kernel<T, VEC, 64>, 64);
}

template <typename O, int VEC> int32_t zero_table(const GradArgs &a, void *stream) {
  auto go = [&](auto kernel, int64_t rows, int64_t vecs, int64_t dim) {
    const int64_t blocks = std::max<int64_t>(1, ceil_div64(rows * vecs, 256 * kZeroItems));
    return launch(kernel, dim3(std::min(blocks, kMostBlocks)), dim3(256), stream,
                  static_cast<O *>(a.out), rows, dim, a.out_stride);
  };
  constexpr int kWhole = 16 / sizeof(O);
  if ((a.out_stride == a.dim || a.rows == 1) && aligned_to(a.out, 16))
    return go(embedding_zero_kernel<O, kWhole>, 1, a.rows * a.dim / kWhole, a.rows * a.dim);
  return go(embedding_zero_kernel<O, VEC>, a.rows, a.dim / VEC, a.dim);
}

template <typename T, typename O, int VEC> int32_t grad_vec(GradArgs a, void *stream) {
  if (a.tiles == 0) {
    auto go = [&](auto kernel, int64_t blocks) {
      return launch(kernel, dim3(blocks), dim3(256), stream, a);
    };
    if (!a.large)
      return a.count <= 1024   ? go(embedding_few_kernel<T, O, VEC, 1024>, a.spans)
             : a.count <= 4096 ? go(embedding_few_kernel<T, O, VEC, 4096>, a.spans)
                               : go(embedding_few_kernel<T, O, VEC, kFewMost>, a.spans);
    const int32_t rc = zero_table<O, VEC>(a, stream);
    if (rc != SPORDER_OK || a.count == 0) return rc;
    const int64_t vecs = a.dim / VEC, wide = hub_lanes(static_cast<uint32_t>(vecs));
    const int64_t pieces = ceil_div64(vecs, wide);
    const int64_t slice = ceil_div64(pieces, std::min(pieces, kTokenSlices)) * wide * VEC;
    auto sum = [&](auto kernel) {
      return launch(kernel, dim3(a.count, ceil_div64(a.dim, slice)), dim3(256), stream, a, slice);
    };
    return a.count <= 512 ? sum(embedding_token_kernel<T, O, VEC, 512>)
                          : sum(embedding_token_kernel<T, O, VEC, kLargeFewMost>);
  }
  int32_t rc = a.tile == kSmallTile
                   ? launch(embedding_tile_kernel<kSmallTile>, dim3(a.tiles),
                            dim3(kSmallTile / kTileRounds), stream, a)
                   : launch(embedding_tile_kernel<kLargeTile>, dim3(a.tiles),
                            dim3(kLargeTile / kTileRounds), stream, a);
  if (rc == SPORDER_OK) rc = run_spans<T, VEC>(a, stream);
  if (rc != SPORDER_OK) return rc;
  // About one turn of sum_rows per workgroup, with one row in rows / count
  // taken to have entries.
  const int64_t vecs = a.dim / VEC, turn = 512;
  const int64_t sparse = std::clamp<int64_t>(a.rows / a.count, 1, kSparse);
  a.row_block = static_cast<int>(std::clamp<int64_t>(turn * sparse / vecs, 1, kRowsMost));
  return launch(embedding_row_kernel<T, O, VEC>,
                dim3(kHubBlocks + std::min(ceil_div64(a.rows, a.row_block), kMostBlocks)), dim3(256),
                stream, a);
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
// 2^32 threads, and the runs' launch takes 2 per token and slice.
constexpr int64_t kMostRows = (int64_t(1) << 31) - 2;
constexpr int64_t kMostTokens = (int64_t(1) << 28) - kLargeTile;

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
                     dim,     table_stride, out_stride, scale, token_bits == 64,
                     count * dim * type_bytes(type) >= kStreamBytes, 0};
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
                   rows * dim * type_bytes(out_type) >= kStreamBytes,
                   l.large,
                   bits_for(rows),
                   0,
                   l.span,
                   l.spans,
                   l.tile,
                   l.tiles,
                   reinterpret_cast<uint32_t *>(w + l.keys),
                   reinterpret_cast<uint32_t *>(w + l.sources),
                   reinterpret_cast<uint16_t *>(w + l.order),
                   reinterpret_cast<uint32_t *>(w + l.runs),
                   reinterpret_cast<int32_t *>(w + l.run_count),
                   reinterpret_cast<uint16_t *>(w + l.starts),
                   reinterpret_cast<float *>(w + l.sums),
                   reinterpret_cast<uint32_t *>(w + l.list),
                   reinterpret_cast<int32_t *>(w + l.row_start),
                   reinterpret_cast<int32_t *>(w + l.hubs),
                   l.hub_stride};
  if (type == SPORDER_TYPE_F32) return grad_typed<float, float>(a, stream);
  if (type == SPORDER_TYPE_BF16)
    return out_type == type ? grad_typed<bf16_t, bf16_t>(a, stream)
                            : grad_typed<bf16_t, float>(a, stream);
  return out_type == type ? grad_typed<f16_t, f16_t>(a, stream)
                          : grad_typed<f16_t, float>(a, stream);
}

} // extern "C"
