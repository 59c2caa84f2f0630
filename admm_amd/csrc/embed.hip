// Row lookup of a weight matrix (X W) and its gradient (X^T R) by sorted ids.
#include "rows_common.h"

namespace admm_impl {

constexpr uint64_t kMaxCount = 0xFFFFFF00ull;  // entries, rows: counted in 32 bits with room for a step beyond
constexpr int kSortSmall = 16384;  // entries that one workgroup can sort in its LDS

// ---- lookup -----------------------------------------------------------------------------------

// One id per row: a copy with a factor, bound by memory.  2^lanes_log2 lanes share a row, N elements each at a time, four of
// those on the way.  16384 rows of 4096 in 16 bits: 36 us, 134 MB written and the distinct rows (56 MB) read, 5.3 TB/s; 8 rows: 2.3 us.
template <class T, class TO, int N, class Id>
__global__ void __launch_bounds__(256) k_embed_rows(const Id *__restrict__ ids, uint64_t nrows, const T *__restrict__ table,
                                                    uint64_t tstride, uint64_t trows, TO *__restrict__ out, uint64_t ostride,
                                                    uint64_t cols, float scale, int lanes_log2) {
  const unsigned lanes = 1u << lanes_log2, lane = threadIdx.x & (lanes - 1);
  const uint64_t per = 256u >> lanes_log2, whole = cols / N * N;
  for (uint64_t r = (uint64_t)blockIdx.x * per + (threadIdx.x >> lanes_log2); r < nrows; r += (uint64_t)gridDim.x * per) {
    const uint64_t id = sizeof(Id) == 4 ? (uint64_t)(uint32_t)ids[r] : (uint64_t)ids[r];
    const bool there = id < trows;
    const T *from = table + (there ? id : 0) * tstride;
    TO *to = out + r * ostride;
    const float f = there ? scale : 0.0f;
    for (uint64_t j = (uint64_t)lane * N; j < whole; j += (uint64_t)lanes * N * 4) {
      float v[4][N];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint64_t at = j + (uint64_t)u * lanes * N;
        if (at < whole) load_n<T, N>(from + at, v[u]);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint64_t at = j + (uint64_t)u * lanes * N;
        if (at >= whole) continue;
#pragma unroll
        for (int k = 0; k < N; ++k) v[u][k] = there ? v[u][k] * f : 0.0f;
        store_n<TO, N>(to + at, v[u]);
      }
    }
    for (uint64_t j = whole + lane; j < cols; j += lanes) to[j] = (TO)(there ? (float)from[j] * f : 0.0f);
  }
}

// Sums the rows `src(e)` for e in [b, end) into acc: the lanes of a wave are groups of 2^lanes_log2, a group takes every
// groups-th entry and its lanes the columns; then the groups' sums are added, so that every lane has the total.
template <int N, class Load>
__device__ inline void sum_entries(uint64_t b, uint64_t end, int lanes_log2, unsigned first, unsigned step, Load load, float (&acc)[N]) {
#pragma unroll
  for (int k = 0; k < N; ++k) acc[k] = 0.0f;
  for (uint64_t e = b + first; e < end; e += (uint64_t)step * 4) {
    float v[4][N];
    float f[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const uint64_t at = e + (uint64_t)u * step;
      f[u] = 0.0f;
      if (at < end) f[u] = load(at, v[u]);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (e + (uint64_t)u * step >= end || f[u] == 0.0f) continue;
#pragma unroll
      for (int k = 0; k < N; ++k) acc[k] += v[u][k] * f[u];
    }
  }
}

template <int N>
__device__ inline void add_groups(int lanes_log2, float (&acc)[N]) {
  for (int off = 1 << lanes_log2; off < 64; off <<= 1) {
#pragma unroll
    for (int k = 0; k < N; ++k) acc[k] += __shfl_xor(acc[k], off, 64);
  }
}

// Rows of several ids.  WAVES waves share a row (1, or 16 for few long ones), each of them as 64 /
// 2^lanes_log2 groups of lanes that take entries in turn.  65536 rows of 40 entries over 16 floats: 36 us, bound by scattered
// requests to memory: 1.17 million of them (half of the 2.34 million that reach L2 hit there), 32 a ns, where a lookup of 2^24
// distinct rows of 64 bytes in random order reaches 40 (2.5 TB/s; rows of 128 bytes 33 a ns, 4.2 TB/s).  Waves wait for 69 % of
// their cycles, the units that form the addresses are busy for 45 %.  65536 x 40 x 256: 441 us, 6.1 TB/s.
template <class T, class TO, int N, class Id, int WAVES>
__global__ void __launch_bounds__(WAVES == 1 ? 256 : 64 * WAVES)
    k_embed_bags(const Id *__restrict__ ids, const uint64_t *__restrict__ rowptr, const float *__restrict__ val, uint64_t nrows,
                 uint64_t nnz, const T *__restrict__ table, uint64_t tstride, uint64_t trows, TO *__restrict__ out,
                 uint64_t ostride, uint64_t cols, float scale, int lanes_log2) {
  constexpr int kRows = WAVES == 1 ? 4 : 1;
  __shared__ float sh[WAVES == 1 ? 1 : WAVES * 64 * N];
  const unsigned lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const unsigned lanes = 1u << lanes_log2, groups = 64u >> lanes_log2;
  const unsigned group = lane >> lanes_log2, sub = lane & (lanes - 1);
  const uint64_t col = ((uint64_t)blockIdx.y * lanes + sub) * N;
  const int here = col >= cols ? 0 : cols - col < N ? (int)(cols - col) : N;
  for (uint64_t r0 = (uint64_t)blockIdx.x * kRows; r0 < nrows; r0 += (uint64_t)gridDim.x * kRows) {
    const uint64_t r = WAVES == 1 ? r0 + wave : r0;
    uint64_t b = 0, end = 0;
    if (r < nrows) {
      b = rowptr[r];
      end = rowptr[r + 1];
      end = end < nnz ? end : nnz;
    }
    float acc[N];
    const unsigned first = WAVES == 1 ? group : wave * groups + group, step = WAVES == 1 ? groups : WAVES * groups;
    sum_entries<N>(b, end, lanes_log2, first, step,
                   [&](uint64_t e, float(&v)[N]) -> float {
                     const uint64_t id = sizeof(Id) == 4 ? (uint64_t)(uint32_t)ids[e] : (uint64_t)ids[e];
                     if (id >= trows || here == 0) return 0.0f;
                     const T *from = table + id * tstride + col;
                     if (here == N) {
                       load_n<T, N>(from, v);
                     } else {
#pragma unroll
                       for (int k = 0; k < N; ++k) v[k] = k < here ? (float)from[k < here ? k : 0] : 0.0f;
                     }
                     return val ? val[e] : 1.0f;
                   },
                   acc);
    add_groups<N>(lanes_log2, acc);
    if (WAVES > 1) {
      __syncthreads();
#pragma unroll
      for (int k = 0; k < N; ++k) sh[(wave * N + k) * 64 + lane] = acc[k];
      __syncthreads();
      if (wave == 0) {
#pragma unroll
        for (int k = 0; k < N; ++k) {
          float s = 0.0f;
          for (int w = 0; w < WAVES; ++w) s += sh[(w * N + k) * 64 + lane];
          acc[k] = s;
        }
      }
    }
    if (r < nrows && group == 0 && here && (WAVES == 1 || wave == 0)) {
      TO *to = out + r * ostride + col;
#pragma unroll
      for (int k = 0; k < N; ++k) acc[k] *= scale;
      if (here == N) {
        store_n<TO, N>(to, acc);
      } else {
#pragma unroll
        for (int k = 0; k < N; ++k)
          if (k < here) to[k] = (TO)acc[k];
      }
    }
  }
}

// ---- sorting the entries by id --------------------------------------------------------------------

// the sort's key of an entry: its id, or `trows` for what is outside the table (sorted behind everything else)
template <class Id>
__device__ inline uint32_t key_of(Id id, uint32_t trows) {
  const uint64_t v = sizeof(Id) == 4 ? (uint64_t)(uint32_t)id : (uint64_t)id;
  return v < trows ? (uint32_t)v : trows;
}

// Stable ranks among equal digits, wave by wave: the lanes with the same digit find each other by one ballot per bit, and
// the first of them takes their places from the wave's counter of that digit.
template <int ITEMS>
__device__ inline void rank_items(const uint32_t (&digit)[ITEMS], uint32_t (&rank)[ITEMS], int items, int bits, uint32_t *counters) {
  const unsigned lane = threadIdx.x & 63;
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    if (i >= items) break;
    unsigned long long same = ~0ull;
    for (int b = 0; b < bits; ++b) {
      const bool bit = (digit[i] >> b) & 1;
      const unsigned long long on = __ballot(bit);
      same &= bit ? on : ~on;
    }
    const int leader = __ffsll(same) - 1;
    uint32_t old = 0;
    if ((int)lane == leader) old = atomicAdd(&counters[digit[i]], (uint32_t)__popcll(same));
    old = __shfl(old, leader, 64);
    rank[i] = old + (uint32_t)__popcll(same & ((1ull << lane) - 1));
  }
}

// counters[wave][digit] -> the items with that digit in the waves before; their sum to totals; one thread a digit
template <int WAVES>
__device__ inline void totals_of_waves(uint32_t *counters, uint32_t *totals) {
  if (threadIdx.x < 256) {
    uint32_t n[WAVES], sum = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) n[w] = counters[w * 256 + threadIdx.x];
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      counters[w * 256 + threadIdx.x] = sum;
      sum += n[w];
    }
    totals[threadIdx.x] = sum;
  }
}

// exclusive sums of v[0..255] in place, by the first wave (4 values a lane); everybody waits
__device__ inline void scan_256(uint32_t *v) {
  __syncthreads();
  if (threadIdx.x < 64) {
    uint32_t x[4], s = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      x[k] = v[threadIdx.x * 4 + k];
      s += x[k];
    }
    uint32_t up = s;
    for (int off = 1; off < 64; off <<= 1) {
      const uint32_t y = __shfl_up(up, off, 64);
      if ((int)threadIdx.x >= off) up += y;
    }
    up -= s;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[threadIdx.x * 4 + k] = up;
      up += x[k];
    }
  }
  __syncthreads();
}

// what the sort leaves: per entry in the order of the ids, its id, its row and its factor
struct Sorted {
  uint32_t *ids, *rows;
  float *val;
  const uint32_t *row_of;  // row of every entry in the caller's order; NULL: entry e is row e
  const float *val_of;     // the caller's factors or NULL
  const uint64_t *rowptr;
  uint32_t nrows;
  // the row of an entry; one that does not exist where no row holds the entry (row_of is not written there)
  __device__ uint32_t row(uint32_t entry) const {
    if (!row_of) return entry;
    const uint32_t r = row_of[entry];
    return r < nrows && rowptr[r] <= entry && entry < rowptr[r + 1] ? r : 0xFFFFFFFFu;
  }
  // of several entries, whose loads are on the way together
  template <int N>
  __device__ void rows_of(const uint32_t (&entry)[N], uint32_t (&out)[N]) const {
    uint64_t from[N], end[N];
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = row_of ? row_of[entry[i]] : entry[i];
    if (!row_of) return;
    if (nrows == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) out[i] = 0xFFFFFFFFu;
      return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t r = out[i] < nrows ? out[i] : nrows - 1;
      from[i] = rowptr[r];
      end[i] = rowptr[(uint64_t)r + 1];
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (out[i] >= nrows || entry[i] < from[i] || entry[i] >= end[i]) out[i] = 0xFFFFFFFFu;
  }
};

// Up to kSortSmall entries, in one launch: every workgroup looks at all keys and sorts those of its own range of them in its
// LDS; how many are below its range says where they go.  (All passes over all keys in one workgroup: 17.5 us for 4001 keys of
// 15 bits; this: 8, and 12.5 for 16384 keys of 17 bits.  Keys loaded one after the other instead of all at once: 10 and 17.)
template <class Id, int kItems>
__global__ void __launch_bounds__(1024) k_sort_small(const Id *__restrict__ ids, uint32_t n, uint32_t trows, Sorted to) {
  extern __shared__ uint32_t sort_sh[];  // counters [16][256], totals [256], 16 + 16 counts of the waves, keys [n], entries [n]
  uint32_t *counters = sort_sh, *totals = counters + 16 * 256, *mine = totals + 256, *less = mine + 16, *keys = less + 16, *entries = keys + n;
  const unsigned lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t width = (uint32_t)(((uint64_t)trows + gridDim.x) / gridDim.x);  // of the trows + 1 keys
  const uint64_t from = (uint64_t)width * blockIdx.x, to_key = from + width;
  uint32_t key[kItems], entry[kItems];
  // a wave's items are consecutive, so what it keeps of them follows the order
  const uint32_t base = wave * (uint32_t)(kItems * 64) + lane;
  uint32_t kept = 0, below = 0;
  Id id[kItems];  // all on the way before the first is looked at
#pragma unroll
  for (int i = 0; i < kItems; ++i) id[i] = ids[base + i * 64 < n ? base + i * 64 : n - 1];
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const uint32_t at = base + i * 64;
    key[i] = at < n ? key_of(id[i], trows) : 0xFFFFFFFFu;
    const bool in = at < n && key[i] >= from && key[i] < to_key;
    const unsigned long long on = __ballot(in);
    below += (uint32_t)__popcll(__ballot(key[i] < from));
    entry[i] = in ? kept + (uint32_t)__popcll(on & ((1ull << lane) - 1)) : 0xFFFFFFFFu;
    kept += (uint32_t)__popcll(on);
  }
  if (lane == 0) {
    mine[wave] = kept;
    less[wave] = below;
  }
  __syncthreads();
  uint32_t count = 0, first = 0, place = 0;
  for (unsigned w = 0; w < 16; ++w) {
    if (w == wave) place = count;
    count += mine[w];
    first += less[w];
  }
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    if (entry[i] == 0xFFFFFFFFu) continue;
    keys[place + entry[i]] = key[i] - (uint32_t)from;
    entries[place + entry[i]] = base + i * 64;
  }
  __syncthreads();
  int bits = 0;
  while (bits < 32 && (width - 1) >> bits) ++bits;
  const int passes = (bits + 7) / 8, digits = passes ? (bits + passes - 1) / passes : 0;
  const int items = (int)((count + 1023) / 1024);
  const uint32_t b2 = wave * (uint32_t)(items * 64) + lane;
  for (int p = 0; p < passes; ++p) {
    uint32_t digit[kItems], rank[kItems];
    for (int i = threadIdx.x; i < 16 * 256; i += 1024) counters[i] = 0;
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      if (i >= items) break;
      const uint32_t at = b2 + i * 64;
      key[i] = at < count ? keys[at] : 0xFFFFFFFFu;
      entry[i] = at < count ? entries[at] : 0;
      digit[i] = (key[i] >> (p * digits)) & ((1u << digits) - 1);
    }
    __syncthreads();
    rank_items<kItems>(digit, rank, items, digits, counters + wave * 256);
    __syncthreads();
    totals_of_waves<16>(counters, totals);
    scan_256(totals);
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      if (i >= items) break;
      // the padding's digit is the largest and it comes behind everything: its places are `count` and beyond
      const uint32_t at = totals[digit[i]] + counters[wave * 256 + digit[i]] + rank[i];
      if (at >= count) continue;
      keys[at] = key[i];
      entries[at] = entry[i];
    }
    __syncthreads();
  }
  for (uint32_t i = threadIdx.x; i < count; i += 1024) {
    const uint32_t e = entries[i];
    to.ids[first + i] = keys[i] + (uint32_t)from;
    to.rows[first + i] = to.row(e);
    if (to.val_of) to.val[first + i] = to.val_of[e];
  }
}

// row of every entry that a row holds, 16 lanes a row
__device__ inline void entry_rows(const uint64_t *rowptr, uint64_t nrows, uint64_t nnz, uint32_t *row_of, unsigned block, unsigned blocks) {
  const unsigned lane = threadIdx.x & 15;
  for (uint64_t r = (uint64_t)block * 16 + (threadIdx.x >> 4); r < nrows; r += (uint64_t)blocks * 16) {
    const uint64_t b = rowptr[r], e1 = rowptr[r + 1], end = e1 < nnz ? e1 : nnz;
    for (uint64_t e = b + lane; e < end; e += 16) row_of[e] = (uint32_t)r;
  }
}

__global__ void __launch_bounds__(256) k_entry_rows(const uint64_t *__restrict__ rowptr, uint64_t nrows, uint64_t nnz, uint32_t *__restrict__ row_of) {
  entry_rows(rowptr, nrows, nnz, row_of, blockIdx.x, gridDim.x);
}

// More entries: one pass per digit, least significant first: counts per tile, their sums, the move.  What is moved with the key
// is the entry's row, and its factor in the upper half where there are factors.  Up to kFewTiles tiles the move sums their
// counts itself (counts by tile, then digit), which saves a launch a pass (32000 entries: 47 us instead of 53 with the
// gradient; 98 tiles: 59 instead of 56); from more of them the sums are made by a launch of their own (counts by digit, then
// tile).  The first count also finds the entries' rows, with workgroups of its own.  2.6 million entries with factors over 2^20
// ids: 3 passes, 95 us in all, of which the moves 53 and the counts 27; what they read and write would take 25.
constexpr uint32_t kFewTiles = 48;

template <class Id, bool FIRST>
__device__ inline uint32_t sort_key(const Id *ids, const uint32_t *keys, uint32_t at, uint32_t trows) {
  return FIRST ? key_of(ids[at], trows) : keys[at];
}

template <class Id, bool FIRST, int TILE>
__global__ void __launch_bounds__(256) k_sort_count(const Id *__restrict__ ids, const uint32_t *__restrict__ keys, uint32_t n,
                                                    uint32_t trows, int shift, int width, uint32_t *__restrict__ counts, uint32_t tiles,
                                                    const uint64_t *__restrict__ rowptr, uint64_t nrows, uint32_t *__restrict__ row_of) {
  __shared__ uint32_t hist[256];
  if (FIRST && blockIdx.x >= tiles) {
    entry_rows(rowptr, nrows, n, row_of, blockIdx.x - tiles, gridDim.x - tiles);
    return;
  }
  hist[threadIdx.x] = 0;
  __syncthreads();
  const uint32_t base = blockIdx.x * (uint32_t)TILE;
  uint32_t key[TILE / 256];
#pragma unroll
  for (int i = 0; i < TILE / 256; ++i) {
    const uint32_t at = base + i * 256 + threadIdx.x;
    key[i] = sort_key<Id, FIRST>(ids, keys, at < n ? at : n - 1, trows);
  }
#pragma unroll
  for (int i = 0; i < TILE / 256; ++i)
    if (base + i * 256 + threadIdx.x < n) atomicAdd(&hist[(key[i] >> shift) & ((1u << width) - 1)], 1u);
  __syncthreads();
  if (threadIdx.x < (1u << width))
    counts[tiles <= kFewTiles ? (uint64_t)blockIdx.x * 256 + threadIdx.x : (uint64_t)threadIdx.x * tiles + blockIdx.x] = hist[threadIdx.x];
}

// per digit: exclusive sums of its counts over the tiles, and its total
__global__ void __launch_bounds__(256) k_sort_scan(uint32_t *__restrict__ counts, uint32_t ntiles, uint32_t *__restrict__ totals) {
  __shared__ uint32_t sums[4];
  uint32_t *c = counts + (uint64_t)blockIdx.x * ntiles;
  uint32_t carry = 0;
  for (uint32_t t0 = 0; t0 < ntiles; t0 += 1024) {
    uint32_t x[4], s = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t t = t0 + threadIdx.x * 4 + k;
      x[k] = t < ntiles ? c[t] : 0;
      s += x[k];
    }
    uint32_t up = s;
    for (int off = 1; off < 64; off <<= 1) {
      const uint32_t y = __shfl_up(up, off, 64);
      if ((int)(threadIdx.x & 63) >= off) up += y;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 63) sums[threadIdx.x >> 6] = up;
    __syncthreads();
    up += carry - s;
    for (unsigned w = 0; w < 4; ++w) {
      if (w < threadIdx.x >> 6) up += sums[w];
      carry += sums[w];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t t = t0 + threadIdx.x * 4 + k;
      if (t < ntiles) c[t] = up;
      up += x[k];
    }
  }
  if (threadIdx.x == 0) totals[blockIdx.x] = carry;
}

// The tile is put in order in LDS first, so that what goes to one digit's place is written side by side.
template <class Id, class Load, bool FIRST, bool LAST, int TILE>
__global__ void __launch_bounds__(256) k_sort_move(const Id *__restrict__ ids, const uint32_t *__restrict__ keys, const Load *__restrict__ loads,
                                                   uint32_t n, uint32_t trows, int shift, int width, const uint32_t *__restrict__ counts,
                                                   const uint32_t *__restrict__ totals, uint32_t *__restrict__ keys_to,
                                                   Load *__restrict__ loads_to, Sorted to) {
  constexpr int kItems = TILE / 256;
  __shared__ uint32_t counters[4 * 256], start[256], local[256], tile_keys[TILE];
  __shared__ Load tile_loads[TILE];
  const unsigned lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t tile = blockIdx.x * (uint32_t)TILE, count = n - tile < (uint32_t)TILE ? n - tile : (uint32_t)TILE;
  const uint32_t base = wave * (kItems * 64) + lane, mask = (1u << width) - 1;
  uint32_t key[kItems], digit[kItems], rank[kItems];
  Load load[kItems];
  // step by step for all items, so that each step's loads are on the way together; beyond the end the last entry is read
  uint32_t at[kItems];
#pragma unroll
  for (int i = 0; i < kItems; ++i) at[i] = tile + (base + i * 64 < count ? base + i * 64 : count - 1);
  if (FIRST) {
    Id id[kItems];
    uint32_t row[kItems];
    float val[kItems];
#pragma unroll
    for (int i = 0; i < kItems; ++i) id[i] = ids[at[i]];
    if (sizeof(Load) == 8) {
#pragma unroll
      for (int i = 0; i < kItems; ++i) val[i] = to.val_of[at[i]];
    }
    to.rows_of(at, row);
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      key[i] = key_of(id[i], trows);
      load[i] = row[i];
      if (sizeof(Load) == 8) load[i] |= (Load)((unsigned long long)__float_as_uint(val[i]) << 32);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      key[i] = keys[at[i]];
      load[i] = loads[at[i]];
    }
  }
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    if (base + i * 64 >= count) key[i] = 0xFFFFFFFFu;
    digit[i] = (key[i] >> shift) & mask;
  }
  for (int i = threadIdx.x; i < 4 * 256; i += 256) counters[i] = 0;
  uint32_t before = 0, total = 0;  // of this thread's digit: in the tiles before, in all
  if (threadIdx.x <= mask) {
    if (gridDim.x <= kFewTiles) {
#pragma unroll 8
      for (uint32_t i = 0; i < gridDim.x; ++i) {
        const uint32_t c = counts[i * 256 + threadIdx.x];
        total += c;
        before += i < blockIdx.x ? c : 0;
      }
    } else {
      total = totals[threadIdx.x];
      before = counts[(uint64_t)threadIdx.x * gridDim.x + blockIdx.x];
    }
  }
  start[threadIdx.x] = total;
  scan_256(start);
  rank_items<kItems>(digit, rank, kItems, width, counters + wave * 256);
  __syncthreads();
  totals_of_waves<4>(counters, local);
  scan_256(local);
  // a digit's place in the whole, less its place in the tile
  if (threadIdx.x <= mask) start[threadIdx.x] += before - local[threadIdx.x];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    // what pads the last tile has the last digit and comes behind everything: its places are `count` and beyond
    const uint32_t at = local[digit[i]] + counters[wave * 256 + digit[i]] + rank[i];
    tile_keys[at] = key[i];
    tile_loads[at] = load[i];
  }
  __syncthreads();
#pragma unroll 4
  for (uint32_t i = threadIdx.x; i < count; i += 256) {
    const uint32_t k = tile_keys[i], place = start[(k >> shift) & mask] + i;
    const Load l = tile_loads[i];
    if (LAST) {
      to.ids[place] = k;
      to.rows[place] = (uint32_t)l;
      if (sizeof(Load) == 8) to.val[place] = __uint_as_float((uint32_t)((unsigned long long)l >> 32));
    } else {
      keys_to[place] = k;
      loads_to[place] = l;
    }
  }
}

// ---- gradient ---------------------------------------------------------------------------------

template <class T, class TO>
struct GradArgs {
  const uint32_t *ids, *rows;  // sorted by id
  const float *val;            // or NULL
  uint32_t n;
  const T *from;  // grad_out
  uint64_t fstride, frows;
  TO *to;  // grad_table
  uint64_t tstride, cols;
  uint32_t trows;
  float scale;
  int accumulate, lanes_log2;
  uint32_t chunk, nchunks;  // entries per chunk
  float *parts;             // [chunk][2][pitch]
  uint64_t pitch;           // cols, to a multiple of 8
  unsigned chunk_blocks, zero_blocks;
};

// where this thread works: its columns, and its group of lanes among its workgroup's
template <int N>
struct Place {
  unsigned lane, wave, lanes, groups, group, sub;
  uint64_t col;
  int here;  // columns of this thread
  __device__ Place(int lanes_log2, uint64_t cols) {
    lane = threadIdx.x & 63;
    wave = threadIdx.x >> 6;
    lanes = 1u << lanes_log2;
    groups = 64u >> lanes_log2;
    group = lane >> lanes_log2;
    sub = lane & (lanes - 1);
    col = ((uint64_t)blockIdx.y * lanes + sub) * N;
    here = col >= cols ? 0 : cols - col < N ? (int)(cols - col) : N;
  }
};

template <int N, class T, class TO>
__device__ inline void put_row(const GradArgs<T, TO> &a, uint32_t id, const Place<N> &p, const float (&acc)[N]) {
  TO *to = a.to + (uint64_t)id * a.tstride + p.col;
  if (p.here == N) {
    float old[N], v[N];
    if (a.accumulate) load_n<TO, N>(to, old);
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = a.accumulate ? old[k] + acc[k] * a.scale : acc[k] * a.scale;
    store_n<TO, N>(to, v);
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (k < p.here) to[k] = (TO)(a.accumulate ? (float)to[k] + acc[k] * a.scale : acc[k] * a.scale);
  }
}

template <int N, class T, class TO>
__device__ inline void put_part(const GradArgs<T, TO> &a, uint32_t chunk, int slot, const Place<N> &p, const float (&acc)[N]) {
  store_n<float, N>(a.parts + ((uint64_t)chunk * 2 + slot) * a.pitch + p.col, acc);  // columns beyond cols are the pitch's
}

// Two kinds of blocks, every one over one tile of columns (blockIdx.y):
//  * chunks: a group of lanes sums a.chunk consecutive entries of the sorted order, however they fall into runs of one id.  A run
//    that lies in the chunk is written at once; the sum of one that comes in from the chunk before goes to slot 0 of `parts`, that
//    of one that begins here and goes on to slot 1.  So every group has the same work, every row is written by one group, in a
//    fixed order and without atomics, whatever the ids.
//  * zeros (only where every row has to be written): rows of the table that no entry names.
// 16384 entries of 2048 columns, bf16 added to f32: 43 us at 128 MB (reads and writes of touched rows, in no order).  2.6 million
// entries of 16 floats: 47 us; 71 MB are written, 78 read in 1.2 million requests, 26 a ns (scattered as the lookup's).
template <class T, class TO, int N>
__global__ void __launch_bounds__(256) k_grad(GradArgs<T, TO> a) {
  const Place<N> p(a.lanes_log2, a.cols);
  if (blockIdx.x < a.chunk_blocks) {
    // The workgroup's chunks lie side by side: their entries come through LDS, read in one piece.  (Every lane of a group
    // reading its entry from memory cost as much address work as the rows themselves, 81 us for 2.6 million entries of 16 floats.)
    extern __shared__ uint32_t stage[];
    constexpr int kAhead = 4;
    const uint32_t per = 4 * p.groups, pitch = a.chunk + 1;  // one word more, so that the groups' words fall on different banks
    uint32_t *const ids = stage, *const rows = ids + per * pitch;
    float *const val = reinterpret_cast<float *>(rows + per * pitch);
    const uint32_t mine = (p.wave * p.groups + p.group) * pitch;
    for (uint64_t c0 = (uint64_t)blockIdx.x * per; c0 < a.nchunks; c0 += (uint64_t)a.chunk_blocks * per) {
      const uint64_t first = c0 * a.chunk;
      const uint32_t here = (uint32_t)(a.n - first < (uint64_t)per * a.chunk ? a.n - first : (uint64_t)per * a.chunk);
      __syncthreads();
      for (uint32_t i = threadIdx.x; i < here; i += 256) {
        const uint32_t at = i / a.chunk * pitch + i % a.chunk;
        ids[at] = a.ids[first + i];
        rows[at] = a.rows[first + i];
        if (a.val) val[at] = a.val[first + i];
      }
      __syncthreads();
      const uint64_t c = c0 + p.wave * p.groups + p.group;
      if (c >= a.nchunks) continue;
      const uint32_t b = (uint32_t)(c * a.chunk), count = a.n - b < a.chunk ? a.n - b : a.chunk;
      uint32_t cur = ids[mine];
      if (cur >= a.trows) continue;  // padding, which comes last
      bool open = b > 0 && a.ids[b - 1] == cur;
      float acc[N];
#pragma unroll
      for (int k = 0; k < N; ++k) acc[k] = 0.0f;
      for (uint32_t e = 0; e < count; e += kAhead) {
        float v[kAhead][N], f[kAhead];
        uint32_t id[kAhead], at_row[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const uint32_t at = mine + (e + u < count ? e + u : count - 1), row = rows[at];
          id[u] = ids[at];
          f[u] = a.val ? val[at] : 1.0f;
          // an entry without a row, a row beyond grad_out (of an order that is not these bags'), the chunk's end: row 0 is read in
          // its place, so that the loads need no branches (49 us with them for 2.6 million entries of 16 floats, 47 without)
          if (row >= a.frows || e + u >= count || id[u] >= a.trows) f[u] = 0.0f;
          at_row[u] = f[u] == 0.0f ? 0 : row;
        }
        if (p.here == N) {
#pragma unroll
          for (int u = 0; u < kAhead; ++u) load_n<T, N>(a.from + at_row[u] * a.fstride + p.col, v[u]);
        } else {
#pragma unroll
          for (int u = 0; u < kAhead; ++u)
#pragma unroll
            for (int k = 0; k < N; ++k) v[u][k] = k < p.here ? (float)a.from[at_row[u] * a.fstride + p.col + k] : 0.0f;
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          if (e + u >= count) continue;
          if (id[u] != cur) {
            if (cur < a.trows && p.here) {
              if (open) put_part<N>(a, (uint32_t)c, 0, p, acc);
              else put_row<N>(a, cur, p, acc);
            }
            cur = id[u];
            open = false;
#pragma unroll
            for (int k = 0; k < N; ++k) acc[k] = 0.0f;
          }
          if (f[u] == 0.0f) continue;
#pragma unroll
          for (int k = 0; k < N; ++k) acc[k] += v[u][k] * f[u];
        }
      }
      if (cur >= a.trows || !p.here) continue;
      if (open) put_part<N>(a, (uint32_t)c, 0, p, acc);
      else if (b + count < a.n && a.ids[b + count] == cur) put_part<N>(a, (uint32_t)c, 1, p, acc);
      else put_row<N>(a, cur, p, acc);
    }
  } else {
    const uint32_t nsets = (uint32_t)(((uint64_t)a.trows + 63) / 64);
    for (uint32_t q = (blockIdx.x - a.chunk_blocks) * 4 + p.wave; q < nsets; q += a.zero_blocks * 4) {
      // Which of the 64 rows from v0 on have entries: the first position whose id is at least v0, 64 probes at a time; then the ids
      // of the next 64 entries, of 448 more if those do not reach the end of the set, and if there are still more, every lane
      // looks for its own row.  (64 probes for every id behind 64 entries: 23 us for 9096 entries of 262 ids; this: 10.)
      const uint32_t v0 = q * 64;
      uint32_t lo = 0, hi = a.n;
      while (hi > lo) {
        const uint32_t step = (hi - lo + 63) / 64;
        const uint64_t at = lo + (uint64_t)p.lane * step;
        const int small = __popcll(__ballot(at < hi && a.ids[at < hi ? at : hi - 1] < v0));  // the first `small` probes are below
        if (small == 0) {
          hi = lo;
        } else {
          const uint64_t to = lo + (uint64_t)small * step;
          lo = lo + (uint32_t)(small - 1) * step + 1;
          hi = to < hi ? (uint32_t)to : hi;
        }
      }
      constexpr int kMore = 7;
      uint64_t at = (uint64_t)lo + p.lane;
      const uint32_t id = at < a.n ? a.ids[at] : 0xFFFFFFFFu;
      unsigned long long there = id - v0 < 64 ? 1ull << (id - v0) : 0;  // an id beyond the table's end is not asked for below
      if ((uint32_t)__shfl(id, 63, 64) - v0 < 64) {
        uint32_t more[kMore];
#pragma unroll
        for (int i = 0; i < kMore; ++i) more[i] = at + 64 * (i + 1) < a.n ? a.ids[at + 64 * (i + 1)] : 0xFFFFFFFFu;
#pragma unroll
        for (int i = 0; i < kMore; ++i) there |= more[i] - v0 < 64 ? 1ull << (more[i] - v0) : 0;
        if ((uint32_t)__shfl(more[kMore - 1], 63, 64) - v0 < 64) {
          uint32_t from = lo, end = a.n;
          while (from < end) {
            const uint32_t mid = from + ((end - from) >> 1);
            if (a.ids[mid] < v0 + p.lane) from = mid + 1;
            else end = mid;
          }
          there |= from < a.n && a.ids[from] == v0 + p.lane ? 1ull << p.lane : 0;
        }
      }
      for (int off = 1; off < 64; off <<= 1) there |= __shfl_xor(there, off, 64);
      if (!p.here) continue;
      float zero[N];
#pragma unroll
      for (int k = 0; k < N; ++k) zero[k] = 0.0f;
      const unsigned rows = a.trows - v0 < 64 ? a.trows - v0 : 64;
      for (unsigned r = p.group; r < rows; r += p.groups) {
        if ((there >> r) & 1) continue;
        TO *to = a.to + (uint64_t)(v0 + r) * a.tstride + p.col;
        if (p.here == N) {
          store_n<TO, N>(to, zero);
        } else {
          for (int k = 0; k < N; ++k)
            if (k < p.here) to[k] = (TO)0.0f;
        }
      }
    }
  }
}

// Runs that go over the end of the chunk they begin in: the sums of their parts, in the order of the chunks.  Runs of up to
// kShort chunks after the first are summed by a group of lanes each; longer ones by a workgroup, which looks for them in
// kSet chunks at a time.  Bound by latency: 17 us for 82000 chunks of which most end inside a run, and 6 for 501.
constexpr int kShort = 7, kSet = 16;

template <class T, class TO>
__device__ inline bool run_leaves(const GradArgs<T, TO> &a, uint32_t c, uint32_t &id) {
  if (c + 1 >= a.nchunks) return false;
  const uint32_t b = c * a.chunk;
  id = a.ids[b + a.chunk];
  const uint32_t last = a.ids[b + a.chunk - 1], first = a.ids[b], before = a.ids[b ? b - 1 : 0];  // all at once
  return id < a.trows && last == id && (first != id || b == 0 || before != id);  // goes on, and begins here
}

template <class T, class TO, int N>
__global__ void __launch_bounds__(256) k_grad_join(GradArgs<T, TO> a, unsigned short_blocks) {
  __shared__ float sh[4][64 * N];
  const Place<N> p(a.lanes_log2, a.cols);
  auto add = [&](float(&acc)[N], uint32_t c, int slot) {
    float v[N];
    load_n<float, N>(a.parts + ((uint64_t)c * 2 + slot) * a.pitch + p.col, v);
#pragma unroll
    for (int k = 0; k < N; ++k) acc[k] += v[k];
  };
  float acc[N];
  if (blockIdx.x < short_blocks) {
    for (uint64_t c = ((uint64_t)blockIdx.x * 4 + p.wave) * p.groups + p.group; c < a.nchunks; c += (uint64_t)short_blocks * 4 * p.groups) {
      uint32_t id;
      if (!p.here || !run_leaves(a, (uint32_t)c, id)) continue;
      int more = 0;  // chunks after the first; the ids are sorted, so these are its
#pragma unroll
      for (int i = 1; i <= kShort + 1; ++i) more += c + i < a.nchunks && a.ids[(c + i) * a.chunk] == id;
      if (more > kShort) continue;  // a long one
#pragma unroll
      for (int k = 0; k < N; ++k) acc[k] = 0.0f;
      add(acc, (uint32_t)c, 1);
#pragma unroll
      for (int i = 1; i <= kShort; ++i)
        if (i <= more) add(acc, (uint32_t)c + i, 0);
      put_row<N>(a, id, p, acc);
    }
    return;
  }
  for (uint32_t set = blockIdx.x - short_blocks; (uint64_t)set * kSet < a.nchunks; set += gridDim.x - short_blocks) {
    const uint32_t mine = set * kSet + p.lane;
    uint32_t id = 0;
    bool is = false;
    if (p.lane < kSet && mine + 1ull + kShort < a.nchunks && run_leaves(a, mine, id)) is = a.ids[(mine + 1ull + kShort) * a.chunk] == id;
    for (unsigned long long todo = __ballot(is); todo; todo &= todo - 1) {  // the same in every wave
      const int l = __ffsll(todo) - 1;
      const uint32_t c = set * kSet + l, run = __shfl(id, l, 64);
      // the last chunk that begins with it, 64 probes at a time
      uint32_t lo = c + 1 + kShort, hi = a.nchunks;
      while (hi - lo > 1) {
        const uint32_t step = (hi - lo + 63) / 64;
        const uint64_t at = lo + (uint64_t)p.lane * step;
        const int is_run = __popcll(__ballot(at < hi && a.ids[(at < hi ? at : lo) * a.chunk] == run));  // the first one is
        const uint64_t to = lo + (uint64_t)is_run * step;
        lo += (uint32_t)(is_run - 1) * step;
        hi = to < hi ? (uint32_t)to : hi;
      }
#pragma unroll
      for (int k = 0; k < N; ++k) acc[k] = 0.0f;
      if (p.here) {
        constexpr int kAhead = 8;
        const uint32_t step = 4 * p.groups;
        uint64_t q = c + p.wave * p.groups + p.group;
        if (q == c) {
          add(acc, c, 1);
          q += step;
        }
        for (; q + (kAhead - 1) * step <= lo; q += kAhead * step) {
          float v[kAhead][N];
#pragma unroll
          for (int u = 0; u < kAhead; ++u) load_n<float, N>(a.parts + (q + u * step) * 2 * a.pitch + p.col, v[u]);
#pragma unroll
          for (int u = 0; u < kAhead; ++u)
#pragma unroll
            for (int k = 0; k < N; ++k) acc[k] += v[u][k];
        }
        for (; q <= lo; q += step) add(acc, (uint32_t)q, 0);
      }
      add_groups<N>(a.lanes_log2, acc);
      __syncthreads();
#pragma unroll
      for (int k = 0; k < N; ++k) sh[p.wave][k * 64 + p.lane] = acc[k];
      __syncthreads();
      if (p.wave == 0 && p.group == 0 && p.here) {
#pragma unroll
        for (int k = 0; k < N; ++k)
          acc[k] = (sh[0][k * 64 + p.lane] + sh[1][k * 64 + p.lane]) + (sh[2][k * 64 + p.lane] + sh[3][k * 64 + p.lane]);
        put_row<N>(a, run, p, acc);
      }
    }
  }
}

// ---- host side --------------------------------------------------------------------------------

static int check_bags(const admm_bags *b, const char *who) {
  ADMM_REQUIRE(b, "%s: bags is NULL", who);
  ADMM_REQUIRE(b->id_type == ADMM_I32 || b->id_type == ADMM_I64, "%s: ids of type %d", who, b->id_type);
  ADMM_REQUIRE(b->nrows <= kMaxCount && b->nnz <= kMaxCount, "%s: %llu rows, %llu entries: at most 2^32 - 256 are supported",
               who, (unsigned long long)b->nrows, (unsigned long long)b->nnz);
  ADMM_REQUIRE(b->rowptr || b->nnz == b->nrows, "%s: %llu ids for %llu rows without row pointers", who, (unsigned long long)b->nnz,
               (unsigned long long)b->nrows);
  ADMM_REQUIRE(b->rowptr || !b->val, "%s: factors need row pointers", who);
  ADMM_REQUIRE(b->nnz == 0 || b->ids, "%s: ids is NULL", who);
  ADMM_REQUIRE(reinterpret_cast<uintptr_t>(b->ids) % type_bytes(b->id_type) == 0 && reinterpret_cast<uintptr_t>(b->rowptr) % 8 == 0 &&
                   reinterpret_cast<uintptr_t>(b->val) % 4 == 0,
               "%s: ids, row pointers or factors are not aligned to their elements", who);
  return ADMM_OK;
}

static int ceil_log2(uint64_t n) {
  int b = 0;
  while ((1ull << b) < n) ++b;
  return b;
}

// elements a lane handles at once: what 16 bytes of the narrower type hold, halved until both matrices allow it
static int lane_width(const admm_mat *a, const admm_mat *b) {
  int n = type_bytes(a->type) == 2 ? 8 : 4;
  while (n > 1 && !(rows_aligned(a, n) && rows_aligned(b, n))) n >>= 1;
  return n;
}

// f(T, TO, N) with N in {8, 4, 2, 1} for 16-bit T, {4, 2, 1} for float
template <class F>
static int by_types(int type, int out_type, int n, F f) {
#define ADMM_WIDTHS(T, TO)                                                    \
  switch (n) {                                                                \
    case 8: return f(T(), TO(), std::integral_constant<int, 8 / (sizeof(T) / 2)>()); \
    case 4: return f(T(), TO(), std::integral_constant<int, 4>());            \
    case 2: return f(T(), TO(), std::integral_constant<int, 2>());            \
    default: return f(T(), TO(), std::integral_constant<int, 1>());           \
  }
  if (type == ADMM_F32) ADMM_WIDTHS(float, float)
  if (type == ADMM_BF16 && out_type == ADMM_F32) ADMM_WIDTHS(bf16_t, float)
  if (type == ADMM_BF16) ADMM_WIDTHS(bf16_t, bf16_t)
  if (out_type == ADMM_F32) ADMM_WIDTHS(f16_t, float)
  ADMM_WIDTHS(f16_t, f16_t)
#undef ADMM_WIDTHS
}

// column tiles are the second dimension of a grid
static int check_tiles(uint64_t tiles, const char *who, uint64_t cols) {
  ADMM_REQUIRE(tiles <= 65535, "%s: %llu columns are more than rows of this alignment can have", who, (unsigned long long)cols);
  return ADMM_OK;
}

// Entries per tile of the sort's passes: large tiles write longer pieces side by side, small ones keep more of the GPU busy (us
// with 1024 and 2048: 100000 entries 32 and 40, 400000 36 and 42, 800000 45 and 49, 1600000 54 and 57 or, of more ids, 63 and
// 61, 2600000 91 and 74, 20000000 594 and 469).
static uint64_t sort_tile(uint64_t n) { return n <= (1u << 20) ? 1024 : 2048; }

struct OrderLayout {
  uint64_t ids, rows, val, row_of, keys_a, loads_a, keys_b, loads_b, counts, totals, bytes;
  explicit OrderLayout(const admm_bags *b) {
    const uint64_t arr = round_up(4 * b->nnz, 256), tile = sort_tile(b->nnz), tiles = (b->nnz + tile - 1) / tile;
    uint64_t at = 0;
    auto take = [&](uint64_t n) {
      const uint64_t here = at;
      at += n;
      return here;
    };
    ids = take(arr);
    rows = take(arr);
    val = take(b->val ? arr : 0);
    row_of = take(b->rowptr ? arr : 0);
    const bool large = b->nnz > kSortSmall;
    keys_a = take(large ? arr : 0);
    loads_a = take(large ? (b->val ? 2 : 1) * arr : 0);
    keys_b = take(large ? arr : 0);
    loads_b = take(large ? (b->val ? 2 : 1) * arr : 0);
    counts = take(large ? round_up(4 * 256 * tiles, 256) : 0);
    totals = take(1024);
    bytes = at;
  }
};

template <class Id, class Load, int TILE>
static int sort_large(admm_ctx *ctx, const Id *ids, uint32_t n, uint32_t trows, char *order, const OrderLayout &at, const Sorted &to) {
  const int bits = ceil_log2((uint64_t)trows + 1);  // keys are 0 .. trows
  auto u32 = [&](uint64_t off) { return reinterpret_cast<uint32_t *>(order + off); };
  auto loads_at = [&](uint64_t off) { return reinterpret_cast<Load *>(order + off); };
  const uint32_t tiles = (uint32_t)(((uint64_t)n + TILE - 1) / TILE);
  const int passes = (bits + 7) / 8, width = (bits + passes - 1) / passes;
  const uint32_t *keys = nullptr;
  const Load *loads = nullptr;
  for (int p = 0; p < passes; ++p) {
    const int shift = p * width;
    uint32_t *keys_to = u32(p & 1 ? at.keys_b : at.keys_a);
    Load *loads_to = loads_at(p & 1 ? at.loads_b : at.loads_a);
    if (p == 0)
      hipLaunchKernelGGL((k_sort_count<Id, true, TILE>), dim3(tiles + (to.rowptr ? blocks_for(to.nrows, 16) : 0)), dim3(256), 0, ctx->stream, ids,
                         keys, n, trows, shift, width, u32(at.counts), tiles, to.rowptr, (uint64_t)to.nrows, u32(at.row_of));
    else
      hipLaunchKernelGGL((k_sort_count<Id, false, TILE>), dim3(tiles), dim3(256), 0, ctx->stream, ids, keys, n, trows, shift, width,
                         u32(at.counts), tiles, to.rowptr, (uint64_t)to.nrows, u32(at.row_of));
    if (tiles > kFewTiles)
      hipLaunchKernelGGL(k_sort_scan, dim3(1u << width), dim3(256), 0, ctx->stream, u32(at.counts), tiles, u32(at.totals));
#define ADMM_MOVE(FIRST, LAST)                                                                                                  \
  hipLaunchKernelGGL((k_sort_move<Id, Load, FIRST, LAST, TILE>), dim3(tiles), dim3(256), 0, ctx->stream, ids, keys, loads, n, trows, \
                     shift, width, u32(at.counts), u32(at.totals), keys_to, loads_to, to)
    if (p == 0 && p + 1 == passes) ADMM_MOVE(true, true);
    else if (p == 0) ADMM_MOVE(true, false);
    else if (p + 1 == passes) ADMM_MOVE(false, true);
    else ADMM_MOVE(false, false);
#undef ADMM_MOVE
    keys = keys_to;
    loads = loads_to;
  }
  ADMM_HIP_CHECK(hipGetLastError());
  return ADMM_OK;
}

template <class Id>
static int sort_entries(admm_ctx *ctx, const admm_bags *b, uint32_t trows, char *order, const OrderLayout &at) {
  const uint32_t n = (uint32_t)b->nnz;
  const Id *ids = static_cast<const Id *>(b->ids);
  auto u32 = [&](uint64_t off) { return reinterpret_cast<uint32_t *>(order + off); };
  Sorted to{u32(at.ids), u32(at.rows), reinterpret_cast<float *>(order + at.val), b->rowptr ? u32(at.row_of) : nullptr, b->val, b->rowptr, (uint32_t)b->nrows};
  if (n <= kSortSmall) {
    if (b->rowptr)
      hipLaunchKernelGGL(k_entry_rows, dim3(blocks_for(b->nrows, 16)), dim3(256), 0, ctx->stream, b->rowptr, b->nrows, b->nnz, u32(at.row_of));
    const size_t lds = 4 * (17 * 256 + 32 + 2 * (size_t)n);
    auto launch = [&](auto kernel) -> int {
      if (lds > 64 * 1024)
        ADMM_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                           4 * (17 * 256 + 32 + 2 * kSortSmall)));
      hipLaunchKernelGGL(kernel, dim3((n + 511) / 512), dim3(1024), lds, ctx->stream, ids, n, trows, to);
      return ADMM_OK;
    };
    // keys a thread looks at: about as many as there are (8192 entries: 7.8 us with 8, 10.2 with 16)
    ADMM_TRY(n <= 1024   ? launch(&k_sort_small<Id, 1>)
             : n <= 4096 ? launch(&k_sort_small<Id, 4>)
             : n <= 8192 ? launch(&k_sort_small<Id, 8>)
                         : launch(&k_sort_small<Id, kSortSmall / 1024>));
    ADMM_HIP_CHECK(hipGetLastError());
    return ADMM_OK;
  }
  if (sort_tile(n) == 1024)
    return b->val ? sort_large<Id, unsigned long long, 1024>(ctx, ids, n, trows, order, at, to) : sort_large<Id, uint32_t, 1024>(ctx, ids, n, trows, order, at, to);
  return b->val ? sort_large<Id, unsigned long long, 2048>(ctx, ids, n, trows, order, at, to) : sort_large<Id, uint32_t, 2048>(ctx, ids, n, trows, order, at, to);
}

template <class Id>
static int embed(admm_ctx *ctx, const admm_bags *b, const admm_mat *table, float scale, const admm_mat *out) {
  const Id *ids = static_cast<const Id *>(b->ids);
  return by_types(table->type, out->type, lane_width(table, out), [&](auto t, auto to, auto width) -> int {
    using T = decltype(t);
    using TO = decltype(to);
    constexpr int N = decltype(width)::value;
    const uint64_t per_row = (table->cols + N - 1) / N;
    if (!b->rowptr) {
      int lanes = ceil_log2(per_row);
      if (lanes > 8) lanes = 8;
      hipLaunchKernelGGL((k_embed_rows<T, TO, N, Id>), dim3(blocks_for(b->nrows, 256u >> lanes)), dim3(256), 0, ctx->stream, ids, b->nrows,
                         static_cast<const T *>(table->data), table->stride, table->rows, static_cast<TO *>(out->data), out->stride,
                         table->cols, scale, lanes);
    } else {
      int lanes = ceil_log2(per_row);
      if (lanes > 6) lanes = 6;
      const uint64_t tiles = (per_row + (1u << lanes) - 1) >> lanes;
      ADMM_TRY(check_tiles(tiles, "admm_embed", table->cols));
      // 16 waves a row where the rows are too few to fill the GPU and each would keep its wave for many steps (us with 1 and 16:
      // 300 rows of 40 entries of 256 floats 11 and 5, 1000 of 40 20 and 13, 2000 of 40 23 and 24, of 80 44 and 37, 4000 of 600
      // 529 and 537, 6000 of 600 595 and 803; of 16 floats 1000 rows of 130 6 and 9, of 600 22 and 18)
      const uint64_t steps = b->nnz / b->nrows >> (6 - lanes), waves = b->nrows * tiles;
      const bool longrows = waves <= 2048 && steps >= 8 && steps * 32 >= waves;
      if (longrows)
        hipLaunchKernelGGL((k_embed_bags<T, TO, N, Id, 16>), dim3(blocks_for(b->nrows, 1), (unsigned)tiles), dim3(1024), 0, ctx->stream, ids, b->rowptr,
                           b->val, b->nrows, b->nnz, static_cast<const T *>(table->data), table->stride, table->rows,
                           static_cast<TO *>(out->data), out->stride, table->cols, scale, lanes);
      else
        hipLaunchKernelGGL((k_embed_bags<T, TO, N, Id, 1>), dim3(blocks_for(b->nrows, 4), (unsigned)tiles), dim3(256), 0, ctx->stream, ids, b->rowptr,
                           b->val, b->nrows, b->nnz, static_cast<const T *>(table->data), table->stride, table->rows,
                           static_cast<TO *>(out->data), out->stride, table->cols, scale, lanes);
    }
    ADMM_HIP_CHECK(hipGetLastError());
    return ADMM_OK;
  });
}

// Entries per chunk: short chunks keep the GPU busy where there is little to add; every chunk may write two rows of floats, so
// they are longer where there is more.  With 8 / 16 / 32 entries a chunk (us, sort included): 4001 entries of 1024 columns 24 /
// 27 / 37, 262144 of 16 64 / 67 / 79, 16384 of 1024 54 / 46 / 52, 640000 of 16 100 / 95 / 104, 65536 of 1024 177 / 151 / 129,
// 2.6 million of 16 234 / 194 / 163.  One chunk has nothing to join: 16 entries of 1024 in one 17.4, in two 20.4.
static uint64_t grad_chunk(uint64_t nnz, uint64_t cols) {
  const double sums = (double)nnz * (double)cols;
  return nnz <= 16 ? 16 : sums <= 0x1p23 ? 8 : sums <= 0x1p25 ? 16 : 32;
}

static uint64_t grad_parts_bytes(uint64_t nnz, uint64_t cols) {
  return (nnz + grad_chunk(nnz, cols) - 1) / grad_chunk(nnz, cols) * 2 * round_up(cols, 8) * sizeof(float);
}

static int embed_grad(admm_ctx *ctx, const admm_bags *b, const char *order, const admm_mat *from, float scale, int accumulate,
                      const admm_mat *to, float *parts) {
  const OrderLayout at(b);
  return by_types(from->type, to->type, lane_width(from, to), [&](auto t, auto tt, auto width) -> int {
    using T = decltype(t);
    using TO = decltype(tt);
    constexpr int N = decltype(width)::value;
    const uint64_t per_row = (from->cols + N - 1) / N;
    int lanes = ceil_log2(per_row);
    if (lanes > 6) lanes = 6;
    const uint64_t tiles = (per_row + (1u << lanes) - 1) >> lanes;
    ADMM_TRY(check_tiles(tiles, "admm_embed_grad", from->cols));
    GradArgs<T, TO> a;
    a.ids = reinterpret_cast<const uint32_t *>(order + at.ids);
    a.rows = reinterpret_cast<const uint32_t *>(order + at.rows);
    a.val = b->val ? reinterpret_cast<const float *>(order + at.val) : nullptr;
    a.n = b->nrows ? (uint32_t)b->nnz : 0;  // entries of no row add nothing, and there is no row to read
    a.from = static_cast<const T *>(from->data);
    a.fstride = from->stride;
    a.frows = b->nrows;
    a.to = static_cast<TO *>(to->data);
    a.tstride = to->stride;
    a.trows = (uint32_t)to->rows;
    a.cols = from->cols;
    a.scale = scale;
    a.accumulate = accumulate != 0;
    a.lanes_log2 = lanes;
    a.chunk = (uint32_t)grad_chunk(b->nnz, from->cols);
    a.nchunks = (uint32_t)(((uint64_t)a.n + a.chunk - 1) / a.chunk);
    a.parts = parts;
    a.pitch = round_up(from->cols, 8);
    const unsigned groups = 4u * (64u >> lanes);
    a.chunk_blocks = a.nchunks ? blocks_for(a.nchunks, groups) : 0;
    a.zero_blocks = accumulate ? 0 : blocks_for(to->rows, 256);
    if (a.chunk_blocks + a.zero_blocks == 0) return ADMM_OK;
    const size_t lds = (size_t)groups * (a.chunk + 1) * (b->val ? 12 : 8);
    if (lds > 64 * 1024)
      ADMM_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void *>(&k_grad<T, TO, N>), hipFuncAttributeMaxDynamicSharedMemorySize, 128 * 1024));
    hipLaunchKernelGGL((k_grad<T, TO, N>), dim3(a.chunk_blocks + a.zero_blocks, (unsigned)tiles), dim3(256), lds, ctx->stream, a);
    if (a.nchunks > 1) {
      const unsigned short_blocks = blocks_for(a.nchunks, groups), long_blocks = a.nchunks > kShort + 1 ? blocks_for(a.nchunks, kSet) : 0;
      hipLaunchKernelGGL((k_grad_join<T, TO, N>), dim3(short_blocks + long_blocks, (unsigned)tiles), dim3(256), 0, ctx->stream, a, short_blocks);
    }
    ADMM_HIP_CHECK(hipGetLastError());
    return ADMM_OK;
  });
}

}  // namespace admm_impl

using namespace admm_impl;

extern "C" int admm_csr_bags(const admm_csr *csr, admm_bags *out) {
  ADMM_REQUIRE(csr && out, "admm_csr_bags: NULL argument");
  ADMM_TRY(require_rows(csr, "admm_csr_bags"));
  if (csr->d_perm) {
    set_error("admm_csr_bags: the set is relabelled: its stored ids are frequency ranks");
    return ADMM_ERR_STATE;
  }
  ADMM_REQUIRE(csr->nnz <= kMaxCount, "admm_csr_bags: %llu entries: at most 2^32 - 256 are supported", (unsigned long long)csr->nnz);
  out->ids = csr->d_col;
  out->rowptr = csr->d_rowptr;
  out->val = csr->d_val;
  out->nrows = csr->nrows;
  out->nnz = csr->nnz;
  out->id_type = ADMM_I32;
  return ADMM_OK;
}

extern "C" int admm_embed(admm_ctx *ctx, const admm_bags *bags, const admm_mat *table, float scale, const admm_mat *out) {
  ADMM_REQUIRE(ctx, "admm_embed: ctx is NULL");
  ADMM_TRY(check_bags(bags, "admm_embed"));
  ADMM_TRY(check_mat(table, "admm_embed", "table"));
  ADMM_TRY(check_mat(out, "admm_embed", "out"));
  ADMM_REQUIRE(table->rows > 0 && table->rows <= kMaxCount, "admm_embed: a table of %llu rows", (unsigned long long)table->rows);
  ADMM_REQUIRE(out->cols == table->cols && out->rows >= bags->nrows, "admm_embed: out is %llu x %llu for %llu rows of %llu columns",
               (unsigned long long)out->rows, (unsigned long long)out->cols, (unsigned long long)bags->nrows, (unsigned long long)table->cols);
  ADMM_REQUIRE(out->type == table->type || out->type == ADMM_F32, "admm_embed: out has the table's type or ADMM_F32");
  ADMM_REQUIRE(!mats_overlap(table, out), "admm_embed: out overlaps the table");
  if (bags->nrows == 0 || table->cols == 0) return ADMM_OK;
  OnDevice on(ctx->device);
  ADMM_HIP_CHECK(on.error);
  KernelTimer t(ctx, ADMM_K_EMBED);
  return bags->id_type == ADMM_I32 ? embed<int32_t>(ctx, bags, table, scale, out) : embed<int64_t>(ctx, bags, table, scale, out);
}

extern "C" int admm_embed_order_bytes(const admm_bags *bags, uint64_t table_rows, uint64_t *bytes) {
  ADMM_REQUIRE(bytes, "admm_embed_order_bytes: bytes is NULL");
  ADMM_TRY(check_bags(bags, "admm_embed_order_bytes"));
  ADMM_REQUIRE(table_rows > 0 && table_rows <= kMaxCount, "admm_embed_order_bytes: a table of %llu rows", (unsigned long long)table_rows);
  *bytes = OrderLayout(bags).bytes;
  return ADMM_OK;
}

extern "C" int admm_embed_order(admm_ctx *ctx, const admm_bags *bags, uint64_t table_rows, void *order, uint64_t order_bytes) {
  ADMM_REQUIRE(ctx, "admm_embed_order: ctx is NULL");
  uint64_t need = 0;
  ADMM_TRY(admm_embed_order_bytes(bags, table_rows, &need));
  if (bags->nnz == 0) return ADMM_OK;
  ADMM_REQUIRE(order && reinterpret_cast<uintptr_t>(order) % 256 == 0, "admm_embed_order: order is NULL or not on 256 bytes");
  ADMM_REQUIRE(order_bytes >= need, "admm_embed_order: order has %llu bytes, %llu are needed", (unsigned long long)order_bytes,
               (unsigned long long)need);
  OnDevice on(ctx->device);
  ADMM_HIP_CHECK(on.error);
  KernelTimer t(ctx, ADMM_K_EMBED);
  const OrderLayout at(bags);
  return bags->id_type == ADMM_I32 ? sort_entries<int32_t>(ctx, bags, (uint32_t)table_rows, static_cast<char *>(order), at)
                                   : sort_entries<int64_t>(ctx, bags, (uint32_t)table_rows, static_cast<char *>(order), at);
}

extern "C" int admm_embed_grad_workspace(const admm_bags *bags, uint64_t cols, uint64_t *bytes) {
  ADMM_REQUIRE(bytes, "admm_embed_grad_workspace: bytes is NULL");
  ADMM_TRY(check_bags(bags, "admm_embed_grad_workspace"));
  ADMM_REQUIRE(cols < (1ull << 40), "admm_embed_grad_workspace: %llu columns", (unsigned long long)cols);
  *bytes = 0;
  if (bags->nnz <= grad_chunk(bags->nnz, cols)) return ADMM_OK;
  ADMM_TRY(check_tiles((cols + 511) / 512, "admm_embed_grad_workspace", cols));  // more columns are refused, whatever their alignment
  *bytes = grad_parts_bytes(bags->nnz, cols);
  return ADMM_OK;
}

extern "C" int admm_embed_grad(admm_ctx *ctx, const admm_bags *bags, const void *order, uint64_t order_bytes, const admm_mat *grad_out,
                               float scale, int accumulate, const admm_mat *grad_table, void *workspace, uint64_t workspace_bytes) {
  ADMM_REQUIRE(ctx, "admm_embed_grad: ctx is NULL");
  ADMM_TRY(check_bags(bags, "admm_embed_grad"));
  ADMM_TRY(check_mat(grad_out, "admm_embed_grad", "grad_out"));
  ADMM_TRY(check_mat(grad_table, "admm_embed_grad", "grad_table"));
  ADMM_REQUIRE(grad_table->rows > 0 && grad_table->rows <= kMaxCount, "admm_embed_grad: a table of %llu rows",
               (unsigned long long)grad_table->rows);
  ADMM_REQUIRE(grad_out->cols == grad_table->cols && grad_out->rows >= bags->nrows,
               "admm_embed_grad: grad_out is %llu x %llu for %llu rows of %llu columns", (unsigned long long)grad_out->rows,
               (unsigned long long)grad_out->cols, (unsigned long long)bags->nrows, (unsigned long long)grad_table->cols);
  ADMM_REQUIRE(grad_table->type == grad_out->type || grad_table->type == ADMM_F32, "admm_embed_grad: grad_table has grad_out's type or ADMM_F32");
  ADMM_REQUIRE(!mats_overlap(grad_out, grad_table), "admm_embed_grad: grad_out overlaps grad_table");
  if (grad_table->cols == 0 || (bags->nnz == 0 && accumulate)) return ADMM_OK;
  if (bags->nnz) {
    ADMM_REQUIRE(order && reinterpret_cast<uintptr_t>(order) % 256 == 0, "admm_embed_grad: order is NULL or not on 256 bytes");
    ADMM_REQUIRE(order_bytes >= OrderLayout(bags).bytes, "admm_embed_grad: order has %llu bytes, %llu are needed",
                 (unsigned long long)order_bytes, (unsigned long long)OrderLayout(bags).bytes);
    uint64_t need = 0;
    ADMM_TRY(admm_embed_grad_workspace(bags, grad_out->cols, &need));
    ADMM_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && reinterpret_cast<uintptr_t>(workspace) % 16 == 0),
                 "admm_embed_grad: the workspace is NULL, not on 16 bytes or smaller than %llu bytes", (unsigned long long)need);
  }
  OnDevice on(ctx->device);
  ADMM_HIP_CHECK(on.error);
  KernelTimer t(ctx, ADMM_K_EMBED);
  return embed_grad(ctx, bags, static_cast<const char *>(order), grad_out, scale, accumulate, grad_table, static_cast<float *>(workspace));
}
