// Row lookup of a weight matrix (X W) and its gradient (X^T R) by sorted ids.
#include "rows_common.h"

namespace admm_impl {

constexpr int kRun = 64;         // entries of one id that one unit sums; longer runs are cut at multiples of it
constexpr int kSortTile = 4096;  // entries per workgroup of the sort's passes
constexpr int kSortSmall = 8192; // entries that one workgroup sorts in its LDS

// ---- lookup -----------------------------------------------------------------------------------

// One id per row: a copy with a factor, bound by memory.  2^lanes_log2 lanes share a row, N elements each at a time.
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

// Rows of several ids.  WAVES waves share a row (1 for short ones, 16 for rows of hundreds of entries), each of them as 64 /
// 2^lanes_log2 groups of lanes that take entries in turn.
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
__device__ inline void rank_items(const uint32_t (&digit)[ITEMS], uint32_t (&rank)[ITEMS], int bits, uint32_t *counters) {
  const unsigned lane = threadIdx.x & 63;
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
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

// counters[wave][digit] -> first place of that wave's items with that digit, counted from `from(digit)`; one thread a digit
template <int WAVES, class From>
__device__ inline void waves_before(uint32_t *counters, int digits, From from) {
  for (int d = threadIdx.x; d < digits; d += WAVES * 64) {
    uint32_t sum = from(d);
    for (int w = 0; w < WAVES; ++w) {
      const uint32_t n = counters[w * 256 + d];
      counters[w * 256 + d] = sum;
      sum += n;
    }
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
  __device__ void put(uint32_t at, uint32_t key, uint32_t entry) const {
    ids[at] = key;
    rows[at] = row_of ? row_of[entry] : entry;
    if (val_of) val[at] = val_of[entry];
  }
};

// up to kSortSmall entries: all passes in one workgroup, keys and entries in its LDS
template <class Id>
__global__ void __launch_bounds__(1024) k_sort_small(const Id *__restrict__ ids, uint32_t n, uint32_t trows, int bits, Sorted to) {
  constexpr int kItems = kSortSmall / 1024;
  extern __shared__ uint32_t sort_sh[];  // keys [kSortSmall], entries [kSortSmall], counters [16][256], totals [256]
  uint32_t *keys = sort_sh, *entries = keys + kSortSmall, *counters = entries + kSortSmall, *totals = counters + 16 * 256;
  const unsigned lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t base = wave * (kItems * 64) + lane;  // a wave's items are consecutive, so ranks follow the order
  uint32_t key[kItems], entry[kItems];
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const uint32_t at = base + i * 64;
    key[i] = at < n ? key_of(ids[at], trows) : 0xFFFFFFFFu;
    entry[i] = at;
  }
  const int passes = (bits + 7) / 8, width = (bits + passes - 1) / passes;
  for (int p = 0; p < passes; ++p) {
    uint32_t digit[kItems], rank[kItems];
    for (int i = threadIdx.x; i < 16 * 256; i += 1024) counters[i] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kItems; ++i) digit[i] = (key[i] >> (p * width)) & ((1u << width) - 1);
    rank_items<kItems>(digit, rank, width, counters + wave * 256);
    __syncthreads();
    if (threadIdx.x < 256) {
      uint32_t s = 0;
      for (int w = 0; w < 16; ++w) s += counters[w * 256 + threadIdx.x];
      totals[threadIdx.x] = s;
    }
    scan_256(totals);
    waves_before<16>(counters, 256, [&](int d) { return totals[d]; });
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const uint32_t at = counters[wave * 256 + digit[i]] + rank[i];
      keys[at] = key[i];
      entries[at] = entry[i];
    }
    __syncthreads();
    if (p + 1 < passes) {
#pragma unroll
      for (int i = 0; i < kItems; ++i) {
        key[i] = keys[base + i * 64];
        entry[i] = entries[base + i * 64];
      }
      __syncthreads();
    }
  }
  // the padding's keys are all ones in every digit and came last in every pass: they are behind the n entries
  for (uint32_t at = threadIdx.x; at < n; at += 1024) to.put(at, keys[at], entries[at]);
}

// one pass over more entries, least significant digit first: counts per tile, their sums, the move
template <class Id, bool FIRST>
__device__ inline void load_tile(const Id *ids, const uint32_t *keys, const uint32_t *entries, uint32_t n, uint32_t trows,
                                 uint32_t base, uint32_t (&key)[kSortTile / 256], uint32_t (&entry)[kSortTile / 256]) {
#pragma unroll
  for (int i = 0; i < kSortTile / 256; ++i) {
    const uint32_t at = base + i * 64;
    key[i] = 0xFFFFFFFFu;
    entry[i] = 0;
    if (at < n) {
      key[i] = FIRST ? key_of(ids[at], trows) : keys[at];
      entry[i] = FIRST ? at : entries[at];
    }
  }
}

template <class Id, bool FIRST>
__global__ void __launch_bounds__(256) k_sort_count(const Id *__restrict__ ids, const uint32_t *__restrict__ keys, uint32_t n,
                                                    uint32_t trows, int shift, int width, uint32_t *__restrict__ counts) {
  __shared__ uint32_t hist[256];
  hist[threadIdx.x] = 0;
  __syncthreads();
  const uint32_t base = blockIdx.x * (uint32_t)kSortTile;
  for (int i = 0; i < kSortTile / 256; ++i) {
    const uint32_t at = base + i * 256 + threadIdx.x;
    if (at < n) atomicAdd(&hist[((FIRST ? key_of(ids[at], trows) : keys[at]) >> shift) & ((1u << width) - 1)], 1u);
  }
  __syncthreads();
  counts[(uint64_t)threadIdx.x * gridDim.x + blockIdx.x] = hist[threadIdx.x];
}

// per digit: exclusive sums of its counts over the tiles, and its total
__global__ void __launch_bounds__(256) k_sort_scan(uint32_t *__restrict__ counts, uint32_t ntiles, uint32_t *__restrict__ totals) {
  __shared__ uint32_t sums[256];
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
    sums[threadIdx.x] = s;
    __syncthreads();
    for (int off = 1; off < 256; off <<= 1) {
      const uint32_t y = (int)threadIdx.x >= off ? sums[threadIdx.x - off] : 0;
      __syncthreads();
      sums[threadIdx.x] += y;
      __syncthreads();
    }
    uint32_t up = carry + sums[threadIdx.x] - s;
    carry += sums[255];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t t = t0 + threadIdx.x * 4 + k;
      if (t < ntiles) c[t] = up;
      up += x[k];
    }
  }
  if (threadIdx.x == 0) totals[blockIdx.x] = carry;
}

template <class Id, bool FIRST, bool LAST>
__global__ void __launch_bounds__(256) k_sort_move(const Id *__restrict__ ids, const uint32_t *__restrict__ keys,
                                                   const uint32_t *__restrict__ entries, uint32_t n, uint32_t trows, int shift,
                                                   int width, const uint32_t *__restrict__ counts,
                                                   const uint32_t *__restrict__ totals, uint32_t *__restrict__ keys_to,
                                                   uint32_t *__restrict__ entries_to, Sorted to) {
  constexpr int kItems = kSortTile / 256;
  __shared__ uint32_t counters[4 * 256], start[256];
  const unsigned lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t key[kItems], entry[kItems], digit[kItems], rank[kItems];
  load_tile<Id, FIRST>(ids, keys, entries, n, trows, blockIdx.x * (uint32_t)kSortTile + wave * (kItems * 64) + lane, key, entry);
  for (int i = threadIdx.x; i < 4 * 256; i += 256) counters[i] = 0;
  start[threadIdx.x] = totals[threadIdx.x];
  scan_256(start);
#pragma unroll
  for (int i = 0; i < kItems; ++i) digit[i] = (key[i] >> shift) & ((1u << width) - 1);
  rank_items<kItems>(digit, rank, width, counters + wave * 256);
  __syncthreads();
  waves_before<4>(counters, 256, [&](int d) { return start[d] + counts[(uint64_t)d * gridDim.x + blockIdx.x]; });
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    // what pads the last tile has the last digit and comes behind everything: its places are n and beyond
    const uint32_t at = counters[wave * 256 + digit[i]] + rank[i];
    if (at >= n) continue;
    if (LAST) {
      to.put(at, key[i], entry[i]);
    } else {
      keys_to[at] = key[i];
      entries_to[at] = entry[i];
    }
  }
}

// row of every entry; entries that no row holds get a row that does not exist
__global__ void __launch_bounds__(256) k_entry_rows(const uint64_t *__restrict__ rowptr, uint64_t nrows, uint64_t nnz,
                                                    uint32_t *__restrict__ row_of) {
  const unsigned lane = threadIdx.x & 63;
  for (uint64_t r = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < nrows; r += (uint64_t)gridDim.x * 4) {
    const uint64_t b = rowptr[r], e1 = rowptr[r + 1], end = e1 < nnz ? e1 : nnz;
    for (uint64_t e = b + lane; e < end; e += 64) row_of[e] = (uint32_t)r;
  }
}

__global__ void __launch_bounds__(256) k_fill_u32(uint32_t *p, uint64_t n, uint32_t v) {
  for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (uint64_t)gridDim.x * 256) p[i] = v;
}

// ---- gradient ---------------------------------------------------------------------------------

// first position whose id is at least `id`
__device__ inline uint64_t lower_bound(const uint32_t *ids, uint64_t n, uint32_t id) {
  uint64_t lo = 0, hi = n;
  while (lo < hi) {
    const uint64_t mid = (lo + hi) >> 1;
    if (ids[mid] < id) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

template <class T, class TO>
struct GradArgs {
  const uint32_t *ids, *rows;  // sorted by id
  const float *val;            // or NULL
  uint64_t n;
  const T *from;  // grad_out
  uint64_t fstride, frows;
  TO *to;  // grad_table
  uint64_t tstride, trows, cols;
  float scale;
  int accumulate, lanes_log2;
  float *parts;  // [chunk][2][cols] sums of the parts of runs longer than kRun
  unsigned run_blocks, chunk_blocks, zero_blocks;
};

// factor of entry e and its row's values; 0 for an entry without a row
template <int N, class T, class TO>
__device__ inline float load_entry(const GradArgs<T, TO> &a, uint64_t e, uint64_t col, int here, float (&v)[N]) {
  const uint64_t row = a.rows[e];
  if (row >= a.frows || here == 0) return 0.0f;
  const T *from = a.from + row * a.fstride + col;
  if (here == N) {
    load_n<T, N>(from, v);
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = k < here ? (float)from[k < here ? k : 0] : 0.0f;
  }
  return a.val ? a.val[e] : 1.0f;
}

template <int N, class T, class TO>
__device__ inline void put_row(const GradArgs<T, TO> &a, uint32_t id, uint64_t col, int here, float (&acc)[N]) {
  TO *to = a.to + (uint64_t)id * a.tstride + col;
  if (here == N) {
    float old[N];
    if (a.accumulate) load_n<TO, N>(to, old);
#pragma unroll
    for (int k = 0; k < N; ++k) acc[k] = a.accumulate ? old[k] + acc[k] * a.scale : acc[k] * a.scale;
    store_n<TO, N>(to, acc);
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (k < here) to[k] = (TO)(a.accumulate ? (float)to[k] + acc[k] * a.scale : acc[k] * a.scale);
  }
}

// Three kinds of blocks, every one over one tile of columns (blockIdx.y):
//  * chunks: kRun sorted entries that may hold parts of at most two runs longer than kRun (the one that holds the first entry
//    and the one that holds the last): their sums go to `parts`;
//  * runs: one group of lanes per sorted entry; where a run of at most kRun entries begins it sums the run and writes the
//    row.  Every row is written by one group, in a fixed order, without atomics;
//  * zeros (only where every row has to be written): rows of the table that no entry names.
template <class T, class TO, int N>
__global__ void __launch_bounds__(256) k_grad(GradArgs<T, TO> a) {
  const unsigned lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const unsigned lanes = 1u << a.lanes_log2, groups = 64u >> a.lanes_log2;
  const unsigned group = lane >> a.lanes_log2, sub = lane & (lanes - 1);
  const uint64_t col = ((uint64_t)blockIdx.y * lanes + sub) * N;
  const int here = col >= a.cols ? 0 : a.cols - col < N ? (int)(a.cols - col) : N;
  if (blockIdx.x < a.chunk_blocks) {
    const uint64_t nchunks = (a.n + kRun - 1) / kRun;
    for (uint64_t c = (uint64_t)blockIdx.x * 4 + wave; c < nchunks; c += (uint64_t)a.chunk_blocks * 4) {
      const uint64_t p0 = c * kRun, end = p0 + kRun < a.n ? p0 + kRun : a.n;
      const uint32_t mine = p0 + lane < end ? a.ids[p0 + lane] : 0xFFFFFFFFu;
      const uint32_t first = a.ids[p0], last = a.ids[end - 1];
      for (int s = 0; s < 2; ++s) {
        const uint32_t id = s == 0 ? first : last;
        if (id >= a.trows || (s == 1 && last == first)) continue;
        const uint64_t count = (uint64_t)__popcll(__ballot(p0 + lane < end && mine == id));
        const uint64_t b = s == 0 ? p0 : end - count, e = b + count;
        const uint64_t head = s == 0 ? lower_bound(a.ids, a.n, id) : b;
        if (head + kRun >= a.n || a.ids[head + kRun] != id) continue;
        float acc[N];
        sum_entries<N>(b, e, a.lanes_log2, group, groups, [&](uint64_t j, float(&v)[N]) -> float { return load_entry<N>(a, j, col, here, v); }, acc);
        add_groups<N>(a.lanes_log2, acc);
        if (group == 0 && here) {
          float *to = a.parts + (c * 2 + s) * a.cols + col;
          for (int k = 0; k < N; ++k)
            if (k < here) to[k] = acc[k];
        }
      }
    }
  } else if (blockIdx.x < a.chunk_blocks + a.run_blocks) {
    const uint64_t per = 4u * groups;
    for (uint64_t i = (uint64_t)(blockIdx.x - a.chunk_blocks) * per + wave * groups + group; i < a.n; i += (uint64_t)a.run_blocks * per) {
      const uint32_t id = a.ids[i];
      if (id >= a.trows || (i > 0 && a.ids[i - 1] == id) || (i + kRun < a.n && a.ids[i + kRun] == id)) continue;
      float acc[N];
#pragma unroll
      for (int k = 0; k < N; ++k) acc[k] = 0.0f;
      bool on = true;
      for (uint64_t e = i; on; e += 4) {
        float v[4][N], f[4];
        bool in[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          on = on && e + u < a.n && a.ids[e + u < a.n ? e + u : i] == id;
          in[u] = on;
          f[u] = 0.0f;
          if (on) f[u] = load_entry<N>(a, e + u, col, here, v[u]);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (!in[u] || f[u] == 0.0f) continue;
#pragma unroll
          for (int k = 0; k < N; ++k) acc[k] += v[u][k] * f[u];
        }
      }
      if (here) put_row<N>(a, id, col, here, acc);
    }
  } else {
    const uint64_t nsets = (a.trows + 63) / 64;
    for (uint64_t q = (uint64_t)(blockIdx.x - a.chunk_blocks - a.run_blocks) * 4 + wave; q < nsets; q += (uint64_t)a.zero_blocks * 4) {
      const uint64_t v0 = q * 64 + lane;
      bool absent = v0 < a.trows;
      if (absent) {
        const uint64_t at = lower_bound(a.ids, a.n, (uint32_t)v0);
        absent = at >= a.n || a.ids[at] != (uint32_t)v0;
      }
      const unsigned long long todo = __ballot(absent);
      for (unsigned r = group; r < 64; r += groups) {
        if (!((todo >> r) & 1) || !here) continue;
        TO *to = a.to + (q * 64 + r) * a.tstride + col;
        float zero[N];
#pragma unroll
        for (int k = 0; k < N; ++k) zero[k] = 0.0f;
        if (here == N) {
          store_n<TO, N>(to, zero);
        } else {
          for (int k = 0; k < N; ++k)
            if (k < here) to[k] = (TO)0.0f;
        }
      }
    }
  }
}

// Runs longer than kRun: the sums of their parts, in the order of the chunks, by the block of the chunk they begin in
// (only the run that holds a chunk's last entry can begin in it and be that long).
template <class T, class TO, int N>
__global__ void __launch_bounds__(256) k_grad_join(GradArgs<T, TO> a) {
  __shared__ float sh[4][64 * N];
  const unsigned lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const unsigned lanes = 1u << a.lanes_log2, groups = 64u >> a.lanes_log2;
  const unsigned group = lane >> a.lanes_log2, sub = lane & (lanes - 1);
  const uint64_t col = ((uint64_t)blockIdx.y * lanes + sub) * N;
  const int here = col >= a.cols ? 0 : a.cols - col < N ? (int)(a.cols - col) : N;
  const uint64_t nchunks = (a.n + kRun - 1) / kRun;
  for (uint64_t c = blockIdx.x; c < nchunks; c += gridDim.x) {  // uniform over the block, so are the conditions below
    const uint64_t p0 = c * kRun, end = p0 + kRun < a.n ? p0 + kRun : a.n;
    const uint32_t id = a.ids[end - 1];
    if (id >= a.trows || end >= a.n || a.ids[end] != id) continue;  // ends in this chunk
    const bool whole = a.ids[p0] == id;
    if (whole && p0 > 0 && a.ids[p0 - 1] == id) continue;  // began before it
    uint64_t b = p0;
    if (!whole) {
      uint64_t lo = p0, hi = end;
      while (lo < hi) {
        const uint64_t mid = (lo + hi) >> 1;
        if (a.ids[mid] < id) lo = mid + 1;
        else hi = mid;
      }
      b = lo;
    }
    if (b + kRun >= a.n || a.ids[b + kRun] != id) continue;
    const uint64_t stop = lower_bound(a.ids, a.n, id + 1);
    const uint64_t clast = (stop - 1) / kRun;
    float acc[N];
#pragma unroll
    for (int k = 0; k < N; ++k) acc[k] = 0.0f;
    for (uint64_t q = c + wave * groups + group; q <= clast; q += 4 * groups) {
      const float *p = a.parts + (q * 2 + (q == c && !whole ? 1 : 0)) * a.cols + col;
#pragma unroll
      for (int k = 0; k < N; ++k)
        if (k < here) acc[k] += p[k];
    }
    add_groups<N>(a.lanes_log2, acc);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) sh[wave][k * 64 + lane] = acc[k];
    __syncthreads();
    if (wave == 0 && group == 0 && here) {
#pragma unroll
      for (int k = 0; k < N; ++k) acc[k] = (sh[0][k * 64 + lane] + sh[1][k * 64 + lane]) + (sh[2][k * 64 + lane] + sh[3][k * 64 + lane]);
      put_row<N>(a, id, col, here, acc);
    }
    __syncthreads();
  }
}

// ---- host side --------------------------------------------------------------------------------

static int check_bags(const admm_bags *b, const char *who) {
  ADMM_REQUIRE(b, "%s: bags is NULL", who);
  ADMM_REQUIRE(b->id_type == ADMM_I32 || b->id_type == ADMM_I64, "%s: ids of type %d", who, b->id_type);
  ADMM_REQUIRE(b->nrows < 0xFFFFFFFFull && b->nnz < 0xFFFFFFFFull, "%s: %llu rows, %llu entries: fewer than 2^32 - 1 are supported",
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

struct OrderLayout {
  uint64_t ids, rows, val, row_of, keys_a, entries_a, keys_b, entries_b, counts, totals, bytes;
  explicit OrderLayout(const admm_bags *b) {
    const uint64_t arr = round_up(4 * b->nnz, 256), tiles = (b->nnz + kSortTile - 1) / kSortTile;
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
    entries_a = take(large ? arr : 0);
    keys_b = take(large ? arr : 0);
    entries_b = take(large ? arr : 0);
    counts = take(large ? round_up(4 * 256 * tiles, 256) : 0);
    totals = take(1024);
    bytes = at;
  }
};

template <class Id>
static int sort_entries(admm_ctx *ctx, const admm_bags *b, uint32_t trows, char *order, const OrderLayout &at) {
  const uint32_t n = (uint32_t)b->nnz;
  const Id *ids = static_cast<const Id *>(b->ids);
  auto u32 = [&](uint64_t off) { return reinterpret_cast<uint32_t *>(order + off); };
  Sorted to{u32(at.ids), u32(at.rows), reinterpret_cast<float *>(order + at.val), b->rowptr ? u32(at.row_of) : nullptr, b->val};
  if (b->rowptr) {
    hipLaunchKernelGGL(k_fill_u32, dim3(blocks_for(n, 2048, 4096)), dim3(256), 0, ctx->stream, u32(at.row_of), (uint64_t)n, 0xFFFFFFFFu);
    hipLaunchKernelGGL(k_entry_rows, dim3(blocks_for(b->nrows, 4)), dim3(256), 0, ctx->stream, b->rowptr, b->nrows, b->nnz, u32(at.row_of));
  }
  const int bits = ceil_log2((uint64_t)trows + 1);  // keys are 0 .. trows
  if (n <= kSortSmall) {
    constexpr size_t lds = 4 * (2 * kSortSmall + 17 * 256);
    ADMM_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void *>(&k_sort_small<Id>), hipFuncAttributeMaxDynamicSharedMemorySize, lds));
    hipLaunchKernelGGL(k_sort_small<Id>, dim3(1), dim3(1024), lds, ctx->stream, ids, n, trows, bits, to);
    ADMM_HIP_CHECK(hipGetLastError());
    return ADMM_OK;
  }
  const uint32_t tiles = (n + kSortTile - 1) / kSortTile;
  const int passes = (bits + 7) / 8, width = (bits + passes - 1) / passes;
  const uint32_t *keys = nullptr, *entries = nullptr;
  for (int p = 0; p < passes; ++p) {
    const int shift = p * width;
    uint32_t *keys_to = u32(p & 1 ? at.keys_b : at.keys_a), *entries_to = u32(p & 1 ? at.entries_b : at.entries_a);
    if (p == 0)
      hipLaunchKernelGGL((k_sort_count<Id, true>), dim3(tiles), dim3(256), 0, ctx->stream, ids, keys, n, trows, shift, width, u32(at.counts));
    else
      hipLaunchKernelGGL((k_sort_count<Id, false>), dim3(tiles), dim3(256), 0, ctx->stream, ids, keys, n, trows, shift, width, u32(at.counts));
    hipLaunchKernelGGL(k_sort_scan, dim3(256), dim3(256), 0, ctx->stream, u32(at.counts), tiles, u32(at.totals));
#define ADMM_MOVE(FIRST, LAST)                                                                                             \
  hipLaunchKernelGGL((k_sort_move<Id, FIRST, LAST>), dim3(tiles), dim3(256), 0, ctx->stream, ids, keys, entries, n, trows, \
                     shift, width, u32(at.counts), u32(at.totals), keys_to, entries_to, to)
    if (p == 0 && p + 1 == passes) ADMM_MOVE(true, true);
    else if (p == 0) ADMM_MOVE(true, false);
    else if (p + 1 == passes) ADMM_MOVE(false, true);
    else ADMM_MOVE(false, false);
#undef ADMM_MOVE
    keys = keys_to;
    entries = entries_to;
  }
  ADMM_HIP_CHECK(hipGetLastError());
  return ADMM_OK;
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
      // a wave takes a row of 40 entries in a few steps; one of many hundreds would keep it alone on its CU
      const bool longrows = b->nnz / b->nrows >= 512;
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

static uint64_t grad_parts_bytes(uint64_t nnz, uint64_t cols) { return (nnz + kRun - 1) / kRun * 2 * cols * sizeof(float); }

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
    a.n = b->nnz;
    a.from = static_cast<const T *>(from->data);
    a.fstride = from->stride;
    a.frows = b->nrows;
    a.to = static_cast<TO *>(to->data);
    a.tstride = to->stride;
    a.trows = to->rows;
    a.cols = from->cols;
    a.scale = scale;
    a.accumulate = accumulate != 0;
    a.lanes_log2 = lanes;
    a.parts = parts;
    a.chunk_blocks = b->nnz > kRun ? blocks_for(b->nnz, 4 * kRun) : 0;  // a run longer than kRun needs more entries than that
    a.run_blocks = b->nnz ? blocks_for(b->nnz, 4u * (64u >> lanes)) : 0;
    a.zero_blocks = accumulate ? 0 : blocks_for(to->rows, 256);
    if (a.chunk_blocks + a.run_blocks + a.zero_blocks == 0) return ADMM_OK;
    hipLaunchKernelGGL((k_grad<T, TO, N>), dim3(a.chunk_blocks + a.run_blocks + a.zero_blocks, (unsigned)tiles), dim3(256), 0, ctx->stream, a);
    if (a.chunk_blocks)
      hipLaunchKernelGGL((k_grad_join<T, TO, N>), dim3(blocks_for(b->nnz, kRun), (unsigned)tiles), dim3(256), 0, ctx->stream, a);
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
  ADMM_REQUIRE(csr->nnz < 0xFFFFFFFFull, "admm_csr_bags: %llu entries: fewer than 2^32 - 1 are supported", (unsigned long long)csr->nnz);
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
  ADMM_REQUIRE(table->rows > 0 && table->rows < 0xFFFFFFFFull, "admm_embed: a table of %llu rows", (unsigned long long)table->rows);
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
  ADMM_REQUIRE(table_rows > 0 && table_rows < 0xFFFFFFFFull, "admm_embed_order_bytes: a table of %llu rows", (unsigned long long)table_rows);
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
  *bytes = bags->nnz > kRun ? grad_parts_bytes(bags->nnz, cols) : 0;
  return ADMM_OK;
}

extern "C" int admm_embed_grad(admm_ctx *ctx, const admm_bags *bags, const void *order, uint64_t order_bytes, const admm_mat *grad_out,
                               float scale, int accumulate, const admm_mat *grad_table, void *workspace, uint64_t workspace_bytes) {
  ADMM_REQUIRE(ctx, "admm_embed_grad: ctx is NULL");
  ADMM_TRY(check_bags(bags, "admm_embed_grad"));
  ADMM_TRY(check_mat(grad_out, "admm_embed_grad", "grad_out"));
  ADMM_TRY(check_mat(grad_table, "admm_embed_grad", "grad_table"));
  ADMM_REQUIRE(grad_table->rows > 0 && grad_table->rows < 0xFFFFFFFFull, "admm_embed_grad: a table of %llu rows",
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
