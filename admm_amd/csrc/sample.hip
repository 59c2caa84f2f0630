// Draws a class per row from softmax(logits / temperature) after top-k, top-p and min-p, with given uniform numbers.
//
// The weight of a class is w = 2^((x - max) L / T), L = log2(e), computed in double and held as the integer
// rint(w 2^S): sums of integers do not depend on their order, so a row's token does not depend on how it is summed.  S is 51,
// or less where a row of ones would not fit 63 bits.
//
// Every filter keeps a prefix of the classes in the order (logit descending, index ascending), and the draw is the first
// class in index order at which the cumulative weight passes a bound.  Both are one question -- the first class, by some
// key, at which the cumulative amount (a count, or the weight) reaches a target -- and are answered digit by digit: amounts
// per value of the digit in LDS, the value at which the target falls, and on with the classes of that value.
#include "rows_common.h"

namespace admm_impl {

constexpr int kThreads = 512;
constexpr int kDigit = 8;

struct SampleArgs {
  const void *logits;
  uint64_t stride, rows, cols;
  const float *temperature, *top_p, *min_p, *uniform;
  const int32_t *top_k;
  int32_t *token;
  float *logprob;
  int index_bits, shift;  // 2^index_bits >= cols; S
  float *tops;            // [rows][groups] largest logits of kGroup granules each
  int64_t groups;
  unsigned long long *sums;  // [rows of a batch][kParts][kSums]
};

// larger logits have smaller keys; -0 counts as 0 and NaN as -inf
__device__ inline uint32_t key_of(float x) {
  x = x == x ? x + 0.0f : -INFINITY;
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? b : ~(b | 0x80000000u);
}
__device__ inline float logit_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key : ~key & 0x7FFFFFFFu);
}

struct Weights {
  float top;      // the row's largest logit
  double per;     // L / T
  double least;   // 2^S min-p, or 0
  int shift;      // S <= 51
  __device__ Weights(float top_, float t, float min_p, int shift_) : top(top_), shift(shift_) {
    per = fmax(1.44269504088896340736 / (double)t, 1e-300);  // not 0 at an infinite temperature: -inf stays -inf
    least = min_p > 0.0f ? ldexp((double)min_p, shift) : 0.0;
  }
  // 2^S times the weight of a class: 2^(n + S) times a polynomial of the rest of the exponent (|f ln 2| <= 0.35: the series'
  // term of degree 11 is 2e-13, where the draw of a flat row of 2^17 classes sees 8e-6 a class).  0 for -inf and NaN; a top of
  // +inf is not meant here.
  __device__ double scaled(float x) const {
    const double y = fmax(((double)x - (double)top) * per, -1100.0);
    const double n = rint(y), f = y - n;
    double p = 7.054911620801121e-09;  // ln(2)^k / k!
    p = fma(p, f, 1.0178086009239699e-07);
    p = fma(p, f, 1.3215486790144307e-06);
    p = fma(p, f, 1.525273380405984e-05);
    p = fma(p, f, 0.0001540353039338161);
    p = fma(p, f, 0.0013333558146428443);
    p = fma(p, f, 0.009618129107628477);
    p = fma(p, f, 0.05550410866482158);
    p = fma(p, f, 0.2402265069591007);
    p = fma(p, f, 0.6931471805599453);
    p = fma(p, f, 1.0);
    return ldexp(p, (int)n + shift);
  }
  // rounded to an integer below 2^52: what is left in the mantissa after 2^52 is added
  __device__ static unsigned long long units(double v) { return __double_as_longlong(v + 0x1p52) & 0xFFFFFFFFFFFFFull; }
};

// the classes of a row, each of them to one thread
template <class T>
struct RowSource {
  const T *row;
  int64_t cols;
  template <class F>
  __device__ void each(F f) const {
#pragma unroll 1
    for (int64_t j = threadIdx.x; j < cols; j += kThreads) f((float)row[j], (uint32_t)j);
  }
};

struct Shared {
  unsigned long long hist[1 << kDigit];
  unsigned long long sums[kThreads / 64];
  unsigned long long found, before;
};

template <int NT = kThreads>
__device__ inline unsigned long long block_sum(unsigned long long v, Shared &sh) {
  for (int off = 1; off < 64; off <<= 1) v += __shfl_xor(v, off, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh.sums[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) v += sh.sums[i];
  return v;
}

template <int NT = kThreads>
__device__ inline unsigned long long block_min(unsigned long long v, Shared &sh) {
  for (int off = 1; off < 64; off <<= 1) {
    const unsigned long long o = __shfl_xor(v, off, 64);
    v = o < v ? o : v;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh.sums[threadIdx.x >> 6] = v;
  __syncthreads();
  v = sh.sums[0];
#pragma unroll
  for (int i = 1; i < NT / 64; ++i) v = sh.sums[i] < v ? sh.sums[i] : v;
  return v;
}

// The key of `bits` bits of the first class, in ascending order of the keys, at which the amounts add up to `target` (>= 1);
// all ones where they never do.  visit(f) calls f(key, amount) for this thread's classes.
template <class Visit>
__device__ inline unsigned long long select_key(int bits, unsigned long long target, Shared &sh, Visit visit) {
  unsigned long long prefix = 0;
  const unsigned long long all = bits >= 64 ? ~0ull : (1ull << bits) - 1;
  for (int top = bits; top > 0;) {
    const int width = top < kDigit ? top : kDigit, low = top - width;
    __syncthreads();
    for (int i = threadIdx.x; i < 1 << kDigit; i += kThreads) sh.hist[i] = 0;
    if (threadIdx.x == 0) sh.found = ~0ull;
    __syncthreads();
    visit([&](unsigned long long key, unsigned long long amount) {
      if (amount && (top >= 64 || key >> top == prefix)) atomicAdd(&sh.hist[(key >> low) & ((1u << width) - 1)], amount);
    });
    __syncthreads();
    if (threadIdx.x < 64) {  // 4 values a lane
      unsigned long long x[4], s = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        x[k] = sh.hist[threadIdx.x * 4 + k];
        s += x[k];
      }
      unsigned long long up = s;
      for (int off = 1; off < 64; off <<= 1) {
        const unsigned long long y = __shfl_up(up, off, 64);
        if ((int)threadIdx.x >= off) up += y;
      }
      up -= s;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (up < target && target <= up + x[k]) {
          sh.found = threadIdx.x * 4 + k;
          sh.before = up;
        }
        up += x[k];
      }
    }
    __syncthreads();
    if (sh.found == ~0ull) return all;
    prefix = prefix << width | sh.found;
    target -= sh.before;
    top = low;
  }
  return prefix;
}

struct Params {
  float t, p, m, u;
  int32_t k;  // 0: no top-k
};

// the target of top-p: kept while the mass before is below p times all, up to the first class at which the sum reaches that
__device__ inline unsigned long long mass_target(float p, unsigned long long mass) {
  const double bound = p > 0.0f ? ceil((double)p * (double)mass) : 0.0;
  return bound < 1.0 ? 1ull : (unsigned long long)bound;
}

// the draw's: the first class at which the sum exceeds u times all
__device__ inline unsigned long long draw_target(float u, unsigned long long total) {
  const double at = floor((double)u * (double)total);
  const unsigned long long target = at < (double)total ? (unsigned long long)at + 1 : total;
  return target < total ? target : total;
}

__device__ inline void write_token(const SampleArgs &a, uint64_t r, uint32_t token, float x, const Weights &w, float t, unsigned long long total) {
  a.token[r] = (int32_t)token;
  if (!a.logprob) return;
  const double y = x == w.top ? 0.0 : ((double)x - (double)w.top) / (double)t;
  a.logprob[r] = (float)(y - log(ldexp((double)total, -w.shift)));
}

// The token of one row from the classes that `source` gives out; any row, any parameters.  `first`: the key of the first class.
template <class Source>
__device__ inline void draw_row(const SampleArgs &a, uint64_t r, const Params &q, const Weights &weight, unsigned long long first, const Source &source, Shared &sh) {
  const int bits = 32 + a.index_bits;
  auto order = [&](float x, uint32_t j) { return (unsigned long long)key_of(x) << a.index_bits | j; };
  auto scaled = [&](float x) { return x == weight.top ? ldexp(1.0, weight.shift) : weight.scaled(x); };  // also where top is +inf
  unsigned long long last = ~0ull;  // the last class that is kept
  if (q.k > 0) last = select_key(bits, (unsigned long long)q.k, sh, [&](auto f) { source.each([&](float x, uint32_t j) { f(order(x, j), 1ull); }); });
  if (q.p < 1.0f) {
    unsigned long long mass = 0;
    source.each([&](float x, uint32_t j) { mass += order(x, j) <= last ? weight.units(scaled(x)) : 0; });
    mass = block_sum(mass, sh);
    const unsigned long long end = select_key(bits, mass_target(q.p, mass), sh, [&](auto f) {
      source.each([&](float x, uint32_t j) {
        const unsigned long long o = order(x, j);
        f(o, o <= last ? weight.units(scaled(x)) : 0ull);
      });
    });
    last = end < last ? end : last;
  }
  auto kept = [&](float x, uint32_t j) -> unsigned long long {
    const unsigned long long o = order(x, j);
    if (o > last) return 0;
    const double w = scaled(x);
    return w >= weight.least || o == first ? weight.units(w) : 0;
  };
  unsigned long long total = 0;
  source.each([&](float x, uint32_t j) { total += kept(x, j); });
  total = block_sum(total, sh);
  unsigned long long token;
  if (q.u > 0.0f) {
    token = select_key(a.index_bits, draw_target(q.u, total), sh, [&](auto f) { source.each([&](float x, uint32_t j) { f(j, kept(x, j)); }); });
  } else {  // the first class of any weight, however small
    token = ~0ull;
    source.each([&](float x, uint32_t j) {
      const unsigned long long o = order(x, j);
      const double w = scaled(x);
      if (o <= last && w > 0.0 && (w >= weight.least || o == first) && j < token) token = j;
    });
    token = block_min(token, sh);
  }
  source.each([&](float x, uint32_t j) {
    if (j == token) write_token(a, r, j, x, weight, q.t, total);
  });
}

// ---- rows in a few launches ----------------------------------------------------------------------------
//
//  * k_sample_tops reads the logits once, with as many workgroups as there are, and leaves the largest logit of every kGroup
//    granules.  What follows knows from those the row's largest logit and reads the row again from the caches.
//  * k_sample_list (where top-k is given), a workgroup per row: the k-th largest logit is not below the k-th largest of the
//    groups'.  The classes from that bound on are few; everything else happens among them in LDS.
//  * k_sample_sums (the rows without top-k), kParts workgroups per row: for top-p the weights are summed by kBuckets buckets of
//    the logit.  Weights below (1 - p) / cols of the largest take no part in the buckets: together they are less than 1 - p of
//    the whole.  Without top-p there is one sum; min-p is a bound on the weight.
//  * k_sample_rest, a workgroup per row: the target of top-p falls into one bucket, whose classes are put in order; what is kept
//    of each part is known then, and only the part where the draw falls is read again.  Rows that do not fit any of this
//    (too many classes between a bound and a border, a large k, u <= 0, logits of +inf) are drawn by draw_row from the whole
//    row, to the same result: all sums are the same integers.
// A row that is left to a later kernel has the token kLeft.  One kernel for all of it took 43 us for a row of 128000 classes
// with top-k, where k_sample_list takes 15, and 290 for 512 rows with top-p.

constexpr int kGroup = 32;       // granules
constexpr int kTopsPer = 512;    // granules per workgroup of k_sample_tops
constexpr int kMaxGroups = 4096; // groups whose largest logits fit LDS beside the rest
constexpr int kList = 2048;      // classes kept in LDS
constexpr int kPairs = 512;      // of which all pairs are compared, not sorted digit by digit
constexpr int kBuckets = 512, kParts = 8;
constexpr int kSums = kBuckets + 2;   // the buckets of a part, what is below them, what passes min-p
constexpr uint64_t kBatch = 1024;     // rows whose sums the workspace holds at once
constexpr int32_t kLeft = -2;

struct ListShared {
  float tops[kMaxGroups];
  unsigned int hits[kMaxGroups];
  unsigned long long list[kPairs];   // keys of draw_row's order
  unsigned long long units[kPairs];  // their weights
  Shared sh;
  unsigned int count, nhits, bound;
};

struct RestShared {
  unsigned long long hist[kParts][kBuckets];
  unsigned long long list[kList], units[kPairs];
  Shared sh;
  unsigned int count;
};

__device__ inline Params params_of(const SampleArgs &a, uint64_t r) {
  return Params{a.temperature ? a.temperature[r] : 1.0f, a.top_p ? a.top_p[r] : 1.0f, a.min_p ? a.min_p[r] : 0.0f, a.uniform[r],
                a.top_k && (uint64_t)a.top_k[r] < a.cols ? a.top_k[r] : 0};
}

__device__ inline bool is_greedy(const Params &q) { return !(q.t > 0.0f) || q.m > 1.0f; }  // no class but the first has a weight above 1

__device__ inline void write_none(const SampleArgs &a, uint64_t r) {
  if (threadIdx.x != 0) return;
  a.token[r] = -1;
  if (a.logprob) a.logprob[r] = -INFINITY;
}

// the row's largest logit, from the groups'
template <int NT>
__device__ inline float row_top(const SampleArgs &a, uint64_t r, Shared &sh) {
  float top = -INFINITY;
  for (int64_t g = threadIdx.x; g < a.groups; g += NT) top = fmaxf(top, a.tops[r * a.groups + g]);
  return logit_of((uint32_t)block_min<NT>(key_of(top), sh));
}

// Buckets of equal width in the logit, for top-p: down to weights of (1 - p) / cols, and one power of two more for the
// roundings; kBuckets and beyond: below them.
struct Buckets {
  float top, scale;
  __device__ Buckets(const Params &q, const Weights &w, uint64_t cols) : top(w.top) {
    const double depth = log2((double)cols / (1.0 - (double)q.p)) + 1.0;
    scale = fminf((float)(w.per * kBuckets / (depth > 1.0 ? depth : 1.0)), 0x1p100f);  // 0 times infinity would be no bucket
  }
  __device__ int of(float x) const { return (int)fminf((top - x) * scale, (float)kBuckets); }
};

// is a row of this kind drawn by its sums?
__device__ inline bool by_sums(const Params &q, float top) { return q.k == 0 && q.u > 0.0f && top > -INFINITY && top < INFINITY && !is_greedy(q); }

template <class T>
__global__ void __launch_bounds__(256) k_sample_tops(SampleArgs a) {
  constexpr int K = 16 / sizeof(T);
  const Chunks<T> row(static_cast<const T *>(a.logits) + (uint64_t)blockIdx.y * a.stride, (int64_t)a.cols);
  const int64_t c0 = (int64_t)blockIdx.x * kTopsPer + threadIdx.x;
  vec_t<T, K> x[kTopsPer / 256];
#pragma unroll
  for (int i = 0; i < kTopsPer / 256; ++i) {
    x[i] = (T)-INFINITY;
    if (c0 + i * 256 < row.count) x[i] = row.load(c0 + i * 256, (T)-INFINITY);
  }
#pragma unroll
  for (int i = 0; i < kTopsPer / 256; ++i) {
    float m = -INFINITY;
#pragma unroll
    for (int k = 0; k < K; ++k) m = fmaxf(m, (float)x[i][k]);
    for (int off = 1; off < kGroup; off <<= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
    const int64_t g = (c0 + i * 256) / kGroup;
    if (threadIdx.x % kGroup == 0 && g < a.groups) a.tops[(uint64_t)blockIdx.y * a.groups + g] = m;
  }
}

// the classes in the list, each of them to one thread
struct ListSource {
  const unsigned long long *list;
  int count, index_bits;
  template <class F>
  __device__ void each(F f) const {
    for (int i = threadIdx.x; i < count; i += kThreads) f(logit_of((uint32_t)(list[i] >> index_bits)), (uint32_t)(list[i] & ((1ull << index_bits) - 1)));
  }
};

// sum of `v` over the `each` threads that share a class
template <class V>
__device__ inline V among(V v, int each) {
  for (int off = 1; off < each; off <<= 1) v += __shfl_xor(v, off, 64);
  return v;
}

// All filters and the draw among up to kPairs classes: every class against every other, `each` threads a class.
__device__ inline void draw_pairs(const SampleArgs &a, uint64_t r, const Params &q, const Weights &weight, unsigned long long first, ListShared &s, int count) {
  int log_each = 0;
  while (log_each < 6 && (count << (log_each + 1)) <= kThreads) ++log_each;
  const int each = 1 << log_each, mine = threadIdx.x >> log_each, part = threadIdx.x & (each - 1);
  const unsigned long long mask = (1ull << a.index_bits) - 1;
  const bool in = mine < count;
  const unsigned long long o = in ? s.list[mine] : ~0ull;
  const float x = logit_of((uint32_t)(o >> a.index_bits));
  const double w = in ? weight.scaled(x) : 0.0;
  const unsigned long long units = in ? weight.units(w) : 0;
  int rank = 0;
  for (int i = part; i < count; i += each) rank += s.list[i] < o;
  rank = among(rank, each);
  const bool top = in && (q.k <= 0 || rank < q.k);
  if (in && part == 0) s.units[mine] = top ? units : 0;
  const unsigned long long mass = block_sum(top && part == 0 ? units : 0, s.sh);
  bool kept = top;
  if (q.p < 1.0f) {
    unsigned long long before = 0;
    for (int i = part; i < count; i += each) before += s.list[i] < o ? s.units[i] : 0;
    before = among(before, each);
    kept = kept && before < mass_target(q.p, mass);
  }
  kept = kept && (w >= weight.least || o == first);
  __syncthreads();
  if (in && part == 0) s.units[mine] = kept ? units : 0;
  const unsigned long long total = block_sum(kept && part == 0 ? units : 0, s.sh);
  const unsigned long long target = draw_target(q.u, total);
  unsigned long long upto = 0;
  for (int i = part; i < count; i += each) upto += (s.list[i] & mask) <= (o & mask) ? s.units[i] : 0;
  upto = among(upto, each);
  const unsigned long long token = block_min(kept && upto >= target ? o & mask : ~0ull, s.sh);
  if (kept && part == 0 && (o & mask) == token) write_token(a, r, (uint32_t)token, x, weight, q.t, total);
}

// The first class, in the order of the indexes, at which the amounts of the granules [c0, c1) reach `target`; visit(x, j) is
// a class's amount, hit(x, j) gets the class.
template <class T, class Amount, class Hit>
__device__ inline void find_class(const Chunks<T, 8> &row, int64_t c0, int64_t c1, unsigned long long target, Shared &sh, Amount amount, Hit hit) {
  constexpr int K = 8 / sizeof(T);
#pragma unroll 1
  for (int64_t b = c0; b < c1; b += kThreads) {
    const int64_t c = b + threadIdx.x;
    vec_t<T, K> x = (T)-INFINITY;
    if (c < c1) x = row.load(c, (T)-INFINITY);
    unsigned long long u[K], mine = 0;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      u[k] = amount((float)x[k], c * K + k - row.lead);
      mine += u[k];
    }
    unsigned long long up = mine;
    for (int off = 1; off < 64; off <<= 1) {
      const unsigned long long y = __shfl_up(up, off, 64);
      if ((int)(threadIdx.x & 63) >= off) up += y;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 63) sh.sums[threadIdx.x >> 6] = up;
    __syncthreads();
    unsigned long long all = 0;
    for (int i = 0; i < kThreads / 64; ++i) {
      if (i == (int)(threadIdx.x >> 6)) up += all;
      all += sh.sums[i];
    }
    if (all >= target) {  // uniform
      unsigned long long sum = up - mine;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (sum < target && target <= sum + u[k]) hit((float)x[k], c * K + k - row.lead);
        sum += u[k];
      }
      return;
    }
    target -= all;
  }
}

// granules of a part of a row
struct Part {
  int64_t first, last;
  __device__ Part(int64_t count, int part) {
    const int64_t span = (count + kParts - 1) / kParts;
    first = part * span < count ? part * span : count;
    last = first + span < count ? first + span : count;
  }
};

template <class T>
__global__ void __launch_bounds__(256) k_sample_sums(SampleArgs a, uint64_t r0) {
  constexpr int K = 8 / sizeof(T);  // narrow granules: the arithmetic is the bound, and eight classes at once take too many registers
  __shared__ unsigned long long hist[kBuckets];
  __shared__ Shared sh;
  const uint64_t r = r0 + blockIdx.y;
  if (a.top_k && a.token[r] != kLeft) return;
  const Params q = params_of(a, r);
  const float top = row_top<256>(a, r, sh);
  if (!by_sums(q, top)) return;
  const Weights weight(top, q.t, q.m, a.shift);
  const Chunks<T, 8> row(static_cast<const T *>(a.logits) + r * a.stride, (int64_t)a.cols);
  const Part part(row.count, (int)blockIdx.x);
  const T none = (T)-INFINITY;
  unsigned long long *to = a.sums + (blockIdx.y * kParts + blockIdx.x) * (uint64_t)kSums;
  unsigned long long rest = 0, above = 0;  // below the buckets; passing min-p
  if (q.p < 1.0f) {
    const Buckets buckets(q, weight, a.cols);
    for (int i = threadIdx.x; i < kBuckets; i += 256) hist[i] = 0;
    __syncthreads();
    for (int64_t c = part.first + threadIdx.x; c < part.last; c += 256) {
      const vec_t<T, K> x = row.load(c, none);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const double w = weight.scaled((float)x[k]);
        const unsigned long long u = weight.units(w);
        const int b = buckets.of((float)x[k]);
        if (b < kBuckets) atomicAdd(&hist[b], u);
        else rest += u;
        if (q.m > 0.0f) above += w >= weight.least ? u : 0;
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kBuckets; i += 256) to[i] = hist[i];
    rest = block_sum<256>(rest, sh);
  }
  if (q.p < 1.0f && q.m > 0.0f) {
    above = block_sum<256>(above, sh);
  } else if (!(q.p < 1.0f)) {
    for (int64_t c = part.first + threadIdx.x; c < part.last; c += 256) {
      const vec_t<T, K> x = row.load(c, none);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const double w = weight.scaled((float)x[k]);
        above += w >= weight.least ? weight.units(w) : 0;
      }
    }
    above = block_sum<256>(above, sh);
  }
  if (threadIdx.x == 0) {
    to[kBuckets] = rest;
    to[kBuckets + 1] = above;
  }
}

// A row with its parts' sums; false where its border's bucket holds too many classes.
template <class T>
__device__ inline bool draw_sums(const SampleArgs &a, uint64_t r, const unsigned long long *sums, const Params &q, const Weights &weight, RestShared &s) {
  const Chunks<T, 8> row(static_cast<const T *>(a.logits) + r * a.stride, (int64_t)a.cols);
  bool nucleus = q.p < 1.0f;
  const Buckets buckets(q, weight, a.cols);
  int border = 0;
  unsigned long long last = 0;
  if (nucleus) {
    unsigned long long mine = 0, above = 0;
    static_assert(kThreads == kBuckets, "a bucket each");
#pragma unroll
    for (int part = 0; part < kParts; ++part) {
      const unsigned long long v = sums[part * kSums + threadIdx.x];
      s.hist[part][threadIdx.x] = v;
      mine += v;
      above += sums[part * kSums + kBuckets + 1];
    }
    unsigned long long up = mine;  // of the buckets up to this one
    for (int off = 1; off < 64; off <<= 1) {
      const unsigned long long y = __shfl_up(up, off, 64);
      if ((int)(threadIdx.x & 63) >= off) up += y;
    }
    if (threadIdx.x == 0) {
      s.count = 0;
      s.sh.found = ~0ull;
    }
    if ((threadIdx.x & 63) == 63) s.sh.sums[threadIdx.x >> 6] = up;
    __syncthreads();
    unsigned long long total = 0;
    for (int i = 0; i < kThreads / 64; ++i) {
      if (i == (int)(threadIdx.x >> 6)) up += total;
      total += s.sh.sums[i];
    }
    for (int part = 0; part < kParts; ++part) total += sums[part * kSums + kBuckets];
    const unsigned long long target = mass_target(q.p, total);
    // where the target is beyond all that passes min-p, top-p keeps all of that and more
    nucleus = !(q.m > 0.0f && target > above);
    if (nucleus) {
      if (up - mine < target && target <= up) {
        s.sh.found = threadIdx.x;
        s.sh.before = up - mine;
      }
      __syncthreads();
      if (s.sh.found == ~0ull) return false;
      border = (int)s.sh.found;
      const unsigned long long within = target - s.sh.before;
      // the classes of the bucket that the target falls into
      const Chunks<T> wide(static_cast<const T *>(a.logits) + r * a.stride, (int64_t)a.cols);
      constexpr int K = 16 / sizeof(T), kAhead = 4;
      for (int64_t c0 = threadIdx.x; c0 < wide.count; c0 += kAhead * kThreads) {
        vec_t<T, K> x[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          x[u] = (T)-INFINITY;
          if (c0 + u * kThreads < wide.count) x[u] = wide.load(c0 + u * kThreads, (T)-INFINITY);
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
#pragma unroll
          for (int k = 0; k < K; ++k) {
            if (buckets.of((float)x[u][k]) != border) continue;  // what is not of the row is below all buckets
            const unsigned at = atomicAdd(&s.count, 1u);
            if (at < (unsigned)kList) s.list[at] = (unsigned long long)key_of((float)x[u][k]) << a.index_bits | (unsigned long long)((c0 + u * kThreads) * K + k - wide.lead);
          }
        }
      }
      __syncthreads();
      const int count = (int)(s.count < (unsigned)kList + 1 ? s.count : (unsigned)kList + 1);
      if (count > kList) return false;
      const ListSource list{s.list, count, a.index_bits};
      if (count <= kPairs) {
        int log_each = 0;
        while (log_each < 6 && (count << (log_each + 1)) <= kThreads) ++log_each;
        const int each = 1 << log_each, me = threadIdx.x >> log_each;
        const unsigned long long o = me < count ? s.list[me] : ~0ull;
        if (threadIdx.x < count) s.units[threadIdx.x] = weight.units(weight.scaled(logit_of((uint32_t)(s.list[threadIdx.x] >> a.index_bits))));
        __syncthreads();
        unsigned long long upto = 0;
        for (int i = threadIdx.x & (each - 1); i < count; i += each) upto += s.list[i] <= o ? s.units[i] : 0;
        upto = among(upto, each);
        last = block_min(me < count && upto >= within ? o : ~0ull, s.sh);
      } else {
        last = select_key(32 + a.index_bits, within, s.sh, [&](auto f) {
          list.each([&](float x, uint32_t j) { f((unsigned long long)key_of(x) << a.index_bits | j, weight.units(weight.scaled(x))); });
        });
      }
      // what is kept of every part
      if (threadIdx.x < kParts) s.hist[threadIdx.x][border] = 0;
      __syncthreads();
      const int64_t span = (row.count + kParts - 1) / kParts;
      list.each([&](float x, uint32_t j) {
        if (((unsigned long long)key_of(x) << a.index_bits | j) > last) return;
        atomicAdd(&s.hist[((int64_t)j + row.lead) / (8 / (int)sizeof(T)) / span][border], weight.units(weight.scaled(x)));
      });
      __syncthreads();
      static_assert(kThreads / 64 == kParts, "a wave each");
      unsigned long long kept = 0;
      for (int b = threadIdx.x & 63; b <= border; b += 64) kept += s.hist[threadIdx.x / 64][b];
      for (int off = 1; off < 64; off <<= 1) kept += __shfl_xor(kept, off, 64);
      __syncthreads();
      if ((threadIdx.x & 63) == 0) s.units[threadIdx.x / 64] = kept;
    }
  }
  if (!nucleus && threadIdx.x < kParts) s.units[threadIdx.x] = sums[threadIdx.x * kSums + kBuckets + 1];
  __syncthreads();
  unsigned long long total = 0;
  for (int part = 0; part < kParts; ++part) total += s.units[part];
  unsigned long long at = draw_target(q.u, total);
  int part = 0;
  while (part < kParts - 1 && at > s.units[part]) at -= s.units[part++];
  const Part span(row.count, part);
  find_class(row, span.first, span.last, at, s.sh,
             [&](float x, int64_t j) -> unsigned long long {
               const double w = weight.scaled(x);
               bool kept = w >= weight.least;
               if (nucleus) {
                 const int b = buckets.of(x);
                 kept = b < border || (b == border && ((unsigned long long)key_of(x) << a.index_bits | (unsigned long long)j) <= last);
               }
               return kept ? weight.units(w) : 0;
             },
             [&](float x, int64_t j) { write_token(a, r, (uint32_t)j, x, weight, q.t, total); });
  return true;
}

template <class T>
__global__ void __launch_bounds__(kThreads, 4) k_sample_list(SampleArgs a) {
  constexpr int K = 16 / sizeof(T);
  __shared__ ListShared s;
  const T none = (T)-INFINITY;
  for (uint64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    __syncthreads();
    const Chunks<T> row(static_cast<const T *>(a.logits) + r * a.stride, (int64_t)a.cols);
    const Params q = params_of(a, r);
    const int64_t small = (row.count + kGroup - 1) / kGroup, size = (small + kMaxGroups - 1) / kMaxGroups;
    const int groups = (int)((small + size - 1) / size);  // of `size` times kGroup granules
    // the groups' largest logits, and the row's
    float top = -INFINITY;
    for (int g = threadIdx.x; g < groups; g += kThreads) {
      float m = -INFINITY;
      for (int64_t i = g * size; i < (g + 1) * size && i < small; ++i) m = fmaxf(m, a.tops[r * a.groups + i]);
      s.tops[g] = m;
      top = fmaxf(top, m);
    }
    if (threadIdx.x == 0) s.count = s.nhits = 0;
    top = logit_of((uint32_t)block_min(key_of(top), s.sh));
    if (top == -INFINITY) {  // uniform, as everything that skips a barrier here
      write_none(a, r);
      continue;
    }
    const bool greedy = is_greedy(q);
    const int want = greedy ? 1 : q.k;
    if (!greedy && (want == 0 || want > groups || !(q.u > 0.0f) || top == INFINITY)) {
      if (threadIdx.x == 0) a.token[r] = kLeft;
      continue;
    }
    // the want-th largest of the groups' largest logits: by one wave, bisecting their keys; a bound that a few more reach does
    // as well
    if (threadIdx.x < 64) {
      uint32_t lo = key_of(top), hi = key_of(-INFINITY);  // the bound's key is between them
      uint32_t mine[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) mine[i] = (int)threadIdx.x + 64 * i < groups ? key_of(s.tops[threadIdx.x + 64 * i]) : 0xFFFFFFFFu;
      while (lo < hi) {
        const uint32_t mid = lo + ((hi - lo) >> 1);
        int have = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) have += __popcll(__ballot(mine[i] <= mid));
        for (int g = 512 + threadIdx.x; g < (groups + 63) / 64 * 64; g += 64) have += __popcll(__ballot(g < groups && key_of(s.tops[g]) <= mid));
        if (have >= want) hi = mid;
        else lo = mid + 1;
        if (have >= want && have <= want + want / 8) break;
      }
      if (threadIdx.x == 0) s.bound = hi;
    }
    __syncthreads();
    const float bound = logit_of(s.bound);
    for (int g = threadIdx.x; g < groups; g += kThreads)
      if (s.tops[g] >= bound) s.hits[atomicAdd(&s.nhits, 1u)] = g;
    __syncthreads();
    // the classes from the bound on
    unsigned long long first = ~0ull;
    const unsigned per = (unsigned)(size * kGroup), granules = s.nhits * per;  // at most the row's 2^31 / K and kMaxGroups' rounding
    for (unsigned i = threadIdx.x; i < granules; i += 4 * kThreads) {
      vec_t<T, K> x[4];
      int64_t c[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const unsigned at = i + u * kThreads;
        c[u] = at < granules ? (int64_t)s.hits[at / per] * per + at % per : row.count;
        if (c[u] < row.count) x[u] = row.load(c[u], none);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (c[u] >= row.count) continue;
#pragma unroll
        for (int k = 0; k < K; ++k) {
          const float v = (float)x[u][k];
          const int64_t j = c[u] * K + k - row.lead;
          if (v >= bound && j >= 0 && j < row.cols) {
            const unsigned at = atomicAdd(&s.count, 1u);
            const unsigned long long o = (unsigned long long)key_of(v) << a.index_bits | (unsigned long long)j;
            if (at < (unsigned)kPairs) s.list[at] = o;
            first = o < first ? o : first;
          }
        }
      }
    }
    first = block_min(first, s.sh);
    if (greedy) {
      if (threadIdx.x == 0) {
        a.token[r] = (int32_t)(first & ((1ull << a.index_bits) - 1));
        if (a.logprob) a.logprob[r] = 0.0f;
      }
    } else if (s.count <= (unsigned)kPairs) {
      draw_pairs(a, r, q, Weights(top, q.t, q.m, a.shift), first, s, (int)s.count);
    } else if (threadIdx.x == 0) {
      a.token[r] = kLeft;
    }
  }
}

template <class T>
__global__ void __launch_bounds__(kThreads) k_sample_rest(SampleArgs a, uint64_t r0, uint64_t r1) {
  __shared__ RestShared s;
  const uint64_t r = r0 + blockIdx.x;
  if (r >= r1 || (a.top_k && a.token[r] != kLeft)) return;
  const Params q = params_of(a, r);
  const float top = row_top<kThreads>(a, r, s.sh);
  if (top == -INFINITY) {
    write_none(a, r);
    return;
  }
  const Weights weight(top, q.t, q.m, a.shift);
  __syncthreads();
  if (by_sums(q, top) && draw_sums<T>(a, r, a.sums + blockIdx.x * (uint64_t)(kParts * kSums), q, weight, s)) return;
  __syncthreads();
  const Chunks<T> row(static_cast<const T *>(a.logits) + r * a.stride, (int64_t)a.cols);
  unsigned long long first = ~0ull;  // the lowest index of the largest logit
  for (int64_t c = threadIdx.x; c < row.count && first == ~0ull; c += kThreads) {
    const vec_t<T, 16 / sizeof(T)> x = row.load(c, (T)-INFINITY);
#pragma unroll
    for (int k = 16 / sizeof(T) - 1; k >= 0; --k)
      if ((float)x[k] == top) first = (unsigned long long)(c * (int64_t)(16 / sizeof(T)) + k - row.lead);
  }
  first = block_min(first, s.sh);
  if (is_greedy(q)) {
    if (threadIdx.x == 0) {
      a.token[r] = (int32_t)first;
      if (a.logprob) a.logprob[r] = 0.0f;
    }
    return;
  }
  draw_row(a, r, q, weight, (unsigned long long)key_of(top) << a.index_bits | first, RowSource<T>{row.base + row.lead, row.cols}, s.sh);
}

static uint64_t tops_groups(uint64_t cols, uint64_t per) { return ((cols + per - 1) / per + 1 + kGroup - 1) / kGroup; }

static uint64_t tops_bytes(uint64_t rows, uint64_t groups) { return round_up(rows * groups * sizeof(float), 256); }

template <class T>
static int sample(admm_ctx *ctx, SampleArgs a, void *workspace) {
  a.groups = (int64_t)tops_groups(a.cols, 16 / sizeof(T));
  a.tops = static_cast<float *>(workspace);
  a.sums = reinterpret_cast<unsigned long long *>(static_cast<char *>(workspace) + tops_bytes(a.rows, a.groups));
  const dim3 block(kThreads);
  const unsigned per_row = (unsigned)((a.groups * kGroup + kTopsPer - 1) / kTopsPer);
  for (uint64_t r = 0; r < a.rows; r += 65535) {  // rows are the second dimension of the grid
    SampleArgs b = a;
    b.logits = static_cast<const T *>(a.logits) + r * a.stride;
    b.tops = a.tops + r * a.groups;
    const unsigned rows = (unsigned)(a.rows - r < 65535 ? a.rows - r : 65535);
    hipLaunchKernelGGL(k_sample_tops<T>, dim3(per_row, rows), dim3(256), 0, ctx->stream, b);
  }
  if (a.top_k) hipLaunchKernelGGL(k_sample_list<T>, dim3(blocks_for(a.rows, 1)), block, 0, ctx->stream, a);
  for (uint64_t r = 0; r < a.rows; r += kBatch) {
    const uint64_t end = r + kBatch < a.rows ? r + kBatch : a.rows;
    hipLaunchKernelGGL(k_sample_sums<T>, dim3(kParts, (unsigned)(end - r)), dim3(256), 0, ctx->stream, a, r);
    hipLaunchKernelGGL(k_sample_rest<T>, dim3((unsigned)(end - r)), block, 0, ctx->stream, a, r, end);
  }
  ADMM_HIP_CHECK(hipGetLastError());
  return ADMM_OK;
}

}  // namespace admm_impl

using namespace admm_impl;

extern "C" int admm_sample_workspace(uint64_t rows, uint64_t cols, uint64_t *bytes) {
  ADMM_REQUIRE(bytes, "admm_sample_workspace: bytes is NULL");
  ADMM_REQUIRE(rows < (1ull << 40) && cols < (1ull << 31), "admm_sample_workspace: %llu x %llu logits", (unsigned long long)rows,
               (unsigned long long)cols);
  // enough for logits of any type: granules of four floats are the most
  *bytes = tops_bytes(rows, tops_groups(cols, 4)) + (rows < kBatch ? rows : kBatch) * (kParts * kSums * sizeof(unsigned long long));
  return ADMM_OK;
}

extern "C" int admm_sample(admm_ctx *ctx, const admm_mat *logits, const admm_sample_params *params, const float *uniform, int32_t *token,
                           float *logprob, void *workspace, uint64_t workspace_bytes) {
  ADMM_REQUIRE(ctx, "admm_sample: ctx is NULL");
  ADMM_TRY(check_mat(logits, "admm_sample", "logits"));
  if (logits->rows == 0) return ADMM_OK;
  ADMM_REQUIRE(logits->cols > 0 && logits->cols < (1ull << 31), "admm_sample: %llu classes", (unsigned long long)logits->cols);
  ADMM_REQUIRE(uniform && token, "admm_sample: uniform or token is NULL");
  uint64_t need = 0;
  ADMM_TRY(admm_sample_workspace(logits->rows, logits->cols, &need));
  ADMM_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && reinterpret_cast<uintptr_t>(workspace) % 256 == 0),
               "admm_sample: the workspace is NULL, not on 256 bytes or smaller than %llu bytes", (unsigned long long)need);
  OnDevice on(ctx->device);
  ADMM_HIP_CHECK(on.error);
  KernelTimer t(ctx, ADMM_K_SAMPLE);
  SampleArgs a = {};
  a.logits = logits->data;
  a.stride = logits->stride;
  a.rows = logits->rows;
  a.cols = logits->cols;
  if (params) {
    a.temperature = params->temperature;
    a.top_k = params->top_k;
    a.top_p = params->top_p;
    a.min_p = params->min_p;
  }
  a.uniform = uniform;
  a.token = token;
  a.logprob = logprob;
  a.index_bits = 1;
  while ((1ull << a.index_bits) < a.cols) ++a.index_bits;
  a.shift = 62 - a.index_bits < 51 ? 62 - a.index_bits : 51;
  return logits->type == ADMM_F32 ? sample<float>(ctx, a, workspace) : logits->type == ADMM_BF16 ? sample<bf16_t>(ctx, a, workspace) : sample<f16_t>(ctx, a, workspace);
}
