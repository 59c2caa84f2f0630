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
constexpr int kDigit = 9;  // a value of the digit for every thread
static_assert(1 << kDigit == kThreads, "");

struct SampleArgs {
  const void *logits;
  uint64_t stride, rows, cols;
  const float *temperature, *top_p, *min_p, *uniform;
  const int32_t *top_k;
  int32_t *token;
  float *logprob;
  int index_bits, shift;  // 2^index_bits >= cols; S
  float *tops;            // [rows][groups] largest logits of 2^group_log2 granules each
  int64_t groups;
  int group_log2;
  unsigned long long *sums;  // [rows of a batch][kParts][kSums]
  int split;                 // workgroups per part that add to its sums; more than one where there are few rows
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

// p f + c.  The compiler's own choice for a polynomial is the form that adds to its third operand in place, with a copy of
// the coefficient before every step: a tenth of k_sample_sums.
__device__ inline double fma3(double p, double f, double c) {
  double d;
  asm("v_fma_f64 %0, %1, %2, %3" : "=v"(d) : "v"(p), "v"(f), "v"(c));
  return d;
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
  // The exponent of a class' weight, at least -64 (less than half a unit for every S); NaN counts as -inf.  A top of +inf is
  // not meant here.
  __device__ double exponent(float x) const { return fmax(((double)x - (double)top) * per, -64.0); }
  // 2^(y + S): the integer part n of y is what is left in the low bits of y + 1.5 2^52 and goes to the exponent of 2^S times a
  // polynomial of the rest.  That is 1 + f q(f), q through the Chebyshev points of (2^f - 1) / f on [-1/2, 1/2]: off by
  // 2.2e-12 of the weight at most (the draw from a flat row of 2^17 classes sees 8e-6 a class), and 1 where f is 0.
  __device__ double scaled(double y) const {
    const double t = y + 0x1.8p52, f = y - (t - 0x1.8p52);
    double p = 1.325080551750225e-06;
    p = fma3(p, f, 1.5303700711365693e-05);
    p = fma3(p, f, 0.00015403475186530786);
    p = fma3(p, f, 0.0013333478473685416);
    p = fma3(p, f, 0.00961812913523614);
    p = fma3(p, f, 0.055504109063258665);
    p = fma3(p, f, 0.24022650695888503);
    p = fma3(p, f, 0.6931471805568324);
    p = fma3(p, f, 1.0);
    const int n = (int)(unsigned)__double_as_longlong(t);
    return __hiloint2double(__double2hiint(p) + ((n + shift) << 20), __double2loint(p));
  }
  __device__ double scaled(float x) const { return scaled(exponent(x)); }
  // rounded to an integer below 2^52: what is left in the mantissa after 2^52 is added
  __device__ static unsigned long long units(double v) { return __double_as_longlong(v + 0x1p52) & 0xFFFFFFFFFFFFFull; }
};

// the classes of a row, each of them to one thread
template <class T>
struct RowSource {
  const T *row;
  int cols;
  template <class F>
  __device__ void each(F f) const {
#pragma unroll 1
    for (int64_t j = threadIdx.x; j < cols; j += kThreads) f((float)row[j], (uint32_t)j);
  }
};

struct Shared {
  unsigned long long hist[1 << kDigit];
  unsigned long long sums[kThreads / 64], tops[kThreads / 64];
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

// Sums over sh.hist up to and with every thread's value: where they reach `target` goes to sh.found (else all ones), what comes
// before it to sh.before; everybody waits.  Returns the sum of all.
__device__ inline unsigned long long find_value(Shared &sh, unsigned long long v, unsigned long long target) {
  unsigned long long up = v;
  for (int off = 1; off < 64; off <<= 1) {
    const unsigned long long y = __shfl_up(up, off, 64);
    if ((int)(threadIdx.x & 63) >= off) up += y;
  }
  if (threadIdx.x == 0) sh.found = ~0ull;
  if ((threadIdx.x & 63) == 63) sh.sums[threadIdx.x >> 6] = up;
  __syncthreads();
  unsigned long long all = 0;
#pragma unroll
  for (int i = 0; i < kThreads / 64; ++i) {
    if (i == (int)(threadIdx.x >> 6)) up += all;
    all += sh.sums[i];
  }
  if (up - v < target && target <= up) {
    sh.found = threadIdx.x;
    sh.before = up - v;
  }
  __syncthreads();
  return all;
}

// The key of `bits` bits of the first class, in ascending order of the keys, at which the amounts add up to `target` (>= 1);
// all ones where they never do.  visit(f) calls f(key, amount) for this thread's classes.
template <class Visit>
__device__ inline unsigned long long select_key(int bits, unsigned long long target, Shared &sh, Visit visit) {
  unsigned long long prefix = 0;
  for (int top = bits; top > 0;) {
    const int width = top < kDigit ? top : kDigit, low = top - width;
    __syncthreads();
    sh.hist[threadIdx.x] = 0;
    __syncthreads();
    visit([&](unsigned long long key, unsigned long long amount) {
      if (amount && (top >= 64 || key >> top == prefix)) atomicAdd(&sh.hist[(key >> low) & ((1u << width) - 1)], amount);
    });
    __syncthreads();
    find_value(sh, sh.hist[threadIdx.x], target);
    if (sh.found == ~0ull) return ~0ull;
    prefix = prefix << width | sh.found;
    target -= sh.before;
    top = low;
  }
  return prefix;
}

// The same among classes that the threads hold, kHeld each, with keys that differ; an amount of 0: not among them.  The range
// of the keys that are left is cut into 512 until there is one.
constexpr int kHeld = 4;
__device__ inline unsigned long long select_held(const unsigned long long (&key)[kHeld], const unsigned long long (&amount)[kHeld],
                                                 unsigned long long target, Shared &sh) {
  bool on[kHeld];
#pragma unroll
  for (int i = 0; i < kHeld; ++i) on[i] = amount[i] != 0;
  for (;;) {
    unsigned long long lo = ~0ull, hi = 0;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      if (on[i] && key[i] < lo) lo = key[i];
      if (on[i] && key[i] > hi) hi = key[i];
    }
    for (int off = 1; off < 64; off <<= 1) {
      const unsigned long long l = __shfl_xor(lo, off, 64), h = __shfl_xor(hi, off, 64);
      lo = l < lo ? l : lo;
      hi = h > hi ? h : hi;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
      sh.sums[threadIdx.x >> 6] = lo;
      sh.tops[threadIdx.x >> 6] = hi;
    }
    sh.hist[threadIdx.x] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kThreads / 64; ++i) {
      lo = sh.sums[i] < lo ? sh.sums[i] : lo;
      hi = sh.tops[i] > hi ? sh.tops[i] : hi;
    }
    if (lo >= hi) return lo;  // one, or none: all ones
    const int bits = 64 - __clzll((long long)(lo ^ hi)), shift = bits > kDigit ? bits - kDigit : 0;
    const unsigned long long from = lo >> shift;
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
      if (on[i]) atomicAdd(&sh.hist[(key[i] >> shift) - from], amount[i]);
    __syncthreads();
    find_value(sh, sh.hist[threadIdx.x], target);
    if (sh.found == ~0ull) return ~0ull;
    target -= sh.before;
    const unsigned long long at = from + sh.found;
    if (shift == 0) return at;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) on[i] = on[i] && key[i] >> shift == at;
  }
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
      const bool any = x == weight.top || ((double)x - (double)weight.top) * weight.per > -1075.0;
      if (o <= last && any && (scaled(x) >= weight.least || o == first) && j < token) token = j;
    });
    token = block_min(token, sh);
  }
  source.each([&](float x, uint32_t j) {
    if (j == token) write_token(a, r, j, x, weight, q.t, total);
  });
}

// ---- rows in a few launches ----------------------------------------------------------------------------
//
//  * k_sample_tops reads the logits once, with as many workgroups as there are, and leaves the largest logit of every group
//    of granules.  What follows knows from those the row's largest logit and reads the row again from the caches.
//  * k_sample_list (where top-k is given), a workgroup per row: the k-th largest logit is not below the k-th largest of the
//    groups'.  The classes from that bound on are few; everything else happens among them in LDS.
//  * k_sample_sums (the rows without top-k), kParts workgroups per row, or up to eight times as many for few rows: for top-p
//    the weights are summed by kBuckets buckets of the logit.  Weights below (1 - p) / cols of the largest take no part in the buckets: together they are less than 1 - p of
//    the whole.  Without top-p there is one sum; min-p is a bound on the weight.
//  * k_sample_rest, a workgroup per row: the target of top-p falls into one bucket, whose classes are put in order; what is kept
//    of each part is known then, and only the part where the draw falls is read again.  Rows that do not fit any of this
//    (too many classes between a bound and a border, a large k, u <= 0, logits of +inf) are drawn by draw_row from the whole
//    row, to the same result: all sums are the same integers.
// A row that is left to a later kernel has the token kLeft.  One kernel for all of it took 43 us for a row of 128000 classes
// with top-k, where k_sample_list takes 18, and 290 for 512 rows with top-p.  512 rows of 128000 in 16 bits with top-p: tops 21
// us (131 MB at 6.2 TB/s), sums 75 (bound by arithmetic: 33 instructions a class, most of them in 64 bits, issued three quarters
// of the time), rest 58 (17 for the border's bucket, 7 for the draw, 12 of steps that wait for each other; rows that share a CU with
// a slower one end last).

constexpr int kTopsPer = 512;    // granules per workgroup of k_sample_tops
constexpr int kMaxGroups = 4096; // groups whose largest logits fit LDS beside the rest
constexpr int kList = kHeld * kThreads;  // classes kept in LDS
constexpr int kPairs = 128;      // up to so many all pairs are compared: 3 us for the filters and the draw, where selecting takes 12
constexpr int kBuckets = 512, kParts = 8;
constexpr int kSums = kBuckets + 2;   // the buckets of a part, what is below them, what passes min-p
constexpr uint64_t kBatch = 1024;     // rows whose sums the workspace holds at once
constexpr int32_t kLeft = -2;

struct ListShared {
  float tops[kMaxGroups];
  unsigned int hits[kMaxGroups];
  unsigned long long list[kList];    // keys of draw_row's order
  unsigned long long units[kPairs];  // their weights
  Shared sh;
  unsigned int count, nhits, bound;
};

struct RestShared {
  unsigned long long hist[kParts][kBuckets];
  unsigned long long list[kList], units[kParts];
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

// Buckets of equal width in the weight's exponent, for top-p: down to weights of (1 - p) / cols, and one power of two more for
// the roundings; kBuckets and beyond: below them.
struct Buckets {
  double per;
  __device__ Buckets(const Params &q, uint64_t cols) {
    const double depth = log2((double)cols / (1.0 - (double)q.p)) + 1.0;
    per = -kBuckets / (depth > 1.0 ? depth : 1.0);
  }
  // y in [-64, 0]: the rounded product is what is left in the low bits after 2^52 is added
  __device__ unsigned of(double y) const { return (unsigned)__double_as_longlong(fma(y, per, 0x1p52)); }
};

// is a row of this kind drawn by its sums?
__device__ inline bool by_sums(const Params &q, float top) { return q.k == 0 && q.u > 0.0f && top > -INFINITY && top < INFINITY && !is_greedy(q); }

template <class T>
__global__ void __launch_bounds__(256) k_sample_tops(SampleArgs a) {
  constexpr int K = 16 / sizeof(T);
  const Chunks<T> row(static_cast<const T *>(a.logits) + (uint64_t)blockIdx.y * a.stride, (int)a.cols);
  if (a.split > 1)  // the sums are added to by several workgroups of the next launch
    for (unsigned i = blockIdx.x * 256 + threadIdx.x; i < kParts * kSums; i += gridDim.x * 256) a.sums[blockIdx.y * (uint64_t)(kParts * kSums) + i] = 0;
  const int c0 = (int)(blockIdx.x * kTopsPer + threadIdx.x);
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
    for (int off = 1; off < 1 << a.group_log2; off <<= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
    const int g = (c0 + i * 256) >> a.group_log2;
    if ((threadIdx.x & ((1u << a.group_log2) - 1)) == 0 && g < a.groups) a.tops[(uint64_t)blockIdx.y * a.groups + g] = m;
  }
}

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

// what a thread holds of a list
struct Held {
  unsigned long long o[kHeld], units[kHeld];
  double w[kHeld];
  __device__ Held(const unsigned long long *list, int count, const Weights &weight, int index_bits) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int at = threadIdx.x + i * kThreads;
      o[i] = at < count ? list[at] : ~0ull;
      w[i] = at < count ? weight.scaled(logit_of((uint32_t)(o[i] >> index_bits))) : 0.0;
      units[i] = Weights::units(w[i]);
    }
  }
};

// All filters and the draw among up to kList classes.
__device__ inline void draw_held(const SampleArgs &a, uint64_t r, const Params &q, const Weights &weight, unsigned long long first,
                                 const unsigned long long *list, int count, Shared &sh) {
  Held h(list, count, weight, a.index_bits);
  unsigned long long amount[kHeld], last = ~0ull;
  if (q.k > 0) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i) amount[i] = (int)threadIdx.x + i * kThreads < count ? 1 : 0;
    last = select_held(h.o, amount, (unsigned long long)q.k, sh);
  }
  if (q.p < 1.0f) {
    unsigned long long mass = 0;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      amount[i] = h.o[i] <= last ? h.units[i] : 0;
      mass += amount[i];
    }
    mass = block_sum(mass, sh);
    const unsigned long long end = select_held(h.o, amount, mass_target(q.p, mass), sh);
    last = end < last ? end : last;
  }
  unsigned long long total = 0, index[kHeld];
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    amount[i] = h.o[i] <= last && (h.w[i] >= weight.least || h.o[i] == first) ? h.units[i] : 0;
    total += amount[i];
    index[i] = h.o[i] & ((1ull << a.index_bits) - 1);
  }
  total = block_sum(total, sh);
  const unsigned long long token = select_held(index, amount, draw_target(q.u, total), sh);
#pragma unroll
  for (int i = 0; i < kHeld; ++i)
    if (amount[i] && index[i] == token) write_token(a, r, (uint32_t)token, logit_of((uint32_t)(h.o[i] >> a.index_bits)), weight, q.t, total);
}

// The first class, in the order of the indexes, at which the amounts of the granules [c0, c1) reach `target`; amount(x, j) is a
// class's, hit(x, j) gets the class.  Every wave leaves the sums of eight of its steps of 64 granules, then all look among the 64
// sums, and the wave that has the class goes through that step again; a single step is looked at by all.  (All looking after
// every step: 512 rows of 128000 floats 131 us instead of 122; the sums for a single step too: 4096 rows of 5000 144, not 134.)
template <class T, class Amount, class Hit>
__device__ inline void find_class(const Chunks<T, 8> &row, int c0, int c1, unsigned long long target, Shared &sh, Amount amount, Hit hit) {
  constexpr int K = 8 / sizeof(T), kWaves = kThreads / 64, kSteps = 64 / kWaves;
  const T none = (T)-INFINITY;
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
  auto load = [&](int c) {
    vec_t<T, K> x = none;
    if (c < c1) x = row.load(c, none);
    return x;
  };
  auto scan = [&](unsigned long long v) {
    for (int off = 1; off < 64; off <<= 1) {
      const unsigned long long y = __shfl_up(v, off, 64);
      if (lane >= off) v += y;
    }
    return v;
  };
  unsigned long long u[K];
  auto amounts = [&](const vec_t<T, K> &x, int c) {
    unsigned long long sum = 0;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      u[k] = amount((float)x[k], row.column(c, k));
      sum += u[k];
    }
    return sum;
  };
  auto hit_among = [&](const vec_t<T, K> &x, int c, unsigned long long before) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (before < target && target <= before + u[k]) hit((float)x[k], row.column(c, k));
      before += u[k];
    }
  };
  if (c1 - c0 <= kThreads) {
    const int c = c0 + (int)threadIdx.x;
    const vec_t<T, K> x = load(c);
    const unsigned long long mine = amounts(x, c);
    __syncthreads();
    find_value(sh, mine, target);
    if (sh.found == threadIdx.x) hit_among(x, c, sh.before);
    return;
  }
  for (int b = c0; b < c1; b += kSteps * kThreads) {
    __syncthreads();
    vec_t<T, K> x[kSteps];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) x[i] = load(b + i * kThreads + (int)threadIdx.x);
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      const int c = b + i * kThreads + (int)threadIdx.x;
      unsigned long long mine = 0;
      if (b + i * kThreads < c1) {
#pragma unroll
        for (int k = 0; k < K; ++k) mine += amount((float)x[i][k], row.column(c, k));
        for (int off = 1; off < 64; off <<= 1) mine += __shfl_xor(mine, off, 64);
      }
      if (lane == 0) sh.hist[i * kWaves + wave] = mine;
    }
    __syncthreads();
    const unsigned long long sum = sh.hist[lane], up = scan(sum), all = __shfl(up, 63, 64);
    if (all < target) {  // uniform
      target -= all;
      continue;
    }
    const int at = __ffsll((unsigned long long)__ballot(up >= target)) - 1;
    if (wave != at % kWaves) return;
    const unsigned long long before = __shfl(up - sum, at, 64);
    const int c = b + at / kWaves * kThreads + (int)threadIdx.x;
    vec_t<T, K> y = x[0];
#pragma unroll
    for (int i = 1; i < kSteps; ++i) y = i == at / kWaves ? x[i] : y;
    const unsigned long long mine = amounts(y, c);
    hit_among(y, c, before + scan(mine) - mine);
    return;
  }
}

// granules of a part of a row
struct Part {
  int first, last;
  __device__ Part(int count, int part) {
    const int span = (count + kParts - 1) / kParts;
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
  const Chunks<T, 8> row(static_cast<const T *>(a.logits) + r * a.stride, (int)a.cols);
  const Part part(row.count, (int)blockIdx.x / a.split);
  const int step = 256 * a.split, start = part.first + (int)blockIdx.x % a.split * 256 + (int)threadIdx.x;
  const T none = (T)-INFINITY;
  unsigned long long *to = a.sums + (blockIdx.y * kParts + blockIdx.x / a.split) * (uint64_t)kSums;
  auto put_sum = [&](int i, unsigned long long v) {
    if (a.split == 1) to[i] = v;
    else if (v) atomicAdd(to + i, v);  // integers: in any order
  };
  unsigned long long rest = 0, above = 0;  // below the buckets; passing min-p
  auto each = [&](auto f) {
    for (int c = start; c < part.last; c += step) {
      const vec_t<T, K> x = row.load(c, none);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const double y = weight.exponent((float)x[k]), w = weight.scaled(y);
        f(y, w, weight.units(w));
      }
    }
  };
  if (q.p < 1.0f) {
    const Buckets buckets(q, a.cols);
    for (int i = threadIdx.x; i < kBuckets; i += 256) hist[i] = 0;
    __syncthreads();
    auto put = [&](double y, unsigned long long u) {
      const unsigned b = buckets.of(y);
      if (b < (unsigned)kBuckets) atomicAdd(&hist[b], u);
      else rest += u;
    };
    if (q.m > 0.0f) {
      each([&](double y, double w, unsigned long long u) {
        put(y, u);
        above += w >= weight.least ? u : 0;
      });
    } else {
      each([&](double y, double, unsigned long long u) { put(y, u); });
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kBuckets; i += 256) put_sum(i, hist[i]);
    rest = block_sum<256>(rest, sh);
  } else {
    each([&](double, double w, unsigned long long u) { above += w >= weight.least ? u : 0; });
  }
  above = block_sum<256>(above, sh);
  if (threadIdx.x == 0) {
    put_sum(kBuckets, rest);
    put_sum(kBuckets + 1, above);
  }
}

// A row with its parts' sums; false where its border's bucket holds too many classes.
template <class T>
__device__ inline bool draw_sums(const SampleArgs &a, uint64_t r, const unsigned long long *sums, const Params &q, const Weights &weight, RestShared &s) {
  const Chunks<T, 8> row(static_cast<const T *>(a.logits) + r * a.stride, (int)a.cols);
  bool nucleus = q.p < 1.0f;
  const Buckets buckets(q, a.cols);
  unsigned border = 0;
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
    unsigned long long total = mine;
    if (threadIdx.x < kParts) total += sums[threadIdx.x * kSums + kBuckets];
    total = block_sum(total, s.sh);
    const unsigned long long target = mass_target(q.p, total);
    // where the target is beyond all that passes min-p, top-p keeps all of that and more
    nucleus = !(q.m > 0.0f && target > above);
    if (nucleus) {
      if (threadIdx.x == 0) s.count = 0;
      __syncthreads();
      find_value(s.sh, mine, target);
      if (s.sh.found == ~0ull) return false;
      border = (unsigned)s.sh.found;
      const unsigned long long within = target - s.sh.before;
      // the classes of the bucket that the target falls into
      const Chunks<T> wide(static_cast<const T *>(a.logits) + r * a.stride, (int)a.cols);
      constexpr int K = 16 / sizeof(T), kAhead = 8;
      // The logits of the bucket lie between two floats; these are a little farther apart.  What lies outside is left out by
      // them, the rest is asked for its bucket (asked all: 16 instructions a class, 62 us instead of 58 at 512 x 128000 bf16,
      // where the rows come at 12 bytes a clock per CU).  Classes whose exponent is held at -64 weigh nothing and may be left out.
      const double high = weight.top + (border - 0.5) / buckets.per / weight.per, low = weight.top + (border + 0.5) / buckets.per / weight.per;
      const float from = (float)(low - fabs(low) * 0x1p-22 - fabs((double)weight.top) * 0x1p-48 - 0x1p-140);
      const float to = (float)(high + fabs(high) * 0x1p-22 + fabs((double)weight.top) * 0x1p-48 + 0x1p-140);
      for (int c0 = threadIdx.x; c0 < wide.count; c0 += kAhead * kThreads) {
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
            if (!((float)x[u][k] >= from && (float)x[u][k] <= to) || buckets.of(weight.exponent((float)x[u][k])) != border) continue;
            const int j = wide.column(c0 + u * kThreads, k);
            if (j < 0 || j >= wide.cols) continue;
            const unsigned at = atomicAdd(&s.count, 1u);
            if (at < (unsigned)kList) s.list[at] = (unsigned long long)key_of((float)x[u][k]) << a.index_bits | (unsigned long long)j;
          }
        }
      }
      __syncthreads();
      if (s.count > (unsigned)kList) return false;
      const Held h(s.list, (int)s.count, weight, a.index_bits);
      last = select_held(h.o, h.units, within, s.sh);
      // what is kept of every part
      if (threadIdx.x < kParts) s.hist[threadIdx.x][border] = 0;
      __syncthreads();
      const int span = (row.count + kParts - 1) / kParts;
#pragma unroll
      for (int i = 0; i < kHeld; ++i) {
        if ((int)threadIdx.x + i * kThreads >= (int)s.count || h.o[i] > last) continue;
        const int j = (int)(h.o[i] & ((1ull << a.index_bits) - 1));
        atomicAdd(&s.hist[(j + row.lead) / (8 / (int)sizeof(T)) / span][border], h.units[i]);
      }
      __syncthreads();
      static_assert(kThreads / 64 == kParts, "a wave each");
      unsigned long long kept = 0;
      for (unsigned b = threadIdx.x & 63; b <= border; b += 64) kept += s.hist[threadIdx.x / 64][b];
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
             [&](float x, int j) -> unsigned long long {
               const double y = weight.exponent(x), w = weight.scaled(y);
               bool kept = w >= weight.least;
               if (nucleus) {
                 const unsigned b = buckets.of(y);
                 kept = b < border || (b == border && ((unsigned long long)key_of(x) << a.index_bits | (unsigned long long)j) <= last);
               }
               return kept ? weight.units(w) : 0;
             },
             [&](float x, int j) { write_token(a, r, (uint32_t)j, x, weight, q.t, total); });
  return true;
}

template <class T>
__global__ void __launch_bounds__(kThreads) k_sample_list(SampleArgs a) {
  constexpr int K = 16 / sizeof(T);
  __shared__ ListShared s;
  const T none = (T)-INFINITY;
  for (uint64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    __syncthreads();
    const Chunks<T> row(static_cast<const T *>(a.logits) + r * a.stride, (int)a.cols);
    const Params q = params_of(a, r);
    const int small = (row.count + (1 << a.group_log2) - 1) >> a.group_log2, size = (small + kMaxGroups - 1) / kMaxGroups;
    const int groups = (small + size - 1) / size;  // of `size` times 2^group_log2 granules
    // the groups' largest logits, and the row's
    float top = -INFINITY;
    for (int g = threadIdx.x; g < groups; g += kThreads) {
      float m = -INFINITY;
      for (int i = g * size; i < (g + 1) * size && i < small; ++i) m = fmaxf(m, a.tops[r * a.groups + i]);
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
    const unsigned per = (unsigned)(size << a.group_log2), granules = s.nhits * per;  // at most the row's 2^31 / K and kMaxGroups' rounding
    for (unsigned i = threadIdx.x; i < granules; i += 4 * kThreads) {
      vec_t<T, K> x[4];
      int c[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const unsigned at = i + u * kThreads;
        c[u] = at < granules ? (int)(s.hits[at / per] * per + at % per) : row.count;
        if (c[u] < row.count) x[u] = row.load(c[u], none);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (c[u] >= row.count) continue;
#pragma unroll
        for (int k = 0; k < K; ++k) {
          const float v = (float)x[u][k];
          const int j = row.column(c[u], k);
          if (v >= bound && j >= 0 && j < row.cols) {
            const unsigned at = atomicAdd(&s.count, 1u);
            const unsigned long long o = (unsigned long long)key_of(v) << a.index_bits | (unsigned long long)j;
            if (at < (unsigned)kList) s.list[at] = o;
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
    } else if (s.count <= (unsigned)kList) {
      draw_held(a, r, q, Weights(top, q.t, q.m, a.shift), first, s.list, (int)s.count, s.sh);
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
  const Chunks<T> row(static_cast<const T *>(a.logits) + r * a.stride, (int)a.cols);
  unsigned long long first = ~0ull;  // the lowest index of the largest logit
  for (int c = threadIdx.x; c < row.count && first == ~0ull; c += kThreads) {
    const vec_t<T, 16 / sizeof(T)> x = row.load(c, (T)-INFINITY);
#pragma unroll
    for (int k = 16 / sizeof(T) - 1; k >= 0; --k)
      if ((float)x[k] == top) first = (unsigned long long)row.column(c, k);
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

// ---- rows of up to 1024 classes ------------------------------------------------------------------------
//
// In one launch: LANES lanes hold a row, EACH consecutive classes a lane, and sort its keys in their registers (bitonic: the
// partner of position p is p ^ j, in the same lane for j < EACH).  The sums over the sorted classes say which is the last that
// is kept, those over the classes where they are give the token.  No row is left to anyone else.  With more than kLaneCols
// classes the sort is long for one wave (33 us where the kernels above take 23), so that fewer than kSmallRows rows that need
// it go there: 64 rows of 1000 with top-k 33 and 24 us, 512 35 and 32, with top-p 37 and 41, 8192 137 and 417; without either
// filter there is no sort and this is faster, 64 rows 8 and 13.  That holds for shorter rows, whose few groups leave a larger k to
// draw_row: 64 rows in 16 bits by the kernels above, and 512 by the sort, with k = 90 of 520 classes 23 and 34 us, of 640 23 and
// 35, of 800 27 and 35; with top-p beside it 30, 30, 34 and 36, 36, 36.
constexpr uint64_t kSmallCols = 1024, kLaneCols = 512, kSmallRows = 512;

template <class T, int LANES, int EACH>
__global__ void __launch_bounds__(256) k_sample_small(SampleArgs a) {
  const int lane = (int)threadIdx.x & (LANES - 1);
  auto sum = [&](unsigned long long v) {
#pragma unroll
    for (int off = 1; off < LANES; off <<= 1) v += __shfl_xor(v, off, 64);
    return v;
  };
  auto sum_before = [&](unsigned long long v) {  // of the lanes before this one
    unsigned long long up = v;
#pragma unroll
    for (int off = 1; off < LANES; off <<= 1) {
      const unsigned long long y = __shfl_up(up, off, LANES);
      if (lane >= off) up += y;
    }
    return up - v;
  };
  for (uint64_t r = (uint64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES; r < a.rows; r += (uint64_t)gridDim.x * (256 / LANES)) {
    const T *row = static_cast<const T *>(a.logits) + r * a.stride;
    const Params q = params_of(a, r);
    float x[EACH];
    unsigned long long mine[EACH], o[EACH];
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      const int j = lane * EACH + e;
      x[e] = j < (int)a.cols ? (float)row[j] : -INFINITY;
      mine[e] = o[e] = j < (int)a.cols ? (unsigned long long)key_of(x[e]) << a.index_bits | (unsigned)j : ~0ull;
    }
    // sorted: position lane * EACH + e (without top-k and top-p the first class is all that is wanted of it)
    const bool sorts = (q.k > 0 || q.p < 1.0f) && !is_greedy(q);
    for (int k = 2; sorts && k <= LANES * EACH; k <<= 1) {
      for (int j = k >> 1; j >= EACH; j >>= 1) {
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
          const unsigned long long other = __shfl_xor(o[e], j / EACH, 64);
          const int p = lane * EACH + e;
          const bool low = ((p & j) == 0) == ((p & k) == 0);
          o[e] = (other < o[e]) == low ? other : o[e];
        }
      }
#pragma unroll
      for (int j = EACH >> 1; j >= 1; j >>= 1) {
        if (j >= k) continue;
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
          if (e & j) continue;
          const bool up = ((lane * EACH + e) & k) == 0;
          const unsigned long long lo = o[e] < o[e ^ j] ? o[e] : o[e ^ j], hi = o[e] < o[e ^ j] ? o[e ^ j] : o[e];
          o[e] = up ? lo : hi;
          o[e ^ j] = up ? hi : lo;
        }
      }
    }
    unsigned long long first = o[0];
    if (!sorts) {
#pragma unroll
      for (int e = 1; e < EACH; ++e) first = o[e] < first ? o[e] : first;
#pragma unroll
      for (int off = 1; off < LANES; off <<= 1) {
        const unsigned long long y = __shfl_xor(first, off, 64);
        first = y < first ? y : first;
      }
    }
    first = __shfl(first, 0, LANES);
    const float top = logit_of((uint32_t)(first >> a.index_bits));
    const uint32_t mask = (1u << a.index_bits) - 1;
    if (top == -INFINITY || is_greedy(q)) {
      if (lane == 0) {
        a.token[r] = top == -INFINITY ? -1 : (int32_t)(first & mask);
        if (a.logprob) a.logprob[r] = top == -INFINITY ? -INFINITY : 0.0f;
      }
      continue;
    }
    const Weights weight(top, q.t, q.m, a.shift);
    // (a top of +inf has all the weight)
    auto scaled = [&](float v) { return top == INFINITY ? (v == top ? ldexp(1.0, a.shift) : 0.0) : weight.scaled(v); };
    unsigned long long last = ~0ull;
    if (q.k > 0 || q.p < 1.0f) {
      unsigned long long u[EACH], all = 0;
      int kept = 0;
#pragma unroll
      for (int e = 0; e < EACH; ++e) {
        const int at = lane * EACH + e;
        const bool in = at < (int)a.cols && (q.k <= 0 || at < q.k);
        u[e] = in && q.p < 1.0f ? weight.units(scaled(logit_of((uint32_t)(o[e] >> a.index_bits)))) : 0;
        all += u[e];
        kept += in;
      }
      if (q.p < 1.0f) {
        const unsigned long long target = mass_target(q.p, sum(all));
        unsigned long long before = sum_before(all);
        int count = 0;
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
          const int at = lane * EACH + e;
          count += at < (int)a.cols && (q.k <= 0 || at < q.k) && before < target;
          before += u[e];
        }
        kept = count;
      }
      // the kept ones are the first in order: the last of them is the largest key
      last = 0;
#pragma unroll
      for (int e = 0; e < EACH; ++e)
        if (e < kept) last = o[e];
#pragma unroll
      for (int off = 1; off < LANES; off <<= 1) {
        const unsigned long long y = __shfl_xor(last, off, 64);
        last = y > last ? y : last;
      }
    }
    unsigned long long amount[EACH], all = 0;
    int lowest = 0x7FFFFFFF;  // class of any weight, however small: the token for u <= 0
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      const double w = scaled(x[e]);
      const bool in = mine[e] <= last && mine[e] != ~0ull && (w >= weight.least || mine[e] == first);
      amount[e] = in ? weight.units(w) : 0;
      all += amount[e];
      const bool any = x[e] == top || ((double)x[e] - (double)top) * weight.per > -1075.0;
      if (in && any && lane * EACH + e < lowest) lowest = lane * EACH + e;
    }
    const unsigned long long total = sum(all);
    int token = -1;
    float value = 0.0f;
    if (q.u > 0.0f) {
      const unsigned long long target = draw_target(q.u, total);
      unsigned long long before = sum_before(all);
#pragma unroll
      for (int e = 0; e < EACH; ++e) {
        if (before < target && target <= before + amount[e]) {
          token = lane * EACH + e;
          value = x[e];
        }
        before += amount[e];
      }
    } else {
      int at = lowest;
#pragma unroll
      for (int off = 1; off < LANES; off <<= 1) at = min(at, __shfl_xor(at, off, 64));
#pragma unroll
      for (int e = 0; e < EACH; ++e) {
        if (lane * EACH + e == at) {
          token = at;
          value = x[e];
        }
      }
    }
    if (token >= 0) write_token(a, r, (uint32_t)token, value, weight, q.t, total);
  }
}

// Granules per group: as many groups as a wave can hold in registers, 256 to 512, so that a large k has its groups too; rows of
// more than 2^14 granules have more groups, of 32 granules.  (With groups of 32 whatever the row, us for k = 50 and 200: 64 rows
// of 5000 floats 34 and 36, 64 of 32000 halves 21 and 137, 2048 of 32000 halves 149 and 912; so: 18 and 27, 19 and 31, 129 and
// 225.)
static int tops_group_log2(uint64_t granules) {
  int log2 = 0;
  while (log2 < 5 && (granules >> log2) >= 512) ++log2;
  return log2;
}

// groups of a row, whatever its alignment
static uint64_t tops_groups(uint64_t cols, uint64_t per) {
  const uint64_t granules = (cols + per - 1) / per + 1;
  const int log2 = tops_group_log2(granules);
  return (granules + (1ull << log2) - 1) >> log2;
}

static uint64_t tops_bytes(uint64_t rows, uint64_t groups) { return round_up(rows * groups * sizeof(float), 256); }

template <class T>
static int sample(admm_ctx *ctx, SampleArgs a, void *workspace) {
  if (a.cols <= kLaneCols || (a.cols <= kSmallCols && (a.rows >= kSmallRows || !(a.top_k || a.top_p)))) {
#define ADMM_SMALL(LANES, EACH) hipLaunchKernelGGL((k_sample_small<T, LANES, EACH>), dim3(blocks_for(a.rows, 256 / LANES)), dim3(256), 0, ctx->stream, a)
    if (a.cols <= 16) ADMM_SMALL(16, 1);
    else if (a.cols <= 64) ADMM_SMALL(64, 1);
    else if (a.cols <= 128) ADMM_SMALL(64, 2);
    else if (a.cols <= 256) ADMM_SMALL(64, 4);
    else if (a.cols <= 512) ADMM_SMALL(64, 8);
    else ADMM_SMALL(64, 16);
#undef ADMM_SMALL
    ADMM_HIP_CHECK(hipGetLastError());
    return ADMM_OK;
  }
  a.groups = (int64_t)tops_groups(a.cols, 16 / sizeof(T));
  a.group_log2 = tops_group_log2((a.cols + 16 / sizeof(T) - 1) / (16 / sizeof(T)) + 1);
  a.tops = static_cast<float *>(workspace);
  a.sums = reinterpret_cast<unsigned long long *>(static_cast<char *>(workspace) + tops_bytes(a.rows, a.groups));
  const dim3 block(kThreads);
  a.split = a.rows * kParts >= 512 ? 1 : (int)(512 / (a.rows * kParts) < 8 ? 512 / (a.rows * kParts) : 8);
  const unsigned per_row = (unsigned)(((a.groups << a.group_log2) + kTopsPer - 1) / kTopsPer);
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
    hipLaunchKernelGGL(k_sample_sums<T>, dim3(kParts * a.split, (unsigned)(end - r)), dim3(256), 0, ctx->stream, a, r);
    hipLaunchKernelGGL(k_sample_rest<T>, dim3((unsigned)(end - r)), block, 0, ctx->stream, a, r, end);
  }
  ADMM_HIP_CHECK(hipGetLastError());
  return ADMM_OK;
}

}  // namespace admm_impl

using namespace admm_impl;

extern "C" int admm_sample_workspace(uint64_t rows, uint64_t cols, uint64_t *bytes) {
  ADMM_REQUIRE(bytes, "admm_sample_workspace: bytes is NULL");
  ADMM_REQUIRE(rows < (1ull << 40) && cols <= kMaxClasses && (unsigned __int128)rows * cols < ((unsigned __int128)1 << 46),
               "admm_sample_workspace: %llu x %llu logits", (unsigned long long)rows, (unsigned long long)cols);
  *bytes = 0;
  if (cols <= kLaneCols || (cols <= kSmallCols && rows >= kSmallRows)) return ADMM_OK;
  // enough for logits of any type: granules of four floats or of eight halves
  const uint64_t wide = tops_groups(cols, 4), narrow = tops_groups(cols, 8);
  *bytes = tops_bytes(rows, wide > narrow ? wide : narrow) + (rows < kBatch ? rows : kBatch) * (kParts * kSums * sizeof(unsigned long long));
  return ADMM_OK;
}

extern "C" int admm_sample(admm_ctx *ctx, const admm_mat *logits, const admm_sample_params *params, const float *uniform, int32_t *token,
                           float *logprob, void *workspace, uint64_t workspace_bytes) {
  ADMM_REQUIRE(ctx, "admm_sample: ctx is NULL");
  ADMM_TRY(check_mat(logits, "admm_sample", "logits"));
  if (logits->rows == 0) return ADMM_OK;
  ADMM_REQUIRE(logits->cols > 0 && logits->cols <= kMaxClasses, "admm_sample: %llu classes", (unsigned long long)logits->cols);
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
