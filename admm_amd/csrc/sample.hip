// Draws a class per row from softmax(logits / temperature) after top-k, top-p and min-p, with given uniform numbers.
//
// The weight of a class is w = 2^((x - max) L / T), L = log2(e), computed in double and held as the integer
// rint(w 2^S): sums of integers do not depend on their order, so a row's token does not depend on how it is summed.  S is
// such that a row of ones still fits 63 bits.
//
// Every filter keeps a prefix of the classes in the order (logit descending, index ascending), and the draw is the first
// class in index order at which the cumulative weight passes a bound.  Both are one question -- the first class, by some
// key, at which the cumulative amount (a count, or the weight) reaches a target -- and are answered digit by digit: amounts
// per value of the digit in LDS, the value at which the target falls, and on with the classes of that value.
#include "rows_common.h"

namespace admm_impl {

constexpr int kThreads = 1024;
constexpr int kDigit = 8;

struct SampleArgs {
  const void *logits;
  uint64_t stride, rows, cols;
  const float *temperature, *top_p, *min_p, *uniform;
  const int32_t *top_k;
  int32_t *token;
  float *logprob;
  int index_bits, shift;  // 2^index_bits >= cols; S
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

// 2^y for y <= 0: 2^rint(y) times a polynomial of the rest (|f ln 2| <= 0.35: the series' term of degree 12 is 1e-16)
__device__ inline double exp2_double(double y) {
  y = y > -1100.0 ? y : -1100.0;
  const double n = rint(y), f = (y - n) * 0.69314718055994530942;
  double p = 1.0 / 479001600.0;
  p = fma(p, f, 1.0 / 39916800.0);
  p = fma(p, f, 1.0 / 3628800.0);
  p = fma(p, f, 1.0 / 362880.0);
  p = fma(p, f, 1.0 / 40320.0);
  p = fma(p, f, 1.0 / 5040.0);
  p = fma(p, f, 1.0 / 720.0);
  p = fma(p, f, 1.0 / 120.0);
  p = fma(p, f, 1.0 / 24.0);
  p = fma(p, f, 1.0 / 6.0);
  p = fma(p, f, 0.5);
  p = fma(p, f, 1.0);
  p = fma(p, f, 1.0);
  return ldexp(p, (int)n);
}

struct Weights {
  float top;
  double per;  // L / T
  int shift;
  // the weight as a double; the class with the largest logit has 1 (also where that is +inf)
  __device__ double of(float x) const { return x == top ? 1.0 : x > -INFINITY ? exp2_double(((double)x - (double)top) * per) : 0.0; }
  __device__ unsigned long long units(double w) const { return (unsigned long long)rint(ldexp(w, shift)); }
};

// the classes of a row, each of them to one thread
template <class T>
struct RowSource {
  Chunks<T> row;
  template <class F>
  __device__ void each(F f) const {
    constexpr int K = 16 / sizeof(T);
    for (int64_t c = threadIdx.x; c < row.count; c += kThreads) {
      const vec_t<T, K> x = row.load(c, (T)-INFINITY);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int64_t j = c * K + k - row.lead;
        if (j >= 0 && j < row.cols) f((float)x[k], (uint32_t)j);
      }
    }
  }
};

struct Shared {
  unsigned long long hist[1 << kDigit];
  unsigned long long sums[kThreads / 64];
  unsigned long long found, before;
};

__device__ inline unsigned long long block_sum(unsigned long long v, Shared &sh) {
  for (int off = 1; off < 64; off <<= 1) v += __shfl_xor(v, off, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh.sums[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int i = 0; i < kThreads / 64; ++i) v += sh.sums[i];
  return v;
}

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
  for (int i = 1; i < kThreads / 64; ++i) v = sh.sums[i] < v ? sh.sums[i] : v;
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

// the token of one row from the classes that `source` gives out
template <class Source>
__device__ inline void draw_row(const SampleArgs &a, uint64_t r, const Source &source, Shared &sh) {
  const int bits = 32 + a.index_bits;
  auto order = [&](float x, uint32_t j) { return (unsigned long long)key_of(x) << a.index_bits | j; };
  unsigned long long first = ~0ull;
  source.each([&](float x, uint32_t j) {
    const unsigned long long k = order(x, j);
    first = k < first ? k : first;
  });
  first = block_min(first, sh);
  const float top = logit_of((uint32_t)(first >> a.index_bits));
  const float t = a.temperature ? a.temperature[r] : 1.0f;
  const bool none = top == -INFINITY;
  if (none || !(t > 0.0f)) {
    if (threadIdx.x == 0) {
      a.token[r] = none ? -1 : (int32_t)(first & ((1ull << a.index_bits) - 1));
      if (a.logprob) a.logprob[r] = none ? -INFINITY : 0.0f;
    }
    return;
  }
  const Weights weight{top, 1.44269504088896340736 / (double)t, a.shift};
  const float m = a.min_p ? a.min_p[r] : 0.0f;
  const int32_t k = a.top_k ? a.top_k[r] : 0;
  const float p = a.top_p ? a.top_p[r] : 1.0f;
  unsigned long long last = ~0ull;  // the last class that is kept
  if (k > 0 && (uint64_t)k < a.cols)
    last = select_key(bits, (unsigned long long)k, sh, [&](auto f) { source.each([&](float x, uint32_t j) { f(order(x, j), 1ull); }); });
  if (p < 1.0f) {
    unsigned long long mass = 0;
    source.each([&](float x, uint32_t j) { mass += order(x, j) <= last ? weight.units(weight.of(x)) : 0; });
    mass = block_sum(mass, sh);
    // kept while the mass before is below p times it: up to the first class at which the sum reaches that
    const double bound = p > 0.0f ? ceil((double)p * (double)mass) : 0.0;
    const unsigned long long target = bound < 1.0 ? 1ull : (unsigned long long)bound;
    const unsigned long long end = select_key(bits, target, sh, [&](auto f) {
      source.each([&](float x, uint32_t j) {
        const unsigned long long o = order(x, j);
        f(o, o <= last ? weight.units(weight.of(x)) : 0ull);
      });
    });
    last = end < last ? end : last;
  }
  auto kept = [&](float x, uint32_t j) -> unsigned long long {
    const unsigned long long o = order(x, j);
    if (o > last) return 0;
    const double w = weight.of(x);
    if (m > 0.0f && !(w >= (double)m) && o != first) return 0;
    return weight.units(w);
  };
  unsigned long long total = 0;
  source.each([&](float x, uint32_t j) { total += kept(x, j); });
  total = block_sum(total, sh);
  const float u = a.uniform[r];
  unsigned long long token;
  if (u > 0.0f) {
    const double at = floor((double)u * (double)total);
    unsigned long long target = at < (double)total ? (unsigned long long)at + 1 : total;
    target = target < total ? target : total;
    token = select_key(a.index_bits, target, sh, [&](auto f) { source.each([&](float x, uint32_t j) { f(j, kept(x, j)); }); });
  } else {  // the first class of any weight, however small
    token = ~0ull;
    source.each([&](float x, uint32_t j) {
      const unsigned long long o = order(x, j);
      const double w = weight.of(x);
      if (o <= last && w > 0.0 && (!(m > 0.0f) || w >= (double)m || o == first) && j < token) token = j;
    });
    token = block_min(token, sh);
  }
  source.each([&](float x, uint32_t j) {
    if (j != token) return;
    a.token[r] = (int32_t)j;
    if (!a.logprob) return;
    const double y = x == top ? 0.0 : ((double)x - (double)top) / (double)t;
    a.logprob[r] = (float)(y - log(ldexp((double)total, -a.shift)));
  });
}

template <class T>
__global__ void __launch_bounds__(kThreads) k_sample_rows(SampleArgs a) {
  __shared__ Shared sh;
  for (uint64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const RowSource<T> source{Chunks<T>(static_cast<const T *>(a.logits) + r * a.stride, (int64_t)a.cols)};
    draw_row(a, r, source, sh);
    __syncthreads();
  }
}

}  // namespace admm_impl

using namespace admm_impl;

extern "C" int admm_sample_workspace(uint64_t rows, uint64_t cols, uint64_t *bytes) {
  ADMM_REQUIRE(bytes, "admm_sample_workspace: bytes is NULL");
  ADMM_REQUIRE(rows < (1ull << 40) && cols < (1ull << 31), "admm_sample_workspace: %llu x %llu logits", (unsigned long long)rows,
               (unsigned long long)cols);
  *bytes = 0;
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
  a.shift = 62 - a.index_bits;
  const dim3 grid(blocks_for(a.rows, 1));
  if (logits->type == ADMM_F32) hipLaunchKernelGGL(k_sample_rows<float>, grid, dim3(kThreads), 0, ctx->stream, a);
  else if (logits->type == ADMM_BF16) hipLaunchKernelGGL(k_sample_rows<bf16_t>, grid, dim3(kThreads), 0, ctx->stream, a);
  else hipLaunchKernelGGL(k_sample_rows<f16_t>, grid, dim3(kThreads), 0, ctx->stream, a);
  ADMM_HIP_CHECK(hipGetLastError());
  return ADMM_OK;
}
