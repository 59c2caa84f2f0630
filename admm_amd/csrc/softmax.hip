// Softmax loss with its gradient: the many-class form of the logistic loss and its residuals.
//
// With L = log2(e) and m the row's largest logit, the exponentials are 2^(x L - m L) (one fused multiply-add and one
// hardware exp2 each), o the sum of all but the label's, s = o + 2^(x_t L - m L), and
//   loss = ln 2 (log2 s - (x_t L - m L)),  grad = 2^(x L - m L) w / s, at the label -w o / s.
// The label is left out of o, not taken off s: a row that is nearly sure of its label has a loss and a gradient far below 1, of
// which p - 1 and log s would keep 2^-24 of 1 only (its loss is log1p of o over the label's power).
// Both read x L - m L through the same rounded m L, so its rounding cancels (log2 s in the exponent instead of the division
// would add half a step of m L to it, 2e-6 of a probability where m is 30).  Where m L would overflow (a mask of the type's
// lowest value over a whole row), 1 takes the place of L: logits of that size are equal or more than 2^100 apart.
#include "rows_common.h"

namespace admm_impl {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct SoftmaxArgs {
  const void *logits;
  void *grad;  // or NULL; may be the logits
  uint64_t stride, gstride, rows, cols;
  const void *labels;
  int label_type;
  const float *weight;  // or NULL
  float grad_scale;
  float *loss, *lse;  // lse or NULL
  int lanes_log2;
  int apart;  // the gradient's rows are aligned otherwise than the logits': written element by element
};

// the row's label, -1 where it is not trained on; w: its weight
__device__ inline int64_t label_of(const SoftmaxArgs &a, uint64_t r, float &w) {
  w = a.weight ? a.weight[r] : 1.0f;
  int64_t t;
  if (a.label_type == ADMM_I64) {
    t = static_cast<const int64_t *>(a.labels)[r];
  } else if (a.label_type == ADMM_I32) {
    t = static_cast<const int32_t *>(a.labels)[r];
  } else {
    const float f = static_cast<const float *>(a.labels)[r];
    t = f > -1.0f && f < 9.0e18f ? (int64_t)f : -1;
  }
  return t >= 0 && (uint64_t)t < a.cols && w != 0.0f ? t : -1;
}

__device__ inline float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// largest element of a chunk, NaN aside
template <class T>
__device__ inline float chunk_max(const vec_t<T, 16 / sizeof(T)> &x, float m) {
#pragma unroll
  for (int k = 0; k < (int)(16 / sizeof(T)); ++k) m = fmaxf(m, (float)x[k]);
  return m;
}

// What is taken off a row's exponents: x l - m2, rounded once.  m2 is m L rounded, by up to 2^-24 of itself; that is in every
// power of the row and cancels, so long as it stays far from the ends of the exponents: by up to 64 at |m| = 2^30.  Larger logits
// that differ are at least 64 apart, so their factor may as well be 1, with which m2 is exact (and does not overflow).
struct Shift {
  float l, m2;
  explicit __device__ Shift(float m) {
    l = fabsf(m) < 0x1p30f || m == -INFINITY ? kLog2e : 1.0f;
    m2 = m == -INFINITY ? 0.0f : m * l;  // without a class every power is 2^(-inf - 0) = 0
  }
};

// What a sum relative to `from` is multiplied by to be relative to `to`, a larger logit's.  Where their factors differ, so do the
// logits, by 64 or more (and m2 is not in their order).
__device__ inline float moved(Shift from, Shift to) { return from.l == to.l ? exp2_fast(from.m2 - to.m2) : 0.0f; }

template <class T>
__device__ inline float chunk_sum(const vec_t<T, 16 / sizeof(T)> &x, Shift b) {
  float s = 0.0f;
#pragma unroll
  for (int k = 0; k < (int)(16 / sizeof(T)); ++k) s += exp2_fast(__fmaf_rn((float)x[k], b.l, -b.m2));
  return s;
}

// Keeps a chunk in its 16 bytes between two uses: without it the compiler holds the unpacked floats instead, twice the
// registers, and spills.
template <class V>
__device__ inline void stay_packed(V &x) {
  u32x4 u = __builtin_bit_cast(u32x4, x);
  asm volatile("" : "+v"(u));
  x = __builtin_bit_cast(V, u);
}

// Takes the label out of a chunk before its sum; `at`: which of its elements it is, or anything else.  On the packed words, three
// instructions each: element by element it is three times as many, and registers with them.
template <class T>
__device__ inline void take_out(vec_t<T, 16 / sizeof(T)> &x, int at) {
  u32x4 u = __builtin_bit_cast(u32x4, x);
  if (sizeof(T) == 4) {
#pragma unroll
    for (int k = 0; k < 4; ++k) u[k] = at == k ? 0xFF800000u : u[k];
  } else {
    constexpr uint32_t none = std::is_same<T, bf16_t>::value ? 0xFF80u : 0xFC00u;  // -inf
    const uint32_t mask = at & 1 ? 0xFFFF0000u : 0xFFFFu, put = none << 16 | none;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t here = at >> 1 == k ? mask : 0u;
      u[k] = (u[k] & ~here) | (put & here);
    }
  }
  x = __builtin_bit_cast(vec_t<T, 16 / sizeof(T)>, u);
}

// the label's power; 0 where there is no label
__device__ inline float label_power(int64_t t, float xt, Shift b) { return t >= 0 ? exp2_fast(__fmaf_rn(xt, b.l, -b.m2)) : 0.0f; }

// the gradient of a chunk; `at`: which of its elements the label is, or anything else; gl: the label's, negated
template <class T>
__device__ inline vec_t<T, 16 / sizeof(T)> chunk_grad(const vec_t<T, 16 / sizeof(T)> &x, Shift b, float share, float gl = 0.0f, int at = -1) {
  constexpr int K = 16 / sizeof(T);
  float v[K];
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = share * exp2_fast(__fmaf_rn((float)x[k], b.l, -b.m2));
  if ((unsigned)at < (unsigned)K) {
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = at == k ? -gl : v[k];
  }
  vec_t<T, K> y;
#pragma unroll
  for (int k = 0; k < K; ++k) y[k] = (T)v[k];
  return y;
}

// log(1 + x) of 0 <= x < 1, right relative to itself: what 1 + x loses of x, log(1 + x) loses too
__device__ inline float log1p_fast(float x) {
  const float y = 1.0f + x, got = y - 1.0f;
  return got == 0.0f ? x : kLn2 * __log2f(y) * (x * __builtin_amdgcn_rcpf(got));
}

// loss and lse of a row with the label t, whose power is e; the others' sum is `others`
__device__ inline void finish_row(const SoftmaxArgs &a, uint64_t r, Shift b, float others, float e, int64_t t, float w, float xt) {
  const float s = others + e;
  const float log2s = __log2f(s);  // -inf where no class is left
  const float nats = b.l == 1.0f ? 1.0f : kLn2;
  if (a.lse) a.lse[r] = s == 0.0f ? -INFINITY : b.m2 * nats + log2s * kLn2;
  // (a label masked by the type's lowest value: x_t L would overflow)
  const float off = fabsf(xt) < 0x1p100f ? nats * __fmaf_rn(xt, b.l, -b.m2) : xt - nats * b.m2;
  a.loss[r] = t < 0 ? 0.0f : s == 0.0f ? INFINITY * w : others < e ? w * log1p_fast(others * __builtin_amdgcn_rcpf(e)) : w * (kLn2 * log2s - off);
}

// Rows of up to 64 CH chunks: 2^lanes_log2 lanes hold a row, CH chunks each, and reduce it among themselves.  With more than one
// chunk a lane the label's is left out of the sum whole, and its other elements are added by one lane each.
template <class T, int CH>
__global__ void __launch_bounds__(256) k_softmax_lanes(SoftmaxArgs a) {
  constexpr int K = 16 / sizeof(T);
  constexpr bool kAside = CH > 1;  // 64 lanes a row, more than a chunk has elements
  const unsigned lanes = 1u << a.lanes_log2, lane = threadIdx.x & (lanes - 1);
  const uint64_t per = 256u >> a.lanes_log2;
  const T none = (T)-INFINITY;
  for (uint64_t r = (uint64_t)blockIdx.x * per + (threadIdx.x >> a.lanes_log2); r < a.rows; r += (uint64_t)gridDim.x * per) {
    float w;
    const int64_t t = label_of(a, r, w);
    const T *const from = static_cast<const T *>(a.logits) + r * a.stride;
    const Chunks<T> row(from, (int)a.cols);
    T *to = a.grad ? static_cast<T *>(a.grad) + r * a.gstride : nullptr;
    vec_t<T, K> x[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c)
      if ((int)(c * lanes + lane) < row.count) x[c] = row.load(c * lanes + lane, none);
      else x[c] = none;
    const float xt = (float)from[t >= 0 ? t : 0];
    const int tc = t < 0 ? -1 : (int)t + row.lead;
    int label_chunk = t < 0 ? -1 : tc / K;
    asm volatile("" : "+v"(label_chunk));  // or the compiler traces it back to the logits' address and no longer sees that they are global memory
    const int aside = kAside && t >= 0 && lane < K ? row.column(label_chunk, (int)lane) : -1;
    const bool is_loose = (aside >= 0) & (aside < row.cols) & (aside != (int)t);
    const float at_loose = kAside ? (float)from[is_loose ? aside : 0] : 0.0f;
    float m = -INFINITY;
#pragma unroll
    for (int c = 0; c < CH; ++c) m = chunk_max<T>(x[c], m);
    for (unsigned off = 1; off < lanes; off <<= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
    const Shift b(m);
    float others = 0.0f;
    const float loose = is_loose ? at_loose : -INFINITY;
    if (kAside) others = exp2_fast(__fmaf_rn(loose, b.l, -b.m2));
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      if (!kAside) take_out<T>(x[c], tc - (c * (int)lanes + (int)lane) * K);
      stay_packed(x[c]);
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const float part = chunk_sum<T>(x[c], b);
      others += kAside && c * (int)lanes + (int)lane == label_chunk ? 0.0f : part;
    }
    for (unsigned off = 1; off < lanes; off <<= 1) others += __shfl_xor(others, off, 64);
    const float e = label_power(t, xt, b), s = others + e;
    if (lane == 0) finish_row(a, r, b, others, e, t, w, xt);
    if (!to) continue;
    const float share = (t < 0 ? 0.0f : w * a.grad_scale) / s, gl = share * others;
#pragma unroll
    for (int c = 0; c < CH; ++c) stay_packed(x[c]);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int at = c * (int)lanes + (int)lane;
      if (at >= row.count) continue;
      const vec_t<T, K> zero = (T)0.0f;
      row.store(to, a.apart, at, t < 0 || s == 0.0f ? zero : chunk_grad<T>(x[c], b, share, gl, kAside ? -1 : tc - at * K));
    }
    // over what this lane has just written there
    if (kAside & (t >= 0) & ((label_chunk & ((int)lanes - 1)) == (int)lane)) to[t] = s == 0.0f ? (T)0.0f : (T)-gl;
  }
}

template <int NT>
__device__ inline float block_max(float v, float *sh) {
  for (int off = 1; off < 64; off <<= 1) v = fmaxf(v, __shfl_xor(v, off, 64));
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  v = sh[0];
#pragma unroll
  for (int i = 1; i < NT / 64; ++i) v = fmaxf(v, sh[i]);
  return v;
}

template <int NT>
__device__ inline float block_sum(float v, float *sh) {
  for (int off = 1; off < 64; off <<= 1) v += __shfl_xor(v, off, 64);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  v = sh[0];
#pragma unroll
  for (int i = 1; i < NT / 64; ++i) v += sh[i];
  return v;
}

// The elements of a row outside its whole granules: up to kPer - 1 at either end, one to each of the first threads.
template <class T>
struct Edges {
  int head, tail_from, count;
  __device__ explicit Edges(const Chunks<T> &row) {
    const int before = row.whole_from ? Chunks<T>::kPer - row.lead : 0;
    head = before < row.cols ? before : row.cols;
    const int after = row.column(row.whole_to, 0);
    tail_from = after > head ? after : head;
    count = head + row.cols - tail_from;
  }
  __device__ int column(int i) const { return i < head ? i : tail_from + i - head; }
};

// Rows of any length, one workgroup each: whole granules, CH a thread, kept in registers (CH > 0) or read again (CH == 0), and
// the edges' elements one a thread.
// Read and written once, this is bound by memory where several rows are at work on a CU: 5.7 TB/s for 8192 rows of 32000 in 16
// bits.  Rows of 10^5 halves fill the registers of a CU alone, and what it computes between reading and writing (two
// exponentials an element) shows: 4.1 TB/s.  Neither keeping a part in LDS so that two rows fit (3.8) nor fetching the next row
// as this one leaves the registers (4.0) nor reading twice (3.4) is faster.
template <class T, int NT, int CH>
__global__ void __launch_bounds__(NT, NT == 512 ? 4 : 1) k_softmax_block(SoftmaxArgs a) {
  constexpr int K = 16 / sizeof(T);
  typedef vec_t<T, K> chunk;
  __shared__ float sh[2][NT / 64];
  const T none = (T)-INFINITY;
  const int tid = (int)threadIdx.x;
  for (uint64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    float w;
    const int64_t t = label_of(a, r, w);
    const Chunks<T> row(static_cast<const T *>(a.logits) + r * a.stride, (int)a.cols);
    const Edges<T> edges(row);
    const T *const from = row.base + row.lead;
    T *const to = a.grad ? static_cast<T *>(a.grad) + r * a.gstride : nullptr;
    const chunk *const in = reinterpret_cast<const chunk *>(row.base) + row.whole_from;
    const int count = row.whole_to - row.whole_from;  // may be negative: then all elements are edges
    auto put = [&](int c, const chunk &x) {
      if (!a.apart) {
        reinterpret_cast<chunk *>(to - row.lead)[row.whole_from + c] = x;
      } else {
#pragma unroll
        for (int k = 0; k < K; ++k) to[row.column(row.whole_from + c, k)] = x[k];
      }
    };
    const chunk zero = (T)0.0f;
    if (t < 0 && !a.lse) {  // nothing of the row is needed
      if (to) {
        for (int c = tid; c < count; c += NT) put(c, zero);
        if (tid < edges.count) to[edges.column(tid)] = (T)0.0f;
      }
      if (tid == 0) a.loss[r] = 0.0f;
      continue;
    }
    const float xt = (float)from[t >= 0 ? t : 0];  // before anyone writes over it
    // The label's chunk is not held or walked through with the others, which so need not ask for the label: its elements are loose
    // ones like the edges', one a thread.  (Every chunk asked: 100 us for 1001 rows of 100003, this: 95.)
    const int tc = t < 0 ? -1 : (int)t + row.lead - row.whole_from * K;
    const int label_chunk = tc >= 0 && tc < count * K ? tc / K : -1;  // or the label is at an edge
    int loose = -1;  // this thread's column
    if (tid < edges.count) loose = edges.column(tid);
    else if (label_chunk >= 0 && tid < edges.count + K) loose = row.column(row.whole_from + label_chunk, tid - edges.count);
    const float at_loose = (float)from[loose >= 0 ? loose : 0];  // without a branch, which would wait for it before the row is asked for
    float edge = loose >= 0 ? at_loose : -INFINITY;
    float m = edge;  // the label is in the maximum, not in the sum
    if (loose >= 0 && loose == (int)t) edge = -INFINITY;
    chunk x[CH ? CH : 1];
    // One pass: the sum is kept relative to the running maximum, so that the exponentials are computed while the row arrives: 177
    // us for 8192 rows of 32000 where a maximum first and the sum after it takes 185.  With 16 granules a thread it needs more
    // registers than there are: 95 us the other way for 1001 rows of 100003, 100 this way.
    constexpr bool kOnePass = CH < 16;
    Shift b(m);
    float s = exp2_fast(__fmaf_rn(edge, b.l, -b.m2));
    auto take = [&](const chunk &y) {
      const float mc = chunk_max<T>(y, m);
      if (mc > m) {
        const Shift next(mc);
        s *= m == -INFINITY ? 1.0f : moved(b, next);  // s is 0 (or NaN) while no class was seen
        m = mc;
        b = next;
      }
      s += chunk_sum<T>(y, b);
    };
    if (CH) {
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int at = c * NT + tid;
        x[c] = none;
        if (at < count && at != label_chunk) x[c] = in[at];
      }
      if (kOnePass) {
#pragma unroll
        for (int c = 0; c < CH; ++c) take(x[c]);
      } else {
#pragma unroll
        for (int c = 0; c < CH; ++c) m = chunk_max<T>(x[c], m);
      }
    } else {
      for (int c = tid; c < count; c += NT)
        if (c != label_chunk) take(in[c]);
    }
    const float mine = m;
    const Shift was = b;
    m = block_max<NT>(m, sh[0]);
    b = Shift(m);
    if (kOnePass) {
      if (mine != -INFINITY) s *= moved(was, b);
    } else {
      s = exp2_fast(__fmaf_rn(edge, b.l, -b.m2));
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        stay_packed(x[c]);
        s += chunk_sum<T>(x[c], b);
      }
    }
    const float others = block_sum<NT>(s, sh[1]), e = label_power(t, xt, b);
    s = others + e;
    if (tid == 0) finish_row(a, r, b, others, e, t, w, xt);
    if (to) {
      const float share = (t < 0 ? 0.0f : w * a.grad_scale) / s, gl = share * others;
      const bool no = t < 0 || s == 0.0f;
      if (loose >= 0) to[loose] = no ? (T)0.0f : (T)(loose == (int)t ? -gl : share * exp2_fast(__fmaf_rn(edge, b.l, -b.m2)));
      if (CH) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          const int at = c * NT + tid;
          stay_packed(x[c]);
          if (at < count && at != label_chunk) put(at, no ? zero : chunk_grad<T>(x[c], b, share));
        }
      } else {
        for (int c = tid; c < count; c += NT)
          if (c != label_chunk) put(c, no ? zero : chunk_grad<T>(in[c], b, share));
      }
    }
    __syncthreads();  // sh is free again
  }
}

// ---- few long rows: several workgroups each -------------------------------------------------------------
//
// A row is cut into pieces of kPiece granules.  The first launch leaves every piece's largest logit and its sum relative to
// that; the second puts a row's pieces together (every workgroup for itself, in the same order) and writes the gradient of
// its own, which it reads again from the cache.
// For fewer than kFewRows rows of more than kLong granules (us for 8 rows in 16 bits, this and a workgroup a row: 48000 classes
// 10.4 and 9.3, 65000 10.2 and 10.4, 80000 10.4 and 13.9, 131000 10.1 and 16.8; 127 rows of 80000 15.2 and 16.9, of 131000 19.9
// and 21.9, but 256 of 128000 35.5 and 28).
constexpr int kPiece = 2048, kLong = 8192;
constexpr uint64_t kFewRows = 128;

struct Piece {
  float m, s;
};

template <class T>
__global__ void __launch_bounds__(256) k_softmax_pieces(SoftmaxArgs a, Piece *pieces, float *label_logits) {
  __shared__ float sh[2][4];
  constexpr int K = 16 / sizeof(T);
  const uint64_t r = blockIdx.y;
  float w;
  const int64_t t = label_of(a, r, w);
  if (t < 0 && !a.lse) return;
  const Chunks<T> row(static_cast<const T *>(a.logits) + r * a.stride, (int)a.cols);
  const T none = (T)-INFINITY;
  const int c0 = (int)blockIdx.x * kPiece + (int)threadIdx.x;
  vec_t<T, K> x[kPiece / 256];
  float m = -INFINITY, s = 0.0f;
#pragma unroll
  for (int i = 0; i < kPiece / 256; ++i) {
    x[i] = none;
    if (c0 + i * 256 < row.count) x[i] = row.load(c0 + i * 256, none);
    m = chunk_max<T>(x[i], m);
  }
  m = block_max<256>(m, sh[0]);
  const Shift b(m);
  // the label is in the maximum, not in the sum
  const int tc = t < 0 ? -1 : (int)t + row.lead, label_chunk = t < 0 ? -1 : tc / K;
#pragma unroll
  for (int i = 0; i < kPiece / 256; ++i) {
    const bool labels = c0 + i * 256 == label_chunk;
    if (__ballot(labels)) take_out<T>(x[i], labels ? tc - label_chunk * K : -1);
    stay_packed(x[i]);
    s += chunk_sum<T>(x[i], b);
  }
  s = block_sum<256>(s, sh[1]);
  if (threadIdx.x != 0) return;
  pieces[r * gridDim.x + blockIdx.x] = Piece{m, s};
  if (blockIdx.x == 0) label_logits[r] = t >= 0 ? (float)row.base[row.lead + t] : 0.0f;  // the next launch may write over it
}

template <class T>
__global__ void __launch_bounds__(256) k_softmax_pieces_grad(SoftmaxArgs a, const Piece *pieces, const float *label_logits, unsigned count) {
  constexpr int K = 16 / sizeof(T);
  const uint64_t r = blockIdx.y;
  float w;
  const int64_t t = label_of(a, r, w);
  const Chunks<T> row(static_cast<const T *>(a.logits) + r * a.stride, (int)a.cols);
  const vec_t<T, K> zero = (T)0.0f;
  const float xt = label_logits[r];  // of a row that is not trained on it may be anything
  float others = 0.0f, e = 0.0f;
  Shift b(0.0f);
  if (t >= 0 || a.lse) {
    // every wave for itself: its lanes take pieces in turn
    float m = -INFINITY;
    for (unsigned i = threadIdx.x & 63; i < count; i += 64) m = fmaxf(m, pieces[r * count + i].m);
    for (int off = 1; off < 64; off <<= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
    b = Shift(m);
    for (unsigned i = threadIdx.x & 63; i < count; i += 64) {
      const Piece p = pieces[r * count + i];
      others += p.m == -INFINITY ? p.s : p.s * moved(Shift(p.m), b);  // s of a piece without classes: 0, or NaN
    }
    for (int off = 1; off < 64; off <<= 1) others += __shfl_xor(others, off, 64);
    e = label_power(t, xt, b);
    if (blockIdx.x == 0 && threadIdx.x == 0) finish_row(a, r, b, others, e, t, w, xt);
  } else if (blockIdx.x == 0 && threadIdx.x == 0) {
    a.loss[r] = 0.0f;
  }
  if (!a.grad) return;
  T *const to = static_cast<T *>(a.grad) + r * a.gstride;
  const float s = others + e, share = (t < 0 ? 0.0f : w * a.grad_scale) / s, gl = share * others;
  const int tc = t < 0 ? -1 : (int)t + row.lead;
#pragma unroll
  for (int i = 0; i < kPiece / 256; ++i) {
    const int at = (int)blockIdx.x * kPiece + (int)threadIdx.x + i * 256;
    if (at >= row.count) break;
    row.store(to, a.apart, at, t < 0 || s == 0.0f ? zero : chunk_grad<T>(row.load(at, (T)-INFINITY), b, share, gl, tc - at * K));
  }
}

// pieces of a row, whatever its alignment
static uint64_t piece_count(uint64_t cols, uint64_t per) { return ((cols + per - 1) / per + 1 + kPiece - 1) / kPiece; }

template <class T>
static int softmax_loss(admm_ctx *ctx, SoftmaxArgs a, void *workspace) {
  constexpr uint64_t K = 16 / sizeof(T);
  auto offset = [](const void *p) { return reinterpret_cast<uintptr_t>(p) & 15; };
  a.apart = a.grad && (offset(a.grad) != offset(a.logits) || (a.rows > 1 && (a.gstride - a.stride) * sizeof(T) % 16 != 0));
  const bool even = offset(a.logits) == 0 && (a.rows == 1 || a.stride * sizeof(T) % 16 == 0);
  const uint64_t chunks = (a.cols + K - 1) / K + (even ? 0 : 1);  // a row between granules touches one more
  // The fewest registers and threads that hold a row.  Up to 256 granules a wave holds rows without barriers (8192 rows of 1000
  // in 16 bits: 9 us, by the next form 22; of 2000: 15 and 24).  Each of the others against the one after it, in 16 bits: 8192
  // rows of 8000 42 and 50 us, of 16000 101 and 128, 4096 of 32000 100 and 116, 2048 of 64000 108 and 153, 1024 of 128000 123
  // and 143.
  if (chunks <= 256) {
    a.lanes_log2 = 0;
    while (a.lanes_log2 < 6 && (1ull << a.lanes_log2) < chunks) ++a.lanes_log2;
    const dim3 grid(blocks_for(a.rows, 256u >> a.lanes_log2));
    if (chunks <= 64) hipLaunchKernelGGL((k_softmax_lanes<T, 1>), grid, dim3(256), 0, ctx->stream, a);
    else if (chunks <= 128) hipLaunchKernelGGL((k_softmax_lanes<T, 2>), grid, dim3(256), 0, ctx->stream, a);
    else hipLaunchKernelGGL((k_softmax_lanes<T, 4>), grid, dim3(256), 0, ctx->stream, a);
  } else if (a.rows < kFewRows && chunks > kLong) {
    const dim3 grid((unsigned)piece_count(a.cols, K), (unsigned)a.rows);
    float *label_logits = static_cast<float *>(workspace);
    Piece *pieces = reinterpret_cast<Piece *>(label_logits + kFewRows);
    hipLaunchKernelGGL(k_softmax_pieces<T>, grid, dim3(256), 0, ctx->stream, a, pieces, label_logits);
    hipLaunchKernelGGL(k_softmax_pieces_grad<T>, a.grad ? grid : dim3(1, grid.y), dim3(256), 0, ctx->stream, a, pieces, label_logits, grid.x);
  } else {
    const dim3 grid(blocks_for(a.rows, 1));
    if (chunks <= 1024) hipLaunchKernelGGL((k_softmax_block<T, 256, 4>), grid, dim3(256), 0, ctx->stream, a);
    else if (chunks <= 2048) hipLaunchKernelGGL((k_softmax_block<T, 256, 8>), grid, dim3(256), 0, ctx->stream, a);
    else if (chunks <= 4096) hipLaunchKernelGGL((k_softmax_block<T, 512, 8>), grid, dim3(512), 0, ctx->stream, a);
    else if (chunks <= 8192) hipLaunchKernelGGL((k_softmax_block<T, 512, 16>), grid, dim3(512), 0, ctx->stream, a);
    else if (chunks <= 16384) hipLaunchKernelGGL((k_softmax_block<T, 1024, 16>), grid, dim3(1024), 0, ctx->stream, a);
    else hipLaunchKernelGGL((k_softmax_block<T, 1024, 0>), grid, dim3(1024), 0, ctx->stream, a);
  }
  ADMM_HIP_CHECK(hipGetLastError());
  return ADMM_OK;
}

}  // namespace admm_impl

using namespace admm_impl;

extern "C" int admm_softmax_loss_workspace(uint64_t rows, uint64_t cols, uint64_t *bytes) {
  ADMM_REQUIRE(bytes, "admm_softmax_loss_workspace: bytes is NULL");
  ADMM_REQUIRE(rows < (1ull << 40) && cols <= kMaxClasses, "admm_softmax_loss_workspace: %llu x %llu logits", (unsigned long long)rows,
               (unsigned long long)cols);
  // of the narrowest granules, for logits of any type
  *bytes = rows && rows < kFewRows && (cols + 3) / 4 + 1 > kLong ? kFewRows * sizeof(float) + rows * piece_count(cols, 4) * sizeof(Piece) : 0;
  return ADMM_OK;
}

extern "C" int admm_softmax_loss(admm_ctx *ctx, const admm_mat *logits, const void *labels, int label_type, const float *weight,
                                 float grad_scale, float *loss, float *lse, const admm_mat *grad, void *workspace,
                                 uint64_t workspace_bytes) {
  ADMM_REQUIRE(ctx, "admm_softmax_loss: ctx is NULL");
  ADMM_TRY(check_mat(logits, "admm_softmax_loss", "logits"));
  ADMM_REQUIRE(label_type == ADMM_I32 || label_type == ADMM_I64 || label_type == ADMM_F32, "admm_softmax_loss: labels of type %d", label_type);
  if (grad) {
    ADMM_TRY(check_mat(grad, "admm_softmax_loss", "grad"));
    ADMM_REQUIRE(grad->rows == logits->rows && grad->cols == logits->cols && grad->type == logits->type,
                 "admm_softmax_loss: grad has another shape or type than the logits");
    const bool same = grad->data == logits->data && (grad->stride == logits->stride || grad->rows <= 1);
    ADMM_REQUIRE(same || !mats_overlap(grad, logits), "admm_softmax_loss: grad overlaps the logits and is not their own memory");
  }
  if (logits->rows == 0) return ADMM_OK;
  ADMM_REQUIRE(logits->cols > 0, "admm_softmax_loss: no classes");
  ADMM_REQUIRE(logits->cols <= kMaxClasses, "admm_softmax_loss: %llu classes", (unsigned long long)logits->cols);
  ADMM_REQUIRE(labels && loss, "admm_softmax_loss: labels or loss is NULL");
  uint64_t need = 0;
  ADMM_TRY(admm_softmax_loss_workspace(logits->rows, logits->cols, &need));
  ADMM_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && reinterpret_cast<uintptr_t>(workspace) % 16 == 0),
               "admm_softmax_loss: the workspace is NULL, not on 16 bytes or smaller than %llu bytes", (unsigned long long)need);
  OnDevice on(ctx->device);
  ADMM_HIP_CHECK(on.error);
  KernelTimer t(ctx, ADMM_K_SOFTMAX);
  SoftmaxArgs a = {};
  a.logits = logits->data;
  a.stride = logits->stride;
  a.grad = grad ? grad->data : nullptr;
  a.gstride = grad ? grad->stride : 0;
  a.rows = logits->rows;
  a.cols = logits->cols;
  a.labels = labels;
  a.label_type = label_type;
  a.weight = weight;
  a.grad_scale = grad_scale;
  a.loss = loss;
  a.lse = lse;
  return logits->type == ADMM_F32 ? softmax_loss<float>(ctx, a, workspace) : logits->type == ADMM_BF16 ? softmax_loss<bf16_t>(ctx, a, workspace) : softmax_loss<f16_t>(ctx, a, workspace);
}
