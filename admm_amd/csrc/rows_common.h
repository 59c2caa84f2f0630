// Shared by the many-class operators (embed.hip, softmax.hip, sample.hip): element types, 16-byte chunks of rows of any
// alignment, checks of the matrices in their arguments.
#pragma once

#include "internal.h"

namespace admm_impl {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

template <class T, int N>
using vec_t = T __attribute__((ext_vector_type(N)));

constexpr float kLog2e = 1.44269504088896341f;
constexpr float kLn2 = 0.69314718055994531f;

inline uint64_t type_bytes(int type) { return type == ADMM_F32 || type == ADMM_I32 ? 4 : type == ADMM_I64 ? 8 : 2; }

// N elements from / to `p`, which is aligned to min(16, N * sizeof(T)) bytes
template <class T, int N>
__device__ inline void load_n(const T *p, float (&v)[N]) {
  constexpr int M = N * sizeof(T) > 16 ? (int)(16 / sizeof(T)) : N;
#pragma unroll
  for (int i = 0; i < N; i += M) {
    const vec_t<T, M> x = *reinterpret_cast<const vec_t<T, M> *>(p + i);
#pragma unroll
    for (int k = 0; k < M; ++k) v[i + k] = (float)x[k];
  }
}

template <class T, int N>
__device__ inline void store_n(T *p, const float (&v)[N]) {
  constexpr int M = N * sizeof(T) > 16 ? (int)(16 / sizeof(T)) : N;
#pragma unroll
  for (int i = 0; i < N; i += M) {
    vec_t<T, M> x;
#pragma unroll
    for (int k = 0; k < M; ++k) x[k] = (T)v[i + k];
    *reinterpret_cast<vec_t<T, M> *>(p + i) = x;
  }
}

// A row of `cols` elements at any address, seen as the granules of 16 (or BYTES) bytes of memory that it touches: all but the
// first and the last are whole and are read and written at once, those two element by element, so nothing outside the row
// is touched.  Element k of chunk c is column c * kPer + k - lead.
template <class T, int BYTES = 16>
struct Chunks {
  static constexpr int kPer = BYTES / sizeof(T);
  const T *base;  // on BYTES bytes; the row begins `lead` elements after it
  int lead, cols, count;
  int whole_from, whole_to;  // chunks that lie in the row altogether
  __device__ Chunks(const T *row, int n) {
    lead = (int)((reinterpret_cast<uintptr_t>(row) & (BYTES - 1)) / sizeof(T));
    base = row - lead;
    cols = n;
    count = (int)(((unsigned)lead + (unsigned)n + kPer - 1) / kPer);
    whole_from = lead ? 1 : 0;
    whole_to = (int)(((unsigned)lead + (unsigned)n) / kPer);
  }
  __device__ int column(int c, int k) const { return c * kPer + k - lead; }
  __device__ vec_t<T, kPer> load(int c, T other) const {
    if (c >= whole_from && c < whole_to) return *reinterpret_cast<const vec_t<T, kPer> *>(base + (int64_t)c * kPer);
    vec_t<T, kPer> x;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int j = column(c, k);
      x[k] = other;
      if (j >= 0 && j < cols) x[k] = base[(int64_t)c * kPer + k];
    }
    return x;
  }
  // to another row; `apart`: of another alignment
  __device__ void store(T *row, bool apart, int c, vec_t<T, kPer> x) const {
    T *to = row - lead;
    if (!apart && c >= whole_from && c < whole_to) {
      *reinterpret_cast<vec_t<T, kPer> *>(to + (int64_t)c * kPer) = x;
      return;
    }
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int j = column(c, k);
      if (j >= 0 && j < cols) to[(int64_t)c * kPer + k] = x[k];
    }
  }
};

constexpr uint64_t kMaxClasses = 0x7FFFFF00;  // chunks and columns of a row of logits are counted in ints

// ---- host side ----------------------------------------------------------------------------------

// type, stride, alignment to the element and size of a matrix argument
inline int check_mat(const admm_mat *m, const char *who, const char *name) {
  ADMM_REQUIRE(m, "%s: %s is NULL", who, name);
  ADMM_REQUIRE(m->type == ADMM_F32 || m->type == ADMM_BF16 || m->type == ADMM_F16, "%s: %s has type %d", who, name, m->type);
  if (m->rows == 0 || m->cols == 0) return ADMM_OK;
  ADMM_REQUIRE(m->data, "%s: %s has no memory", who, name);
  ADMM_REQUIRE(m->stride >= m->cols || m->rows == 1, "%s: %s has rows of %llu elements, %llu apart", who, name,
               (unsigned long long)m->cols, (unsigned long long)m->stride);
  ADMM_REQUIRE(reinterpret_cast<uintptr_t>(m->data) % type_bytes(m->type) == 0, "%s: %s is not aligned to its elements", who, name);
  ADMM_REQUIRE(m->cols < (1ull << 40) && m->rows < (1ull << 40) &&
                   (unsigned __int128)m->rows * (m->stride > m->cols ? m->stride : m->cols) < ((unsigned __int128)1 << 46),
               "%s: %s is too large", who, name);
  return ADMM_OK;
}

inline bool overlap(const void *a, uint64_t na, const void *b, uint64_t nb) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return na && nb && x < y + nb && y < x + na;
}

// from the first element to the last
inline uint64_t mat_span(const admm_mat *m) {
  return m->rows && m->cols ? ((m->rows - 1) * m->stride + m->cols) * type_bytes(m->type) : 0;
}

// Do they share an element?  Rows of one stride may lie side by side: then their places within the stride tell.
inline bool mats_overlap(const admm_mat *a, const admm_mat *b) {
  if (!overlap(a->data, mat_span(a), b->data, mat_span(b))) return false;
  const uint64_t na = a->cols * type_bytes(a->type), nb = b->cols * type_bytes(b->type);
  const uint64_t sa = a->stride * type_bytes(a->type), sb = b->stride * type_bytes(b->type);
  if ((a->rows <= 1 && b->rows <= 1) || (a->rows > 1 && b->rows > 1 && sa != sb)) return true;
  const uint64_t stride = a->rows > 1 ? sa : sb;
  const uintptr_t x = reinterpret_cast<uintptr_t>(a->data), y = reinterpret_cast<uintptr_t>(b->data);
  const uint64_t from = y >= x ? (y - x) % stride : (stride - (x - y) % stride) % stride;  // where b's rows begin, from a's on
  return from < na || from + nb > stride;
}

// can rows of this matrix be read and written n elements at a time from column 0 on?
inline bool rows_aligned(const admm_mat *m, uint64_t n) {
  const uint64_t bytes = n * type_bytes(m->type) < 16 ? n * type_bytes(m->type) : 16;
  return reinterpret_cast<uintptr_t>(m->data) % bytes == 0 && (m->rows <= 1 || m->stride * type_bytes(m->type) % bytes == 0);
}

inline uint64_t round_up(uint64_t n, uint64_t to) { return (n + to - 1) / to * to; }

// blocks for `units` of work at `per_block` a block; kernels go on by gridDim.x blocks where it is not enough
inline unsigned blocks_for(uint64_t units, uint64_t per_block, uint64_t most = 1u << 21) {
  const uint64_t b = (units + per_block - 1) / per_block;
  return (unsigned)(b < 1 ? 1 : b > most ? most : b);
}

}  // namespace admm_impl
