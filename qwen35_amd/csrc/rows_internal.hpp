// rows_internal.hpp -- what the operators on rows of heads share (norms, rotary
// positions, linear attention): the checks of qhip_rows descriptors and pieces of
// eight elements.
#pragma once
#include "kv_internal.hpp"

namespace qhip {

// Rows that are read: elements of `size` bytes, strides that are not negative
// (0: the same elements for every token or head).
inline bool rows_ok(const qhip_rows* r, int size) {
  return r && r->at && (uintptr_t)r->at % size == 0 && r->token_stride >= 0 && r->head_stride >= 0 &&
         r->token_stride <= 0x7FFFFFFFL && r->head_stride <= 0x7FFFFFFFFFFFL;
}
// elements from the first to behind the last
inline long rows_span(const qhip_rows* r, int tokens, int heads, int dim) {
  return (long)(tokens - 1) * r->token_stride + (long)(heads - 1) * r->head_stride + dim;
}
// Rows that are written: no element of them twice (heads inside a token's row, or
// tokens inside a head's).
inline bool rows_apart(const qhip_rows* r, int tokens, int heads, int dim) {
  const long t = r->token_stride, h = r->head_stride;
  if (tokens == 1) return heads == 1 || h >= dim;
  if (heads == 1) return t >= dim;
  return (h >= dim && t >= (heads - 1) * h + dim) || (t >= dim && h >= (tokens - 1) * t + dim);
}
inline bool rows_same(const qhip_rows* a, const qhip_rows* b) {
  return a->at == b->at && a->token_stride == b->token_stride && a->head_stride == b->head_stride;
}
// Whether two sets of rows may share memory.  Columns of one wider array (equal token
// strides, heads inside them) do not, though their ranges meet.
inline bool rows_overlap(const qhip_rows* a, int a_heads, int a_dim, const qhip_rows* b, int b_heads, int b_dim, int tokens,
                         int size) {
  const char *pa = (const char*)a->at, *pb = (const char*)b->at;
  if (pa >= pb + rows_span(b, tokens, b_heads, b_dim) * size || pb >= pa + rows_span(a, tokens, a_heads, a_dim) * size) return false;
  const long row = a->token_stride * size;
  if (tokens > 1 && a->token_stride == b->token_stride && row > 0) {
    const long wa = ((a_heads - 1) * a->head_stride + a_dim) * size, wb = ((b_heads - 1) * b->head_stride + b_dim) * size;
    const long off = (((pb - pa) % row) + row) % row;  // of b's columns in a's row
    if (wa <= row && wb <= row && off >= wa && off + wb <= row) return false;
  }
  // nor do parts of one array's heads
  const long head = a->head_stride * size;
  if (head > 0 && a->head_stride == b->head_stride &&
      (tokens == 1 || (a->token_stride == b->token_stride && a->token_stride % a->head_stride == 0))) {
    const long off = (((pb - pa) % head) + head) % head;
    if (off >= (long)a_dim * size && off + (long)b_dim * size <= head) return false;
  }
  return true;
}
// bytes [p, p + n) against the rows' range
inline bool rows_meet(const qhip_rows* r, int tokens, int heads, int dim, int size, const void* p, long n) {
  const char *a = (const char*)r->at, *b = (const char*)p;
  return n > 0 && b < a + rows_span(r, tokens, heads, dim) * size && a < b + n;
}

// Eight elements at p, or the n < 8 that there are (0 behind them), as floats.
template <typename T>
__device__ __forceinline__ void get8(const T* p, int n, float (&v)[8]) {
  if (n >= 8) {
    const Raw8<T> r = load8(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)r.e[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? (float)p[i] : 0.0f;
  }
}
template <typename T>
__device__ __forceinline__ void put8(T* p, int n, const float (&v)[8]) {
  if (n >= 8) {
    typedef uint32_t piece __attribute__((ext_vector_type(4), aligned(2)));
    Raw8<T> r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r.e[i] = (T)v[i];
    struct Pieces {
      kv_u32x4 x[sizeof(Raw8<T>) / 16];
    } out = __builtin_bit_cast(Pieces, r);
#pragma unroll
    for (unsigned i = 0; i < sizeof(out) / 16; ++i) ((piece*)p)[i] = out.x[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = (T)v[i];
  }
}

}  // namespace qhip
