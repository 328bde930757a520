// kv_attention.hip -- attention over the 8-bit key/value cache.
//
// One wave per packed token and query head: 64 keys at a time, a key a lane
// for the scores, eight or fewer dimensions' sums a lane for the output, with
// the running maximum and sum of the softmax in f32.
#include "kv_internal.hpp"

namespace qhip {

struct KvAttnArgs {
  const int8_t *k, *v;
  const float *k_scale, *v_scale;
  const int *offsets, *kv_lens, *table;
  const void* q;
  void* out;
  float* lse;
  long q_token, q_head, out_token, out_head;
  int nseq, tokens, width, shift, num_blocks, kv_heads, q_heads;
  float scale;
  int causal, window;
};

template <typename T, int D>
__global__ __launch_bounds__(64) void k_kv_attention(KvAttnArgs a) {
  constexpr int R = D / 64;
  __shared__ float s_q[D], s_p[64];
  __shared__ long s_at[64];
  const int t = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
  int lo = 0, hi = a.nseq;  // the token's sequence
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.offsets[mid] <= t) lo = mid; else hi = mid;
  }
  if (t >= a.offsets[a.nseq]) return;
  const int len = a.kv_lens[lo], p = len - a.offsets[lo + 1] + t;
  const int end = a.causal ? min(p + 1, len) : len;
  const int begin = a.causal && a.window > 0 ? max(0, p - a.window + 1) : 0;
  const int kh = h / (a.q_heads / a.kv_heads), mask = (1 << a.shift) - 1;
  const T* q = (const T*)a.q + (long)t * a.q_token + (long)h * a.q_head;
  for (int d = lane; d < D; d += 64) s_q[d] = (float)q[d];
  __syncthreads();
  float m = -INFINITY, l = 0.0f, acc[R] = {};
  for (int j0 = begin; j0 < end; j0 += 64) {
    const int j = j0 + lane;
    float s = -INFINITY, vs = 0.0f;
    long at = 0;
    if (j < end) {
      const int b = j >> a.shift, id = b < a.width ? a.table[(long)lo * a.width + b] : -1;
      const bool in = (unsigned)id < (unsigned)a.num_blocks;
      const long bh = in ? (long)id * a.kv_heads + kh : 0;
      at = (bh << a.shift | (j & mask)) * D;
      float dot = 0.0f;
      for (int d = 0; d < D; ++d) dot = __builtin_fmaf(s_q[d], (float)a.k[at + d], dot);
      const float ks = in ? a.k_scale[bh] : __builtin_nanf("");
      s = finite_bits(__float_as_uint(ks)) ? dot * ks * a.scale : __builtin_nanf("");
      vs = a.v_scale[bh];
      vs = finite_bits(__float_as_uint(vs)) ? vs : __builtin_nanf("");
    }
    float top = s;
    for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
    const float m1 = fmaxf(m, top), alpha = m == -INFINITY ? 0.0f : expf(m - m1);
    const float e = j < end ? (s == -INFINITY ? 0.0f : expf(s - m1)) : 0.0f;
    float sum = e;
    for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d, 64);
    l = l * alpha + sum;
    m = m1;
    __syncthreads();
    s_p[lane] = j < end ? e * vs : 0.0f;
    s_at[lane] = at;
    __syncthreads();
    for (int r = 0; r < R; ++r) {
      float o = acc[r] * alpha;
      for (int i = 0; i < min(64, end - j0); ++i) o = __builtin_fmaf(s_p[i], (float)a.v[s_at[i] + lane + 64 * r], o);
      acc[r] = o;
    }
  }
  T* out = (T*)a.out + (long)t * a.out_token + (long)h * a.out_head;
  for (int r = 0; r < R; ++r) out[lane + 64 * r] = (T)(end > begin ? acc[r] / l : 0.0f);
  if (a.lse && lane == 0) a.lse[(long)t * a.q_heads + h] = end > begin ? m + logf(l) : -INFINITY;
}

template <typename T>
static void launch_attention(const KvAttnArgs& a, int dim, hipStream_t s) {
  const dim3 grid((unsigned)a.tokens, (unsigned)a.q_heads);
  if (dim == 64) hipLaunchKernelGGL((k_kv_attention<T, 64>), grid, dim3(64), 0, s, a);
  else if (dim == 128) hipLaunchKernelGGL((k_kv_attention<T, 128>), grid, dim3(64), 0, s, a);
  else hipLaunchKernelGGL((k_kv_attention<T, 256>), grid, dim3(64), 0, s, a);
}

// 0, hipErrorInvalidValue or QHIP_DECLINE
static int check_batch(const qhip_kv_cache* cache, const qhip_kv_batch* b, int q_heads) {
  const int rc = kv_check_cache(cache);
  if (rc == (int)hipErrorInvalidValue || !b) return (int)hipErrorInvalidValue;
  if (b->nseq < 0 || b->tokens < 0 || b->max_new < 0 || b->max_kv < 0 || b->table_width < 0) return (int)hipErrorInvalidValue;
  if (q_heads <= 0 || q_heads > 65535 || q_heads % cache->kv_heads) return (int)hipErrorInvalidValue;
  return rc;
}

}  // namespace qhip

using namespace qhip;

extern "C" long qhip_kv_attention_work_bytes(const qhip_kv_cache* cache, const qhip_kv_batch* batch, int q_heads) {
  return check_batch(cache, batch, q_heads) ? -1 : 0;
}

extern "C" int qhip_launch_kv_attention(const qhip_kv_cache* cache, const qhip_kv_batch* batch, int type,
                                        const void* d_q, long q_token_stride, long q_head_stride, int q_heads,
                                        float softmax_scale, int causal, int window, void* d_out,
                                        long out_token_stride, long out_head_stride, float* d_lse, void* d_work,
                                        long work_bytes, void* stream) {
  const int rc = check_batch(cache, batch, q_heads), size = kv_type_size(type);
  if (rc == (int)hipErrorInvalidValue || !size || (causal != 0 && causal != 1) || window < 0 || (window > 0 && !causal) ||
      work_bytes < 0 || !aligned16(d_work))
    return (int)hipErrorInvalidValue;
  if (batch->tokens > 0 && batch->nseq > 0 &&
      (!d_q || !d_out || ((uintptr_t)d_q % size) || ((uintptr_t)d_out % size) || !batch->offsets || !batch->kv_lens ||
       (batch->table_width > 0 && !batch->table)))
    return (int)hipErrorInvalidValue;
  if (rc) return rc;
  if (batch->tokens == 0 || batch->nseq == 0) return 0;
  const KvAttnArgs a{(const int8_t*)cache->k, (const int8_t*)cache->v, cache->k_scale, cache->v_scale, batch->offsets,
                     batch->kv_lens, batch->table, d_q, d_out, d_lse, q_token_stride, q_head_stride, out_token_stride,
                     out_head_stride, batch->nseq, batch->tokens, batch->table_width, kv_block_shift(cache->block_size),
                     cache->num_blocks, cache->kv_heads, q_heads, softmax_scale, causal, window};
  hipStream_t s = (hipStream_t)stream;
  if (type == QHIP_TT_F32) launch_attention<float>(a, cache->head_dim, s);
  else if (type == QHIP_TT_F16) launch_attention<f16_t>(a, cache->head_dim, s);
  else launch_attention<bf16_t>(a, cache->head_dim, s);
  return (int)hipGetLastError();
}
