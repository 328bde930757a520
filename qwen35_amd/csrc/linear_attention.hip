// linear_attention.hip -- linear attention with a decay for each head, over a pool
// of states.  For a head with state S [key_dim, value_dim] and a token's q, k, v,
// a = exp(log_decay):
//
//   S <- a S;  u = beta (v - k S) with the delta rule, else v
//   S <- S + k^T u;  out = scale q S
//
// Columns of S (value dimensions) do not see each other.
#include "qhip_device.hpp"
#include "qhip_internal.hpp"
#include "rows_internal.hpp"

namespace qhip {

typedef float f32x4 __attribute__((ext_vector_type(4)));

struct LinearArgs {
  const void *q, *k, *v;
  void* out;
  long q_token, q_head, k_token, k_head, v_token, v_head, out_token, out_head;
  const float *log_decay, *beta;
  long decay_token, beta_token;
  float* states;
  const int *offsets, *slots, *source;
  int nseq, tokens, max_new, num_states, k_heads, v_heads, value_dim, group;
  float scale;
};

// A sequence's packed tokens (those among `tokens`, at most max_new) and the
// states that it reads and writes (nullptr: zeros, and nowhere).
struct LinearSeq {
  int first, n;
  const float* from;
  float* to;
  bool bad;  // the source is no state
};
__device__ __forceinline__ LinearSeq linear_seq(const LinearArgs& a, int i, int head, int key_dim) {
  LinearSeq s{a.offsets[i], 0, nullptr, nullptr, false};
  const int end = min(a.offsets[i + 1], a.tokens);
  if (s.first >= 0 && end > s.first) s.n = min(end - s.first, a.max_new);
  const long size = (long)key_dim * a.value_dim;
  const int to = a.slots[i], from = a.source ? a.source[i] : to;
  if ((unsigned)to < (unsigned)a.num_states) s.to = a.states + ((long)to * a.v_heads + head) * size;
  if ((unsigned)from < (unsigned)a.num_states) s.from = a.states + ((long)from * a.v_heads + head) * size;
  else s.bad = from != -1;
  return s;
}

// sum over lanes l, l ^ 16, l ^ 32, l ^ 48
__device__ __forceinline__ float sum_rows(float v) {
  auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(x[0]) + __uint_as_float(x[1]);
  x = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(x[0]) + __uint_as_float(x[1]);
}

// ---- token by token --------------------------------------------------------------------
//
// A workgroup holds 64 columns of a head's state in registers: lane l of a wave
// columns 4 (l mod 16) ..+3 of DK / 16 rows.  A token's products k S and q S (of the
// state before it) are summed over the rows together, so that one exchange between
// the waves serves both:  out = scale (a q S + (q . k) u).
template <typename T, int DK>
__global__ __launch_bounds__(256) void k_linear_steps(LinearArgs a) {
  constexpr int R = DK / 16;  // rows of a thread
  __shared__ float s_part[2][4][2][64];
  __shared__ float s_qk[2][4];
  const int tid = threadIdx.x, wave = tid >> 6, col = (tid & 15) * 4, row0 = (tid >> 4) * R;
  const int seq = blockIdx.z, head = blockIdx.y, d0 = blockIdx.x * 64 + col;
  const LinearSeq s = linear_seq(a, seq, head, DK);
  if (s.n == 0 && s.from == s.to) return;
  f32x4 st[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    st[r] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    if (s.from) st[r] = *(const f32x4*)(s.from + (long)(row0 + r) * a.value_dim + d0);
    if (s.bad) st[r] = f32x4{__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
  }
  const int kh = head / a.group;
  const T* q = (const T*)a.q + s.first * a.q_token + kh * a.q_head + row0;
  const T* k = (const T*)a.k + s.first * a.k_token + kh * a.k_head + row0;
  const T* v = (const T*)a.v + s.first * a.v_token + head * a.v_head + d0;
  T* out = (T*)a.out + s.first * a.out_token + head * a.out_head + d0;
  const float* decay = a.log_decay + s.first * a.decay_token + head;
  const float* beta = a.beta ? a.beta + s.first * a.beta_token + head : nullptr;
  for (int t = 0; t < s.n; ++t) {
    float kr[R], qr[R], vc[4];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      kr[r] = (float)k[t * a.k_token + r];
      qr[r] = (float)q[t * a.q_token + r];
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) vc[c] = (float)v[t * a.v_token + c];
    const float keep = expf(decay[t * a.decay_token]), b = beta ? beta[t * a.beta_token] : 0.0f;
    float ks[4] = {}, qs[4] = {}, qk = 0.0f;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      qk = __builtin_fmaf(qr[r], kr[r], qk);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        ks[c] = __builtin_fmaf(kr[r], st[r][c], ks[c]);
        qs[c] = __builtin_fmaf(qr[r], st[r][c], qs[c]);
      }
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      ks[c] = sum_rows(ks[c]);
      qs[c] = sum_rows(qs[c]);
    }
    qk = sum_rows(qk);
    const int buf = t & 1;
    if ((tid & 63) < 16) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        s_part[buf][wave][0][col + c] = ks[c];
        s_part[buf][wave][1][col + c] = qs[c];
      }
      if ((tid & 63) == 0) s_qk[buf][wave] = qk;
    }
    __syncthreads();  // (the buffer after next is written behind the next token's barrier)
    qk = (s_qk[buf][0] + s_qk[buf][1]) + (s_qk[buf][2] + s_qk[buf][3]);
    float u[4], o[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const float(*p)[2][64] = s_part[buf];
      const float kc = (p[0][0][col + c] + p[1][0][col + c]) + (p[2][0][col + c] + p[3][0][col + c]);
      const float qc = (p[0][1][col + c] + p[1][1][col + c]) + (p[2][1][col + c] + p[3][1][col + c]);
      u[c] = a.beta ? b * (vc[c] - keep * kc) : vc[c];
      o[c] = a.scale * __builtin_fmaf(qk, u[c], keep * qc);
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int c = 0; c < 4; ++c) st[r][c] = __builtin_fmaf(kr[r], u[c], keep * st[r][c]);
    if (tid < 16) {
#pragma unroll
      for (int c = 0; c < 4; ++c) out[t * a.out_token + c] = (T)o[c];
    }
  }
  if (s.to) {
#pragma unroll
    for (int r = 0; r < R; ++r) *(f32x4*)(s.to + (long)(row0 + r) * a.value_dim + d0) = st[r];
  }
}

template <typename T>
static void launch_steps(const LinearArgs& a, int key_dim, hipStream_t s) {
  const dim3 grid((unsigned)(a.value_dim / 64), (unsigned)a.v_heads, (unsigned)a.nseq);
  if (key_dim == 64) hipLaunchKernelGGL((k_linear_steps<T, 64>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((k_linear_steps<T, 128>), grid, dim3(256), 0, s, a);
}

}  // namespace qhip

using namespace qhip;

// Whether rows share memory with one f32 a token and head at p.  (Those of one array
// with the rows are seen as columns of it.)
static bool numbers_meet(const qhip_rows* r, int heads, int dim, int tokens, int size, const float* p, long stride) {
  if (!p) return false;
  const qhip_rows n{(void*)p, stride * (4 / size), 0};
  return rows_overlap(r, heads, dim, &n, 1, heads * (4 / size), tokens, size);
}

// 0, hipErrorInvalidValue or QHIP_DECLINE (dimensions without kernels)
static int check_linear(const qhip_linear_batch* b, int type) {
  if (!b || !kv_type_size(type) || b->nseq < 0 || b->nseq > 65535 || b->tokens < 0 || b->tokens > kMaxCount || b->max_new < 0 ||
      b->num_states < 0 || b->k_heads <= 0 || b->v_heads <= 0 || b->v_heads > 65535 || b->v_heads % b->k_heads ||
      b->key_dim <= 0 || b->value_dim <= 0)
    return (int)hipErrorInvalidValue;
  if ((b->key_dim != 64 && b->key_dim != 128) || (b->value_dim != 64 && b->value_dim != 128 && b->value_dim != 256))
    return QHIP_DECLINE;
  return 0;
}

extern "C" long qhip_linear_attention_work_bytes(const qhip_linear_batch* batch, int type, int delta) {
  if (check_linear(batch, type)) return -1;
  return 0;
}

extern "C" int qhip_launch_linear_attention(const qhip_linear_batch* batch, int type, const qhip_rows* q, const qhip_rows* k,
                                            const qhip_rows* v, const float* d_log_decay, long decay_stride,
                                            const float* d_beta, long beta_stride, float scale, float* d_states,
                                            const qhip_rows* out, void* d_work, long work_bytes, void* stream) {
  const int rc = check_linear(batch, type), size = kv_type_size(type);
  if (rc == (int)hipErrorInvalidValue) return rc;
  const int nseq = batch->nseq, tokens = batch->tokens;
  if (nseq > 0 && (!batch->offsets || !batch->slots || ((uintptr_t)batch->offsets & 3u) || ((uintptr_t)batch->slots & 3u) ||
                   ((uintptr_t)batch->source & 3u)))
    return (int)hipErrorInvalidValue;
  if (batch->num_states > 0 && (!d_states || !aligned16(d_states))) return (int)hipErrorInvalidValue;
  if (rc) return rc;
  if (nseq == 0) return 0;
  if (tokens > 0) {
    if (!rows_ok(q, size) || !rows_ok(k, size) || !rows_ok(v, size) || !rows_ok(out, size) || !d_log_decay ||
        ((uintptr_t)d_log_decay & 3u) || decay_stride < 0 || ((uintptr_t)d_beta & 3u) || beta_stride < 0)
      return (int)hipErrorInvalidValue;
    const long state_bytes = 4L * batch->num_states * batch->v_heads * batch->key_dim * batch->value_dim;
    if (!rows_apart(out, tokens, batch->v_heads, batch->value_dim) ||
        rows_meet(out, tokens, batch->v_heads, batch->value_dim, size, d_states, state_bytes))
      return (int)hipErrorInvalidValue;
    const qhip_rows* read[] = {q, k, v};
    const int heads[] = {batch->k_heads, batch->k_heads, batch->v_heads}, dims[] = {batch->key_dim, batch->key_dim, batch->value_dim};
    for (int i = 0; i < 3; ++i)
      if (rows_overlap(out, batch->v_heads, batch->value_dim, read[i], heads[i], dims[i], tokens, size) ||
          rows_meet(read[i], tokens, heads[i], dims[i], size, d_states, state_bytes))
        return (int)hipErrorInvalidValue;
    if (numbers_meet(out, batch->v_heads, batch->value_dim, tokens, size, d_log_decay, decay_stride) ||
        numbers_meet(out, batch->v_heads, batch->value_dim, tokens, size, d_beta, beta_stride))
      return (int)hipErrorInvalidValue;
  }
  LinearArgs a{};
  if (tokens > 0) {
    const qhip_rows* rows[] = {q, k, v, out};
    a.q = q->at;
    a.k = k->at;
    a.v = v->at;
    a.out = out->at;
    long* strides[][2] = {{&a.q_token, &a.q_head}, {&a.k_token, &a.k_head}, {&a.v_token, &a.v_head}, {&a.out_token, &a.out_head}};
    for (int i = 0; i < 4; ++i) {
      *strides[i][0] = rows[i]->token_stride;
      *strides[i][1] = rows[i]->head_stride;
    }
  }
  a.log_decay = d_log_decay;
  a.beta = d_beta;
  a.decay_token = decay_stride;
  a.beta_token = beta_stride;
  a.states = d_states;
  a.offsets = batch->offsets;
  a.slots = batch->slots;
  a.source = batch->source;
  a.nseq = nseq;
  a.tokens = tokens;
  a.max_new = batch->max_new;
  a.num_states = batch->num_states;
  a.k_heads = batch->k_heads;
  a.v_heads = batch->v_heads;
  a.value_dim = batch->value_dim;
  a.group = batch->v_heads / batch->k_heads;
  a.scale = scale;
  hipStream_t st = (hipStream_t)stream;
  if (type == QHIP_TT_F32) launch_steps<float>(a, batch->key_dim, st);
  else if (type == QHIP_TT_F16) launch_steps<f16_t>(a, batch->key_dim, st);
  else launch_steps<bf16_t>(a, batch->key_dim, st);
  return (int)hipGetLastError();
}
