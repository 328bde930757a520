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

#include <type_traits>

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
  int few;        // sequences of more tokens go in chunks
  uint8_t* work;  // of the chunks
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

// Sequences of at most this many new tokens go token by token.
constexpr int kFew = 12;

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
  if (s.n > a.few || (s.n == 0 && s.from == s.to)) return;
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

// ---- chunks of 32 tokens ---------------------------------------------------------------
//
// Inside a chunk with G_i = log_decay_0 + .. + log_decay_i, S the state before it and
// D_ij = exp(G_i - G_j):
//
//   L_ij = beta_i (k_i . k_j) D_ij  (j < i),   T = (1 + L)^-1 diag(beta)
//   A_ij = scale (q_i . k_j) D_ij   (j <= i)
//   U = T (V - diag(exp(G)) K S)    (U = V without the delta rule)
//   O = scale diag(exp(G)) Q S + A U
//   S <- exp(G_31) S + (diag(exp(G_31 - G)) K)^T U
//
// k_linear_prepare makes T, A and the exponentials of every chunk side by side;
// k_linear_scan then walks a sequence's chunks with 16 columns of a state in a wave's
// registers.  All differences G_i - G_j are taken in f64: G is a long sum where the
// decay between near tokens is small.
//
// Products run on bf16 matrix tiles.  An f32 value goes in as a sum of planes of 8
// bits: three hold it whole, and of their products those up to 2^-16 are summed, so a
// product is good to f32; 16-bit inputs need one plane (bf16) or two (f16).
constexpr int kChunk = 32;

typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <typename T>
constexpr int kPlanes = sizeof(T) == 4 ? 3 : 1;  // that hold an element whole
template <>
constexpr int kPlanes<f16_t> = 2;
template <typename T>
constexpr int kSome = sizeof(T) == 4 ? 3 : 2;  // of states read, weights inside a chunk

// N planes of eight values (the last of two rounds to nearest, else bits are cut off:
// no plane overflows)
template <int N>
__device__ __forceinline__ void split8(f32x4 x, f32x4 y, u32x4* out) {
  float rest[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    rest[i] = x[i];
    rest[4 + i] = y[i];
  }
#pragma unroll
  for (int p = 0; p < N; ++p) {
    if (p == N - 1 && N < 3) {
      b16x8 b;
#pragma unroll
      for (int i = 0; i < 8; ++i) b[i] = (__bf16)rest[i];
      out[p] = __builtin_bit_cast(u32x4, b);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        out[p][i] = __builtin_amdgcn_perm(__float_as_uint(rest[2 * i + 1]), __float_as_uint(rest[2 * i]), 0x07060302u);
      if (p + 1 < N) {
#pragma unroll
        for (int i = 0; i < 8; ++i) rest[i] -= __uint_as_float(__float_as_uint(rest[i]) & 0xFFFF0000u);
      }
    }
  }
}
// the same of four values, two dwords a plane
template <int N>
__device__ __forceinline__ void split4(const float* x, u32x2* out) {
  float rest[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) rest[i] = x[i];
#pragma unroll
  for (int p = 0; p < N; ++p) {
    out[p] = u32x2{__builtin_amdgcn_perm(__float_as_uint(rest[1]), __float_as_uint(rest[0]), 0x07060302u),
                   __builtin_amdgcn_perm(__float_as_uint(rest[3]), __float_as_uint(rest[2]), 0x07060302u)};
#pragma unroll
    for (int i = 0; i < 4; ++i) rest[i] -= __uint_as_float(__float_as_uint(rest[i]) & 0xFFFF0000u);
  }
}

__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b16x8, a), __builtin_bit_cast(b16x8, b), c, 0, 0, 0);
}
// the product of planes, smallest terms first
template <int NA, int NB>
__device__ __forceinline__ f32x4 mfma_planes(const u32x4* a, const u32x4* b, f32x4 c) {
#pragma unroll
  for (int sum = 2; sum >= 0; --sum)
#pragma unroll
    for (int i = 0; i <= sum; ++i)
      if (i < NA && sum - i < NB) c = mfma(a[i], b[sum - i], c);
  return c;
}

// What prepare leaves for a chunk and value head, as matrix operands (lane l: row l mod
// 16, columns 4 (l / 16) ..+3): T's tiles (0, 0), (1, 0) and (1, 1) in f32; A's the
// same way for f32 rows, else its two rows of tiles in two planes; then exp(G),
// exp(G_31 - G) and exp(G_31).
template <typename T, bool DELTA>
struct ChunkWork {
  static constexpr bool whole = sizeof(T) == 4;
  static constexpr int solve = 0, inside = DELTA ? 3 * 1024 : 0, numbers = inside + (whole ? 3 : 4) * 1024, bytes = numbers + 512;
};

// The chunk slot of a sequence's first: no two sequences' slots meet, and there are at
// most tokens / 32 + nseq.
__device__ __forceinline__ long first_slot(const LinearSeq& s, int i) { return s.first / kChunk + i; }

// (LDS between the lanes of a wave: in order in the hardware, kept in order here)
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Sixteen rows of DK elements, a row to the lanes of equal l mod 16: either operand of
// row_product, which gives the 16 x 16 products of two of them.
template <typename T, int DK>
struct RowTiles {
  u32x4 v[sizeof(T) == 4 ? DK / 16 : DK / 32];
  __device__ __forceinline__ void load(const T* row, bool in) {  // (the row of !in is there, but not this chunk's)
    const int g = (threadIdx.x & 63) >> 4;
    typedef uint32_t piece __attribute__((ext_vector_type(4), aligned(2)));
    constexpr int W = 16 / sizeof(T);  // elements of a piece
#pragma unroll
    for (int s = 0; s < (int)(sizeof(v) / 16); ++s) {
      v[s] = *(const piece*)(row + (4 * s + g) * W);
    }
#pragma unroll
    for (int s = 0; s < (int)(sizeof(v) / 16); ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i) v[s][i] = in ? v[s][i] : 0u;
  }
};
template <typename T, int DK>
__device__ __forceinline__ f32x4 row_product(const RowTiles<T, DK>& a, const RowTiles<T, DK>& b) {
  f32x4 c = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int s = 0; s < (int)(sizeof(a.v) / 16); ++s) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.v[s][j]), __uint_as_float(b.v[s][j]), c, 0, 0, 0);
    } else if constexpr (std::is_same<T, f16_t>::value) {
      c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h16x8, a.v[s]), __builtin_bit_cast(h16x8, b.v[s]), c, 0, 0, 0);
    } else {
      c = mfma(a.v[s], b.v[s], c);
    }
  }
  return c;
}

constexpr int kRowPad = 36;  // floats of a row of a 32 x 32 matrix in LDS

__device__ __forceinline__ f32x4 mfma4(f32x4 a, f32x4 b, f32x4 c) {  // 16 columns of a against 16 rows of b
#pragma unroll
  for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
  return c;
}

// A wave takes a chunk of two value heads, a half of its lanes for each where the work
// goes by tokens or columns.
template <typename T, int DK, bool DELTA>
__global__ __launch_bounds__(256) void k_linear_prepare(LinearArgs a) {
  typedef ChunkWork<T, DELTA> W;
  __shared__ __attribute__((aligned(16))) float s_mat[4][2][32 * kRowPad];
  __shared__ double s_sum[4][2][32];
  __shared__ __attribute__((aligned(16))) float s_beta[4][2][32];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, m = lane & 15, half = lane >> 5, token = lane & 31;
  const int slot = blockIdx.x, head0 = __builtin_amdgcn_readfirstlane((blockIdx.y * 4 + wave) * 2);
  if (head0 >= a.v_heads) return;  // (waves do not wait for each other)
  const int heads = min(2, a.v_heads - head0);
  // the slot's sequence: the last whose first slot is not behind it
  int seq = -1;
  for (int i0 = 0; i0 < a.nseq; i0 += 64) {
    const int i = i0 + lane;
    const uint64_t before = __ballot(i < a.nseq && a.offsets[min(i, a.nseq - 1)] / kChunk + i <= slot);
    seq += __builtin_popcountll(before);
    if (before != ~0ull) break;
  }
  if (seq < 0) return;
  LinearSeq s{a.offsets[seq], 0, nullptr, nullptr, false};
  const int end = min(a.offsets[seq + 1], a.tokens);
  if (s.first >= 0 && end > s.first) s.n = min(end - s.first, a.max_new);
  const int chunk = (int)(slot - first_slot(s, seq)), n = s.n - chunk * kChunk;  // tokens from the chunk's first on
  if (chunk < 0 || n <= 0 || s.n <= a.few) return;
  const long t0 = s.first + (long)chunk * kChunk;

  // G (times log2 e) in f64; a decay of exp(-200) is 0 in f32, and sums of -infinity
  // have no differences
  uint8_t* out = a.work + ((long)slot * a.v_heads + head0) * W::bytes;
  {
    const int h = head0 + min(half, heads - 1);
    const long t = t0 + min(token, n - 1);
    const float x = a.log_decay[t * a.decay_token + h];
    const float beta = DELTA ? a.beta[t * a.beta_token + h] : 0.0f;
    double sum = token < n ? (x < -200.0f ? -200.0 : (double)x) * 1.4426950408889634 : 0.0;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const double up = __shfl_up(sum, d, 64);
      if (token >= d) sum += up;
    }
    s_sum[wave][half][token] = sum;
    s_beta[wave][half][token] = token < n ? beta : 0.0f;
    wave_sync();
    const double last = s_sum[wave][half][31];
    if (half < heads) {
      float* numbers = (float*)(out + half * W::bytes + W::numbers);
      numbers[token] = __builtin_amdgcn_exp2f((float)sum);
      numbers[32 + token] = __builtin_amdgcn_exp2f((float)(last - sum));
      if (token == 0) numbers[64] = __builtin_amdgcn_exp2f((float)last);
    }
  }

  // tiles (0, 0), (1, 0), (1, 1): rows 16 i + 4 g + r, column 16 j + m
  f32x4 kk[3], qk[3], in[2][3];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    if (x >= heads) break;
    const int kh = (head0 + x) / a.group;
    if (x == 0 || kh != (head0 + x - 1) / a.group) {
      RowTiles<T, DK> k0, k1, q0, q1;
      const T* k = (const T*)a.k + t0 * a.k_token + kh * a.k_head;
      const T* q = (const T*)a.q + t0 * a.q_token + kh * a.q_head;
      k0.load(k + min(m, n - 1) * a.k_token, m < n);
      k1.load(k + min(m + 16, n - 1) * a.k_token, m + 16 < n);
      q0.load(q + min(m, n - 1) * a.q_token, m < n);
      q1.load(q + min(m + 16, n - 1) * a.q_token, m + 16 < n);
      if constexpr (DELTA) {
        kk[0] = row_product(k0, k0);
        kk[1] = row_product(k1, k0);
        kk[2] = row_product(k1, k1);
      }
      qk[0] = row_product(q0, k0);
      qk[1] = row_product(q1, k0);
      qk[2] = row_product(q1, k1);
    }
    float* mat = s_mat[wave][x];
#pragma unroll
    for (int t = 0; t < 3; ++t) {
      const int i0 = t > 0 ? 16 : 0, j = (t == 2 ? 16 : 0) + m;
      const double gj = s_sum[wave][x][j];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = i0 + 4 * g + r;
        const float d = __builtin_amdgcn_exp2f((float)(s_sum[wave][x][i] - gj));
        in[x][t][r] = i >= j && i < n ? a.scale * qk[t][r] * d : 0.0f;
        if constexpr (DELTA) mat[i * kRowPad + j] = i > j ? s_beta[wave][x][i] * kk[t][r] * d : 0.0f;
      }
    }
  }
  wave_sync();
  if constexpr (DELTA) {
    // (1 + L)^-1: the two blocks of 16 on the diagonal by substitution, a column a lane
    {
      float* mat = s_mat[wave][half];
      const int b = lane & 16;
      float x[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float y = i == m ? 1.0f : 0.0f;
#pragma unroll
        for (int l = 0; l < i; ++l) y = __builtin_fmaf(-mat[(b + i) * kRowPad + b + l], x[l], y);
        x[i] = i < m ? 0.0f : y;
      }
      wave_sync();
      if (half < heads) {
#pragma unroll
        for (int i = 0; i < 16; ++i) mat[(b + i) * kRowPad + b + m] = x[i];
      }
      wave_sync();
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      if (x >= heads) break;
      // the block below them: -X22 L21 X11 (a result's rows 4 g + r are an operand's)
      float* mat = s_mat[wave][x];
      const float* row = mat + m * kRowPad + 4 * g;
      f32x4 top, low = *(const f32x4*)(row + 16 * kRowPad), diag = *(const f32x4*)(row + 16 * kRowPad + 16);
#pragma unroll
      for (int j = 0; j < 4; ++j) top[j] = mat[(4 * g + j) * kRowPad + m];
      const f32x4 none = {0.0f, 0.0f, 0.0f, 0.0f};
      const f32x4 y = mfma4(-diag, mfma4(low, top, none), none);
      wave_sync();
#pragma unroll
      for (int r = 0; r < 4; ++r) mat[(16 + 4 * g + r) * kRowPad + m] = y[r];
      wave_sync();
      // T = X diag(beta)
      const f32x4 b0 = *(const f32x4*)(s_beta[wave][x] + 4 * g), b1 = *(const f32x4*)(s_beta[wave][x] + 16 + 4 * g);
      f32x4 t00 = *(const f32x4*)row, t10 = *(const f32x4*)(row + 16 * kRowPad) * b0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {  // (nothing above the diagonal, whatever beta holds)
        t00[j] = 4 * g + j <= m ? t00[j] * b0[j] : 0.0f;
        diag[j] = 4 * g + j <= m ? diag[j] * b1[j] : 0.0f;
      }
      f32x4* to = (f32x4*)(out + x * W::bytes + W::solve) + lane;
      to[0] = t00;
      to[64] = t10;
      to[128] = diag;
    }
    wave_sync();
  }
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    if (x >= heads) break;
    float* mat = s_mat[wave][x];
#pragma unroll
    for (int t = 0; t < 3; ++t) {
      const int i0 = t > 0 ? 16 : 0, j = (t == 2 ? 16 : 0) + m;
#pragma unroll
      for (int r = 0; r < 4; ++r) mat[(i0 + 4 * g + r) * kRowPad + j] = in[x][t][r];
    }
  }
  wave_sync();
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    if (x >= heads) break;
    const float* row = s_mat[wave][x] + m * kRowPad + 4 * g;
    const f32x4 none = {0.0f, 0.0f, 0.0f, 0.0f};
    const f32x4 t00 = *(const f32x4*)row, t10 = *(const f32x4*)(row + 16 * kRowPad), t11 = *(const f32x4*)(row + 16 * kRowPad + 16);
    u32x4* to = (u32x4*)(out + x * W::bytes + W::inside) + lane;
    if constexpr (W::whole) {
      to[0] = __builtin_bit_cast(u32x4, t00);
      to[64] = __builtin_bit_cast(u32x4, t10);
      to[128] = __builtin_bit_cast(u32x4, t11);
    } else {
      u32x4 planes[2];
      split8<2>(t00, none, planes);
      to[0] = planes[0];
      to[64] = planes[1];
      split8<2>(t10, t11, planes);
      to[128] = planes[0];
      to[192] = planes[1];
    }
  }
}

// DK / 32 waves have the same 16 columns, 32 rows of the state each: they share the
// products with the state out between them, hand their parts round in LDS (one
// barrier a chunk), and go on with the sums by themselves.
template <typename T, int DK, bool DELTA>
__global__ __launch_bounds__(256) void k_linear_scan(LinearArgs a) {
  typedef ChunkWork<T, DELTA> W;
  constexpr bool F32 = sizeof(T) == 4;       // f32 rows: f32 products throughout
  constexpr int P = F32 ? 1 : kPlanes<T>;    // planes of keys and queries
  constexpr int PARTS = DK / 32, SETS = 4 / PARTS, COLS = 16 * SETS;
  // the keys of a chunk, turned: operands of 16 dimensions and 32 tokens.  A tile is 1 KB
  // (f32: two, of 16 tokens) and 16 bytes, so that a thread's stores fall on all banks.
  constexpr int TURNED = F32 ? 2 * 1024 + 16 : 1024 + 16, KEYS = P * (DK / 16) * TURNED;
  __shared__ __attribute__((aligned(16))) uint8_t s_keys[2 * KEYS];
  __shared__ f32x4 s_part[2][SETS][4][PARTS][64];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, g = lane >> 4, m = lane & 15;
  const int set = wave / PARTS, part = wave % PARTS;
  // the workgroups of a sequence's head follow each other on one XCD
  const int blocks = a.value_dim / COLS, id = (int)blockIdx.x;
  const int pair = id / (8 * blocks) * 8 + (id & 7), seq = pair / a.v_heads, head = pair - seq * a.v_heads;
  if (seq >= a.nseq) return;
  const int col = (id >> 3) % blocks * COLS + set * 16 + m;
  const LinearSeq s = linear_seq(a, seq, head, DK);
  if (s.n <= a.few) return;
  const int kh = head / a.group, chunks = (s.n + kChunk - 1) / kChunk, tail = s.n - (chunks - 1) * kChunk;

  // state: tile i has rows 16 i + 4 g + r of the wave's 32, and the wave's columns
  f32x4 st[2];
  const long state_at = (long)(32 * part + 4 * g) * a.value_dim + col;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      st[i][r] = s.from ? s.from[state_at + (16 * i + r) * a.value_dim] : s.bad ? __builtin_nanf("") : 0.0f;

  // Everything of a chunk is loaded for the next one when the present one is done with
  // it, without branches: uniform bases that go on by 32 tokens, offsets of 32 bits, and
  // the last token's in the place of those behind it.
  const char* k_at = (const char*)((const T*)a.k + s.first * a.k_token + kh * a.k_head);
  const char* q_at = (const char*)((const T*)a.q + s.first * a.q_token + kh * a.q_head);
  const char* v_at = (const char*)((const T*)a.v + s.first * a.v_token + head * a.v_head);
  char* out_at = (char*)((T*)a.out + s.first * a.out_token + head * a.out_head);
  // (global memory by name: through a flat address, a load would count as one of LDS too)
  typedef const __attribute__((address_space(1))) uint8_t* Work;
  Work work = (Work)a.work + (first_slot(s, seq) * a.v_heads + head) * W::bytes;
  const long k_step = kChunk * a.k_token * (long)sizeof(T), q_step = kChunk * a.q_token * (long)sizeof(T),
             v_step = kChunk * a.v_token * (long)sizeof(T), out_step = kChunk * a.out_token * (long)sizeof(T),
             work_step = (long)a.v_heads * W::bytes;

  typedef typename std::conditional<F32, u32x4, u32x2>::type Four;  // elements
  typedef typename std::conditional<F32, uint32_t, uint16_t>::type Word;
  typedef uint32_t four __attribute__((ext_vector_type(sizeof(Four) / 4), aligned(sizeof(Word))));
  // rows 16 t + m: dimensions 4 g ..+3 of the wave's 32 and 16 more
  Four kr[2][2], qr[2][2];
  // four tokens x four dimensions a thread, to be turned (DK = 64: every second wave)
  const int dq = tid & (DK / 4 - 1), tq = tid / (DK / 4) & 7;
  const bool turns = tid < 2 * DK;
  Four held[4];
  T val[8];
  uint32_t k_off[2], q_off[2], held_off[4], v_off[8];
  auto place = [&](int rows) {  // of a chunk with that many tokens
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      k_off[t] = (uint32_t)(min(16 * t + m, rows - 1) * (int)a.k_token + 32 * part + 4 * g) * (uint32_t)sizeof(T);
      q_off[t] = (uint32_t)(min(16 * t + m, rows - 1) * (int)a.q_token + 32 * part + 4 * g) * (uint32_t)sizeof(T);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) held_off[i] = (uint32_t)(min(4 * tq + i, rows - 1) * (int)a.k_token + 4 * dq) * (uint32_t)sizeof(T);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      v_off[e] = (uint32_t)(min((e & 4) * 4 + 4 * g + (e & 3), rows - 1) * (int)a.v_token + col) * (uint32_t)sizeof(T);
  };
  auto fetch_rows = [&](const char* k, const char* q) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (DELTA) kr[t][h] = *(const four*)(k + k_off[t] + 16 * h * sizeof(T));
        qr[t][h] = *(const four*)(q + q_off[t] + 16 * h * sizeof(T));
      }
  };
  auto fetch_held = [&](const char* k) {
#pragma unroll
    for (int i = 0; i < 4; ++i) held[i] = *(const four*)(k + held_off[i]);
  };
  auto fetch_values = [&](const char* v) {
#pragma unroll
    for (int e = 0; e < 8; ++e) val[e] = *(const T*)(v + v_off[e]);
  };
  typedef const __attribute__((address_space(1))) f32x4* GlobalF4;
  f32x4 solve[3], since[2], left[2];
  f32x4 inside[3];  // f32 rows: the three tiles; else two planes of the wave's output tile
  float total;
  const int out_tile = part & 1;  // of the chunk's two, and of its rows 4 g + r those from out_row on
  constexpr int OUT_ROWS = PARTS == 4 ? 2 : 4;
  const int out_row = PARTS == 4 ? part & 2 : 0;
  auto fetch_solve = [&](Work w) {
    if constexpr (DELTA) {
#pragma unroll
      for (int i = 0; i < 3; ++i) solve[i] = *(GlobalF4)(w + W::solve + i * 1024 + lane * 16);
#pragma unroll
      for (int t = 0; t < 2; ++t) since[t] = *(GlobalF4)(w + W::numbers + (16 * t + 4 * g) * 4);
    }
  };
  auto fetch_left = [&](Work w) {
#pragma unroll
    for (int t = 0; t < 2; ++t) left[t] = *(GlobalF4)(w + W::numbers + (32 + 16 * t + 4 * g) * 4);
    total = *(const __attribute__((address_space(1))) float*)(w + W::numbers + 256);
  };
  f32x4 out_since;
  auto fetch_inside = [&](Work w) {
#pragma unroll
    for (int i = 0; i < (F32 ? 3 : 2); ++i) inside[i] = *(GlobalF4)(w + W::inside + (F32 ? i : 2 * out_tile + i) * 1024 + lane * 16);
    out_since = *(GlobalF4)(w + W::numbers + (16 * out_tile + 4 * g) * 4);
  };
  // the held keys into LDS, turned; `rows` of the chunk are there
  uint8_t* const to_turned = s_keys + (dq >> 2) * TURNED + (dq & 3) * 64 +
                             (F32 ? (tq >> 2) * 1024 + (tq & 3) * 256 : (tq & 3) * 256 + (tq >> 2) * 8);
  auto turn = [&](int buffer, int rows) {
    if (rows < kChunk) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < (int)(sizeof(Four) / 4); ++j) held[i][j] = 4 * tq + i < rows ? held[i][j] : 0u;
    }
    if constexpr (F32) {
#pragma unroll
      for (int j = 0; j < 4; ++j) *(u32x4*)(to_turned + buffer + j * 16) = u32x4{held[0][j], held[1][j], held[2][j], held[3][j]};
    } else {
      u32x2 planes[4][P];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (P == 1) {
          planes[i][0] = held[i];
        } else {
          typedef T Four_t __attribute__((ext_vector_type(4)));
          const Four_t x = __builtin_bit_cast(Four_t, held[i]);
          const float y[4] = {(float)x[0], (float)x[1], (float)x[2], (float)x[3]};
          split4<P>(y, planes[i]);
        }
      }
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t pick = j & 1 ? 0x07060302u : 0x05040100u;
          *(u32x2*)(to_turned + buffer + p * (DK / 16) * TURNED + j * 16) =
              u32x2{__builtin_amdgcn_perm(planes[1][p][j >> 1], planes[0][p][j >> 1], pick),
                    __builtin_amdgcn_perm(planes[3][p][j >> 1], planes[2][p][j >> 1], pick)};
        }
    }
  };
  // a part of 16 rows' product with the state
  u32x4 sp[2];
  auto with_state = [&](const Four(&row)[2]) {
    f32x4 c = {0.0f, 0.0f, 0.0f, 0.0f};
    if constexpr (F32) {
      c = mfma4(__builtin_bit_cast(f32x4, row[0]), st[0], c);
      return mfma4(__builtin_bit_cast(f32x4, row[1]), st[1], c);
    } else if constexpr (P == 1) {
      const u32x4 x[1] = {u32x4{row[0][0], row[0][1], row[1][0], row[1][1]}};
      return mfma_planes<1, 2>(x, sp, c);
    } else {
      typedef T Four_t __attribute__((ext_vector_type(4)));
      f32x4 y[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const Four_t z = __builtin_bit_cast(Four_t, row[h]);
        y[h] = f32x4{(float)z[0], (float)z[1], (float)z[2], (float)z[3]};
      }
      u32x4 x[P];
      split8<P>(y[0], y[1], x);
      return mfma_planes<P, 2>(x, sp, c);
    }
  };

  place(chunks > 1 ? kChunk : tail);
  fetch_rows(k_at, q_at);
  fetch_held(k_at);
  fetch_values(v_at);
  fetch_solve(work);
  fetch_left(work);
  fetch_inside(work);
  for (int c = 0; c < chunks; ++c) {
    const bool more = c + 1 < chunks;
    const int rows = more ? kChunk : tail, buffer = (c & 1) * KEYS;
    if (more) {
      work += work_step;
      v_at += v_step;
      k_at += k_step;
      q_at += q_step;
      if (c + 2 == chunks && tail < kChunk) place(tail);
    }
    // this wave's part of K S and Q S
    if constexpr (!F32) split8<2>(st[0], st[1], sp);
    f32x4(*parts)[PARTS][64] = s_part[c & 1][set];
    if (turns) turn(buffer, rows);
    fetch_held(k_at);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      if (DELTA) parts[t][part][lane] = with_state(kr[t]);
      parts[2 + t][part][lane] = with_state(qr[t]);
    }
    fetch_rows(k_at, q_at);
    __syncthreads();  // (the buffers after next are written behind the next chunk's barrier)
    // what U is made of, then U
    f32x4 u[2];
    float sum = 0.0f;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int r = 0; r < 4; ++r) u[t][r] = (float)val[4 * t + r];
      if (rows < kChunk) {
#pragma unroll
        for (int r = 0; r < 4; ++r) u[t][r] = 16 * t + 4 * g + r < rows ? u[t][r] : 0.0f;
      }
      if constexpr (DELTA) {
        f32x4 ks = parts[t][0][lane];
#pragma unroll
        for (int i = 1; i < PARTS; ++i) ks += parts[t][i][lane];
        // (rows behind the sequence's end have the last row's keys: their T is 0)
        u[t] -= since[t] * ks;
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) sum = __builtin_fmaf(u[t][r], 0.0f, sum);
    }
    fetch_values(v_at);
    // a value that is not finite spoils its column from its token on; in a product it
    // would spoil the tokens before as well (0 * NaN), so it stays out of them
    const bool any = __ballot(sum != 0.0f) != 0;
    int spoilt = kChunk;  // the column's first such token
    auto clear = [&]() {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if ((e & 4) * 4 + 4 * g + (e & 3) >= spoilt) u[e >> 2][e & 3] = 0.0f;
    };
    if (any) {
#pragma unroll
      for (int e = 7; e >= 0; --e)
        if (!(__builtin_fabsf(u[e >> 2][e & 3]) < INFINITY)) spoilt = (e & 4) * 4 + 4 * g + (e & 3);
      spoilt = min(spoilt, __shfl_xor(spoilt, 16, 64));
      spoilt = min(spoilt, __shfl_xor(spoilt, 32, 64));
      clear();
    }
    const f32x4 none = {0.0f, 0.0f, 0.0f, 0.0f};
    if constexpr (DELTA) {
      f32x4 y0 = none, y1 = none;
#pragma unroll
      for (int j = 0; j < 4; ++j) {  // (side by side: each waits for the one before it)
        y1 = __builtin_amdgcn_mfma_f32_16x16x4f32(solve[1][j], u[0][j], y1, 0, 0, 0);
        y0 = __builtin_amdgcn_mfma_f32_16x16x4f32(solve[0][j], u[0][j], y0, 0, 0, 0);
      }
      u[1] = mfma4(solve[2], u[1], y1);
      u[0] = y0;
      fetch_solve(work);
      if (any) clear();
    }
    // the state
    const uint8_t* turned = s_keys + buffer + 2 * part * TURNED + lane * 16;
    if constexpr (F32) {
      const f32x4 w0 = left[0] * u[0], w1 = left[1] * u[1];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        st[i] = mfma4(*(const f32x4*)(turned + i * TURNED), w0, st[i] * total);
        st[i] = mfma4(*(const f32x4*)(turned + i * TURNED + 1024), w1, st[i]);
      }
    } else {
      u32x4 planes[3];
      split8<3>(left[0] * u[0], left[1] * u[1], planes);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        u32x4 x[P];
#pragma unroll
        for (int p = 0; p < P; ++p) x[p] = *(const u32x4*)(turned + (p * (DK / 16) + i) * TURNED);
        st[i] = mfma_planes<P, 3>(x, planes, st[i] * total);
      }
    }
    fetch_left(work);
    if (any && spoilt < kChunk) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) st[i][r] = __builtin_nanf("");
    }
    // the wave's rows of the output
    f32x4 o = parts[2 + out_tile][0][lane];
#pragma unroll
    for (int i = 1; i < PARTS; ++i) o += parts[2 + out_tile][i][lane];
    o *= a.scale * out_since;
    if constexpr (F32) {
      o = mfma4(out_tile ? inside[1] : inside[0], u[0], o);
      if (out_tile) o = mfma4(inside[2], u[1], o);
    } else {
      u32x4 planes[2];
      split8<2>(u[0], u[1], planes);
      const u32x4 x[2] = {__builtin_bit_cast(u32x4, inside[0]), __builtin_bit_cast(u32x4, inside[1])};
      o = mfma_planes<2, 2>(x, planes, o);
    }
    fetch_inside(work);
    float left_rows[OUT_ROWS];
#pragma unroll
    for (int r = 0; r < OUT_ROWS; ++r) {
      left_rows[r] = PARTS == 4 && out_row ? o[2 + (r & 1)] : o[r];
      if (any && 16 * out_tile + 4 * g + out_row + r >= spoilt) left_rows[r] = __builtin_nanf("");
    }
    const int out0 = 16 * out_tile + 4 * g + out_row;
#pragma unroll
    for (int r = 0; r < OUT_ROWS; ++r)
      if (rows == kChunk || out0 + r < rows)
        *(T*)(out_at + (uint32_t)((out0 + r) * (int)a.out_token + col) * (uint32_t)sizeof(T)) = (T)left_rows[r];
    out_at += out_step;
  }
  if (s.to) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) s.to[state_at + (16 * i + r) * a.value_dim] = st[i][r];
  }
}

template <typename T, int DK, bool DELTA>
static void launch_chunks(const LinearArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((k_linear_prepare<T, DK, DELTA>), dim3((unsigned)(a.tokens / kChunk + a.nseq), (unsigned)((a.v_heads + 7) / 8)),
                     dim3(256), 0, s, a);
  const long pairs = ((long)a.nseq * a.v_heads + 7) / 8 * 8;
  hipLaunchKernelGGL((k_linear_scan<T, DK, DELTA>), dim3((unsigned)(pairs * (a.value_dim / (2048 / DK)))), dim3(256), 0, s, a);
}

template <typename T>
static void launch_linear(const LinearArgs& a, int key_dim, bool steps, bool chunks, hipStream_t s) {
  if (steps) launch_steps<T>(a, key_dim, s);
  if (!chunks) return;
  if (key_dim == 64) a.beta ? launch_chunks<T, 64, true>(a, s) : launch_chunks<T, 64, false>(a, s);
  else a.beta ? launch_chunks<T, 128, true>(a, s) : launch_chunks<T, 128, false>(a, s);
}

static long chunk_bytes(int type, bool delta) {
  if (type == QHIP_TT_F32) return delta ? ChunkWork<float, true>::bytes : ChunkWork<float, false>::bytes;
  return delta ? ChunkWork<f16_t, true>::bytes : ChunkWork<f16_t, false>::bytes;
}
static long linear_work(const qhip_linear_batch* b, int type, bool delta) {
  if (b->max_new <= kFew || b->nseq == 0 || b->tokens == 0) return 0;
  return ((long)b->tokens / kChunk + b->nseq) * b->v_heads * chunk_bytes(type, delta);
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
  return linear_work(batch, type, delta != 0);
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
    const qhip_rows* all[] = {q, k, v, out};
    for (const qhip_rows* r : all)  // (a chunk's offsets are 32 bits)
      if (!rows_ok(r, size) || r->token_stride > 1 << 23) return (int)hipErrorInvalidValue;
    if (!d_log_decay ||
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
  // without a workspace every sequence goes token by token; where all have more than
  // a few tokens the other kernel has nothing to do
  const long need = linear_work(batch, type, d_beta != nullptr);
  const bool chunks = need > 0 && d_work;
  if (chunks && (work_bytes < need || !aligned16(d_work))) return (int)hipErrorInvalidValue;
  const bool steps = !chunks || (long)nseq * batch->max_new != tokens;
  a.few = chunks ? kFew : 0x7FFFFFFF;
  a.work = (uint8_t*)d_work;
  hipStream_t st = (hipStream_t)stream;
  if (type == QHIP_TT_F32) launch_linear<float>(a, batch->key_dim, steps, chunks, st);
  else if (type == QHIP_TT_F16) launch_linear<f16_t>(a, batch->key_dim, steps, chunks, st);
  else launch_linear<bf16_t>(a, batch->key_dim, steps, chunks, st);
  return (int)hipGetLastError();
}
