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
__device__ __forceinline__ void split8(const float* x, u32x4* out) {
  float rest[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) rest[i] = x[i];
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
#pragma unroll
      for (int i = 0; i < 8; ++i) rest[i] -= __uint_as_float(__float_as_uint(rest[i]) & 0xFFFF0000u);
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

// What prepare leaves for a chunk and value head: matrix operands, a plane of 16 rows
// in 1 KB (lane l: row l mod 16, columns 4 (l / 16) ..+3 and 16 more), then exp(G),
// exp(G_31 - G) and exp(G_31).
template <typename T, bool DELTA>
struct ChunkWork {
  static constexpr int solve = 0, inside = DELTA ? 2 * 3 * 1024 : 0, numbers = inside + 2 * kSome<T> * 1024,
                       bytes = numbers + 512;
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
  __device__ __forceinline__ void load(const T* row, bool in) {
    const int g = (threadIdx.x & 63) >> 4;
    typedef uint32_t piece __attribute__((ext_vector_type(4), aligned(2)));
    constexpr int W = 16 / sizeof(T);  // elements of a piece
#pragma unroll
    for (int s = 0; s < (int)(sizeof(v) / 16); ++s) {
      v[s] = u32x4{0, 0, 0, 0};
      if (in) v[s] = *(const piece*)(row + (4 * s + g) * W);
    }
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

// A wave takes a chunk of one key head and all of its value heads.
template <typename T, int DK, bool DELTA>
__global__ __launch_bounds__(256) void k_linear_prepare(LinearArgs a) {
  typedef ChunkWork<T, DELTA> W;
  __shared__ __attribute__((aligned(16))) float s_mat[4][32 * kRowPad];
  __shared__ double s_sum[4][32];
  __shared__ __attribute__((aligned(16))) float s_beta[4][32];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, m = lane & 15;
  const int slot = blockIdx.x, kh = blockIdx.y * 4 + wave;
  if (kh >= a.k_heads) return;  // (waves do not wait for each other)
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

  RowTiles<T, DK> k0, k1, q0, q1;
  {
    const T* k = (const T*)a.k + t0 * a.k_token + kh * a.k_head;
    const T* q = (const T*)a.q + t0 * a.q_token + kh * a.q_head;
    k0.load(k + m * a.k_token, m < n);
    k1.load(k + (m + 16) * a.k_token, m + 16 < n);
    q0.load(q + m * a.q_token, m < n);
    q1.load(q + (m + 16) * a.q_token, m + 16 < n);
  }
  // tiles (0, 0), (1, 0), (1, 1): rows 16 i + 4 g + r, column 16 j + m
  f32x4 kk[3], qk[3];
  if constexpr (DELTA) {
    kk[0] = row_product(k0, k0);
    kk[1] = row_product(k1, k0);
    kk[2] = row_product(k1, k1);
  }
  qk[0] = row_product(q0, k0);
  qk[1] = row_product(q1, k0);
  qk[2] = row_product(q1, k1);

  float* mat = s_mat[wave];
  for (int h = kh * a.group; h < (kh + 1) * a.group; ++h) {
    uint8_t* out = a.work + ((long)slot * a.v_heads + h) * W::bytes;
    // G in f64; a decay of exp(-200) is 0 in f32, and sums of -infinity have no differences
    double sum = 0.0;
    float beta = 0.0f;
    if (lane < 32 && lane < n) {
      const float x = a.log_decay[(t0 + lane) * a.decay_token + h];
      sum = x < -200.0f ? -200.0 : (double)x;
      if (DELTA) beta = a.beta[(t0 + lane) * a.beta_token + h];
    }
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const double up = __shfl_up(sum, d, 64);
      if ((lane & 31) >= d) sum += up;
    }
    wave_sync();
    if (lane < 32) {
      s_sum[wave][lane] = sum;
      s_beta[wave][lane] = beta;
    }
    wave_sync();
    const double last = s_sum[wave][31];
    if (lane < 32) {
      float* numbers = (float*)(out + W::numbers);
      numbers[lane] = expf((float)sum);
      numbers[32 + lane] = expf((float)(last - sum));
      if (lane == 0) numbers[64] = expf((float)last);
    }
    f32x4 in[3];
#pragma unroll
    for (int t = 0; t < 3; ++t) {
      const int i0 = t > 0 ? 16 : 0, j = (t == 2 ? 16 : 0) + m;
      const double gj = s_sum[wave][j];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = i0 + 4 * g + r;
        const float d = expf((float)(s_sum[wave][i] - gj));
        in[t][r] = i >= j && i < n ? a.scale * qk[t][r] * d : 0.0f;
        if constexpr (DELTA) mat[i * kRowPad + j] = i > j ? s_beta[wave][i] * kk[t][r] * d : 0.0f;
      }
    }
    wave_sync();
    if constexpr (DELTA) {
      // the two blocks of 16 on the diagonal by substitution, a column a lane
      const int b = (lane & 16), c = m;
      float x[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float y = i == c ? 1.0f : 0.0f;
#pragma unroll
        for (int l = 0; l < i; ++l) y = __builtin_fmaf(-mat[(b + i) * kRowPad + b + l], x[l], y);
        x[i] = i < c ? 0.0f : y;
      }
      // the block below: -X22 L21 X11, on the matrix cores (column 4 g + j of one is row 4 g + j of the other)
      const f32x4 low = *(const f32x4*)(mat + (16 + m) * kRowPad + 4 * g);
      wave_sync();
      if (lane < 32) {
#pragma unroll
        for (int i = 0; i < 16; ++i) mat[(b + i) * kRowPad + b + c] = x[i];
      }
      wave_sync();
      f32x4 p = {0.0f, 0.0f, 0.0f, 0.0f}, y = p;
#pragma unroll
      for (int j = 0; j < 4; ++j) p = __builtin_amdgcn_mfma_f32_16x16x4f32(low[j], mat[(4 * g + j) * kRowPad + m], p, 0, 0, 0);
      const f32x4 diag = *(const f32x4*)(mat + (16 + m) * kRowPad + 16 + 4 * g);
#pragma unroll
      for (int j = 0; j < 4; ++j) y = __builtin_amdgcn_mfma_f32_16x16x4f32(-diag[j], p[j], y, 0, 0, 0);
#pragma unroll
      for (int r = 0; r < 4; ++r) mat[(16 + 4 * g + r) * kRowPad + m] = y[r];
      wave_sync();
    }
    // rows in the order of a matrix operand, split into planes
    auto leave = [&](int at, auto planes, bool with_beta) {
      constexpr int N = decltype(planes)::value;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int j = (e & 4) * 4 + 4 * g + (e & 3);
          v[e] = t == 0 && e >= 4 ? 0.0f : mat[(16 * t + m) * kRowPad + j];
          if (with_beta) v[e] = j <= 16 * t + m ? v[e] * s_beta[wave][j] : 0.0f;
        }
        u32x4 planes_of[N];
        split8<N>(v, planes_of);
#pragma unroll
        for (int q = 0; q < N; ++q) *(u32x4*)(out + at + (t * N + q) * 1024 + lane * 16) = planes_of[q];
      }
    };
    if constexpr (DELTA) {
      leave(W::solve, std::integral_constant<int, 3>{}, true);
      wave_sync();
    }
#pragma unroll
    for (int t = 0; t < 3; ++t) {
      const int i0 = t > 0 ? 16 : 0, j = (t == 2 ? 16 : 0) + m;
#pragma unroll
      for (int r = 0; r < 4; ++r) mat[(i0 + 4 * g + r) * kRowPad + j] = in[t][r];
    }
    wave_sync();
    leave(W::inside, std::integral_constant<int, kSome<T>>{}, false);
  }
}

// A workgroup's four waves have 16 columns each and share the chunk's keys and queries
// in LDS, as matrix operands: rows of 16 tokens (for products with the state), and of
// 16 dimensions (for its update).
template <typename T, int DK>
struct ScanLds {
  static constexpr int P = kPlanes<T>;
  // a plane of 16 rows: 1 KB and a little, so that the stores of a row's pieces and
  // of a column's fall on all banks
  static constexpr int group = 272, tile = 4 * group, across = 1040;
  static constexpr int keys = 0, queries = P * (DK / 16) * tile, turned = 2 * queries, buffer = turned + P * (DK / 16) * across;
};

template <typename T, int DK, bool DELTA>
__global__ __launch_bounds__(256) void k_linear_scan(LinearArgs a) {
  typedef ChunkWork<T, DELTA> W;
  typedef ScanLds<T, DK> L;
  constexpr int P = L::P, TILES = DK / 16, STEPS = DK / 32, SOME = kSome<T>;
  __shared__ __attribute__((aligned(16))) uint8_t lds[2 * L::buffer];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, g = lane >> 4, m = lane & 15;
  const int seq = blockIdx.z, head = blockIdx.y, col = blockIdx.x * 64 + wave * 16 + m;
  const LinearSeq s = linear_seq(a, seq, head, DK);
  if (s.n <= a.few) return;
  const int kh = head / a.group, chunks = (s.n + kChunk - 1) / kChunk;
  const uint8_t* work = a.work + (first_slot(s, seq) * a.v_heads + head) * W::bytes;
  const long work_step = (long)a.v_heads * W::bytes;
  const T* k = (const T*)a.k + s.first * a.k_token + kh * a.k_head;
  const T* q = (const T*)a.q + s.first * a.q_token + kh * a.q_head;
  const T* v = (const T*)a.v + s.first * a.v_token + head * a.v_head + col;
  T* out = (T*)a.out + s.first * a.out_token + head * a.out_head + col;

  // state: tile i has rows 16 i + 4 g + r of the wave's columns
  f32x4 st[TILES];
#pragma unroll
  for (int i = 0; i < TILES; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      st[i][r] = s.from ? s.from[(long)(16 * i + 4 * g + r) * a.value_dim + col] : s.bad ? __builtin_nanf("") : 0.0f;

  // four tokens x four dimensions of keys or queries a thread
  constexpr int BLOCKS = 8 * (DK / 4), EACH = BLOCKS / 128;  // of one of them; of both a thread
  typedef T Four __attribute__((ext_vector_type(4)));
  struct FourRows {
    Four row[4];
  } held[EACH];
  auto block_of = [&](int e, bool& keys, int& tq, int& dq) {
    const int b = EACH == 2 ? tid : tid & 127;
    keys = EACH == 2 ? e == 0 : tid < 128;
    dq = b & (DK / 4 - 1);
    tq = b / (DK / 4);
  };
  auto fetch = [&](int c) {
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      bool keys;
      int tq, dq;
      block_of(e, keys, tq, dq);
      const long stride = keys ? a.k_token : a.q_token;
      const T* from = (keys ? k : q) + 4 * dq;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = c * kChunk + 4 * tq + i;
        typedef T four __attribute__((ext_vector_type(4), aligned(sizeof(T))));
        held[e].row[i] = Four{(T)0.0f, (T)0.0f, (T)0.0f, (T)0.0f};
        if (t < s.n) held[e].row[i] = *(const four*)(from + t * stride);
      }
    }
  };
  auto put = [&](int buffer) {
    uint8_t* to = lds + buffer * L::buffer;
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      bool keys;
      int tq, dq;
      block_of(e, keys, tq, dq);
      float x[4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) x[i][j] = (float)held[e].row[i][j];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        u32x2 planes[P];
        split4<P>(x[i], planes);
        const int t = 4 * tq + i;
#pragma unroll
        for (int p = 0; p < P; ++p)
          *(u32x2*)(to + (keys ? L::keys : L::queries) + ((p * 2 + (t >> 4)) * STEPS + (dq >> 3)) * L::tile + (dq & 3) * L::group +
                    (t & 15) * 16 + ((dq >> 2) & 1) * 8) = planes[p];
      }
      if (keys) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float y[4] = {x[0][j], x[1][j], x[2][j], x[3][j]};
          u32x2 planes[P];
          split4<P>(y, planes);
#pragma unroll
          for (int p = 0; p < P; ++p)
            *(u32x2*)(to + L::turned + (p * TILES + (dq >> 2)) * L::across + (tq & 3) * 256 + (4 * (dq & 3) + j) * 16 + (tq >> 2) * 8) =
                planes[p];
        }
      }
    }
  };
  // a chunk's operands from prepare, and its values: rows 16 t + 4 g + r
  u32x4 solve[2][3], inside[2][SOME];
  f32x4 since[2], left[2];
  float total, val[8];
  auto fetch_work = [&](int c) {
    const uint8_t* w = work + c * work_step;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      if constexpr (DELTA) {
#pragma unroll
        for (int p = 0; p < 3; ++p) solve[t][p] = *(const u32x4*)(w + W::solve + (t * 3 + p) * 1024 + lane * 16);
      }
#pragma unroll
      for (int p = 0; p < SOME; ++p) inside[t][p] = *(const u32x4*)(w + W::inside + (t * SOME + p) * 1024 + lane * 16);
      since[t] = *(const f32x4*)(w + W::numbers + (16 * t + 4 * g) * 4);
      left[t] = *(const f32x4*)(w + W::numbers + (32 + 16 * t + 4 * g) * 4);
    }
    total = *(const float*)(w + W::numbers + 256);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int t = c * kChunk + (e & 4) * 4 + 4 * g + (e & 3);
      val[e] = t < s.n ? (float)v[t * a.v_token] : 0.0f;
    }
  };
  auto operand = [&](int at, u32x4(&x)[P], int plane_bytes) {
#pragma unroll
    for (int p = 0; p < P; ++p) x[p] = *(const u32x4*)(lds + at + p * plane_bytes);
  };

  fetch(0);
  put(0);
  __syncthreads();
  for (int c = 0; c < chunks; ++c) {
    fetch_work(c);
    if (c + 1 < chunks) fetch(c + 1);
    const int base = (c & 1) * L::buffer;
    // Q S and K S
    f32x4 qs[2] = {}, ks[2] = {};
#pragma unroll
    for (int step = 0; step < STEPS; ++step) {
      float x[8];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        x[r] = st[2 * step][r];
        x[4 + r] = st[2 * step + 1][r];
      }
      u32x4 sp[SOME];
      split8<SOME>(x, sp);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int at = base + (t * STEPS + step) * L::tile + g * L::group + m * 16;
        u32x4 x[P];
        if constexpr (DELTA) {
          operand(at + L::keys, x, 2 * STEPS * L::tile);
          ks[t] = mfma_planes<P, SOME>(x, sp, ks[t]);
        }
        operand(at + L::queries, x, 2 * STEPS * L::tile);
        qs[t] = mfma_planes<P, SOME>(x, sp, qs[t]);
      }
    }
    // U
    float u[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) u[e] = DELTA ? val[e] - since[e >> 2][e & 3] * ks[e >> 2][e & 3] : val[e];
    // a value that is not finite spoils its column from its token on; in a product it
    // would spoil the tokens before as well (0 * NaN), so it stays out of them
    int spoilt = kChunk;  // the column's first such token
#pragma unroll
    for (int e = 7; e >= 0; --e)
      if (!(__builtin_fabsf(u[e]) < INFINITY)) spoilt = (e & 4) * 4 + 4 * g + (e & 3);
    const bool any = __ballot(spoilt < kChunk) != 0;
    auto clear = [&]() {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if ((e & 4) * 4 + 4 * g + (e & 3) >= spoilt) u[e] = 0.0f;
    };
    if (any) {
      spoilt = min(spoilt, __shfl_xor(spoilt, 16, 64));
      spoilt = min(spoilt, __shfl_xor(spoilt, 32, 64));
      clear();
    }
    if constexpr (DELTA) {
      u32x4 planes[3];
      split8<3>(u, planes);
      const f32x4 none = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const f32x4 y = mfma_planes<3, 3>(solve[t], planes, none);
#pragma unroll
        for (int r = 0; r < 4; ++r) u[4 * t + r] = y[r];
      }
      if (any) clear();
    }
    // the state, then the outputs
    float w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = left[e >> 2][e & 3] * u[e];
    u32x4 planes[3];
    split8<3>(w, planes);
#pragma unroll
    for (int i = 0; i < TILES; ++i) {
      u32x4 x[P];
      operand(base + L::turned + i * L::across + lane * 16, x, TILES * L::across);
      st[i] = mfma_planes<P, 3>(x, planes, st[i] * total);
    }
    if (any && spoilt < kChunk) {
#pragma unroll
      for (int i = 0; i < TILES; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) st[i][r] = __builtin_nanf("");
    }
    split8<SOME>(u, planes);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      f32x4 o;
#pragma unroll
      for (int r = 0; r < 4; ++r) o[r] = a.scale * since[t][r] * qs[t][r];
      o = mfma_planes<SOME, SOME>(inside[t], planes, o);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = 16 * t + 4 * g + r, at = c * kChunk + i;
        if (any && i >= spoilt) o[r] = __builtin_nanf("");
        if (at < s.n) out[at * a.out_token] = (T)o[r];
      }
    }
    if (c + 1 < chunks) put((c + 1) & 1);
    __syncthreads();
  }
  if (s.to) {
#pragma unroll
    for (int i = 0; i < TILES; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) s.to[(long)(16 * i + 4 * g + r) * a.value_dim + col] = st[i][r];
  }
}

template <typename T, int DK, bool DELTA>
static void launch_chunks(const LinearArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((k_linear_prepare<T, DK, DELTA>), dim3((unsigned)(a.tokens / kChunk + a.nseq), (unsigned)((a.k_heads + 3) / 4)),
                     dim3(256), 0, s, a);
  hipLaunchKernelGGL((k_linear_scan<T, DK, DELTA>), dim3((unsigned)(a.value_dim / 64), (unsigned)a.v_heads, (unsigned)a.nseq),
                     dim3(256), 0, s, a);
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
