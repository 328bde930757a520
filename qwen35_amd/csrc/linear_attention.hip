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

// Beside sequences that go in chunks, those of at most this many new tokens go token by
// token: a chunk takes one sequence of 16 heads 13 (bf16) to 18 us (f32), a token 0.8.
constexpr int kFew = 16;
// A batch whose sequences all have at most this many does without chunks.  Of sequences
// that fill the card (256 workgroups of 64 columns) a chunk costs more tokens.  16 heads of
// 128 x 128, us token by token / in chunks of f32 / of bf16:
//    1 sequence   17 tokens  18 /  18 /  13   32:  30 /  18 /  14   64:  56 /  20 /  14
//    8 sequences  33 tokens  35 /  37 /  28   48:  47 /  40 /  29   64:  60 /  42 /  30
//   64 sequences  33 tokens 119 / 233 / 159   48: 170 / 247 / 167   64: 217 / 275 / 178
//                 96 tokens 318 / 382 / 238  128: 418 / 401 / 246
// So it is right where the card is empty or just filled.  For many times as many sequences
// chunks pay from 48 (bf16) or 110 tokens (f32) on, and below that take up to twice as long.
static int few_alone(const qhip_linear_batch* b) { return (long)b->nseq * b->v_heads * (b->value_dim / 64) < 256 ? kFew : 2 * kFew; }

// sum over lanes l, l ^ 16, l ^ 32, l ^ 48
__device__ __forceinline__ float sum_rows(float v) {
  auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(x[0]) + __uint_as_float(x[1]);
  x = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(x[0]) + __uint_as_float(x[1]);
}

// N elements side by side, from any element's address
template <typename T, int N>
struct Some {
  T e[N];
  __device__ __forceinline__ void load(const T* p) {
    typedef uint32_t words __attribute__((ext_vector_type(N * sizeof(T) / 4 > 4 ? 4 : N * sizeof(T) / 4), aligned(2)));
    struct Words {
      words w[(N * sizeof(T) + 15) / 16];
    } x;
#pragma unroll
    for (unsigned i = 0; i < sizeof(x.w) / sizeof(words); ++i) x.w[i] = ((const words*)p)[i];
    *this = __builtin_bit_cast(Some, x);
  }
};

// ---- token by token --------------------------------------------------------------------
//
// A workgroup holds 64 columns of a head's state in registers: a lane four of them, of DK /
// 16 rows.  A token's products k S and q S (of the state before it) are summed over the rows
// together, so that one exchange between the waves serves both:  out = scale (a q S + (q . k)
// u).  (16 columns a workgroup: one token of one sequence of 16 heads 4.0 us instead of 4.2, of
// eight 8.8 instead of 5.5.)
//
// For one token the states' memory bounds it: 64 sequences of 32 heads of 128 x 128 read and
// write 268 MB in 56 us, 4.75 TB/s.  They pass the caches by (nontemporal): a layer's states
// are not met again before all other layers' have been; through the caches it takes 66 us, or
// 46 where no other work comes between the calls.
template <typename T, int DK>
__global__ __launch_bounds__(256) void k_linear_steps(LinearArgs a) {
  constexpr int COLS = 64, ACROSS = COLS / 4, R = DK * ACROSS / 256;  // lanes of a row, rows of a thread
  __shared__ __attribute__((aligned(16))) float s_part[2][4][2][COLS];
  __shared__ float s_qk[2][4];
  const int tid = threadIdx.x, wave = tid >> 6, col = (tid % ACROSS) * 4, row0 = tid / ACROSS * R;
  const int seq = blockIdx.z, head = blockIdx.y, d0 = blockIdx.x * COLS + col;
  const LinearSeq s = linear_seq(a, seq, head, DK);
  if (s.n > a.few || (s.n == 0 && s.from == s.to)) return;
  f32x4 st[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    st[r] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    if (s.from) st[r] = __builtin_nontemporal_load((const f32x4*)(s.from + (long)(row0 + r) * a.value_dim + d0));
    if (s.bad) st[r] = f32x4{__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
  }
  const int kh = head / a.group;
  const T* q = (const T*)a.q + s.first * a.q_token + kh * a.q_head + row0;
  const T* k = (const T*)a.k + s.first * a.k_token + kh * a.k_head + row0;
  const T* v = (const T*)a.v + s.first * a.v_token + head * a.v_head + d0;
  T* out = (T*)a.out + s.first * a.out_token + head * a.out_head + d0;
  const float* decay = a.log_decay + s.first * a.decay_token + head;
  const float* beta = a.beta ? a.beta + s.first * a.beta_token + head : nullptr;
  Some<T, R> kr, qr;
  Some<T, 4> vr;
  float log_keep = 0.0f, b = 0.0f;
  auto fetch = [&](int t) {
    kr.load(k + t * a.k_token);
    qr.load(q + t * a.q_token);
    vr.load(v + t * a.v_token);
    log_keep = decay[t * a.decay_token];
    if (beta) b = beta[t * a.beta_token];
  };
  if (s.n > 0) fetch(0);
  for (int t = 0; t < s.n; ++t) {
    float kf[R], vc[4], ks[4] = {}, qs[4] = {}, qk = 0.0f;
    const float keep = expf(log_keep), rate = b;
#pragma unroll
    for (int c = 0; c < 4; ++c) vc[c] = (float)vr.e[c];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float qf = (float)qr.e[r];
      kf[r] = (float)kr.e[r];
      qk = __builtin_fmaf(qf, kf[r], qk);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        ks[c] = __builtin_fmaf(kf[r], st[r][c], ks[c]);
        qs[c] = __builtin_fmaf(qf, st[r][c], qs[c]);
      }
    }
    if (t + 1 < s.n) fetch(t + 1);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      ks[c] = sum_rows(ks[c]);
      qs[c] = sum_rows(qs[c]);
    }
    qk = sum_rows(qk);
    const int buf = t & 1;
    if ((tid & 63) < ACROSS) {
      *(f32x4*)&s_part[buf][wave][0][col] = f32x4{ks[0], ks[1], ks[2], ks[3]};
      *(f32x4*)&s_part[buf][wave][1][col] = f32x4{qs[0], qs[1], qs[2], qs[3]};
      if ((tid & 63) == 0) s_qk[buf][wave] = qk;
    }
    __syncthreads();  // (the buffer after next is written behind the next token's barrier)
    qk = (s_qk[buf][0] + s_qk[buf][1]) + (s_qk[buf][2] + s_qk[buf][3]);
    f32x4 kc = {0.0f, 0.0f, 0.0f, 0.0f}, qc = kc;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      kc += *(const f32x4*)&s_part[buf][w][0][col];
      qc += *(const f32x4*)&s_part[buf][w][1][col];
    }
    float u[4], o[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      u[c] = beta ? rate * (vc[c] - keep * kc[c]) : vc[c];
      o[c] = a.scale * __builtin_fmaf(qk, u[c], keep * qc[c]);
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int c = 0; c < 4; ++c) st[r][c] = __builtin_fmaf(kf[r], u[c], keep * st[r][c]);
    if (tid < ACROSS) {
#pragma unroll
      for (int c = 0; c < 4; ++c) out[t * a.out_token + c] = (T)o[c];
    }
  }
  if (s.to) {
#pragma unroll
    for (int r = 0; r < R; ++r) __builtin_nontemporal_store(st[r], (f32x4*)(s.to + (long)(row0 + r) * a.value_dim + d0));
  }
}

template <typename T>
static void launch_steps(const LinearArgs& a, int key_dim, hipStream_t s) {
  const dim3 grid((unsigned)(a.value_dim / 64), (unsigned)a.v_heads, (unsigned)a.nseq);
  if (key_dim == 64) hipLaunchKernelGGL((k_linear_steps<T, 64>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((k_linear_steps<T, 128>), grid, dim3(256), 0, s, a);
}

// ---- chunks of 64 tokens ---------------------------------------------------------------
//
// Inside a chunk with G_i = log_decay_0 + .. + log_decay_i, S the state before it and
// D_ij = exp(G_i - G_j):
//
//   L_ij = beta_i (k_i . k_j) D_ij  (j < i),   T = (1 + L)^-1 diag(beta)
//   A_ij = scale (q_i . k_j) D_ij   (j <= i)
//   R = V - diag(exp(G)) K S,   U = T R    (U = V without the delta rule)
//   O = scale diag(exp(G)) Q S + A U
//   S <- exp(G_63) S + K^T (diag(exp(G_63 - G)) U)
//
// k_linear_prepare makes T, A and the exponentials of every chunk side by side;
// k_linear_scan then walks a sequence's chunks with 16 columns of a state in the
// registers of a workgroup.  G is summed in f64 and kept in two f32 parts, of which
// differences are taken: it is a long sum where the decay between near tokens is small.
//
// f32 rows take f32 matrix tiles throughout.  16-bit rows take bf16 ones for products with
// keys and queries, for which an f32 value goes in as a sum of three planes of 8 bits, which
// hold it whole; of products of planes those down to 2^-16 are summed.  So all sums are good
// to f32, and an output is rounded once, to its type.  (With the state, U and A in two planes
// for the outputs, 2^-16 off, 0.6% of bf16 outputs and 3% of f16 ones were rounded otherwise
// than the f64 results, instead of 0.02% and 0.09%: 253 us for 8192 tokens instead of 264.)
// Keys and queries need one plane (bf16) or two (f16).  T R and A U take f32 tiles for all
// types (A U in planes: as fast, with three times the registers or half as much again to read).
constexpr int kChunk = 64, kTiles = kChunk / 16;

typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// N planes of four values, two dwords a plane: all but the last cut off (no plane
// overflows), the last rounded to nearest.  (The third of three is exact.)
template <int N>
__device__ __forceinline__ void split4(f32x4 x, u32x2* out) {
#pragma unroll
  for (int p = 0; p < N; ++p) {
    if (p == N - 1) {
      typedef __bf16 b16x4 __attribute__((ext_vector_type(4)));
      out[p] = __builtin_bit_cast(u32x2, b16x4{(__bf16)x[0], (__bf16)x[1], (__bf16)x[2], (__bf16)x[3]});
    } else {
      out[p] = u32x2{__builtin_amdgcn_perm(__float_as_uint(x[1]), __float_as_uint(x[0]), 0x07060302u),
                     __builtin_amdgcn_perm(__float_as_uint(x[3]), __float_as_uint(x[2]), 0x07060302u)};
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] -= __uint_as_float(__float_as_uint(x[i]) & 0xFFFF0000u);
    }
  }
}
// four f16 values
__device__ __forceinline__ f32x4 floats(uint32_t x, uint32_t y) {
  typedef _Float16 h16x4 __attribute__((ext_vector_type(4)));
  const h16x4 z = __builtin_bit_cast(h16x4, u32x2{x, y});
  return f32x4{(float)z[0], (float)z[1], (float)z[2], (float)z[3]};
}
template <int N>
__device__ __forceinline__ void split8(f32x4 x, f32x4 y, u32x4* out) {
  u32x2 a[N], b[N];
  split4<N>(x, a);
  split4<N>(y, b);
#pragma unroll
  for (int p = 0; p < N; ++p) out[p] = u32x4{a[p][0], a[p][1], b[p][0], b[p][1]};
}

// Products of 16 x 16 results.  Lane l = 16 g + m holds row m of the left operand, column
// m of the right one and rows 4 g ..+3 of column m of the result: a result is a right
// operand for the products that follow, with 4 g ..+3 as its rows.
__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {  // 32 of bf16: 4 g ..+3 and 16 + 4 g ..+3
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b16x8, a), __builtin_bit_cast(b16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma4(f32x4 a, f32x4 b, f32x4 c) {  // 16 of f32: 4 g ..+3
#pragma unroll
  for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
  return c;
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

// What prepare leaves for a chunk and value head, as left operands of 1 KB: T's and A's tiles
// (i, j), j <= i, in f32; then exp(G), exp(G_63 - G), exp(G_63) and the
// first token whose row of L, or beta, is not finite (64: none).
constexpr int kWhole = 2 * kChunk, kSound = kWhole + 1, kNumbers = kWhole + 2;
template <bool DELTA>
struct ChunkWork {
  static constexpr int tiles = kTiles * (kTiles + 1) / 2 * 1024;
  static constexpr int solve = 0, inside = DELTA ? tiles : 0, numbers = inside + tiles, bytes = numbers + 576;
  __host__ __device__ static constexpr int tile(int i, int j) { return (i * (i + 1) / 2 + j) * 1024; }
};

// The chunk slot of a sequence's first: no two sequences' slots meet, and there are at
// most tokens / 64 + nseq.
__device__ __forceinline__ long first_slot(const LinearSeq& s, int i) { return s.first / kChunk + i; }

// A value that the compiler takes as new here.
__device__ __forceinline__ int fresh(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

// (LDS between the lanes of a wave: in order in the hardware, kept in order here)
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// One step of sixteen rows against sixteen others: 16 bytes of a row a lane.
template <typename T>
__device__ __forceinline__ f32x4 row_product(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (sizeof(T) == 4) return mfma4(__builtin_bit_cast(f32x4, a), __builtin_bit_cast(f32x4, b), c);
  else if constexpr (std::is_same<T, f16_t>::value)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h16x8, a), __builtin_bit_cast(h16x8, b), c, 0, 0, 0);
  else return mfma(a, b, c);
}

// A workgroup takes a chunk of one key head, and its value heads in turn.  The ten tiles of K
// K^T are two waves', those of K Q^T the others': with the keys on the left, a result has row
// m, columns 4 g ..+3 of L or A, as they go into LDS and out.  (1 + L)^-1 goes by blocks of
// 16: those on the diagonal by substitution, a column a lane; then each column of blocks
// downwards, X_ij = -X_ii sum of L_ik X_kj, a wave a column.
template <typename T, int DK, bool DELTA>
__global__ __launch_bounds__(256) void k_linear_prepare(LinearArgs a) {
  typedef ChunkWork<DELTA> W;
  constexpr int ROW = kChunk + 4;  // floats of a row in LDS
  constexpr int PIECES = DK * sizeof(T) / 64, TILE = PIECES * 64;  // 16-byte pieces of a row a lane, of 16 rows
  __shared__ u32x4 s_rows[2][kTiles][TILE];  // keys and queries; then L and its inverse
  __shared__ __attribute__((aligned(16))) float s_sum[2][kChunk];  // G in two parts
  __shared__ __attribute__((aligned(16))) float s_beta[kChunk];
  __shared__ int s_sound[3];  // the first token that is not finite: beta, L's rows of either wave
  static_assert(sizeof(s_rows) >= kChunk * ROW * 4 || DK == 64, "L");
  constexpr int MORE = sizeof(s_rows) >= kChunk * ROW * 4 ? 1 : kChunk * ROW;  // (16-bit rows of 64)
  __shared__ __attribute__((aligned(16))) float s_more[MORE];
  float* const mat = MORE > 1 ? s_more : (float*)s_rows;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, g = lane >> 4, m = lane & 15;
  // (heads side by side: a head's rows, a token's stride apart, lie in few memory channels)
  const int slot = blockIdx.x / a.k_heads, kh = blockIdx.x - slot * a.k_heads;
  // the slot's sequence: the last whose first slot is not behind it
  int seq = -1, first = 0, end = 0;
  for (int i0 = 0; i0 < a.nseq; i0 += 64) {
    const int i = min(i0 + lane, a.nseq - 1), from = a.offsets[i], to = a.offsets[i + 1];
    const uint64_t before = __ballot(i0 + lane < a.nseq && from / kChunk + i <= slot);
    const int count = __builtin_popcountll(before);
    if (count == 0) break;
    seq = i0 + count - 1;
    first = __builtin_amdgcn_readlane(from, count - 1);
    end = __builtin_amdgcn_readlane(to, count - 1);
    if (count < 64) break;
  }
  if (seq < 0) return;
  LinearSeq s{first, 0, nullptr, nullptr, false};
  end = min(end, a.tokens);
  if (first >= 0 && end > first) s.n = min(end - first, a.max_new);
  const int chunk = (int)(slot - first_slot(s, seq)), n = s.n - chunk * kChunk;  // tokens from the chunk's first on
  if (chunk < 0 || n <= 0 || s.n <= a.few) return;
  const long t0 = first + (long)chunk * kChunk;
  {
    const char* k = (const char*)((const T*)a.k + t0 * a.k_token + kh * a.k_head);
    const char* q = (const char*)((const T*)a.q + t0 * a.q_token + kh * a.q_head);
    typedef uint32_t piece __attribute__((ext_vector_type(4), aligned(2)));
    constexpr int EACH = TILE / 256 ? TILE / 256 : 1;  // pieces of a tile a thread
    const int tid = threadIdx.x, step = tid >> 6;
    if (TILE >= 256 || tid < TILE) {
      u32x4 x[2][kTiles][EACH];  // (rows behind the sequence's end: the last again)
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        const long row = min(16 * t + m, n - 1);
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
          const int at = 64 * (step + 4 * e) + 16 * g;
          x[0][t][e] = *(const piece*)(k + row * a.k_token * (long)sizeof(T) + at);
          x[1][t][e] = *(const piece*)(q + row * a.q_token * (long)sizeof(T) + at);
        }
      }
#pragma unroll
      for (int t = 0; t < kTiles; ++t)
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
          s_rows[0][t][tid + 256 * e] = x[0][t][e];
          s_rows[1][t][tid + 256 * e] = x[1][t][e];
        }
    }
  }
  __syncthreads();
  // rows of tiles 3 and 0, or 1 and 2, of L or A: five tiles each
  const bool keys = wave < 2, outer = (wave & 1) == 0;
  f32x4 product[5] = {};
  if (DELTA || !keys) {
    const u32x4(*rows)[TILE] = s_rows[keys ? 0 : 1];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int at = i * 64 + lane;
      const u32x4 x0 = rows[outer ? 3 : 1][at], x1 = rows[outer ? 0 : 2][at];
      const u32x4 y0 = s_rows[0][0][at], y1 = s_rows[0][1][at], y2 = s_rows[0][2][at];
      product[0] = row_product<T>(y0, x0, product[0]);
      product[1] = row_product<T>(y1, x0, product[1]);
      if (outer) {
        product[2] = row_product<T>(y2, x0, product[2]);
        product[3] = row_product<T>(s_rows[0][3][at], x0, product[3]);
        product[4] = row_product<T>(y0, x1, product[4]);
      } else {
        product[2] = row_product<T>(y0, x1, product[2]);
        product[3] = row_product<T>(y1, x1, product[3]);
        product[4] = row_product<T>(y2, x1, product[4]);
      }
    }
  }
  for (int head = kh * a.group; head < (kh + 1) * a.group; ++head) {
    // (lanes as something new in each pass: what follows from them would fill the registers)
    const int lane = fresh(threadIdx.x & 63), g = lane >> 4, m = lane & 15;
    uint8_t* out = a.work + ((long)slot * a.v_heads + head) * W::bytes;
    if (wave == 0) {
      // G (times log2 e) in f64; a decay of exp(-200) is 0 in f32, and sums of -infinity
      // have no differences
      const long t = t0 + min(lane, n - 1);
      const float decay = a.log_decay[t * a.decay_token + head], beta = DELTA ? a.beta[t * a.beta_token + head] : 0.0f;
      double sum = lane < n ? (decay < -200.0f ? -200.0 : (double)decay) * 1.4426950408889634 : 0.0;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const double up = __shfl_up(sum, d, 64);
        if (lane >= d) sum += up;
      }
      s_sum[0][lane] = (float)sum;
      s_sum[1][lane] = (float)(sum - (float)sum);
      s_beta[lane] = lane < n ? beta : 0.0f;
      const uint64_t bad = __ballot(lane < n && !(__builtin_fabsf(beta) < INFINITY));
      if (lane == 0) s_sound[2] = bad ? __builtin_ctzll(bad) : kChunk;
    }
    __syncthreads();
    f32x4 tile[5];
    if (DELTA || !keys) {
      // of tiles (3, 0) .. (3, 3), (0, 0), or (1, 0), (1, 1), (2, 0) .. (2, 2)
      const float scales[2] = {keys ? s_beta[outer ? 48 + m : 16 + m] : a.scale, keys ? s_beta[outer ? m : 32 + m] : a.scale};
#pragma unroll
      for (int e = 0; e < 5; ++e) {
        const int first_of = outer ? 4 : 2, second = e >= first_of;
        const int i = (outer ? (second ? 0 : 48) : (second ? 32 : 16)) + m, j0 = 16 * (second ? e - first_of : e) + 4 * g;
        const f32x4 far = s_sum[0][i] - *(const f32x4*)&s_sum[0][j0], near = s_sum[1][i] - *(const f32x4*)&s_sum[1][j0];
        const float scale = second ? scales[1] : scales[0];
        const int seen = i < n ? i + !keys - j0 : 0;  // columns of the four that the row has
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float x = product[e][r] * (__builtin_amdgcn_exp2f(far[r] + near[r]) * scale);
          tile[e][r] = r < seen ? x : 0.0f;
        }
        if (DELTA && keys) *(f32x4*)&mat[i * ROW + j0] = tile[e];
      }
      if (DELTA && keys) {
        const int second_of = outer ? 4 : 2;  // (rows of two tiles, as above)
        int bad = kChunk;
#pragma unroll
        for (int e = 0; e < 5; ++e) {
          const f32x4 none = tile[e] * 0.0f;
          if ((none[0] + none[1]) + (none[2] + none[3]) != 0.0f) bad = min(bad, (outer ? (e >= second_of ? 0 : 48) : (e >= second_of ? 32 : 16)) + m);
        }
        if (__ballot(bad < kChunk)) {
#pragma unroll
          for (int d = 1; d < 64; d <<= 1) bad = min(bad, __shfl_xor(bad, d, 64));
        }
        if (lane == 0) s_sound[outer] = bad;
      }
    }
    if (!keys) {  // A
#pragma unroll
      for (int e = 0; e < 5; ++e) {
        const int at = outer ? (e < 4 ? W::tile(3, e) : W::tile(0, 0)) : e < 2 ? W::tile(1, e) : W::tile(2, e - 2);
        *((f32x4*)(out + W::inside + at) + lane) = tile[e];
      }
    }
    if (wave == 3) {
      float* numbers = (float*)(out + W::numbers);
      const float sum = s_sum[0][lane];
      numbers[lane] = __builtin_amdgcn_exp2f(sum);
      numbers[64 + lane] = __builtin_amdgcn_exp2f((s_sum[0][63] - sum) + (s_sum[1][63] - s_sum[1][lane]));
      if (lane == 63) numbers[kWhole] = __builtin_amdgcn_exp2f(sum);
    }
    if constexpr (DELTA) {
      __syncthreads();
      // Rows of the inverse from the first that is not finite on are left out (0): in the
      // products below they would spoil the rows before, with 0 * NaN.
      const int sound = min(min(s_sound[0], s_sound[1]), s_sound[2]);
      if (sound < kChunk) {
        for (int e = threadIdx.x; e < (kChunk - sound) * ROW; e += 256) mat[sound * ROW + e] = 0.0f;
        __syncthreads();
      }
      if (wave == 3 && lane == 0) ((float*)(out + W::numbers))[kSound] = (float)sound;
      if (wave == 0) {
        const int b = lane & 48;
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float y = i == m ? 1.0f : 0.0f;
#pragma unroll
          for (int l = 0; l < i; ++l) y = __builtin_fmaf(-mat[(b + i) * ROW + b + l], x[l], y);
          x[i] = i < m ? 0.0f : y;
        }
        wave_sync();
#pragma unroll
        for (int i = 0; i < 16; ++i) mat[(b + i) * ROW + b + m] = x[i];
      }
      __syncthreads();
      auto block = [&](int i, int j) { return mat + (16 * i + m) * ROW + 16 * j + 4 * g; };  // as a left operand
      // T = X diag(beta) (nothing above the diagonal, whatever beta holds)
      auto leave = [&](int i, int j, f32x4 x) {
        const f32x4 b = *(const f32x4*)(s_beta + 16 * j + 4 * g);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = 16 * i + m < sound && (i > j || 4 * g + e <= m) ? x[e] * b[e] : 0.0f;
        *((f32x4*)(out + W::solve + W::tile(i, j)) + lane) = x;
      };
      const f32x4 none = {0.0f, 0.0f, 0.0f, 0.0f};
      if (wave == 3) {
#pragma unroll
        for (int i = 0; i < kTiles; ++i) leave(i, i, *(const f32x4*)block(i, i));
      } else {
        const int j = wave;
        f32x4 x[kTiles];
#pragma unroll
        for (int r = 0; r < 4; ++r) x[0][r] = mat[(16 * j + 4 * g + r) * ROW + 16 * j + m];
#pragma unroll
        for (int d = 1; d < kTiles; ++d) {  // x[d] is X_{j + d, j}
          if (j + d >= kTiles) break;
          f32x4 sum[2] = {none, none};  // (side by side: each product waits for the one before it)
#pragma unroll
          for (int e = 0; e < d; ++e) sum[e & 1] = mfma4(*(const f32x4*)block(j + d, j + e), x[e], sum[e & 1]);
          sum[0] += sum[1];
          // a sum that overflowed would, by the zeros of X_ii, spoil the rows before its own:
          // it stays out of the product, and its row of X is NaN
          const f32x4 over = sum[0] * 0.0f;
          const bool some = __ballot((over[0] + over[1]) + (over[2] + over[3]) != 0.0f);
          if (some) {
#pragma unroll
            for (int r = 0; r < 4; ++r) sum[0][r] = over[r] == 0.0f ? sum[0][r] : 0.0f;
          }
          x[d] = mfma4(-*(const f32x4*)block(j + d, j + d), sum[0], none);
          if (some) x[d] += over;
          // turned by way of the blocks above the diagonal, which nothing reads
          wave_sync();
#pragma unroll
          for (int r = 0; r < 4; ++r) mat[(16 * j + 4 * g + r) * ROW + 16 * (j + d) + m] = x[d][r];
          wave_sync();
          leave(j + d, j, *(const f32x4*)block(j, j + d));
        }
      }
    }
    if (head + 1 < (kh + 1) * a.group) __syncthreads();
  }
}

// Four waves carry the state and four others make the outputs, each pair on one SIMD.  DK /
// 32 of either kind have the same 16 columns: of the first, each keeps 32 rows of the state
// in registers, and all have their share of the chunk's four tiles of 16 tokens.  Between
// three barriers a chunk:
//
//   the state, in planes, into LDS, and all tokens' K S over the own rows
//   R of the own tokens        | Q S of the own tokens
//   U of the own tokens        | the next chunk's keys into LDS, as rows and turned
//   the state's update         | the outputs
//
// A chunk waits for the one before it, so its chain bounds a sequence.  bf16 rows of 128 with
// the delta rule: 2.0 us, of which products fill three tenths and vector instructions a quarter,
// the rest being LDS, barriers and waits for each other (loads a chunk ahead do not show); 8192
// tokens of 32 value heads, a workgroup on every CU, 252 to 262 us, beside 41 of prepare, and
// of 16 heads, on half of the CUs, 236 and 27.  f32 rows: 3.4 us (16 heads), 3700 cycles of f32
// products on each SIMD among them; eight prompts of up to 256 tokens of 16 heads, four rounds of
// workgroups, 58 and 15.  (Of the bf16 prompt, before outputs took three planes, 223: with K S of
// the own tokens over all rows of the state, read by every wave from LDS, 229; with T in three
// planes of bf16, so that its product takes a third of the cycles, 263, for the splits and the
// larger loads.)  A second workgroup on a CU has no room in LDS (with the delta rule 86 to 141
// KB, f32 and f16 rows of 128 without it 87 and 98) or in registers (keys of 64: 146 to 162);
// bf16 rows of 128 without it (61 KB, 110 registers) would fit, but for amdgpu_waves_per_eu.
template <typename T, int DK, bool DELTA>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2))) void k_linear_scan(LinearArgs a) {
  typedef ChunkWork<DELTA> W;
  constexpr bool F32 = sizeof(T) == 4;
  constexpr int P = std::is_same<T, f16_t>::value ? 2 : 1;  // planes of keys and queries
  constexpr int PARTS = DK / 32, SETS = 4 / PARTS, COLS = 16 * SETS, OWN = kTiles / PARTS;
  constexpr int PIECES = DK * sizeof(T) / 64;  // of 16 bytes of a row a lane
  // Keys, as left operands of 16 tokens, and turned, as those of 16 dimensions: steps of 32
  // tokens (f32: 16), a step's lanes of equal l / 16 272 bytes apart.  The strides are such
  // that the lanes of a store, which hold other tokens, fall on all banks.
  constexpr int GROUP = 272, STEP = F32 ? 4 * GROUP : 4 * GROUP + 64, TURNED = (F32 ? 4 : 2) * STEP, KEYS = P * (DK / 16) * TURNED;
  __shared__ u32x4 s_rows[DELTA ? kTiles : 1][PIECES * 64 + 1];
  __shared__ __attribute__((aligned(16))) uint8_t s_keys[2 * KEYS];
  __shared__ __attribute__((aligned(16))) float s_numbers[2][kNumbers + 2];
  constexpr int SP = F32 ? 2 : 3;
  __shared__ u32x4 s_state[SETS][PARTS][SP][64];  // three planes, f32: two tiles
  __shared__ f32x4 s_part[DELTA ? SETS : 1][PARTS][kTiles][64];  // K S over the dimensions of a wave
  __shared__ f32x4 s_rest[DELTA ? SETS : 1][kTiles][64];
  __shared__ __attribute__((aligned(16))) int s_spoilt[DELTA ? 2 : 1][SETS][16][kTiles];  // by R; by U too
  __shared__ u32x4 s_new[SETS][F32 ? 1 : 3][kTiles / (F32 ? 1 : 2)][64];  // U as it enters the state
  __shared__ f32x4 s_old[SETS][kTiles][64];  // U for the outputs
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, g = lane >> 4, m = lane & 15;
  const int set = (wave & 3) / PARTS, part = (wave & 3) % PARTS;
  // the workgroups of a sequence's head follow each other on one XCD
  const int blocks = a.value_dim / COLS, id = (int)blockIdx.x;
  const int pair = id / (8 * blocks) * 8 + (id & 7), seq = pair / a.v_heads, head = pair - seq * a.v_heads;
  if (seq >= a.nseq) return;
  const int col = (id >> 3) % blocks * COLS + set * 16 + m;
  const LinearSeq s = linear_seq(a, seq, head, DK);
  if (s.n <= a.few) return;
  const int kh = head / a.group, chunks = (s.n + kChunk - 1) / kChunk, tail = s.n - (chunks - 1) * kChunk;
  // the wave's tiles of tokens (of two the first and last, or those between: T has 1 to 4
  // tiles in a row, and so has A, which a SIMD's other wave takes the other way round)
  auto own = [&](int o) { return (o == 0) == (wave < 4) ? part : 3 - part; };
  auto rows_of = [&](int c) { return c + 1 < chunks ? kChunk : tail; };

  // Everything of a chunk is loaded for the next one when the present one is done with
  // it, without branches: uniform bases that go on by 64 tokens, offsets of 32 bits, and
  // the last token's in the place of those behind it.
  // (global memory by name: through a flat address, a load would count as one of LDS too)
  typedef const __attribute__((address_space(1))) uint8_t* Work;
  typedef const __attribute__((address_space(1))) f32x4* GlobalF4;
  Work work = (Work)a.work + (first_slot(s, seq) * a.v_heads + head) * W::bytes;
  const long work_step = (long)a.v_heads * W::bytes;
  typedef uint32_t piece __attribute__((ext_vector_type(4), aligned(2)));
  // exp(G) or (64) exp(G_63 - G) of tile t's rows 4 g ..+3
  auto number = [&](int c, int at, int t) { return *(const f32x4*)&s_numbers[c & 1][at + 16 * t + 4 * g]; };
  // sixteen rows' product with the state, in two sums side by side (each product waits
  // for the one before it)
  auto with_state = [&](auto row) {
    f32x4 c[2] = {};
#pragma unroll
    for (int i = 0; i < PARTS; ++i) {
      u32x4 sp[SP];
#pragma unroll
      for (int p = 0; p < SP; ++p) sp[p] = s_state[set][i][p][lane];
      if constexpr (F32) {
#pragma unroll
        for (int h = 0; h < 2; ++h) c[h] = mfma4(__builtin_bit_cast(f32x4, row(2 * i + h)), __builtin_bit_cast(f32x4, sp[h]), c[h]);
      } else {
        const u32x4 y = row(i);
        u32x4 x[P];
        if constexpr (P == 1) x[0] = y;
        else split8<P>(floats(y[0], y[1]), floats(y[2], y[3]), x);
        c[i & 1] = mfma_planes<P, 3>(x, sp, c[i & 1]);
      }
    }
    return c[0] + c[1];
  };
  // a column's first token whose R (or U) is not finite
  auto first_spoilt = [&](int by) {
    const u32x4 all = *(const u32x4*)s_spoilt[by][set][m];
    return min(min((int)all[0], (int)all[1]), min((int)all[2], (int)all[3]));
  };

  if (wave < 4) {
    // state: row 4 g + r of tile i is dimension 8 g + 4 i + r of the wave's 32, so that the
    // eight of a lane are side by side in a key (f32: tiles of 16 dimensions as they lie)
    f32x4 st[2];
    auto state_at = [&](int i, int r) { return (long)(32 * part + (F32 ? 16 * i + 4 * g : 8 * g + 4 * i) + r) * a.value_dim + col; };
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) st[i][r] = s.from ? s.from[state_at(i, r)] : s.bad ? __builtin_nanf("") : 0.0f;

    const char* v_at = (const char*)((const T*)a.v + s.first * a.v_token + head * a.v_head);
    const long v_step = kChunk * a.v_token * (long)sizeof(T);
    T val[OWN][4];
    uint32_t v_off[OWN][4];
    auto place = [&](int rows) {  // of a chunk with that many tokens
#pragma unroll
      for (int o = 0; o < OWN; ++o)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          v_off[o][r] = (uint32_t)(min(16 * own(o) + 4 * g + r, rows - 1) * (int)a.v_token + col) * (uint32_t)sizeof(T);
    };
    auto fetch_values = [&]() {
#pragma unroll
      for (int o = 0; o < OWN; ++o)
#pragma unroll
        for (int r = 0; r < 4; ++r) val[o][r] = *(const T*)(v_at + v_off[o][r]);
    };
    f32x4 solve[OWN][kTiles];
    auto fetch_solve = [&]() {
#pragma unroll
      for (int o = 0; o < OWN; ++o) {
        if constexpr (DELTA) {
#pragma unroll
          for (int j = 0; j < kTiles; ++j) solve[o][j] = *(GlobalF4)(work + W::solve + W::tile(own(o), min(j, own(o))) + lane * 16);
        }
      }
    };
    // What is not finite spoils its column from its token on; in a product it would spoil
    // the tokens before as well (0 * NaN), so it stays out of them.
    auto leave_out = [&](f32x4& x, int t, int first, int by) {
      float sum = 0.0f;
#pragma unroll
      for (int r = 0; r < 4; ++r) sum = __builtin_fmaf(x[r], 0.0f, sum);
      if (__ballot(sum != 0.0f)) {
#pragma unroll
        for (int r = 3; r >= 0; --r)
          if (!(__builtin_fabsf(x[r]) < INFINITY)) {
            first = min(first, 16 * t + 4 * g + r);
            x[r] = 0.0f;
          }
        first = min(first, __shfl_xor(first, 16, 64));
        first = min(first, __shfl_xor(first, 32, 64));
      }
      if (lane < 16) s_spoilt[by][set][m][t] = first;
    };
    place(rows_of(0));
    fetch_values();
    fetch_solve();
    __syncthreads();  // (the first chunk's keys)
    // (the last chunk apart: with branches around them, loads are waited for in vain)
    auto step = [&](int c, auto last) {
      constexpr bool LAST = decltype(last)::value;
      if constexpr (!LAST) {
        work += work_step;
        v_at += v_step;
        if (c + 2 == chunks) place(tail);
      }
      if constexpr (F32) {
        s_state[set][part][0][lane] = __builtin_bit_cast(u32x4, st[0]);
        s_state[set][part][1][lane] = __builtin_bit_cast(u32x4, st[1]);
      } else {
        u32x4 sp[3];
        split8<3>(st[0], st[1], sp);
#pragma unroll
        for (int p = 0; p < 3; ++p) s_state[set][part][p][lane] = sp[p];
        if constexpr (DELTA) {
#pragma unroll
          for (int t = 0; t < kTiles; ++t) {
            const u32x4 y = s_rows[t][part * 64 + lane];
            u32x4 x[P];
            if constexpr (P == 1) x[0] = y;
            else split8<P>(floats(y[0], y[1]), floats(y[2], y[3]), x);
            s_part[set][part][t][lane] = mfma_planes<P, 3>(x, sp, f32x4{0.0f, 0.0f, 0.0f, 0.0f});
          }
        }
      }
      if constexpr (DELTA && F32) {
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
          f32x4 x[2];
#pragma unroll
          for (int h = 0; h < 2; ++h)
            x[h] = mfma4(__builtin_bit_cast(f32x4, s_rows[t][(2 * part + h) * 64 + lane]), st[h], f32x4{0.0f, 0.0f, 0.0f, 0.0f});
          s_part[set][part][t][lane] = x[0] + x[1];
        }
      }
      __syncthreads();
      f32x4 u[OWN];
#pragma unroll
      for (int w = 0; w < OWN; ++w) {
        const int t = own(w);
#pragma unroll
        for (int r = 0; r < 4; ++r) u[w][r] = (float)val[w][r];
        if constexpr (LAST) {
#pragma unroll
          for (int r = 0; r < 4; ++r) u[w][r] = 16 * t + 4 * g + r < tail ? u[w][r] : 0.0f;
        }
        // (rows behind the sequence's end have the last row's keys: their T is 0)
        if constexpr (DELTA) {
          f32x4 ks = s_part[set][0][t][lane];
#pragma unroll
          for (int p = 1; p < PARTS; ++p) ks += s_part[set][p][t][lane];
          u[w] -= number(c, 0, t) * ks;
        }
        leave_out(u[w], t, DELTA ? (int)s_numbers[c & 1][kSound] : kChunk, 0);
        if constexpr (DELTA) s_rest[set][t][lane] = u[w];
      }
      if constexpr (!LAST) fetch_values();
      if constexpr (DELTA) {
        __syncthreads();
        f32x4 rest[kTiles];
#pragma unroll
        for (int j = 0; j < kTiles; ++j) rest[j] = s_rest[set][j][lane];
        const int spoilt = first_spoilt(0);
#pragma unroll
        for (int w = 0; w < OWN; ++w) {
          const int t = own(w);
          f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f}, y = x;
#pragma unroll
          for (int j = 0; j < kTiles; ++j)
            if (j <= t) {
              if (j & 1) y = mfma4(solve[w][j], rest[j], y);
              else x = mfma4(solve[w][j], rest[j], x);
            }
          u[w] = x + y;
          if (__ballot(spoilt < kChunk)) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (16 * t + 4 * g + r >= spoilt) u[w][r] = 0.0f;
          }
          leave_out(u[w], t, spoilt, 1);  // (T or the product may have overflowed)
        }
      }
#pragma unroll
      for (int w = 0; w < OWN; ++w) {
        const int t = own(w);
        const f32x4 in = number(c, kChunk, t) * u[w];
        s_old[set][t][lane] = u[w];
        if constexpr (F32) {
          s_new[set][0][t][lane] = __builtin_bit_cast(u32x4, in);
        } else {
          u32x2 planes[3];
          split4<3>(in, planes);
#pragma unroll
          for (int p = 0; p < 3; ++p) ((u32x2*)&s_new[set][p][t >> 1][lane])[t & 1] = planes[p];
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) st[i] *= s_numbers[c & 1][kWhole];
      if constexpr (!LAST) fetch_solve();
      __syncthreads();
      const uint8_t* turned = s_keys + (c & 1) * KEYS + 2 * part * TURNED + g * GROUP + m * 16;
      if constexpr (F32) {
#pragma unroll
        for (int j = 0; j < kTiles; ++j) {
          const f32x4 x = __builtin_bit_cast(f32x4, s_new[set][0][j][lane]);
#pragma unroll
          for (int i = 0; i < 2; ++i) st[i] = mfma4(*(const f32x4*)(turned + i * TURNED + j * STEP), x, st[i]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < kTiles / 2; ++j) {
          const u32x4 x[3] = {s_new[set][0][j][lane], s_new[set][1][j][lane], s_new[set][2][j][lane]};
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            u32x4 y[P];
#pragma unroll
            for (int p = 0; p < P; ++p) y[p] = *(const u32x4*)(turned + (p * (DK / 16) + i) * TURNED + j * STEP);
            st[i] = mfma_planes<P, 3>(y, x, st[i]);
          }
        }
      }
      const int spoilt = first_spoilt(DELTA);
      if (__ballot(spoilt < kChunk)) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) st[i][r] = spoilt < kChunk ? __builtin_nanf("") : st[i][r];
      }
    };
    for (int c = 0; c + 1 < chunks; ++c) step(c, std::false_type{});
    step(chunks - 1, std::true_type{});
    if (s.to) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) s.to[state_at(i, r)] = st[i][r];
    }
    return;
  }

  const int tid = threadIdx.x & 255;
  const char* k_at = (const char*)((const T*)a.k + s.first * a.k_token + kh * a.k_head);
  const char* q_at = (const char*)((const T*)a.q + s.first * a.q_token + kh * a.q_head);
  char* out_at = (char*)((T*)a.out + s.first * a.out_token + head * a.out_head);
  const long k_step = kChunk * a.k_token * (long)sizeof(T), q_step = kChunk * a.q_token * (long)sizeof(T),
             out_step = kChunk * a.out_token * (long)sizeof(T);
  // the wave's tokens' queries: row m, piece i has 16 bytes from byte 64 i + 16 g on
  u32x4 qr[OWN][PIECES];
  Work key_work = work;
  // keys: four tokens x 16 bytes a thread (f32 of 128 dimensions twice)
  constexpr int ACROSS = DK * sizeof(T) / 16, TURNS = 16 * ACROSS > 256 ? 16 * ACROSS / 256 : 1;
  const int dq = tid / (16 / TURNS) % ACROSS, tq = tid % (16 / TURNS);
  const bool turns = tid < 16 * ACROSS;
  u32x4 held[TURNS][4];
  float held_number;
  uint32_t q_off[OWN], held_off[TURNS][4];
  auto place_queries = [&](int rows) {  // of a chunk with that many tokens
#pragma unroll
    for (int o = 0; o < OWN; ++o)
      q_off[o] = (uint32_t)(min(16 * own(o) + m, rows - 1) * (int)a.q_token) * (uint32_t)sizeof(T) + 16 * g;
  };
  auto place_keys = [&](int rows) {
#pragma unroll
    for (int e = 0; e < TURNS; ++e)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        held_off[e][i] = (uint32_t)(min(4 * tq + 64 / TURNS * e + i, rows - 1) * (int)a.k_token) * (uint32_t)sizeof(T) + 16 * dq;
  };
  auto fetch_queries = [&]() {
#pragma unroll
    for (int o = 0; o < OWN; ++o)
#pragma unroll
      for (int i = 0; i < PIECES; ++i) qr[o][i] = *(const piece*)(q_at + q_off[o] + 64 * i);
  };
  auto fetch_keys = [&]() {
#pragma unroll
    for (int e = 0; e < TURNS; ++e)
#pragma unroll
      for (int i = 0; i < 4; ++i) held[e][i] = *(const piece*)(k_at + held_off[e][i]);
    held_number = *(const __attribute__((address_space(1))) float*)(key_work + W::numbers + 4 * min(tid, kNumbers - 1));
  };
  f32x4 inside[OWN][kTiles];
  auto fetch_inside = [&]() {
#pragma unroll
    for (int o = 0; o < OWN; ++o)
#pragma unroll
      for (int j = 0; j < kTiles; ++j) inside[o][j] = *(GlobalF4)(work + W::inside + W::tile(own(o), min(j, own(o))) + lane * 16);
  };
  // the held keys and numbers into LDS (behind the sequence's end the last key: U is 0 there)
  auto put_keys = [&](int buffer) {
    if (tid < kNumbers) s_numbers[buffer][tid] = held_number;
    if (!turns) return;
#pragma unroll
    for (int e = 0; e < TURNS; ++e) {
      const int quad = tq + 16 / TURNS * e;  // of tokens
      if constexpr (DELTA) {
#pragma unroll
        for (int i = 0; i < 4; ++i) s_rows[quad >> 2][(dq >> 2) * 64 + (dq & 3) * 16 + (quad & 3) * 4 + i] = held[e][i];
      }
      uint8_t* to = s_keys + buffer * KEYS + (dq & 3) * 64 + (quad & 3) * GROUP;
      if constexpr (F32) {  // dimensions 4 dq ..+3
        to += (dq >> 2) * TURNED + (quad >> 2) * STEP;
#pragma unroll
        for (int j = 0; j < 4; ++j) *(u32x4*)(to + j * 16) = u32x4{held[e][0][j], held[e][1][j], held[e][2][j], held[e][3][j]};
      } else {  // dimensions 8 dq ..+7: rows 4 (dq mod 4) ..+3 of two tiles
        to += (dq >> 2) * 2 * TURNED + (quad >> 3) * STEP + ((quad >> 2) & 1) * 8;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          u32x2 planes[4][P];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if constexpr (P == 1) planes[i][0] = u32x2{held[e][i][2 * h], held[e][i][2 * h + 1]};
            else split4<P>(floats(held[e][i][2 * h], held[e][i][2 * h + 1]), planes[i]);
          }
#pragma unroll
          for (int p = 0; p < P; ++p)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint32_t pick = j & 1 ? 0x07060302u : 0x05040100u;
              *(u32x2*)(to + (p * (DK / 16) + h) * TURNED + j * 16) =
                  u32x2{__builtin_amdgcn_perm(planes[1][p][j >> 1], planes[0][p][j >> 1], pick),
                        __builtin_amdgcn_perm(planes[3][p][j >> 1], planes[2][p][j >> 1], pick)};
            }
        }
      }
    }
  };
  place_queries(rows_of(0));
  place_keys(rows_of(0));
  fetch_keys();
  fetch_queries();
  fetch_inside();
  put_keys(0);
  if (chunks > 1) {
    k_at += k_step;
    key_work += work_step;
    if (chunks == 2) place_keys(tail);
  }
  fetch_keys();
  __syncthreads();
  auto step = [&](int c, auto last) {
    constexpr bool LAST = decltype(last)::value;
    if constexpr (!LAST) {
      work += work_step;
      q_at += q_step;
      if (c + 2 == chunks) place_queries(tail);
    }
    __syncthreads();
    f32x4 o[OWN];
#pragma unroll
    for (int w = 0; w < OWN; ++w) o[w] = a.scale * number(c, 0, own(w)) * with_state([&](int i) { return qr[w][i]; });
    if constexpr (!LAST) fetch_queries();
    if constexpr (DELTA) __syncthreads();
    if constexpr (!LAST) {
      put_keys((c + 1) & 1);
      if (c + 2 < chunks) {
        k_at += k_step;
        key_work += work_step;
        if (c + 3 == chunks) place_keys(tail);
      }
      fetch_keys();
    }
    __syncthreads();
    const int spoilt = first_spoilt(DELTA);
#pragma unroll
    for (int w = 0; w < OWN; ++w) {
      const int t = own(w), row = 16 * t + 4 * g;
      f32x4 more = {0.0f, 0.0f, 0.0f, 0.0f};  // a second sum beside o[w], as above
#pragma unroll
      for (int j = 0; j < kTiles; ++j)
        if (j <= t) {
          f32x4& sum = j & 1 ? more : o[w];
          sum = mfma4(inside[w][j], s_old[set][j][lane], sum);
        }
      o[w] += more;
      if (__ballot(spoilt < kChunk)) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (row + r >= spoilt) o[w][r] = __builtin_nanf("");
      }
      auto store = [&](int r) {
        *(T*)(out_at + (uint32_t)((row + r) * (int)a.out_token + col) * (uint32_t)sizeof(T)) = (T)o[w][r];
      };
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (!LAST || row + r < tail) store(r);
    }
    if constexpr (!LAST) fetch_inside();
    out_at += out_step;
  };
  for (int c = 0; c + 1 < chunks; ++c) step(c, std::false_type{});
  step(chunks - 1, std::true_type{});
}

template <typename T, int DK, bool DELTA>
static void launch_chunks(const LinearArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((k_linear_prepare<T, DK, DELTA>), dim3((unsigned)((a.tokens / kChunk + a.nseq) * a.k_heads)), dim3(256), 0, s, a);
  const long pairs = ((long)a.nseq * a.v_heads + 7) / 8 * 8;
  hipLaunchKernelGGL((k_linear_scan<T, DK, DELTA>), dim3((unsigned)(pairs * (a.value_dim / (2048 / DK)))), dim3(512), 0, s, a);
}

template <typename T>
static void launch_linear(const LinearArgs& a, int key_dim, bool chunks, hipStream_t s) {
  launch_steps<T>(a, key_dim, s);
  if (!chunks) return;
  if (key_dim == 64) a.beta ? launch_chunks<T, 64, true>(a, s) : launch_chunks<T, 64, false>(a, s);
  else a.beta ? launch_chunks<T, 128, true>(a, s) : launch_chunks<T, 128, false>(a, s);
}

// 0: token by token (also where a grid would pass 2^32 threads)
static long linear_work(const qhip_linear_batch* b, bool delta) {
  if (b->max_new <= few_alone(b) || b->nseq == 0 || b->tokens == 0) return 0;
  const long slots = (long)b->tokens / kChunk + b->nseq, pairs = (long)b->nseq * b->v_heads + 8;
  if (slots * b->k_heads >= 1L << 24 || pairs * (b->value_dim / 16) >= 1L << 23) return 0;
  return slots * b->v_heads * (delta ? ChunkWork<true>::bytes : ChunkWork<false>::bytes);
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

struct Bytes {
  const void* at;
  long n;
};
static bool bytes_meet(Bytes a, Bytes b) {
  return a.n > 0 && b.n > 0 && (const char*)a.at < (const char*)b.at + b.n && (const char*)b.at < (const char*)a.at + a.n;
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
  return linear_work(batch, delta != 0);
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
  const long need = linear_work(batch, d_beta != nullptr);
  const bool chunks = need > 0 && d_work;
  if (chunks && (work_bytes < need || !aligned16(d_work))) return (int)hipErrorInvalidValue;
  // the states and the workspace are written: nothing else of the call may lie in them
  const long state_bytes = 4L * batch->num_states * batch->v_heads * batch->key_dim * batch->value_dim;
  const Bytes states{d_states, state_bytes}, work{d_work, chunks ? need : 0};
  const Bytes lists[] = {{batch->offsets, 4L * (nseq + 1)}, {batch->slots, 4L * nseq}, {batch->source, batch->source ? 4L * nseq : 0}};
  if (bytes_meet(states, work)) return (int)hipErrorInvalidValue;
  for (const Bytes& list : lists)
    if (bytes_meet(list, states) || bytes_meet(list, work)) return (int)hipErrorInvalidValue;
  if (tokens > 0) {
    const qhip_rows* all[] = {q, k, v, out};
    for (const qhip_rows* r : all)  // (a chunk's offsets are 32 bits)
      if (!rows_ok(r, size) || (tokens > 1 && r->token_stride > 1 << 23)) return (int)hipErrorInvalidValue;
    if (!d_log_decay ||
        ((uintptr_t)d_log_decay & 3u) || decay_stride < 0 || ((uintptr_t)d_beta & 3u) || beta_stride < 0)
      return (int)hipErrorInvalidValue;
    const auto meets = [&](const qhip_rows* rows, int heads, int dim, Bytes b) { return rows_meet(rows, tokens, heads, dim, size, b.at, b.n); };
    if (!rows_apart(out, tokens, batch->v_heads, batch->value_dim) || meets(out, batch->v_heads, batch->value_dim, states) ||
        meets(out, batch->v_heads, batch->value_dim, work))
      return (int)hipErrorInvalidValue;
    for (const Bytes& list : lists)
      if (meets(out, batch->v_heads, batch->value_dim, list)) return (int)hipErrorInvalidValue;
    const Bytes numbers[] = {{d_log_decay, 4 * ((tokens - 1) * decay_stride + batch->v_heads)},
                             {d_beta, d_beta ? 4 * ((tokens - 1) * beta_stride + batch->v_heads) : 0}};
    for (const Bytes& n : numbers)
      if (bytes_meet(n, states) || bytes_meet(n, work)) return (int)hipErrorInvalidValue;
    const qhip_rows* read[] = {q, k, v};
    const int heads[] = {batch->k_heads, batch->k_heads, batch->v_heads}, dims[] = {batch->key_dim, batch->key_dim, batch->value_dim};
    for (int i = 0; i < 3; ++i)
      if (rows_overlap(out, batch->v_heads, batch->value_dim, read[i], heads[i], dims[i], tokens, size) ||
          meets(read[i], heads[i], dims[i], states) || meets(read[i], heads[i], dims[i], work))
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
  // Without a workspace every sequence goes token by token.  Beside chunks short sequences do:
  // how many new tokens each has stands on the device, so both forms are launched always
  // (without a short one the first is idle, 5 us; rows for max_new tokens of every sequence
  // say nothing, a captured step has them whatever comes: 64 single tokens of 16 f32 heads in
  // rows for 64 each 50 us, in chunks 201).
  a.few = chunks ? kFew : 0x7FFFFFFF;
  a.work = (uint8_t*)d_work;
  hipStream_t st = (hipStream_t)stream;
  if (type == QHIP_TT_F32) launch_linear<float>(a, batch->key_dim, chunks, st);
  else if (type == QHIP_TT_F16) launch_linear<f16_t>(a, batch->key_dim, chunks, st);
  else launch_linear<bf16_t>(a, batch->key_dim, chunks, st);
  return (int)hipGetLastError();
}
