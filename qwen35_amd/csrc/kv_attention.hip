// kv_attention.hip -- attention over the 8-bit key/value cache.
//
// Two kernels, each for its own sequences of a batch: those of a few rows, whose
// cost is reading the codes, and those of many, whose cost is the products.
#include "kv_internal.hpp"
#include "qhip_device.hpp"
#include "qhip_internal.hpp"

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
  int type, group, few_tokens;  // group: query heads of a key head; sequences of up to few_tokens new tokens are few rows
  bool q_vec, out_vec;          // rows that 16-byte accesses may touch
  // the cut of long sequences: off, or items aimed for, fewest key units of one,
  // bound of a sequence's units, rows of a chunk's partial results
  bool cut;
  int target, least, max_units, max_chunks, rows;
  long slots;  // chunks that the workspace holds
  unsigned* counters;
  float* partial;
};

// ---- sequences of a few rows: the cache streamed once ------------------------------
//
// The rows of a sequence are its new tokens' query heads of one key head (row =
// token * G + head of the group), up to 64 in tiles of 16.  The work is one
// pass over the codes, 2 D bytes a key, so the kernel is built to keep loads in
// flight and never puts a code anywhere but in a register:
//
//   S^T = K Q^T   16 keys x 16 rows a v_mfma_f32_16x16x32_f16; lane 16 g + i
//                 loads 16-byte pieces of key i, whose dimensions (64 j + 16 g
//                 ..+15) the query fragment has in the same order
//   O^T = V^T P^T the accumulator of S^T (lane 16 g + r: row r, keys 4 g ..+3
//                 of each of two tiles) is P's operand as it stands; lane 16 g +
//                 i loads dimensions i D/16 ..+(D/16-1) of just those eight
//                 keys, whole 16-lane rows contiguous, and picks a dimension's
//                 eight codes with byte permutes
//
// so that a row's maximum, sum and output all stay in the four lanes 16 g + r.
// Codes become f16 exactly: (code + 128) as a subnormal is (code + 128) 2^-24,
// and one packed fma makes it code * 2^-9.  Queries are scaled by a power of two
// per row to below 2^14 and f32 ones split into two f16 parts (22 bits); softmax
// weights are scaled to 2^14 and, for f32 rows, split alike.  f16 and bf16 rows
// take weights of 11 bits: their outputs are rounded to 11 and 8.  A block's key
// scale multiplies the scores; its value scale, relative to the largest's power
// of two, the weights.
//
// A workgroup's four waves take steps of 32 keys in turn (one, two or four row
// tiles share a step's waves) and are merged in LDS.  Long sequences are cut
// into chunks over workgroups; the chunk length follows from all sequences'
// lengths, so that ragged batches spread evenly, and the last workgroup of a
// sequence's key head joins the partial results in order.

typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 h16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kFewRows = 64;         // most rows of a sequence's key head
constexpr long kCountBytes = 32768;
constexpr int kMaxCut = kCountBytes / 4;  // most row tiles that are cut
constexpr float kCodeScale = 0x1p9f;  // codes are held as code * 2^-9
constexpr float kMinusInf = -INFINITY;

// pairs of codes (bytes 0 and 2 of p, biased by 128) as f16, times 2^-9
__device__ __forceinline__ h16x2 codes2(uint32_t p) {
  return __builtin_elementwise_fma(__builtin_bit_cast(h16x2, p), h16x2{(_Float16)32768.0f, (_Float16)32768.0f},
                                   h16x2{(_Float16)-0.25f, (_Float16)-0.25f});
}
// eight codes of two dwords (biased) in order
__device__ __forceinline__ h16x8 codes8(uint32_t a, uint32_t b) {
  const h16x2 p0 = codes2(__builtin_amdgcn_perm(0u, a, 0x0C010C00u)), p1 = codes2(__builtin_amdgcn_perm(0u, a, 0x0C030C02u));
  const h16x2 p2 = codes2(__builtin_amdgcn_perm(0u, b, 0x0C010C00u)), p3 = codes2(__builtin_amdgcn_perm(0u, b, 0x0C030C02u));
  return h16x8{p0[0], p0[1], p1[0], p1[1], p2[0], p2[1], p3[0], p3[1]};
}
// byte B of two dwords (biased)
template <int B>
__device__ __forceinline__ h16x2 codes_of(uint32_t a, uint32_t b) {
  return codes2(__builtin_amdgcn_perm(b, a, 0x0C000C00u | (unsigned)B | ((4u + B) << 16)));
}

// maximum and sum over the four lanes of a row (lanes r, r + 16, r + 32, r + 48)
__device__ __forceinline__ float row_max(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float row_sum(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

__device__ __forceinline__ int wave_sum(int v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d, 64);
  return v;
}
__device__ __forceinline__ int wave_scan(int v, int lane) {  // inclusive
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int o = __shfl_up(v, d, 64);
    if (lane >= d) v += o;
  }
  return v;
}

struct FewSeq {
  int n, len, lo, units;  // rows of queries (0: not one of these sequences), tokens, first key, 32-key units to plan for
};
__device__ __forceinline__ FewSeq few_seq(const KvAttnArgs& a, int i) {
  FewSeq s{0, 0, 0, 0};
  if (i >= a.nseq) return s;
  const int n = a.offsets[i + 1] - a.offsets[i];
  if (n <= 0 || n > a.few_tokens) return s;
  s.n = n;
  s.len = max(a.kv_lens[i], 0);
  if (a.causal && a.window > 0) s.lo = max(0, s.len - n - a.window + 1) & ~31;
  s.units = min(max(s.len - s.lo + 31, 0) >> 5, a.max_units);
  return s;
}

// The item of a workgroup: key head, sequence and chunk.
struct FewItem {
  int seq, head, chunk, chunks, slot;  // slot: of the first chunk's partial results
  FewSeq s;
};
__device__ __forceinline__ bool few_item(const KvAttnArgs& a, int lane, FewItem& it) {
  const int at = blockIdx.x / a.kv_heads;
  it.head = blockIdx.x - at * a.kv_heads;
  int unit = 0x7FFFFFFF;
  FewSeq s = few_seq(a, lane);
  if (a.cut) {
    int total = s.units;
    for (int i = 64 + lane; i - lane < a.nseq; i += 64) total += few_seq(a, i).units;
    total = wave_sum(total);
    // about `target` items in all, none of fewer than `least` units
    unit = max(a.least, (int)(((long)total * a.kv_heads + a.target - 1) / a.target));
  }
  int items = 0, slots = 0;
  for (int i0 = 0; i0 < a.nseq; i0 += 64) {
    if (i0) s = few_seq(a, i0 + lane);
    const int c = s.n ? min(a.max_chunks, max(1, (int)(((long)s.units + unit - 1) / unit))) : 0, cut = c > 1 ? c : 0;
    const int ci = wave_scan(c, lane), cs = wave_scan(cut, lane);
    const int all = __shfl(ci, 63, 64);
    if (at < items + all) {
      const int owner = __builtin_ctzll(__ballot(items + ci > at));
      it.seq = i0 + owner;
      it.chunks = __shfl(c, owner, 64);
      it.chunk = at - (items + __shfl(ci, owner, 64) - it.chunks);
      it.slot = (slots + __shfl(cs, owner, 64) - it.chunks) * a.kv_heads + it.head * it.chunks;
      it.s = FewSeq{__shfl(s.n, owner, 64), __shfl(s.len, owner, 64), __shfl(s.lo, owner, 64), __shfl(s.units, owner, 64)};
      return true;
    }
    items += all;
    slots += __shfl(cs, 63, 64);
  }
  return false;
}

// eight query values from d on as f32
__device__ __forceinline__ void load_q8(const void* q, long at, int type, bool vec, float* v) {
  if (type == QHIP_TT_F32) {
    const Raw8<float> r = vec ? load8<float, true>((const float*)q + at) : load8<float, false>((const float*)q + at);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = r.e[i];
  } else if (type == QHIP_TT_F16) {
    const Raw8<f16_t> r = vec ? load8<f16_t, true>((const f16_t*)q + at) : load8<f16_t, false>((const f16_t*)q + at);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)r.e[i];
  } else {
    const Raw8<bf16_t> r = vec ? load8<bf16_t, true>((const bf16_t*)q + at) : load8<bf16_t, false>((const bf16_t*)q + at);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)r.e[i];
  }
}
__device__ __forceinline__ void store1(void* out, long at, int type, float v) {
  if (type == QHIP_TT_F32) ((float*)out)[at] = v;
  else if (type == QHIP_TT_F16) ((f16_t*)out)[at] = (f16_t)v;
  else ((bf16_t*)out)[at] = (bf16_t)v;
}
// N (a power of two) consecutive values, in pieces of up to 16 bytes where vec
template <typename T, int N>
__device__ __forceinline__ void store_pieces(T* out, const float* v) {
  constexpr int P = N * sizeof(T) < 16 ? N : 16 / sizeof(T);
  typedef T piece __attribute__((ext_vector_type(P)));
#pragma unroll
  for (int i = 0; i < N; i += P) {
    piece x;
#pragma unroll
    for (int j = 0; j < P; ++j) x[j] = (T)v[i + j];
    *(piece*)(out + i) = x;
  }
}
template <int N>
__device__ __forceinline__ void store_n(void* out, long at, int type, bool vec, const float* v) {
  if (!vec) {
#pragma unroll
    for (int i = 0; i < N; ++i) store1(out, at + i, type, v[i]);
  } else if (type == QHIP_TT_F32) {
    store_pieces<float, N>((float*)out + at, v);
  } else if (type == QHIP_TT_F16) {
    store_pieces<f16_t, N>((f16_t*)out + at, v);
  } else {
    store_pieces<bf16_t, N>((bf16_t*)out + at, v);
  }
}

// power of two of a value scale (a zero or a NaN has none)
constexpr int kNoScale = -1000;
__device__ __forceinline__ int scale_exp(float v) { return fabsf(v) > 0.0f ? __builtin_amdgcn_frexp_expf(v) : kNoScale; }

// log(sum e^s) of a row whose maximum and sum are in powers of two
__device__ __forceinline__ float row_lse(float m, float l) {
  return l == 0.0f ? kMinusInf : (m + __builtin_log2f(l)) * 0.693147180559945309f;
}

// what e^-(m - M) leaves of a part whose maximum is m (both may be -infinity)
__device__ __forceinline__ float weight_of(float m, float top) { return m == top ? 1.0f : __builtin_amdgcn_exp2f(m - top); }

// ---- joining the chunks of a sequence's rows ----------------------------------------
//
// A chunk's partial results are `rows` x D outputs of its own keys, then each
// row's maximum m and sum l, `stride` floats in all, stored and loaded through
// to the agent's point of coherence (sc1: sk_store's and sk_load's policy, 16
// bytes at a time).  Every chunk adds one to the tile's counter; the last one
// joins all in chunk order, so the result does not depend on which was last.
constexpr int kSc1 = 16;  // cache policy of a buffer access: sc1

__device__ __forceinline__ __amdgpu_buffer_rsrc_t part_rsrc(float* p, long floats) {
  return __builtin_amdgcn_make_buffer_rsrc(p, 0, (int)(4 * floats), 0x00027000);  // raw, 32-bit, bounds-checked
}
// N (2, 4, 8 or 16) consecutive values from float `at` on
template <int N>
__device__ __forceinline__ void part_store(__amdgpu_buffer_rsrc_t r, int at, const float* v) {
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    if constexpr (N == 2)
      __builtin_amdgcn_raw_buffer_store_b64(kv_u32x2{__float_as_uint(v[0]), __float_as_uint(v[1])}, r, 4 * at, 0, kSc1);
    else
      __builtin_amdgcn_raw_buffer_store_b128(kv_u32x4{__float_as_uint(v[i]), __float_as_uint(v[i + 1]), __float_as_uint(v[i + 2]),
                                                      __float_as_uint(v[i + 3])}, r, 4 * (at + i), 0, kSc1);
  }
}

// LDS of a join: m (then weights) and l of `rows` x `chunks`, 1 / sum of each
// row, and 4 KB of sums
constexpr int kJoinLds = 16384;
constexpr int kJoinPairs = (kJoinLds - 4096 - 4 * 128) / 8;  // most rows x chunks

// All 256 threads: the rows seq_row .. seq_row + count of key head `head`.
template <int D>
__device__ __forceinline__ void join_rows(const KvAttnArgs& a, float* lds, __amdgpu_buffer_rsrc_t parts, int stride, int rows,
                                          int count, int chunks, int first_token, int seq_row, int head) {
  const int tid = threadIdx.x;
  float* s_acc = lds;               // [256][4]
  float* s_inv = lds + 1024;        // [128]
  float* s_m = lds + 1024 + 128;    // [chunks][count]
  float* s_l = s_m + chunks * count;
  for (int i = tid; i < chunks * count; i += 256) {
    const int c = i / count, r = i - c * count;
    const kv_u32x2 x = __builtin_amdgcn_raw_buffer_load_b64(parts, 4 * (c * stride + rows * D + 2 * r), 0, kSc1);
    s_m[i] = __uint_as_float(x[0]);
    s_l[i] = __uint_as_float(x[1]);
  }
  __syncthreads();
  {
    int team = 64;  // lanes of a row
    while (team * count > 256) team >>= 1;
    const int r = tid / team, tl = tid & (team - 1);
    float top = kMinusInf, sum = 0.0f;
    if (r < count)
      for (int c = tl; c < chunks; c += team) top = fmaxf(top, s_m[c * count + r]);
    for (int d = 1; d < team; d <<= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
    if (r < count)
      for (int c = tl; c < chunks; c += team) {
        const float f = weight_of(s_m[c * count + r], top) * s_l[c * count + r];
        s_m[c * count + r] = f;
        sum += f;
      }
    for (int d = 1; d < team; d <<= 1) sum += __shfl_xor(sum, d, 64);
    if (r < count && tl == 0) {
      s_inv[r] = sum == 0.0f ? 0.0f : 1.0f / sum;
      const int tok = (seq_row + r) / a.group, t = first_token + tok, qh = head * a.group + (seq_row + r - tok * a.group);
      if (a.lse && t >= 0 && t < a.tokens) a.lse[(long)t * a.q_heads + qh] = row_lse(top, sum);
    }
  }
  __syncthreads();
  // four values a thread; with fewer than 256 of them, slices of the chunks
  const int pieces = count * (D / 4), slices = pieces < 256 ? 256 / pieces : 1;
  for (int e0 = 0; e0 < pieces; e0 += 256) {
    const int sl = slices > 1 ? tid / pieces : 0, e = slices > 1 ? tid - sl * pieces : e0 + tid;
    const int r = e / (D / 4);
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    if (e < pieces && sl < slices)
      for (int c0 = sl; c0 < chunks; c0 += 8 * slices) {
        kv_u32x4 x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)  // past the last chunk: out of the buffer's bounds, 0
          x[j] = __builtin_amdgcn_raw_buffer_load_b128(parts, 4 * ((c0 + j * slices) * stride + 4 * e), 0, kSc1);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int c = c0 + j * slices;
          const float f = c < chunks ? s_m[c * count + r] : 0.0f;
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[i] += f * __uint_as_float(x[j][i]);
        }
      }
    if (slices > 1) {
      ((f32x4*)s_acc)[tid] = acc;
      __syncthreads();
      if (sl == 0)
        for (int k = 1; k < slices; ++k) acc += ((f32x4*)s_acc)[k * pieces + e];
    }
    const int tok = (seq_row + r) / a.group, t = first_token + tok, qh = head * a.group + (seq_row + r - tok * a.group);
    if (e < pieces && sl == 0 && t >= 0 && t < a.tokens) {
      const float inv = s_inv[r], v[4] = {acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv};
      store_n<4>(a.out, (long)t * a.out_token + (long)qh * a.out_head + 4 * (e % (D / 4)), a.type, a.out_vec, v);
    }
  }
}

// SPLIT 2: f32 rows, queries and weights in two f16 parts each
template <int D, int SPLIT>
__global__ __launch_bounds__(256, D == 256 ? 2 : D == 128 ? 3 : 4) void k_kv_attention_few(KvAttnArgs a) {
  constexpr int J = D / 64, C = D / 16, W = D / 64;  // 64-dimension pieces, output tiles, dwords of a value load
  constexpr int R = C * 4 * 64;  // floats of a wave's output
  __shared__ __attribute__((aligned(16))) float s_o[2 * R > kJoinLds / 4 ? 2 * R : kJoinLds / 4];
  __shared__ float s_m[2][64], s_l[2][64];
  __shared__ int s_e[2][64];
  const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  FewItem it;
  if (!few_item(a, lane, it)) return;  // all four waves alike
  const int seq = __builtin_amdgcn_readfirstlane(it.seq), n = __builtin_amdgcn_readfirstlane(it.s.n);
  const int len = __builtin_amdgcn_readfirstlane(it.s.len), lo = __builtin_amdgcn_readfirstlane(it.s.lo);
  const int chunks = __builtin_amdgcn_readfirstlane(it.chunks), chunk = __builtin_amdgcn_readfirstlane(it.chunk);
  const int head = __builtin_amdgcn_readfirstlane(it.head);
  const int rows = n * a.group, tiles = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
  const int units = max(0, len - lo + 31) >> 5;
  const int key0 = lo + 32 * (int)((long)units * chunk / chunks);
  const int key1 = min(len, lo + 32 * (int)((long)units * (chunk + 1) / chunks));
  const int part = wave / tiles, parts = 4 / tiles;
  const int row = (wave % tiles) * 16 + r16;  // this lane's row
  const bool own_row = row < rows;
  const int tok = own_row ? row / a.group : 0, p = len - n + tok;
  const int t = a.offsets[seq] + tok, qh = head * a.group + (row - tok * a.group);
  const bool live = own_row && t >= 0 && t < a.tokens;
  const int vis_hi = a.causal ? p + 1 : len, vis_lo = a.causal && a.window > 0 ? p - a.window + 1 : 0;
  // keys that every row of the sequence sees
  const int all_hi = a.causal ? len - n + 1 : len, all_lo = a.causal && a.window > 0 ? len - a.window : 0;

  // the row's queries, scaled by a power of two
  h16x8 qh_[J][2], ql_[SPLIT == 2 ? J : 1][2];
  float c_row;
  {
    float v[J][2][8], top = 0.0f;
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (live)
          load_q8(a.q, (long)t * a.q_token + (long)qh * a.q_head + 64 * j + 16 * g + 8 * h, a.type, a.q_vec, v[j][h]);
        else
#pragma unroll
          for (int i = 0; i < 8; ++i) v[j][h][i] = 0.0f;
      }
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(v[j][h][i]));
    const int e = 14 - __builtin_amdgcn_frexp_expf(row_max(top));
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float x = __builtin_ldexpf(v[j][h][i], e);
          const _Float16 hi = (_Float16)x;
          qh_[j][h][i] = hi;
          if constexpr (SPLIT == 2) ql_[j][h][i] = (_Float16)(x - (float)hi);
        }
    c_row = __builtin_ldexpf(a.scale * 1.44269504088896341f * kCodeScale, -e);
  }

  f32x4 o[C];
#pragma unroll
  for (int c = 0; c < C; ++c) o[c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float m = kMinusInf, l = 0.0f;
  int ve = kNoScale;  // power of two of the largest value scale that the row has seen: o is in units of 2^(ve - 14 + 9)

  const uint8_t* kc = (const uint8_t*)a.k;
  const uint8_t* vc = (const uint8_t*)a.v;
  const int mask = (1 << a.shift) - 1;
  const uint32_t koff = (uint32_t)(r16 * D + 16 * g), voff = (uint32_t)(4 * g * D + r16 * C);
  for (int s0 = part; key0 + 32 * s0 < key1; s0 += 32 * parts) {
    // lane i: tile i & 1 of this wave's step i / 2
    const int mine = key0 + 32 * (s0 + parts * (lane >> 1)) + 16 * (lane & 1);
    int id = 0;
    float ks = 0.0f, vs = 0.0f;
    if (mine < key1) {
      const int b = mine >> a.shift;
      id = b < a.width ? a.table[(long)seq * a.width + b] : -1;
      const bool in = (unsigned)id < (unsigned)a.num_blocks;
      id = in ? id : 0;
      ks = a.k_scale[(long)id * a.kv_heads + head];
      vs = a.v_scale[(long)id * a.kv_heads + head];
      ks = in && finite_bits(__float_as_uint(ks)) ? ks : __builtin_nanf("");
      vs = in && finite_bits(__float_as_uint(vs)) ? vs : __builtin_nanf("");
    }
    const int steps = min(32, (key1 - key0 - 32 * s0 + 32 * parts - 1) / (32 * parts));

    kv_u32x4 kr[2][J];
    uint32_t vr[8][W];
    auto tile_at = [&](int i) {  // byte offset of tile i's first code
      const long b = __builtin_amdgcn_readlane(id, i);
      const int first = (key0 + 32 * (s0 + parts * (i >> 1)) + 16 * (i & 1)) & mask;
      return ((b * a.kv_heads + head) << a.shift | first) * D;
    };
    auto load_k = [&](int st) {
#pragma unroll
      for (int tt = 0; tt < 2; ++tt) {
        const uint8_t* b = kc + tile_at(2 * st + tt);
#pragma unroll
        for (int j = 0; j < J; ++j) kr[tt][j] = *(const kv_u32x4*)(b + koff + 64 * j);
      }
    };
    auto load_v = [&](int st) {
#pragma unroll
      for (int tt = 0; tt < 2; ++tt) {
        const uint8_t* b = vc + tile_at(2 * st + tt);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t* x = (const uint32_t*)(b + voff + i * D);
          if constexpr (W == 4) {
            const kv_u32x4 y = *(const kv_u32x4*)x;
#pragma unroll
            for (int w = 0; w < 4; ++w) vr[4 * tt + i][w] = y[w];
          } else if constexpr (W == 2) {
            const kv_u32x2 y = *(const kv_u32x2*)x;
            vr[4 * tt + i][0] = y[0];
            vr[4 * tt + i][1] = y[1];
          } else {
            vr[4 * tt + i][0] = x[0];
          }
        }
      }
    };
    load_k(0);
    load_v(0);
    for (int st = 0; st < steps; ++st) {
      const int key = key0 + 32 * (s0 + parts * st);
      float s[2][4];
#pragma unroll
      for (int tt = 0; tt < 2; ++tt) {
        f32x4 hi = {0.0f, 0.0f, 0.0f, 0.0f}, low = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const kv_u32x4 x = kr[tt][j] ^ 0x80808080u;
          const h16x8 k0 = codes8(x[0], x[1]), k1 = codes8(x[2], x[3]);
          hi = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qh_[j][0], hi, 0, 0, 0);
          hi = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, qh_[j][1], hi, 0, 0, 0);
          if constexpr (SPLIT == 2) {
            low = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, ql_[j][0], low, 0, 0, 0);
            low = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, ql_[j][1], low, 0, 0, 0);
          }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) s[tt][r] = SPLIT == 2 ? hi[r] + low[r] : hi[r];
      }
      if (st + 1 < steps) load_k(st + 1);
      const float c0 = c_row * __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ks), 2 * st));
      const float c1 = c_row * __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ks), 2 * st + 1));
      const float v0 = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(vs), 2 * st));
      const float v1 = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(vs), 2 * st + 1));
      float top = kMinusInf;
      const bool edge = key < all_lo || key + 32 > min(all_hi, key1);  // some row does not see some key
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[0][r] *= c0;
        s[1][r] *= c1;
      }
      int e0 = scale_exp(v0), e1 = scale_exp(v1);
      if (edge) {
        const int end = min(vis_hi, key1);
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int j = key + 16 * tt + 4 * g + r;
            if (j < vis_lo || j >= end) s[tt][r] = kMinusInf;
          }
        if (key >= end || key + 16 <= vis_lo) e0 = kNoScale;
        if (key + 16 >= end || key + 32 <= vis_lo) e1 = kNoScale;
      }
      e0 = max(ve, max(e0, e1));
#pragma unroll
      for (int r = 0; r < 4; ++r) top = fmaxf(top, fmaxf(s[0][r], s[1][r]));
      top = fmaxf(m, row_max(top));
      if (__any(top != m || e0 != ve)) {
        const float f = weight_of(m, top), fo = __builtin_ldexpf(f, ve - e0);
        l *= f;
#pragma unroll
        for (int c = 0; c < C; ++c) o[c] *= fo;
        m = top;
        ve = e0;
      }
      const float w0 = __builtin_ldexpf(v0, 14 - ve), w1 = __builtin_ldexpf(v1, 14 - ve);
      h16x8 ph, pl;
      float sum = 0.0f;
#pragma unroll
      for (int tt = 0; tt < 2; ++tt)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          // m is -infinity where the row has seen nothing yet; what it does not
          // see has weight 0 whatever its block's scales are
          float e = __builtin_amdgcn_exp2f(s[tt][r] - m), x = e * (tt ? w1 : w0);
          if (edge) {
            const int j = key + 16 * tt + 4 * g + r;
            if (j < vis_lo || j >= vis_hi || j >= key1) e = x = 0.0f;
          }
          sum += e;
          const _Float16 hi = (_Float16)x;
          ph[4 * tt + r] = hi;
          if constexpr (SPLIT == 2) pl[4 * tt + r] = (_Float16)(x - (float)hi);
        }
      l += sum;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        uint32_t x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = vr[i][w] ^ 0x80808080u;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          h16x2 y[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            y[i] = b == 0 ? codes_of<0>(x[2 * i], x[2 * i + 1]) : b == 1 ? codes_of<1>(x[2 * i], x[2 * i + 1])
                 : b == 2 ? codes_of<2>(x[2 * i], x[2 * i + 1]) : codes_of<3>(x[2 * i], x[2 * i + 1]);
          const h16x8 v8 = {y[0][0], y[0][1], y[1][0], y[1][1], y[2][0], y[2][1], y[3][0], y[3][1]};
          o[4 * w + b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v8, ph, o[4 * w + b], 0, 0, 0);
          if constexpr (SPLIT == 2) o[4 * w + b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v8, pl, o[4 * w + b], 0, 0, 0);
        }
      }
      if (st + 1 < steps) load_v(st + 1);
    }
  }
  l = row_sum(l);

  // merge the waves that share a row tile: the upper half of the parts into the lower
  for (int half = parts / 2; half >= 1; half >>= 1) {
    const int slot = wave - half * tiles;  // waves [half * tiles, 2 half * tiles) give
    if (slot >= 0 && slot < half * tiles) {
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r) s_o[slot * R + (4 * c + r) * 64 + lane] = o[c][r];
      s_m[slot][lane] = m;
      s_l[slot][lane] = l;
      s_e[slot][lane] = ve;
    }
    __syncthreads();
    if (wave < half * tiles) {
      const float m2 = s_m[wave][lane], top = fmaxf(m, m2);
      const int ve2 = s_e[wave][lane], e = max(ve, ve2);
      const float f1 = weight_of(m, top), f2 = weight_of(m2, top);
      const float g1 = __builtin_ldexpf(f1, ve - e), g2 = __builtin_ldexpf(f2, ve2 - e);
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[c][r] = o[c][r] * g1 + s_o[wave * R + (4 * c + r) * 64 + lane] * g2;
      l = l * f1 + s_l[wave][lane] * f2;
      m = top;
      ve = e;
    }
    __syncthreads();
  }

  // a row that sees nothing: 0 and -infinity (l is 0); NaN stays
  const float norm = l == 0.0f ? 0.0f : 1.0f / l;
  if (chunks == 1) {
    if (wave < tiles && live) {
      const long at = (long)t * a.out_token + (long)qh * a.out_head + (4 * g) * C;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float v[C];
#pragma unroll
        for (int c = 0; c < C; ++c) v[c] = __builtin_ldexpf(o[c][r] * norm, ve - 14 + 9);
        store_n<C>(a.out, at + r * C, a.type, a.out_vec, v);
      }
      if (a.lse && g == 0) a.lse[(long)t * a.q_heads + qh] = row_lse(m, l);
    }
    return;
  }
  // partial results of the chunk: out [rows][D] (of its own keys), then m and l
  if (it.slot + chunks > a.slots) return;  // offsets or lengths that are none
  const int stride = a.rows * (D + 2);
  const __amdgpu_buffer_rsrc_t parts_at = part_rsrc(a.partial + (long)it.slot * stride, (long)chunks * stride);
  if (wave < tiles && own_row) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float v[C];
#pragma unroll
      for (int c = 0; c < C; ++c) v[c] = __builtin_ldexpf(o[c][r] * norm, ve - 14 + 9);
      part_store<C>(parts_at, chunk * stride + row * D + (4 * g + r) * C, v);
    }
    const float stat[2] = {m, l};
    if (g == 0) part_store<2>(parts_at, chunk * stride + a.rows * D + 2 * row, stat);
  }
  unsigned* count = a.counters + (long)seq * a.kv_heads + head;
  if (!sk_arrive(count, (unsigned)chunks)) return;
  sk_reset(count);
  join_rows<D>(a, s_o, parts_at, stride, a.rows, rows, chunks, a.offsets[seq], 0, head);
}

// ---- sequences of many rows: key tiles staged in LDS ---------------------------------
//
// A workgroup takes kManyRows rows of one key head (row = token * G + head of
// the group, so that the heads of a group share every key), a wave 32 of them.
// Per tile of 64 keys the codes are read once from memory, turned into f16 and
// laid down in LDS as v_mfma_f32_32x32x16_f16 wants them: keys row by row
// (16-byte pieces of 8 dimensions), values dimension by dimension (16-byte
// pieces of the 8 keys that a lane's weights belong to), both with the piece
// index xor-ed so that eight lanes hit eight pieces of a 128-byte row of banks.
// S^T and O^T as for few rows: lane 32 h + r holds row r; keys 8 i + 4 h ..+3 of
// a 32-key half are its scores and its half of the weights' operand, and output
// tile c holds dimensions i D/32 + c.  The next tile's codes are in flight in
// registers while this one is multiplied.

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kManyRows = 128;
constexpr int kManyKeys = 64;


struct ManySeq {
  int n, len, tiles, units;  // new tokens (0: not one of these sequences), tokens, row tiles, key tiles to plan for
};
__device__ __forceinline__ ManySeq many_seq(const KvAttnArgs& a, int i) {
  ManySeq s{0, 0, 0, 0};
  if (i >= a.nseq) return s;
  const int n = a.offsets[i + 1] - a.offsets[i];
  if (n <= a.few_tokens || n > a.tokens) return s;
  s.n = n;
  s.len = max(a.kv_lens[i], 0);
  s.tiles = (int)(((long)(min(a.offsets[i + 1], a.tokens) - a.offsets[i]) * a.group + kManyRows - 1) / kManyRows);
  if (s.tiles <= 0) return ManySeq{0, 0, 0, 0};
  int keys = s.len;
  if (a.causal && a.window > 0) keys = (int)min((long)keys, (long)a.window + kManyRows / a.group + 2 * kManyKeys);
  s.units = min((keys + kManyKeys - 1) / kManyKeys, a.max_units);
  return s;
}
struct ManyItem {
  int seq, head, tile, chunk, chunks, slot, counter;
  ManySeq s;
};
__device__ __forceinline__ bool many_item(const KvAttnArgs& a, int lane, ManyItem& it) {
  const int at = blockIdx.x / a.kv_heads;
  it.head = blockIdx.x - at * a.kv_heads;
  int unit = 0x7FFFFFFF;
  ManySeq s = many_seq(a, lane);
  if (a.cut) {
    int total = s.tiles * s.units;
    for (int i = 64 + lane; i - lane < a.nseq; i += 64) {
      const ManySeq x = many_seq(a, i);
      total += x.tiles * x.units;
    }
    total = wave_sum(total);
    unit = max(a.least, (int)(((long)total * a.kv_heads + a.target - 1) / a.target));
  }
  int items = 0, slots = 0, tiles = 0;
  for (int i0 = 0; i0 < a.nseq; i0 += 64) {
    if (i0) s = many_seq(a, i0 + lane);
    const int c = min(a.max_chunks, max(1, (int)(((long)s.units + unit - 1) / unit))), n = s.tiles * c, cut = c > 1 ? n : 0;
    const int ci = wave_scan(n, lane), cs = wave_scan(cut, lane), ct = wave_scan(s.tiles, lane);
    const int all = __shfl(ci, 63, 64);
    if (at < items + all) {
      const int owner = __builtin_ctzll(__ballot(items + ci > at));
      it.seq = i0 + owner;
      it.s = ManySeq{__shfl(s.n, owner, 64), __shfl(s.len, owner, 64), __shfl(s.tiles, owner, 64), 0};
      it.chunks = __shfl(c, owner, 64);
      const int local = at - (items + __shfl(ci, owner, 64) - it.s.tiles * it.chunks);
      const int tile = local / it.chunks;
      it.chunk = local - tile * it.chunks;
      it.tile = it.s.tiles - 1 - tile;  // the last rows see the most keys: they begin first
      it.slot = (slots + __shfl(cs, owner, 64) - (it.s.tiles - tile) * it.chunks) * a.kv_heads + it.head * it.chunks;
      it.counter = (tiles + __shfl(ct, owner, 64) - it.s.tiles + it.tile) * a.kv_heads + it.head;
      return true;
    }
    items += all;
    slots += __shfl(cs, 63, 64);
    tiles += __shfl(ct, 63, 64);
  }
  return false;
}

// the 16-byte piece of a value row that holds piece x of dimension `dim`
template <int D>
__device__ __forceinline__ int value_piece(int dim, int x) {
  if constexpr (D == 64) return x ^ (((dim >> 1) ^ (dim >> 4)) & 7);
  else return x ^ ((dim / (D / 32)) & 7);
}

template <int D, int SPLIT>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void k_kv_attention_many(KvAttnArgs a) {
  constexpr int S = D / 16, C = D / 32;      // 16-dimension steps, output tiles
  constexpr int KP = D / 64;                 // 16-byte pieces of a key tile a thread stages
  constexpr int VW = D == 256 ? 2 : 1;       // dwords of a value row a thread stages (8 keys of 4 VW dimensions)
  constexpr int VT = 8 * (D / (4 * VW));     // threads that stage values
  __shared__ __attribute__((aligned(16))) uint8_t s_kv[2 * kManyKeys * D * 2];
  uint8_t *const s_k = s_kv, *const s_v = s_kv + kManyKeys * D * 2;
  static_assert(sizeof(s_kv) >= kJoinLds, "the join's LDS");
  const int tid = threadIdx.x, lane = tid & 63, r32 = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  ManyItem it;
  if (!many_item(a, lane, it)) return;
  const int seq = __builtin_amdgcn_readfirstlane(it.seq), n = __builtin_amdgcn_readfirstlane(it.s.n);
  const int len = __builtin_amdgcn_readfirstlane(it.s.len), head = __builtin_amdgcn_readfirstlane(it.head);
  const int chunks = __builtin_amdgcn_readfirstlane(it.chunks), chunk = __builtin_amdgcn_readfirstlane(it.chunk);
  const int row_first = __builtin_amdgcn_readfirstlane(it.tile) * kManyRows;
  const int rows = (int)min((long)kManyRows, (long)n * a.group - row_first);
  const int first = len - n;  // place of the sequence's first new token
  const bool windowed = a.causal && a.window > 0;
  // the tile's keys, and this chunk's
  const int tok_a = row_first / a.group, tok_b = (row_first + rows - 1) / a.group;
  const int lo = windowed ? max(0, first + tok_a - a.window + 1) & ~(kManyKeys - 1) : 0;
  const int hi = a.causal ? first + tok_b + 1 : len;
  const int all_tiles = max(0, hi - lo + kManyKeys - 1) / kManyKeys;
  const int tile0 = (int)((long)all_tiles * chunk / chunks), tile1 = (int)((long)all_tiles * (chunk + 1) / chunks);
  const int key0 = lo + tile0 * kManyKeys, count = tile1 - tile0;

  // this lane's row, and what the wave's rows see
  const int wrow = wave * 32, row = wrow + r32;
  const bool own_row = row < rows;
  const int tok = own_row ? (row_first + row) / a.group : tok_a, p = first + tok;
  const int t = a.offsets[seq] + tok, qh = head * a.group + (row_first + row - tok * a.group);
  const bool live = own_row && t >= 0 && t < a.tokens;
  const int vis_hi = a.causal ? p + 1 : len, vis_lo = windowed ? p - a.window + 1 : 0;
  const int wtok_a = (row_first + wrow) / a.group, wtok_b = (row_first + min(wrow + 31, rows - 1)) / a.group;
  const bool busy = wrow < rows;
  const int all_hi = a.causal ? first + wtok_a + 1 : len, all_lo = windowed ? first + wtok_b - a.window + 1 : 0;
  const int any_hi = a.causal ? first + wtok_b + 1 : len, any_lo = windowed ? first + wtok_a - a.window + 1 : 0;

  h16x8 q_hi[S], q_lo[SPLIT == 2 ? S : 1];
  float c_row;
  {
    float top = 0.0f;
    const long at = (long)t * a.q_token + (long)qh * a.q_head + 8 * h;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      float v[8] = {};
      if (live) load_q8(a.q, at + 16 * s, a.type, a.q_vec, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(v[i]));
    }
    const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
    const int e = 14 - __builtin_amdgcn_frexp_expf(fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1])));
#pragma unroll
    for (int s = 0; s < S; ++s) {
      float v[8] = {};
      if (live) load_q8(a.q, at + 16 * s, a.type, a.q_vec, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = __builtin_ldexpf(v[i], e);
        q_hi[s][i] = (_Float16)x;
        if constexpr (SPLIT == 2) q_lo[s][i] = (_Float16)(x - (float)q_hi[s][i]);
      }
    }
    c_row = __builtin_ldexpf(a.scale * 1.44269504088896341f * kCodeScale, -e);
  }

  f32x16 o[C];
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[c][i] = 0.0f;
  float m = kMinusInf, l = 0.0f;
  int ve = kNoScale;

  // lane i: the 16-key tile i of a round of 16 key tiles
  struct Info {
    int id;
    float ks, vs;
  };
  auto load_info = [&](int round) {
    Info x{0, 0.0f, 0.0f};
    const int mine = key0 + round * 16 * kManyKeys + 16 * lane;
    if (mine < hi) {
      const int b = mine >> a.shift;
      const int id = b < a.width ? a.table[(long)seq * a.width + b] : -1;
      const bool in = (unsigned)id < (unsigned)a.num_blocks;
      x.id = in ? id : 0;
      x.ks = a.k_scale[(long)x.id * a.kv_heads + head];
      x.vs = a.v_scale[(long)x.id * a.kv_heads + head];
      x.ks = in && finite_bits(__float_as_uint(x.ks)) ? x.ks : __builtin_nanf("");
      x.vs = in && finite_bits(__float_as_uint(x.vs)) ? x.vs : __builtin_nanf("");
    }
    return x;
  };
  const int mask = (1 << a.shift) - 1;
  // staging: pieces of keys (D / 16 a key), then 8 keys of 4 VW dimensions of the values
  const int kkey = tid / (D / 16), kpc = tid % (D / 16);   // first key (a step of 4096 / D further each piece)
  const int vgrp = tid / (D / (4 * VW)), vdim = (tid % (D / (4 * VW))) * 4 * VW;
  // group x of the values' eight: keys 32 (x >> 2) + 16 (x >> 1 & 1) + 4 (x & 1) + {0..3, 8..11}
  const int vkey = 32 * (vgrp >> 2) + 16 * ((vgrp >> 1) & 1) + 4 * (vgrp & 1);
  kv_u32x4 kr[KP];
  uint32_t vr[8][VW];
  auto load_tile = [&](const Info& x, int i) {  // key tile i of the round
    auto at = [&](int key) {  // byte offset of a key's codes
      const long id = __shfl(x.id, 4 * i + (key >> 4), 64);
      return ((id * a.kv_heads + head) << a.shift | ((16 * (4 * i + (key >> 4)) + key0 + (key & 15)) & mask)) * D;
    };
#pragma unroll
    for (int j = 0; j < KP; ++j) kr[j] = *(const kv_u32x4*)((const uint8_t*)a.k + at(kkey + j * (4096 / D)) + 16 * kpc);
    if (VT == 256 || tid < VT) {
      const uint8_t* b = (const uint8_t*)a.v + at(vkey) + vdim;  // all eight keys lie in one 16-key tile
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t* y = (const uint32_t*)(b + (j < 4 ? j : j + 4) * D);
        if constexpr (VW == 2) {
          const kv_u32x2 z = *(const kv_u32x2*)y;
          vr[j][0] = z[0];
          vr[j][1] = z[1];
        } else {
          vr[j][0] = y[0];
        }
      }
    }
  };
  auto store_tile = [&]() {
#pragma unroll
    for (int j = 0; j < KP; ++j) {
      const int key = kkey + j * (4096 / D);
      const kv_u32x4 x = kr[j] ^ 0x80808080u;
      uint8_t* row_at = s_k + key * (D * 2);
      *(h16x8*)(row_at + ((2 * kpc) ^ (key & 7)) * 16) = codes8(x[0], x[1]);
      *(h16x8*)(row_at + ((2 * kpc + 1) ^ (key & 7)) * 16) = codes8(x[2], x[3]);
    }
    if (VT == 256 || tid < VT) {
#pragma unroll
      for (int w = 0; w < VW; ++w) {
        uint32_t x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = vr[j][w] ^ 0x80808080u;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          h16x2 y[4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            y[j] = b == 0 ? codes_of<0>(x[2 * j], x[2 * j + 1]) : b == 1 ? codes_of<1>(x[2 * j], x[2 * j + 1])
                 : b == 2 ? codes_of<2>(x[2 * j], x[2 * j + 1]) : codes_of<3>(x[2 * j], x[2 * j + 1]);
          const int dim = vdim + 4 * w + b;
          *(h16x8*)(s_v + dim * 128 + value_piece<D>(dim, vgrp) * 16) =
              h16x8{y[0][0], y[0][1], y[1][0], y[1][1], y[2][0], y[2][1], y[3][0], y[3][1]};
        }
      }
    }
  };

  Info info = load_info(0), next = load_info(1);
  if (count > 0) load_tile(info, 0);
  for (int i = 0; i < count; ++i) {
    const int ri = i & 15;
    if (ri == 0 && i) {
      info = next;
      next = load_info((i >> 4) + 1);
    }
    __syncthreads();  // the previous tile has been read
    store_tile();
    __syncthreads();
    if (i + 1 < count) {
      if (ri == 15) load_tile(next, 0);
      else load_tile(info, ri + 1);
    }
    const int key = key0 + i * kManyKeys;
#pragma unroll 1
    for (int mt = 0; mt < 2; ++mt) {
      const int kt = key + 32 * mt;
      if (!busy || kt >= any_hi || kt + 32 <= any_lo) continue;  // no row of the wave sees it
      f32x16 s = {}, sl = {};
#pragma unroll
      for (int st = 0; st < S; ++st) {
        const int kk = 32 * mt + r32;
        const h16x8 x = *(const h16x8*)(s_k + kk * (D * 2) + ((2 * st + h) ^ (kk & 7)) * 16);
        s = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, q_hi[st], s, 0, 0, 0);
        if constexpr (SPLIT == 2) sl = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, q_lo[st], sl, 0, 0, 0);
      }
      const int sc = 4 * ri + 2 * mt;
      const float c0 = c_row * __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(info.ks), sc));
      const float c1 = c_row * __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(info.ks), sc + 1));
      const float v0 = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(info.vs), sc));
      const float v1 = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(info.vs), sc + 1));
      const bool edge = kt < all_lo || kt + 32 > all_hi;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = (SPLIT == 2 ? s[r] + sl[r] : s[r]) * (r < 8 ? c0 : c1);
      int e0 = scale_exp(v0), e1 = scale_exp(v1);
      if (edge) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int j = kt + 8 * (r >> 2) + 4 * h + (r & 3);
          if (j < vis_lo || j >= vis_hi) s[r] = kMinusInf;
        }
        if (kt >= vis_hi || kt + 16 <= vis_lo) e0 = kNoScale;
        if (kt + 16 >= vis_hi || kt + 32 <= vis_lo) e1 = kNoScale;
      }
      e0 = max(ve, max(e0, e1));
      float top = s[0];
#pragma unroll
      for (int r = 1; r < 16; ++r) top = fmaxf(top, s[r]);
      const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
      top = fmaxf(m, fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1])));
      if (__any(top != m || e0 != ve)) {
        const float f = weight_of(m, top), fo = __builtin_ldexpf(f, ve - e0);
        l *= f;
#pragma unroll
        for (int c = 0; c < C; ++c) o[c] *= fo;
        m = top;
        ve = e0;
      }
      const float w0 = __builtin_ldexpf(v0, 14 - ve), w1 = __builtin_ldexpf(v1, 14 - ve);
      h16x8 p_hi[2], p_lo[2];
      float sum = 0.0f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float e = __builtin_amdgcn_exp2f(s[r] - m), x = e * (r < 8 ? w0 : w1);
        if (edge) {
          const int j = kt + 8 * (r >> 2) + 4 * h + (r & 3);
          if (j < vis_lo || j >= vis_hi) e = x = 0.0f;
        }
        sum += e;
        const _Float16 y = (_Float16)x;
        p_hi[r >> 3][r & 7] = y;
        if constexpr (SPLIT == 2) p_lo[r >> 3][r & 7] = (_Float16)(x - (float)y);
      }
      l += sum;
#pragma unroll
      for (int st = 0; st < 2; ++st)
#pragma unroll
        for (int c = 0; c < C; ++c) {
          const int dim = r32 * C + c;
          const h16x8 x = *(const h16x8*)(s_v + dim * 128 + value_piece<D>(dim, 4 * mt + 2 * st + h) * 16);
          o[c] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, p_hi[st], o[c], 0, 0, 0);
          if constexpr (SPLIT == 2) o[c] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, p_lo[st], o[c], 0, 0, 0);
        }
    }
  }
  {
    const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
    l = __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
  }
  const float norm = l == 0.0f ? 0.0f : 1.0f / l;
  if (chunks == 1) {
    if (live) {
      const long at = (long)t * a.out_token + (long)qh * a.out_head;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float v[C];
#pragma unroll
        for (int c = 0; c < C; ++c) v[c] = __builtin_ldexpf(o[c][r] * norm, ve - 14 + 9);
        store_n<C>(a.out, at + (8 * (r >> 2) + 4 * h + (r & 3)) * C, a.type, a.out_vec, v);
      }
      if (a.lse && h == 0) a.lse[(long)t * a.q_heads + qh] = row_lse(m, l);
    }
    return;
  }
  if (it.slot + chunks > a.slots || it.counter >= kMaxCut) return;  // offsets or lengths that are none
  constexpr int kStride = kManyRows * (D + 2);
  const __amdgpu_buffer_rsrc_t parts_at = part_rsrc(a.partial + (long)it.slot * kStride, (long)chunks * kStride);
  if (own_row) {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      float v[C];
#pragma unroll
      for (int c = 0; c < C; ++c) v[c] = __builtin_ldexpf(o[c][r] * norm, ve - 14 + 9);
      part_store<C>(parts_at, chunk * kStride + row * D + (8 * (r >> 2) + 4 * h + (r & 3)) * C, v);
    }
    const float stat[2] = {m, l};
    if (h == 0) part_store<2>(parts_at, chunk * kStride + kManyRows * D + 2 * row, stat);
  }
  unsigned* counter = a.counters + it.counter;
  if (!sk_arrive(counter, (unsigned)chunks)) return;
  sk_reset(counter);
  join_rows<D>(a, (float*)s_kv, parts_at, kStride, kManyRows, rows, chunks, a.offsets[seq], row_first, head);
}

template <int SPLIT>
static void launch_few(const KvAttnArgs& a, int dim, unsigned grid, hipStream_t s) {
  if (dim == 64) hipLaunchKernelGGL((k_kv_attention_few<64, SPLIT>), dim3(grid), dim3(256), 0, s, a);
  else if (dim == 128) hipLaunchKernelGGL((k_kv_attention_few<128, SPLIT>), dim3(grid), dim3(256), 0, s, a);
  else hipLaunchKernelGGL((k_kv_attention_few<256, SPLIT>), dim3(grid), dim3(256), 0, s, a);
}

template <int SPLIT>
static void launch_many(const KvAttnArgs& a, int dim, unsigned grid, hipStream_t s) {
  if (dim == 64) hipLaunchKernelGGL((k_kv_attention_many<64, SPLIT>), dim3(grid), dim3(256), 0, s, a);
  else if (dim == 128) hipLaunchKernelGGL((k_kv_attention_many<128, SPLIT>), dim3(grid), dim3(256), 0, s, a);
  else hipLaunchKernelGGL((k_kv_attention_many<256, SPLIT>), dim3(grid), dim3(256), 0, s, a);
}

// 0, hipErrorInvalidValue or QHIP_DECLINE
static int check_batch(const qhip_kv_cache* cache, const qhip_kv_batch* b, int q_heads) {
  const int rc = kv_check_cache(cache);
  if (rc == (int)hipErrorInvalidValue || !b) return (int)hipErrorInvalidValue;
  if (b->nseq < 0 || b->tokens < 0 || b->max_new < 0 || b->max_kv < 0 || b->table_width < 0) return (int)hipErrorInvalidValue;
  if (q_heads <= 0 || q_heads > 65535 || q_heads % cache->kv_heads) return (int)hipErrorInvalidValue;
  return rc;
}

// How one of the two kernels' sequences are cut: grid without and with a cut,
// key units of the longest sequence, items aimed for, fewest units of one, and
// the workspace (0: no cut).
struct AttnPlan {
  int rows, max_units, target, least;
  long grid, cut_grid, work;
};
// `tiles`: bound of the row tiles over all sequences and key heads; a sequence
// that is cut has less than twice units / unit chunks, where a chunk's unit is
// at least a target-th of all units, so the chunks are less than twice target.
static AttnPlan attn_plan(long tiles, int rows, int units, int target, int least, int dim) {
  AttnPlan p{rows, units, target, least, tiles, tiles, 0};
  const long most = (units + least - 1) / least;
  if (tiles > 0 && most > 1 && tiles <= kMaxCut && tiles * units < 0x7FFFFFFFL) {
    p.cut_grid = tiles * most < target + tiles ? tiles * most : target + tiles;
    const long slots = tiles * most < 2L * target ? tiles * most : 2L * target;
    p.work = kCountBytes + slots * rows * (dim + 2) * 4;
  }
  return p;
}
// most new tokens of a few-row sequence
static int few_tokens(const qhip_kv_cache* c, const qhip_kv_batch* b, int q_heads) {
  const int most = kFewRows / (q_heads / c->kv_heads);
  return most < b->max_new ? most : b->max_new;
}
static AttnPlan few_plan(const qhip_kv_cache* c, const qhip_kv_batch* b, int q_heads) {
  const int rows = few_tokens(c, b, q_heads) * (q_heads / c->kv_heads);
  const long tiles = rows ? (long)b->nseq * c->kv_heads : 0;
  return attn_plan(tiles, rows, (int)(((long)b->max_kv + 31) / 32), rows <= 16 ? 1024 : 512, 16, c->head_dim);
}
static AttnPlan many_plan(const qhip_kv_cache* c, const qhip_kv_batch* b, int q_heads) {
  if (b->max_new <= few_tokens(c, b, q_heads)) return AttnPlan{};
  const long tiles = ((long)b->tokens * (q_heads / c->kv_heads) / kManyRows + b->nseq) * c->kv_heads;
  const int target = 512;
  AttnPlan p = attn_plan(tiles, kManyRows, (int)(((long)b->max_kv + kManyKeys - 1) / kManyKeys), target, 8, c->head_dim);
  if (tiles >= 2 * target) p.work = 0;  // enough workgroups as it is
  return p;
}

}  // namespace qhip

using namespace qhip;

extern "C" long qhip_kv_attention_work_bytes(const qhip_kv_cache* cache, const qhip_kv_batch* batch, int q_heads) {
  if (check_batch(cache, batch, q_heads)) return -1;
  const long few = few_plan(cache, batch, q_heads).work, many = many_plan(cache, batch, q_heads).work;
  return few > many ? few : many;
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
  const AttnPlan few = few_plan(cache, batch, q_heads), many = many_plan(cache, batch, q_heads);
  // rows and workgroups are counted in 32 bits
  if (few.grid > 0x7FFFFFFFL || many.grid > 0x7FFFFFFFL || (long)batch->tokens * q_heads > 0x7FFFFFFFL) return (int)hipErrorInvalidValue;
  KvAttnArgs a{(const int8_t*)cache->k, (const int8_t*)cache->v, cache->k_scale, cache->v_scale, batch->offsets,
               batch->kv_lens, batch->table, d_q, d_out, d_lse, q_token_stride, q_head_stride, out_token_stride,
               out_head_stride, batch->nseq, batch->tokens, batch->table_width, kv_block_shift(cache->block_size),
               cache->num_blocks, cache->kv_heads, q_heads, softmax_scale, causal, window, type, q_heads / cache->kv_heads,
               few_tokens(cache, batch, q_heads), kv_rows_aligned(d_q, q_token_stride, q_head_stride, size),
               kv_rows_aligned(d_out, out_token_stride, out_head_stride, size)};
  a.counters = (unsigned*)d_work;
  a.partial = (float*)((char*)d_work + kCountBytes);
  hipStream_t s = (hipStream_t)stream;
  // the two kernels share the workspace: they follow each other on the stream
  // and each leaves the counters at zero
  auto launch = [&](const AttnPlan& p, void (*f32_rows)(const KvAttnArgs&, int, unsigned, hipStream_t),
                    void (*f16_rows)(const KvAttnArgs&, int, unsigned, hipStream_t)) {
    if (p.grid == 0) return;
    a.cut = p.work > 0 && d_work && work_bytes >= p.work;
    a.target = p.target;
    a.least = p.least;
    a.max_units = p.max_units;
    a.max_chunks = kJoinPairs / p.rows;
    a.rows = p.rows;
    a.slots = a.cut ? (p.work - kCountBytes) / ((long)p.rows * (cache->head_dim + 2) * 4) : 0;
    (type == QHIP_TT_F32 ? f32_rows : f16_rows)(a, cache->head_dim, (unsigned)(a.cut ? p.cut_grid : p.grid), s);
  };
  launch(few, launch_few<2>, launch_few<1>);
  launch(many, launch_many<2>, launch_many<1>);
  return (int)hipGetLastError();
}
