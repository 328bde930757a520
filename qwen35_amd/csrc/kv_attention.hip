// kv_attention.hip -- attention over the 8-bit key/value cache.
//
// One wave per packed token and query head: 64 keys at a time, a key a lane
// for the scores, eight or fewer dimensions' sums a lane for the output, with
// the running maximum and sum of the softmax in f32.
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
  // the cut of long sequences (few rows): off, or items aimed for, least 32-key units of one, bound of a sequence's units
  bool cut;
  int few_target, few_min, max_units, few_rows;
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
constexpr long kFewCountBytes = 32768;
constexpr int kFewPairs = kFewCountBytes / 4;  // most (sequence, key head) pairs that are cut
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
  int seq, head, chunk, chunks, slot, unit;  // slot: of the first chunk's partial results; unit: 32-key units of a chunk
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
    // about few_target items in all, none of fewer than few_min units
    unit = max(a.few_min, (int)(((long)total * a.kv_heads + a.few_target - 1) / a.few_target));
  }
  int items = 0, slots = 0;
  for (int i0 = 0; i0 < a.nseq; i0 += 64) {
    if (i0) s = few_seq(a, i0 + lane);
    const int c = s.n ? max(1, (int)(((long)s.units + unit - 1) / unit)) : 0, cut = c > 1 ? c : 0;
    const int ci = wave_scan(c, lane), cs = wave_scan(cut, lane);
    const int all = __shfl(ci, 63, 64);
    if (at < items + all) {
      const int owner = __builtin_ctzll(__ballot(items + ci > at));
      it.seq = i0 + owner;
      it.chunks = __shfl(c, owner, 64);
      it.chunk = at - (items + __shfl(ci, owner, 64) - it.chunks);
      it.slot = (slots + __shfl(cs, owner, 64) - it.chunks) * a.kv_heads + it.head * it.chunks;
      it.unit = unit;
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
// N consecutive values (16-byte stores where vec)
template <int N>
__device__ __forceinline__ void store_n(void* out, long at, int type, bool vec, const float* v) {
  if (vec && type == QHIP_TT_F32) {
#pragma unroll
    for (int i = 0; i < N; i += 4) *(f32x4*)((float*)out + at + i) = f32x4{v[i], v[i + 1], v[i + 2], v[i + 3]};
  } else if (vec) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      uint64_t w = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint16_t b = type == QHIP_TT_F16 ? __builtin_bit_cast(uint16_t, (f16_t)v[i + j])
                                               : __builtin_bit_cast(uint16_t, (bf16_t)v[i + j]);
        w |= (uint64_t)b << (16 * j);
      }
      *(uint64_t*)((uint16_t*)out + at + i) = w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) store1(out, at + i, type, v[i]);
  }
}

// what e^-(m - M) leaves of a part whose maximum is m (both may be -infinity)
__device__ __forceinline__ float weight_of(float m, float top) { return m == top ? 1.0f : __builtin_amdgcn_exp2f(m - top); }

// SPLIT 2: f32 rows, queries and weights in two f16 parts each
template <int D, int SPLIT>
__global__ __launch_bounds__(256, D == 256 ? 2 : D == 128 ? 3 : 4) void k_kv_attention_few(KvAttnArgs a) {
  constexpr int J = D / 64, C = D / 16, W = D / 64;  // 64-dimension pieces, output tiles, dwords of a value load
  __shared__ float s_o[2][C * 4 * 64], s_m[2][64], s_l[2][64];
  __shared__ int s_e[2];
  const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  FewItem it;
  if (!few_item(a, lane, it)) return;  // all four waves alike
  const int seq = __builtin_amdgcn_readfirstlane(it.seq), n = __builtin_amdgcn_readfirstlane(it.s.n);
  const int len = __builtin_amdgcn_readfirstlane(it.s.len), lo = __builtin_amdgcn_readfirstlane(it.s.lo);
  const int chunks = __builtin_amdgcn_readfirstlane(it.chunks), chunk = __builtin_amdgcn_readfirstlane(it.chunk);
  const int head = __builtin_amdgcn_readfirstlane(it.head), unit = __builtin_amdgcn_readfirstlane(it.unit);
  const int rows = n * a.group, tiles = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
  const int key0 = lo + (chunks > 1 ? chunk * unit * 32 : 0);
  const int key1 = chunk == chunks - 1 ? len : key0 + unit * 32;
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
  int ve = -1000;  // the values' power of two: o is in units of 2^(ve - 14) / 2^9

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
    // the largest value scale's power of two (a NaN is never the larger)
    int e = vs > 0.0f ? __builtin_amdgcn_frexp_expf(vs) : -1000;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) e = max(e, __shfl_xor(e, d, 64));
    e = max(e, ve);
    if (e != ve) {
      const float f = __builtin_ldexpf(1.0f, ve - e);
#pragma unroll
      for (int c = 0; c < C; ++c) o[c] *= f;
      ve = e;
    }
    vs = __builtin_ldexpf(vs, 14 - ve);
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
      const float w0 = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(vs), 2 * st));
      const float w1 = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(vs), 2 * st + 1));
      float top = kMinusInf;
      const bool edge = key < all_lo || key + 32 > min(all_hi, key1);  // some row does not see some key
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[0][r] *= c0;
        s[1][r] *= c1;
      }
      if (edge) {
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int j = key + 16 * tt + 4 * g + r;
            if (j < vis_lo || j >= vis_hi || j >= key1) s[tt][r] = kMinusInf;
          }
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) top = fmaxf(top, fmaxf(s[0][r], s[1][r]));
      top = fmaxf(m, row_max(top));
      if (__any(top != m)) {
        const float f = weight_of(m, top);
        l *= f;
#pragma unroll
        for (int c = 0; c < C; ++c) o[c] *= f;
        m = top;
      }
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
        for (int r = 0; r < 4; ++r) s_o[slot][(4 * c + r) * 64 + lane] = o[c][r];
      s_m[slot][lane] = m;
      s_l[slot][lane] = l;
      if (lane == 0) s_e[slot] = ve;
    }
    __syncthreads();
    if (wave < half * tiles) {
      const float m2 = s_m[wave][lane], top = fmaxf(m, m2);
      const int e = max(ve, s_e[wave]);
      const float f1 = weight_of(m, top), f2 = weight_of(m2, top);
      const float g1 = __builtin_ldexpf(f1, ve - e), g2 = __builtin_ldexpf(f2, s_e[wave] - e);
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[c][r] = o[c][r] * g1 + s_o[wave][(4 * c + r) * 64 + lane] * g2;
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
      if (a.lse && g == 0) a.lse[(long)t * a.q_heads + qh] = l == 0.0f ? kMinusInf : (m + __builtin_log2f(l)) * 0.693147180559945309f;
    }
    return;
  }
  // partial results of the chunk: out [rows][D] (of its own keys), then m and l
  const long stride = (long)a.few_rows * (D + 2);
  float* parts_at = a.partial + (long)it.slot * stride;
  if (wave < tiles && own_row) {
    float* mine = parts_at + chunk * stride;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int c = 0; c < C; ++c)
        sk_store(mine + row * D + (4 * g + r) * C + c, __builtin_ldexpf(o[c][r] * norm, ve - 14 + 9));
    if (g == 0) {
      sk_store(mine + a.few_rows * D + 2 * row, m);
      sk_store(mine + a.few_rows * D + 2 * row + 1, l);
    }
  }
  unsigned* count = a.counters + (long)seq * a.kv_heads + head;
  if (!sk_arrive(count, (unsigned)chunks)) return;
  sk_reset(count);
  // the last workgroup: a wave a row, D / 64 values a lane
  for (int rw = wave; rw < rows; rw += 4) {
    float top = kMinusInf;
    for (int c0 = 0; c0 < chunks; c0 += 64) {
      float x = c0 + lane < chunks ? sk_load(parts_at + (c0 + lane) * stride + a.few_rows * D + 2 * rw) : kMinusInf;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) x = fmaxf(x, __shfl_xor(x, d, 64));
      top = fmaxf(top, x);
    }
    float acc[W], sum = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w) acc[w] = 0.0f;
    for (int c0 = 0; c0 < chunks; c0 += 64) {
      const int cnt = min(64, chunks - c0);
      float f = 0.0f;
      if (lane < cnt) {
        const float* x = parts_at + (c0 + lane) * stride + a.few_rows * D + 2 * rw;
        f = weight_of(sk_load(x), top) * sk_load(x + 1);
      }
      for (int i = 0; i < cnt; ++i) {
        const float fi = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f), i));
        const float* x = parts_at + (c0 + i) * stride + rw * D + lane * W;
        sum += fi;
#pragma unroll
        for (int w = 0; w < W; ++w) acc[w] += fi * sk_load(x + w);
      }
    }
    const int tk = rw / a.group, tt = a.offsets[seq] + tk, h = head * a.group + (rw - tk * a.group);
    if (tt < 0 || tt >= a.tokens) continue;
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int w = 0; w < W; ++w) store1(a.out, (long)tt * a.out_token + (long)h * a.out_head + lane * W + w, a.type, acc[w] * inv);
    if (a.lse && lane == 0) a.lse[(long)tt * a.q_heads + h] = sum == 0.0f ? kMinusInf : (top + __builtin_log2f(sum)) * 0.693147180559945309f;
  }
}

// ---- every other sequence ------------------------------------------------------------

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
  if (t >= a.offsets[a.nseq] || a.offsets[lo + 1] - a.offsets[lo] <= a.few_tokens) return;
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

template <int SPLIT>
static void launch_few(const KvAttnArgs& a, int dim, unsigned grid, hipStream_t s) {
  if (dim == 64) hipLaunchKernelGGL((k_kv_attention_few<64, SPLIT>), dim3(grid), dim3(256), 0, s, a);
  else if (dim == 128) hipLaunchKernelGGL((k_kv_attention_few<128, SPLIT>), dim3(grid), dim3(256), 0, s, a);
  else hipLaunchKernelGGL((k_kv_attention_few<256, SPLIT>), dim3(grid), dim3(256), 0, s, a);
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

// How the few-row sequences are cut: items aimed for, and the workspace (0: no cut).
struct FewPlan {
  int tokens, rows, max_units, target, least;
  long grid, work;
};
static FewPlan few_plan(const qhip_kv_cache* c, const qhip_kv_batch* b, int q_heads) {
  const int group = q_heads / c->kv_heads;
  FewPlan p{};
  p.tokens = kFewRows / group < b->max_new ? kFewRows / group : b->max_new;
  p.rows = p.tokens * group;
  p.max_units = (int)(((long)b->max_kv + 31) / 32);
  p.target = p.rows <= 16 ? 1024 : 512;
  p.least = 16;
  const long pairs = (long)b->nseq * c->kv_heads, most = (p.max_units + p.least - 1) / p.least;
  p.grid = pairs;
  if (p.tokens > 0 && most > 1 && pairs <= kFewPairs && (long)b->nseq * p.max_units < 0x7FFFFFFFL) {
    p.grid = pairs * most < p.target + pairs ? pairs * most : p.target + pairs;
    // sequences that are cut have less than twice target chunks: a chunk holds
    // at least a target-th of all units
    const long slots = pairs * most < 2L * p.target ? pairs * most : 2L * p.target;
    p.work = kFewCountBytes + slots * p.rows * (c->head_dim + 2) * 4;
  }
  return p;
}

}  // namespace qhip

using namespace qhip;

extern "C" long qhip_kv_attention_work_bytes(const qhip_kv_cache* cache, const qhip_kv_batch* batch, int q_heads) {
  return check_batch(cache, batch, q_heads) ? -1 : few_plan(cache, batch, q_heads).work;
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
  const FewPlan plan = few_plan(cache, batch, q_heads);
  const bool cut = plan.work > 0 && d_work && work_bytes >= plan.work;
  const int group = q_heads / cache->kv_heads;
  const KvAttnArgs a{(const int8_t*)cache->k, (const int8_t*)cache->v, cache->k_scale, cache->v_scale, batch->offsets,
                     batch->kv_lens, batch->table, d_q, d_out, d_lse, q_token_stride, q_head_stride, out_token_stride,
                     out_head_stride, batch->nseq, batch->tokens, batch->table_width, kv_block_shift(cache->block_size),
                     cache->num_blocks, cache->kv_heads, q_heads, softmax_scale, causal, window, type, group, plan.tokens,
                     kv_rows_aligned(d_q, q_token_stride, q_head_stride, size),
                     kv_rows_aligned(d_out, out_token_stride, out_head_stride, size), cut, plan.target, plan.least,
                     plan.max_units, plan.rows, (unsigned*)d_work, (float*)((char*)d_work + kFewCountBytes)};
  hipStream_t s = (hipStream_t)stream;
  if (plan.tokens > 0) {
    const unsigned grid = (unsigned)(cut ? plan.grid : (long)batch->nseq * cache->kv_heads);
    if (type == QHIP_TT_F32) launch_few<2>(a, cache->head_dim, grid, s);
    else launch_few<1>(a, cache->head_dim, grid, s);
  }
  if (batch->max_new > plan.tokens) {
    if (type == QHIP_TT_F32) launch_attention<float>(a, cache->head_dim, s);
    else if (type == QHIP_TT_F16) launch_attention<f16_t>(a, cache->head_dim, s);
    else launch_attention<bf16_t>(a, cache->head_dim, s);
  }
  return (int)hipGetLastError();
}
