// kv_attention.hip -- attention over the 8-bit key/value cache.
//
//   s_j = scale * q . k_j over the keys j that the row sees, out = sum
//   softmax(s)_j v_j, lse = log(sum exp(s_j)); k_j = code * key scale of j's
//   block, v_j likewise
//
// in one pass over the keys with a running maximum m and sum l in f32.  Two
// kernels, each for its own sequences of a batch: one for those of a few rows,
// whose cost is reading the codes, and one for those of many, whose cost is the
// products.  A row is a query head of a new token; the rows of one key head (row
// = token * G + head of the group) share every key.
#include "kv_internal.hpp"
#include "qhip_device.hpp"
#include "qhip_internal.hpp"

namespace qhip {

typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 h16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

struct KvAttnArgs {
  const int8_t *k, *v;
  const float *k_scale, *v_scale;
  const int *offsets, *kv_lens, *table;
  const void* q;
  void* out;
  float* lse;
  long q_token, q_head, out_token, out_head;
  int nseq, tokens, width, shift, num_blocks, kv_heads, q_heads;
  float scale, sign;  // the softmax scale's absolute value and sign
  int causal, window, type, group;
  int group_inv;  // 2^20 / group, rounded up
  // the kernel's sequences (those of min_tokens < new tokens <= max_tokens), the
  // rows of a workgroup and log2 of the keys of a unit
  int min_tokens, max_tokens, tile_rows, key_shift;
  // the cut of long sequences: off, or a unit count's share of the items aimed
  // for, fewest key units of an item, bound of a sequence's units, most chunks,
  // and the chunks that the workspace holds
  bool cut;
  float share;
  int least, max_units, max_chunks;
  long slots;
  unsigned* counters;
  float* partial;
};

constexpr float kMinusInf = -INFINITY;
constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.693147180559945309f;

// ---- codes as f16 ---------------------------------------------------------------------
// A code + 128 read as a subnormal f16 is (code + 128) 2^-24; one packed fma
// makes it code * 2^-9, exactly.
constexpr float kCodeScale = 0x1p9f;

// bytes 0 and 2 of p (biased by 128, bytes 1 and 3 zero)
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
// byte B of eight dwords (biased): one dimension of eight keys
template <int B>
__device__ __forceinline__ h16x8 codes_across(const uint32_t* x) {
  constexpr uint32_t sel = 0x0C000C00u | (unsigned)B | ((4u + B) << 16);
  const h16x2 p0 = codes2(__builtin_amdgcn_perm(x[1], x[0], sel)), p1 = codes2(__builtin_amdgcn_perm(x[3], x[2], sel));
  const h16x2 p2 = codes2(__builtin_amdgcn_perm(x[5], x[4], sel)), p3 = codes2(__builtin_amdgcn_perm(x[7], x[6], sel));
  return h16x8{p0[0], p0[1], p1[0], p1[1], p2[0], p2[1], p3[0], p3[1]};
}

// ---- lanes ------------------------------------------------------------------------------

// maximum of a value over lanes l and l ^ 32 / over the four lanes l mod 16
__device__ __forceinline__ float max32(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float sum32(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}
__device__ __forceinline__ float max16(float v) {
  v = max32(v);
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float sum16(float v) {
  v = sum32(v);
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
__device__ __forceinline__ float lane_f(float v, int i) {
  return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), i));
}
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// A uniform value that the compiler takes as new here, so that what is computed
// from it stays in its branch (it would otherwise be done on every path).
__device__ __forceinline__ int here(int v) {
  asm volatile("" : "+s"(v));
  return v;
}

// ---- a workgroup's item -------------------------------------------------------------------
//
// Sequences that are cut into chunks of keys come first, so that the short ones
// fill the end; a sequence's row tiles from the last (which sees the most keys),
// a tile's chunks, and fastest the key heads.  The chunk count follows from a
// sequence's share of all sequences' row tiles times key units, so that a ragged
// batch spreads evenly over the workgroups; every wave works the plan out for
// itself, 64 sequences at a time.  c = round(units / unit) chunks, at least one:
// sequences that are cut have fewer than 4/3 of their units / unit, so all
// chunks of cut sequences are fewer than 4/3 of the items aimed for.
struct Item {
  int seq, head, off, n, len, tile, chunk, chunks;  // off: the sequence's first packed token
  int slot, counter;  // of the tile's first chunk among the partial results, of the tile
};
struct SeqPlan {
  int first, n, len, tiles, units;
};
__device__ __forceinline__ SeqPlan plan_seq(const KvAttnArgs& a, int i) {
  SeqPlan s{0, 0, 0, 0, 0};
  if (i >= a.nseq) return s;
  const int first = a.offsets[i], end = a.offsets[i + 1], len = a.kv_lens[i];
  if (first < 0 || end <= first) return s;
  const int n = end - first, here = min(end, a.tokens) - first;  // new tokens, and those among the packed rows
  if (n <= a.min_tokens || n > a.max_tokens || n > kMaxLen || here <= 0) return s;
  s.first = first;
  s.n = n;
  s.len = min(max(len, 0), kMaxLen);
  s.tiles = (here * a.group + a.tile_rows - 1) / a.tile_rows;
  int keys = s.len;
  if (a.window > 0) keys = (int)min((long)keys, (long)a.window + a.tile_rows + (2 << a.key_shift));
  s.units = min((keys + (1 << a.key_shift) - 1) >> a.key_shift, a.max_units);
  return s;
}
__device__ __forceinline__ bool find_item(const KvAttnArgs& a, int lane, Item& it) {
  const int at = blockIdx.x / a.kv_heads;
  SeqPlan s = plan_seq(a, lane);
  float per_unit = 0.0f;  // chunks of a key unit
  if (a.cut) {
    int total = s.tiles * s.units;
    for (int i = 64 + lane; i - lane < a.nseq; i += 64) {
      const SeqPlan x = plan_seq(a, i);
      total += x.tiles * x.units;
    }
    total = __builtin_amdgcn_readlane(scan64(total), 63);
    per_unit = 1.0f / fmaxf((float)a.least, (float)total * a.share);
  }
  int items = 0, tiles = 0;  // before the 64 sequences, of the cut ones
  for (int pass = a.cut ? 0 : 1; pass < 2; ++pass)
    for (int i0 = 0; i0 < a.nseq; i0 += 64) {
      if (a.nseq > 64) s = plan_seq(a, i0 + lane);
      const int c = min(a.max_chunks, max(1, (int)((float)s.units * per_unit + 0.5f)));
      const int here = (c > 1) == (pass == 0) ? s.tiles : 0;
      const int ni = scan64(here * c), ti = scan64(here);
      const int all = __builtin_amdgcn_readlane(ni, 63);
      if (at < items + all) {
        const int owner = __builtin_ctzll(__ballot(items + ni > at));
        const int count = __builtin_amdgcn_readlane(s.tiles, owner);
        it.seq = uniform(i0 + owner);
        it.head = uniform(blockIdx.x - at * a.kv_heads);
        it.off = __builtin_amdgcn_readlane(s.first, owner);
        it.n = __builtin_amdgcn_readlane(s.n, owner);
        it.len = __builtin_amdgcn_readlane(s.len, owner);
        it.chunks = __builtin_amdgcn_readlane(c, owner);
        const int first = items + __builtin_amdgcn_readlane(ni, owner) - count * it.chunks;
        const int tile = uniform((at - first) / it.chunks);
        it.chunk = uniform(at - first - tile * it.chunks);
        it.tile = count - 1 - tile;
        it.slot = uniform((first + tile * it.chunks) * a.kv_heads + it.head * it.chunks);
        it.counter = uniform((tiles + __builtin_amdgcn_readlane(ti, owner) - 1 - tile) * a.kv_heads + it.head);
        return true;
      }
      items += all;
      tiles += __builtin_amdgcn_readlane(ti, 63);
    }
  return false;
}

constexpr int kBehind = 1 << 20;

// The item's rows and keys.
struct Span {
  int row0, rows;    // first row and rows of the tile
  int first;         // place of the sequence's first new token
  int key0, key1;    // this chunk's keys, from a unit's start
};
__device__ __forceinline__ Span find_span(const KvAttnArgs& a, const Item& it) {
  Span s;
  s.row0 = it.tile * a.tile_rows;
  s.rows = (int)min((long)a.tile_rows, (long)it.n * a.group - s.row0);
  s.first = it.len - it.n;
  const int tok_a = uniform(s.row0 / a.group), tok_b = uniform((s.row0 + s.rows - 1) / a.group);
  const int lo = a.window > 0 ? max(0, s.first + tok_a - a.window + 1) >> a.key_shift << a.key_shift : 0;
  // (lengths that the table cannot hold end a little behind it: enough for their rows to be NaN)
  const long cap = max((long)a.width << a.shift, (long)lo) + kBehind;
  const int hi = (int)min((long)(a.causal ? s.first + tok_b + 1 : it.len), cap);
  const int units = max(0, hi - lo + (1 << a.key_shift) - 1) >> a.key_shift;
  const int q = uniform(units / it.chunks), r = units - q * it.chunks;  // the first r chunks have one more
  const int u0 = q * it.chunk + min(it.chunk, r), u1 = u0 + q + (it.chunk < r ? 1 : 0);
  s.key0 = lo + (u0 << a.key_shift);
  s.key1 = min(hi, lo + (u1 << a.key_shift));
  return s;
}
// row r of the tile: its token among the sequence's new ones and its query head
struct RowAt {
  int tok, head;
};
__device__ __forceinline__ RowAt row_at(const KvAttnArgs& a, const Span& s, int r, int head) {
  const int base = s.row0 / a.group, x = s.row0 - base * a.group + r;
  const int t = (x * a.group_inv) >> 20;  // x / group, exact: x < 128 + group, so x * group < 2^20
  return RowAt{base + t, head * a.group + (x - t * a.group)};
}

// ---- a 16-key tile's block ------------------------------------------------------------------
// (a block holds whole 16-key tiles)  NaN scales where the table names no block
// of the pool: the rows that see the tile become NaN; the address is block 0's.
struct TileInfo {
  int id;
  float ks, vs;
};
__device__ __forceinline__ int tile_id(const KvAttnArgs& a, int seq, int key, int end) {
  const int b = key >> a.shift;
  return key >= end ? -2 : (unsigned)b < (unsigned)a.width ? a.table[(long)seq * a.width + b] : -1;
}
__device__ __forceinline__ TileInfo tile_info(const KvAttnArgs& a, int id, int head) {
  const bool in = (unsigned)id < (unsigned)a.num_blocks;
  TileInfo x{in ? id : 0, 0.0f, 0.0f};
  if (id != -2) {  // -2: past the last key, never seen
    x.ks = a.k_scale[(long)x.id * a.kv_heads + head];
    x.vs = a.v_scale[(long)x.id * a.kv_heads + head];
    x.ks = in && finite_bits(__float_as_uint(x.ks)) ? x.ks : __builtin_nanf("");
    x.vs = in && finite_bits(__float_as_uint(x.vs)) ? x.vs : __builtin_nanf("");
  }
  return x;
}

// ---- queries ----------------------------------------------------------------------------------
// A lane's pieces of eight query values as they lie in memory (f32 rows where
// SPLIT is 2, else 16-bit ones).
template <int SPLIT>
using QElem = typename std::conditional<SPLIT == 2, float, uint16_t>::type;
template <int SPLIT>
using QRaw = Raw8<QElem<SPLIT>>;

template <int SPLIT>
__device__ __forceinline__ float q_value(const QRaw<SPLIT>& raw, int i, int type) {
  if constexpr (SPLIT == 2) return raw.e[i];
  else if (type == QHIP_TT_F16) return (float)__builtin_bit_cast(f16_t, raw.e[i]);
  else return __uint_as_float((uint32_t)raw.e[i] << 16);
}
// The row's values times a power of two that brings the largest to below 2^14
// (and the softmax scale's sign), as f16 or, SPLIT 2, as the sum of two (22
// bits); returns the power.
template <int SPLIT, int N, typename RowMax>
__device__ __forceinline__ int split_q(const QRaw<SPLIT>* raw, int type, float sign, RowMax row_max, h16x8* hi, h16x8* lo) {
  float top = 0.0f;
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(q_value<SPLIT>(raw[n], i, type)));
  const int e = 14 - __builtin_amdgcn_frexp_expf(row_max(top));
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = __builtin_ldexpf(q_value<SPLIT>(raw[n], i, type) * sign, e);
      hi[n][i] = (_Float16)x;
      if constexpr (SPLIT == 2) lo[n][i] = (_Float16)(x - (float)hi[n][i]);
    }
  return e;
}

// ---- results ------------------------------------------------------------------------------------
// N (a power of two) consecutive values of a row, in pieces of up to 16 bytes
template <int SPLIT, int N>
__device__ __forceinline__ void store_row(void* out, long at, int type, const float* v) {
  typedef QElem<SPLIT> T;
  constexpr int P = N * sizeof(T) < 16 ? N : 16 / sizeof(T);
  typedef T value __attribute__((ext_vector_type(P)));
  struct __attribute__((packed, aligned(2))) piece { value x; };
#pragma unroll
  for (int i = 0; i < N; i += P) {
    value x;
#pragma unroll
    for (int j = 0; j < P; ++j) {
      if constexpr (SPLIT == 2) x[j] = v[i + j];
      else x[j] = type == QHIP_TT_F16 ? __builtin_bit_cast(uint16_t, (f16_t)v[i + j]) : __builtin_bit_cast(uint16_t, (bf16_t)v[i + j]);
    }
    ((piece*)((T*)out + at + i))->x = x;
  }
}
// log(sum e^s) of a row whose maximum is in powers of two
__device__ __forceinline__ float row_lse(float m, float l) {
  return l == 0.0f ? kMinusInf : (m + __builtin_log2f(l)) * kLn2;
}
// what 2^(m - top) leaves of a part whose maximum is m (both may be -infinity)
__device__ __forceinline__ float weight_of(float m, float top) { return m == top ? 1.0f : __builtin_amdgcn_exp2f(m - top); }

// A row's weights are taken relative to a maximum m and to the power of two e of
// a value scale, times 2^kShift: its output is in units of 2^(e - kShift) times
// kCodeScale.  m and e are those of what the row itself has seen (so that hidden
// blocks change no bit of it), and move only when a score passes m by more than
// kLag or a scale 2^(e + kLagExp): the output is then rescaled, which at every
// new maximum would cost a tile of many rows a tenth of its time.  Weights stay
// below 2^15, inside f16.  Two-part weights keep the larger shift: what is below
// 2^-24 of it is lost, and they are to be good to 22 bits.
template <int SPLIT>
constexpr int kShift = SPLIT == 2 ? 14 : 7;
template <int SPLIT>
constexpr float kLag = SPLIT == 2 ? 1.0f : 7.0f;
template <int SPLIT>
constexpr int kLagExp = SPLIT == 2 ? 0 : 1;
constexpr int kNoScale = -1000;  // of a zero or a NaN
__device__ __forceinline__ int scale_exp(float v) { return fabsf(v) > 0.0f ? __builtin_amdgcn_frexp_expf(v) : kNoScale; }
template <int SPLIT>
__device__ __forceinline__ float in_units(float o, int e) { return __builtin_ldexpf(o, e - kShift<SPLIT> + 9); }

// ---- joining a tile's chunks ----------------------------------------------------------------------
//
// A chunk's partial results are tile_rows x D outputs of its own keys, then each
// row's maximum m and sum l, stored and loaded through to the agent's point of
// coherence (sc1: sk_store's and sk_load's policy, 16 bytes at a time).  Every
// chunk adds one to the tile's counter; the last one joins all in chunk order,
// so the result does not depend on which was last.  A join is bound by the
// latency of its loads, so 16 pieces a thread are in flight: 4 chunks of 128 rows
// of 128 dimensions take 10 us, a decode's chunks of 4 rows 3.7.  (32 in
// flight spill the products' registers: 96 us against 86 for 512 rows behind 8000
// keys.)
constexpr int kSc1 = 16;  // cache policy of a buffer access
constexpr long kCountBytes = 32768;
constexpr int kMaxCut = kCountBytes / 4;  // most row tiles that are cut

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

// LDS of a join: 4 KB of sums, 1 / sum of each row, m (then weights) and l of
// rows x chunks
constexpr int kJoinLds = 16384;  // least that a kernel has
constexpr int join_pairs(int lds) { return (lds - 4096 - 4 * 128) / 8; }  // most rows x chunks

// All 256 threads.  EB pieces of four values a thread and CB chunks are loaded
// at a time; with fewer than 256 pieces the threads share out the chunks.
template <int D, int SPLIT, int EB, int CB>
__device__ __forceinline__ void join_rows(const KvAttnArgs& a, float* lds, __amdgpu_buffer_rsrc_t parts, const Item& it,
                                          const Span& sp) {
  const int tid = threadIdx.x, count = sp.rows, chunks = it.chunks, stride = a.tile_rows * (D + 2);
  float* s_acc = lds;             // [256][4]
  float* s_inv = lds + 1024;      // [128]
  float* s_m = lds + 1024 + 128;  // [chunks][count]
  float* s_l = s_m + chunks * count;
  const int pieces = count * (D / 4), slices = EB == 1 ? 256 / pieces : 1;
  const int sl = EB == 1 ? tid / pieces : 0, e0 = EB == 1 ? tid - sl * pieces : tid;
  kv_u32x4 x[EB][CB];
  auto load = [&](int e, int c) {  // past the last piece or chunk: out of the buffer's bounds, 0
#pragma unroll
    for (int j = 0; j < EB; ++j)
#pragma unroll
      for (int k = 0; k < CB; ++k)
        x[j][k] = __builtin_amdgcn_raw_buffer_load_b128(
            parts, 4 * (e + 256 * j < pieces && sl < slices ? (c + k * slices) * stride + 4 * (e + 256 * j) : chunks * stride), 0, kSc1);
  };
  load(e0, sl);
  for (int i = tid; i < chunks * count; i += 256) {
    const int c = i / count, r = i - c * count;
    const kv_u32x2 y = __builtin_amdgcn_raw_buffer_load_b64(parts, 4 * (c * stride + a.tile_rows * D + 2 * r), 0, kSc1);
    s_m[i] = __uint_as_float(y[0]);
    s_l[i] = __uint_as_float(y[1]);
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
      const RowAt w = row_at(a, sp, r, it.head);
      const int t = it.off + w.tok;
      if (a.lse && t >= 0 && t < a.tokens) a.lse[(long)t * a.q_heads + w.head] = row_lse(top, sum);
    }
  }
  __syncthreads();
  for (int e = e0; e - tid < pieces; e += 256 * EB) {
    f32x4 acc[EB] = {};
    for (int c = sl; c < chunks; c += CB * slices) {
      if (e != e0 || c != sl) load(e, c);
#pragma unroll
      for (int j = 0; j < EB; ++j)
#pragma unroll
        for (int k = 0; k < CB; ++k) {
          const int cc = c + k * slices, r = (e + 256 * j) / (D / 4);
          const float f = cc < chunks && r < count ? s_m[cc * count + r] : 0.0f;
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[j][i] += f * __uint_as_float(x[j][k][i]);
        }
    }
    if constexpr (EB == 1) {
      ((f32x4*)s_acc)[tid] = acc[0];
      __syncthreads();
      if (sl == 0)
        for (int k = 1; k < slices; ++k) acc[0] += ((f32x4*)s_acc)[k * pieces + e];
    }
#pragma unroll
    for (int j = 0; j < EB; ++j) {
      const int ee = e + 256 * j, r = ee / (D / 4);
      if (ee >= pieces || sl != 0) continue;
      const RowAt w = row_at(a, sp, r, it.head);
      const int t = it.off + w.tok;
      if (t < 0 || t >= a.tokens) continue;
      const float inv = s_inv[r], v[4] = {acc[j][0] * inv, acc[j][1] * inv, acc[j][2] * inv, acc[j][3] * inv};
      store_row<SPLIT, 4>(a.out, (long)t * a.out_token + (long)w.head * a.out_head + 4 * (ee % (D / 4)), a.type, v);
    }
    if constexpr (EB == 1) break;
  }
}
// Whether each chunk of the item's tile has its place in the workspace and its
// workgroup in the grid.  Always, but for offsets that are none and sequences of
// more than the stated tokens, whose counters would stay behind.
__device__ __forceinline__ bool all_arrive(const KvAttnArgs& a, const Item& it) {
  const int last = it.slot + (it.chunks - 1) * a.kv_heads - it.head * (it.chunks - 1);  // workgroup of the last chunk
  return it.slot + it.chunks <= a.slots && it.counter < kMaxCut && last < (int)gridDim.x;
}
// After every thread's part_stores: whether this workgroup was the tile's last,
// which then joins.
template <int D, int SPLIT>
__device__ __forceinline__ void arrive_and_join(const KvAttnArgs& a, float* lds, __amdgpu_buffer_rsrc_t parts, const Item& it,
                                                const Span& sp) {
  unsigned* counter = a.counters + it.counter;
  if (!sk_arrive(counter, (unsigned)it.chunks)) return;
  sk_reset(counter);
  constexpr int F = D == 64 ? 2 : 4;  // 16 pieces in flight a thread, where the registers allow it
  if (sp.rows * (D / 4) <= 256) join_rows<D, SPLIT, 1, 4 * F>(a, lds, parts, it, sp);
  else join_rows<D, SPLIT, F, 4>(a, lds, parts, it, sp);
}

// ---- sequences of a few rows: the cache streamed once ------------------------------
//
// A wave has 16 rows (NT = 2: two times 16, on each step's codes), a workgroup that
// many or twice as many (attn_plans).  The work is one pass over the codes, 2 D bytes a key, so the kernel is built to keep loads in flight and
// never puts a code anywhere but in a register:
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
// f32 rows (SPLIT 2) take queries and softmax weights in two f16 parts each, 22
// bits; f16 and bf16 rows, whose outputs are rounded to 11 and 8 bits, weights of
// 11.  A block's key scale multiplies the scores, its value scale the weights.
//
// A workgroup's four waves take steps of 32 keys in turn (with twice a wave's rows,
// two and two of them) and are merged in LDS.  Long sequences are cut into chunks
// over workgroups (find_item).
//
// Bound by memory where sequences are long: one f32 token on 131071 keys (4 key
// heads of 256, 268 MB) 60 us, 4.5 TB/s; 64 tokens on 2000 keys each (262 MB), 54 us at
// 4.9 TB/s (4 heads of 256) and 51 us at 5.1 (8 of 128).  Short ones are bound by
// chains of latencies: lengths - plan - table - scales 5 us and codes 3 us before
// the first product, 2 us to merge the waves, partial results - counter - join 5
// us where a sequence is cut: one token on 333 keys takes 13 us.  Every wave walks
// all sequences for the plan, so many short ones cost more: 512 decodes of up to
// 2000 keys 104 us (306 MB, 62 at the copy's rate), 1000 of them 199 (547 MB, 111).
// f32 rows in number are bound by the matrix pipe at twice the products for either
// operand: 4096 tokens, 16 heads of 128, 170 to 195 us by the card (350 to 400
// TFLOP/s), of 256 365 to 375.  The registers allow two waves a SIMD for D = 256 and three for
// 128; a fourth would spill (60 us against 44 for 64 ragged decodes).
constexpr int kFewRows = 64;  // rows up to which a sequence beside long ones is this kernel's

template <int D, int SPLIT, int NT>
__global__ __launch_bounds__(256, NT == 1 ? (D == 256 ? 2 : D == 128 ? 3 : 4) : 2)
void k_kv_attention_few(KvAttnArgs a) {
  constexpr int J = D / 64, C = D / 16, W = D / 64;  // 64-dimension pieces, output tiles, dwords of a value load
  constexpr int R = NT * C * 4 * 64;                 // floats of a wave's output
  __shared__ __attribute__((aligned(16))) float s_o[4 * R];
  static_assert(sizeof(s_o) >= kJoinLds, "the join's LDS");
  __shared__ float s_m[4][NT][64], s_l[4][NT][64];
  __shared__ int s_e[4][NT][64];
  const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, g = lane >> 4;
  const int wave = uniform(tid >> 6);
  Item it;
  if (!find_item(a, lane, it)) return;  // all four waves alike
  const Span sp = find_span(a, it);
  const int tiles = sp.rows <= 16 * NT ? 1 : 2, part = wave / tiles, parts = 4 / tiles;

  // lane i: tile i & 1 of this wave's step i / 2 of a round of 32 steps
  int s0 = part;
  auto round_id = [&]() { return tile_id(a, it.seq, sp.key0 + 32 * (s0 + parts * (lane >> 1)) + 16 * (lane & 1), sp.key1); };
  const int id0 = round_id();

  // this lane's rows
  int vis_hi[NT], vis_lo[NT];
  QRaw<SPLIT> raw[NT][2 * J] = {};
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int row = ((wave % tiles) * NT + nt) * 16 + r16;
    const RowAt w = row_at(a, sp, row < sp.rows ? row : 0, it.head);
    const int p = sp.first + w.tok, t = it.off + w.tok;
    vis_hi[nt] = min(a.causal ? p + 1 : it.len, sp.key1);  // of this chunk
    vis_lo[nt] = a.window > 0 ? p - a.window + 1 : 0;
    if (row < sp.rows && t >= 0 && t < a.tokens) {
      const long at = (long)t * a.q_token + (long)w.head * a.q_head + 16 * g;
#pragma unroll
      for (int i = 0; i < 2 * J; ++i) raw[nt][i] = load8((const QElem<SPLIT>*)a.q + at + 64 * (i >> 1) + 8 * (i & 1));
    }
  }
  // keys that every row of the tile sees
  const int all_hi = a.causal ? sp.first + uniform(sp.row0 / a.group) + 1 : it.len;
  const int all_lo = a.window > 0 ? sp.first + uniform(row_at(a, sp, sp.rows - 1, it.head).tok) - a.window + 1 : 0;

  TileInfo info = tile_info(a, id0, it.head);
  const uint8_t* kc = (const uint8_t*)a.k;
  const uint8_t* vc = (const uint8_t*)a.v;
  const int mask = (1 << a.shift) - 1;
  const uint32_t koff = (uint32_t)(r16 * D + 16 * g), voff = (uint32_t)(4 * g * D + r16 * C);
  kv_u32x4 kr[2][J];
  uint32_t vr[8][W];
  auto tile_at = [&](int i) {  // byte offset of tile i's first code
    const uint64_t b = (uint32_t)__builtin_amdgcn_readlane(info.id, i);
    const unsigned first = (sp.key0 + 32 * (s0 + parts * (i >> 1)) + 16 * (i & 1)) & mask;
    return ((b * (uint32_t)a.kv_heads + (uint32_t)it.head) << a.shift | first) * D;
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
  const bool any = sp.key0 + 32 * s0 < sp.key1;
  if (any) {
    load_k(0);
    load_v(0);
  }

  h16x8 q_hi[NT][2 * J], q_lo[NT][SPLIT == 2 ? 2 * J : 1];
  float c_row[NT], m[NT], l[NT];
  int ve[NT];
  f32x4 o[NT][C];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int qe = split_q<SPLIT, 2 * J>(raw[nt], a.type, a.sign, max16, q_hi[nt], q_lo[nt]);
    c_row[nt] = __builtin_ldexpf(a.scale * kLog2e * kCodeScale, -qe);
    m[nt] = kMinusInf;
    l[nt] = 0.0f;
    ve[nt] = kNoScale;
#pragma unroll
    for (int c = 0; c < C; ++c) o[nt][c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  // a wave's results into its part of the LDS, and those of a wave's part added to this one's
  // (the lane counted anew, here and for the results: what is kept over the loop spills)
  auto lane_here = [&]() { return (int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, (unsigned)here(0))); };
  auto give = [&]() {
    const int lane = lane_here();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r) s_o[wave * R + ((nt * C + c) * 4 + r) * 64 + lane] = o[nt][c][r];
      s_m[wave][nt][lane] = m[nt];
      s_l[wave][nt][lane] = l[nt];
      s_e[wave][nt][lane] = ve[nt];
    }
  };
  auto take = [&](int from) {
    const int lane = lane_here();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float m2 = s_m[from][nt][lane], top = fmaxf(m[nt], m2);
      const int ve2 = s_e[from][nt][lane], e = max(ve[nt], ve2);
      const float f1 = weight_of(m[nt], top), f2 = weight_of(m2, top);
      const float g1 = __builtin_ldexpf(f1, ve[nt] - e), g2 = __builtin_ldexpf(f2, ve2 - e);
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[nt][c][r] = o[nt][c][r] * g1 + s_o[from * R + ((nt * C + c) * 4 + r) * 64 + lane] * g2;
      l[nt] = l[nt] * f1 + s_l[from][nt][lane] * f2;
      m[nt] = top;
      ve[nt] = e;
    }
  };
  bool aside = false;  // results of earlier rounds wait in the LDS
  while (any) {
    const int steps = min(32, (sp.key1 - sp.key0 - 32 * s0 + 32 * parts - 1) / (32 * parts));
    for (int st = 0; st < steps; ++st) {
      const int key = sp.key0 + 32 * (s0 + parts * st);
      float s[NT][2][4];
#pragma unroll
      for (int tt = 0; tt < 2; ++tt) {
        f32x4 hi[NT], low[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) hi[nt] = low[nt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < 2 * J; ++j) {
          const kv_u32x4 x = kr[tt][j >> 1] ^ 0x80808080u;
          const h16x8 k = j & 1 ? codes8(x[2], x[3]) : codes8(x[0], x[1]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            hi[nt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, q_hi[nt][j], hi[nt], 0, 0, 0);
            if constexpr (SPLIT == 2) low[nt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, q_lo[nt][j], low[nt], 0, 0, 0);
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int r = 0; r < 4; ++r) s[nt][tt][r] = SPLIT == 2 ? hi[nt][r] + low[nt][r] : hi[nt][r];
      }
      if (st + 1 < steps) load_k(st + 1);
      const float k0 = lane_f(info.ks, 2 * st), k1 = lane_f(info.ks, 2 * st + 1);
      const float v0 = lane_f(info.vs, 2 * st), v1 = lane_f(info.vs, 2 * st + 1);
      const bool edge = key < all_lo || key + 32 > min(all_hi, sp.key1);  // some row does not see some key
      h16x8 ph[NT], pl[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float c0 = c_row[nt] * k0, c1 = c_row[nt] * k1;
        int e0 = scale_exp(v0), e1 = scale_exp(v1);
        if (edge) {
          const int from = vis_lo[nt], to = vis_hi[nt];
#pragma unroll
          for (int tt = 0; tt < 2; ++tt)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int j = key + 16 * tt + 4 * g + r;
              s[nt][tt][r] = j < from || j >= to ? kMinusInf : s[nt][tt][r];
            }
          e0 = key >= to || key + 16 <= from ? kNoScale : e0;
          e1 = key + 16 >= to || key + 32 <= from ? kNoScale : e1;
        }
        e0 = max(e0, e1);
        // the scores' factors c0, c1 are not negative, so each tile's largest is that of the products
        const float top0 = fmaxf(fmaxf(s[nt][0][0], s[nt][0][1]), fmaxf(s[nt][0][2], s[nt][0][3]));
        const float top1 = fmaxf(fmaxf(s[nt][1][0], s[nt][1][1]), fmaxf(s[nt][1][2], s[nt][1][3]));
        const float top = max16(fmaxf(top0 * c0, top1 * c1));
        if (__any(top > m[nt] + kLag<SPLIT> || e0 > ve[nt] + kLagExp<SPLIT>)) {
          const float m1 = top > m[nt] + kLag<SPLIT> ? top : m[nt];
          e0 = e0 > ve[nt] + kLagExp<SPLIT> ? e0 : ve[nt];
          const float f = weight_of(m[nt], m1), fo = __builtin_ldexpf(f, ve[nt] - e0);
          l[nt] *= f;
#pragma unroll
          for (int c = 0; c < C; ++c) o[nt][c] *= fo;
          m[nt] = m1;
          ve[nt] = e0;
        }
        const float w0 = __builtin_ldexpf(v0, kShift<SPLIT> - ve[nt]), w1 = __builtin_ldexpf(v1, kShift<SPLIT> - ve[nt]);
        auto hide = [&]() {  // what the row does not see has weight 0 whatever its block's scales are
          const int from = vis_lo[nt], to = vis_hi[nt], first = here(key);
#pragma unroll
          for (int tt = 0; tt < 2; ++tt)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int j = first + 16 * tt + 4 * g + r;
              s[nt][tt][r] = j < from || j >= to ? 0.0f : s[nt][tt][r];
            }
        };
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
          for (int r = 0; r < 4; ++r) s[nt][tt][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[nt][tt][r], tt ? c1 : c0, -m[nt]));
        if (edge) hide();
        float sum = 0.0f;
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            sum += s[nt][tt][r];
            s[nt][tt][r] *= tt ? w1 : w0;
          }
        if (edge && __any(!(w0 * 0.0f + w1 * 0.0f == 0.0f))) hide();  // 0 * NaN, 0 * infinity
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            ph[nt][4 * tt + r] = (_Float16)s[nt][tt][r];
            if constexpr (SPLIT == 2) pl[nt][4 * tt + r] = (_Float16)(s[nt][tt][r] - (float)ph[nt][4 * tt + r]);
          }
        l[nt] += sum;
      }
#pragma unroll
      for (int w = 0; w < W; ++w) {
        uint32_t x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = vr[i][w] ^ 0x80808080u;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const h16x8 v8 = b == 0 ? codes_across<0>(x) : b == 1 ? codes_across<1>(x) : b == 2 ? codes_across<2>(x) : codes_across<3>(x);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            f32x4& y = o[nt][4 * w + b];
            y = __builtin_amdgcn_mfma_f32_16x16x32_f16(v8, ph[nt], y, 0, 0, 0);
            if constexpr (SPLIT == 2) y = __builtin_amdgcn_mfma_f32_16x16x32_f16(v8, pl[nt], y, 0, 0, 0);
          }
        }
      }
      if (st + 1 < steps) load_v(st + 1);
    }
    s0 += 32 * parts;
    const bool more = sp.key0 + 32 * s0 < sp.key1;
    // One long sum of like terms would round the same way each time (1.2e-4 of an
    // output in 131,072 keys, now 2e-6): two rounds are summed by themselves and then
    // added to what waits in the LDS.
    if (!more || !((s0 >> 5) & parts)) {
      if (aside) take(wave);
      if (!more) break;
      give();
      aside = true;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        l[nt] = 0.0f;
#pragma unroll
        for (int c = 0; c < C; ++c) o[nt][c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      }
    }
    info = tile_info(a, round_id(), it.head);
    load_k(0);
    load_v(0);
  }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) l[nt] = sum16(l[nt]);

  // merge the waves that share a row tile: the upper half of the parts into the lower
  for (int half = parts / 2; half >= 1; half >>= 1) {
    const int at = wave - half * tiles;  // waves [half * tiles, 2 half * tiles) give
    if (at >= 0 && at < half * tiles) give();
    __syncthreads();
    if (at < 0) take(wave + half * tiles);
  }

#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    // a row that sees nothing: 0 and -infinity (l is 0); NaN stays
    const float norm = l[nt] == 0.0f ? 0.0f : 1.0f / l[nt];
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int r = 0; r < 4; ++r) o[nt][c][r] = in_units<SPLIT>(o[nt][c][r] * norm, ve[nt]);
  }
  const int lane_end = lane_here(), g_end = lane_end >> 4, row_end = (wave % tiles) * NT * 16 + (lane_end & 15);
  if (it.chunks == 1) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = row_end + 16 * nt;
      const RowAt w = row_at(a, sp, row < sp.rows ? row : 0, it.head);
      const int t = it.off + w.tok;
      if (wave < tiles && row < sp.rows && t >= 0 && t < a.tokens) {
        const long at = (long)t * a.out_token + (long)w.head * a.out_head + 4 * g_end * C;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float v[C];
#pragma unroll
          for (int c = 0; c < C; ++c) v[c] = o[nt][c][r];
          store_row<SPLIT, C>(a.out, at + r * C, a.type, v);
        }
        if (a.lse && g_end == 0) a.lse[(long)t * a.q_heads + w.head] = row_lse(m[nt], l[nt]);
      }
    }
    return;
  }
  if (!all_arrive(a, it)) return;
  const int stride = a.tile_rows * (D + 2);
  const __amdgpu_buffer_rsrc_t parts_at = part_rsrc(a.partial + (long)it.slot * stride, (long)it.chunks * stride);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
    if (wave < tiles && row_end + 16 * nt < sp.rows) {
      const int row = row_end + 16 * nt;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float v[C];
#pragma unroll
        for (int c = 0; c < C; ++c) v[c] = o[nt][c][r];
        part_store<C>(parts_at, it.chunk * stride + row * D + (4 * g_end + r) * C, v);
      }
      const float stat[2] = {m[nt], l[nt]};
      if (g_end == 0) part_store<2>(parts_at, it.chunk * stride + a.tile_rows * D + 2 * row, stat);
    }
  arrive_and_join<D, SPLIT>(a, s_o, parts_at, it, sp);
}

// ---- sequences of many rows: key tiles staged in LDS ---------------------------------
//
// A workgroup takes kManyRows rows of one key head (row = token * G + head of
// the group, so that the heads of a group share every key), a wave 32 of them.
// Per tile of 64 keys the codes are read once from memory, turned into f16 and
// laid down in LDS as v_mfma_f32_32x32x16_f16 wants them: keys row by row
// (16-byte pieces of 8 dimensions), values dimension by dimension (16-byte
// pieces of the 8 keys that a lane's weights belong to; dimensions in the order
// of the output tiles' rows), the rows padded by 16 bytes so that eight lanes hit
// eight different 16-byte banks.
// S^T and O^T as for few rows: lane 32 h + r holds row r; keys 8 i + 4 h ..+3 of
// a 32-key half are its scores and its half of the weights' operand, and output
// tile c holds dimensions i D/32 + c.  The next tile's codes are in flight in
// registers while this one is multiplied.
//
// Bound by the SIMDs' issue: of a tile's time the matrix pipe is busy for 38% and
// the vector pipe issues for 61% (32 exponentials and some 300 other operations a
// lane and tile of 64 keys, a quarter of them the staging), and the two hardly
// overlap with two waves a SIMD.  A prompt of 8192 tokens, 32 heads of 128 on 8,
// takes 650 us (850 TFLOP/s); 4096 tokens of 16 heads 127 us (531), of 256
// dimensions 245 us (560), of 64 92 us (370: half the products to the same
// exponentials); 8192 tokens of 16 heads of 256 900 us (610).  Tried and not kept: LDS for two tiles with one barrier (the
// same for 128, 285 us against 242 for 256), loops of their own for tiles without
// masks (64: 88 against 94, but 256: 402 against 242 for its spills), three waves a
// SIMD for 64 (116 against 99), priority for the products (702 us against 696).

constexpr int kManyRows = 128;
constexpr int kManyKeys = 64;
// LDS: a tile's keys and values, and for 31 chunks of a tile or more in a join
// (64 tokens of 16 heads of 128 behind 100,000 keys, 8 tiles: 182 us, 287 with 11)
constexpr int many_lds(int dim) {
  const int tile = kManyKeys * (2 * dim + 16) + dim * (2 * kManyKeys + 16);
  return tile > 36864 ? tile : 36864;
}

template <int D>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void k_kv_attention_many(KvAttnArgs a) {
  constexpr int SPLIT = 1;
  constexpr int S = D / 16, C = D / 32;      // 16-dimension steps, output tiles
  constexpr int KP = D / 64;                 // 16-byte pieces of a key tile a thread stages
  constexpr int VW = D == 256 ? 2 : 1;       // dwords of a value row a thread stages (8 keys of 4 VW dimensions)
  constexpr int VT = 8 * (D / (4 * VW));     // threads that stage values
  constexpr int KB = 2 * D + 16, VB = 2 * kManyKeys + 16;  // bytes of a key row, of a dimension's row
  __shared__ __attribute__((aligned(16))) uint8_t s_kv[many_lds(D)];
  uint8_t *const s_k = s_kv, *const s_v = s_kv + kManyKeys * KB;
  static_assert(sizeof(s_kv) >= kManyKeys * KB + D * VB && sizeof(s_kv) >= kJoinLds, "a tile's and the join's LDS");
  const int tid = threadIdx.x, lane = tid & 63, r32 = lane & 31, h = lane >> 5;
  const int wave = uniform(tid >> 6);
  Item it;
  if (!find_item(a, lane, it)) return;
  const Span sp = find_span(a, it);
  const int count = max(0, sp.key1 - sp.key0 + kManyKeys - 1) / kManyKeys;  // key tiles

  // lane i: 16-key tile i of a round of 16 key tiles
  auto round_id = [&](int round) { return tile_id(a, it.seq, sp.key0 + round * 16 * kManyKeys + 16 * lane, sp.key1); };
  const int id0 = round_id(0), id1 = round_id(1);

  // this lane's row, and what the wave's rows see
  const int wrow = wave * 32, row = wrow + r32;
  const bool busy = wrow < sp.rows;
  const RowAt w = row_at(a, sp, row < sp.rows ? row : 0, it.head);
  const int p = sp.first + w.tok, t = it.off + w.tok;
  const bool live = row < sp.rows && t >= 0 && t < a.tokens;
  const int vis_hi = a.causal ? p + 1 : it.len, vis_lo = a.window > 0 ? p - a.window + 1 : 0;
  const int tok_a = uniform(row_at(a, sp, wrow, it.head).tok);
  const int tok_b = uniform(row_at(a, sp, min(wrow + 31, sp.rows - 1), it.head).tok);
  const int all_hi = a.causal ? sp.first + tok_a + 1 : it.len, all_lo = a.window > 0 ? sp.first + tok_b - a.window + 1 : 0;
  const int any_hi = a.causal ? sp.first + tok_b + 1 : it.len, any_lo = a.window > 0 ? sp.first + tok_a - a.window + 1 : 0;
  QRaw<SPLIT> raw[S] = {};
  if (live) {
    const long at = (long)t * a.q_token + (long)w.head * a.q_head + 8 * h;
#pragma unroll
    for (int i = 0; i < S; ++i) raw[i] = load8((const QElem<SPLIT>*)a.q + at + 16 * i);
  }

  TileInfo info = tile_info(a, id0, it.head), next = tile_info(a, id1, it.head);
  const int mask = (1 << a.shift) - 1;
  // staging: pieces of keys (D / 16 a key), then 8 keys of 4 VW dimensions of the values
  const int kkey = tid / (D / 16), kpc = tid % (D / 16);  // first key (4096 / D further each piece)
  const int vgrp = tid / (D / (4 * VW)), vdim = (tid % (D / (4 * VW))) * 4 * VW;
  // group x of the values' eight: keys 32 (x >> 2) + 16 (x >> 1 & 1) + 4 (x & 1) + {0..3, 8..11}
  const int vkey = 32 * (vgrp >> 2) + 16 * ((vgrp >> 1) & 1) + 4 * (vgrp & 1);
  kv_u32x4 kr[KP];
  uint32_t vr[8][VW];
  auto load_tile = [&](const TileInfo& x, int i) {  // key tile i of the round
    auto at = [&](int key) {  // byte offset of a key's codes
      const long id = __shfl(x.id, 4 * i + (key >> 4), 64);
      return ((id * a.kv_heads + it.head) << a.shift | ((sp.key0 + 16 * (4 * i + (key >> 4)) + (key & 15)) & mask)) * D;
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
      *(h16x8*)(s_k + key * KB + 32 * kpc) = codes8(x[0], x[1]);
      *(h16x8*)(s_k + key * KB + 32 * kpc + 16) = codes8(x[2], x[3]);
    }
    if (VT == 256 || tid < VT) {
#pragma unroll
      for (int w = 0; w < VW; ++w) {
        uint32_t x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = vr[j][w] ^ 0x80808080u;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const int dim = vdim + 4 * w + b;
          *(h16x8*)(s_v + ((dim % C) * 32 + dim / C) * VB + 16 * vgrp) =
              b == 0 ? codes_across<0>(x) : b == 1 ? codes_across<1>(x) : b == 2 ? codes_across<2>(x) : codes_across<3>(x);
        }
      }
    }
  };
  if (count > 0) load_tile(info, 0);

  h16x8 qf[S];
  const int qe = split_q<SPLIT, S>(raw, a.type, a.sign, max32, qf, nullptr);
  const float c_row = __builtin_ldexpf(a.scale * kLog2e * kCodeScale, -qe);
  f32x16 o[C];
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[c][i] = 0.0f;
  float m = kMinusInf, l = 0.0f, l_before = 0.0f;  // l: of this round of tiles
  int ve = kNoScale;

  const uint8_t *const k_at = s_k + r32 * KB + 16 * h, *const v_at = s_v + r32 * VB + 16 * h;  // this lane's operands
  for (int i = 0; i < count; ++i) {
    const int ri = i & 15;
    if (ri == 0 && i) {
      info = next;
      next = tile_info(a, round_id((i >> 4) + 1), it.head);
      // One long sum of like terms would round the same way each time (4e-5 in 90,000
      // keys).  The outputs' accumulators stay: uncut rows of 131,072 keys alike are off
      // by up to 6e-4, where f16 rows allow 1e-3 and 128 rows' outputs of 128 dimensions
      // would take another 64 KB of LDS, half the workgroups.
      l_before += l;
      l = 0.0f;
    }
    __syncthreads();  // the previous tile has been read
    store_tile();
    __syncthreads();
    if (i + 1 < count) {
      if (ri == 15) load_tile(next, 0);
      else load_tile(info, ri + 1);
    }
    const int key = sp.key0 + i * kManyKeys;
    if (!busy || key >= any_hi || key + kManyKeys <= any_lo) continue;  // no row of the wave sees it
    // both 32-key halves' scores, then both halves' weights: the second half's
    // products run beside the first's exponentials
    f32x16 s[2];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      f32x16 x = {};
#pragma unroll
      for (int st = 0; st < S; ++st) {
        const h16x8 k = *(const h16x8*)(k_at + 32 * mt * KB + 32 * st);
        x = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, qf[st], x, 0, 0, 0);
      }
      s[mt] = x;
    }
    const bool edge = key < all_lo || key + kManyKeys > all_hi;
    float cs[4], vs[4];  // of the four 16-key tiles
    int e0 = kNoScale;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      cs[q] = c_row * lane_f(info.ks, 4 * ri + q);
      vs[q] = lane_f(info.vs, 4 * ri + q);
      // frexp_exp of a normal number, on the scalar unit (0 and what is below 2^-126 count as 2^-126)
      const int e = ((int)__float_as_uint(vs[q]) >> 23) - 126;
      e0 = max(e0, e < 129 ? e : kNoScale);
    }
    const int from = vis_lo, to = vis_hi;
    auto hide = [&](int mt, float with) {
      const int lo = from - 4 * h - here(key), hi = to - 4 * h - here(key);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int j = 32 * mt + 8 * (r >> 2) + (r & 3);
        s[mt][r] = j < lo || j >= hi ? with : s[mt][r];
      }
    };
    if (edge) {
      hide(0, kMinusInf);
      hide(1, kMinusInf);
      e0 = kNoScale;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int e = scale_exp(vs[q]);
        e0 = max(e0, key + 16 * q >= to || key + 16 * q + 16 <= from ? kNoScale : e);
      }
    }
    // the scores' factors are not negative, so each 16-key tile's largest is that of the products
    float top = kMinusInf;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float x = s[q >> 1][8 * (q & 1)];
#pragma unroll
      for (int r = 1; r < 8; ++r) x = fmaxf(x, s[q >> 1][8 * (q & 1) + r]);
      top = fmaxf(top, x * cs[q]);
    }
    top = max32(top);
    if (__any(top > m + kLag<SPLIT> || e0 > ve + kLagExp<SPLIT>)) {
      const float m1 = top > m + kLag<SPLIT> ? top : m;
      e0 = e0 > ve + kLagExp<SPLIT> ? e0 : ve;
      const float f = weight_of(m, m1), fo = __builtin_ldexpf(f, ve - e0);
      l *= f;
      l_before *= f;
#pragma unroll
      for (int c = 0; c < C; ++c) o[c] *= fo;
      m = m1;
      ve = e0;
    }
    float ws[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) ws[q] = __builtin_ldexpf(vs[q], kShift<SPLIT> - ve);
    float sum[2] = {};
    auto weights = [&](auto masked) {
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[mt][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[mt][r], cs[2 * mt + (r >> 3)], -m));
        if constexpr (masked) hide(mt, 0.0f);  // what the row does not see has weight 0 whatever its block's scales are
#pragma unroll
        for (int r = 0; r < 16; ++r) sum[mt] += s[mt][r];
#pragma unroll
        for (int r = 0; r < 16; ++r) s[mt][r] *= ws[2 * mt + (r >> 3)];
        if constexpr (masked) hide(mt, 0.0f);  // 0 * NaN, 0 * infinity
      }
    };
    if (edge) weights(std::true_type{});
    else weights(std::false_type{});
    l += sum[0];
    l += sum[1];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      h16x8 pf[2];
#pragma unroll
      for (int r = 0; r < 16; ++r) pf[r >> 3][r & 7] = (_Float16)s[mt][r];
#pragma unroll
      for (int st = 0; st < 2; ++st)
#pragma unroll
        for (int c = 0; c < C; ++c) {
          const h16x8 v = *(const h16x8*)(v_at + 64 * mt + 32 * st + 32 * c * VB);
          o[c] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, pf[st], o[c], 0, 0, 0);
        }
    }
  }
  l = sum32(l_before + l);
  const float norm = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[c][r] = in_units<SPLIT>(o[c][r] * norm, ve);
  if (it.chunks == 1) {
    if (live) {
      const long at = (long)t * a.out_token + (long)w.head * a.out_head;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float v[C];
#pragma unroll
        for (int c = 0; c < C; ++c) v[c] = o[c][r];
        store_row<SPLIT, C>(a.out, at + (8 * (r >> 2) + 4 * h + (r & 3)) * C, a.type, v);
      }
      if (a.lse && h == 0) a.lse[(long)t * a.q_heads + w.head] = row_lse(m, l);
    }
    return;
  }
  if (!all_arrive(a, it)) return;
  constexpr int kStride = kManyRows * (D + 2);
  const __amdgpu_buffer_rsrc_t parts_at = part_rsrc(a.partial + (long)it.slot * kStride, (long)it.chunks * kStride);
  if (row < sp.rows) {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      float v[C];
#pragma unroll
      for (int c = 0; c < C; ++c) v[c] = o[c][r];
      part_store<C>(parts_at, it.chunk * kStride + row * D + (8 * (r >> 2) + 4 * h + (r & 3)) * C, v);
    }
    const float stat[2] = {m, l};
    if (h == 0) part_store<2>(parts_at, it.chunk * kStride + kManyRows * D + 2 * row, stat);
  }
  arrive_and_join<D, SPLIT>(a, (float*)s_kv, parts_at, it, sp);
}

template <int D>
static void launch_few(const KvAttnArgs& a, bool f32, bool pairs, unsigned grid, hipStream_t s) {
  if constexpr (D < 256)
    if (pairs) {
      if (f32) hipLaunchKernelGGL((k_kv_attention_few<D, 2, 2>), dim3(grid), dim3(256), 0, s, a);
      else hipLaunchKernelGGL((k_kv_attention_few<D, 1, 2>), dim3(grid), dim3(256), 0, s, a);
      return;
    }
  if (f32) hipLaunchKernelGGL((k_kv_attention_few<D, 2, 1>), dim3(grid), dim3(256), 0, s, a);
  else hipLaunchKernelGGL((k_kv_attention_few<D, 1, 1>), dim3(grid), dim3(256), 0, s, a);
}
static void launch_few(const KvAttnArgs& a, int dim, bool f32, bool pairs, unsigned grid, hipStream_t s) {
  if (dim == 64) launch_few<64>(a, f32, pairs, grid, s);
  else if (dim == 128) launch_few<128>(a, f32, pairs, grid, s);
  else launch_few<256>(a, f32, pairs, grid, s);
}
static void launch_many(const KvAttnArgs& a, int dim, unsigned grid, hipStream_t s) {
  if (dim == 64) hipLaunchKernelGGL(k_kv_attention_many<64>, dim3(grid), dim3(256), 0, s, a);
  else if (dim == 128) hipLaunchKernelGGL(k_kv_attention_many<128>, dim3(grid), dim3(256), 0, s, a);
  else hipLaunchKernelGGL(k_kv_attention_many<256>, dim3(grid), dim3(256), 0, s, a);
}

constexpr int kMaxGroup = 512;  // most query heads of a key head (row_at)
// 0, hipErrorInvalidValue or QHIP_DECLINE
static int check_batch(const qhip_kv_cache* cache, const qhip_kv_batch* b, int q_heads) {
  const int rc = kv_check_cache(cache);
  if (rc == (int)hipErrorInvalidValue || !b) return (int)hipErrorInvalidValue;
  if (b->nseq < 0 || b->nseq > kMaxCount || b->tokens < 0 || b->max_new < 0 || b->max_kv < 0 || b->table_width < 0) return (int)hipErrorInvalidValue;
  if (q_heads <= 0 || q_heads > 65535 || q_heads % cache->kv_heads) return (int)hipErrorInvalidValue;
  return rc ? rc : q_heads / cache->kv_heads > kMaxGroup ? QHIP_DECLINE : 0;
}

// One kernel's share of a batch: its sequences, tile and unit sizes, grid without
// and with a cut, items aimed for, and the workspace (0: no cut).
struct AttnPlan {
  int min_tokens, max_tokens, rows, key_shift, units, target, least;
  long grid, cut_grid, work;
};
// `tiles`: bound of the row tiles over all sequences and key heads.  Chunks of
// cut sequences are fewer than 4/3 of target (find_item), items than target +
// tiles.  Twice as many tiles as items aimed for are enough as they are.
static void plan_cut(AttnPlan& p, long tiles, int dim) {
  p.grid = p.cut_grid = tiles;
  const long most = (p.units + p.least - 1) / p.least;  // chunks of a tile
  if (tiles > 0 && most > 1 && tiles < 2L * p.target && tiles <= kMaxCut && tiles * p.units < 0x7FFFFFFFL) {
    p.cut_grid = tiles * most < p.target + tiles ? tiles * most : p.target + tiles;
    const long slots = tiles * most < 4L * p.target / 3 + 1 ? tiles * most : 4L * p.target / 3 + 1;
    p.work = kCountBytes + slots * p.rows * (dim + 2) * 4;
  }
}
static int units_of(int keys, int shift) { return (int)(((long)keys + (1 << shift) - 1) >> shift); }

// the few-row kernel's plan, then the many-row kernel's
static void attn_plans(const qhip_kv_cache* c, const qhip_kv_batch* b, int q_heads, int window, bool f32, AttnPlan* p) {
  const int group = q_heads / c->kv_heads;
  const long rows = (long)b->tokens * q_heads, most_rows = (long)b->max_new * group;  // in all, of a sequence's key head
  AttnPlan &few = p[0], &many = p[1];
  few = many = AttnPlan{};
  if (b->max_new == 0) return;
  const long many_tiles = rows / kManyRows + (long)b->nseq * c->kv_heads;
  // row tiles times key tiles (at most) from which the many-row kernel runs
  const long work = many_tiles * units_of(window > 0 && window < b->max_kv ? window : b->max_kv, 6);
  // (us, few-row / many-row kernel, bf16, 16 heads on 4: 2048 tokens of 128 48 / 57,
  // 4096 129 / 127, of 256 100 / 116 and 321 / 242; 512 tokens behind 8000 keys of 128
  // 97 / 87, 256 behind 4000 37 / 51; 256 behind 30,000 of 256 337 / 254, 64 behind
  // 100,000 332 / 349; of 64 512 behind 8000 66 / 51, 8192 tokens 288 /
  // 262, but 4096 87 / 95, whose 512 uneven tiles are one round of workgroups.)
  const bool use_many = !f32 && most_rows > kFewRows && work >= (c->head_dim == 256 ? 12000 : 8500);
  // where the sequences are half as long as the longest on average, what single
  // tokens there may be are few beside the tiles of the others, and a launch
  // that mostly finds no sequence costs 3 to 4 us
  const bool alike = use_many && (long)b->nseq * b->max_new <= 2L * b->tokens;
  few.max_tokens = many.min_tokens = alike ? 0 : use_many ? kFewRows / group : 0x7FFFFFFF;
  many.max_tokens = 0x7FFFFFFF;
  if (few.max_tokens > 0) {
    // Rows of a workgroup: more of them share the codes, fewer make more
    // workgroups.  (us at 16 / 32 / 64 rows, f32, 16 heads: 512 tokens of 128
    // dimensions 18.5 / 17.5 / 22.4, 1024 32 / 29 / 36, 4096 224 / 181 / 170, of 64
    // dimensions 131 / 128 / 127; of 256 512 tokens 23 / 26, 1024 52 / 46.  13
    // sequences of 5 tokens with 24 heads of 256: 24 / 30.  64 rows of 256
    // dimensions do not fit the registers.)  Twice a wave's rows at most: 32 of 256
    // dimensions, and beyond 16 (pairs) 64 of fewer.
    few.rows = most_rows <= 16 ? (int)most_rows : use_many || rows <= 8192 ? 16 : c->head_dim == 256 || rows < 40000 ? 32 : 64;
    few.key_shift = 5;
    few.units = units_of(b->max_kv, 5);
    // Items aimed for: a cut costs partial results and a join, too few leave CUs
    // idle.  (us at 384 / 512 / 768: 64 sequences of 2000 keys of 128 dimensions 30 /
    // 34 / 35, of 256 at 256 / 512 / 768 52 / 59 / 69.)  Fewest 32-key units of an
    // item: one token on 8000 keys 15.5 us with 4, 14.8 with 8; 256 f32 tokens behind
    // 4000 45.3 with 8, 44.0 with 16.
    few.target = c->head_dim == 256 ? 256 : 384;
    few.least = few.rows <= 16 ? 8 : 16;
    // beyond one a sequence and key head
    long more = most_rows <= few.rows ? 0 : rows / few.rows;
    if (use_many && more > 3L * b->nseq * c->kv_heads) more = 3L * b->nseq * c->kv_heads;
    plan_cut(few, more + (long)b->nseq * c->kv_heads, c->head_dim);
  }
  if (use_many) {
    many.rows = kManyRows;
    many.key_shift = 6;
    many.units = units_of(b->max_kv, 6);
    // two workgroups a CU, one where they have 256 dimensions (1021 tokens behind 5000
    // keys of 128: 103 us with 512, 115 with 256, 140 with 768; 512 behind 8000 of 256:
    // 156 with 256, 229 with 512)
    many.target = c->head_dim == 256 ? 256 : 512;
    many.least = 8;  // 64-key units (4: 91 us, 8: 88, 16: 87 for 512 tokens behind 8000)
    plan_cut(many, many_tiles, c->head_dim);
  }
}

}  // namespace qhip

using namespace qhip;

extern "C" long qhip_kv_attention_work_bytes(const qhip_kv_cache* cache, const qhip_kv_batch* batch, int q_heads) {
  if (check_batch(cache, batch, q_heads)) return -1;
  long work = 0;
  for (int f32 = 0; f32 < 2; ++f32) {
    AttnPlan p[2];
    attn_plans(cache, batch, q_heads, 0, f32, p);  // a window may only move rows to the plan of f32 rows
    for (const AttnPlan& x : p) work = x.work > work ? x.work : work;
  }
  return work;
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
  AttnPlan plans[2];
  attn_plans(cache, batch, q_heads, window, type == QHIP_TT_F32, plans);
  // rows and workgroups are counted in 32 bits
  if (plans[0].cut_grid > 0x7FFFFFFFL || plans[1].cut_grid > 0x7FFFFFFFL || (long)batch->tokens * q_heads > 0x7FFFFFFFL)
    return (int)hipErrorInvalidValue;
  KvAttnArgs a{};
  a.k = (const int8_t*)cache->k;
  a.v = (const int8_t*)cache->v;
  a.k_scale = cache->k_scale;
  a.v_scale = cache->v_scale;
  a.offsets = batch->offsets;
  a.kv_lens = batch->kv_lens;
  a.table = batch->table;
  a.q = d_q;
  a.out = d_out;
  a.lse = d_lse;
  a.q_token = q_token_stride;
  a.q_head = q_head_stride;
  a.out_token = out_token_stride;
  a.out_head = out_head_stride;
  a.nseq = batch->nseq;
  a.tokens = batch->tokens;
  a.width = batch->table_width;
  a.shift = kv_block_shift(cache->block_size);
  a.num_blocks = cache->num_blocks;
  a.kv_heads = cache->kv_heads;
  a.q_heads = q_heads;
  a.scale = fabsf(softmax_scale);
  a.sign = softmax_scale < 0.0f ? -1.0f : 1.0f;
  a.causal = causal;
  a.window = window < kMaxLen ? window : kMaxLen;
  a.type = type;
  a.group = q_heads / cache->kv_heads;
  a.group_inv = ((1 << 20) + a.group - 1) / a.group;
  a.counters = (unsigned*)d_work;
  a.partial = (float*)((char*)d_work + kCountBytes);
  // the two kernels share the workspace: they follow each other on the stream
  // and each leaves the counters at zero
  for (int i = 0; i < 2; ++i) {
    const AttnPlan& p = plans[i];
    if (p.grid == 0) continue;
    a.min_tokens = p.min_tokens;
    a.max_tokens = p.max_tokens;
    a.tile_rows = p.rows;
    a.key_shift = p.key_shift;
    a.cut = p.work > 0 && d_work && work_bytes >= p.work;
    // a little above kv_heads / target, so that rounding makes no item too many
    a.share = (float)cache->kv_heads / (float)p.target * 1.00001f;
    a.least = p.least;
    a.max_units = p.units;
    a.max_chunks = join_pairs(i == 0 ? kJoinLds : many_lds(cache->head_dim)) / p.rows;
    a.slots = a.cut ? (p.work - kCountBytes) / ((long)p.rows * (cache->head_dim + 2) * 4) : 0;
    const unsigned grid = (unsigned)(a.cut ? p.cut_grid : p.grid);
    if (i == 0) launch_few(a, cache->head_dim, type == QHIP_TT_F32, p.rows > 16, grid, (hipStream_t)stream);
    else launch_many(a, cache->head_dim, grid, (hipStream_t)stream);
  }
  return (int)hipGetLastError();
}
