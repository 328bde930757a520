// kv_cache.hip -- the 8-bit key/value cache without its attention: block
// tables and slot maps from request lengths, the append of new tokens, and
// reading blocks back.
#include "kv_internal.hpp"

#include <type_traits>

namespace qhip {

// ---- block tables and slot maps --------------------------------------------------
//
// With B tokens a block, sequence i has before_i = ceil(c_i / B) blocks and
// needs need_i = ceil((c_i + n_i) / B); its fresh ones are entries F_i = taken +
// sum_{j<i} (need_j - before_j) on of the free list, its packed tokens start at
// O_i = sum_{j<i} n_j.  Everything follows from the two prefix sums, so each
// workgroup computes them for itself, 1024 sequences at a time (four a thread,
// two scans), and then fills its own share of the tokens and of the table's
// new entries, each by a search in the sums: one launch, nothing handed from
// one workgroup to another.
//
// Bound by the launch and one chain of loads (lengths, held entry, free entry):
// 4.2 us for 64 sequences of a token each (1.5 KB), 7.5 us for 1000 sequences of
// 100,000 tokens (0.8 MB), of which the scans and searches are about 2.
constexpr int kTabSeqs = 1024;  // sequences of a chunk (256 threads x 4)

struct KvTablesArgs {
  const int *cached, *fresh, *free_list, *taken;
  int nseq, nfree, shift, width, tokens, each, entries;  // tokens of a thread, table entries of a workgroup
  int *table, *offsets, *kv_lens, *slots, *positions, *taken_out;
};

// largest i in [0, cnt) with a[i] <= x (a ascending, a[0] <= x)
__device__ __forceinline__ int find_le(const int* a, int cnt, int x) {
  int lo = 0, hi = cnt;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

__global__ __launch_bounds__(256) void k_kv_tables(KvTablesArgs a) {
  __shared__ int s_len[kTabSeqs], s_off[kTabSeqs + 1], s_fresh[kTabSeqs + 1], s_wave[2][4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const bool last = blockIdx.x == gridDim.x - 1;
  const int t_lo = (int)blockIdx.x * 256 * a.each, t_hi = min(a.tokens, t_lo + 256 * a.each);
  const int e_lo = (int)blockIdx.x * a.entries, e_hi = last ? 0x7FFFFF00 : e_lo + a.entries;
  const int mask = (1 << a.shift) - 1;
  const int taken = a.taken ? a.taken[0] : 0;
  int off0 = 0, fresh0 = 0;  // sums before the chunk
  for (int s0 = 0; s0 < a.nseq; s0 += kTabSeqs) {
    int c[4], n[4], f[4], nsum = 0, fsum = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = s0 + 4 * tid + k;
      c[k] = i < a.nseq ? min(max(a.cached[i], 0), kMaxLen) : 0;
      n[k] = i < a.nseq ? min(max(a.fresh[i], 0), kMaxLen - c[k]) : 0;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      f[k] = ((c[k] + n[k] + mask) >> a.shift) - ((c[k] + mask) >> a.shift);
      nsum += n[k];
      fsum += f[k];
    }
    const int ni = scan64(nsum), fi = scan64(fsum);
    if (lane == 63) {
      s_wave[0][wave] = ni;
      s_wave[1][wave] = fi;
    }
    __syncthreads();
    int o = off0 + ni - nsum, r = fresh0 + fi - fsum;
    for (int w = 0; w < wave; ++w) {
      o += s_wave[0][w];
      r += s_wave[1][w];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      s_len[4 * tid + k] = c[k];
      s_off[4 * tid + k] = o;
      s_fresh[4 * tid + k] = r;
      o += n[k];
      r += f[k];
    }
    if (tid == 255) {
      s_off[kTabSeqs] = o;
      s_fresh[kTabSeqs] = r;
    }
    __syncthreads();
    const int cnt = min(kTabSeqs, a.nseq - s0);
    const int off1 = s_off[kTabSeqs], fresh1 = s_fresh[kTabSeqs];
    if ((unsigned)(s0 / kTabSeqs) % gridDim.x == blockIdx.x)
      for (int i = tid; i < cnt; i += 256) {
        a.offsets[s0 + i] = s_off[i];
        a.kv_lens[s0 + i] = s_len[i] + (s_off[i + 1] - s_off[i]);
      }
    // a.each consecutive tokens a thread
    const int t0 = t_lo + a.each * tid, t1 = min(min(t0 + a.each, t_hi), off1), tb = max(t0, off0);
    if (tb < t1) {
      int i = find_le(s_off, cnt, tb), slot[4], place[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int t = t0 + k;
        if (t < tb || t >= t1) continue;
        while (i + 1 < cnt && s_off[i + 1] <= t) ++i;
        const int p = s_len[i] + (t - s_off[i]);
        const int j = p >> a.shift, before = (s_len[i] + mask) >> a.shift;
        int entry = -1;
        if ((unsigned)j < (unsigned)a.width) {
          const int at = taken + s_fresh[i] + (j - before);
          if (j < before)
            entry = a.table[(long)(s0 + i) * a.width + j];
          else if ((unsigned)at < (unsigned)a.nfree)
            entry = a.free_list[at];
        }
        // (a larger id is outside every pool, and its slot would not fit 31 bits)
        slot[k] = (unsigned)entry <= 0x7FFFFFFFu >> a.shift ? (entry << a.shift) | (p & mask) : -1;
        place[k] = p;
      }
      typedef int int4_a4 __attribute__((ext_vector_type(4), aligned(4)));
      if (t1 - tb == 4) {
        *(int4_a4*)(a.slots + t0) = int4_a4{slot[0], slot[1], slot[2], slot[3]};
        if (a.positions) *(int4_a4*)(a.positions + t0) = int4_a4{place[0], place[1], place[2], place[3]};
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (t0 + k >= tb && t0 + k < t1) {
            a.slots[t0 + k] = slot[k];
            if (a.positions) a.positions[t0 + k] = place[k];
          }
      }
    }
    for (int e = max(e_lo, fresh0) + tid; e < min(e_hi, fresh1); e += 256) {
      const int i = find_le(s_fresh, cnt, e);
      const int j = ((s_len[i] + mask) >> a.shift) + (e - s_fresh[i]), at = taken + e;
      if ((unsigned)j < (unsigned)a.width)
        a.table[(long)(s0 + i) * a.width + j] = (unsigned)at < (unsigned)a.nfree ? a.free_list[at] : -1;
    }
    off0 = off1;
    fresh0 = fresh1;
    __syncthreads();
  }
  for (int t = max(t_lo, off0) + tid; t < t_hi; t += 256) {  // padding
    a.slots[t] = -1;
    if (a.positions) a.positions[t] = 0;
  }
  if (last && tid == 0) {
    a.offsets[a.nseq] = off0;
    a.taken_out[0] = taken + fresh0;
  }
}

// ---- append -----------------------------------------------------------------------
//
// A run is the new tokens of one block: a token begins one unless its slot
// follows the previous token's in the same block.  A workgroup finds the runs
// that begin among its kAppTokens (or, in a batch of few tokens, at its one)
// token, for one head of the keys or of the values.  A run whose values fit one
// wave's registers is a wave's, so that a batch of single tokens keeps all four
// busy; a longer one is the workgroup's.  The values are read once, into
// registers (kAppKeep pieces of eight a thread; what a run has beyond them is
// read again), their largest |x| taken as the maximum of the bit patterns (a
// NaN's is above an infinity's, so neither is lost), and the codes written.  The
// scale is the product with the f32 nearest 1/127: within one unit in the last
// place of the quotient, and one multiply.
//
// Prompts are bound by reading the new values: 4600 f32 tokens of 4 heads of 256
// (47 MB) 12.4 us, 3.8 TB/s.  16-bit ones take as long for 28 MB (13.0 us, of 8 heads of
// 128 13.6): as many pieces in flight, each of half the bytes, and of blocks of 64
// tokens three tiles in four find no run.  Single tokens are bound by the chain slots - values
// - maximum - codes: 64 tokens of 8 heads of 128 in 4.5 us.
constexpr int kAppKeep = 8;
// One token a workgroup up to kAppFew tokens: single tokens are a run each, which
// a wave would otherwise take in turn, a prompt's workgroups mostly find no run.
// (us, one / 16 a workgroup, bf16 8 heads of 128: 32 single tokens 3.7 / 9.8, 128
// 5.9 / 11.2, 256 8.9 / 11.2, 512 15.2 / 11.3; a prompt of 32 4.3 / 4.1, of 128 7.8 /
// 4.7, of 256 12.3 / 4.8, of 1024 45 / 5.6)
constexpr int kAppTokens = 16;
constexpr int kAppFew = 128;

struct KvAppendArgs {
  int8_t* codes[2];
  float* scales[2];
  const void* x[2];
  long token_stride[2], head_stride[2];
  const int* slots;
  int tokens, num_slots, shift, heads, dim, tile, tiles, span;  // span: log2 of the tiles of a block
};

__device__ __forceinline__ int code8(float x, float m) {
  const float r = __builtin_rintf(x * m);
  return r == r ? (int)fminf(fmaxf(r, -127.0f), 127.0f) : 0;
}
// four codes in a dword
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d, float m) {
  return (code8(a, m) & 0xFF) | (code8(b, m) & 0xFF) << 8 | (code8(c, m) & 0xFF) << 16 | (uint32_t)code8(d, m) << 24;
}
__device__ __forceinline__ float sbyte(uint32_t w, int i) { return (float)(int8_t)(w >> (8 * i)); }

// The run of `n` tokens from token t on, at `slot`; this thread is `id` of NT
// (a wave, or the workgroup's four with s_max between them), keeping KEEP pieces.
template <typename T, int NT, int KEEP>
__device__ __forceinline__ void append_run(const KvAppendArgs& a, int t, int slot, int n, int h, int z, int id, uint32_t* s_max) {
  const int size = 1 << a.shift, place = slot & (size - 1);
  const int lanes = a.dim >> 3, rows = NT / lanes;  // lanes of a row, rows of a pass
  const int row0 = id / lanes, d0 = (id & (lanes - 1)) * 8;
  const long stride = a.token_stride[z];
  const T* x = (const T*)a.x[z] + (long)t * stride + (long)h * a.head_stride[z] + d0;
  const long bh = (long)(slot >> a.shift) * a.heads + h;
  const float old = place > 0 ? a.scales[z][bh] : 0.0f;
  Raw8<T> keep[KEEP];
  uint32_t top = 0;
#pragma unroll
  for (int k = 0; k < KEEP; ++k)
    if (row0 + k * rows < n) keep[k] = load8(x + (row0 + k * rows) * stride);
  auto see = [&](const Raw8<T>& v) {
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint((float)v.e[i]) & 0x7FFFFFFFu);
  };
#pragma unroll
  for (int k = 0; k < KEEP; ++k)
    if (row0 + k * rows < n) see(keep[k]);
  for (int r = row0 + KEEP * rows; r < n; r += rows) see(load8(x + r * stride));
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d, 64));
  if constexpr (NT > 64) {
    if ((id & 63) == 0) s_max[id >> 6] = top;
    __syncthreads();
    top = max(max(s_max[0], s_max[1]), max(s_max[2], s_max[3]));
    __syncthreads();  // read before the next run's
  }
  // maximum of non-negative floats as integers: NaN above infinity above all others
  const uint32_t sbits = max(__float_as_uint(__uint_as_float(top) * (1.0f / 127.0f)) & 0x7FFFFFFFu, __float_as_uint(old));
  const float scale = __uint_as_float(sbits);
  const float inv = scale > 0.0f ? 1.0f / scale : 0.0f;
  int8_t* codes = a.codes[z] + bh * ((long)size * a.dim);
  if (place > 0 && sbits != __float_as_uint(old)) {  // the tokens before the run, to the new scale
    const float ratio = scale > 0.0f ? old / scale : 0.0f;
    for (int i = id; i < place * a.dim / 8; i += NT) {
      const kv_u32x2 v = ((const kv_u32x2*)codes)[i];
      ((kv_u32x2*)codes)[i] = kv_u32x2{codes4(sbyte(v[0], 0), sbyte(v[0], 1), sbyte(v[0], 2), sbyte(v[0], 3), ratio),
                                       codes4(sbyte(v[1], 0), sbyte(v[1], 1), sbyte(v[1], 2), sbyte(v[1], 3), ratio)};
    }
  }
  auto put = [&](int r, const Raw8<T>& v) {
    *(kv_u32x2*)(codes + (long)(place + r) * a.dim + d0) =
        kv_u32x2{codes4((float)v.e[0], (float)v.e[1], (float)v.e[2], (float)v.e[3], inv),
                 codes4((float)v.e[4], (float)v.e[5], (float)v.e[6], (float)v.e[7], inv)};
  };
#pragma unroll
  for (int k = 0; k < KEEP; ++k)
    if (row0 + k * rows < n) put(row0 + k * rows, keep[k]);
  for (int r = row0 + KEEP * rows; r < n; r += rows) put(r, load8(x + r * stride));
  if (id == 0) a.scales[z][bh] = scale;
}

template <typename T>
__global__ __launch_bounds__(256) void k_kv_append(KvAppendArgs a) {
  __shared__ uint32_t s_max[4];
  const int tid = threadIdx.x, lane = tid & 63, size = 1 << a.shift;
  int item = blockIdx.x, h = blockIdx.y, z = blockIdx.z;
  if (a.tile > 1) {  // eight blocks' tiles side by side (an XCD each), of a tile all heads, keys and values
    const unsigned parts = 2u * a.heads, at = blockIdx.x >> 3;
    const unsigned tile = __builtin_amdgcn_readfirstlane(at / parts), part = at - tile * parts;  // (a division is a vector's)
    item = (int)(((((tile >> a.span) << 3) + (blockIdx.x & 7)) << a.span) + (tile & ((1u << a.span) - 1)));
    if (item >= a.tiles) return;
    z = (int)part >= a.heads;
    h = (int)part - z * a.heads;
  }
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int t0 = item * a.tile;
  // the tokens of the tile that begin a run (a lane each)
  int slot = -1;
  bool begins = false;
  if (lane < a.tile && t0 + lane < a.tokens) {
    slot = a.slots[t0 + lane];
    const int before = t0 + lane > 0 ? a.slots[t0 + lane - 1] : -1;
    begins = (unsigned)slot < (unsigned)a.num_slots && ((slot & (size - 1)) == 0 || before != slot - 1 || t0 + lane == 0);
  }
  uint64_t runs = __ballot(begins);
  for (int i = 0; runs; ++i, runs &= runs - 1) {
    const int at = __builtin_ctzll(runs), t = t0 + at, first = __builtin_amdgcn_readlane(slot, at);
    // its length: the tokens whose slots follow, up to the block's end
    int n = 0;
    for (int c = 0; c < size; c += 64) {
      const int j = c + lane;
      const bool in = j < size - (first & (size - 1)) && t + j < a.tokens && a.slots[t + j] == first + j;
      const uint64_t m = __ballot(in);
      n += m == ~0ull ? 64 : __builtin_ctzll(~m);
      if (m != ~0ull) break;
    }
    if (n * a.dim <= 64 * 8) {
      if ((i & 3) == wave) append_run<T, 64, 1>(a, t, first, n, h, z, lane, s_max);
    } else {
      append_run<T, 256, kAppKeep>(a, t, first, n, h, z, tid, s_max);
    }
  }
}

// ---- read back ----------------------------------------------------------------------
//
// A workgroup's share of one block's head: kReadCodes codes, a 16-byte piece of
// the output a thread and pass, so that a wave's stores are contiguous.  Bound by
// the writes: f32 out of 9 MB of codes (46 MB in all) 9.5 us, 4.8 TB/s.
constexpr int kReadCodes = 4096;

struct KvReadArgs {
  const int8_t* codes[2];
  const float* scales[2];
  void* out[2];
  const int* blocks;
  int size, num_blocks, heads;  // size: codes of a block's head
};

template <typename T>
__global__ __launch_bounds__(256) void k_kv_read(KvReadArgs a) {
  constexpr int P = 16 / sizeof(T);  // values of a piece
  typedef typename std::conditional<P == 4, uint32_t, kv_u32x2>::type Codes;
  const int z = blockIdx.z;
  if (!a.out[z]) return;
  const int i = (int)blockIdx.x / a.heads, h = (int)blockIdx.x - i * a.heads, id = a.blocks[i];
  const bool in = (unsigned)id < (unsigned)a.num_blocks;
  const long bh = in ? (long)id * a.heads + h : 0;
  const float scale = in ? a.scales[z][bh] : __builtin_nanf("");
  const int8_t* codes = a.codes[z] + bh * a.size;
  T* out = (T*)a.out[z] + (long)blockIdx.x * a.size;
  const int c0 = (int)blockIdx.y * kReadCodes, c1 = min(a.size, c0 + kReadCodes);
#pragma unroll
  for (int k = 0; k < kReadCodes / (256 * P); ++k) {
    const int c = c0 + (k * 256 + (int)threadIdx.x) * P;
    if (c >= c1) break;
    const Codes x = *(const Codes*)(codes + c);
    const uint32_t* w = (const uint32_t*)&x;
    T v[P];
#pragma unroll
    for (int j = 0; j < P; ++j) v[j] = (T)(sbyte(w[j >> 2], j & 3) * scale);
    *(kv_u32x4*)(out + c) = *(const kv_u32x4*)v;
  }
}

}  // namespace qhip

using namespace qhip;

struct Ints {
  const int* at;
  long n;
};
static bool overlap(const Ints& a, const Ints& b) {
  return a.at && b.at && a.n > 0 && b.n > 0 && a.at < b.at + b.n && b.at < a.at + a.n;
}

extern "C" int qhip_launch_kv_tables(const int* d_cached, const int* d_new, int nseq, const int* d_free, int nfree,
                                     const int* d_taken, int block_size, int* d_table, int table_width, int tokens,
                                     int* d_offsets, int* d_kv_lens, int* d_slots, int* d_positions, int* d_taken_out,
                                     void* stream) {
  const int shift = kv_block_shift(block_size);
  if (shift < 0 || nseq < 0 || nseq > kMaxCount || nfree < 0 || table_width < 0 || tokens < 0 || tokens > kMaxCount)
    return (int)hipErrorInvalidValue;
  if (!d_offsets || !d_taken_out || (nseq > 0 && (!d_cached || !d_new || !d_kv_lens)) || (nfree > 0 && !d_free) ||
      (nseq > 0 && table_width > 0 && !d_table) || (tokens > 0 && !d_slots))
    return (int)hipErrorInvalidValue;
  // (an output in an input's place would be read by workgroups that start later)
  const Ints table{d_table, (long)nseq * table_width}, in[] = {{d_cached, nseq}, {d_new, nseq}, {d_taken, 1}, {d_free, nfree}},
             out[] = {{d_offsets, nseq + 1L}, {d_kv_lens, nseq}, {d_slots, tokens}, {d_positions, tokens}, {d_taken_out, 1}};
  for (const Ints& x : in)
    if (overlap(x, table)) return (int)hipErrorInvalidValue;
  for (const Ints& y : out) {
    for (const Ints& x : in)
      if (overlap(x, y)) return (int)hipErrorInvalidValue;
    for (const Ints& z : out)
      if (&z != &y && overlap(z, y)) return (int)hipErrorInvalidValue;
    if (overlap(table, y)) return (int)hipErrorInvalidValue;
  }
  // every workgroup walks all sequences, so the grid follows the tokens; the
  // fresh blocks number at most tokens / block_size + nseq
  // (four tokens a thread share a search and 16-byte stores: 100,000 tokens of
  // 1000 ragged sequences 7.1 us against 7.8; the 64 of a decode step 5.7 us
  // against 4.4)
  const int each = tokens > 4096 ? 4 : 1;
  const int grid = tokens > 0 ? (tokens - 1) / (256 * each) + 1 : 1;
  const int entries = (int)((((long)tokens >> shift) + nseq) / grid + 1);
  hipLaunchKernelGGL(k_kv_tables, dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream,
                     KvTablesArgs{d_cached, d_new, d_free, d_taken, nseq, nfree, shift, table_width, tokens, each, entries,
                                  d_table, d_offsets, d_kv_lens, d_slots, d_positions, d_taken_out});
  return (int)hipGetLastError();
}

extern "C" int qhip_launch_kv_append(const qhip_kv_cache* cache, int type, const void* d_k, long k_token_stride,
                                     long k_head_stride, const void* d_v, long v_token_stride, long v_head_stride,
                                     const int* d_slots, int tokens, void* stream) {
  const int rc = kv_check_cache(cache), size = kv_type_size(type);
  if (rc == (int)hipErrorInvalidValue || !size || tokens < 0 || tokens > kMaxCount) return (int)hipErrorInvalidValue;
  if (tokens > 0 && (!d_k || !d_v || !d_slots || ((uintptr_t)d_k % size) || ((uintptr_t)d_v % size)))
    return (int)hipErrorInvalidValue;
  if (rc) return rc;
  if (tokens == 0) return 0;
  const int num_slots = cache->num_blocks * cache->block_size, tile = tokens > kAppFew ? kAppTokens : 1;
  const int tiles = (tokens - 1) / tile + 1, span = kv_block_shift(cache->block_size) - 4;
  static_assert(kAppTokens == 16, "span");
  const KvAppendArgs a{{(int8_t*)cache->k, (int8_t*)cache->v}, {cache->k_scale, cache->v_scale}, {d_k, d_v},
                       {k_token_stride, v_token_stride}, {k_head_stride, v_head_stride}, d_slots, tokens, num_slots,
                       kv_block_shift(cache->block_size), cache->kv_heads, cache->head_dim,
                       tile, tiles, span};
  // An XCD takes all heads of a block's tokens: whole rows through one L2, and a
  // run (mostly a whole block) on each of the eight.  4600 tokens, us, so / the
  // tokens in the grid's order, whose runs fall on two XCDs / one XCD a head: bf16 8
  // heads of 128 13.7 / 24.1 / 15.4, 4 of 256 12.8 / 21.9 / 18.8, f32 12.2 / 19.5 / 15.4.
  // Single tokens in the grid's order (64 of 8 heads: 4.5 against 5.8 by head).
  const long round = 8L << span, parts = 2L * cache->kv_heads, items = (tiles + round - 1) / round * round * parts;
  if (tile > 1 && items > 0x7FFFFFFFL) return (int)hipErrorInvalidValue;
  const dim3 grid = tile > 1 ? dim3((unsigned)items) : dim3(tiles, cache->kv_heads, 2);
  hipStream_t s = (hipStream_t)stream;
  if (type == QHIP_TT_F32) hipLaunchKernelGGL(k_kv_append<float>, grid, dim3(256), 0, s, a);
  else if (type == QHIP_TT_F16) hipLaunchKernelGGL(k_kv_append<f16_t>, grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL(k_kv_append<bf16_t>, grid, dim3(256), 0, s, a);
  return (int)hipGetLastError();
}

extern "C" int qhip_launch_kv_read(const qhip_kv_cache* cache, const int* d_blocks, int nblocks, int type,
                                   void* d_k_out, void* d_v_out, void* stream) {
  const int rc = kv_check_cache(cache), size = kv_type_size(type);
  if (rc == (int)hipErrorInvalidValue || !size || nblocks < 0 || !aligned16(d_k_out) || !aligned16(d_v_out) ||
      (nblocks > 0 && !d_blocks))
    return (int)hipErrorInvalidValue;
  if (rc) return rc;
  if (nblocks == 0 || (!d_k_out && !d_v_out)) return 0;
  const KvReadArgs a{{(const int8_t*)cache->k, (const int8_t*)cache->v}, {cache->k_scale, cache->v_scale},
                     {d_k_out, d_v_out}, d_blocks, cache->block_size * cache->head_dim, cache->num_blocks, cache->kv_heads};
  if ((long)nblocks * a.heads > 0x7FFFFFFFL) return (int)hipErrorInvalidValue;
  const dim3 grid((unsigned)(nblocks * a.heads), (unsigned)((a.size + kReadCodes - 1) / kReadCodes), 2);
  hipStream_t s = (hipStream_t)stream;
  if (type == QHIP_TT_F32) hipLaunchKernelGGL(k_kv_read<float>, grid, dim3(256), 0, s, a);
  else if (type == QHIP_TT_F16) hipLaunchKernelGGL(k_kv_read<f16_t>, grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL(k_kv_read<bf16_t>, grid, dim3(256), 0, s, a);
  return (int)hipGetLastError();
}
