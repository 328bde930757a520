// kv_cache.hip -- the 8-bit key/value cache without its attention: block
// tables and slot maps from request lengths, the append of new tokens, and
// reading blocks back.
#include "kv_internal.hpp"

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
constexpr int kTabSeqs = 1024;    // sequences of a chunk (256 threads x 4)
constexpr int kTabTokens = 1024;  // tokens of a workgroup

struct KvTablesArgs {
  const int *cached, *fresh, *free_list, *taken;
  int nseq, nfree, shift, width, tokens, entries;  // entries: table entries of a workgroup
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
  const int t_lo = (int)blockIdx.x * kTabTokens, t_hi = min(a.tokens, t_lo + kTabTokens);
  const int e_lo = (int)blockIdx.x * a.entries, e_hi = last ? 0x7FFFFFFF : e_lo + a.entries;
  const int mask = (1 << a.shift) - 1;
  const int taken = a.taken ? a.taken[0] : 0;
  int off0 = 0, fresh0 = 0;  // sums before the chunk
  for (int s0 = 0; s0 < a.nseq; s0 += kTabSeqs) {
    int c[4], n[4], f[4], nsum = 0, fsum = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = s0 + 4 * tid + k;
      c[k] = i < a.nseq ? max(a.cached[i], 0) : 0;
      n[k] = i < a.nseq ? max(a.fresh[i], 0) : 0;
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
    for (int t = max(t_lo, off0) + tid; t < min(t_hi, off1); t += 256) {
      const int i = find_le(s_off, cnt, t);
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
      a.slots[t] = entry >= 0 ? (entry << a.shift) | (p & mask) : -1;
      if (a.positions) a.positions[t] = p;
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
// follows the previous token's in the same block.  The workgroup of a run's
// first token handles the run for one head of the keys or of the values, the
// others end.  The values are read once into registers (up to kAppKeep pieces
// of eight a thread; what a longer run has beyond them is read again), their
// largest |x| taken as the maximum of the bit patterns (a NaN's is above an
// infinity's, so neither is lost), and the codes written.
constexpr int kAppKeep = 8;

struct KvAppendArgs {
  int8_t* codes[2];
  float* scales[2];
  const void* x[2];
  long token_stride[2], head_stride[2];
  const int* slots;
  int tokens, num_slots, shift, heads, dim;
};

__device__ __forceinline__ int code8(float x, float m) {
  const float r = __builtin_rintf(x * m);
  return r == r ? (int)fminf(fmaxf(r, -127.0f), 127.0f) : 0;
}

template <typename T>
__global__ __launch_bounds__(256) void k_kv_append(KvAppendArgs a) {
  __shared__ uint32_t s_max[4];
  const int t = blockIdx.x, h = blockIdx.y, z = blockIdx.z, tid = threadIdx.x, lane = tid & 63;
  const int slot = a.slots[t], size = 1 << a.shift, place = slot & (size - 1);
  if ((unsigned)slot >= (unsigned)a.num_slots) return;
  if (place > 0 && t > 0 && a.slots[t - 1] == slot - 1) return;
  // the run's length: the tokens whose slots follow, up to the block's end
  int n = 0;
  for (int c = 0; c < size; c += 64) {
    const int i = c + lane;
    const bool in = i < size - place && t + i < a.tokens && a.slots[t + i] == slot + i;
    const uint64_t m = __ballot(in);
    n += m == ~0ull ? 64 : __builtin_ctzll(~m);
    if (m != ~0ull) break;
  }
  const int lanes = a.dim >> 3, rows = 256 / lanes;  // lanes of a row, rows of a pass
  const int row0 = tid / lanes, d0 = (tid & (lanes - 1)) * 8;
  const T* x = (const T*)a.x[z] + (long)t * a.token_stride[z] + (long)h * a.head_stride[z] + d0;
  const long stride = a.token_stride[z];
  Raw8<T> keep[kAppKeep];
  uint32_t top = 0;
#pragma unroll
  for (int k = 0; k < kAppKeep; ++k) {
    const int r = row0 + k * rows;
    if (r < n) keep[k] = load8(x + r * stride);
  }
#pragma unroll
  for (int k = 0; k < kAppKeep; ++k)
    if (row0 + k * rows < n)
#pragma unroll
      for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint((float)keep[k].e[i]) & 0x7FFFFFFFu);
  for (int r = row0 + kAppKeep * rows; r < n; r += rows) {
    const Raw8<T> v = load8(x + r * stride);
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint((float)v.e[i]) & 0x7FFFFFFFu);
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d, 64));
  if (lane == 0) s_max[tid >> 6] = top;
  const long bh = (long)(slot >> a.shift) * a.heads + h;
  const float old = place > 0 ? a.scales[z][bh] : 0.0f;
  __syncthreads();
  top = max(max(s_max[0], s_max[1]), max(s_max[2], s_max[3]));
  // maximum of non-negative floats as integers: NaN above infinity above all others
  const uint32_t sbits = max(__float_as_uint(__uint_as_float(top) / 127.0f) & 0x7FFFFFFFu, __float_as_uint(old));
  const float scale = __uint_as_float(sbits);
  const float inv = scale > 0.0f ? 1.0f / scale : 0.0f;
  int8_t* codes = a.codes[z] + bh * ((long)size * a.dim);
  if (place > 0 && sbits != __float_as_uint(old)) {
    const float ratio = scale > 0.0f ? old / scale : 0.0f;
    for (int i = tid; i < place * a.dim / 8; i += 256) {
      kv_u32x2 v = ((kv_u32x2*)codes)[i];
      int8_t* b = (int8_t*)&v;
#pragma unroll
      for (int j = 0; j < 8; ++j) b[j] = (int8_t)code8((float)b[j], ratio);
      ((kv_u32x2*)codes)[i] = v;
    }
  }
  auto put = [&](int r, const Raw8<T>& v) {
    kv_u32x2 w;
    int8_t* b = (int8_t*)&w;
#pragma unroll
    for (int j = 0; j < 8; ++j) b[j] = (int8_t)code8((float)v.e[j], inv);
    *(kv_u32x2*)(codes + (long)(place + r) * a.dim + d0) = w;
  };
#pragma unroll
  for (int k = 0; k < kAppKeep; ++k)
    if (row0 + k * rows < n) put(row0 + k * rows, keep[k]);
  for (int r = row0 + kAppKeep * rows; r < n; r += rows) put(r, load8(x + r * stride));
  if (tid == 0) a.scales[z][bh] = scale;
}

// ---- read back ----------------------------------------------------------------------

struct KvReadArgs {
  const int8_t* codes[2];
  const float* scales[2];
  void* out[2];
  const int* blocks;
  long pieces;  // 16-code pieces of one block's head
  int num_blocks, heads;
};

template <typename T>
__global__ __launch_bounds__(256) void k_kv_read(KvReadArgs a) {
  const int h = blockIdx.y, z = blockIdx.z;
  if (!a.out[z]) return;
  const int id = a.blocks[blockIdx.x];
  const bool in = (unsigned)id < (unsigned)a.num_blocks;
  const long bh = in ? (long)id * a.heads + h : 0;
  const float scale = in ? a.scales[z][bh] : __builtin_nanf("");
  const long to = ((long)blockIdx.x * a.heads + h) * a.pieces;
  for (long i = threadIdx.x; i < a.pieces; i += 256) {
    kv_u32x4 c = {0, 0, 0, 0};
    if (in) c = ((const kv_u32x4*)a.codes[z])[bh * a.pieces + i];
    const int8_t* b = (const int8_t*)&c;
    T v[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = (T)((float)b[j] * scale);
    kv_u32x4* o = (kv_u32x4*)((T*)a.out[z] + 16 * (to + i));
#pragma unroll
    for (unsigned j = 0; j < sizeof(v) / 16; ++j) o[j] = ((const kv_u32x4*)v)[j];
  }
}

}  // namespace qhip

using namespace qhip;

extern "C" int qhip_launch_kv_tables(const int* d_cached, const int* d_new, int nseq, const int* d_free, int nfree,
                                     const int* d_taken, int block_size, int* d_table, int table_width, int tokens,
                                     int* d_offsets, int* d_kv_lens, int* d_slots, int* d_positions, int* d_taken_out,
                                     void* stream) {
  const int shift = kv_block_shift(block_size);
  if (shift < 0 || nseq < 0 || nfree < 0 || table_width < 0 || tokens < 0) return (int)hipErrorInvalidValue;
  if (!d_offsets || !d_taken_out || (nseq > 0 && (!d_cached || !d_new || !d_kv_lens)) || (nfree > 0 && !d_free) ||
      (nseq > 0 && table_width > 0 && !d_table) || (tokens > 0 && !d_slots))
    return (int)hipErrorInvalidValue;
  // every workgroup walks all sequences, so the grid follows the tokens; the
  // fresh blocks number at most tokens / block_size + nseq
  const int grid = tokens > 0 ? (tokens - 1) / kTabTokens + 1 : 1;
  const int entries = (int)((((long)tokens >> shift) + nseq) / grid + 1);
  hipLaunchKernelGGL(k_kv_tables, dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream,
                     KvTablesArgs{d_cached, d_new, d_free, d_taken, nseq, nfree, shift, table_width, tokens, entries,
                                  d_table, d_offsets, d_kv_lens, d_slots, d_positions, d_taken_out});
  return (int)hipGetLastError();
}

extern "C" int qhip_launch_kv_append(const qhip_kv_cache* cache, int type, const void* d_k, long k_token_stride,
                                     long k_head_stride, const void* d_v, long v_token_stride, long v_head_stride,
                                     const int* d_slots, int tokens, void* stream) {
  const int rc = kv_check_cache(cache), size = kv_type_size(type);
  if (rc == (int)hipErrorInvalidValue || !size || tokens < 0) return (int)hipErrorInvalidValue;
  if (tokens > 0 && (!d_k || !d_v || !d_slots || ((uintptr_t)d_k % size) || ((uintptr_t)d_v % size)))
    return (int)hipErrorInvalidValue;
  if (rc) return rc;
  if (tokens == 0) return 0;
  const int num_slots = cache->num_blocks * cache->block_size;
  const KvAppendArgs a{{(int8_t*)cache->k, (int8_t*)cache->v}, {cache->k_scale, cache->v_scale}, {d_k, d_v},
                       {k_token_stride, v_token_stride}, {k_head_stride, v_head_stride}, d_slots, tokens, num_slots,
                       kv_block_shift(cache->block_size), cache->kv_heads, cache->head_dim};
  const dim3 grid((unsigned)tokens, (unsigned)cache->kv_heads, 2);
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
                     {d_k_out, d_v_out}, d_blocks, (long)cache->block_size * cache->head_dim / 16, cache->num_blocks,
                     cache->kv_heads};
  const dim3 grid((unsigned)nblocks, (unsigned)cache->kv_heads, 2);
  hipStream_t s = (hipStream_t)stream;
  if (type == QHIP_TT_F32) hipLaunchKernelGGL(k_kv_read<float>, grid, dim3(256), 0, s, a);
  else if (type == QHIP_TT_F16) hipLaunchKernelGGL(k_kv_read<f16_t>, grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL(k_kv_read<bf16_t>, grid, dim3(256), 0, s, a);
  return (int)hipGetLastError();
}
