// rope.hip -- rotary positions of queries and keys.
//
// Pair i of a head's first rot_dim values is turned by position * f_i radians:
//   (a, b) -> gain (a cos - b sin, b cos + a sin)
// with a, b = values i and i + rot_dim / 2 (halves) or 2 i and 2 i + 1 (pairs side
// by side); the values behind rot_dim are copied.
//
// An angle is kept in turns: steps[i] is f_i / 2 pi as a fraction of 2^64, so
// position * steps[i] mod 2^64 is the place on the circle, exact to 2^-32 turns at
// any position, without a floating reduction of a large angle.
//
// Memory bounds it: 4097 tokens of 10 heads of 256 in f32 22 us (3.8 TB/s of the 5.1 of a copy),
// 8192 of 40 heads of 128 in bf16 38 us (4.4), inputs from memory and outputs into memory not
// used before; 18 and 30 us into what the call before wrote, which the last cache still holds.
// 64 tokens of 20 heads 5.8 us, a chain of loads and the angles.
#include "qhip_internal.hpp"
#include "rows_internal.hpp"

#include <algorithm>
#include <cmath>

namespace qhip {

// most values that turn, and that are copied: 256 lanes hold a head
constexpr int kRopeMost = 1024;

struct RopeArgs {
  const void* x[2];
  void* out[2];
  long token[2], head[2], out_token[2], out_head[2];
  const uint64_t* steps;
  const int* positions;
  float gain;
  int tokens, q_heads, heads, dim, rot, interleaved;
  int lanes, pieces;  // lanes of a head (a power of two), pieces of eight pairs or values that they hold
  int each;           // heads of a lane
  int first;          // token of this launch
};

// cos and sin of `turn` / 2^32 turns: the nearest quarter by its top bits, then the
// Taylor sums of the rest, |y| <= pi / 4 (terms left out: 2e-9 and 1e-10).
__device__ __forceinline__ void cos_sin(uint32_t turn, float& c, float& s) {
  const uint32_t q = (turn + 0x20000000u) >> 30;
  const float y = (float)(int)(turn - (q << 30)) * 1.4629180792671596e-9f;  // 2 pi / 2^32
  const float z = y * y;
  float p = __builtin_fmaf(z, 2.7557319e-6f, -1.9841270e-4f);  // 1 / 9!, 1 / 7!
  p = __builtin_fmaf(z, p, 8.3333333e-3f);
  p = __builtin_fmaf(z, p, -1.6666667e-1f);
  const float sn = __builtin_fmaf(y * z, p, y);
  p = __builtin_fmaf(z, -2.7557319e-7f, 2.4801587e-5f);  // 1 / 10!, 1 / 8!
  p = __builtin_fmaf(z, p, -1.3888889e-3f);
  p = __builtin_fmaf(z, p, 4.1666667e-2f);
  p = __builtin_fmaf(z, p, -0.5f);
  const float cs = __builtin_fmaf(z, p, 1.0f);
  c = q & 1 ? sn : cs;
  s = q & 1 ? cs : sn;
  if (q == 1 || q == 2) c = -c;
  if (q >= 2) s = -s;
}

// `lanes` lanes hold a head; a lane keeps the same piece of `each` heads of one
// token, and with it the cosines and sines.
template <typename T, bool PAIRS>
__global__ __launch_bounds__(256) void k_rope(RopeArgs a) {
  constexpr int N = PAIRS ? 4 : 8;  // pairs of a piece
  const int piece = threadIdx.x & (a.lanes - 1);
  const int t = a.first + (int)blockIdx.x * (256 / a.lanes) + threadIdx.x / a.lanes;
  if (t >= a.tokens || piece >= a.pieces) return;
  const int half = a.rot >> 1, turned = (half + N - 1) / N;
  const int h0 = blockIdx.y * a.each, h1 = min(a.heads, h0 + a.each);
  auto in = [&](int h) {
    const int z = h >= a.q_heads;
    return (const T*)a.x[z] + t * a.token[z] + (h - (z ? a.q_heads : 0)) * a.head[z];
  };
  auto to = [&](int h) {
    const int z = h >= a.q_heads;
    return (T*)a.out[z] + t * a.out_token[z] + (h - (z ? a.q_heads : 0)) * a.out_head[z];
  };
  if (piece >= turned) {
    const int d = a.rot + (piece - turned) * 8;
    for (int h = h0; h < h1; ++h) {
      float v[8];
      get8(in(h) + d, a.dim - d, v);
      put8(to(h) + d, a.dim - d, v);
    }
    return;
  }
  const int i0 = piece * N, n = min(N, half - i0);
  float c[N], s[N];
  const int64_t place = a.positions[t];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint64_t turn = (uint64_t)place * a.steps[min(i0 + i, half - 1)];
    cos_sin((uint32_t)((turn + 0x80000000u) >> 32), c[i], s[i]);
    c[i] *= a.gain;
    s[i] *= a.gain;
  }
#pragma unroll 2
  for (int h = h0; h < h1; ++h) {
    const T* x = in(h);
    T* y = to(h);
    if constexpr (PAIRS) {
      float v[8];
      get8(x + 2 * i0, 2 * n, v);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float p = v[2 * i], q = v[2 * i + 1];
        v[2 * i] = __builtin_fmaf(p, c[i], -(q * s[i]));
        v[2 * i + 1] = __builtin_fmaf(q, c[i], p * s[i]);
      }
      put8(y + 2 * i0, 2 * n, v);
    } else {
      float p[8], q[8];
      get8(x + i0, n, p);
      get8(x + i0 + half, n, q);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float u = p[i];
        p[i] = __builtin_fmaf(u, c[i], -(q[i] * s[i]));
        q[i] = __builtin_fmaf(q[i], c[i], u * s[i]);
      }
      put8(y + i0, n, p);
      put8(y + i0 + half, n, q);
    }
  }
}

template <typename T>
static void launch_rope(RopeArgs a, unsigned slices, hipStream_t s) {
  constexpr long most = 1 << 23;  // workgroups of a launch (2^32 threads are too many)
  const int rows = 256 / a.lanes;
  for (long at = 0; at < a.tokens; at += most * rows) {
    a.first = (int)at;
    const dim3 grid((unsigned)((std::min(a.tokens - at, most * rows) + rows - 1) / rows), slices);
    if (a.interleaved) hipLaunchKernelGGL((k_rope<T, true>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((k_rope<T, false>), grid, dim3(256), 0, s, a);
  }
}

}  // namespace qhip

using namespace qhip;

extern "C" int qhip_rope_steps(int rot_dim, double base, int scaling, double factor, int original, double fast, double slow,
                               unsigned long long* h_steps, float* h_gain) {
  if (rot_dim < 2 || (rot_dim & 1) || !(base > 1.0) || !(base < INFINITY) || !(factor > 0.0) || !(factor < INFINITY) ||
      !h_steps || !h_gain)
    return (int)hipErrorInvalidValue;
  const long double turn = 2.0L * 3.14159265358979323846264338327950288L;
  const int half = rot_dim / 2;
  long double b = base, low = 0, high = 0;
  float gain = 1.0f;
  switch (scaling) {
    case QHIP_ROPE_PLAIN: break;
    case QHIP_ROPE_LINEAR: break;
    case QHIP_ROPE_NTK:
      if (rot_dim == 2) return (int)hipErrorInvalidValue;
      b = base * powl(factor, (long double)rot_dim / (rot_dim - 2));
      break;
    case QHIP_ROPE_YARN:
      if (original <= 0 || !(slow > 0.0) || !(fast > slow) || !(factor >= 1.0)) return (int)hipErrorInvalidValue;
      // the pair that turns `n` times over the original context
      low = floorl(rot_dim * logl(original / (turn * fast)) / (2 * logl(base)));
      high = ceill(rot_dim * logl(original / (turn * slow)) / (2 * logl(base)));
      low = low < 0 ? 0 : low;
      high = high > rot_dim - 1 ? rot_dim - 1 : high;
      gain = (float)(1.0L + 0.1L * logl(factor));
      break;
    default: return (int)hipErrorInvalidValue;
  }
  for (int i = 0; i < half; ++i) {
    long double f = powl(b, -2.0L * i / rot_dim);
    if (scaling == QHIP_ROPE_LINEAR) f /= factor;
    if (scaling == QHIP_ROPE_YARN) {
      const long double span = high - low > 0.001L ? high - low : 0.001L;
      long double ramp = (i - low) / span;
      ramp = ramp < 0 ? 0 : ramp > 1 ? 1 : ramp;
      f = f * (1 - ramp) + f / factor * ramp;
    }
    f /= turn;
    f -= floorl(f);
    const long double r = roundl(f * 0x1p64L);
    h_steps[i] = r >= 0x1p64L ? 0ull : (unsigned long long)r;
  }
  *h_gain = gain;
  return 0;
}

extern "C" int qhip_launch_rope(int type, const qhip_rows* q, const qhip_rows* q_out, int q_heads, const qhip_rows* k,
                                const qhip_rows* k_out, int k_heads, int dim, int rot_dim,
                                const unsigned long long* d_steps, float gain, int interleaved, const int* d_positions,
                                int tokens, void* stream) {
  const int size = kv_type_size(type);
  if (!size || q_heads <= 0 || k_heads < 0 || dim <= 0 || rot_dim < 2 || (rot_dim & 1) || rot_dim > dim || tokens < 0 ||
      tokens > kMaxCount || (interleaved != 0 && interleaved != 1) || (long)(q_heads + (long)k_heads) * dim > 0x7FFFFFFFL)
    return (int)hipErrorInvalidValue;
  if (rot_dim > kRopeMost || dim - rot_dim > kRopeMost) return QHIP_DECLINE;
  if (tokens == 0) return 0;
  if (!rows_ok(q, size) || !rows_ok(q_out, size) || (k_heads > 0 && (!rows_ok(k, size) || !rows_ok(k_out, size))) || !d_steps ||
      ((uintptr_t)d_steps & 7u) || !d_positions || ((uintptr_t)d_positions & 3u))
    return (int)hipErrorInvalidValue;
  // a head is read and written by its own lanes: an output may take its input's
  // place, and no other's
  const qhip_rows *ins[] = {q, k}, *outs[] = {q_out, k_out};
  const int heads[] = {q_heads, k_heads};
  for (int o = 0; o < 2; ++o) {
    if (!heads[o]) continue;
    if (!rows_apart(outs[o], tokens, heads[o], dim) || rows_meet(outs[o], tokens, heads[o], dim, size, d_positions, 4L * tokens) ||
        rows_meet(outs[o], tokens, heads[o], dim, size, d_steps, 4L * rot_dim))
      return (int)hipErrorInvalidValue;
    for (int i = 0; i < 2; ++i)
      if (heads[i] && rows_overlap(outs[o], heads[o], dim, ins[i], heads[i], dim, tokens, size) && (i != o || !rows_same(outs[o], ins[i])))
        return (int)hipErrorInvalidValue;
  }
  if (k_heads && rows_overlap(q_out, q_heads, dim, k_out, k_heads, dim, tokens, size)) return (int)hipErrorInvalidValue;
  RopeArgs a{};
  for (int i = 0; i < 2; ++i) {
    if (!heads[i]) continue;
    a.x[i] = ins[i]->at;
    a.out[i] = outs[i]->at;
    a.token[i] = ins[i]->token_stride;
    a.head[i] = ins[i]->head_stride;
    a.out_token[i] = outs[i]->token_stride;
    a.out_head[i] = outs[i]->head_stride;
  }
  a.steps = (const uint64_t*)d_steps;
  a.positions = d_positions;
  a.gain = gain;
  a.tokens = tokens;
  a.q_heads = q_heads;
  a.heads = q_heads + k_heads;
  a.dim = dim;
  a.rot = rot_dim;
  a.interleaved = interleaved;
  // values that stay in place need no lanes
  const bool in_place = rows_same(q, q_out) && (!k_heads || rows_same(k, k_out));
  const int pairs = interleaved ? 4 : 8;
  a.pieces = (rot_dim / 2 + pairs - 1) / pairs + (in_place ? 0 : (dim - rot_dim + 7) / 8);
  a.lanes = 1;
  while (a.lanes < a.pieces) a.lanes *= 2;
  const long blocks = ((long)tokens * a.lanes + 255) / 256;
  // heads of a lane: as many as leave eight workgroups a CU (4097 tokens of 10 heads of 256,
  // 8192 of 40 of 128, into new memory: with two 25.9 and 47.3 us, four 22.9 and 40.2, eight 22.2
  // and 37.4, sixteen 23.0 and 38.7; into what the call before wrote 21.4 and 45.4, 19.8 and
  // 33.1, 17.9 and 30.0, 20.4 and 31.2)
  a.each = (int)((long)a.heads * blocks / 2048);
  a.each = a.each < 1 ? 1 : a.each > a.heads ? a.heads : a.each;
  const unsigned slices = (unsigned)((a.heads + a.each - 1) / a.each);  // fewer than 4096
  if (type == QHIP_TT_F32) launch_rope<float>(a, slices, (hipStream_t)stream);
  else if (type == QHIP_TT_F16) launch_rope<f16_t>(a, slices, (hipStream_t)stream);
  else launch_rope<bf16_t>(a, slices, (hipStream_t)stream);
  return (int)hipGetLastError();
}
