// norm.hip -- root-mean-square norms of rows or heads, with the residual's
// addition in front, a gate behind, and an output in 8 bits.
//
//   h = x + residual (residual becomes h);  r = 1 / sqrt(mean(h^2) + eps)
//   y = (h * r) * weight [* gate / (1 + exp(-gate))]
//   out = y in the rows' type, codes = the activation quantizers' rows of y
//
// The mean square is summed in f64 (a product of two f32 is exact there) and r
// rounded once to f32; all else is single f32 operations.  So a row's bits do not
// depend on how its sum is cut over lanes, and the codes are those of the
// quantizers applied to the f32 y.
//
// Memory bounds it: each value is read once, held in registers over the sum and written
// once.  Inputs from memory, outputs into memory not used before (in brackets: into what the
// call before wrote, which the last cache still holds): 4096 bf16 rows of 5120 with the residual
// 37 us, 4.5 TB/s of the 5.1 of a copy (33); 131,056 heads of 128 in f32 with gates 40 us, 5.0
// (40); 1673 f32 rows of 5120 with the residual to Q8_0 codes 29 us, 3.9 (27: one uneven round
// of workgroups), to Q8_K 27.5 us; the heads with gates to Q8_0 codes 40.5 us, 3.8, to Q8_K 42;
// one row of 2560 4.3 us, a chain of loads, two sums and stores.
#include "qhip_device.hpp"
#include "qhip_internal.hpp"
#include "rows_internal.hpp"

#include <algorithm>

namespace qhip {

struct NormArgs {
  const void *x, *gate;
  void *residual, *out;
  long x_token, x_head, res_token, res_head, gate_token, gate_head, out_token, out_head;
  const float* weight;
  uint8_t* xq;
  long groups;  // tokens * heads
  long first;   // row of this launch
  int heads, dim, lanes;
  int act;  // 32: Q8_0 rows, 256: Q8_K rows
  float eps;
};

template <int CTRL>
__device__ __forceinline__ double move_f64(double v) {
  const int lo = __double2loint(v), hi = __double2hiint(v);
  return __hiloint2double(__builtin_amdgcn_update_dpp(0, hi, CTRL, 0xF, 0xF, false),
                          __builtin_amdgcn_update_dpp(0, lo, CTRL, 0xF, 0xF, false));
}
// sum over aligned groups of `lanes` (a power of two, uniform) lanes, in each of them
__device__ __forceinline__ double sum_f64(double v, int lanes) {
  if (lanes > 1) v += move_f64<0xB1>(v);   // quad_perm [1, 0, 3, 2]
  if (lanes > 2) v += move_f64<0x4E>(v);   // quad_perm [2, 3, 0, 1]
  if (lanes > 4) v += move_f64<0x141>(v);  // row_half_mirror
  if (lanes > 8) v += move_f64<0x140>(v);  // row_mirror
  if (lanes > 16) {
    const auto lo = __builtin_amdgcn_permlane16_swap(__double2loint(v), __double2loint(v), false, false);
    const auto hi = __builtin_amdgcn_permlane16_swap(__double2hiint(v), __double2hiint(v), false, false);
    v = __hiloint2double(hi[0], lo[0]) + __hiloint2double(hi[1], lo[1]);
  }
  if (lanes > 32) {
    const auto lo = __builtin_amdgcn_permlane32_swap(__double2loint(v), __double2loint(v), false, false);
    const auto hi = __builtin_amdgcn_permlane32_swap(__double2hiint(v), __double2hiint(v), false, false);
    v = __hiloint2double(hi[0], lo[0]) + __hiloint2double(hi[1], lo[1]);
  }
  return v;
}
__device__ __forceinline__ float inverse_root(double sum, const NormArgs& a) {
  return (float)(1.0 / sqrt(sum / a.dim + (double)a.eps));
}

// The codes of eight values of one row at value `at` of all rows (whole blocks of
// lanes are in or out together).
__device__ __forceinline__ void put_codes(const NormArgs& a, const float (&y)[8], long at, bool in) {
  if (a.act == 32) {
    uint32_t bits, w[2];
    quant_q8_0_lane8(y, w, bits);
    if (!in) return;
    uint16_t* block = (uint16_t*)(a.xq + (at >> 5) * 34);
    const int pt = (int)(at >> 3) & 3;
    block[1 + 4 * pt] = (uint16_t)w[0];
    block[2 + 4 * pt] = (uint16_t)(w[0] >> 16);
    block[3 + 4 * pt] = (uint16_t)w[1];
    block[4 + 4 * pt] = (uint16_t)(w[1] >> 16);
    if (pt == 0) block[0] = (uint16_t)bits;
  } else {
    uint32_t w[2];
    int sum;
    float scale;
    quant_q8_K_lane8(y, w, sum, scale);
    if (!in) return;
    uint8_t* block = a.xq + (at >> 8) * 292;
    const int pt = (int)(at >> 3) & 31;
    ((uint32_t*)(block + 4))[2 * pt] = w[0];
    ((uint32_t*)(block + 4))[2 * pt + 1] = w[1];
    if ((pt & 1) == 0) ((int16_t*)(block + 260))[pt >> 1] = (int16_t)sum;
    if (pt == 0) *(float*)block = scale;
  }
}

// A row a workgroup of NT threads (a wave's lanes would hold 40 values of 2560 each, and one
// row would wait for one wave), P pieces of eight values a thread in
// registers; P = 0: rows of any length, read a second time (from L2).
template <typename T, int NT, int P>
__global__ __launch_bounds__(NT) void k_norm_row(NormArgs a) {
  __shared__ double s_sum[NT / 64];
  const int tid = threadIdx.x;
  const long g = a.first + blockIdx.x, token = a.heads == 1 ? g : (unsigned)g / (unsigned)a.heads, head = g - token * a.heads;
  const T* x = (const T*)a.x + token * a.x_token + head * a.x_head;
  T* res = a.residual ? (T*)a.residual + token * a.res_token + head * a.res_head : nullptr;
  const T* gate = a.gate ? (const T*)a.gate + token * a.gate_token + head * a.gate_head : nullptr;
  T* out = a.out ? (T*)a.out + token * a.out_token + head * a.out_head : nullptr;
  constexpr int K = P ? P : 1;
  float h[K][8];
  double sum = 0.0;
  auto square = [&](const float(&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = __builtin_fma((double)v[i], (double)v[i], sum);
  };
  auto added = [&](int d, float(&v)[8], bool keep) {  // v += residual
    float r[8];
    get8(res + d, a.dim - d, r);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += r[i];
    if (keep) put8(res + d, a.dim - d, v);
  };
  if constexpr (P > 0) {
#pragma unroll
    for (int p = 0; p < P; ++p) get8(x + (p * NT + tid) * 8, a.dim - (p * NT + tid) * 8, h[p]);
    if (res) {
#pragma unroll
      for (int p = 0; p < P; ++p) added((p * NT + tid) * 8, h[p], true);
    }
#pragma unroll
    for (int p = 0; p < P; ++p) square(h[p]);
  } else {
    for (int d = tid * 8; d < a.dim; d += NT * 8) {
      get8(x + d, a.dim - d, h[0]);
      if (res) added(d, h[0], false);
      square(h[0]);
    }
  }
  sum = sum_f64(sum, 64);
  if ((tid & 63) == 0) s_sum[tid >> 6] = sum;
  __syncthreads();
  sum = s_sum[0];
#pragma unroll
  for (int w = 1; w < NT / 64; ++w) sum += s_sum[w];
  const float r = inverse_root(sum, a);
  auto finish = [&](int d, float(&v)[8]) {
    const int n = a.dim - d;
    float w[8];
    if (a.weight) get8(a.weight + d, n, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = a.weight ? (v[i] * r) * w[i] : v[i] * r;
    if (gate) {
      float t[8];
      get8(gate + d, n, t);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] *= t[i] / (1.0f + expf(-t[i]));
    }
    if (out) put8(out + d, n, v);
    if (a.xq) {
      if (n <= 0) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.0f;
      }
      put_codes(a, v, g * a.dim + d, n > 0);
    }
  };
  if constexpr (P > 0) {
#pragma unroll
    for (int p = 0; p < P; ++p) finish((p * NT + tid) * 8, h[p]);
  } else {
    for (int d0 = 0; d0 < a.dim; d0 += NT * 8) {
      const int d = d0 + tid * 8;
      get8(x + d, a.dim - d, h[0]);
      if (res) added(d, h[0], true);
      finish(d, h[0]);
    }
  }
}

// Rows of up to 512 values: `lanes` lanes a row, eight values each, several rows a
// wave.
template <typename T>
__global__ __launch_bounds__(256) void k_norm_heads(NormArgs a) {
  const int lane = threadIdx.x & (a.lanes - 1), d = lane * 8, n = a.dim - d;
  const long g = a.first + (long)blockIdx.x * (256 / a.lanes) + threadIdx.x / a.lanes;
  const bool in = g < a.groups && n > 0;
  const long token = (unsigned)g / (unsigned)a.heads, head = g - token * a.heads;
  float h[8] = {}, t[8], w[8];
  if (in) {
    get8((const T*)a.x + token * a.x_token + head * a.x_head + d, n, h);
    if (a.gate) get8((const T*)a.gate + token * a.gate_token + head * a.gate_head + d, n, t);
    if (a.weight) get8(a.weight + d, n, w);
    if (a.residual) {
      T* res = (T*)a.residual + token * a.res_token + head * a.res_head + d;
      float r[8];
      get8(res, n, r);
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] += r[i];
      put8(res, n, h);
    }
  }
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < 8; ++i) sum = __builtin_fma((double)h[i], (double)h[i], sum);
  const float r = inverse_root(sum_f64(sum, a.lanes), a);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    h[i] = in ? h[i] * r : 0.0f;
    if (in && a.weight) h[i] *= w[i];
    if (in && a.gate) h[i] *= t[i] / (1.0f + expf(-t[i]));
  }
  if (in && a.out) put8((T*)a.out + token * a.out_token + head * a.out_head + d, n, h);
  if (a.xq) put_codes(a, h, g * a.dim + d, in);
}

constexpr int kHeadMost = 512;  // values of a row that a wave's lanes hold
// values of a row at most: 1024 lanes of eight step past its end within an int
constexpr int kRowMost = 0x7FFFFFFF - 8192;

template <typename T>
static void launch_norm_part(const NormArgs& a, long count, hipStream_t s) {
  if (a.dim <= kHeadMost) {
    const long rows = 256 / a.lanes;
    hipLaunchKernelGGL(k_norm_heads<T>, dim3((unsigned)((count + rows - 1) / rows)), dim3(256), 0, s, a);
    return;
  }
  const dim3 grid((unsigned)count);
  if (a.dim <= 2048) hipLaunchKernelGGL((k_norm_row<T, 256, 1>), grid, dim3(256), 0, s, a);
  else if (a.dim <= 4096) hipLaunchKernelGGL((k_norm_row<T, 256, 2>), grid, dim3(256), 0, s, a);
  else if (a.dim <= 8192) hipLaunchKernelGGL((k_norm_row<T, 256, 4>), grid, dim3(256), 0, s, a);
  else if (a.dim <= 16384) hipLaunchKernelGGL((k_norm_row<T, 512, 4>), grid, dim3(512), 0, s, a);
  else hipLaunchKernelGGL((k_norm_row<T, 1024, 0>), grid, dim3(1024), 0, s, a);
}

template <typename T>
static void launch_norm(NormArgs a, hipStream_t s) {
  constexpr long most = 1 << 21;  // workgroups of a launch (2^32 threads are too many)
  const long rows = a.dim <= kHeadMost ? 256 / a.lanes : 1;
  for (; a.first < a.groups; a.first += most * rows) launch_norm_part<T>(a, std::min(a.groups - a.first, most * rows), s);
}

}  // namespace qhip

using namespace qhip;

extern "C" int qhip_launch_rms_norm(int type, const qhip_rows* x, const qhip_rows* residual, const qhip_rows* gate,
                                    const float* d_weight, float eps, const qhip_rows* out, int ttype, void* d_xq,
                                    int tokens, int heads, int dim, void* stream) {
  const int size = kv_type_size(type);
  if (!size || tokens < 0 || heads <= 0 || dim <= 0 || dim > kRowMost || !(eps >= 0.0f) ||
      (long)heads * dim > 0x7FFFFFFFL)
    return (int)hipErrorInvalidValue;
  NormArgs a{};
  if (d_xq) {
    const long cols = (long)heads * dim;
    a.act = qhip_quant_act_block_elems(ttype);
    if (!a.act || cols % a.act || (uintptr_t)d_xq % (a.act == 32 ? 2 : 4)) return (int)hipErrorInvalidValue;
    // a block's lanes are side by side: blocks inside a row, or rows that fill their lanes
    if (dim % a.act && (dim > kHeadMost || dim % 8 || (dim & (dim - 1)))) return QHIP_DECLINE;
  }
  if (tokens == 0) return 0;
  if ((!out && !d_xq) || (long)tokens * heads > 0x7FFFFFFFL) return (int)hipErrorInvalidValue;
  if (!rows_ok(x, size) || (residual && !rows_ok(residual, size)) || (gate && !rows_ok(gate, size)) ||
      (out && !rows_ok(out, size)) || ((uintptr_t)d_weight & 3u))
    return (int)hipErrorInvalidValue;
  // every row is read and written by its own workgroup or lanes: an output may
  // take the place of an input with the same rows, and of no other
  const long code_bytes = d_xq ? (long)tokens * heads * dim / a.act * (a.act == 32 ? 34 : 292) : 0;
  const qhip_rows* written[] = {residual, out};
  for (const qhip_rows* w : written) {
    if (!w) continue;
    if (!rows_apart(w, tokens, heads, dim) || rows_meet(w, tokens, heads, dim, size, d_xq, code_bytes) ||
        (d_weight && rows_meet(w, tokens, heads, dim, size, d_weight, 4L * dim)))
      return (int)hipErrorInvalidValue;
    for (const qhip_rows* r : {x, gate})
      if (r && rows_overlap(w, heads, dim, r, heads, dim, tokens, size) && (w == residual || !rows_same(w, r)))
        return (int)hipErrorInvalidValue;
  }
  if (residual && out && rows_overlap(residual, heads, dim, out, heads, dim, tokens, size)) return (int)hipErrorInvalidValue;
  for (const qhip_rows* r : {x, gate})
    if (r && rows_meet(r, tokens, heads, dim, size, d_xq, code_bytes)) return (int)hipErrorInvalidValue;
  if (d_xq && d_weight && (const char*)d_weight < (const char*)d_xq + code_bytes && (const char*)d_xq < (const char*)(d_weight + dim))
    return (int)hipErrorInvalidValue;
  a.x = x->at;
  a.x_token = x->token_stride;
  a.x_head = x->head_stride;
  if (residual) {
    a.residual = residual->at;
    a.res_token = residual->token_stride;
    a.res_head = residual->head_stride;
  }
  if (gate) {
    a.gate = gate->at;
    a.gate_token = gate->token_stride;
    a.gate_head = gate->head_stride;
  }
  if (out) {
    a.out = out->at;
    a.out_token = out->token_stride;
    a.out_head = out->head_stride;
  }
  a.weight = d_weight;
  a.xq = (uint8_t*)d_xq;
  a.groups = (long)tokens * heads;
  a.heads = heads;
  a.dim = dim;
  a.eps = eps;
  a.lanes = 1;
  while (a.lanes * 8 < dim && a.lanes < 64) a.lanes *= 2;
  if (type == QHIP_TT_F32) launch_norm<float>(a, (hipStream_t)stream);
  else if (type == QHIP_TT_F16) launch_norm<f16_t>(a, (hipStream_t)stream);
  else launch_norm<bf16_t>(a, (hipStream_t)stream);
  return (int)hipGetLastError();
}
