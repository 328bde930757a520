// kv_internal.hpp -- what the kernels of the 8-bit key/value cache share: the
// element types of keys, values, queries and outputs, and the checks of a
// cache descriptor.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/qwen35_hip.h"

namespace qhip {

typedef uint32_t kv_u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t kv_u32x2 __attribute__((ext_vector_type(2)));

// Longest sequence: places are ints, and some are counted a round of steps past
// the last.
constexpr int kMaxLen = 1 << 30;
// Most tokens and sequences of a call: indexes run up to a workgroup's or a block's
// past the last.
constexpr int kMaxCount = 0x7FFFFFFF - 1024;

// NaN payloads aside, (float)T is exact and T(float) rounds to nearest even.
typedef _Float16 f16_t;
typedef __bf16 bf16_t;

// Eight consecutive elements as they lie in memory, in 16-byte loads from any
// element's address (rows inside a wider tensor may begin anywhere).
template <typename T>
struct Raw8 {
  T e[8];
};
template <typename T>
__device__ __forceinline__ Raw8<T> load8(const T* p) {
  typedef uint32_t piece __attribute__((ext_vector_type(4), aligned(2)));
  kv_u32x4 r[sizeof(Raw8<T>) / 16];
#pragma unroll
  for (unsigned i = 0; i < sizeof(r) / 16; ++i) r[i] = ((const piece*)p)[i];
  return __builtin_bit_cast(Raw8<T>, r);
}

__device__ __forceinline__ bool finite_bits(uint32_t u) { return (u & 0x7F800000u) != 0x7F800000u; }

// inclusive sum over the wave's lanes up to this one (rows of 16, then their ends
// handed on)
__device__ __forceinline__ int scan64(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);  // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast:15 into rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // row_bcast:31 into rows 2 and 3
  return v;
}

inline int kv_type_size(int type) {
  return type == QHIP_TT_F32 ? 4 : type == QHIP_TT_F16 || type == QHIP_TT_BF16 ? 2 : 0;
}

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

// log2 of a supported block size, else -1
inline int kv_block_shift(int block_size) {
  for (int s = 4; s <= 8; ++s)
    if (block_size == 1 << s) return s;
  return -1;
}

// 0, hipErrorInvalidValue or QHIP_DECLINE (a head width without kernels)
inline int kv_check_cache(const qhip_kv_cache* c) {
  if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale) return (int)hipErrorInvalidValue;
  if (!aligned16(c->k) || !aligned16(c->v) || ((uintptr_t)c->k_scale & 3u) || ((uintptr_t)c->v_scale & 3u))
    return (int)hipErrorInvalidValue;
  if (c->num_blocks <= 0 || c->kv_heads <= 0 || c->kv_heads > 65535 || c->head_dim <= 0) return (int)hipErrorInvalidValue;
  if (kv_block_shift(c->block_size) < 0 || (long)c->num_blocks * c->block_size > 0x7FFFFFFFL)
    return (int)hipErrorInvalidValue;
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return QHIP_DECLINE;
  return 0;
}

}  // namespace qhip
