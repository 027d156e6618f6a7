// attn_dev.hpp -- device helpers of the attention kernels on 32x32x16 matrix
// products (tree_attention.hip, shared_attention.hip): K and V tiles in LDS and
// reductions over the two lanes that share a query row.
#pragma once

#include "gemm_dev.hpp"

namespace whd {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));  // four floats of the caller's arrays
typedef short s16x4 __attribute__((ext_vector_type(4)));

// LDS rows of K and V are D f16 without padding (the copies write 16 lanes'
// chunks in a row), so the 16-byte chunks of row r are permuted: chunk c lies
// at c ^ swz(r).  K: a wave's operand read takes one chunk of 32 rows; V: a
// transposing read takes four chunks of each of 4 rows.  With these every 16
// (32) lanes reach all 64 banks once.
template <int D>
__device__ __forceinline__ int swz_k(int r) { return D == 128 ? (r & 15) : ((r >> 1) & 7); }
template <int D>
__device__ __forceinline__ int swz_v(int r) { return D == 128 ? (r & 3) << 2 : ((r >> 1) & 1) << 2; }

__device__ __forceinline__ s16x4 read_tr(uint32_t lds) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(uintptr_t)lds);
}

// The largest of this lane's and lane ^ 32's value: NaN passed over, or kept.
__device__ __forceinline__ float swap_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
  return fmaxf(__builtin_bit_cast(float, static_cast<uint32_t>(r[0])), __builtin_bit_cast(float, static_cast<uint32_t>(r[1])));
}
__device__ __forceinline__ float swap_max_nan(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
  return __builtin_elementwise_maximum(__builtin_bit_cast(float, static_cast<uint32_t>(r[0])),
                                       __builtin_bit_cast(float, static_cast<uint32_t>(r[1])));
}
__device__ __forceinline__ float swap_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
  return __builtin_bit_cast(float, static_cast<uint32_t>(r[0])) + __builtin_bit_cast(float, static_cast<uint32_t>(r[1]));
}

}  // namespace whd
