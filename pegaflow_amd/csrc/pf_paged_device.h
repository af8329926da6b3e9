// pf_paged_device.h — device helpers of the paged-cache kernels.
#pragma once

#include <hip/hip_runtime.h>

#include "pf_paged.h"

namespace pf {

typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(1))) uint8_t g_u8;
typedef __attribute__((address_space(1))) uint16_t g_u16;
typedef __attribute__((address_space(1))) uint32_t g_u32;
typedef __attribute__((address_space(1))) u32x2 g_u32x2;
typedef __attribute__((address_space(1))) u32x4 g_u32x4;
typedef __attribute__((address_space(1))) float g_f32;

// Row types.
struct BF16 {
  static constexpr uint32_t kType = PF_KV_BF16;
  static constexpr uint32_t kInf = 0x7f80;  // |bits| from here on: infinity or NaN
  static __device__ __forceinline__ float to_float(uint32_t bits) {
    return __builtin_bit_cast(float, bits << 16);
  }
  static __device__ __forceinline__ uint32_t from_float(float x) {
    return __builtin_bit_cast(uint16_t, static_cast<__bf16>(x));
  }
};
struct FP16 {
  static constexpr uint32_t kType = PF_KV_FP16;
  static constexpr uint32_t kInf = 0x7c00;
  static __device__ __forceinline__ float to_float(uint32_t bits) {
    return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(bits)));
  }
  static __device__ __forceinline__ uint32_t from_float(float x) {
    return __builtin_bit_cast(uint16_t, static_cast<_Float16>(x));
  }
};

// The four codes of a word as floats.
template <uint32_t TYPE>
__device__ __forceinline__ void codes_to_float(uint32_t word, float* out) {
  if constexpr (TYPE == PF_KV_E4M3) {
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(word, false);
    const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8(word, true);
    out[0] = lo[0];
    out[1] = lo[1];
    out[2] = hi[0];
    out[3] = hi[1];
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      out[i] = static_cast<float>(static_cast<int8_t>(word >> (8 * i)));
  }
}

// x / block_size for x < 2^31 (set_division).
__device__ __forceinline__ uint32_t page_of(const PagedView& p, uint32_t x) {
  return static_cast<uint32_t>(static_cast<uint64_t>(x) * p.div_mul >> (31 + p.div_shift));
}

}  // namespace pf
