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

// 8 values of a row as 4 words.
template <bool ALIGNED>
__device__ __forceinline__ u32x4 load_row8(uint64_t at) {
  if constexpr (ALIGNED) return *reinterpret_cast<const g_u32x4*>(at);
  const g_u16* p = reinterpret_cast<const g_u16*>(at);
  u32x4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    v[i] = p[2 * i] | (static_cast<uint32_t>(p[2 * i + 1]) << 16);
  return v;
}

template <bool ALIGNED>
__device__ __forceinline__ void store_row8(uint64_t at, u32x4 v) {
  if constexpr (ALIGNED) {
    *reinterpret_cast<g_u32x4*>(at) = v;
  } else {
    g_u16* p = reinterpret_cast<g_u16*>(at);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      p[2 * i] = static_cast<uint16_t>(v[i]);
      p[2 * i + 1] = static_cast<uint16_t>(v[i] >> 16);
    }
  }
}

__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }

// The largest x of a group of LANES aligned lanes, in all of them.  Within 16 lanes by
// cross-lane operands of the vector instructions, which cost no trip through LDS.
template <uint32_t LANES>
__device__ __forceinline__ uint32_t group_max(uint32_t x) {
  constexpr int kSwap1 = 0xb1, kSwap2 = 0x4e;  // lanes 1 0 3 2 and 2 3 0 1 of each four
  constexpr int kMirror8 = 0x141, kMirror16 = 0x140;
  x = umax(x, __builtin_amdgcn_mov_dpp(x, kSwap1, 0xf, 0xf, true));
  x = umax(x, __builtin_amdgcn_mov_dpp(x, kSwap2, 0xf, 0xf, true));
  if constexpr (LANES >= 8) x = umax(x, __builtin_amdgcn_mov_dpp(x, kMirror8, 0xf, 0xf, true));
  if constexpr (LANES >= 16) x = umax(x, __builtin_amdgcn_mov_dpp(x, kMirror16, 0xf, 0xf, true));
  if constexpr (LANES >= 32) x = umax(x, static_cast<uint32_t>(__shfl_xor(static_cast<int>(x), 16)));
  return x;
}

// L and 1 / L of a row's scale max|x| / L.
template <uint32_t TYPE>
constexpr float kLargest = TYPE == PF_KV_E4M3 ? 448.0f : 127.0f;
template <uint32_t TYPE>
constexpr float kInverseLargest = 1.0f / kLargest<TYPE>;

// 8 values q as codes of scale s (s > 0).
//
// The quotients are IEEE divisions, at 5 operations each instead of the compiler's 10
// or so: with y = 1 / s rounded to nearest, q = x y, and twice q += y (x - q s), each
// step one fused operation.  The first correction leaves q within an ulp, and the second
// then gives x / s rounded to nearest (Markstein's theorem), provided that x - q s is
// exact, which it is where its last bit, 2^-24 x or more, is not below 2^-149.  With s >=
// 2^-100 that holds for every x that does not round to code 0 anyway (|x| >= 2^-11 s);
// rows smaller than that are divided, and cut to L: of 32-bit values a scale may have a bit
// or two only, and be far off.
template <uint32_t TYPE>
__device__ __forceinline__ u32x2 encode(float (&q)[8], float s) {
  if (s >= 0x1p-100f) {
    const float y = 1.0f / s;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float v = q[i];
      float z = v * y;
      z = __builtin_fmaf(__builtin_fmaf(-z, s, v), y, z);
      z = __builtin_fmaf(__builtin_fmaf(-z, s, v), y, z);
      q[i] = __builtin_copysignf(z, v);  // also of 0
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = fminf(fmaxf(q[i] / s, -kLargest<TYPE>), kLargest<TYPE>);
  }
  u32x2 c;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    if constexpr (TYPE == PF_KV_E4M3) {
      int v = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * w], q[4 * w + 1], 0, false);
      c[w] = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * w + 2], q[4 * w + 3], v, true);
    } else {
      // Added to 1.5 * 2^23 a quotient is rounded to an integer, ties to even, and the
      // sum's low byte is its code.
      uint32_t v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = __builtin_bit_cast(uint32_t, q[4 * w + i] + 12582912.0f);
      const uint32_t lo = __builtin_amdgcn_perm(v[1], v[0], 0x0c0c0400u);
      const uint32_t hi = __builtin_amdgcn_perm(v[3], v[2], 0x04000c0cu);
      c[w] = lo | hi;
    }
  }
  return c;
}

// x / block_size for x < 2^31 (set_division).
__device__ __forceinline__ uint32_t page_of(const PagedView& p, uint32_t x) {
  return static_cast<uint32_t>(static_cast<uint64_t>(x) * p.div_mul >> (31 + p.div_shift));
}

}  // namespace pf
