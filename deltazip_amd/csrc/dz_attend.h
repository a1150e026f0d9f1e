// What the attention kernels over a paged cache share: element types, sums over a wavefront, the joining of pieces.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "dz_device.h"

namespace {

typedef float f2_t __attribute__((ext_vector_type(2)));
typedef __bf16 b8_t __attribute__((ext_vector_type(8)));

template <bool BF>
struct Type;
template <>
struct Type<false> {
  typedef h8_t v8;
  static constexpr float BIAS = 14.0f;
  static __device__ __forceinline__ f4_t mma(v8 a, v8 b, f4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ uint16_t round(float x) { return __builtin_bit_cast(uint16_t, (_Float16)x); }
  static __device__ __forceinline__ _Float16 one(float x) { return (_Float16)x; }
};
template <>
struct Type<true> {
  typedef b8_t v8;
  static constexpr float BIAS = 0.0f;
  static __device__ __forceinline__ f4_t mma(v8 a, v8 b, f4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ uint16_t round(float x) { return __builtin_bit_cast(uint16_t, (__bf16)x); }
  static __device__ __forceinline__ __bf16 one(float x) { return (__bf16)x; }
};

// Sums over the lanes in front of and at each, by shifts within the wavefront's rows of 16 lanes and broadcasts of their last ones.
template <typename T>
__device__ __forceinline__ T scan_add(T x) {
  auto add = [&](auto ctrl, auto mask) {
    x += __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctrl)::value, decltype(mask)::value, 0xf, false));
  };
  using std::integral_constant;
  add(integral_constant<int, 0x111>(), integral_constant<int, 0xf>());     // row_shr:1, 2, 4, 8
  add(integral_constant<int, 0x112>(), integral_constant<int, 0xf>());
  add(integral_constant<int, 0x114>(), integral_constant<int, 0xf>());
  add(integral_constant<int, 0x118>(), integral_constant<int, 0xf>());
  add(integral_constant<int, 0x142>(), integral_constant<int, 0xa>());     // row_bcast:15
  add(integral_constant<int, 0x143>(), integral_constant<int, 0xc>());     // row_bcast:31
  return x;
}

// What the sums of a piece of a row with the maximum `top` count for in sums with the maximum `up`.  A piece without a maximum
// has sums of zero, or of NaN (a score that is NaN raises no maximum), and these have to stay.
__device__ __forceinline__ float weight_of(float top, float up) { return top == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(top - up); }

}  // namespace
