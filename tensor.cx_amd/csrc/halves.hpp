// float32 numbers as two float16 halves for matrix instructions: hi = half(x) and
// lo = half(x - hi) hold 22 bits of x together. float16 has five bits of exponent,
// so a row of numbers is first multiplied by a power of two (exact) that brings
// its largest magnitude into [2^14, 2^15): numbers down to 2^-29 of the largest
// then keep their 22 bits, and below that an absolute error of 2^-40 of it.
#pragma once

#include "common.hpp"

namespace tcx {

using half2_t = _Float16 __attribute__((ext_vector_type(2)));
using half4_t = _Float16 __attribute__((ext_vector_type(4)));
using half8_t = _Float16 __attribute__((ext_vector_type(8)));
using float2v_t = float __attribute__((ext_vector_type(2)));
using acc_t = float __attribute__((ext_vector_type(4)));

// hi and lo halves of N scaled numbers.
template <int N, typename H>
__device__ __forceinline__ void split_halves(const float (&x)[N], H& hi, H& lo) {
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const half2_t h = __builtin_convertvector((float2v_t{x[i], x[i + 1]}), half2_t);
    const half2_t l = __builtin_convertvector(
        (float2v_t{x[i] - static_cast<float>(h[0]), x[i + 1] - static_cast<float>(h[1])}), half2_t);
    hi[i] = h[0];
    hi[i + 1] = h[1];
    lo[i] = l[0];
    lo[i + 1] = l[1];
  }
}

__device__ __forceinline__ std::uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffU; }

// The largest of kLanes neighbouring lanes' words, in all of them.
template <int kLanes>
__device__ __forceinline__ std::uint32_t lanes_most(std::uint32_t x) {
  auto with = [&]<int kControl>() {
    x = max(x, static_cast<std::uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), kControl, 0xf, 0xf, true)));
  };
  with.template operator()<0xb1>();
  with.template operator()<0x4e>();
  if constexpr (kLanes >= 8) with.template operator()<0x141>();
  if constexpr (kLanes >= 16) with.template operator()<0x140>();
  if constexpr (kLanes >= 32)
    x = max(x, static_cast<std::uint32_t>(__builtin_amdgcn_ds_swizzle(static_cast<int>(x), 0x401f)));
  return x;
}

// Sum and maximum over the four lanes of a column of a matrix operand (16 apart), in
// all of them: two swaps of rows of lanes, without LDS.
__device__ __forceinline__ float across_sum(float x) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
__device__ __forceinline__ float across_max(float x) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ std::uint32_t across_max(std::uint32_t x) {
  const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = max(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return max(b[0], b[1]);
}
// Over the four lanes of sixteen that are 4 apart, in all of them.
__device__ __forceinline__ float ror4(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x124, 0xf, 0xf, true));
}
__device__ __forceinline__ float ror8(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x128, 0xf, 0xf, true));
}
__device__ __forceinline__ float shares_sum(float x) {
  x += ror8(x);
  return x + ror4(x);
}
__device__ __forceinline__ float shares_max(float x) {
  x = fmaxf(x, ror8(x));
  return fmaxf(x, ror4(x));
}

// The exponent field of the power of two that brings a magnitude into [2^14,
// 2^15), at most `most`.
__device__ __forceinline__ int scale_field(std::uint32_t magnitude_bits, int most) {
  return min(268 - static_cast<int>(magnitude_bits >> 23), most);
}
__device__ __forceinline__ float power_field(int field) { return __int_as_float(field << 23); }

}  // namespace tcx
