// float32 numbers as two float16 halves for matrix instructions: hi = half(x) and
// lo = half(x - hi) hold 22 bits of x together. float16 has five bits of exponent,
// so a row of numbers is first multiplied by a power of two (exact) that brings
// its largest magnitude into [2^14, 2^15): numbers down to 2^-29 of the largest
// then keep their 22 bits, and below that an absolute error of 2^-40 of it. RowBase
// does the like for a softmax's weights.
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
// A whole number as an exponent (past those of float32 it makes no difference).
__device__ __forceinline__ int exponent(float x) { return static_cast<int>(fminf(fmaxf(x, -400.F), 400.F)); }

// What the scores of a row, in units of log2, are taken from: p = 2^(s - base), whose
// sum is the softmax's, and p 2^(e + rest) for a key whose values are held times 2^-e,
// which goes into halves. Both are whole numbers, so that moving them is exact. base is
// such that the largest product is 2^kAim when it is set, as far as that leaves the
// largest weight between 2^-kNear and 2^kNear; rest makes up for where it does not, and
// is 0 otherwise. The five powers of two up to 2^kMost, which float16 still holds, are
// what scores can rise before base is set anew (with three 241 us in place of 230 for a
// prompt of 8192 rows, 16 heads of 64 features, window 2048).
//
// A row is held by several lanes, which all have its base, but each the largest of its
// own scores: what a tile shows is put together only where a base moves. A row whose
// base does not stays as it is to the bit: why others do, and why this is asked at
// all, may be keys that it does not see.
struct RowBase {
  static constexpr float kAim = 11.F, kMost = 15.99F, kNear = 60.F, kFar = 64.F;
  static constexpr float kWhole = 8388608.F;  // from here on float32 has no fractions
  float base, rest;
  float top;   // the lane's largest score, from base on
  bool first;  // nothing is seen yet

  __device__ __forceinline__ void start() {
    base = rest = 0.F;
    top = -__builtin_inff();
    first = true;
  }
  // Takes note of a lane's largest score of a tile, from base on; whether that, or its
  // largest score and exponent, may move the row.
  __device__ __forceinline__ bool see(float most, float high) {
    top = fmaxf(top, most);
    return first | (most > kFar) | (high + rest > kMost);
  }
  // Moves it where it has to be. row(x): the largest x of the row's lanes; each(f): f on
  // the lane's scores; product(): its largest score and exponent; l: a sum of weights.
  // Returns the exponent by which the outputs are to be scaled.
  template <typename Row, typename Each, typename Product>
  __device__ __forceinline__ int move(float& l, Row&& row, Each&& each, Product&& product) {
    top = row(top);
    const float high = row(product());
    const bool past = first || high + rest > kMost, need = top > -__builtin_inff() && (past || top > kFar);
    float to = base, aim = rest, gone = 0.F;
    bool plain = true, far = false;
    if (need) {
      const float all = past ? ceilf(high) - kAim : 0.F, peak = ceilf(top);
      const float by = fminf(fmaxf(all, peak - kNear), peak + kNear);
      to += by;
      far = fabsf(to) >= kWhole;
      if (far) to = base + top;  // the largest score itself, which the others are then rounded like
      plain = by == all && !far;
      if (past && plain) aim = 0.F;
      gone = to - base;
    }
    if (__any(!plain)) [[unlikely]] {
      each([&](float s) { return far ? (s + base) - to : s - gone; });
      top = far ? 0.F : top - gone;
      gone = 0.F;
      const float now = row(product());
      if (!plain && (past || now + rest > kMost)) aim = kAim - ceilf(now);
    }
    top -= gone;
    each([&](float s) { return s - gone; });
    l = ldexpf(l, exponent(base - to));
    const int scale = first ? 0 : exponent((base - to) + (aim - rest));
    base = to;
    rest = aim;
    first = first && !need;
    return scale;
  }
  // The row's largest score, rounded up, from base on, and as it is, once `top` is that of
  // all its lanes: sums over parts of the keys are joined from there.
  __device__ __forceinline__ int whole() const { return top > -__builtin_inff() ? exponent(ceilf(top)) : 0; }
  __device__ __forceinline__ float most() const { return top > -__builtin_inff() ? base + static_cast<float>(whole()) : top; }
};

}  // namespace tcx
