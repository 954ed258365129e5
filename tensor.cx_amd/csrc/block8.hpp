// Rows in 8-bit floating point: each value a code of four exponent and three
// mantissa bits (e4m3: 448 at most, steps of 2^-9 at least, no infinities), each
// 128 of a row in units of a power of two of their own. Codes are held four to an
// int32 word in whole blocks, zeros behind the last feature; the exponents, a byte
// e + 127 each, four to a word behind each other. A block's exponent is the least
// from -100 on that leaves its largest finite value at 448 units or below: its
// values stay normal bfloat16 numbers (2^-109 to 2^128), which the products rely on.
#pragma once

#include <cstdint>

#include "common.hpp"

namespace tcx {

constexpr int kBlock8 = 128;      // features that share an exponent
constexpr int kLowestByte8 = 27;  // of the exponent -100

constexpr std::int64_t blocks8(std::int64_t features) { return (features + kBlock8 - 1) / kBlock8; }
// Words of a row's exponents.
constexpr std::int64_t scale_words8(std::int64_t features) { return (blocks8(features) + 3) / 4; }

// float32 at any multiple of 4 bytes.
using float4_any = float __attribute__((ext_vector_type(4), aligned(4)));

// Features [f, f + 4) of a row; zeros behind its end.
__device__ __forceinline__ float4_t load_features(const float* row, int f, int features) {
  if (f + 4 <= features) return *reinterpret_cast<const float4_any*>(row + f);
  float4_t v = {0.0F, 0.0F, 0.0F, 0.0F};
#pragma unroll
  for (int e = 0; e < 3; ++e)
    if (f + e < features) v[e] = row[f + e];
  return v;
}
__device__ __forceinline__ void store_features(float* row, int f, int features, float4_t v) {
  if (f + 4 <= features) {
    *reinterpret_cast<float4_any*>(row + f) = v;
    return;
  }
#pragma unroll
  for (int e = 0; e < 3; ++e)
    if (f + e < features) row[f + e] = v[e];
}

__device__ __forceinline__ float4_t add4(float4_t p, float4_t q) {
  return float4_t{p[0] + q[0], p[1] + q[1], p[2] + q[2], p[3] + q[3]};
}

// Maximum over the sixteen lanes of a group, in all of them.
__device__ __forceinline__ std::uint32_t lanes16_max(std::uint32_t x) {
  auto take = [&]<int kControl>() {
    const auto y = static_cast<std::uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), kControl, 0xf, 0xf, true));
    x = x > y ? x : y;
  };
  take.template operator()<0xb1>();   // lane ^ 1
  take.template operator()<0x4e>();   // lane ^ 2
  take.template operator()<0x141>();  // mirror in eight lanes
  take.template operator()<0x140>();  // mirror in sixteen
  return x;
}

// The exponent's byte for a block whose largest finite value has these bits. 448 is
// 1.75 * 2^8: the next power is taken where the mantissa is above .75.
__device__ __forceinline__ int exponent_byte(std::uint32_t top) {
  const int byte = static_cast<int>((top + 0x1fffffU) >> 23) - 8;
  return byte > kLowestByte8 ? byte : kLowestByte8;
}

// Four values in units of 2^-e as a word of codes, each rounded to the nearest, ties
// to even. The instruction makes NaN's code of NaN and infinities.
__device__ __forceinline__ std::uint32_t code_word(float4_t v, float inverse) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inverse, v[1] * inverse, 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * inverse, v[3] * inverse, w, true);
  return static_cast<std::uint32_t>(w);
}

// A block held by sixteen lanes: lane i of them has features 4 i to 4 i + 3 in v[0]
// and 64 + 4 i on in v[1], so that every load and store of a wave is of whole lines.
// Gives the lane's two words of codes and the block's exponent byte.
struct Coded8 {
  std::uint32_t word[2];
  int byte;
};
__device__ __forceinline__ Coded8 encode_block(const float4_t (&v)[2]) {
  std::uint32_t top = 0;
  auto widest = [&](bool finite_only) {
    top = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const std::uint32_t u = __float_as_uint(v[h][e]) & 0x7fffffffU;
        top = top > u || (finite_only && u >= 0x7f800000U) ? top : u;
      }
    top = lanes16_max(top);
  };
  widest(false);
  if (__any(top >= 0x7f800000U)) widest(true);  // the exponent goes by the finite values
  Coded8 c;
  c.byte = exponent_byte(top);
  const float inverse = __uint_as_float(static_cast<std::uint32_t>(254 - c.byte) << 23);
  c.word[0] = code_word(v[0], inverse);
  c.word[1] = code_word(v[1], inverse);
  return c;
}

// Where a wave's lane stands in group g (four blocks, a word of exponents) of a row.
struct Place8 {
  int i, block, feature;  // lane of its block, block and first feature of the row
};
__device__ __forceinline__ Place8 place8(int lane, int g) {
  const int i = lane & 15, block = 4 * g + (lane >> 4);
  return {i, block, block * kBlock8 + 4 * i};
}
// Writes a group's codes and its word of exponents (zeros for blocks past the row).
__device__ __forceinline__ void store_group(std::uint32_t* __restrict__ code_row, std::uint8_t* __restrict__ scale_row,
                                            const Place8& p, int blocks, const Coded8& c) {
  if (p.block < blocks) {
    code_row[static_cast<std::int64_t>(p.block) * 32 + p.i] = c.word[0];
    code_row[static_cast<std::int64_t>(p.block) * 32 + 16 + p.i] = c.word[1];
  }
  if (p.i == 0) scale_row[p.block] = p.block < blocks ? static_cast<std::uint8_t>(c.byte) : 0;
}

// The activations of the fused products (TCX_ACT_*).
inline bool activation_known(int activation) {
  return activation == TCX_ACT_NONE || activation == TCX_ACT_SILU || activation == TCX_ACT_GELU;
}
__device__ __forceinline__ float activate8(float v, int activation) {
  if (activation == TCX_ACT_SILU) return v / (1.0F + expf(-v));
  if (activation == TCX_ACT_GELU) {
    const float inner = 0.7978845608028654F * (v + 0.044715F * v * v * v);
    return 0.5F * v * (1.0F + tanhf(inner));
  }
  return v;
}

inline bool aligned8(const void* p, std::uintptr_t bytes) { return (reinterpret_cast<std::uintptr_t>(p) & (bytes - 1)) == 0; }

}  // namespace tcx
