// Attention over a 4-bit cache on matrix instructions.
//
// Products. A code c of 0..15 enters as (c - 7.5) 2^-9, which float16 holds: the
// bits c are the float16 c 2^-24, and one packed fused multiply-add of those yields
// it. (Matrix instructions would take the subnormals themselves, but keep five bits
// less of a sum; and codes around zero, with the middle of a group in the place of
// its low end, do not cancel against it in sums over many tokens. Both together: an
// error of 3.6e-5 of the outputs' size over 512 tokens, where this form's is 3e-7.) Their other factor
// is float32 held as two float16 halves of 22 bits together (queries times a power
// of two of their row), so a score is
//   s_j = sum over groups G of step_jG (sum over G of q (c_j - 7.5)) + mid_jG (sum over G of q),
// mid = low + 7.5 step. The second term is one product on the scale words as they
// are: a word is the bfloat16 pair (step, low), and meets 7.5 times the sum of q and
// the sum, in three bfloat16 parts of 24 bits.
//
// Weights. The outputs are sums of (p_j step_jG) (c_j - 7.5) and, apart from the
// codes, of p_j mid_jG. With e_j the exponent of token j's largest low or step, RowBase
// keeps p_j 2^e_j, and so p_j step_jG, in the range of two halves, which hold it to 22
// bits; of a row only what it sees decides, and the softmax's sum is of p_j alone.
//
// Layout. A wave takes 16 or 4 rows of a key head and tiles of 32 tokens, with a
// state of its own; the four waves of a block are joined in LDS, key splits by
// join_splits. Scores are transposed, S^T = K Q^T, so that lane (n, g) holds column
// n's scores of tokens 16 b + 4 g + v, just the k indices it supplies to O^T =
// V^T P^T. A lane's 16 bytes of key codes are four columns of a token, of which
// byte G of each makes group G's operand; its eight values of a V operand are
// the bytes of column n of eight tokens. Steps and middles go through LDS (for each
// group a row of the tile's tokens), where every lane finds its tokens'.
//
// With 16 rows a column is a row. With 4, which is what most models ask of a
// decoding step, columns 4 q + r are four shares of row r: of its scores, group q's
// (the other columns' queries are zeros there, the shares are added across the
// lanes), and of its weights, those of two of a lane's eight tokens, with zeros for
// the rest (the outputs are added across the columns at the end). The work of a
// weight - exponential, a product for each group, halves - is then done once and
// not four times.
//
// Measured: 16 sequences of up to 8192 tokens, 32 heads on 8 of 128 features, 129
// MB in 38.5 us and 4.7 more for the join (a vector kernel of a key at a time: 98 us);
// 131072 tokens of 16 heads of 64, 168 MB, in 47 and 7. A copy would take 23 and 31.
// One sequence of 8192, 32 heads on 8 of 128: 16 rows 23 and 5, 64 rows 52 and 5, 512
// rows 295, each block of 16 rows unpacking all that it sees. What bounds it is issue
// and latency together: a tile of 32 tokens is some 500 instructions on 5 KB, 20 us
// of the 38.5 on vector pipes, and waves wait 38 % of their time (four query rows that
// share a key head, and one, take the same time). Tiles brought by asynchronous copies
// into an LDS ring, and splits of a fixed length, were no faster.
#pragma once

#include "decoding.hpp"
#include "halves.hpp"

namespace tcx {

using short8_t = short __attribute__((ext_vector_type(8)));
using bf8_t = __bf16 __attribute__((ext_vector_type(8)));
using word2_t = std::uint32_t __attribute__((ext_vector_type(2)));
using word4_t = std::uint32_t __attribute__((ext_vector_type(4)));

// Byte `byte` of a in bits 0..7 and of b in bits 16..23.
template <int kByteA, int kByteB>
__device__ __forceinline__ std::uint32_t byte_pair(std::uint32_t a, std::uint32_t b) {
  // Selectors 0..3 are b's bytes, 4..7 a's, 12 is zero.
  return __builtin_amdgcn_perm(a, b, 0x0c000c00U | (kByteB << 16) | (4 + kByteA));
}
// The codes of a pair's low or high half bytes as operands, (c - 7.5) / 512.
template <int kBits>
__device__ __forceinline__ std::uint32_t centred(std::uint32_t bits) {
  const half2_t c = __builtin_bit_cast(half2_t, bits);
  constexpr _Float16 kBy = static_cast<_Float16>(32768.F / (1 << kBits)), kMiddle = static_cast<_Float16>(-7.5F / 512.F);
  return __builtin_bit_cast(std::uint32_t, __builtin_elementwise_fma(c, half2_t{kBy, kBy}, half2_t{kMiddle, kMiddle}));
}
__device__ __forceinline__ std::uint32_t low_codes(std::uint32_t pair) { return centred<0>(pair & 0x000f000fU); }
__device__ __forceinline__ std::uint32_t high_codes(std::uint32_t pair) { return centred<4>(pair & 0x00f000f0U); }
constexpr float kCodeUnit = 512.F;

// Rows of the cache as a lane takes them.
template <int D>
struct CacheLanes {
  static constexpr int kGroups = D / 32, kRowBytes = 20 * kGroups, kScaleBytes = D / 2;
  // Columns c and c + 1 (c = 0 or 2) of a lane's four, byte G of each.
  template <int kG, int kC>
  static __device__ __forceinline__ std::uint32_t columns(const std::uint32_t (&w)[kGroups]) {
    if constexpr (D == 128) return byte_pair<kG, kG>(w[kC], w[kC + 1]);
    else if constexpr (D == 64) return byte_pair<kG, 2 + kG>(w[kC / 2], w[kC / 2]);
    else return byte_pair<kC, kC + 1>(w[0], w[0]);
  }
  // kGroups words, and one lane's byte for each group, at `offset` of a tile.
  static __device__ __forceinline__ void load_words(__amdgpu_buffer_rsrc_t tile, int offset, std::uint32_t (&w)[kGroups]) {
    if constexpr (D == 128) {
      const word4_t v = __builtin_amdgcn_raw_buffer_load_b128(tile, offset, 0, 0);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = v[i];
    } else if constexpr (D == 64) {
      const word2_t v = __builtin_amdgcn_raw_buffer_load_b64(tile, offset, 0, 0);
      w[0] = v[0];
      w[1] = v[1];
    } else {
      w[0] = __builtin_amdgcn_raw_buffer_load_b32(tile, offset, 0, 0);
    }
  }
  static __device__ __forceinline__ std::uint32_t load_bytes(__amdgpu_buffer_rsrc_t tile, int offset) {
    if constexpr (D == 128) return __builtin_amdgcn_raw_buffer_load_b32(tile, offset, 0, 0);
    else if constexpr (D == 64) return static_cast<std::uint16_t>(__builtin_amdgcn_raw_buffer_load_b16(tile, offset, 0, 0));
    else return static_cast<std::uint8_t>(__builtin_amdgcn_raw_buffer_load_b8(tile, offset, 0, 0));
  }
};

// Calls f<0>(), .. f<kN - 1>().
template <int kN, typename F>
__device__ __forceinline__ void for_groups(F&& f) {
  f.template operator()<0>();
  if constexpr (kN > 1) f.template operator()<1>();
  if constexpr (kN > 2) {
    f.template operator()<2>();
    f.template operator()<3>();
  }
}

template <int D, int kRows>
__global__ __launch_bounds__(256, D == 128 && kRows == 16 ? 2 : 3) void cache_attention_kernel(DecodeArgs a, std::uint32_t items, int row_tiles) {
  using Lanes = CacheLanes<D>;
  constexpr int kGroups = D / 32, kT = D / 16, kRow = Lanes::kRowBytes;
  constexpr int kShare = 16 / kRows;  // columns of a row
  constexpr int kTokens = 8 / kShare; // of a lane's weights
  constexpr float kLog2e = 1.44269502F;
  static_assert(kRows == 16 || kRows == 4);
  struct Wave {  // of a group, a token each
    float key_step[kGroups][32], value_step[kGroups][32], value_mid[kGroups][32];
    float value_exp[32];
  };
  constexpr int kPitch = D + 4;
  __shared__ alignas(16) union {
    Wave wave[4];
    float part[4][kRows][kPitch];
  } shared;
  __shared__ float part_m[4][kRows], part_l[4][kRows];
  __shared__ half8_t q_halves[kGroups][2][64];  // the rows' operands, the same for every wave
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int n16 = lane & 15, g = lane >> 4;
  const int column = n16 % kRows, q = n16 / kRows;  // row of the column, and its share
  // The first of the lane's tokens with weights: all of them, or 2 q and 2 q + 1.
  const int token0 = kRows == 16 ? 4 * g : 16 * (q >> 1) + 4 * g + 2 * (q & 1);
  const float neg_inf = -__builtin_inff();
  const int total = a.rows * a.share;
  Wave& mine = shared.wave[wave];
  for (std::uint32_t item = blockIdx.x; item < items; item += gridDim.x) {
    const auto [split, tile_of, head, b, kv] = block_work(a, item, row_tiles);
    const int r0 = tile_of * kRows, r1 = min(r0 + kRows, total) - 1;
    const int n = checked_length(a, b);
    const int i0 = row_query(a, r0), i1 = row_query(a, r1);
    const SeenKeys seen = seen_keys(n, a.rows, i0, i1, a.window, a.sinks);
    const int u0 = split_start<128>(a, seen.count(), split), u1 = split_start<128>(a, seen.count(), split + 1);
    // The split's keys as two runs, of the sinks and of the window, in tiles of 32.
    const int sink_end = min(u1, seen.sinks);
    const int from = seen.key(max(u0, seen.sinks)), to = from + max(u1 - max(u0, seen.sinks), 0);
    const int sink_tiles = u0 < sink_end ? (sink_end - u0 + 31) / 32 : 0, tiles = sink_tiles + (to - from + 31) / 32;
    const char* kb = static_cast<const char*>(a.k) + 4 * (b * a.k_stride[0] + kv * a.k_stride[1]);
    const char* vb = static_cast<const char*>(a.v) + 4 * (b * a.v_stride[0] + kv * a.v_stride[1]);
    const int p_first = n - a.rows + i0, p_last = n - a.rows + i1;

    auto place = [&](int i, int& j0, int& count) {
      const bool sink = i < sink_tiles;
      j0 = __builtin_amdgcn_readfirstlane(sink ? u0 + 32 * i : from + 32 * (i - sink_tiles));
      count = __builtin_amdgcn_readfirstlane(min(32, (sink ? sink_end : to) - j0));  // below 1 past the last tile
    };
    // A tile's key codes of token 16 w + n16, columns 4 g .., and its scale words;
    // value codes of tokens 16 (k / 4) + 4 g + k % 4, column n16, and the scale
    // words of token n16 + 16 (g & 1). Each is loaded again as soon as the tile in
    // hand has used it. A tile is a buffer of its tokens: past a run's end (and past
    // the last tile, which spares the loads a branch) it reads as zeros, and an
    // offset in it has no more than 32 bits.
    std::uint32_t key[2][kGroups], key_scale[2][kGroups], value[8], value_scale[kGroups];
    auto tile_buffer = [&](const char* base, int i) {
      int j0, count;
      place(i, j0, count);
      return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base + static_cast<std::int64_t>(j0) * kRow), 0,
                                               max(count, 0) * kRow, 0x00020000);
    };
    const int at_key = n16 * kRow + 4 * g * kGroups, at_key_scale = n16 * kRow + Lanes::kScaleBytes;
    const int at_value = 4 * g * kRow + n16 * kGroups, at_value_scale = at_key_scale + 16 * (g & 1) * kRow;
    auto load_keys = [&](int i) {
      const auto tile = tile_buffer(kb, i);
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        Lanes::load_words(tile, at_key + 16 * w * kRow, key[w]);
        Lanes::load_words(tile, at_key_scale + 16 * w * kRow, key_scale[w]);
      }
    };
    auto load_value_scales = [&](int i) { Lanes::load_words(tile_buffer(vb, i), at_value_scale, value_scale); };
    auto load_values = [&](int i) {
      const auto tile = tile_buffer(vb, i);
#pragma unroll
      for (int k = 0; k < 8; ++k) value[k] = Lanes::load_bytes(tile, at_value + (16 * (k / 4) + k % 4) * kRow);
    };
    load_keys(wave);
    load_value_scales(wave);
    load_values(wave);

    // The rows: halves of q in the order of the key operands, and the sums of a
    // group's q (those of the bfloat16 parts this lane supplies).
    const RowPlace at = row_place(a, kv, min(r0 + column, r1));
    const int p_row = n - a.rows + at.query;
    short8_t q_sums{};
    float row_factor;
    {
      const float* row = a.q + b * a.q_stride[0] + at.head * a.q_stride[1] + at.query * a.q_stride[2];
      float x[kGroups][8];
      std::uint32_t most = 0;
#pragma unroll
      for (int y = 0; y < kGroups; ++y) {
        const float4_t low = *reinterpret_cast<const float4_t*>(row + 32 * y + 4 * g);
        const float4_t high = *reinterpret_cast<const float4_t*>(row + 32 * y + 16 + 4 * g);
        // Columns 0 and 1: low and high features; then columns 2 and 3.
        const float order[8] = {low[0], low[1], high[0], high[1], low[2], low[3], high[2], high[3]};
        float sum = 0.F;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[y][e] = order[e] * (a.scale * kLog2e);
          most = max(most, magnitude(x[y][e]));
          sum += x[y][e];
        }
        sum = across_sum(sum);
        // Three bfloat16 parts, lanes g = 0, 1 and 2 one each.
        auto part = [&](float value) {
          const __bf16 first = static_cast<__bf16>(value);
          const float rest1 = value - static_cast<float>(first);
          const __bf16 second = static_cast<__bf16>(rest1);
          const __bf16 third = static_cast<__bf16>(rest1 - static_cast<float>(second));
          return g == 3 ? short{0} : __builtin_bit_cast(short, g == 0 ? first : g == 1 ? second : third);
        };
        q_sums[2 * y] = part(7.5F * sum);
        q_sums[2 * y + 1] = part(sum);
      }
      most = across_max(most);
      const int field = scale_field(most, 253);
      row_factor = power_field(254 - field) * kCodeUnit;
#pragma unroll
      for (int y = 0; y < kGroups; ++y) {
        const bool mine_y = kRows == 16 || q == y;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[y][e] = mine_y ? x[y][e] * power_field(field) : 0.F;
        if (wave == y % 4) split_halves<8>(x[y], q_halves[y][0][lane], q_halves[y][1][lane]);
      }
    }
    __syncthreads();

    acc_t o[kT];
    float mid[kGroups], l = 0.F;
    RowBase weights;
    weights.start();
#pragma unroll
    for (int y = 0; y < kT; ++y) o[y] = acc_t{0.F, 0.F, 0.F, 0.F};
#pragma unroll
    for (int y = 0; y < kGroups; ++y) mid[y] = 0.F;

    for (int i = wave; i < tiles; i += 4) {
      int j0, count;
      place(i, j0, count);
      const bool whole = count == 32 && j0 + 31 <= p_first && (a.window == 0 || j0 > p_last - a.window || j0 + 31 < a.sinks);

      // Steps and middles into LDS, a token's by a lane that loaded it.
      {
        std::uint32_t finite = 0;
#pragma unroll
        for (int y = 0; y < kGroups; ++y) {
          const std::uint32_t large = max(value_scale[y] & 0x7fff0000U, value_scale[y] << 16);
          if (large < 0x7f800000U) finite = max(finite, large);
        }
        if (g < 2) {
          const int k = n16 + 16 * g;
#pragma unroll
          for (int y = 0; y < kGroups; ++y) {
            const std::uint32_t even = key_scale[0][y], odd = key_scale[1][y];
            mine.key_step[y][k] = __uint_as_float((g == 0 ? even : odd) << 16);
            const float step = __uint_as_float(value_scale[y] << 16);
            mine.value_step[y][k] = step;
            mine.value_mid[y][k] = fmaf(7.5F, step, __uint_as_float(value_scale[y] & 0xffff0000U));
          }
          // Not below 2^-100, so that what makes up for it stays finite.
          mine.value_exp[k] = static_cast<float>(max(static_cast<int>(finite >> 23) + 1, 27) - 127);
        }
      }
      load_value_scales(i + 4);
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");

      // Scores of tokens 16 w + 4 g + v.
      float s[8];
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        word4_t words{0, 0, 0, 0};
#pragma unroll
        for (int y = 0; y < kGroups; ++y) words[y] = key_scale[w][y];
        const acc_t base = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8_t, words),
                                                                   __builtin_bit_cast(bf8_t, q_sums),
                                                                   acc_t{0.F, 0.F, 0.F, 0.F}, 0, 0, 0);
        acc_t sum{0.F, 0.F, 0.F, 0.F};
        for_groups<kGroups>([&]<int kG>() {
          const std::uint32_t c01 = Lanes::template columns<kG, 0>(key[w]), c23 = Lanes::template columns<kG, 2>(key[w]);
          const half8_t codes = __builtin_bit_cast(
              half8_t, (word4_t{low_codes(c01), high_codes(c01), low_codes(c23), high_codes(c23)}));
          if (kRows == 16) sum = acc_t{0.F, 0.F, 0.F, 0.F};
          sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes, q_halves[kG][1][lane], sum, 0, 0, 0);
          sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes, q_halves[kG][0][lane], sum, 0, 0, 0);
          if constexpr (kRows == 16) {
            const float4_t step = *reinterpret_cast<const float4_t*>(&mine.key_step[kG][16 * w + 4 * g]);
#pragma unroll
            for (int v = 0; v < 4; ++v) s[4 * w + v] = kG == 0 ? step[v] * sum[v] : fmaf(step[v], sum[v], s[4 * w + v]);
          }
        });
        if constexpr (kRows == 4) {
          // Column 4 q + r has group q's sums (zeros past the last group).
          const float4_t step = *reinterpret_cast<const float4_t*>(&mine.key_step[min(q, kGroups - 1)][16 * w + 4 * g]);
#pragma unroll
          for (int v = 0; v < 4; ++v) s[4 * w + v] = shares_sum(step[v] * sum[v]);
        }
#pragma unroll
        for (int v = 0; v < 4; ++v) s[4 * w + v] = fmaf(s[4 * w + v], row_factor, base[v]);
      }
      load_keys(i + 4);
      // The lane's tokens: token(k) of the tile.
      float x[kTokens];
      auto token = [&](int k) { return kRows == 16 ? 16 * (k / 4) + token0 + k % 4 : token0 + k; };
#pragma unroll
      for (int k = 0; k < kTokens; ++k) {
        if constexpr (kRows == 16) x[k] = s[k];
        else x[k] = q & 2 ? (q & 1 ? s[6 + k] : s[4 + k]) : (q & 1 ? s[2 + k] : s[k]);
      }
      std::uint32_t hidden = 0;
      if (!whole) {
#pragma unroll
        for (int k = 0; k < kTokens; ++k) {
          const int j = j0 + token(k), until = a.window == 0 || j < a.sinks ? 0x7fffffff : j + a.window;
          const bool in = token(k) < count && j <= p_row && until > p_row;
          x[k] = in ? x[k] : neg_inf;
          hidden |= (in ? 0U : 1U) << k;
        }
      }
      auto row = [](float y) {
        if constexpr (kRows == 4) y = shares_max(y);
        return across_max(y);
      };
      auto product = [&] {
        float high = neg_inf;
#pragma unroll
        for (int k = 0; k < kTokens; k += 2) {
          const float2v_t add = *reinterpret_cast<const float2v_t*>(&mine.value_exp[token(k)]);
          high = fmaxf(fmaxf(high, x[k] + add[0]), x[k + 1] + add[1]);
        }
        return high;
      };
      float most = neg_inf;
#pragma unroll
      for (int k = 0; k < kTokens; ++k) {
        x[k] -= weights.base;
        most = fmaxf(most, x[k]);
      }
      if (__any(weights.see(most, product()))) [[unlikely]] {
        auto each = [&](auto&& change) {
#pragma unroll
          for (int k = 0; k < kTokens; ++k) x[k] = change(x[k]);
        };
        const int scale = weights.move(l, row, each, product);
        if (__any(scale != 0)) {
#pragma unroll
          for (int y = 0; y < kT; ++y)
#pragma unroll
            for (int v = 0; v < 4; ++v) o[y][v] = ldexpf(o[y][v], scale);
#pragma unroll
          for (int y = 0; y < kGroups; ++y) mid[y] = ldexpf(mid[y], scale);
        }
      }
#pragma unroll
      for (int k = 0; k < kTokens; ++k) {
        x[k] = __builtin_amdgcn_exp2f(x[k]);
        l += x[k];
      }
      const bool scaled = __any(weights.rest != 0.F);

      // A group's weights and its part of the outputs.
      for_groups<kGroups>([&]<int kG>() {
        float step[kTokens], mids[kTokens];
#pragma unroll
        for (int k = 0; k < kTokens; k += 2) {
          const float2v_t u = *reinterpret_cast<const float2v_t*>(&mine.value_step[kG][token(k)]);
          const float2v_t v = *reinterpret_cast<const float2v_t*>(&mine.value_mid[kG][token(k)]);
          step[k] = u[0];
          step[k + 1] = u[1];
          mids[k] = v[0];
          mids[k + 1] = v[1];
        }
        if (!whole) {  // a token that is not seen may hold NaN
#pragma unroll
          for (int k = 0; k < kTokens; ++k) {
            const bool out = hidden >> k & 1U;
            step[k] = out ? 0.F : step[k];
            mids[k] = out ? 0.F : mids[k];
          }
        }
        float weight[kTokens];
#pragma unroll
        for (int k = 0; k < kTokens; ++k) weight[k] = x[k] * step[k];
        if (scaled) [[unlikely]] {
#pragma unroll
          for (int k = 0; k < kTokens; ++k) {
            weight[k] = ldexpf(weight[k], exponent(weights.rest));
            mid[kG] += ldexpf(x[k] * mids[k], exponent(weights.rest));
          }
        } else {
#pragma unroll
          for (int k = 0; k < kTokens; ++k) mid[kG] = fmaf(x[k], mids[k], mid[kG]);
        }
        word4_t w_hi, w_lo;
        if constexpr (kRows == 16) {
          half8_t hi, lo;
          split_halves<8>(weight, hi, lo);
          w_hi = __builtin_bit_cast(word4_t, hi);
          w_lo = __builtin_bit_cast(word4_t, lo);
        } else {
          half2_t hi, lo;
          split_halves<2>(weight, hi, lo);
          const auto pair_hi = __builtin_bit_cast(std::uint32_t, hi), pair_lo = __builtin_bit_cast(std::uint32_t, lo);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            w_hi[k] = q == k ? pair_hi : 0U;
            w_lo[k] = q == k ? pair_lo : 0U;
          }
        }
        word4_t even, odd;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const std::uint32_t p = byte_pair<kG, kG>(value[2 * k], value[2 * k + 1]);
          even[k] = low_codes(p);
          odd[k] = high_codes(p);
        }
        const half8_t c0 = __builtin_bit_cast(half8_t, even), c1 = __builtin_bit_cast(half8_t, odd);
        const half8_t hi = __builtin_bit_cast(half8_t, w_hi), lo = __builtin_bit_cast(half8_t, w_lo);
        o[2 * kG] = __builtin_amdgcn_mfma_f32_16x16x32_f16(c0, lo, o[2 * kG], 0, 0, 0);
        o[2 * kG + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(c1, lo, o[2 * kG + 1], 0, 0, 0);
        o[2 * kG] = __builtin_amdgcn_mfma_f32_16x16x32_f16(c0, hi, o[2 * kG], 0, 0, 0);
        o[2 * kG + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(c1, hi, o[2 * kG + 1], 0, 0, 0);
      });
      load_values(i + 4);
      __builtin_amdgcn_wave_barrier();
    }

    // A row's columns, then the waves' states, joined in LDS.
    l = across_sum(l);
#pragma unroll
    for (int y = 0; y < kGroups; ++y) mid[y] = across_sum(mid[y]);
    weights.top = across_max(weights.top);
    if constexpr (kRows == 4) {
      l = shares_sum(l);
      weights.top = shares_max(weights.top);
#pragma unroll
      for (int y = 0; y < kGroups; ++y) mid[y] = shares_sum(mid[y]);
#pragma unroll
      for (int y = 0; y < kT; ++y)
#pragma unroll
        for (int v = 0; v < 4; ++v) o[y][v] = shares_sum(o[y][v]);
    }
    __syncthreads();  // every wave is done with its part of the union
    if (q == 0) {
      const int whole = weights.whole(), back = -exponent(weights.rest) - whole;
#pragma unroll
      for (int y = 0; y < kT; ++y) {
        float4_t part;
#pragma unroll
        for (int v = 0; v < 4; ++v) part[v] = ldexpf(fmaf(o[y][v], kCodeUnit, mid[y / 2]), back);
        *reinterpret_cast<float4_t*>(&shared.part[wave][column][16 * y + 4 * g]) = part;
      }
      if (g == 0) {
        part_m[wave][column] = weights.most();
        part_l[wave][column] = ldexpf(l, -whole);
      }
    }
    __syncthreads();
    for (int i = t; i < (r1 - r0 + 1) * (D / 4); i += 256) {
      const int r = i / (D / 4), f = 4 * (i % (D / 4));
      float most = part_m[0][r];
#pragma unroll
      for (int w = 1; w < 4; ++w) most = fmaxf(most, part_m[w][r]);
      const float by = most == neg_inf ? 0.F : most;
      float sum = 0.F;
      float4_t value{0.F, 0.F, 0.F, 0.F};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float weight = __builtin_amdgcn_exp2f(part_m[w][r] - by);
        sum = fmaf(part_l[w][r], weight, sum);
        const float4_t part = *reinterpret_cast<const float4_t*>(&shared.part[w][r][f]);
#pragma unroll
        for (int e = 0; e < 4; ++e) value[e] = fmaf(part[e], weight, value[e]);
      }
      if (a.splits == 1) {
        const RowPlace to_row = row_place(a, kv, r0 + r);
        if (sum == 0.F) value = float4_t{0.F, 0.F, 0.F, 0.F};  // a row that sees nothing
        else value /= sum;
        *reinterpret_cast<float4_t*>(a.out + b * a.out_stride[0] + to_row.head * a.out_stride[1] +
                                     to_row.query * a.out_stride[2] + f) = value;
      } else {
        const std::int64_t row = (static_cast<std::int64_t>(split) * a.batch * a.kv_heads + head) * total + r0 + r;
        *reinterpret_cast<float4_t*>(a.part + row * D + f) = value;
        if (f == 0) {
          a.part_ml[2 * row] = most;
          a.part_ml[2 * row + 1] = sum;
        }
      }
    }
    __syncthreads();
  }
}

}  // namespace tcx
