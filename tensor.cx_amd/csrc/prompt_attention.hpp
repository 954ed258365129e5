// Windowed attention of many rows (prompts, chunks) on matrix instructions.
//
// Products. The inputs are float32, and a float32 matrix instruction does 256
// operations a cycle and CU where a float16 one does 4096. So every factor is
// held as two float16 numbers, hi = half(x) and lo = half(x - hi), 22 bits
// together, and a product is hi hi' + hi lo' + lo hi' with float32 sums: what is
// left out, lo lo', and what lo rounds off are 2^-22 of the product, less than
// what float32 sums of 64 and more terms lose. float16 has five bits of
// exponent, so what is split is first multiplied by a power of two (exact) that
// brings its largest magnitude into [2^14, 2^15): a query and a key row as a
// whole, the values of a key as a whole. A number down to 2^-29 of the largest
// in its row still keeps its 22 bits, and below that an absolute error of 2^-40
// of the largest.
//
// Weights. With s the score in units of log2, p_j = 2^(s_j - base) for a whole number
// `base` of each row, near its largest score, and the softmax's sum is that of p_j,
// whatever the values are. With V_j = 2^e_j V'_j, the outputs are sums of p_j 2^e_j times
// V'_j: `base` is also such that those products stay below 2^16, which are split as
// above, and where a row's values are too large or small for both, a power of two
// 2^rest goes into the products alone. Only what a row sees moves its base and rest,
// so that nothing else has an influence, and by whole numbers, which is exact. What
// the halves cost: a weight is off by 2^-22 of itself and by 2^-35 of the row's largest
// p_j 2^e_j, which shows where one key's values are 2^13 times another's and more.
//
// Layout. A block takes 16 kQ rows a wave of one key head (row r: query r / share,
// head r % share, so that neighbours see the same keys) and walks the keys that
// its rows see, sinks and window in one run, in tiles of 64. Scores are computed
// transposed, S^T = K Q^T: lane (n, g) = (lane % 16, lane / 16) then holds query
// n's scores of keys 16 b + 4 g + v, which are the k indices 8 g .. 8 g + 7 that
// it has to supply as P^T in O^T = V^T P^T once V's columns in LDS are in the
// order (b even 4 g + v, b odd 4 g + v): the weights never leave their lane, and
// neither do the query's maximum, sum and rescaling. V is transposed on its way
// into LDS (rows are features, feature 4 c + e in row e D / 4 + c, so that the
// lanes of a store and of a load meet 16 different slots of 16 bytes).
//
// Stages. K and V have one buffer each. Between barriers A and B a tile's V goes
// from registers into LDS while its scores are computed and the next K is on its
// way; between B and the next A that K goes into LDS while P V is computed and
// the next V is on its way.
//
// Measured: 3 sequences of 37 rows, 6 heads on 2 of 80 features, windows of 50, in 16 us,
// 12 blocks and a chain of loads, splitting and products for each tile; 2 sequences of
// 64 rows, 16 heads on 4 of 128 features and 8192 keys in 65 us. Asking for a tile's K and
// V together was no faster (50 -> 55 us for 8 sequences of 20 rows): what bounds it
// there is splitting them into halves.
#pragma once

#include "decoding.hpp"
#include "halves.hpp"

namespace tcx {

constexpr int kMostKeyField = 253;   // its inverse is a normal number
constexpr int kMostValueField = 245; // 2^118
constexpr int kLeastExp = 141 - kMostValueField;  // of e_j

// The slot of chunk c of 8 features of key row j, and of the 16 bytes of 8 keys at
// chunk c of value row f: xored so that the lanes of a fragment meet different
// banks.
template <int D>
__device__ __forceinline__ int key_slot(int j, int c) {
  constexpr int kChunks = D / 8, kShift = D >= 128 ? 0 : D == 64 ? 1 : 2;
  return j * kChunks + (c ^ ((j >> kShift) & (kChunks - 1) & 15));
}
__device__ __forceinline__ int value_slot(int row, int chunk) { return row * 8 + (chunk ^ ((row >> 1) & 7)); }

// Chunk c of key j, from registers into the tile's buffers; D / 8 neighbouring
// lanes hold a key. Chunks past the last feature become zeros here: set where they are
// loaded, the program would wait there for each load.
template <int D>
__device__ __forceinline__ void pack_keys(const float4_t (&in)[2], int j, int c, int features, half8_t* key_hi, half8_t* key_lo,
                                          float* key_factor) {
  float x[8];
  std::uint32_t most = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    x[e] = 8 * c < features ? in[e / 4][e % 4] : 0.F;
    most = max(most, magnitude(x[e]));
  }
  const int field = scale_field(lanes_most<D / 8>(most), kMostKeyField);
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] *= power_field(field);
  half8_t hi, lo;
  split_halves<8>(x, hi, lo);
  if (j < 64) {
    key_hi[key_slot<D>(j, c)] = hi;
    key_lo[key_slot<D>(j, c)] = lo;
    if (c == 0) key_factor[j] = power_field(254 - field);
  }
}

// The powers of two of quad c (4 features) of the values of keys 4 h .. 4 h + 3;
// D / 4 neighbouring lanes hold a key. Values that are not finite are taken out
// and marked: a product with them would reach rows that do not see them.
template <int D>
__device__ __forceinline__ void measure_values(float4_t (&in)[4], int h, int c, int features, int (&field)[4], float* value_exp,
                                               float* value_unit, int* bad) {
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    std::uint32_t most = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      in[v][e] = 4 * c < features ? in[v][e] : 0.F;
      most = max(most, magnitude(in[v][e]));
    }
    if (__any(most >= 0x7f800000U)) {
      if (most >= 0x7f800000U) {
        most = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (magnitude(in[v][e]) >= 0x7f800000U) in[v][e] = 0.F;
          most = max(most, magnitude(in[v][e]));
        }
        *bad = 1;
      }
    }
    field[v] = scale_field(lanes_most<D / 4>(most), kMostValueField);
    if (c == 0 && h < 16) {
      value_exp[4 * h + v] = static_cast<float>(141 - field[v]);
      value_unit[4 * h + v] = power_field(268 - field[v]);
    }
  }
}

// The largest e_j of a wave's values: of all lanes' fields.
template <int D, int kTasks>
__device__ __forceinline__ int most_exponent(const int (&field)[kTasks][4]) {
  int least = kMostValueField;
#pragma unroll
  for (int i = 0; i < kTasks; ++i) least = min(least, min(min(field[i][0], field[i][1]), min(field[i][2], field[i][3])));
  auto most = static_cast<std::uint32_t>(kMostValueField - least);
  if constexpr (D < 64) most = lanes_most<16>(most);
  return static_cast<int>(across_max(most)) + kLeastExp;
}

__device__ __forceinline__ float largest(const float (&x)[4]) { return fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])); }

template <int D>
__device__ __forceinline__ void pack_values(const float4_t (&in)[4], int h, int c, const int (&field)[4],
                                            half4_t* value_hi, half4_t* value_lo) {
  if (h >= 16) return;
  // Keys 16 b + 4 g .. of h = 4 b + g: half b % 2 of chunk 4 (b / 2) + g.
  const int chunk = 4 * (h >> 3) + (h & 3), half = (h >> 2) & 1;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float x[4];
#pragma unroll
    for (int v = 0; v < 4; ++v) x[v] = in[v][e] * power_field(field[v]);
    half4_t hi, lo;
    split_halves<4>(x, hi, lo);
    const int slot = 2 * value_slot(e * (D / 4) + c, chunk) + half;
    value_hi[slot] = hi;
    value_lo[slot] = lo;
  }
}

// A wave's 16 kQ rows: queries as B operands, the running maxima, sums and outputs.
template <int D, int kQ>
struct PromptRows {
  static constexpr int kSteps = D / 32, kT = D / 16, kQuads = D / 4;
  half8_t q_hi[kQ][kSteps], q_lo[kQ][kSteps];  // lane (n, g): features 32 s + 8 g .. + 7 of query n
  float row_factor[kQ];
  int p_row[kQ];
  acc_t o[kQ][kT];  // feature 4 (r % (D / 4)) + r / (D / 4) of query n at r = 16 i + 4 g + v
  RowBase weights[kQ];
  float l[kQ];  // the sum of this lane's weights
  int first_row, last_row;  // the keys of the wave's first and last queries
  int row0, n16, g;

  __device__ __forceinline__ void start(const DecodeArgs& a, int b, int kv, int n, int r0, int r1, int lane) {
    constexpr float kLog2e = 1.44269502F;
    row0 = r0;
    n16 = lane & 15;
    g = lane >> 4;
    first_row = n - a.rows + row_query(a, min(r0, r1));
    last_row = n - a.rows + row_query(a, min(r0 + kQ * 16 - 1, r1));
#pragma unroll
    for (int x = 0; x < kQ; ++x) {
      const RowPlace at = row_place(a, kv, min(r0 + 16 * x + n16, r1));
      const float* row = a.q + b * a.q_stride[0] + at.head * a.q_stride[1] + at.query * a.q_stride[2];
      p_row[x] = n - a.rows + at.query;
      float q[kSteps][8];
      std::uint32_t most = 0;
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int f = 32 * s + 8 * g + 4 * c;
          const float4_t w = f < a.features ? *reinterpret_cast<const float4_t*>(row + f) : float4_t{0.F, 0.F, 0.F, 0.F};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            q[s][4 * c + e] = w[e];
            most = max(most, magnitude(w[e]));
          }
        }
      most = across_max(most);
      const int field = scale_field(most, kMostKeyField);
      row_factor[x] = power_field(254 - field) * (a.scale * kLog2e);
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
#pragma unroll
        for (int e = 0; e < 8; ++e) q[s][e] *= power_field(field);
        split_halves<8>(q[s], q_hi[x][s], q_lo[x][s]);
      }
#pragma unroll
      for (int i = 0; i < kT; ++i) o[x][i] = acc_t{0.F, 0.F, 0.F, 0.F};
      weights[x].start();
      l[x] = 0.F;
    }
  }

  // Whether some row sees a key of [j0, j0 + 64), and whether each sees them all.
  __device__ __forceinline__ bool any_seen(const DecodeArgs& a, int j0) const {
    return j0 <= last_row && (a.window == 0 || j0 + 63 > first_row - a.window || j0 < a.sinks);
  }
  __device__ __forceinline__ bool all_seen(const DecodeArgs& a, int j0) const {
    return j0 + 63 <= first_row && (a.window == 0 || j0 > last_row - a.window || j0 + 63 < a.sinks);
  }

  // The largest of this lane's s + exponent of a tile.
  __device__ __forceinline__ float most_product(const acc_t (&s)[4], const float* value_exp) const {
    float most = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4_t add = *reinterpret_cast<const float4_t*>(&value_exp[16 * i + 4 * g]);
#pragma unroll
      for (int v = 0; v < 4; ++v) most = fmaxf(most, s[i][v] + add[v]);
    }
    return most;
  }
  // Moves the base of row x of the lanes that need it.
  __device__ __forceinline__ void move(acc_t (&s)[4], int x, const float* value_exp) {
    auto each = [&](auto&& change) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int v = 0; v < 4; ++v) s[i][v] = change(s[i][v]);
    };
    const int scale = weights[x].move(l[x], [](float y) { return across_max(y); }, each,
                                      [&] { return most_product(s, value_exp); });
    if (__any(scale != 0)) {
#pragma unroll
      for (int i = 0; i < kT; ++i)
#pragma unroll
        for (int v = 0; v < 4; ++v) o[x][i][v] = ldexpf(o[x][i][v], scale);
    }
  }

  // A tile's weights, as B operands of the P V products. key_of(k): the key at
  // place k of the tile, or one past every query.
  template <typename F>
  __device__ __forceinline__ void scores(const DecodeArgs& a, const half8_t* key_hi, const half8_t* key_lo,
                                         const float* key_factor, const float* value_exp, const float* value_unit, float most_exp,
                                         bool whole, F&& key_of, half8_t (&p_hi)[kQ][2], half8_t (&p_lo)[kQ][2]) {
    const float neg_inf = -__builtin_inff();
    acc_t s[kQ][4];
#pragma unroll
    for (int x = 0; x < kQ; ++x)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[x][i] = acc_t{0.F, 0.F, 0.F, 0.F};
    // Two blocks of keys at a time, so that no product waits for the one before it.
#pragma unroll
    for (int st = 0; st < kSteps; ++st)
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        half8_t kh[2], kl[2];
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const int slot = key_slot<D>(16 * (i + w) + n16, 4 * st + g);
          kh[w] = key_hi[slot];
          kl[w] = key_lo[slot];
        }
        multiply<2>(kh, kl, [&](int x) -> const half8_t& { return q_hi[x][st]; },
                    [&](int x) -> const half8_t& { return q_lo[x][st]; },
                    [&](int x, int w) -> acc_t& { return s[x][i + w]; });
      }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4_t factor = *reinterpret_cast<const float4_t*>(&key_factor[16 * i + 4 * g]);
#pragma unroll
      for (int x = 0; x < kQ; ++x)
#pragma unroll
        for (int v = 0; v < 4; ++v) s[x][i][v] = fmaf(s[x][i][v], row_factor[x] * factor[v], -weights[x].base);
    }
    if (!whole) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          // The oldest key in the window of key p is p - window + 1; sinks are in every one.
          const int key = key_of(16 * i + 4 * g + v);
          const int until = a.window == 0 || key < a.sinks ? 0x7fffffff : key + a.window;
#pragma unroll
          for (int x = 0; x < kQ; ++x) s[x][i][v] = key <= p_row[x] && until > p_row[x] ? s[x][i][v] : neg_inf;
        }
    }
#pragma unroll
    for (int x = 0; x < kQ; ++x) {
      float most = s[x][0][0];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int v = 0; v < 4; ++v) most = fmaxf(most, s[x][i][v]);
      // The tile's largest exponent shows of most tiles that no product passes the limit.
      if (__any(weights[x].see(most, most + most_exp))) [[unlikely]]
        move(s[x], x, value_exp);
      // A tile's weights are summed by pairs: one by one they would make a chain of a
      // quarter of the keys, which loses small weights beside a large one.
      float sum[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4_t unit = *reinterpret_cast<const float4_t*>(&value_unit[16 * i + 4 * g]);
#pragma unroll
        for (int v = 0; v < 4; ++v) s[x][i][v] = __builtin_amdgcn_exp2f(s[x][i][v]);
        sum[i] = (s[x][i][0] + s[x][i][1]) + (s[x][i][2] + s[x][i][3]);
#pragma unroll
        for (int v = 0; v < 4; ++v) s[x][i][v] *= unit[v];
      }
      l[x] += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      if (__any(weights[x].rest != 0.F)) [[unlikely]] {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int v = 0; v < 4; ++v) s[x][i][v] = ldexpf(s[x][i][v], exponent(weights[x].rest));
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float w[8] = {s[x][2 * k][0],     s[x][2 * k][1],     s[x][2 * k][2],     s[x][2 * k][3],
                            s[x][2 * k + 1][0], s[x][2 * k + 1][1], s[x][2 * k + 1][2], s[x][2 * k + 1][3]};
        split_halves<8>(w, p_hi[x][k], p_lo[x][k]);
      }
    }
  }

  __device__ __forceinline__ void outputs(const half8_t* value_hi, const half8_t* value_lo, const half8_t (&p_hi)[kQ][2],
                                          const half8_t (&p_lo)[kQ][2]) {
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int i = 0; i < kT; i += 2) {
        half8_t vh[2], vl[2];
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const int slot = value_slot(16 * (i + w) + n16, 4 * k + g);
          vh[w] = value_hi[slot];
          vl[w] = value_lo[slot];
        }
        multiply<2>(vh, vl, [&](int x) -> const half8_t& { return p_hi[x][k]; },
                    [&](int x) -> const half8_t& { return p_lo[x][k]; },
                    [&](int x, int w) -> acc_t& { return o[x][i + w]; });
      }
  }

  // sum(x, w) += (hi + lo)[w] (hi + lo)(x) without lo lo, term by term.
  template <int kN, typename H, typename L, typename S>
  __device__ __forceinline__ static void multiply(const half8_t (&hi)[kN], const half8_t (&lo)[kN], H&& b_hi, L&& b_lo,
                                                  S&& sum) {
#pragma unroll
    for (int term = 0; term < 3; ++term)
#pragma unroll
      for (int w = 0; w < kN; ++w)
#pragma unroll
        for (int x = 0; x < kQ; ++x)
          sum(x, w) = __builtin_amdgcn_mfma_f32_16x16x32_f16(term == 0 ? lo[w] : hi[w], term == 1 ? b_lo(x) : b_hi(x),
                                                             sum(x, w), 0, 0, 0);
  }

  // The values that were taken out of a tile of `count` keys, for the rows that see them.
  template <typename F>
  __device__ __forceinline__ void add_bad(const DecodeArgs& a, const float* vb, int count, F&& key_of) {
    for (int k = 0; k < count; ++k) {
      const int key = key_of(k);
      const float* row = vb + key * a.v_stride[2];
#pragma unroll
      for (int i = 0; i < kT; ++i)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const int at = 16 * i + 4 * g + v, f = 4 * (at % kQuads) + at / kQuads;
          const float value = f < a.features ? row[f] : 0.F;
          if (magnitude(value) < 0x7f800000U) continue;
#pragma unroll
          for (int x = 0; x < kQ; ++x)
            if (sees(p_row[x], key, a.window, a.sinks)) o[x][i][v] += value;
        }
    }
  }

  __device__ __forceinline__ void finish(const DecodeArgs& a, int b, int kv, int head, int split, int r1) {
    const int total = a.rows * a.share;
#pragma unroll
    for (int x = 0; x < kQ; ++x) {
      l[x] = across_sum(l[x]);
      weights[x].top = across_max(weights[x].top);
      const int r = row0 + 16 * x + n16;
      if (r > r1) continue;
      const RowPlace place = row_place(a, kv, r);
      const std::int64_t row = (static_cast<std::int64_t>(split) * a.batch * a.kv_heads + head) * total + r;
      float* out = a.splits == 1
                       ? a.out + b * a.out_stride[0] + place.head * a.out_stride[1] + place.query * a.out_stride[2]
                       : a.part + row * a.features;
      // Outputs are held times 2^rest, and 2^14 of V'.
      const int whole = weights[x].whole(), back = -14 - exponent(weights[x].rest) - (a.splits > 1 ? whole : 0);
      const float by = a.splits > 1 ? 1.F : l[x] == 0.F ? 0.F : 1.F / l[x];
      auto result = [&](float y) { return ldexpf(y * by, back); };
      if constexpr (kQuads % 16 == 0) {
        // Rows e D / 4 + c for e = 0..3 are features 4 c + e: one store of four.
#pragma unroll
        for (int i = 0; i < kT / 4; ++i)
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const int f = 4 * (16 * i + 4 * g + v);
            if (f < a.features)
              *reinterpret_cast<float4_t*>(out + f) = float4_t{result(o[x][i][v]), result(o[x][i + kT / 4][v]),
                                                               result(o[x][i + kT / 2][v]), result(o[x][i + 3 * kT / 4][v])};
          }
      } else {
#pragma unroll
        for (int i = 0; i < kT; ++i)
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const int at = 16 * i + 4 * g + v, f = 4 * (at % kQuads) + at / kQuads;
            if (f < a.features) out[f] = result(o[x][i][v]);
          }
      }
      if (a.splits > 1 && g == 0) {
        a.part_ml[2 * row] = weights[x].most();
        a.part_ml[2 * row + 1] = ldexpf(l[x], -whole);
      }
    }
  }
};

// Rows of a block, 16 a wave.
constexpr int kPromptRows = 64;

template <int D>
__global__ __launch_bounds__(256, 2) void prompt_attention_kernel(DecodeArgs a, std::uint32_t items, int row_tiles) {
  constexpr int kThreads = 256, kRows = kPromptRows, kTile = 64;
  constexpr int kKeyChunks = D / 8;  // of 8 features a key
  constexpr int kKeyTasks = (kTile * kKeyChunks + kThreads - 1) / kThreads;
  constexpr int kQuads = D / 4;      // of 4 features of a key's values
  constexpr int kValueTasks = (kTile / 4 * kQuads + kThreads - 1) / kThreads;
  __shared__ half8_t key_hi[8 * D], key_lo[8 * D], value_hi[8 * D], value_lo[8 * D];
  __shared__ alignas(16) float key_factor[kTile];    // 2^-scale of a key
  __shared__ alignas(16) float value_exp[2][kTile];  // e_j of a key
  __shared__ alignas(16) float value_unit[2][kTile];
  __shared__ alignas(16) float value_most[2][4];     // the largest e_j that each wave found
  __shared__ int value_bad[2];                       // some value is not finite
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int total = a.rows * a.share;
  for (std::uint32_t item = blockIdx.x; item < items; item += gridDim.x) {
    const auto [split, from_end, head, b, kv] = block_work(a, item, row_tiles);
    // The last tiles of a prompt see the most keys: they start first.
    const int r0 = (row_tiles - 1 - from_end) * kRows, r1 = min(r0 + kRows, total) - 1;
    const int n = checked_length(a, b);
    const SeenKeys seen = seen_keys(n, a.rows, row_query(a, r0), row_query(a, r1), a.window, a.sinks);
    const int u0 = split_start<kTile>(a, seen.count(), split), u1 = split_start<kTile>(a, seen.count(), split + 1);
    const float* kb = static_cast<const float*>(a.k) + b * a.k_stride[0] + kv * a.k_stride[1];
    const float* vb = static_cast<const float*>(a.v) + b * a.v_stride[0] + kv * a.v_stride[1];

    // Keys and values by turns.
    constexpr int kStage = 2 * kKeyTasks > 4 * kValueTasks ? 2 * kKeyTasks : 4 * kValueTasks;
    float4_t stage[kStage];
    auto& key = reinterpret_cast<float4_t(&)[kKeyTasks][2]>(stage);
    auto& value = reinterpret_cast<float4_t(&)[kValueTasks][4]>(stage);
    int field[kValueTasks][4];
    auto load_keys = [&](int u) {
#pragma unroll
      for (int i = 0; i < kKeyTasks; ++i) {
        const int task = t + i * kThreads, j = task / kKeyChunks, f = 8 * (task % kKeyChunks);
        // Keys past the end are the last one again, which no row sees there.
        const float* row = kb + seen.key(min(u + j, u1 - 1)) * a.k_stride[2] + (f < a.features ? f : 0);
        key[i][0] = *reinterpret_cast<const float4_t*>(row);
        key[i][1] = *reinterpret_cast<const float4_t*>(row + 4);
      }
    };
    auto store_keys = [&] {
#pragma unroll
      for (int i = 0; i < kKeyTasks; ++i) {
        const int task = t + i * kThreads;
        pack_keys<D>(key[i], task / kKeyChunks, task % kKeyChunks, a.features, key_hi, key_lo, key_factor);
      }
    };
    auto load_values = [&](int u) {
#pragma unroll
      for (int i = 0; i < kValueTasks; ++i) {
        const int task = t + i * kThreads, f = 4 * (task % kQuads), h = task / kQuads;
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const float* row = vb + seen.key(min(u + 4 * h + v, u1 - 1)) * a.v_stride[2] + (f < a.features ? f : 0);
          value[i][v] = *reinterpret_cast<const float4_t*>(row);
        }
      }
    };
    auto measure = [&](int buffer) {
#pragma unroll
      for (int i = 0; i < kValueTasks; ++i) {
        const int task = t + i * kThreads;
        measure_values<D>(value[i], task / kQuads, task % kQuads, a.features, field[i], value_exp[buffer], value_unit[buffer],
                          &value_bad[buffer]);
      }
      const int most = most_exponent<D>(field);
      if (lane == 0) value_most[buffer][wave] = static_cast<float>(most);
    };
    auto store_values = [&] {
#pragma unroll
      for (int i = 0; i < kValueTasks; ++i) {
        const int task = t + i * kThreads;
        pack_values<D>(value[i], task / kQuads, task % kQuads, field[i], reinterpret_cast<half4_t*>(value_hi),
                       reinterpret_cast<half4_t*>(value_lo));
      }
    };

    PromptRows<D, 1> rows;
    if (t < 2) value_bad[t] = 0;
    __syncthreads();
    if (u0 < u1) load_keys(u0);
    rows.start(a, b, kv, n, r0 + wave * 16, r1, lane);
    if (u0 < u1) {
      store_keys();
      load_values(u0);
      measure(0);
    }
    int buffer = 0;
    for (int u = u0; u < u1; u += kTile, buffer ^= 1) {
      const bool more = u + kTile < u1;
      __syncthreads();  // A: this tile's keys and value powers are in LDS, the last tile's values are free
      if (t == 0) value_bad[buffer ^ 1] = 0;  // the last tile's mark has been read
      store_values();
      if (more) load_keys(u + kTile);
      // Which of the tile's keys the wave's rows see: the sinks in it by all; its
      // part of the window runs from `from` to `last`.
      const int last = seen.key(min(u + kTile, u1) - 1), from = u >= seen.sinks ? seen.key(u) : seen.first;
      const bool with_window = last >= seen.first;
      const bool any_seen = u < seen.sinks || (from <= rows.last_row && (a.window == 0 || last > rows.first_row - a.window ||
                                                                         from < a.sinks));
      const bool all_seen = u + kTile <= u1 &&
                            (!with_window || (last <= rows.first_row && (a.window == 0 || from > rows.last_row - a.window)));
      auto key_of = [&](int k) { return u + k < u1 ? seen.key(u + k) : 1 << 30; };
      half8_t p_hi[1][2], p_lo[1][2];
      if (any_seen)
        rows.scores(a, key_hi, key_lo, key_factor, value_exp[buffer], value_unit[buffer],
                    largest(value_most[buffer]), all_seen, key_of, p_hi, p_lo);
      __syncthreads();  // B: this tile's values are in LDS, its keys are free
      if (more) {
        store_keys();
        load_values(u + kTile);
      }
      if (any_seen) {
        rows.outputs(value_hi, value_lo, p_hi, p_lo);
        if (value_bad[buffer]) rows.add_bad(a, vb, min(kTile, u1 - u), key_of);
      }
      if (more) measure(buffer ^ 1);
    }
    rows.finish(a, b, kv, head, split, r1);
    __syncthreads();
  }
}

// ------------------------------------------------------------------ long prompts
// Where many blocks see the same keys, splitting them into halves anew in each
// costs more than the products (790 vector instructions a wave and tile, half of
// them for that). A first kernel then writes each tile of 64 keys once, as the
// block's buffers hold it, to the workspace, and prompt_tile_kernel takes the
// tiles from there straight into LDS, two buffers and one barrier a tile.
//
// Measured: 4096 rows, 16 heads on 4 of 128 features, window 1024, in 9.6 us of packing
// (its chain of load, split and store; a block a CU) and some 108 of products, 91
// GFLOP in halves at 0.8 PFLOP/s, of a call of 117 (128 for the products alone under the
// profiler, which runs them with pauses between, at a lower clock); 8192 rows, 16 heads
// of 64 features, window 2048: 26 (134 MB, at a copy's rate) and 209 of 235 (250).
// Counters: matrix pipes busy 96 k cycles of 230 k a SIMD, 182 k of 430 k for the latter,
// where 58 k vector instructions a SIMD at four cycles are as much again; a third of the
// waves' time waits (LDS, barrier) and a third waits to issue.
// A higher priority for half of the waves, and operands read from LDS one step ahead
// (127 -> 123 us under the profiler for the scores; for both products the registers
// spill), gave little.

// A tile as it lies in the workspace and in LDS.
template <int D>
struct PromptTile {
  half8_t key_hi[8 * D], key_lo[8 * D];
  half8_t value_hi[8 * D], value_lo[8 * D];
  float key_factor[64], value_exp[64];
  float value_unit[64];
  int most;  // the largest e_j
  int bad;   // some value is not finite
  int pad[14];
};

// The tiles that a call sees: those of its sinks, then the window's; tile i is
// keys 64 i .. 64 i + 63.
struct SeenTiles {
  int sinks, first, end;  // tiles [0, sinks) and [first, end)
  __host__ __device__ int count() const { return sinks + end - first; }
  __device__ int tile(int i) const { return i < sinks ? i : i - sinks + first; }
  __device__ int place(int tile) const { return tile < sinks ? tile : tile - first + sinks; }
};
__host__ __device__ inline SeenTiles seen_tiles(const SeenKeys& s) {
  SeenTiles t;
  t.sinks = (s.sinks + 63) / 64;
  t.end = (s.end + 63) / 64;
  t.first = s.first / 64 > t.sinks ? s.first / 64 : t.sinks;
  if (t.first > t.end) t.first = t.end;
  return t;
}

template <int D>
__global__ __launch_bounds__(256) void prompt_pack_kernel(DecodeArgs a, PromptTile<D>* tiles, int places) {
  constexpr int kTile = 64, kThreads = 256;
  constexpr int kKeyChunks = D / 8, kKeyTasks = (kTile * kKeyChunks + kThreads - 1) / kThreads;
  constexpr int kQuads = D / 4, kValueTasks = (kTile / 4 * kQuads + kThreads - 1) / kThreads;
  __shared__ PromptTile<D> out;
  const int t = threadIdx.x, place = blockIdx.x;
  const int heads = a.batch * a.kv_heads;
  for (int head = blockIdx.y; head < heads; head += gridDim.y) {
    const int b = __builtin_amdgcn_readfirstlane(head / a.kv_heads), kv = head - b * a.kv_heads;
    const int n = checked_length(a, b);
    const SeenTiles seen = seen_tiles(seen_keys(n, a.rows, 0, a.rows - 1, a.window, a.sinks));
    if (place >= seen.count()) continue;  // the same for the whole block
    const int j0 = 64 * seen.tile(place);
    const float* kb = static_cast<const float*>(a.k) + b * a.k_stride[0] + kv * a.k_stride[1];
    const float* vb = static_cast<const float*>(a.v) + b * a.v_stride[0] + kv * a.v_stride[1];
    if (t == 0) {
      out.most = kLeastExp;
      out.bad = 0;
    }
    float4_t key[kKeyTasks][2], value[kValueTasks][4];
    int field[kValueTasks][4];
#pragma unroll
    for (int i = 0; i < kKeyTasks; ++i) {
      const int task = t + i * kThreads, j = task / kKeyChunks, f = 8 * (task % kKeyChunks);
      const float* row = kb + min(j0 + j, n - 1) * a.k_stride[2] + (f < a.features ? f : 0);
      key[i][0] = *reinterpret_cast<const float4_t*>(row);
      key[i][1] = *reinterpret_cast<const float4_t*>(row + 4);
    }
#pragma unroll
    for (int i = 0; i < kValueTasks; ++i) {
      const int task = t + i * kThreads, f = 4 * (task % kQuads), h = task / kQuads;
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const float* row = vb + min(j0 + 4 * h + v, n - 1) * a.v_stride[2] + (f < a.features ? f : 0);
        value[i][v] = *reinterpret_cast<const float4_t*>(row);
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kKeyTasks; ++i) {
      const int task = t + i * kThreads;
      pack_keys<D>(key[i], task / kKeyChunks, task % kKeyChunks, a.features, out.key_hi, out.key_lo, out.key_factor);
    }
#pragma unroll
    for (int i = 0; i < kValueTasks; ++i) {
      const int task = t + i * kThreads, h = task / kQuads;
      measure_values<D>(value[i], h, task % kQuads, a.features, field[i], out.value_exp, out.value_unit, &out.bad);
      pack_values<D>(value[i], h, task % kQuads, field[i], reinterpret_cast<half4_t*>(out.value_hi),
                     reinterpret_cast<half4_t*>(out.value_lo));
    }
    const int most = most_exponent<D>(field);
    if ((t & 63) == 0) atomicMax(&out.most, most);
    __syncthreads();
    auto* to = reinterpret_cast<float4_t*>(tiles + static_cast<std::int64_t>(head) * places + place);
    const auto* from = reinterpret_cast<const float4_t*>(&out);
    for (int i = t; i < static_cast<int>(sizeof(out) / 16); i += kThreads) to[i] = from[i];
    __syncthreads();
  }
}

// Copies `bytes` (a multiple of 16) from global memory into LDS, straight, 16 bytes a
// lane: instruction p of wave w fills 1024 bytes from (p waves + w) 1024 on.
template <int kWaves, int kBytes>
__device__ __forceinline__ void copy_to_lds(const void* from, void* to, int wave, int lane) {
  using int4v = int __attribute__((ext_vector_type(4)));
  const auto address = reinterpret_cast<std::uint64_t>(from);
  // The resource's size: reads past it give zeros.
  const int4v rsrc{static_cast<int>(address), static_cast<int>(address >> 32), kBytes, 0x00020000};
  const auto lds = static_cast<unsigned>(
      reinterpret_cast<std::uintptr_t>((__attribute__((address_space(3))) void*)to));
  constexpr int kInst = (kBytes + 1024 * kWaves - 1) / (1024 * kWaves);
#pragma unroll
  for (int p = 0; p < kInst; ++p) {
    const int at = (p * kWaves + wave) * 1024;
    if (at >= kBytes) continue;
    // The last lanes of the last piece would write past the tile in LDS.
    if (at + 1024 > kBytes && at + 16 * lane >= kBytes) continue;
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds + at),
                 "v"(at + 16 * lane), "s"(rsrc)
                 : "memory", "m0");
#pragma clang diagnostic pop
  }
}

template <int D, int kWaves, int kQ>
__global__ __launch_bounds__(64 * kWaves, 2) void prompt_tile_kernel(DecodeArgs a, const PromptTile<D>* tiles, int places,
                                                                     std::uint32_t items, std::uint32_t per_xcd,
                                                                     int row_tiles) {
  constexpr int kRows = 16 * kQ * kWaves;
  extern __shared__ __align__(16) char shared[];
  auto* stage = reinterpret_cast<PromptTile<D>*>(shared);  // two
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int total = a.rows * a.share;
  for (std::uint32_t block = blockIdx.x; block < 8 * per_xcd; block += gridDim.x) {
    const std::uint32_t item = block % 8 * per_xcd + block / 8;
    if (item >= items) continue;
    const auto [split, from_end, head, b, kv] = block_work(a, item, row_tiles);
    // The last tiles of a prompt see the most keys: they start first.
    const int r0 = (row_tiles - 1 - from_end) * kRows, r1 = min(r0 + kRows, total) - 1;
    const int n = checked_length(a, b);
    const SeenTiles all = seen_tiles(seen_keys(n, a.rows, 0, a.rows - 1, a.window, a.sinks));
    const SeenTiles seen = seen_tiles(seen_keys(n, a.rows, row_query(a, r0), row_query(a, r1), a.window, a.sinks));
    const PromptTile<D>* from = tiles + static_cast<std::int64_t>(head) * places;
    const float* vb = static_cast<const float*>(a.v) + b * a.v_stride[0] + kv * a.v_stride[1];
    PromptRows<D, kQ> rows;
    const int t0 = split_start<1>(a, seen.count(), split), t1 = split_start<1>(a, seen.count(), split + 1);
    auto copy = [&](int i) {
      copy_to_lds<kWaves, static_cast<int>(sizeof(PromptTile<D>))>(from + all.place(seen.tile(i)), &stage[i & 1], wave, lane);
    };
    if (t0 < t1) copy(t0);
    rows.start(a, b, kv, n, r0 + wave * kQ * 16, r1, lane);
    for (int i = t0; i < t1; ++i) {
      // This tile has landed, for every wave, and the other buffer is free.
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      if (i + 1 < t1) copy(i + 1);
      const PromptTile<D>& now = stage[i & 1];
      const int j0 = 64 * seen.tile(i);
      if (!rows.any_seen(a, j0)) continue;
      half8_t p_hi[kQ][2], p_lo[kQ][2];
      rows.scores(a, now.key_hi, now.key_lo, now.key_factor, now.value_exp, now.value_unit,
                  static_cast<float>(now.most), rows.all_seen(a, j0), [&](int k) { return j0 + k; }, p_hi, p_lo);
      rows.outputs(now.value_hi, now.value_lo, p_hi, p_lo);
      if (now.bad) rows.add_bad(a, vb, min(64, n - j0), [&](int k) { return j0 + k; });
    }
    rows.finish(a, b, kv, head, split, r1);
    __syncthreads();  // both buffers are free again
  }
}

}  // namespace tcx
