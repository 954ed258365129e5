// Attention of a few rows over a long run of keys that streams past them.
//
// A block takes kRows rows of one key head (queries of the heads that share it,
// neighbours first) and a share of the keys that they see. Sixteen lanes hold a
// key, D / 16 features each, so that a wave takes four keys at a time and a
// block sixteen; each group of lanes keeps an online softmax of its own (the
// running maximum m in units of log2, the sum l, the outputs o) and the sixteen
// states are joined at the end, in registers across a wave's groups and in LDS
// across the waves. Matrix instructions would have their rows idle: a step has as
// many rows as heads share a key head, up to 8.
//
// Measured: 8 sequences of 1028 keys seen, 32 heads on 8 of 128 features, 67 MB in 17.4
// us and 3.9 for the join; a plain read takes 10.5. The rest is a block's start (its
// length, then its queries and first keys) and end around four passes.
#pragma once

#include "decoding.hpp"
#include "halves.hpp"

namespace tcx {

template <class Source, int kRows, int kEach>
__global__ __launch_bounds__(256) void stream_attention_kernel(DecodeArgs a, std::uint32_t items, int row_tiles) {
  constexpr int kF = Source::kFeatures, D = 16 * kF;
  constexpr float kLog2e = 1.44269502F;
  __shared__ float part_o[4][kRows][D];
  __shared__ float part_m[4][kRows], part_l[4][kRows];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, li = lane & 15, group = t >> 4;
  const float neg_inf = -__builtin_inff();
  const int total = a.rows * a.share;
  for (std::uint32_t item = blockIdx.x; item < items; item += gridDim.x) {
    const auto [split, tile, head, b, kv] = block_work(a, item, row_tiles);
    const int r0 = tile * kRows, r1 = min(r0 + kRows, total) - 1;
    const int n = checked_length(a, b);
    const int i0 = row_query(a, r0), i1 = row_query(a, r1);
    const SeenKeys seen = seen_keys(n, a.rows, i0, i1, a.window, a.sinks);
    const int u0 = split_start<16 * kEach>(a, seen.count(), split), u1 = split_start<16 * kEach>(a, seen.count(), split + 1);

    const Source source(a, b, kv, li);
    float q[kRows][kF], o[kRows][kF], m[kRows], l[kRows];
    typename Source::Raw q_raw[kRows];
    int p_row[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const RowPlace at = row_place(a, kv, min(r0 + r, r1));
      const float* row = a.q + b * a.q_stride[0] + at.head * a.q_stride[1] + at.query * a.q_stride[2];
      source.load(row, 0, 0, 0, q_raw[r]);
      p_row[r] = n - a.rows + at.query;
      m[r] = neg_inf;
      l[r] = 0.F;
    }

    // Keys of [u0, u1) from `base` on, whose loads are under way; each is followed
    // by the load of the next pass as soon as it has been used. (Past the end they
    // read the last key again.)
    typename Source::Raw kr[kEach], vr[kEach];
    auto place = [&](int base, int u) { return seen.key(min(base + 16 * u + group, u1 - 1)); };
    auto load_keys = [&](int base) {
#pragma unroll
      for (int u = 0; u < kEach; ++u) source.load(a.k, source.k_base, a.k_stride[2], place(base, u), kr[u]);
    };
    auto load_values = [&](int base) {
#pragma unroll
      for (int u = 0; u < kEach; ++u) source.load(a.v, source.v_base, a.v_stride[2], place(base, u), vr[u]);
    };
    // kMasked: some key is not seen by all of the rows, or lies past the end; its
    // value is left out, not weighted with 0, which would let a NaN through.
    auto pass = [&]<bool kMasked>(int base) {
      float s[kRows][kEach];
      bool in[kRows][kEach];
#pragma unroll
      for (int u = 0; u < kEach; ++u) {
        const int j = place(base, u);
        float x[kF];
        source.values(kr[u], x);
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          float dot = 0.F;
#pragma unroll
          for (int e = 0; e < kF; ++e) dot = fmaf(q[r][e], x[e], dot);
          s[r][u] = lanes16_sum(dot);
          in[r][u] = !kMasked || ((base + 16 * u + group < u1) & sees(p_row[r], j, a.window, a.sinks));
          s[r][u] = in[r][u] ? s[r][u] : neg_inf;
        }
      }
      load_keys(base + 16 * kEach);
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        float top = m[r];
#pragma unroll
        for (int u = 0; u < kEach; ++u) top = fmaxf(top, s[r][u]);
        const float at = top == neg_inf ? 0.F : top;  // nothing seen yet
        const float f = __builtin_amdgcn_exp2f(m[r] - at);
        m[r] = top;
        l[r] *= f;
#pragma unroll
        for (int e = 0; e < kF; ++e) o[r][e] *= f;
#pragma unroll
        for (int u = 0; u < kEach; ++u) {
          s[r][u] = __builtin_amdgcn_exp2f(s[r][u] - at);
          l[r] += s[r][u];
        }
      }
#pragma unroll
      for (int u = 0; u < kEach; ++u) {
        float x[kF];  // past the last feature anything: such outputs are not written
        source.values_all(vr[u], x);
#pragma unroll
        for (int r = 0; r < kRows; ++r)
#pragma unroll
          for (int e = 0; e < kF; ++e) o[r][e] = in[r][u] ? fmaf(s[r][u], x[e], o[r][e]) : o[r][e];
      }
      load_values(base + 16 * kEach);
    };
    int base = u0;
    if (base < u1) {
      load_keys(base);
      load_values(base);
    }
    // The scale and log2 e go into the query: scores come out in units of log2.
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      source.values(q_raw[r], q[r]);
#pragma unroll
      for (int e = 0; e < kF; ++e) {
        q[r][e] *= a.scale * kLog2e;
        o[r][e] = 0.F;
      }
    }
    if (i0 == i1)
      for (; base + 16 * kEach <= u1; base += 16 * kEach) pass.template operator()<false>(base);
    for (; base < u1; base += 16 * kEach) pass.template operator()<true>(base);

    // The wave's four groups, then the block's four waves.
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const float top = across_max(m[r]);
      const float f = __builtin_amdgcn_exp2f(m[r] - (top == neg_inf ? 0.F : top));
      l[r] = across_sum(l[r] * f);
#pragma unroll
      for (int e = 0; e < kF; ++e) {
        const float v = across_sum(o[r][e] * f);
        if (lane < 16) part_o[wave][r][Source::feature(li, e)] = v;
      }
      if (lane == 0) {
        part_m[wave][r] = top;
        part_l[wave][r] = l[r];
      }
    }
    __syncthreads();
    for (int i = t; i < (r1 - r0 + 1) * D; i += 256) {
      const int r = i / D, f = i % D;
      if (f >= a.features) continue;
      float top = part_m[0][r];
#pragma unroll
      for (int w = 1; w < 4; ++w) top = fmaxf(top, part_m[w][r]);
      const float at = top == neg_inf ? 0.F : top;
      float sum = 0.F, value = 0.F;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float weight = __builtin_amdgcn_exp2f(part_m[w][r] - at);
        sum = fmaf(part_l[w][r], weight, sum);
        value = fmaf(part_o[w][r][f], weight, value);
      }
      if (a.splits == 1) {
        const RowPlace place = row_place(a, kv, r0 + r);
        a.out[b * a.out_stride[0] + place.head * a.out_stride[1] + place.query * a.out_stride[2] + f] =
            sum == 0.F ? 0.F : value / sum;  // a row that sees nothing: zeros
      } else {
        const std::int64_t row = (static_cast<std::int64_t>(split) * a.batch * a.kv_heads + head) * total + r0 + r;
        a.part[row * a.features + f] = value;
        if (f == 0) {
          a.part_ml[2 * row] = top;
          a.part_ml[2 * row + 1] = sum;
        }
      }
    }
    __syncthreads();
  }
}

// Rows a block of stream_attention_kernel takes.
inline int stream_rows(const DecodeArgs& a) {
  const int total = a.rows * a.share;
  return total <= 1 ? 1 : total <= 2 ? 2 : total <= 4 ? 4 : 8;
}

template <class Source>
int launch_stream(const DecodeArgs& a, hipStream_t s) {
  const int rows = stream_rows(a), tiles = (a.rows * a.share + rows - 1) / rows;
  std::uint32_t items;
  if (int rc = count_items(a, tiles, items); rc != TCX_OK) return rc;
  const unsigned grid = grid_for(items, 1, 1 << 22);
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(grid), dim3(256), 0, s, a, items, tiles); };
  if (rows == 1) go(stream_attention_kernel<Source, 1, 4>);
  else if (rows == 2) go(stream_attention_kernel<Source, 2, 4>);
  else if (rows == 4) go(stream_attention_kernel<Source, 4, 2>);
  else go(stream_attention_kernel<Source, 8, 2>);
  return check(hipGetLastError(), "attention launch");
}

}  // namespace tcx
