// Rows in 8-bit floating point (block8.hpp): quantised, read back, and as the
// output of the root-mean-square norm with a residual.
#include <algorithm>
#include <cstdint>

#include "block8.hpp"

namespace tcx {
namespace {

// A wave's unit of work is a group of a row: four blocks, 512 features.
struct Rows8 {
  std::int64_t stride;  // floats between rows
  int features, blocks, groups;
  std::uint32_t items;
  FastDiv by_groups;
};

// Reads 4 bytes a feature and writes 1, a group a wave so that enough loads are under
// way without a loop over the row: 11264 x 4096 in 55 us, 4.2 TB/s; 333 x 1100 in 3.0, of
// which 2.4 are the launch.
__global__ __launch_bounds__(256) void quantise_kernel(const float* __restrict__ x, std::uint32_t* __restrict__ codes,
                                                       std::uint8_t* __restrict__ scales, Rows8 a) {
  const int lane = threadIdx.x & 63;
  const std::uint32_t step = gridDim.x * 4;
  for (std::uint32_t item = blockIdx.x * 4 + (threadIdx.x >> 6); item < a.items; item += step) {
    const std::uint32_t row = a.by_groups(item);
    const Place8 p = place8(lane, static_cast<int>(item - row * a.groups));
    const float* from = x + row * a.stride;
    const float4_t v[2] = {load_features(from, p.feature, a.features), load_features(from, p.feature + 64, a.features)};
    store_group(codes + static_cast<std::int64_t>(row) * a.blocks * 32, scales + static_cast<std::int64_t>(row) * a.groups * 4, p,
                a.blocks, encode_block(v));
  }
}

// The other way round, bound by its writes: 11264 x 4096 in 34 us, 6.7 TB/s.
__global__ __launch_bounds__(256) void dequantise_kernel(const std::uint32_t* __restrict__ codes,
                                                         const std::uint8_t* __restrict__ scales, float* __restrict__ out, Rows8 a) {
  const int lane = threadIdx.x & 63;
  const std::uint32_t step = gridDim.x * 4;
  for (std::uint32_t item = blockIdx.x * 4 + (threadIdx.x >> 6); item < a.items; item += step) {
    const std::uint32_t row = a.by_groups(item);
    const Place8 p = place8(lane, static_cast<int>(item - row * a.groups));
    if (p.block >= a.blocks) continue;
    const std::uint32_t* from = codes + (static_cast<std::int64_t>(row) * a.blocks + p.block) * 32 + p.i;
    const std::uint32_t word[2] = {from[0], from[16]};
    const float unit =
        __uint_as_float(static_cast<std::uint32_t>(scales[static_cast<std::int64_t>(row) * a.groups * 4 + p.block]) << 23);
    float* to = out + row * a.stride;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const auto low = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(word[h]), false);
      const auto high = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(word[h]), true);
      store_features(to, p.feature + 64 * h, a.features, float4_t{low[0] * unit, low[1] * unit, high[0] * unit, high[1] * unit});
    }
  }
}

struct Norm8 {
  const float* x;
  const float* residual;
  const float* weight;
  float* sum;
  std::uint32_t* codes;
  std::uint8_t* scales;
  std::int64_t rows, x_stride, residual_stride, sum_stride;
  int features, blocks, groups;
  float epsilon;
};

// Sum over the block's waves of v (a wave's own sum in all its lanes).
__device__ __forceinline__ float block_sum(float v, float* slots) {
  v = wave_sum(v);
  const int waves = blockDim.x >> 6;
  if (waves == 1) return v;
  if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = v;
  __syncthreads();
  float total = 0.0F;
  for (int w = 0; w < waves; ++w) total += slots[w];
  __syncthreads();
  return total;
}
__device__ __forceinline__ float inverse_rms(const Norm8& a, float squares) {
  return 1.0F / sqrtf(squares / static_cast<float>(a.features) + a.epsilon);
}

// Behind a row's last feature zeros times an inverse of NaN or infinity are NaN: their codes
// are set back to zeros once the block's waves have written the row (`inverse` is the same in
// all threads). Selecting zeros before the codes are made, or only for such rows, costs every
// row 1 % (8192 x 8192 with residual 164.3 and 164.6 us, without 162.7).
__device__ __forceinline__ void zeros_behind(const Norm8& a, std::int64_t row, float inverse) {
  if (inverse <= 3.402823466e38F) return;
  __syncthreads();
  std::uint8_t* const codes = reinterpret_cast<std::uint8_t*>(a.codes + row * a.blocks * 32);
  for (int f = a.features + static_cast<int>(threadIdx.x); f < a.blocks * kBlock8; f += blockDim.x) codes[f] = 0;
}

__device__ __forceinline__ float squares4(float4_t v) { return (v[0] * v[0] + v[1] * v[1]) + (v[2] * v[2] + v[3] * v[3]); }

// A block a row, U groups of it in each wave's registers: one read of x and the
// residual, one write of their sum and of the codes. Waves and U are the fewest that hold
// the row, so a short one has more blocks on a CU. Bound by memory: 8192 x 8192 with
// residual, weight and sum in 163 us, 5.4 TB/s; 1 x 4096 in 2.8, nearly all of it the launch
// and three dependent steps (load, sum over the block, store).
template <int U>
__global__ __launch_bounds__(512) void rmsnorm_kernel(Norm8 a) {
  __shared__ float slots[8];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  for (std::int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    float4_t v[U][2];
    float squares = 0.0F;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        v[u][h] = load_features(a.x + row * a.x_stride, place8(lane, wave + u * waves).feature + 64 * h, a.features);
    if (a.residual != nullptr) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          v[u][h] = add4(v[u][h], load_features(a.residual + row * a.residual_stride,
                                                place8(lane, wave + u * waves).feature + 64 * h, a.features));
    }
    if (a.sum != nullptr) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          store_features(a.sum + row * a.sum_stride, place8(lane, wave + u * waves).feature + 64 * h, a.features, v[u][h]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) squares += squares4(v[u][0]) + squares4(v[u][1]);
    const float inverse = inverse_rms(a, block_sum(squares, slots));
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int g = wave + u * waves;
      if (g >= a.groups) break;
      const Place8 p = place8(lane, g);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float4_t w = a.weight != nullptr ? load_features(a.weight, p.feature + 64 * h, a.features) : float4_t{1.0F, 1.0F, 1.0F, 1.0F};
#pragma unroll
        for (int e = 0; e < 4; ++e) v[u][h][e] = v[u][h][e] * inverse * w[e];
      }
      store_group(a.codes + row * a.blocks * 32, a.scales + row * a.groups * 4, p, a.blocks, encode_block(v[u]));
    }
    zeros_behind(a, row, inverse);
  }
}

// Rows that no block's registers hold (above 32768 features): read twice, the second
// time from the cache.
__global__ __launch_bounds__(512) void rmsnorm_long_kernel(Norm8 a) {
  __shared__ float slots[8];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  for (std::int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const float* x = a.x + row * a.x_stride;
    const float* residual = a.residual != nullptr ? a.residual + row * a.residual_stride : nullptr;
    auto read = [&](int f) {
      const float4_t v = load_features(x, f, a.features);
      return residual != nullptr ? add4(v, load_features(residual, f, a.features)) : v;
    };
    float squares = 0.0F;
    for (int g = wave; g < a.groups; g += waves) {
      const Place8 p = place8(lane, g);
#pragma unroll
      for (int h = 0; h < 2; ++h) squares += squares4(read(p.feature + 64 * h));
    }
    const float inverse = inverse_rms(a, block_sum(squares, slots));
    for (int g = wave; g < a.groups; g += waves) {
      const Place8 p = place8(lane, g);
      float4_t v[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        v[h] = read(p.feature + 64 * h);
        if (a.sum != nullptr) store_features(a.sum + row * a.sum_stride, p.feature + 64 * h, a.features, v[h]);
        const float4_t w = a.weight != nullptr ? load_features(a.weight, p.feature + 64 * h, a.features) : float4_t{1.0F, 1.0F, 1.0F, 1.0F};
#pragma unroll
        for (int e = 0; e < 4; ++e) v[h][e] = v[h][e] * inverse * w[e];
      }
      store_group(a.codes + row * a.blocks * 32, a.scales + row * a.groups * 4, p, a.blocks, encode_block(v));
    }
    zeros_behind(a, row, inverse);
  }
}

constexpr std::int64_t kMostFeatures = std::int64_t{1} << 30, kMostItems = std::int64_t{1} << 31;

// Checks what quantise8, dequantise8 and rmsnorm8 share; groups of all rows are
// counted in 31 bits, which 2^31 blocks of 128 bytes and more never reach on a card.
int check_rows(std::int64_t rows, std::int64_t features, const char* what) {
  if (rows < 0 || features < 0) return fail(TCX_INVALID_ARGUMENT, std::string(what) + " extents must be non-negative");
  if (features >= kMostFeatures) return fail(TCX_INVALID_ARGUMENT, std::string(what) + " features must be below 2^30");
  if (features > 0 && rows >= kMostItems / scale_words8(features))
    return fail(TCX_INVALID_ARGUMENT, std::string(what) + " has too many rows");
  return TCX_OK;
}
int check_stride(std::int64_t& stride, std::int64_t features, const char* what) {
  if (stride == 0) stride = features;
  if (stride < 0) return fail(TCX_INVALID_ARGUMENT, std::string(what) + " strides must be non-negative");
  return TCX_OK;
}
int check_words(const void* codes, const void* scales, const char* what) {
  if (codes == nullptr || scales == nullptr) return fail(TCX_INVALID_ARGUMENT, std::string(what) + " buffers are null");
  if (!aligned8(codes, 16) || !aligned8(scales, 4))
    return fail(TCX_INVALID_ARGUMENT, std::string(what) + " codes must be 16-byte aligned and scales 4-byte aligned");
  return TCX_OK;
}
int check_floats(const void* p, const char* what) {
  return aligned8(p, 4) ? TCX_OK : fail(TCX_INVALID_ARGUMENT, std::string(what) + " float32 buffers must be 4-byte aligned");
}

Rows8 rows8(std::int64_t rows, std::int64_t features, std::int64_t stride) {
  Rows8 a;
  a.stride = stride;
  a.features = static_cast<int>(features);
  a.blocks = static_cast<int>(blocks8(features));
  a.groups = static_cast<int>(scale_words8(features));
  a.items = static_cast<std::uint32_t>(rows * a.groups);
  a.by_groups = FastDiv(static_cast<std::uint32_t>(a.groups));
  return a;
}

}  // namespace
}  // namespace tcx

extern "C" {

int64_t tcx_hip_block8_code_words(int64_t features) { return features < 0 ? 0 : tcx::blocks8(features) * 32; }
int64_t tcx_hip_block8_scale_words(int64_t features) { return features < 0 ? 0 : tcx::scale_words8(features); }

int tcx_hip_quantise8(const float* x, int32_t* codes, int32_t* scales, int64_t rows, int64_t features, int64_t x_stride,
                      tcx_stream_t stream) {
  using namespace tcx;
  if (int rc = check_rows(rows, features, "quantise8"); rc != TCX_OK) return rc;
  if (int rc = check_stride(x_stride, features, "quantise8"); rc != TCX_OK) return rc;
  if (rows == 0 || features == 0) return TCX_OK;
  if (x == nullptr) return fail(TCX_INVALID_ARGUMENT, "quantise8 buffers are null");
  if (int rc = check_words(codes, scales, "quantise8"); rc != TCX_OK) return rc;
  if (int rc = check_floats(x, "quantise8"); rc != TCX_OK) return rc;
  if (int rc = ready(); rc != TCX_OK) return rc;
  const Rows8 a = rows8(rows, features, x_stride);
  hipLaunchKernelGGL(quantise_kernel, dim3(grid_for(a.items, 4, kStrideBlocks)), dim3(256), 0, static_cast<hipStream_t>(stream), x,
                     reinterpret_cast<std::uint32_t*>(codes), reinterpret_cast<std::uint8_t*>(scales), a);
  return check(hipGetLastError(), "quantise8 launch");
}

int tcx_hip_dequantise8(const int32_t* codes, const int32_t* scales, float* out, int64_t rows, int64_t features,
                        int64_t out_stride, tcx_stream_t stream) {
  using namespace tcx;
  if (int rc = check_rows(rows, features, "dequantise8"); rc != TCX_OK) return rc;
  if (int rc = check_stride(out_stride, features, "dequantise8"); rc != TCX_OK) return rc;
  if (out_stride < features) return fail(TCX_INVALID_ARGUMENT, "dequantise8 output rows must not overlap");
  if (rows == 0 || features == 0) return TCX_OK;
  if (out == nullptr) return fail(TCX_INVALID_ARGUMENT, "dequantise8 buffers are null");
  if (int rc = check_words(codes, scales, "dequantise8"); rc != TCX_OK) return rc;
  if (int rc = check_floats(out, "dequantise8"); rc != TCX_OK) return rc;
  if (int rc = ready(); rc != TCX_OK) return rc;
  const Rows8 a = rows8(rows, features, out_stride);
  hipLaunchKernelGGL(dequantise_kernel, dim3(grid_for(a.items, 4, kStrideBlocks)), dim3(256), 0, static_cast<hipStream_t>(stream),
                     reinterpret_cast<const std::uint32_t*>(codes), reinterpret_cast<const std::uint8_t*>(scales), out, a);
  return check(hipGetLastError(), "dequantise8 launch");
}

int tcx_hip_rmsnorm8(const float* x, const float* residual, const float* weight, float* sum, int32_t* codes, int32_t* scales,
                     const tcx_hip_rmsnorm8_desc_t* desc, tcx_stream_t stream) {
  using namespace tcx;
  if (desc == nullptr) return fail(TCX_INVALID_ARGUMENT, "rmsnorm8 descriptor is null");
  auto d = *desc;
  if (int rc = check_rows(d.rows, d.features, "rmsnorm8"); rc != TCX_OK) return rc;
  for (std::int64_t* stride : {&d.x_stride, &d.residual_stride, &d.sum_stride})
    if (int rc = check_stride(*stride, d.features, "rmsnorm8"); rc != TCX_OK) return rc;
  if (sum != nullptr && d.sum_stride < d.features) return fail(TCX_INVALID_ARGUMENT, "rmsnorm8 output rows must not overlap");
  if (!(d.epsilon >= 0.0F) || d.epsilon > 3.402823466e38F)
    return fail(TCX_INVALID_ARGUMENT, "rmsnorm8 epsilon must be finite and non-negative");
  if (d.rows == 0 || d.features == 0) return TCX_OK;
  if (x == nullptr) return fail(TCX_INVALID_ARGUMENT, "rmsnorm8 buffers are null");
  if (int rc = check_words(codes, scales, "rmsnorm8"); rc != TCX_OK) return rc;
  for (const float* p : {x, residual, weight, const_cast<const float*>(sum)})
    if (int rc = check_floats(p, "rmsnorm8"); rc != TCX_OK) return rc;
  if (int rc = ready(); rc != TCX_OK) return rc;
  Norm8 a{};
  a.x = x;
  a.residual = residual;
  a.weight = weight;
  a.sum = sum;
  a.codes = reinterpret_cast<std::uint32_t*>(codes);
  a.scales = reinterpret_cast<std::uint8_t*>(scales);
  a.rows = d.rows;
  a.x_stride = d.x_stride;
  a.residual_stride = d.residual_stride;
  a.sum_stride = d.sum_stride;
  a.features = static_cast<int>(d.features);
  a.blocks = static_cast<int>(blocks8(d.features));
  a.groups = static_cast<int>(scale_words8(d.features));
  a.epsilon = d.epsilon;
  const auto s = static_cast<hipStream_t>(stream);
  const unsigned grid = grid_for(d.rows, 1, kStrideBlocks);
  auto go = [&](auto kernel, int waves) {
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(static_cast<unsigned>(waves) * 64), 0, s, a);
    return check(hipGetLastError(), "rmsnorm8 launch");
  };
  if (a.groups <= 8) return go(rmsnorm_kernel<1>, a.groups);
  if (a.groups <= 16) return go(rmsnorm_kernel<2>, 8);
  if (a.groups <= 32) return go(rmsnorm_kernel<4>, 8);
  if (a.groups <= 64) return go(rmsnorm_kernel<8>, 8);
  return go(rmsnorm_long_kernel, 8);
}

}  // extern "C"
