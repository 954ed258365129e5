// Products of rows in 8-bit floating point (block8.hpp) with weights in that form:
// out = act(x w^T + bias) as float32, and the gated product whose result goes back to
// 8 bits.
//
// A code times its block's power of two is a bfloat16 number, exactly, and one
// instruction makes two of them. So codes stay 8 bits wide up to the registers, and
// the products are bfloat16 matrix instructions with float32 sums: exact products.
// The matrix instructions for 8-bit operands have twice the rate, but keep of each
// product only what lies above about 2^-17 of the largest: an error of 1.4e-5 of the
// result's size at any length, where float32 sums have 1e-7.
#include <algorithm>
#include <cstdint>

#include "block8.hpp"

namespace tcx {
namespace {

using bf2_t = __bf16 __attribute__((ext_vector_type(2)));
using bf8_t = __bf16 __attribute__((ext_vector_type(8)));
using acc16_t = float __attribute__((ext_vector_type(16)));

struct Product8 {
  const std::uint8_t* x;         // codes [m][pitch]
  const std::uint8_t* w;         // codes [n][pitch]
  const std::uint32_t* x_scale;  // exponents [m][scale_pitch]
  const std::uint32_t* w_scale;
  const float* bias;  // [n], may be null
  float* out;         // [m][out_stride]
  std::int64_t out_stride;
  int m, n, blocks, pitch, scale_pitch;  // blocks of 128 features; bytes and words between rows
  int activation;
  int tiles_m, tiles_n;
};

// Sixteen codes as two operands of eight.
struct Wide8 {
  bf8_t half[2];
};
__device__ __forceinline__ Wide8 widen(int4_t codes, float unit) {
  Wide8 r;
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const bf2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes[2 * s], unit, false);
    const bf2_t b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes[2 * s], unit, true);
    const bf2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes[2 * s + 1], unit, false);
    const bf2_t d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes[2 * s + 1], unit, true);
    r.half[s] = bf8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
  }
  return r;
}
// The unit of block kt, from the word of exponents that has it.
__device__ __forceinline__ float unit_of(std::uint32_t word, int kt) {
  return __uint_as_float(((word >> (8 * (kt & 3))) & 255U) << 23);
}

// Tile (row, column) of work item `id`: consecutive items share panels, eight tile
// rows deep, and each of the 8 XCDs (which take blocks by turns) gets a run of them,
// so that its L2 serves its blocks.
struct Tile8 {
  int m, n;
};
__device__ __forceinline__ Tile8 tile_of(int block, int tiles_m, int tiles_n) {
  const int total = tiles_m * tiles_n, share = total / 8, rest = total % 8, xcd = block % 8;
  const int id = xcd * share + min(xcd, rest) + block / 8;
  const int width = 8 * tiles_n, group = id / width, first = group * 8, deep = min(tiles_m - first, 8), in = id - group * width;
  return {first + in % deep, in / deep};
}

// Sixteen bytes a lane straight into LDS, lane after lane from `lds` on.
__device__ __forceinline__ void load_lds16(__amdgpu_buffer_rsrc_t r, void* lds, int voffset, int soffset) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)lds, 16, voffset, soffset, 0, 0);
}

// A tile of kM x kN results, a wave's part of it kWM x kWN in 32 x 32 blocks. Each
// step brings a block of 128 features of the tile's rows from memory straight into
// one of two buffers in LDS while the other is computed. Row r's sixteen-byte pieces
// stand in the order piece ^ (r & 7), so that the reads of eight neighbouring rows
// lie in different banks.
template <int kM, int kN, int kWM, int kWN>
__global__ __launch_bounds__(kM / kWM * (kN / kWN) * 64) void product_kernel(Product8 a) {
  constexpr int kWavesN = kN / kWN, kWaves = kM / kWM * kWavesN, kI = kWM / 32, kJ = kWN / 32;
  constexpr int kRows = kM + kN;  // LDS rows of a buffer: x, then w
  constexpr int kLoads = kRows / 8 / kWaves;
  static_assert(kM % (8 * kWaves) == 0 && kN % (8 * kWaves) == 0, "a load is of one operand");
  __shared__ __attribute__((aligned(1024))) std::uint8_t lds[2][kRows * 128];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Tile8 tile = tile_of(blockIdx.x, a.tiles_m, a.tiles_n);
  const int m0 = tile.m * kM, n0 = tile.n * kN;
  const int r = lane & 31, g = lane >> 5;

  // Loads: instruction t of a wave brings rows 8 (t kWaves + wave) on of the buffer; rows
  // past the operand's end are its last one again.
  const auto x_rsrc = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<std::uint8_t*>(a.x + static_cast<std::int64_t>(m0) * a.pitch), static_cast<short>(0),
      min(a.m - m0, kM) * a.pitch, 0x00020000);
  const auto w_rsrc = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<std::uint8_t*>(a.w + static_cast<std::int64_t>(n0) * a.pitch), static_cast<short>(0),
      min(a.n - n0, kN) * a.pitch, 0x00020000);
  int offset[kLoads];
#pragma unroll
  for (int t = 0; t < kLoads; ++t) {
    const int first = 8 * (t * kWaves + wave), row = first + (lane >> 3);
    const int in = t * 8 * kWaves < kM ? min(row, a.m - m0 - 1) : min(row - kM, a.n - n0 - 1);
    offset[t] = in * a.pitch + (((lane & 7) ^ (lane >> 3)) << 4);
  }
  auto load = [&](int kt, int buffer) {
#pragma unroll
    for (int t = 0; t < kLoads; ++t) {
      const int first = 8 * (t * kWaves + wave);
      load_lds16(t * 8 * kWaves < kM ? x_rsrc : w_rsrc, lds[buffer] + first * 128, offset[t], kt * 128);
    }
  };

  // Exponents: a lane's rows of the tile, a word every four steps.
  const int wm = wave / kWavesN * kWM, wn = wave % kWavesN * kWN;
  const std::uint32_t* x_scale[kI];
  const std::uint32_t* w_scale[kJ];
  std::uint32_t x_word[kI], w_word[kJ];
#pragma unroll
  for (int i = 0; i < kI; ++i)
    x_scale[i] = a.x_scale + static_cast<std::int64_t>(min(m0 + wm + 32 * i + r, a.m - 1)) * a.scale_pitch;
#pragma unroll
  for (int j = 0; j < kJ; ++j)
    w_scale[j] = a.w_scale + static_cast<std::int64_t>(min(n0 + wn + 32 * j + r, a.n - 1)) * a.scale_pitch;

  acc16_t acc[kI][kJ];
#pragma unroll
  for (int i = 0; i < kI; ++i)
#pragma unroll
    for (int j = 0; j < kJ; ++j) acc[i][j] = acc16_t{};

  if (a.blocks > 0) load(0, 0);
  for (int kt = 0; kt < a.blocks; ++kt) {
    if ((kt & 3) == 0) {
#pragma unroll
      for (int i = 0; i < kI; ++i) x_word[i] = x_scale[i][kt >> 2];
#pragma unroll
      for (int j = 0; j < kJ; ++j) w_word[j] = w_scale[j][kt >> 2];
    }
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (kt + 1 < a.blocks) load(kt + 1, (kt + 1) & 1);
    const std::uint8_t* x_lds = lds[kt & 1] + (wm + r) * 128;
    const std::uint8_t* w_lds = lds[kt & 1] + (kM + wn + r) * 128;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int piece = ((2 * q + g) ^ (r & 7)) << 4;
      Wide8 x[kI], w[kJ];
#pragma unroll
      for (int i = 0; i < kI; ++i) x[i] = widen(*reinterpret_cast<const int4_t*>(x_lds + i * 4096 + piece), unit_of(x_word[i], kt));
#pragma unroll
      for (int j = 0; j < kJ; ++j) w[j] = widen(*reinterpret_cast<const int4_t*>(w_lds + j * 4096 + piece), unit_of(w_word[j], kt));
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int i = 0; i < kI; ++i)
#pragma unroll
          for (int j = 0; j < kJ; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[i].half[s], w[j].half[s], acc[i][j], 0, 0, 0);
    }
  }

  // Lane (r, g) has column r of rows 8 (e / 4) + 4 g + e % 4 of each block.
#pragma unroll
  for (int j = 0; j < kJ; ++j) {
    const int n = n0 + wn + 32 * j + r;
    if (n >= a.n) continue;
    const float bias = a.bias != nullptr ? a.bias[n] : 0.0F;
#pragma unroll
    for (int i = 0; i < kI; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int m = m0 + wm + 32 * i + 8 * (e / 4) + 4 * g + e % 4;
        if (m < a.m) a.out[static_cast<std::int64_t>(m) * a.out_stride + n] = activate8(acc[i][j][e] + bias, a.activation);
      }
  }
}

template <int kM, int kN, int kWM, int kWN>
int launch_product(Product8 a, hipStream_t s) {
  a.tiles_m = (a.m + kM - 1) / kM;
  a.tiles_n = (a.n + kN - 1) / kN;
  constexpr int kThreads = kM / kWM * (kN / kWN) * 64;
  const std::int64_t tiles = static_cast<std::int64_t>(a.tiles_m) * a.tiles_n;
  if (tiles * kThreads > kMaxLaunchWorkItems || tiles >= (std::int64_t{1} << 30))
    return fail(TCX_INVALID_ARGUMENT, "linear8 has too many results");
  hipLaunchKernelGGL((product_kernel<kM, kN, kWM, kWN>), dim3(static_cast<unsigned>(tiles)), dim3(kThreads), 0, s, a);
  return check(hipGetLastError(), "linear8 launch");
}

// act(gate) * up of float32 rows [gate | up], in 8 bits: a wave a group of four blocks.
struct Gate8 {
  const float* gate_up;  // [rows][2 * width]
  std::uint32_t* codes;
  std::uint8_t* scales;
  int width, blocks, groups, activation;
  std::uint32_t items;
  FastDiv by_groups;
};
__global__ __launch_bounds__(256) void gate_kernel(Gate8 a) {
  const int lane = threadIdx.x & 63;
  const std::uint32_t step = gridDim.x * 4;
  for (std::uint32_t item = blockIdx.x * 4 + (threadIdx.x >> 6); item < a.items; item += step) {
    const std::uint32_t row = a.by_groups(item);
    const Place8 p = place8(lane, static_cast<int>(item - row * a.groups));
    const float* gate = a.gate_up + static_cast<std::int64_t>(row) * 2 * a.width;
    float4_t v[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float4_t first = load_features(gate, p.feature + 64 * h, a.width);
      const float4_t second = load_features(gate + a.width, p.feature + 64 * h, a.width);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[h][e] = activate8(first[e], a.activation) * second[e];
    }
    store_group(a.codes + static_cast<std::int64_t>(row) * a.blocks * 32, a.scales + static_cast<std::int64_t>(row) * a.groups * 4, p,
                a.blocks, encode_block(v));
  }
}

// Checks a descriptor and fills what follows from it; `gated`: weights of 2 * outputs rows.
int product_args(const tcx_hip_linear8_desc_t* desc, bool gated, Product8& a) {
  if (desc == nullptr) return fail(TCX_INVALID_ARGUMENT, "linear8 descriptor is null");
  const auto& d = *desc;
  constexpr std::int64_t kMost = std::int64_t{1} << 30, kMostFeatures = std::int64_t{1} << 22;
  if (d.rows < 0 || d.features < 0 || d.outputs < 0) return fail(TCX_INVALID_ARGUMENT, "linear8 extents must be non-negative");
  if (d.rows >= kMost || d.outputs >= kMost / 2 || d.features >= kMostFeatures)
    return fail(TCX_INVALID_ARGUMENT, "linear8 rows must be below 2^30, outputs below 2^29 and features below 2^22");
  if (!activation_known(d.activation)) return fail(TCX_INVALID_ARGUMENT, "linear8 has no such activation");
  if (!aligned8(d.bias, 4)) return fail(TCX_INVALID_ARGUMENT, "linear8 float32 buffers must be 4-byte aligned");
  a = Product8{};
  a.bias = d.bias;
  a.m = static_cast<int>(d.rows);
  a.n = static_cast<int>(gated ? 2 * d.outputs : d.outputs);
  a.blocks = static_cast<int>(blocks8(d.features));
  a.pitch = a.blocks * kBlock8;
  a.scale_pitch = static_cast<int>(scale_words8(d.features));
  a.activation = gated ? TCX_ACT_NONE : d.activation;
  a.out_stride = gated || d.out_stride == 0 ? a.n : d.out_stride;
  if (a.out_stride < a.n) return fail(TCX_INVALID_ARGUMENT, "linear8 output rows must not overlap");
  return TCX_OK;
}
int operand_args(const std::int32_t* x_codes, const std::int32_t* x_scales, const std::int32_t* w_codes,
                 const std::int32_t* w_scales, Product8& a) {
  if (a.blocks > 0) {
    for (const std::int32_t* p : {x_codes, x_scales, w_codes, w_scales})
      if (p == nullptr) return fail(TCX_INVALID_ARGUMENT, "linear8 buffers are null");
    if (!aligned8(x_codes, 16) || !aligned8(w_codes, 16) || !aligned8(x_scales, 4) || !aligned8(w_scales, 4))
      return fail(TCX_INVALID_ARGUMENT, "linear8 codes must be 16-byte aligned and scales 4-byte aligned");
  }
  a.x = reinterpret_cast<const std::uint8_t*>(x_codes);
  a.w = reinterpret_cast<const std::uint8_t*>(w_codes);
  a.x_scale = reinterpret_cast<const std::uint32_t*>(x_scales);
  a.w_scale = reinterpret_cast<const std::uint32_t*>(w_scales);
  return TCX_OK;
}

int run_product(const Product8& a, hipStream_t s) { return launch_product<128, 128, 64, 64>(a, s); }

std::size_t gate_bytes(const Product8& a) { return static_cast<std::size_t>(a.m) * a.n * sizeof(float); }

}  // namespace
}  // namespace tcx

extern "C" {

size_t tcx_hip_linear8_workspace_bytes(const tcx_hip_linear8_desc_t* desc) {
  using namespace tcx;
  Product8 a;
  if (product_args(desc, false, a) != TCX_OK || a.m == 0 || a.n == 0) return 0;
  return 0;
}

int tcx_hip_linear8(const int32_t* x_codes, const int32_t* x_scales, const int32_t* w_codes, const int32_t* w_scales, float* out,
                    const tcx_hip_linear8_desc_t* desc, void* workspace, size_t workspace_bytes, tcx_stream_t stream) {
  using namespace tcx;
  Product8 a;
  if (int rc = product_args(desc, false, a); rc != TCX_OK) return rc;
  if (a.m == 0 || a.n == 0) return TCX_OK;
  if (out == nullptr) return fail(TCX_INVALID_ARGUMENT, "linear8 buffers are null");
  if (!aligned8(out, 4)) return fail(TCX_INVALID_ARGUMENT, "linear8 float32 buffers must be 4-byte aligned");
  if (!aligned8(workspace, 16)) return fail(TCX_INVALID_ARGUMENT, "linear8 workspace must be 16-byte aligned");
  if (int rc = operand_args(x_codes, x_scales, w_codes, w_scales, a); rc != TCX_OK) return rc;
  if (int rc = ready(); rc != TCX_OK) return rc;
  a.out = out;
  (void)workspace_bytes;
  return run_product(a, static_cast<hipStream_t>(stream));
}

size_t tcx_hip_gated_linear8_workspace_bytes(const tcx_hip_linear8_desc_t* desc) {
  using namespace tcx;
  Product8 a;
  if (product_args(desc, true, a) != TCX_OK || a.m == 0 || a.n == 0) return 0;
  return gate_bytes(a);
}

int tcx_hip_gated_linear8(const int32_t* x_codes, const int32_t* x_scales, const int32_t* w_codes, const int32_t* w_scales,
                          int32_t* codes, int32_t* scales, const tcx_hip_linear8_desc_t* desc, void* workspace,
                          size_t workspace_bytes, tcx_stream_t stream) {
  using namespace tcx;
  Product8 a;
  if (int rc = product_args(desc, true, a); rc != TCX_OK) return rc;
  if (desc->out_stride != 0) return fail(TCX_INVALID_ARGUMENT, "gated_linear8 writes contiguous rows");
  if (a.m == 0 || a.n == 0) return TCX_OK;
  if (codes == nullptr || scales == nullptr) return fail(TCX_INVALID_ARGUMENT, "linear8 buffers are null");
  if (!aligned8(codes, 16) || !aligned8(scales, 4))
    return fail(TCX_INVALID_ARGUMENT, "linear8 codes must be 16-byte aligned and scales 4-byte aligned");
  if (int rc = operand_args(x_codes, x_scales, w_codes, w_scales, a); rc != TCX_OK) return rc;
  if (workspace == nullptr || !aligned8(workspace, 16) || workspace_bytes < gate_bytes(a))
    return fail(TCX_INVALID_ARGUMENT, "gated_linear8 needs a 16-byte aligned workspace of the query's size");
  Gate8 t{};
  t.width = static_cast<int>(desc->outputs);
  t.blocks = static_cast<int>(blocks8(t.width));
  t.groups = static_cast<int>(scale_words8(t.width));
  if (a.m >= (std::int64_t{1} << 31) / t.groups) return fail(TCX_INVALID_ARGUMENT, "linear8 has too many results");
  if (int rc = ready(); rc != TCX_OK) return rc;
  const auto s = static_cast<hipStream_t>(stream);
  a.out = static_cast<float*>(workspace);
  if (int rc = run_product(a, s); rc != TCX_OK) return rc;
  t.gate_up = a.out;
  t.codes = reinterpret_cast<std::uint32_t*>(codes);
  t.scales = reinterpret_cast<std::uint8_t*>(scales);
  t.activation = desc->activation;
  t.items = static_cast<std::uint32_t>(static_cast<std::int64_t>(a.m) * t.groups);
  t.by_groups = FastDiv(static_cast<std::uint32_t>(t.groups));
  hipLaunchKernelGGL(gate_kernel, dim3(grid_for(t.items, 4, kStrideBlocks)), dim3(256), 0, s, t);
  return check(hipGetLastError(), "gated_linear8 launch");
}

}  // extern "C"
