// Attention with a sliding window and sinks over float32 keys and values, the
// choice of its kernels, and what the attentions of a decoding loop share on
// the host: checked arguments, key splits and their join.

#include <algorithm>
#include <cmath>
#include <limits>

#include "decode_stream.hpp"
#include "prompt_attention.hpp"

namespace tcx {
namespace {

// Rows of float32, `features` of them (a multiple of 8) in D: a lane holds the
// chunks of four (two for D = 32) at 16 lanes' distance.
template <int D>
struct FloatRows {
  static constexpr int kFeatures = D / 16, kChunk = D >= 64 ? 4 : 2, kChunks = kFeatures / kChunk;
  using Chunk = float __attribute__((ext_vector_type(kChunk)));
  struct Raw {
    Chunk c[kChunks];
  };
  static __device__ __forceinline__ int feature(int li, int e) {
    return kChunk * (16 * (e / kChunk) + li) + e % kChunk;
  }
  std::int64_t k_base, v_base;
  int li, features;
  __device__ FloatRows(const DecodeArgs& a, int b, int kv, int lane)
      : k_base(b * a.k_stride[0] + kv * a.k_stride[1]), v_base(b * a.v_stride[0] + kv * a.v_stride[1]), li(lane),
        features(a.features) {}
  __device__ __forceinline__ void load(const void* p, std::int64_t base, std::int64_t stride, int key, Raw& raw) const {
    const float* row = static_cast<const float*>(p) + base + key * stride;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const int f = feature(li, c * kChunk);
      raw.c[c] = stream_load(reinterpret_cast<const Chunk*>(row + (f < features ? f : 0)));
    }
  }
  // Chunks past the last feature hold chunk 0 and count as zeros. (Not set to zeros
  // where they are loaded: that would wait for the load.)
  __device__ __forceinline__ void values(const Raw& raw, float (&x)[kFeatures]) const {
    values_all(raw, x);
#pragma unroll
    for (int e = 0; e < kFeatures; ++e)
      if (e >= kChunk || kChunks == 1) x[e] = feature(li, e) < features ? x[e] : 0.F;
  }
  __device__ __forceinline__ void values_all(const Raw& raw, float (&x)[kFeatures]) const {
#pragma unroll
    for (int e = 0; e < kFeatures; ++e) x[e] = raw.c[e / kChunk][e % kChunk];
  }
};

// Joins the split states of a row: a wave each, a lane a split for the weights. Two
// dependent loads and little else: 256 rows of 8 splits 3.9 us, 16 rows of 48 splits
// 6.8 (sixteen splits' loads at a time 6.5).
__global__ __launch_bounds__(256) void join_splits_kernel(DecodeArgs a, std::int64_t rows) {
  const int lane = threadIdx.x & 63, total = a.rows * a.share;
  const std::int64_t step = static_cast<std::int64_t>(gridDim.x) * 4;
  for (std::int64_t row = static_cast<std::int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6); row < rows; row += step) {
    // Lanes past the last split or feature read the last one: loads without branches
    // pass together.
    const auto ml = reinterpret_cast<const float2v_t*>(a.part_ml)[min(lane, a.splits - 1) * rows + row];
    const float m = lane < a.splits ? ml[0] : -__builtin_inff(), l = lane < a.splits ? ml[1] : 0.F;
    float top = m;
#pragma unroll
    for (int offset = 32; offset > 0; offset >>= 1) top = fmaxf(top, __shfl_xor(top, offset, kWave));
    const float weight = __builtin_amdgcn_exp2f(m - (top == -__builtin_inff() ? 0.F : top));
    const float sum = wave_sum(l * weight);
    const int head = static_cast<int>(row / total), b = head / a.kv_heads;
    const RowPlace place = row_place(a, head % a.kv_heads, static_cast<int>(row % total));
    float* out = a.out + b * a.out_stride[0] + place.head * a.out_stride[1] + place.query * a.out_stride[2];
    const bool low = lane < a.features, high = lane + 64 < a.features;
    float x = 0.F, y = 0.F;
    // Eight splits' loads at a time, so that their latencies pass together.
    for (int first = 0; first < a.splits; first += 8) {
      float px[8], py[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float* part = a.part + (min(first + u, a.splits - 1) * rows + row) * a.features;
        px[u] = part[min(lane, a.features - 1)];
        py[u] = part[min(lane + 64, a.features - 1)];
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        // A split past the last has weight 0; it is left out, in case the last holds NaN.
        const float w = __shfl(weight, first + u, kWave);
        if (first + u < a.splits) {
          x = fmaf(px[u], w, x);
          y = fmaf(py[u], w, y);
        }
      }
    }
    if (low) out[lane] = sum == 0.F ? 0.F : x / sum;
    if (high) out[lane + 64] = sum == 0.F ? 0.F : y / sum;
  }
}

constexpr std::int64_t kMostIndex = std::int64_t{1} << 30;

bool all_zero(const std::int64_t (&s)[3]) { return s[0] == 0 && s[1] == 0 && s[2] == 0; }

// The strides asked for, or the contiguous ones of (batch, heads, tokens, features).
bool fill_strides(const std::int64_t (&in)[3], std::int64_t heads, std::int64_t tokens, std::int64_t features,
                  std::int64_t (&out)[3]) {
  if (all_zero(in)) {
    out[2] = features;
    out[1] = tokens * features;
    out[0] = heads * tokens * features;
    return true;
  }
  for (int i = 0; i < 3; ++i) {
    if (in[i] < 0 || in[i] % 4 != 0) return false;
    out[i] = in[i];
  }
  return true;
}

constexpr int kMostSplits = 64;  // join_splits_kernel: a lane each

}  // namespace

int decode_args(const float* q, const void* k, const void* v, float* out, const tcx_hip_window_attention_desc_t* desc,
                bool cache, DecodeArgs& a, bool& done) {
  if (desc == nullptr) return fail(TCX_INVALID_ARGUMENT, "attention descriptor is null");
  const auto& d = *desc;
  if (d.batch < 0 || d.heads < 0 || d.kv_heads < 0 || d.rows < 0 || d.cols < 0)
    return fail(TCX_INVALID_ARGUMENT, "attention extents must be non-negative");
  if (cache ? tcx_hip_cache4_words(d.features) == 0 : !tcx_hip_window_attention_supported(d.features))
    return fail(TCX_INVALID_ARGUMENT, cache ? "a 4-bit cache holds 32, 64 or 128 features"
                                            : "window attention takes a multiple of 8 features from 16 to 128");
  if (d.kv_heads == 0 ? d.heads != 0 : d.heads % d.kv_heads != 0)
    return fail(TCX_INVALID_ARGUMENT, "attention heads must be a multiple of the key heads");
  if (d.window < 0 || d.sinks < 0) return fail(TCX_INVALID_ARGUMENT, "attention window and sinks must be non-negative");
  if (!std::isfinite(d.scale)) return fail(TCX_INVALID_ARGUMENT, "attention scale must be finite");
  done = d.batch == 0 || d.heads == 0 || d.rows == 0;
  if (done) return TCX_OK;
  const std::int64_t share = d.heads / d.kv_heads;
  if (d.cols >= kMostIndex || d.rows >= kMostIndex / share || d.batch >= kMostIndex / d.kv_heads)
    return fail(TCX_INVALID_ARGUMENT, "attention sizes must be below 2^30");
  // Lengths may leave cols keys unread, but a call of no keys needs none.
  if (q == nullptr || out == nullptr || (d.cols > 0 && (k == nullptr || v == nullptr)))
    return fail(TCX_INVALID_ARGUMENT, "attention buffers are null");
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out))
    return fail(TCX_INVALID_ARGUMENT, "attention buffers must be 16-byte aligned");
  a.q = q;
  a.k = k;
  a.v = v;
  a.out = out;
  a.lengths = d.lengths;
  a.flag = d.flag;
  a.batch = static_cast<int>(d.batch);
  a.heads = static_cast<int>(d.heads);
  a.kv_heads = static_cast<int>(d.kv_heads);
  a.share = static_cast<int>(share);
  a.rows = static_cast<int>(d.rows);
  a.cols = static_cast<int>(d.cols);
  a.features = static_cast<int>(d.features);
  // A window of cols keys hides none.
  a.window = d.window >= d.cols ? 0 : static_cast<int>(d.window);
  a.sinks = static_cast<int>(std::min(d.sinks, d.cols));
  a.scale = d.scale;
  const std::int64_t words = cache ? tcx_hip_cache4_words(d.features) : 0;
  static constexpr std::int64_t kContiguous[3] = {0, 0, 0};
  if (!fill_strides(d.q_strides, d.heads, d.rows, d.features, a.q_stride) ||
      !fill_strides(d.out_strides, d.heads, d.rows, d.features, a.out_stride) ||
      !fill_strides(cache ? kContiguous : d.k_strides, d.kv_heads, d.cols, cache ? words : d.features, a.k_stride) ||
      !fill_strides(cache ? kContiguous : d.v_strides, d.kv_heads, d.cols, cache ? words : d.features, a.v_stride))
    return fail(TCX_INVALID_ARGUMENT, "attention strides must be non-negative multiples of 4");
  a.splits = 1;
  a.part = a.part_ml = nullptr;
  return TCX_OK;
}

std::size_t split_bytes(const DecodeArgs& a, int splits) {
  if (splits <= 1) return 0;
  return sizeof(float) * static_cast<std::size_t>(splits) * a.batch * a.kv_heads * a.rows * a.share * (a.features + 2);
}

void place_split(DecodeArgs& a, int splits, void* workspace) {
  a.splits = splits;
  if (splits <= 1) return;
  a.part = static_cast<float*>(workspace);
  a.part_ml = a.part + static_cast<std::size_t>(splits) * a.batch * a.kv_heads * a.rows * a.share * a.features;
}

int plan_splits(const DecodeArgs& a, std::int64_t blocks, int wanted, int split_keys, int least_keys,
                std::size_t workspace_bytes) {
  std::int64_t keys = a.cols;  // a block's rows see at most this many
  if (a.window > 0) keys = std::min<std::int64_t>(keys, std::int64_t{a.window} + a.sinks + a.rows - 1);
  if (keys < least_keys) return 1;
  // The nearest number of parts (2000 keys in parts of 128: 16 of two rounds of 64, not
  // 15 of up to three: 4 sequences of 12 rows, 8 heads of 128 features 32 -> 25 us).
  std::int64_t splits = std::min<std::int64_t>({kMostSplits, wanted / std::max<std::int64_t>(1, blocks), (keys + split_keys / 2) / split_keys});
  while (splits > 1 && split_bytes(a, static_cast<int>(splits)) > workspace_bytes) --splits;
  return static_cast<int>(std::max<std::int64_t>(1, splits));
}

int count_items(const DecodeArgs& a, std::int64_t row_tiles, std::uint32_t& items) {
  const std::int64_t heads = static_cast<std::int64_t>(a.batch) * a.kv_heads;
  if (row_tiles * a.splits > (kMostIndex * 2) / heads) return fail(TCX_INVALID_ARGUMENT, "attention is too large for one call");
  items = static_cast<std::uint32_t>(heads * row_tiles * a.splits);
  return TCX_OK;
}

int join_splits(const DecodeArgs& a, hipStream_t s) {
  const std::int64_t rows = static_cast<std::int64_t>(a.batch) * a.kv_heads * a.rows * a.share;
  hipLaunchKernelGGL(join_splits_kernel, dim3(grid_for(rows, 4, kStrideBlocks)), dim3(256), 0, s, a, rows);
  return check(hipGetLastError(), "attention join launch");
}

namespace {

// How a call runs.
struct WindowForm {
  bool prompt;      // on matrix instructions: `waves` waves of 16 `each` rows
  bool packed;      // from tiles that a first kernel writes to the workspace
  int waves, each, rows;
  int splits;
  std::size_t tiles, bytes;  // of the packed tiles, and of the whole workspace
};

// Tiles of 64 keys that the rows of a head see, at most.
std::int64_t most_tiles(const DecodeArgs& a) {
  const std::int64_t all = (std::int64_t{a.cols} + 63) / 64;
  if (a.window == 0) return all;
  return std::min(all, (std::int64_t{a.sinks} + 63) / 64 + (std::int64_t{a.window} + a.rows + 62) / 64 + 1);
}

std::size_t tile_bytes(const DecodeArgs& a) {
  return a.features <= 32 ? sizeof(PromptTile<32>) : a.features <= 64 ? sizeof(PromptTile<64>) : sizeof(PromptTile<128>);
}

// Which kernel, for `total` rows of `heads` key heads:
// * up to 8 rows stream the keys past them (4 sequences of 12 rows, 8 heads of 128
//   features, 2000 keys: 44 -> 27 us on matrix instructions; of 8 rows 26.7 and 26.2,
//   and one row would leave fifteen columns of sixteen idle);
// * more take matrix instructions, in blocks of 64 rows that pack what they see for
//   themselves (prompt_attention_kernel);
// * where a tile of keys would be packed by four blocks and more of a GPU that is
//   nearly full, or by sixteen, it is packed once instead (prompt_pack_kernel and
//   prompt_tile_kernel): 4 sequences of 200 rows, 16 heads on 8 of 128 features and
//   1000 keys 68 -> 55 us, a prompt of 2048, 16 heads on 4 of 64, 109 -> 63; 2
//   sequences of 64 rows, 16 heads on 4 of 128 features and 8192 keys, 32 blocks, 65
//   -> 80 the other way, one of 512, 8 heads of 64 features, 64 blocks, 17 -> 20;
// * in blocks of 128 rows where those are at least 256, one a CU (2048 rows, 16
//   heads on 4 of 128 features: 131 -> 102 us; the 200 rows above, 128 blocks: 55 ->
//   62 the other way), and of 256 where those are, heads have more than 64
//   features and a window leaves the blocks alike (4096 rows, window 1024: 134 ->
//   118 us; without a window 286 -> 296 the other way).
WindowForm window_form(const DecodeArgs& a, std::size_t workspace_bytes) {
  const int total = a.rows * a.share;
  const std::int64_t heads = static_cast<std::int64_t>(a.batch) * a.kv_heads;
  const auto blocks = [&](int rows) { return heads * ((total + rows - 1) / rows); };
  WindowForm f{};
  f.splits = 1;
  if (total <= 8) {
    f.rows = stream_rows(a);
  } else {
    f.prompt = true;
    f.waves = 4;
    f.each = 1;
    const auto places = static_cast<std::size_t>(heads * most_tiles(a));  // below 2^55; their bytes may pass 64 bits
    if ((total >= 1024 || (total >= 256 && blocks(64) >= 192)) && places <= workspace_bytes / tile_bytes(a)) {
      f.packed = true;
      f.tiles = places * tile_bytes(a);
      if (blocks(128) >= 256) f.waves = 8;
      if (a.features > 64 && a.window > 0 && blocks(256) >= 256) f.each = 2;
    }
    f.rows = 16 * f.waves * f.each;
  }
  // A CU holds four blocks that stream, two of four waves with tiles in LDS and
  // one of eight. Packed tiles are split only where a part keeps 512 keys (512
  // rows, 16 heads on 4, 512 keys: 32 us whole, 40 in four parts). Others from 512
  // keys on, of 128 (8 heads of 64 features, one row: 256 keys 4.9 us whole, 7.8 in
  // two; of 128 features 512 keys 11.8 whole, 9.8 in four).
  f.splits = plan_splits(a, blocks(f.rows), f.prompt ? 2048 / f.waves : 1024, f.packed ? 512 : 128, f.packed ? 1024 : 512,
                         workspace_bytes - f.tiles);
  f.bytes = f.tiles + split_bytes(a, f.splits);
  return f;
}

template <int D>
int launch_packed(const DecodeArgs& a, const WindowForm& form, void* workspace, hipStream_t s) {
  auto* tiles = static_cast<PromptTile<D>*>(workspace);
  const int places = static_cast<int>(most_tiles(a)), row_tiles = (a.rows * a.share + form.rows - 1) / form.rows;
  const std::int64_t heads = static_cast<std::int64_t>(a.batch) * a.kv_heads;
  std::uint32_t items;
  if (int rc = count_items(a, row_tiles, items); rc != TCX_OK) return rc;
  if (places > 0) {
    const unsigned y = static_cast<unsigned>(std::min<std::int64_t>(heads, 65535));
    hipLaunchKernelGGL(prompt_pack_kernel<D>, dim3(places, y), dim3(256), 0, s, a, tiles, places);
    if (int rc = check(hipGetLastError(), "attention pack launch"); rc != TCX_OK) return rc;
  }
  auto go = [&](auto kernel) -> int {
    constexpr std::size_t kShared = 2 * sizeof(PromptTile<D>);
    if constexpr (kShared > 65536) {
      if (int rc = check(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, kShared),
                         "attention shared memory");
          rc != TCX_OK)
        return rc;
    }
    const std::uint32_t per_xcd = (items + 7) / 8;
    hipLaunchKernelGGL(kernel, dim3(grid_for(8 * std::int64_t{per_xcd}, 1, 1 << 22)), dim3(64 * form.waves), kShared, s, a, tiles, places,
                       items, per_xcd, row_tiles);
    return check(hipGetLastError(), "attention launch");
  };
  if constexpr (D == 128)
    if (form.each == 2) return go(prompt_tile_kernel<D, 8, 2>);
  return form.waves == 8 ? go(prompt_tile_kernel<D, 8, 1>) : go(prompt_tile_kernel<D, 4, 1>);
}

template <int D>
int launch_prompt(const DecodeArgs& a, const WindowForm& form, hipStream_t s) {
  const int tiles = (a.rows * a.share + form.rows - 1) / form.rows;
  std::uint32_t items;
  if (int rc = count_items(a, tiles, items); rc != TCX_OK) return rc;
  hipLaunchKernelGGL(prompt_attention_kernel<D>, dim3(grid_for(items, 1, 1 << 22)), dim3(256), 0, s, a, items, tiles);
  return check(hipGetLastError(), "attention launch");
}

template <int D>
int launch_window(DecodeArgs& a, const WindowForm& form, void* workspace, hipStream_t s) {
  place_split(a, form.splits, static_cast<char*>(workspace) + form.tiles);
  const int rc = form.packed   ? launch_packed<D>(a, form, workspace, s)
                 : form.prompt ? launch_prompt<D>(a, form, s)
                               : launch_stream<FloatRows<D>>(a, s);
  return rc == TCX_OK && a.splits > 1 ? join_splits(a, s) : rc;
}

}  // namespace
}  // namespace tcx

extern "C" {

int tcx_hip_window_attention_supported(int64_t features) {
  return features >= 16 && features <= 128 && features % 8 == 0 ? 1 : 0;
}

size_t tcx_hip_window_attention_workspace_bytes(const tcx_hip_window_attention_desc_t* desc) {
  using namespace tcx;
  DecodeArgs a{};
  bool done = false;
  // Any aligned address passes for the buffers, which are not touched.
  alignas(16) static float any[4];
  if (decode_args(any, any, any, any, desc, false, a, done) != TCX_OK || done) return 0;
  return window_form(a, SIZE_MAX).bytes;
}

int tcx_hip_window_attention_f32(const float* q, const float* k, const float* v, float* out,
                                 const tcx_hip_window_attention_desc_t* desc, void* workspace, size_t workspace_bytes,
                                 tcx_stream_t stream) {
  using namespace tcx;
  DecodeArgs a{};
  bool done = false;
  if (int rc = decode_args(q, k, v, out, desc, false, a, done); rc != TCX_OK || done) return rc;
  if (!aligned16(workspace))
    return fail(TCX_INVALID_ARGUMENT, "attention workspace must be 16-byte aligned");
  if (int rc = ready(); rc != TCX_OK) return rc;
  const auto s = static_cast<hipStream_t>(stream);
  const WindowForm form = window_form(a, workspace != nullptr ? workspace_bytes : 0);
  if (a.features <= 32) return launch_window<32>(a, form, workspace, s);
  if (a.features <= 64) return launch_window<64>(a, form, workspace, s);
  return launch_window<128>(a, form, workspace, s);
}

}  // extern "C"
