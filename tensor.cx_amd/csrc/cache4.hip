// The 4-bit cache of keys and values: storing float32 tokens in it, reading
// them back, and attention over it.
//
// Of 32 features x: low = min x rounded down to bfloat16, step = (max x - low)
// / 15 rounded up to bfloat16, code = round((x - low) / step) in 0..15, which
// stands for low + step * code. Rounding the ends outwards keeps every x inside
// [low, low + 15 step], so that a value is at most half a step off; bfloat16
// costs the step at most 2^-7 of the range plus 2^-7 |low| / 15, and saves a
// fifth of the bytes that float32 ends would make of a row of 128 (80 against
// 96). A row holds its codes in the order that matrix instructions take them:
// lane n of sixteen finds the features 16 e + n in its own D / 32 bytes, byte g
// holding e = 2 g in its low half and e = 2 g + 1 in its high one.

#include <algorithm>

#include "cache4_attention.hpp"

namespace tcx {
namespace {

// The codes of one lane: D / 32 bytes.
template <int D>
struct LaneCodes;
template <>
struct LaneCodes<128> {
  using type = std::uint32_t;
};
template <>
struct LaneCodes<64> {
  using type = std::uint16_t;
};
template <>
struct LaneCodes<32> {
  using type = std::uint8_t;
};

template <int D>
struct CacheRow {
  static constexpr int kGroups = D / 32, kWords = D / 8 + kGroups;
  using Codes = typename LaneCodes<D>::type;
  using Scales = std::uint32_t __attribute__((ext_vector_type(kGroups)));
};
template <>
struct CacheRow<32> {
  static constexpr int kGroups = 1, kWords = 5;
  using Codes = std::uint8_t;
  using Scales = std::uint32_t;
};

__device__ __forceinline__ std::uint32_t scale_word(std::uint32_t v, int) { return v; }
template <typename V>
__device__ __forceinline__ std::uint32_t scale_word(const V& v, int g) {
  return v[g];
}

// y of the lane that differs in bit kBit of sixteen lanes' index (rotated by half a
// cycle for bits 2 and 3, which comes to the same for sums over all of them).
template <int kControl>
__device__ __forceinline__ float lane_other(float y) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(y), kControl, 0xf, 0xf, true));
}
// The largest or smallest of sixteen lanes' values of each group; lane i gets that of
// group i % kGroups. Lanes give away the groups that they do not keep, so that
// four groups take 11 steps and not 16.
template <int kGroups, bool kLargest>
__device__ __forceinline__ float groups_extreme(float (&x)[kGroups], int li) {
  auto best = [](float u, float v) { return kLargest ? fmaxf(u, v) : fminf(u, v); };
  constexpr int kXor1 = 0xb1, kXor2 = 0x4e, kRor4 = 0x124, kRor8 = 0x128;
  float y;
  if constexpr (kGroups == 1) {
    y = best(x[0], lane_other<kXor1>(x[0]));
    y = best(y, lane_other<kXor2>(y));
  } else {
    const bool odd = li & 1;
    float half[kGroups / 2];
#pragma unroll
    for (int i = 0; i < kGroups / 2; ++i)
      half[i] = best(odd ? x[2 * i + 1] : x[2 * i], lane_other<kXor1>(odd ? x[2 * i] : x[2 * i + 1]));
    if constexpr (kGroups == 2) y = best(half[0], lane_other<kXor2>(half[0]));
    else y = best(li & 2 ? half[1] : half[0], lane_other<kXor2>(li & 2 ? half[0] : half[1]));
  }
  y = best(y, lane_other<kRor4>(y));
  return best(y, lane_other<kRor8>(y));
}
// The value of the lane of the same quad that has group kG.
template <int kGroups, int kG>
__device__ __forceinline__ float of_group(float x) {
  if constexpr (kGroups == 1) return x;
  else return lane_other<kG * 0x55>(x);  // quad_perm of four times kG
}

struct StoreArgs {
  const float* x[2];  // keys, values
  std::int32_t* cache[2];
  const std::int32_t* positions;
  std::int32_t* flag;
  std::int64_t stride[2][3];
  std::int64_t heads;  // batch * kv_heads
  int kv_heads, tokens;
  std::int64_t capacity;
};

// Sixteen lanes a token; blocks of 16 tokens of a head, in grid.y the heads, in
// grid.z = 2 the keys and the values.
//
// The quotient is the correctly rounded one: with r the reciprocal of the step,
// correctly rounded by one Newton step, q = y r corrected by r times the exact
// residual y - q step is (Markstein's theorem; the residual must not underflow,
// which holds for steps from 2^-100 on). It lies in [0, 15 + 2^-19], so adding 1.5
// * 2^23 leaves the code, rounded to even, in the lowest bits. What this does not
// cover - lost groups, far steps - a second, plain path does, for a wave at a time.
//
// Measured: 2 sequences of 4096 tokens, 8 heads of 128 features, 67 MB in and 10 MB
// out, in 17.2 us (28.6 with sixteen lanes' extremes of each group in all lanes, the
// compiler's quotient, a token's place by divisions and loads that stay in the
// caches; two and four tokens of a lane were no faster); 10 us of it are its vector
// instructions.
template <int D>
__global__ __launch_bounds__(256) void cache_store_kernel(StoreArgs a) {
  using Row = CacheRow<D>;
  constexpr int kF = D / 16, kGroups = Row::kGroups;
  const int li = threadIdx.x & 15, which = blockIdx.z;
  for (std::int64_t head = blockIdx.y; head < a.heads; head += gridDim.y) {
    const int b = __builtin_amdgcn_readfirstlane(static_cast<int>(head) / a.kv_heads);
    const int kv = static_cast<int>(head) - b * a.kv_heads;
    const float* base = a.x[which] + b * a.stride[which][0] + kv * a.stride[which][1];
    std::int32_t* cache = a.cache[which] + head * a.capacity * Row::kWords;
    for (int t0 = blockIdx.x * 16; t0 < a.tokens; t0 += gridDim.x * 16) {
      const int t = t0 + static_cast<int>(threadIdx.x >> 4);
      const float* row = base + min(t, a.tokens - 1) * a.stride[which][2] + li;
      float x[kF];
#pragma unroll
      for (int e = 0; e < kF; ++e) x[e] = stream_load(row + 16 * e);
      const std::int64_t slot = static_cast<std::int64_t>(a.positions[b]) + t;
      float least[kGroups], most[kGroups], finite = 0.F;
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        least[g] = fminf(x[2 * g], x[2 * g + 1]);
        most[g] = fmaxf(x[2 * g], x[2 * g + 1]);
        finite = fmaf(x[2 * g], 0.F, fmaf(x[2 * g + 1], 0.F, finite));  // else NaN
      }
      const float lowest = groups_extreme<kGroups, false>(least, li) + 0.F;  // no -0
      const float highest = groups_extreme<kGroups, true>(most, li);
      const std::uint32_t bits = __float_as_uint(lowest);
      std::uint32_t low = bits & 0xffff0000U;
      if (low != bits && (bits >> 31)) low += 0x10000U;
      const float span = (highest - __uint_as_float(low)) * (1.F / 15.F) + 0.F;
      std::uint32_t size = (__float_as_uint(span) + 0xffffU) & 0xffff0000U;
      const float from = __uint_as_float(low), by = __uint_as_float(size);
      // Steps of 0 (all codes are 0) and from 2^-100 to 2^100.
      const bool plain = finite == 0.F && (low & 0x7f800000U) != 0x7f800000U &&
                         (by == 0.F || (by >= 0x1p-100F && by <= 0x1p100F));
      std::uint32_t codes = 0;
      if (__all(plain)) {
        const float near = __builtin_amdgcn_rcpf(by);
        const float inverse = by == 0.F ? 0.F : fmaf(fmaf(-by, near, 1.F), near, near);
        std::uint32_t extra = 0;
        for_groups<kGroups>([&]<int kG>() {
          const float f = of_group<kGroups, kG>(from), s = of_group<kGroups, kG>(by), r = of_group<kGroups, kG>(inverse);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float y = x[2 * kG + h] - f, q = y * r;
            const float quotient = fmaf(fmaf(-q, s, y), r, q);
            codes += __float_as_uint(quotient + 12582912.F) << (4 * (2 * kG + h));
            extra += 0x4b400000U << (4 * (2 * kG + h));
          }
        });
        codes -= extra;
      } else {
        std::uint32_t scales = low | (size >> 16);
        for_groups<kGroups>([&]<int kG>() {
          // Whether the group holds a number that is not finite: of the wave's lanes, this token's.
          const float first = fabsf(x[2 * kG]), second = fabsf(x[2 * kG + 1]);
          const bool bad = (__ballot(!(first < __builtin_inff()) || !(second < __builtin_inff())) >> (threadIdx.x & 48)) & 0xffffU;
          const float f = of_group<kGroups, kG>(from), s = of_group<kGroups, kG>(by);
          const bool lost = bad || !(fabsf(f) < __builtin_inff()) || !(s < __builtin_inff());
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float c = fminf(fmaxf(rintf((x[2 * kG + h] - f) / s), 0.F), 15.F);
            if (!lost && s > 0.F) codes |= static_cast<std::uint32_t>(c) << (4 * (2 * kG + h));
          }
          if (lost && (li & (kGroups - 1)) == kG) scales = 0x7fc07fc0U;
        });
        low = scales & 0xffff0000U;
        size = scales << 16;
      }
      if (t >= a.tokens) continue;
      if (slot < 0 || slot >= a.capacity) {
        if (a.flag != nullptr) __hip_atomic_store(a.flag, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
        continue;
      }
      std::int32_t* out = cache + slot * Row::kWords;
      reinterpret_cast<typename Row::Codes*>(out)[li] = static_cast<typename Row::Codes>(codes);
      if (li < kGroups) out[D / 8 + li] = static_cast<std::int32_t>(low | (size >> 16));
    }
  }
}

// Sixteen lanes a token; blocks of 16 tokens of a head, in grid.y the heads. Bound by
// its writes: 80000 tokens of 128 features, 6.4 MB in and 41 MB out, in 10.4 us.
template <int D>
__global__ __launch_bounds__(256) void cache_load_kernel(const std::int32_t* __restrict__ cache, float* __restrict__ out,
                                                         std::int64_t heads, std::int64_t capacity, std::int64_t start,
                                                         std::int64_t count) {
  using Row = CacheRow<D>;
  const int li = threadIdx.x & 15;
  for (std::int64_t head = blockIdx.y; head < heads; head += gridDim.y) {
    const std::int32_t* first = cache + (head * capacity + start) * Row::kWords;
    float* to = out + head * count * D + li;
    for (std::int64_t t = static_cast<std::int64_t>(blockIdx.x) * 16 + (threadIdx.x >> 4); t < count;
         t += static_cast<std::int64_t>(gridDim.x) * 16) {
      const std::int32_t* row = first + t * Row::kWords;
      const std::uint32_t codes = reinterpret_cast<const typename Row::Codes*>(row)[li];
      const auto scales = *reinterpret_cast<const typename Row::Scales*>(row + D / 8);
#pragma unroll
      for (int e = 0; e < D / 16; ++e) {
        const std::uint32_t word = scale_word(scales, e / 2);
        to[t * D + 16 * e] = fmaf(__uint_as_float(word << 16), static_cast<float>((codes >> (4 * e)) & 15U),
                                  __uint_as_float(word & 0xffff0000U));
      }
    }
  }
}

// Rows of a block: 4 where a head has no more, else 16 (cache_attention_kernel:
// 16 sequences of 4096 to 8192 tokens, 8 heads of 128 features, one row each 47.3
// -> 38.5 us, four 46.0 -> 38.7).
int cache_rows(const DecodeArgs& a) { return a.rows * a.share <= 4 ? 4 : 16; }

// 768 blocks fill the GPU three to a CU (512 and 1024: 40.3 and 39.2 us against
// 38.5), and a split of fewer than 256 keys costs more than it spares; nor do two or
// three pay for the join (8 heads of 64 features, one sequence: 512 keys 8.6 us
// whole, 10.1 in two; 1024 keys 12.5 whole, 9.9 in four).
int cache_splits(const DecodeArgs& a, std::size_t workspace_bytes) {
  const int rows = cache_rows(a);
  const std::int64_t blocks = static_cast<std::int64_t>(a.batch) * a.kv_heads * ((a.rows * a.share + rows - 1) / rows);
  return plan_splits(a, blocks, 768, 256, 1024, workspace_bytes);
}

template <int D, int kRows>
int launch_cache(const DecodeArgs& a, hipStream_t s) {
  const int tiles = (a.rows * a.share + kRows - 1) / kRows;
  std::uint32_t items;
  if (int rc = count_items(a, tiles, items); rc != TCX_OK) return rc;
  hipLaunchKernelGGL((cache_attention_kernel<D, kRows>), dim3(grid_for(items, 1, 1 << 22)), dim3(256), 0, s, a, items, tiles);
  return check(hipGetLastError(), "cache attention launch");
}
template <int D>
int launch_cache(const DecodeArgs& a, hipStream_t s) {
  return cache_rows(a) == 4 ? launch_cache<D, 4>(a, s) : launch_cache<D, 16>(a, s);
}

}  // namespace
}  // namespace tcx

extern "C" {

int64_t tcx_hip_cache4_words(int64_t features) {
  return features == 32 || features == 64 || features == 128 ? features / 8 + features / 32 : 0;
}

int tcx_hip_cache4_store(const float* key, const float* value, int32_t* key_cache, int32_t* value_cache,
                         const int32_t* positions, const tcx_hip_cache4_store_desc_t* desc, tcx_stream_t stream) {
  using namespace tcx;
  if (desc == nullptr) return fail(TCX_INVALID_ARGUMENT, "cache store descriptor is null");
  const auto& d = *desc;
  if (d.batch < 0 || d.kv_heads < 0 || d.tokens < 0 || d.capacity < 0)
    return fail(TCX_INVALID_ARGUMENT, "cache store extents must be non-negative");
  if (tcx_hip_cache4_words(d.features) == 0)
    return fail(TCX_INVALID_ARGUMENT, "a 4-bit cache holds 32, 64 or 128 features");
  if (d.batch == 0 || d.kv_heads == 0 || d.tokens == 0) return TCX_OK;
  constexpr std::int64_t kMost = std::int64_t{1} << 30;
  if (d.capacity >= kMost || d.tokens >= kMost || d.batch >= kMost / d.kv_heads)
    return fail(TCX_INVALID_ARGUMENT, "cache store sizes must be below 2^30");
  if (key == nullptr || value == nullptr || positions == nullptr ||
      (d.capacity > 0 && (key_cache == nullptr || value_cache == nullptr)))
    return fail(TCX_INVALID_ARGUMENT, "cache store buffers are null");
  if (!aligned16(key) || !aligned16(value) || !aligned16(key_cache) || !aligned16(value_cache))
    return fail(TCX_INVALID_ARGUMENT, "cache store buffers must be 16-byte aligned");
  StoreArgs a{};
  for (int w = 0; w < 2; ++w) {
    const std::int64_t(&in)[3] = w == 0 ? d.key_strides : d.value_strides;
    const bool contiguous = in[0] == 0 && in[1] == 0 && in[2] == 0;
    a.stride[w][2] = contiguous ? d.features : in[2];
    a.stride[w][1] = contiguous ? d.tokens * d.features : in[1];
    a.stride[w][0] = contiguous ? d.kv_heads * d.tokens * d.features : in[0];
    for (std::int64_t s : a.stride[w])
      if (s < 0 || s % 4 != 0)
        return fail(TCX_INVALID_ARGUMENT, "cache store strides must be non-negative multiples of 4");
  }
  if (int rc = ready(); rc != TCX_OK) return rc;
  a.x[0] = key;
  a.x[1] = value;
  a.cache[0] = key_cache;
  a.cache[1] = value_cache;
  a.positions = positions;
  a.flag = d.flag;
  a.heads = d.batch * d.kv_heads;
  a.kv_heads = static_cast<int>(d.kv_heads);
  a.tokens = static_cast<int>(d.tokens);
  a.capacity = d.capacity;
  const dim3 grid(grid_for(d.tokens, 16, 1 << 20), static_cast<unsigned>(std::min<std::int64_t>(a.heads, 65535)), 2);
  const auto s = static_cast<hipStream_t>(stream);
  if (d.features == 32) hipLaunchKernelGGL(cache_store_kernel<32>, grid, dim3(256), 0, s, a);
  else if (d.features == 64) hipLaunchKernelGGL(cache_store_kernel<64>, grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL(cache_store_kernel<128>, grid, dim3(256), 0, s, a);
  return check(hipGetLastError(), "cache store launch");
}

int tcx_hip_cache4_load(const int32_t* cache, float* out, int64_t heads, int64_t capacity, int64_t start, int64_t count,
                        int64_t features, tcx_stream_t stream) {
  using namespace tcx;
  if (heads < 0 || capacity < 0 || start < 0 || count < 0)
    return fail(TCX_INVALID_ARGUMENT, "cache load extents must be non-negative");
  if (tcx_hip_cache4_words(features) == 0)
    return fail(TCX_INVALID_ARGUMENT, "a 4-bit cache holds 32, 64 or 128 features");
  if (start > capacity || count > capacity - start)
    return fail(TCX_INVALID_ARGUMENT, "cache load slots lie past the capacity");
  if (heads == 0 || count == 0) return TCX_OK;
  if (cache == nullptr || out == nullptr) return fail(TCX_INVALID_ARGUMENT, "cache load buffers are null");
  if (!aligned16(cache) || !aligned16(out))
    return fail(TCX_INVALID_ARGUMENT, "cache load buffers must be 16-byte aligned");
  if (int rc = ready(); rc != TCX_OK) return rc;
  const dim3 grid(grid_for(count, 16, 1 << 20), static_cast<unsigned>(std::min<std::int64_t>(heads, 65535)));
  const auto s = static_cast<hipStream_t>(stream);
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, cache, out, heads, capacity, start, count); };
  if (features == 32) go(cache_load_kernel<32>);
  else if (features == 64) go(cache_load_kernel<64>);
  else go(cache_load_kernel<128>);
  return check(hipGetLastError(), "cache load launch");
}

size_t tcx_hip_cache4_attention_workspace_bytes(const tcx_hip_window_attention_desc_t* desc) {
  using namespace tcx;
  DecodeArgs a{};
  bool done = false;
  alignas(16) static float any[4];  // an aligned address; not touched
  if (decode_args(any, any, any, any, desc, true, a, done) != TCX_OK || done) return 0;
  return split_bytes(a, cache_splits(a, SIZE_MAX));
}

int tcx_hip_cache4_attention_f32(const float* q, const int32_t* key_cache, const int32_t* value_cache, float* out,
                                 const tcx_hip_window_attention_desc_t* desc, void* workspace, size_t workspace_bytes,
                                 tcx_stream_t stream) {
  using namespace tcx;
  DecodeArgs a{};
  bool done = false;
  if (int rc = decode_args(q, key_cache, value_cache, out, desc, true, a, done); rc != TCX_OK || done) return rc;
  if (!aligned16(workspace)) return fail(TCX_INVALID_ARGUMENT, "attention workspace must be 16-byte aligned");
  if (int rc = ready(); rc != TCX_OK) return rc;
  const auto s = static_cast<hipStream_t>(stream);
  place_split(a, cache_splits(a, workspace != nullptr ? workspace_bytes : 0), workspace);
  int rc = a.features == 32 ? launch_cache<32>(a, s) : a.features == 64 ? launch_cache<64>(a, s) : launch_cache<128>(a, s);
  if (rc == TCX_OK && a.splits > 1) rc = join_splits(a, s);
  return rc;
}

}  // extern "C"
