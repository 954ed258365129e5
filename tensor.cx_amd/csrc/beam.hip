// Beam search: the choice of the best continuations over beams and vocabulary,
// and the move of the states to the chosen beams.
//
// A candidate (beam k, token v) scores score_k + (x_v - log sum exp x): within a
// beam the order is that of the logits x, so each part of a beam's row yields
// its `count` first logits, its maximum and its sum of exp(x - maximum); the
// merge then adds score_k - logsumexp, in 64 bits, and takes the best of the
// heads of those sorted lists, `count` times.

#include <algorithm>

#include "common.hpp"

namespace tcx {
namespace {

constexpr int kPart = 8192;        // logits of a part: 32 a thread, in registers
constexpr int kEach = kPart / 256;
constexpr int kListed = 2048;      // candidates of a part in LDS

struct BeamArgs {
  const float* logits;
  const float* scores;
  const std::uint8_t* finished;
  float* out_scores;
  std::int32_t* out_beams;
  std::int32_t* out_tokens;
  std::int64_t batch;
  int beams, vocabulary, count, eos, parts;
  std::uint64_t* places;  // [batch * beams, parts, count]: the key, and the token inverted
  float* sums;            // [batch * beams, parts, 2]: maximum, sum of exp
};

// Larger keys come first; NaN above every number, +0 and -0 alike.
__device__ __forceinline__ std::uint32_t logit_key(float x) {
  const std::uint32_t word = __float_as_uint(x);
  return word_nan(word, true) ? 0xffffffffU : order_key(word);
}
__device__ __forceinline__ float key_logit(std::uint32_t key) {
  if (key == 0xffffffffU) return __builtin_nanf("");
  return __uint_as_float((key & 0x80000000U) ? key ^ 0x80000000U : ~key);
}
__device__ __forceinline__ std::uint64_t place_of(std::uint32_t key, std::uint32_t token) {
  return (static_cast<std::uint64_t>(key) << 32) | static_cast<std::uint32_t>(~token);
}

__device__ __forceinline__ std::uint64_t wave_most(std::uint64_t v) {
#pragma unroll
  for (int offset = 32; offset > 0; offset >>= 1) {
    const std::uint64_t w = __shfl_xor(static_cast<unsigned long long>(v), offset, kWave);
    v = w > v ? w : v;
  }
  return v;
}

// One part of one beam's row. The first `count` keys: a lower bound T of the
// count-th key is the least, over the four waves, of a wave's ceil(count / 4)-th
// largest thread maximum, since at least count keys are >= T; the keys >= T, a
// few times count of them, are listed in LDS and put in order by counting those
// before each. Where they are more than the list holds (long runs of equal
// logits), the first are taken one by one.
__global__ __launch_bounds__(256) void beam_part_kernel(BeamArgs a, std::int64_t items) {
  __shared__ std::uint64_t listed[kListed];
  __shared__ std::uint64_t wave_place[4];
  __shared__ std::uint32_t wave_key[4];
  __shared__ float wave_value[4];
  __shared__ int listed_count;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  for (std::int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const std::int64_t row = item / a.parts;
    const int part = static_cast<int>(item % a.parts);
    if (a.finished != nullptr && a.finished[row]) continue;  // the same for the whole block
    const int v0 = part * kPart, n = min(kPart, a.vocabulary - v0);
    const float* x = a.logits + row * a.vocabulary + v0;
    float value[kEach];
    std::uint32_t most = 0;
#pragma unroll
    for (int e = 0; e < kEach; ++e) value[e] = e * 256 + t < n ? x[e * 256 + t] : 0.F;
#pragma unroll
    for (int e = 0; e < kEach; ++e)
      if (e * 256 + t < n) most = max(most, logit_key(value[e]));

    // The part's maximum and its sum of exponentials.
    std::uint32_t top_key = most;
#pragma unroll
    for (int offset = 32; offset > 0; offset >>= 1)
      top_key = max(top_key, static_cast<std::uint32_t>(__shfl_xor(static_cast<int>(top_key), offset, kWave)));
    // The wave's ceil(count / 4)-th largest thread maximum, bit by bit.
    const int rank = min((a.count + 3) / 4, 64);
    std::uint32_t bound = 0;
    for (int bit = 31; bit >= 0; --bit) {
      const std::uint32_t trial = bound | (1U << bit);
      if (__popcll(__ballot(most >= trial)) >= rank) bound = trial;
    }
    if (lane == 0) {
      wave_key[wave] = bound;
      wave_place[wave] = top_key;
    }
    if (t == 0) listed_count = 0;
    __syncthreads();
    bound = min(min(wave_key[0], wave_key[1]), min(wave_key[2], wave_key[3]));
    top_key = static_cast<std::uint32_t>(max(max(wave_place[0], wave_place[1]), max(wave_place[2], wave_place[3])));
    const float top = key_logit(top_key), at = top == -__builtin_inff() ? 0.F : top;
    float sum = 0.F;
#pragma unroll
    for (int e = 0; e < kEach; ++e)
      if (e * 256 + t < n) {
        sum += exp_softmax(value[e] - at);
        if (logit_key(value[e]) >= bound) {
          const int place = atomicAdd(&listed_count, 1);
          if (place < kListed) listed[place] = place_of(logit_key(value[e]), v0 + e * 256 + t);
        }
      }
    sum = wave_sum(sum);
    if (lane == 0) wave_value[wave] = sum;
    __syncthreads();
    if (t == 0) {
      a.sums[2 * item] = top;
      a.sums[2 * item + 1] = (wave_value[0] + wave_value[1]) + (wave_value[2] + wave_value[3]);
    }
    std::uint64_t* out = a.places + item * a.count;
    const int found = listed_count, wanted = min(a.count, n);
    if (found <= kListed) {
      for (int i = t; i < found; i += 256) {
        const std::uint64_t mine = listed[i];
        int before = 0;
        for (int j = 0; j < found; ++j) before += listed[j] > mine;
        if (before < wanted) out[before] = mine;
      }
    } else {
      std::uint64_t last = ~std::uint64_t{0};
      for (int i = 0; i < wanted; ++i) {
        std::uint64_t best = 0;
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
          const std::uint64_t p = e * 256 + t < n ? place_of(logit_key(value[e]), v0 + e * 256 + t) : 0;
          if (p < last && p > best) best = p;
        }
        best = wave_most(best);
        __syncthreads();
        if (lane == 0) wave_place[wave] = best;
        __syncthreads();
        last = max(max(wave_place[0], wave_place[1]), max(wave_place[2], wave_place[3]));
        if (t == 0) out[i] = last;
      }
    }
    for (int i = wanted + t; i < a.count; i += 256) out[i] = 0;  // no candidate: below every key
    __syncthreads();
  }
}

// Doubles ordered as words: NaN above every number, -0 as +0.
__device__ __forceinline__ std::uint64_t double_key(double x) {
  if (x != x) return ~std::uint64_t{0};
  if (x == 0.0) x = 0.0;
  const std::uint64_t word = static_cast<std::uint64_t>(__double_as_longlong(x == 0.0 ? 0.0 : x));
  return (word >> 63) ? ~word : word ^ (std::uint64_t{1} << 63);
}

// A wave a sequence: lane i walks the lists i, i + 64, ... (a beam's part each)
// and offers the best of their heads.

struct Head {
  std::uint64_t key;    // double_key of the score; 0: none
  std::uint32_t order;  // the flat index inverted
  int list;
};

__global__ __launch_bounds__(64) void beam_merge_kernel(BeamArgs a, std::uint16_t* __restrict__ positions) {
  __shared__ double shift[64];
  const int lane = threadIdx.x;
  const int lists = a.beams * a.parts;
  for (std::int64_t b = blockIdx.x; b < a.batch; b += gridDim.x) {
    std::uint16_t* position = positions + b * lists;
    for (int l = lane; l < lists; l += 64) position[l] = 0;
    // A list's head: its score and its place in the order.
    auto shift_of = [&](int beam) -> double {
      const std::int64_t row = b * a.beams + beam;
      float top = -__builtin_inff();
      for (int p = 0; p < a.parts; ++p) {
        const float m = a.sums[2 * (row * a.parts + p)];
        top = is_nan(m) || is_nan(top) ? __builtin_nanf("") : fmaxf(top, m);
      }
      if (top == -__builtin_inff()) return 0.0;  // every candidate is -inf as it is
      double sum = 0.0;
      for (int p = 0; p < a.parts; ++p) {
        const float m = a.sums[2 * (row * a.parts + p)];
        if (m == -__builtin_inff()) continue;
        sum += static_cast<double>(a.sums[2 * (row * a.parts + p) + 1]) * exp(static_cast<double>(m) - top);
      }
      return static_cast<double>(top) + log(sum);
    };
    auto head = [&](int list, int at, double lse) -> Head {
      Head h{0, 0, list};
      if (at >= a.count) return h;
      const int beam = list / a.parts;
      const std::int64_t row = b * a.beams + beam;
      const double score = a.scores[row];
      double value;
      std::uint32_t token;
      if (a.finished != nullptr && a.finished[row]) {
        // The end token at the beam's score, then the others at -inf by index;
        // a score of -inf leaves nothing but the index to go by.
        if (list % a.parts != 0 || at >= a.vocabulary) return h;
        const bool plain = score == -__builtin_inf();
        token = plain ? at : at == 0 ? a.eos : at - 1 < a.eos ? at - 1 : at;
        value = plain || at > 0 ? -__builtin_inf() : score;
      } else {
        const std::uint64_t place = a.places[(row * a.parts + list % a.parts) * a.count + at];
        if (place == 0) return h;
        token = ~static_cast<std::uint32_t>(place);
        value = (static_cast<double>(key_logit(static_cast<std::uint32_t>(place >> 32))) - lse) + score;
      }
      h.key = double_key(value);
      if (h.key == 0) h.key = 1;
      h.order = ~(static_cast<std::uint32_t>(beam) * static_cast<std::uint32_t>(a.vocabulary) + token);
      return h;
    };
    __syncthreads();
    for (int beam = lane; beam < a.beams; beam += 64)
      if (!(a.finished != nullptr && a.finished[b * a.beams + beam])) shift[beam & 63] = shift_of(beam);
    __syncthreads();
    for (int n = 0; n < a.count; ++n) {
      Head best{0, 0, 0};
      for (int l = lane; l < lists; l += 64) {
        const Head h = head(l, position[l], shift[l / a.parts]);
        if (h.key > best.key || (h.key == best.key && h.order > best.order)) best = h;
      }
      Head win = best;
#pragma unroll
      for (int offset = 32; offset > 0; offset >>= 1) {
        const std::uint64_t key = __shfl_xor(static_cast<unsigned long long>(win.key), offset, kWave);
        const std::uint32_t order = __shfl_xor(static_cast<int>(win.order), offset, kWave);
        const int list = __shfl_xor(win.list, offset, kWave);
        if (key > win.key || (key == win.key && order > win.order)) win = {key, order, list};
      }
      if (lane == (win.list & 63) && win.key != 0) {
        position[win.list] += 1;
        const std::uint32_t flat = ~win.order;
        const std::uint64_t word =
            (win.key >> 63) ? win.key ^ (std::uint64_t{1} << 63) : ~win.key;
        const double value = win.key == ~std::uint64_t{0} ? static_cast<double>(__builtin_nanf(""))
                                                          : __longlong_as_double(static_cast<long long>(word));
        a.out_scores[b * a.count + n] = static_cast<float>(value);
        a.out_beams[b * a.count + n] = static_cast<std::int32_t>(flat / static_cast<std::uint32_t>(a.vocabulary));
        a.out_tokens[b * a.count + n] = static_cast<std::int32_t>(flat % static_cast<std::uint32_t>(a.vocabulary));
      }
    }
    __syncthreads();
  }
}

constexpr int kReorderTensors = 8;
constexpr std::int64_t kReorderChunk = 1024;  // units of a row that a block copies

struct ReorderArgs {
  const void* in[kReorderTensors];
  void* out[kReorderTensors];
  std::int64_t units[kReorderTensors];   // of a row
  std::int64_t chunks[kReorderTensors];  // of a row
  std::int64_t first[kReorderTensors];   // item of the tensor's first chunk
  int width[kReorderTensors];            // bytes of a unit: 16, 4 or 1
  int tensors;
  const std::int32_t* index;
  std::int64_t items, rows;
  int beams, count;
  std::int32_t* flag;
};

template <typename T>
__device__ __forceinline__ void copy_units(const void* in, void* out, std::int64_t from, std::int64_t to,
                                           std::int64_t n, bool zero) {
  const T* src = static_cast<const T*>(in) + from;
  T* dst = static_cast<T*>(out) + to;
  for (std::int64_t i = threadIdx.x; i < n; i += 256) dst[i] = zero ? T{} : src[i];
}

__global__ __launch_bounds__(256) void beam_reorder_kernel(ReorderArgs a) {
  for (std::int64_t item = blockIdx.x; item < a.items; item += gridDim.x) {
    int i = 0;
    while (i + 1 < a.tensors && item >= a.first[i + 1]) ++i;
    const std::int64_t local = item - a.first[i], row = local / a.chunks[i], chunk = local % a.chunks[i];
    const std::int32_t beam = a.index[row];
    const bool bad = beam < 0 || beam >= a.beams;
    if (bad && a.flag != nullptr) __hip_atomic_store(a.flag, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
    const std::int64_t source = row / a.count * a.beams + (bad ? 0 : beam), at = chunk * kReorderChunk;
    const std::int64_t n = min(kReorderChunk, a.units[i] - at);
    const std::int64_t from = source * a.units[i] + at, to = row * a.units[i] + at;
    if (a.width[i] == 16) copy_units<int4_t>(a.in[i], a.out[i], from, to, n, bad);
    else if (a.width[i] == 4) copy_units<std::uint32_t>(a.in[i], a.out[i], from, to, n, bad);
    else copy_units<std::uint8_t>(a.in[i], a.out[i], from, to, n, bad);
  }
}

struct BeamLayout {
  std::int64_t parts;
  std::size_t places, sums, positions, bytes;
};

BeamLayout beam_layout(std::int64_t batch, std::int64_t beams, std::int64_t vocabulary, std::int64_t count) {
  BeamLayout l{};
  l.parts = (vocabulary + kPart - 1) / kPart;
  const auto lists = static_cast<std::size_t>(batch * beams * l.parts);
  const auto up = [](std::size_t v) { return (v + 15) / 16 * 16; };
  l.places = 0;
  l.sums = up(lists * count * sizeof(std::uint64_t));
  l.positions = l.sums + up(lists * 2 * sizeof(float));
  l.bytes = l.positions + up(lists * sizeof(std::uint16_t));
  return l;
}

bool beam_sizes(std::int64_t batch, std::int64_t beams, std::int64_t vocabulary, std::int64_t count) {
  constexpr std::int64_t kMost = std::int64_t{1} << 31;
  if (batch < 0 || beams < 1 || beams > 64 || vocabulary < 1 || count < 1 || count > TCX_HIP_BEAM_MAX_COUNT) return false;
  if (vocabulary >= kMost / beams || count > beams * vocabulary) return false;
  return batch < kMost / beams;
}

}  // namespace
}  // namespace tcx

extern "C" {

size_t tcx_hip_beam_select_workspace_bytes(int64_t batch, int64_t beams, int64_t vocabulary, int64_t count) {
  using namespace tcx;
  return beam_sizes(batch, beams, vocabulary, count) ? beam_layout(batch, beams, vocabulary, count).bytes : 0;
}

int tcx_hip_beam_select_f32(const float* logits, const float* scores, const uint8_t* finished, int32_t eos,
                            float* out_scores, int32_t* out_beams, int32_t* out_tokens, int64_t batch, int64_t beams,
                            int64_t vocabulary, int64_t count, void* workspace, size_t workspace_bytes,
                            tcx_stream_t stream) {
  using namespace tcx;
  if (!beam_sizes(batch, beams, vocabulary, count))
    return fail(TCX_INVALID_ARGUMENT,
                "beam selection takes 1 to 64 beams, a vocabulary with beams * vocabulary below 2^31 and a count of 1 to "
                "256, at most beams * vocabulary");
  if (finished != nullptr && (eos < 0 || eos >= vocabulary))
    return fail(TCX_INVALID_ARGUMENT, "beam selection's end token is outside the vocabulary");
  if (batch == 0) return TCX_OK;
  if (logits == nullptr || scores == nullptr || out_scores == nullptr || out_beams == nullptr || out_tokens == nullptr)
    return fail(TCX_INVALID_ARGUMENT, "beam selection buffers are null");
  const BeamLayout layout = beam_layout(batch, beams, vocabulary, count);
  if (workspace == nullptr || workspace_bytes < layout.bytes)
    return fail(TCX_INVALID_ARGUMENT, "beam selection workspace is too small");
  if (reinterpret_cast<std::uintptr_t>(workspace) & 15U)
    return fail(TCX_INVALID_ARGUMENT, "beam selection workspace must be 16-byte aligned");
  if (int rc = ready(); rc != TCX_OK) return rc;
  BeamArgs a{};
  a.logits = logits;
  a.scores = scores;
  a.finished = finished;
  a.out_scores = out_scores;
  a.out_beams = out_beams;
  a.out_tokens = out_tokens;
  a.batch = batch;
  a.beams = static_cast<int>(beams);
  a.vocabulary = static_cast<int>(vocabulary);
  a.count = static_cast<int>(count);
  a.eos = eos;
  a.parts = static_cast<int>(layout.parts);
  auto* base = static_cast<char*>(workspace);
  a.places = reinterpret_cast<std::uint64_t*>(base + layout.places);
  a.sums = reinterpret_cast<float*>(base + layout.sums);
  auto* positions = reinterpret_cast<std::uint16_t*>(base + layout.positions);
  const auto s = static_cast<hipStream_t>(stream);
  const std::int64_t items = batch * beams * layout.parts;
  hipLaunchKernelGGL(beam_part_kernel, dim3(grid_for(items, 1, kStrideBlocks)), dim3(256), 0, s, a, items);
  if (int rc = check(hipGetLastError(), "beam selection launch"); rc != TCX_OK) return rc;
  hipLaunchKernelGGL(beam_merge_kernel, dim3(grid_for(batch, 1, kStrideBlocks)), dim3(64), 0, s, a, positions);
  return check(hipGetLastError(), "beam merge launch");
}

int tcx_hip_beam_reorder(const void* const* in, void* const* out, const int64_t* row_bytes, int32_t tensors,
                         const int32_t* index, int64_t batch, int64_t beams, int64_t count, int32_t* flag,
                         tcx_stream_t stream) {
  using namespace tcx;
  if (tensors < 0 || batch < 0 || beams < 0 || count < 0)
    return fail(TCX_INVALID_ARGUMENT, "beam reorder extents must be non-negative");
  constexpr std::int64_t kMost = std::int64_t{1} << 31;
  if (beams >= kMost || count >= kMost || (beams > 0 && batch >= kMost / beams) || (count > 0 && batch >= kMost / count))
    return fail(TCX_INVALID_ARGUMENT, "beam reorder sizes must be below 2^31");
  if (tensors > 0 && (in == nullptr || out == nullptr || row_bytes == nullptr))
    return fail(TCX_INVALID_ARGUMENT, "beam reorder lists are null");
  const std::int64_t rows = batch * count;
  if (tensors == 0 || rows == 0) return TCX_OK;
  if (beams == 0) return fail(TCX_INVALID_ARGUMENT, "beam reorder needs beams to choose from");
  if (index == nullptr) return fail(TCX_INVALID_ARGUMENT, "beam reorder index is null");
  for (int i = 0; i < tensors; ++i) {
    if (row_bytes[i] < 0) return fail(TCX_INVALID_ARGUMENT, "beam reorder extents must be non-negative");
    if (row_bytes[i] > 0 && (in[i] == nullptr || out[i] == nullptr))
      return fail(TCX_INVALID_ARGUMENT, "beam reorder buffers are null");
  }
  if (int rc = ready(); rc != TCX_OK) return rc;
  const auto s = static_cast<hipStream_t>(stream);
  for (int from = 0; from < tensors; from += kReorderTensors) {
    ReorderArgs a{};
    a.index = index;
    a.rows = rows;
    a.beams = static_cast<int>(beams);
    a.count = static_cast<int>(count);
    a.flag = flag;
    for (int i = from; i < std::min(tensors, from + kReorderTensors); ++i) {
      if (row_bytes[i] == 0) continue;
      const std::uintptr_t mix = reinterpret_cast<std::uintptr_t>(in[i]) | reinterpret_cast<std::uintptr_t>(out[i]) |
                                 static_cast<std::uintptr_t>(row_bytes[i]);
      const int t = a.tensors++;
      a.in[t] = in[i];
      a.out[t] = out[i];
      a.width[t] = (mix & 15U) == 0 ? 16 : (mix & 3U) == 0 ? 4 : 1;
      a.units[t] = row_bytes[i] / a.width[t];
      a.chunks[t] = (a.units[t] + kReorderChunk - 1) / kReorderChunk;
      a.first[t] = a.items;
      a.items += rows * a.chunks[t];
    }
    if (a.tensors == 0) continue;
    hipLaunchKernelGGL(beam_reorder_kernel, dim3(grid_for(a.items, 1, kStrideBlocks)), dim3(256), 0, s, a);
    if (int rc = check(hipGetLastError(), "beam reorder launch"); rc != TCX_OK) return rc;
  }
  return TCX_OK;
}

}  // extern "C"
