// Beam search: the choice of the best continuations over beams and vocabulary,
// and the move of the states to the chosen beams.
//
// A candidate (beam k, token v) scores score_k + (x_v - log sum exp x): within a
// beam the order is that of the logits x, so each part of a beam's row yields
// its `count` first logits, its maximum and its sum of exp(x - maximum); the
// merge then adds score_k - logsumexp, in 64 bits, to those and takes the first
// `count` of a sequence's.
//
// Both steps find the first of many in the same way. Each thread takes the largest
// of its candidates (the two largest for counts above 128); T is the least, over the
// four waves, of a wave's ceil(count / 4)-th largest of those, so that at least count
// candidates are >= T. Those, up to twice count of them where values are in no special
// order, go to a list in LDS and are put in order by counting those before each. Where
// they are too many for that (long runs of equal values, such as masked tokens) the
// first are taken one by one: by a part from its logits, by the merge from the heads
// of the parts' lists, some 2.3 us each.
//
// The parts read the logits once, and hold them in registers. Measured: 128 beams of
// 128256 logits, 65.7 MB, in 21 us with count 16 (a plain read takes 10.5), and
// 9.6 for the merge; four beams of 32000 with count 4 in 4.9 and 6.8. What is left
// above the read is the work on what was read: a block waits for its loads, then
// for the search, the list and its order, three blocks a CU. Eight beams of 128256:
// count 16 in 33 us, 64 in 110, 128 in 217, 256 in 420: a sequence's merge is one
// block's work. (A bound from the largest alone, over lists in their own order, left
// counts of 64, 128 and 256 to be taken one by one at times: 3.9, 15 and 59 ms.)

#include <algorithm>

#include "common.hpp"

namespace tcx {
namespace {

constexpr int kListed = 2048;   // candidates of a part in LDS
constexpr int kMerged = 1024;   // and of a merge
constexpr int kBeams = 64;

struct BeamArgs {
  const float* logits;
  const float* scores;
  const std::uint8_t* finished;
  float* out_scores;
  std::int32_t* out_beams;
  std::int32_t* out_tokens;
  std::int64_t batch;
  int beams, vocabulary, count, eos, parts;
  std::uint64_t* places;  // [batch * beams, parts, count]: the key, and the token inverted; 0: none
  float* sums;            // [batch * beams, parts, 2]: maximum, sum of exp
  std::int32_t* heads;    // [batch * beams, parts]: of the merge of lists that are too long to be put in order
};

// Larger keys come first; NaN above every number, +0 and -0 alike. No key is 0.
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

// T of the block from its threads' largest keys and, where a wave's rank is above
// kRanked, their second largest (or 0) too; from bit kLast on (a lower one is a bound
// as well, and spares steps of the search). One barrier; `shared` holds a word for
// each wave.
constexpr int kRanked = 32;
template <int kLast>
__device__ __forceinline__ std::uint32_t block_bound(std::uint32_t most, std::uint32_t second, int count, std::uint32_t* shared) {
  const int rank = min((count + 3) / 4, 64);
  std::uint32_t bound = 0;
  auto search = [&](auto&& reaching) {
    for (int bit = 31; bit >= kLast; --bit)
      if (reaching(bound | (1U << bit)) >= rank) bound |= 1U << bit;
  };
  if (rank <= kRanked) search([&](std::uint32_t key) { return __popcll(__ballot(most >= key)); });
  else search([&](std::uint32_t key) { return __popcll(__ballot(most >= key)) + __popcll(__ballot(second >= key)); });
  if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = bound;
  __syncthreads();
  return min(min(shared[0], shared[1]), min(shared[2], shared[3]));
}

// Whether `found` of a list are put in order by counting: that takes a thread some 35
// cycles for each pair, where taking `wanted` one by one costs some 2400 each, of a
// merge 4500 (four beams of 32000 logits, one in a hundred not masked: 245 us by
// counting alone, 16 so).
__device__ __forceinline__ bool counted(int found, int listed, int wanted) {
  return found <= listed && (found + 255) / 256 * found <= wanted * 70;
}

// How many of a list come before one of them.
template <typename F>
__device__ __forceinline__ int count_before(int listed, F&& comes_before) {
  int n = 0, j = 0;
  for (; j + 8 <= listed; j += 8) {  // eight reads of LDS at a time
#pragma unroll
    for (int u = 0; u < 8; ++u) n += comes_before(j + u);
  }
  for (; j < listed; ++j) n += comes_before(j);
  return n;
}

// One part of one beam's row, 256 kEach logits; kWide: loads of four (rows whose
// length is a multiple of 4, from an aligned address; 24.6 -> 20.5 us).
template <int kEach, bool kWide>
__global__ __launch_bounds__(256, kEach == 32 ? 3 : 4) void beam_part_kernel(BeamArgs a, std::uint32_t items) {
  constexpr int kPart = 256 * kEach;
  using Four = float __attribute__((ext_vector_type(4)));
  constexpr float kLog2e = 1.44269502F;
  __shared__ std::uint64_t listed[kListed];
  __shared__ std::uint64_t wave_place[4];
  __shared__ std::uint32_t wave_key[4];
  __shared__ float wave_top[4], wave_value[4];
  __shared__ int listed_count;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  for (std::uint32_t item = blockIdx.x; item < items; item += gridDim.x) {
    const std::uint32_t row = item / static_cast<std::uint32_t>(a.parts);
    const int part = static_cast<int>(item - row * a.parts);
    if (a.finished != nullptr && a.finished[row]) continue;  // the same for the whole block
    const int v0 = part * kPart, n = min(kPart, a.vocabulary - v0);
    const float* x = a.logits + static_cast<std::int64_t>(row) * a.vocabulary + v0;
    float value[kEach];
    auto at = [&](int e) { return kWide ? e / 4 * 1024 + 4 * t + e % 4 : e * 256 + t; };
    if constexpr (kWide) {
#pragma unroll
      for (int e = 0; e < kEach; e += 4) {
        const Four four = stream_load(reinterpret_cast<const Four*>(x + min(at(e), n - 4)));
#pragma unroll
        for (int i = 0; i < 4; ++i) value[e + i] = four[i];
      }
    } else {
#pragma unroll
      for (int e = 0; e < kEach; ++e) value[e] = stream_load(x + min(at(e), n - 1));
    }
    if (n < kPart) {  // -inf behind the end changes neither maximum nor sum
#pragma unroll
      for (int e = 0; e < kEach; ++e) value[e] = at(e) < n ? value[e] : -__builtin_inff();
    }
    // Maximum and sum as numbers; a NaN shows in the sum.
    float top = value[0];
#pragma unroll
    for (int e = 1; e < kEach; ++e) top = fmaxf(top, value[e]);
    const std::uint32_t most = at(0) < n ? logit_key(top) : 0;
    if (t == 0) listed_count = 0;
#pragma unroll
    for (int offset = 32; offset > 0; offset >>= 1) top = fmaxf(top, __shfl_xor(top, offset, kWave));
    if (lane == 0) wave_top[wave] = top;
    std::uint32_t second = 0;
    if (a.count > 4 * kRanked) {
      // (A NaN makes the largest number the second as well, and is itself above it.)
      float first = value[0], next = -__builtin_inff();
#pragma unroll
      for (int e = 1; e < kEach; ++e) {
        next = fmaxf(next, fminf(first, value[e]));
        first = fmaxf(first, value[e]);
      }
      if (at(0) < n) second = logit_key(next);
    }
    const std::uint32_t bound = block_bound<12>(most, second, a.count, wave_key);
    top = fmaxf(fmaxf(wave_top[0], wave_top[1]), fmaxf(wave_top[2], wave_top[3]));
    // Differences from the maximum, which are as good as the logits, and 0 where those
    // are equal, float32's lowest value too. (top log2 e, rounded, would be a factor of
    // the sum: 4e-5 of the scores for logits near 1000.)
    const float shift = top == -__builtin_inff() ? 0.F : top;
    // Four sums by turns: with the wave's and the block's a chain of at most kEach / 4 + 8.
    float part_sum[4] = {0.F, 0.F, 0.F, 0.F};
#pragma unroll
    for (int e = 0; e < kEach; ++e) part_sum[e % 4] += __builtin_amdgcn_exp2f((value[e] - shift) * kLog2e);
    float sum = wave_sum((part_sum[0] + part_sum[1]) + (part_sum[2] + part_sum[3]));
    // With a NaN in this thread's share, its largest number says nothing of the order.
    const bool lost = __any(!(part_sum[0] + part_sum[1] + part_sum[2] + part_sum[3] < __builtin_inff()));
    const float least = key_logit(bound == 0 ? 1U : bound);
    if (!lost && bound > 0x007fffffU) {  // above the key of -inf
#pragma unroll
      for (int e = 0; e < kEach; ++e)
        if (value[e] >= least) {
          const int place = atomicAdd(&listed_count, 1);
          if (place < kListed) listed[place] = place_of(logit_key(value[e]), v0 + at(e));
        }
    } else {
#pragma unroll
      for (int e = 0; e < kEach; ++e)
        if (at(e) < n && logit_key(value[e]) >= bound) {
          const int place = atomicAdd(&listed_count, 1);
          if (place < kListed) listed[place] = place_of(logit_key(value[e]), v0 + at(e));
        }
    }
    if (lane == 0) wave_value[wave] = sum;
    __syncthreads();
    if (t == 0) {
      sum = (wave_value[0] + wave_value[1]) + (wave_value[2] + wave_value[3]);
      a.sums[2 * static_cast<std::int64_t>(item)] = sum != sum ? sum : top;
      a.sums[2 * static_cast<std::int64_t>(item) + 1] = sum;
    }
    std::uint64_t* out = a.places + static_cast<std::int64_t>(item) * a.count;
    const int found = listed_count, wanted = min(a.count, n);
    if (counted(found, kListed, wanted)) {
      for (int i = t; i < found; i += 256) {
        const std::uint64_t mine = listed[i];
        const int rank = count_before(found, [&](int j) { return listed[j] > mine; });
        if (rank < wanted) out[rank] = mine;
      }
    } else {
      std::uint64_t last = ~std::uint64_t{0};  // a place as well: of a NaN in token 0
      for (int i = 0; i < wanted; ++i) {
        std::uint64_t best = 0;
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
          const std::uint64_t p = at(e) < n ? place_of(logit_key(value[e]), v0 + at(e)) : 0;
          if ((i == 0 || p < last) && p > best) best = p;
        }
#pragma unroll
        for (int offset = 32; offset > 0; offset >>= 1) {
          const std::uint64_t other = __shfl_xor(static_cast<unsigned long long>(best), offset, kWave);
          best = other > best ? other : best;
        }
        __syncthreads();
        if (lane == 0) wave_place[wave] = best;
        __syncthreads();
        last = max(max(wave_place[0], wave_place[1]), max(wave_place[2], wave_place[3]));
        if (t == 0) out[i] = last;
      }
    }
    for (int i = wanted + t; i < a.count; i += 256) out[i] = 0;
    __syncthreads();
  }
}

// Doubles ordered as words: NaN above every number, -0 as +0. No key is 0.
__device__ __forceinline__ std::uint64_t double_key(double x) {
  if (x != x) return ~std::uint64_t{0};
  const std::uint64_t word = static_cast<std::uint64_t>(__double_as_longlong(x == 0.0 ? 0.0 : x));
  return (word >> 63) ? ~word : word ^ (std::uint64_t{1} << 63);
}
__device__ __forceinline__ double key_double(std::uint64_t key) {
  if (key == ~std::uint64_t{0}) return __builtin_nan("");
  const std::uint64_t word = (key >> 63) ? key ^ (std::uint64_t{1} << 63) : ~key;
  return __longlong_as_double(static_cast<long long>(word));
}

// A candidate of a sequence: its score's key (0: none), then what orders equal
// scores, the lower beam, of one beam the larger logit, then the lower token.
// (Scores of different logits are equal where a beam's own score is far larger.)
struct Candidate {
  std::uint64_t key, logit;  // logit: its key under the beam, inverted
  std::uint32_t token;       // inverted
};
__device__ __forceinline__ bool before(const Candidate& a, const Candidate& b) {
  if (a.key != b.key) return a.key > b.key;
  return a.logit > b.logit || (a.logit == b.logit && a.token > b.token);
}

// The candidate that thread t of 256 takes in round h. The candidates lie in lists of
// `count`, best first: in their own order a thread would see the same ranks of every list
// where count and 256 have a factor in common, and most threads none of the first
// (counts of 128 and 256 put thousands above the bound). Turned by another
// angle each round, every thread meets all ranks.
__device__ __forceinline__ int merge_candidate(int t, int h) { return 256 * h + ((t + 37 * h) & 255); }

// A block a sequence.
__global__ __launch_bounds__(256) void beam_merge_kernel(BeamArgs a) {
  constexpr int kHeld = 8;  // candidates of a thread that stay in registers
  constexpr float kLog2e = 1.44269502F;
  __shared__ double shift[kBeams];
  __shared__ std::uint64_t listed_key[kMerged], listed_logit[kMerged];
  __shared__ std::uint32_t listed_token[kMerged];
  __shared__ std::uint32_t wave_key[4];
  __shared__ Candidate wave_best[4];
  __shared__ int listed_count;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int each = a.parts * a.count, candidates = a.beams * each;
  for (std::int64_t b = blockIdx.x; b < a.batch; b += gridDim.x) {
    auto done = [&](int beam) { return a.finished != nullptr && a.finished[b * a.beams + beam]; };
    // The first candidates' loads pass while the beams are summed. (A finished beam's
    // places are not written; what is read there is not used.)
    std::uint64_t place[kHeld];
    float score[kHeld];
#pragma unroll
    for (int h = 0; h < kHeld; ++h) {
      const int c = min(merge_candidate(t, h), candidates - 1);
      place[h] = a.places[b * candidates + c];
      score[h] = a.scores[b * a.beams + c / each];
    }
    // log sum exp of each beam: a wave each, a lane a part.
    for (int beam = wave; beam < a.beams; beam += 4) {
      if (done(beam)) continue;
      const auto* sums = reinterpret_cast<const float2*>(a.sums) + (b * a.beams + beam) * a.parts;
      const float2 mine = lane < a.parts ? sums[lane] : float2{-__builtin_inff(), 0.F};
      float top = mine.x;
      bool lost = is_nan(mine.x);
      for (int p = lane + 64; p < a.parts; p += 64) {
        lost |= is_nan(sums[p].x);
        top = fmaxf(top, sums[p].x);
      }
#pragma unroll
      for (int offset = 32; offset > 0; offset >>= 1) top = fmaxf(top, __shfl_xor(top, offset, kWave));
      // A part of nothing but -inf has no weight.
      auto weighted = [&](const float2& s) {
        return s.x == -__builtin_inff() ? 0.F : s.y * __builtin_amdgcn_exp2f((s.x - top) * kLog2e);
      };
      float sum = weighted(mine);
      for (int p = lane + 64; p < a.parts; p += 64) sum += weighted(sums[p]);
      sum = wave_sum(sum);
      // A beam of nothing but -inf leaves them as they are.
      if (__any(lost)) sum = __builtin_nanf("");
      else if (top == -__builtin_inff()) top = 0.F, sum = 1.F;
      if (lane == 0) shift[beam] = static_cast<double>(top) + log(static_cast<double>(sum));
    }
    if (t == 0) listed_count = 0;
    __syncthreads();
    auto make = [&](int c, std::uint64_t place, double score) -> Candidate {
      const int beam = c / each, at = c - beam * each;
      double value;
      std::uint32_t token, logit = 0;
      if (done(beam)) {
        // The end token at the beam's score, then the others at -inf by index; a
        // score of -inf leaves nothing but the index to go by.
        if (at >= min(a.count, a.vocabulary)) return {0, 0, 0};
        const bool plain = score == -__builtin_inf();
        token = plain ? at : at == 0 ? a.eos : at - 1 < a.eos ? at - 1 : at;
        value = plain || at > 0 ? -__builtin_inf() : score;
      } else {
        if (place == 0) return {0, 0, 0};
        token = ~static_cast<std::uint32_t>(place);
        logit = static_cast<std::uint32_t>(place >> 32);
        value = (static_cast<double>(key_logit(logit)) - shift[beam]) + score;
      }
      return {double_key(value), (static_cast<std::uint64_t>(~static_cast<std::uint32_t>(beam)) << 32) | logit, ~token};
    };
    auto candidate = [&](int c) {
      return make(c, a.places[b * candidates + c], a.scores[b * a.beams + c / each]);
    };
    Candidate held[kHeld];
    std::uint32_t most = 0, second = 0;
    auto rank = [&](const Candidate& mine) {
      const auto key = static_cast<std::uint32_t>(mine.key >> 32);
      second = max(second, min(most, key));
      most = max(most, key);
    };
    const int rounds = (candidates + 255) / 256;
#pragma unroll
    for (int h = 0; h < kHeld; ++h) {
      const int c = merge_candidate(t, h);
      held[h] = c < candidates ? make(c, place[h], score[h]) : Candidate{0, 0, 0};
      rank(held[h]);
    }
    for (int h = kHeld; h < rounds; ++h)
      if (const int c = merge_candidate(t, h); c < candidates) rank(candidate(c));
    const std::uint32_t bound = block_bound<4>(most, second, a.count, wave_key);
    auto list = [&](const Candidate& mine) {
      if (mine.key == 0 || static_cast<std::uint32_t>(mine.key >> 32) < bound) return;
      const int place = atomicAdd(&listed_count, 1);
      if (place >= kMerged) return;
      listed_key[place] = mine.key;
      listed_logit[place] = mine.logit;
      listed_token[place] = mine.token;
    };
#pragma unroll
    for (int h = 0; h < kHeld; ++h) list(held[h]);
    for (int h = kHeld; h < rounds; ++h)
      if (const int c = merge_candidate(t, h); c < candidates) list(candidate(c));
    __syncthreads();
    auto write = [&](int n, const Candidate& c) {
      a.out_scores[b * a.count + n] = static_cast<float>(key_double(c.key));
      a.out_beams[b * a.count + n] = static_cast<std::int32_t>(~static_cast<std::uint32_t>(c.logit >> 32));
      a.out_tokens[b * a.count + n] = static_cast<std::int32_t>(~c.token);
    };
    const int found = listed_count;
    if (counted(found, kMerged, a.count)) {
      for (int i = t; i < found; i += 256) {
        const std::uint64_t key = listed_key[i];
        int rank = count_before(found, [&](int j) { return listed_key[j] > key; });
        if (rank >= a.count) continue;
        const Candidate mine{key, listed_logit[i], listed_token[i]};
        // Among equal scores; most have none, and the first pass is over the keys alone.
        if (count_before(found, [&](int j) { return listed_key[j] == key; }) > 1)
          for (int j = 0; j < found; ++j) rank += listed_key[j] == key && before({key, listed_logit[j], listed_token[j]}, mine);
        if (rank < a.count) write(rank, mine);
      }
    } else {
      // The first of all lists' heads, `count` times: a thread has the best of its lists
      // at hand, and looks for it again when that has been taken.
      const int lists = a.beams * a.parts;
      std::int32_t* heads = a.heads + b * lists;
      Candidate best{0, 0, 0};
      int from = 0;
      auto offer = [&](int list, const Candidate& head) {
        if (before(head, best)) best = head, from = list;
      };
      for (int i = t; i < lists; i += 256) {
        heads[i] = 0;
        offer(i, candidate(i * a.count));
      }
      for (int n = 0; n < a.count; ++n) {
        Candidate last = best;
#pragma unroll
        for (int offset = 32; offset > 0; offset >>= 1) {
          const Candidate other{__shfl_xor(static_cast<unsigned long long>(last.key), offset, kWave),
                                __shfl_xor(static_cast<unsigned long long>(last.logit), offset, kWave),
                                static_cast<std::uint32_t>(__shfl_xor(static_cast<int>(last.token), offset, kWave))};
          if (before(other, last)) last = other;
        }
        __syncthreads();
        if (lane == 0) wave_best[wave] = last;
        __syncthreads();
        for (int w = 0; w < 4; ++w)
          if (before(wave_best[w], last)) last = wave_best[w];
        if (t == 0) write(n, last);
        if (best.key != last.key || best.logit != last.logit || best.token != last.token) continue;
        ++heads[from];
        best = {0, 0, 0};
        for (int i = t; i < lists; i += 256)
          if (const int at = heads[i]; at < a.count) offer(i, candidate(i * a.count + at));
      }
    }
    __syncthreads();
  }
}

constexpr int kReorderTensors = 8;
// Units of a row that a block copies: 1024 of 16 bytes, 2048 of others (42 MB in units
// of 16 bytes: 8.4 us, with 2048 9.0; 17 MB in units of 4: 6.5, with 1024 7.9, with
// 4096 8.2).
constexpr std::int64_t reorder_chunk(int width) { return width == 16 ? 1024 : 2048; }

struct ReorderArgs {
  const void* in[kReorderTensors];
  void* out[kReorderTensors];
  std::int64_t units[kReorderTensors];   // of a row
  std::int64_t chunks[kReorderTensors];  // of a row
  std::int64_t first[kReorderTensors];   // item of the tensor's first chunk
  int width[kReorderTensors];            // bytes of a unit: 16, 4 or 1
  int tensors;
  const std::int32_t* index;
  std::int64_t items;
  int beams, count;
  std::int32_t* flag;
};

template <typename T>
__device__ __forceinline__ void copy_units(const void* in, void* out, std::int64_t from, std::int64_t to,
                                           std::int64_t n, bool zero) {
  const T* src = static_cast<const T*>(in) + from;
  T* dst = static_cast<T*>(out) + to;
  constexpr int kHeld = sizeof(T) == 16 ? 1 : 4;
  for (std::int64_t first = threadIdx.x; first < n; first += 256 * kHeld) {
    T held[kHeld];  // narrow loads pass together
#pragma unroll
    for (int u = 0; u < kHeld; ++u) held[u] = src[min<std::int64_t>(first + 256 * u, n - 1)];
#pragma unroll
    for (int u = 0; u < kHeld; ++u)
      if (first + 256 * u < n) dst[first + 256 * u] = zero ? T{} : held[u];
  }
}

__global__ __launch_bounds__(256) void beam_reorder_kernel(ReorderArgs a) {
  for (std::int64_t item = blockIdx.x; item < a.items; item += gridDim.x) {
    int i = 0;
    while (i + 1 < a.tensors && item >= a.first[i + 1]) ++i;
    // Rows and, up to 2^42 units of a row, chunks have 32 bits.
    const std::int64_t local = item - a.first[i];
    std::int64_t row, chunk;
    if ((local | a.chunks[i]) >> 32 == 0) {
      const auto small = static_cast<std::uint32_t>(local), by = static_cast<std::uint32_t>(a.chunks[i]);
      row = __builtin_amdgcn_readfirstlane(small / by);
      chunk = small - static_cast<std::uint32_t>(row) * by;
    } else {
      row = local / a.chunks[i];
      chunk = local % a.chunks[i];
    }
    const std::int32_t beam = a.index[row];
    const bool bad = beam < 0 || beam >= a.beams;
    if (bad && a.flag != nullptr) __hip_atomic_store(a.flag, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
    const std::int64_t source = static_cast<std::int64_t>(static_cast<std::uint32_t>(row) / a.count) * a.beams + (bad ? 0 : beam);
    const std::int64_t at = chunk * reorder_chunk(a.width[i]);
    const std::int64_t n = min(reorder_chunk(a.width[i]), a.units[i] - at);
    const std::int64_t from = source * a.units[i] + at, to = row * a.units[i] + at;
    if (a.width[i] == 16) copy_units<int4_t>(a.in[i], a.out[i], from, to, n, bad);
    else if (a.width[i] == 4) copy_units<std::uint32_t>(a.in[i], a.out[i], from, to, n, bad);
    else copy_units<std::uint8_t>(a.in[i], a.out[i], from, to, n, bad);
  }
}

struct BeamLayout {
  int each;  // logits of a thread
  std::int64_t parts;
  std::size_t sums, heads, bytes;
};

// Parts of 8192 logits, or of 2048 where those would not give every CU a block. (128
// beams of 128256 logits: parts of 4096 20.0 us and twice the candidates for the
// merge, 15.8 us, against 20.8 and 9.6. Four of 32000: parts of 8192 leave all but 16
// CUs without work.)
BeamLayout beam_layout(std::int64_t batch, std::int64_t beams, std::int64_t vocabulary, std::int64_t count) {
  BeamLayout l{};
  l.each = batch * beams * ((vocabulary + 8191) / 8192) < 256 ? 8 : 32;
  l.parts = (vocabulary + 256 * l.each - 1) / (256 * l.each);
  const auto lists = static_cast<std::size_t>(batch * beams * l.parts);
  l.sums = (lists * count * sizeof(std::uint64_t) + 15) / 16 * 16;
  l.heads = l.sums + lists * 2 * sizeof(float);
  l.bytes = l.heads + lists * sizeof(std::int32_t);
  return l;
}

// Parts and candidates are counted in 31 bits.
bool beam_sizes(std::int64_t batch, std::int64_t beams, std::int64_t vocabulary, std::int64_t count) {
  constexpr std::int64_t kMost = std::int64_t{1} << 31;
  if (batch < 0 || beams < 1 || beams > kBeams || vocabulary < 1 || count < 1 || count > TCX_HIP_BEAM_MAX_COUNT) return false;
  if (vocabulary >= kMost / beams || count > beams * vocabulary) return false;
  const std::int64_t lists = beams * ((vocabulary + 2047) / 2048);
  return batch < kMost / lists;
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
  a.places = static_cast<std::uint64_t*>(workspace);
  a.sums = reinterpret_cast<float*>(static_cast<char*>(workspace) + layout.sums);
  a.heads = reinterpret_cast<std::int32_t*>(static_cast<char*>(workspace) + layout.heads);
  const auto s = static_cast<hipStream_t>(stream);
  const auto items = static_cast<std::uint32_t>(batch * beams * layout.parts);
  const dim3 grid(grid_for(items, 1, kStrideBlocks));
  const bool wide = vocabulary % 4 == 0 && reinterpret_cast<std::uintptr_t>(logits) % 16 == 0;
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, a, items); };
  if (layout.each == 8) wide ? go(beam_part_kernel<8, true>) : go(beam_part_kernel<8, false>);
  else wide ? go(beam_part_kernel<32, true>) : go(beam_part_kernel<32, false>);
  if (int rc = check(hipGetLastError(), "beam selection launch"); rc != TCX_OK) return rc;
  hipLaunchKernelGGL(beam_merge_kernel, dim3(grid_for(batch, 1, kStrideBlocks)), dim3(256), 0, s, a);
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
      a.chunks[t] = (a.units[t] + reorder_chunk(a.width[t]) - 1) / reorder_chunk(a.width[t]);
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
