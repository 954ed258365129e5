// What the attentions of a decoding loop share: which keys a query sees, the
// checked arguments, and the join of key splits.
#pragma once

#include <cstddef>
#include <cstdint>

#include "common.hpp"

namespace tcx {

// The keys that queries [i0, i1] of a sequence of n keys see between them: the
// sinks [0, sinks) and [first, end), counted through as count() keys.
struct SeenKeys {
  int sinks, first, end;
  __host__ __device__ int count() const { return sinks + end - first; }
  // The key at place u of them.
  __host__ __device__ int key(int u) const { return u < sinks ? u : u - sinks + first; }
};

// All of them are below 2^30, so that nothing here overflows.
__host__ __device__ inline SeenKeys seen_keys(int n, int rows, int i0, int i1, int window, int sinks) {
  const int p0 = n - rows + i0, p1 = n - rows + i1;
  SeenKeys s;
  s.end = p1 < 0 ? 0 : p1 + 1;
  s.first = window > 0 && p0 >= window ? p0 - window + 1 : 0;
  if (s.first > s.end) s.first = s.end;
  s.sinks = sinks < s.first ? sinks : s.first;
  return s;
}

// Whether the query at key p sees key j.
__device__ __forceinline__ bool sees(int p, int j, int window, int sinks) {
  return (j <= p) & ((window == 0) | (j > p - window) | (j < sinks));
}

// A call with its arguments checked: strides filled in, window and sinks cut to cols.
struct DecodeArgs {
  const float* q;
  const void* k;  // float, or rows of a 4-bit cache
  const void* v;
  float* out;
  const std::int32_t* lengths;
  std::int32_t* flag;
  int batch, heads, kv_heads, share;  // share: query heads that read one head
  int rows, cols, features;
  int window, sinks;
  float scale;
  std::int64_t q_stride[3], k_stride[3], v_stride[3], out_stride[3];
  // Key splits: split s of `splits` takes its share of the keys that its rows
  // see; its state goes to part [splits][batch * kv_heads][rows * share]
  // [features] and part_ml [..][2] (the maximum in units of log2, and the sum).
  int splits;
  float* part;
  float* part_ml;
};

inline bool aligned16(const void* p) { return (reinterpret_cast<std::uintptr_t>(p) & 15U) == 0; }

// Checks desc and fills `a`; true with *rc = TCX_OK in `done` when there is
// nothing to compute. `cache`: k and v are 4-bit caches.
int decode_args(const float* q, const void* k, const void* v, float* out, const tcx_hip_window_attention_desc_t* desc,
                bool cache, DecodeArgs& a, bool& done);
// Bytes of the states of `splits` splits.
std::size_t split_bytes(const DecodeArgs& a, int splits);
// Places part and part_ml in the workspace.
void place_split(DecodeArgs& a, int splits, void* workspace);
// How many splits a call of `blocks` blocks takes to come to `wanted` of them, with
// some split_keys keys and more in each and no more bytes than the workspace has; one
// where its rows see fewer than least_keys, which would not pay for the join.
int plan_splits(const DecodeArgs& a, std::int64_t blocks, int wanted, int split_keys, int least_keys, std::size_t workspace_bytes);
// The blocks' work items of a call of `row_tiles` row tiles a head, as a 32-bit
// count; TCX_INVALID_ARGUMENT where there are more.
int count_items(const DecodeArgs& a, std::int64_t row_tiles, std::uint32_t& items);
// Joins the splits into out.
int join_splits(const DecodeArgs& a, hipStream_t s);

// The keys of sequence b (the same for the whole wave), its length checked; in a
// scalar register, and what follows from it too.
__device__ __forceinline__ int checked_length(const DecodeArgs& a, int b) {
  if (a.lengths == nullptr) return a.cols;
  const int n = __builtin_amdgcn_readfirstlane(a.lengths[b]);
  if (n >= 0 && n <= a.cols) return n;
  if (a.flag != nullptr) __hip_atomic_store(a.flag, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
  return n < 0 ? 0 : a.cols;
}

// What a block does: a split of the keys of row tile `tile` of key head `head` of
// all. Divisions run on vector registers even where their operands are the same
// for the whole wave; the results go back to scalar ones, and with them whatever
// is computed from them (buffer resources most of all, which take a loop over
// the lanes otherwise).
struct BlockWork {
  int split, tile, head, b, kv;
};
__device__ __forceinline__ BlockWork block_work(const DecodeArgs& a, std::uint32_t item, int row_tiles) {
  const std::uint32_t rest = item / static_cast<std::uint32_t>(a.splits), head = rest / static_cast<std::uint32_t>(row_tiles);
  BlockWork w;
  w.split = __builtin_amdgcn_readfirstlane(static_cast<int>(item - rest * a.splits));
  w.tile = __builtin_amdgcn_readfirstlane(static_cast<int>(rest - head * row_tiles));
  w.head = __builtin_amdgcn_readfirstlane(static_cast<int>(head));
  w.b = __builtin_amdgcn_readfirstlane(w.head / a.kv_heads);
  w.kv = w.head - w.b * a.kv_heads;
  return w;
}
// The first of the `count` keys (or tiles of them) that falls to split s: shares that
// differ by one quantum at most, the keys that a block takes in one round, so that no
// round is left to a few keys (8 sequences of 1028 keys, 32 heads on 8 of 128
// features: 18.6 -> 17.4 us; the 4-bit cache of 16 sequences of 4096 to 8192 tokens:
// 38.1 -> 37.6). A fixed number of keys to each split, which leaves the last ones of
// short sequences empty, was slower: 44 us against 38 for the latter.
template <int kQuantum>
__device__ __forceinline__ int split_start(const DecodeArgs& a, int count, int s) {
  if (a.splits == 1) return s == 0 ? 0 : count;
  const int rounds = (count + kQuantum - 1) / kQuantum, each = __builtin_amdgcn_readfirstlane(rounds / a.splits);
  return min((each * s + min(s, rounds - each * a.splits)) * kQuantum, count);
}
// The query of row r.
__device__ __forceinline__ int row_query(const DecodeArgs& a, int r) { return __builtin_amdgcn_readfirstlane(r / a.share); }

// Row r of a head's rows: query r / share of query head kv * share + r % share,
// so that neighbouring rows see the same keys.
struct RowPlace {
  int query, head;
};
__device__ __forceinline__ RowPlace row_place(const DecodeArgs& a, int kv, int r) {
  const int query = r / a.share;
  return {query, kv * a.share + (r - query * a.share)};
}

// Sum over the sixteen lanes of a group, in all of them.
__device__ __forceinline__ float lanes16_sum(float x) {
  auto add = [&]<int kControl>() {
    x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), kControl, 0xf, 0xf, true));
  };
  add.template operator()<0xb1>();   // lane ^ 1
  add.template operator()<0x4e>();   // lane ^ 2
  add.template operator()<0x141>();  // mirror in eight lanes
  add.template operator()<0x140>();  // mirror in sixteen
  return x;
}

}  // namespace tcx
