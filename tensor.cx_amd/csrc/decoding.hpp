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
  return j <= p && (window == 0 || j > p - window || j < sinks);
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

// Checks desc and fills `a`; true with *rc = TCX_OK in `done` when there is
// nothing to compute. `cache`: k and v are 4-bit caches.
int decode_args(const float* q, const void* k, const void* v, float* out, const tcx_hip_window_attention_desc_t* desc,
                bool cache, DecodeArgs& a, bool& done);
// Bytes of the states of `splits` splits.
std::size_t split_bytes(const DecodeArgs& a, int splits);
// Places part and part_ml in the workspace.
void place_split(DecodeArgs& a, int splits, void* workspace);
// How many splits a call of `blocks` blocks takes, of at least split_keys keys
// each and with no more bytes than the workspace has.
int plan_splits(const DecodeArgs& a, std::int64_t blocks, int split_keys, std::size_t workspace_bytes);
// Joins the splits into out.
int join_splits(const DecodeArgs& a, hipStream_t s);

// The keys of sequence b, its length checked.
__device__ __forceinline__ int checked_length(const DecodeArgs& a, int b) {
  if (a.lengths == nullptr) return a.cols;
  const int n = a.lengths[b];
  if (n >= 0 && n <= a.cols) return n;
  if (a.flag != nullptr) __hip_atomic_store(a.flag, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
  return n < 0 ? 0 : a.cols;
}

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
