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
  int tiles_m, tiles_n, whole;  // `whole`: how many of the tiles go to one block each
  FastDiv by_group;  // work items in eight tile rows
  // Sums over shares of the features, one to a row of blocks: share s has `each` blocks
  // (or units of four) and one more if s < extra, and its sums go to parts [s][m][n].
  float* parts;  // null: one share, whose results go to out
  int each, extra;
  // Of a gated product in one launch: w has `outputs` rows of gate, then those of up.
  std::uint32_t* gate_codes;
  std::uint8_t* gate_scales;
  int outputs, gate_blocks, gate_groups, gate_activation;
};
// The features of a share: [first, last).
struct Share8 {
  int first, last;
};
__device__ __forceinline__ Share8 share_of(const Product8& a, int s) {
  const int first = s * a.each + min(s, a.extra);
  return {first, first + a.each + (s < a.extra ? 1 : 0)};
}

// Codes 8 h to 8 h + 7 of sixteen as an operand.
template <int h>
__device__ __forceinline__ bf8_t widen(int4_t codes, float unit) {
  const bf2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes[2 * h], unit, false);
  const bf2_t b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes[2 * h], unit, true);
  const bf2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes[2 * h + 1], unit, false);
  const bf2_t d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes[2 * h + 1], unit, true);
  return bf8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
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
__device__ __forceinline__ int item_of(int block, int total) {
  const int share = total >> 3, rest = total & 7, xcd = block & 7;
  return xcd * share + min(xcd, rest) + (block >> 3);
}
__device__ __forceinline__ Tile8 tile_of(const Product8& a, int id) {
  const int group = static_cast<int>(a.by_group(static_cast<std::uint32_t>(id))), in = id - group * 8 * a.tiles_n;
  const int deep = min(a.tiles_m - group * 8, 8);
  if (deep == 8) return {group * 8 + (in & 7), in >> 3};
  return {group * 8 + in % deep, in / deep};
}

// Rows [first, first + rows) of an operand's codes (or exponents).
__device__ __forceinline__ __amdgpu_buffer_rsrc_t row_buffer(const std::uint8_t* codes, std::int64_t first, int rows, int pitch) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<std::uint8_t*>(codes + first * pitch), static_cast<short>(0), rows * pitch,
                                           0x00020000);
}
__device__ __forceinline__ int4_t load16(__amdgpu_buffer_rsrc_t r, int voffset, int soffset) {
  return __builtin_bit_cast(int4_t, __builtin_amdgcn_raw_buffer_load_b128(r, voffset, soffset, 0));
}

// Sixteen bytes a lane straight into LDS, lane after lane from `lds` on.
__device__ __forceinline__ void load_lds16(__amdgpu_buffer_rsrc_t r, void* lds, int voffset, int soffset) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)lds, 16, voffset, soffset, 0, 0);
}

// An offset past every buffer here (of at most 256 rows of 2^22 bytes): such a load gives
// zeros. Scalar offsets stay inside their buffer, with such a load too: whether they count in
// the check, or are taken from the buffer's size before it, then makes no difference.
constexpr int kNowhere = 0x7fff0000;
// Four bytes a lane straight into LDS.
__device__ __forceinline__ void load_lds4(__amdgpu_buffer_rsrc_t r, void* lds, int voffset, int soffset) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)lds, 4, voffset, soffset, 0, 0);
}
// Waits until at most `count` of this wave's loads are under way.
template <int kCount>
__device__ __forceinline__ void wait_loads() {
  static_assert(kCount < 64);
  __builtin_amdgcn_s_waitcnt((kCount & 15) | (7 << 4) | (15 << 8) | ((kCount >> 4) << 14));
}

// The block's waves meet, their reads of LDS done; loads may still be under way.
__device__ __forceinline__ void block_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// A wave's own reads and writes of LDS are done.
__device__ __forceinline__ void wave_lds_done() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// A tile of kM x kN results, a wave's part of it kWM x kWN in 32 x 32 blocks. Each
// step takes a block of 128 features of the tile's rows, brought from memory straight
// into one of kStages buffers in LDS, kStages - 1 steps ahead. Row r's sixteen-byte
// pieces stand in the order piece ^ (r / 2 & 7): the 64 banks hold two rows, so the reads
// of sixteen neighbouring rows lie in different banks: conflicts in 2 to 3 % of the LDS
// cycles, where the order piece ^ (r & 7) had 46 % (8192^3 takes 780 to 815 us by the GPU's
// clock, and the two orders differ by less than that). Words of exponents, of four steps each,
// have two buffers of their own.
//
// With kSets > 1 there are as many sets of waves, each with the whole tile for every
// kSets-th step and with LDS of its own; their sums meet at the end. A set of one wave
// needs no barriers until then, and makes half the conversions that waves with a quarter of
// a small tile each would make. Sets of more waves share the barriers.
//
// With kGate the tile has 128 columns of gate and the same ones of up, 32 of each by turns,
// and its results leave in 8 bits: 4096 x (2 x 11264) x 4096 in 580 to 595 us, in two
// launches with float32 between them 709.
//
// The features may be split over the grid's rows (Product8::parts).
template <int kM, int kN, int kWM, int kWN, int kSets, int kStages>
struct Tiles8 {
  static constexpr int kWavesN = kN / kWN, kWaves = kM / kWM * kWavesN, kThreads = 64 * kWaves * kSets;  // waves of a set
  static constexpr int kI = kWM / 32, kJ = kWN / 32;
  static constexpr int kRows = kM + kN;  // LDS rows of a buffer: x, then w
  static constexpr int kLoads = kRows / 8 / kWaves;
  static constexpr int kScaleX = (kM + 63) / 64 * 64;  // words of exponents before those of w
  static constexpr int kScaleLoads = (kScaleX + kN) / 64;
  static constexpr int kScaleBuffers = kSets == 1 ? 2 : kStages;
  static constexpr int kStageBytes = kRows * 128, kScales = kStageBytes * kStages;  // where the words of exponents are
  static constexpr int kScaleBytes = kScaleLoads * 256;
  static constexpr int kSetBytes = kScales + kScaleBuffers * kScaleBytes, kLds = kSetBytes * kSets;
  static_assert(kLds <= 160 * 1024 && kStages <= 4);
  static constexpr int kScaled = kSets == 1 ? 0 : (kScaleLoads + kWaves - 1) / kWaves;  // a wave's loads of them in every step
  static_assert(kM % (8 * kWaves) == 0 && kN % (8 * kWaves) == 0 && (kSets > 1 || kM % 64 == 0));
  // Results on their way out through LDS: rows 4 apart lie in different halves of the banks.
  static constexpr int kStride = (kSets == 1 ? kWN : kN) + 8;
  static_assert(kSets == 1 ? kWaves * 32 * kStride * 4 <= kScales : kM * kStride * 4 <= kScales);
};
template <int kM, int kN, int kWM, int kWN, int kSets, int kStages, bool kGate>
__device__ __forceinline__ void product_tile(const Product8& a, Tile8 tile, std::uint8_t* memory) {
  using T = Tiles8<kM, kN, kWM, kWN, kSets, kStages>;
  constexpr int kWavesN = T::kWavesN, kWaves = T::kWaves, kI = T::kI, kJ = T::kJ, kLoads = T::kLoads;
  constexpr int kScaled = T::kScaled;
  const int lane = threadIdx.x & 63, thread_wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int set = thread_wave / kWaves, wave = thread_wave % kWaves;
  std::uint8_t* const lds = memory + set * T::kSetBytes;
  const auto [share_first, last] = share_of(a, static_cast<int>(blockIdx.y));
  const int first = share_first + set;
  const int m0 = tile.m * kM, n0 = tile.n * (kGate ? kN / 2 : kN);
  const int r = lane & 31, g = lane >> 5;

  // Loads: instruction t of a wave brings rows 8 (t kWaves + wave) on of the buffer; rows
  // past the operand's end are its last one again.
  const int m_last = min(a.m - m0, kM) - 1, n_last = kGate ? min(a.outputs - n0, kN / 2) - 1 : min(a.n - n0, kN) - 1;
  // Row of w, from n0 on, that row `row` of w's part of the buffer holds (of gate or up, by bit 5).
  auto w_row = [&](int row) { return min(kGate ? (row >> 6 << 5) + (row & 31) : row, n_last); };
  const std::int64_t w_first = n0 + (kGate && ((wave >> 2) & 1) ? a.outputs : 0);  // a wave's loads are of gate, or of up
  static_assert(!kGate || (kWaves == 8 && 2 * kWM == kM && kN == 256 && kWN == 64 && kSets == 1));
  int offset[kLoads];
  bool of_x[kLoads];
#pragma unroll
  for (int t = 0; t < kLoads; ++t) {
    const int at = 8 * (t * kWaves + wave), row = at + (lane >> 3);
    of_x[t] = t * 8 * kWaves < kM;
    offset[t] = (of_x[t] ? min(row, m_last) : w_row(row - kM)) * a.pitch + (((lane & 7) ^ ((row >> 1) & 7)) << 4);
  }
  // Exponents: words of 64 rows a load, spread over the waves.
  constexpr int kScaleParts = (T::kScaleLoads + kWaves - 1) / kWaves;
  auto scale_part = [&](int t) { return (t * kWaves + wave) % T::kScaleLoads; };
  int scale_offset[kScaleParts];
#pragma unroll
  for (int t = 0; t < kScaleParts; ++t) {
    const int row = 64 * scale_part(t) + lane;
    const int w = row - T::kScaleX;
    scale_offset[t] = 4 * a.scale_pitch * (row < T::kScaleX ? min(row, m_last) : w_row(w) + (kGate && (w >> 5 & 1) ? a.outputs : 0));
  }
  const auto xs_rsrc = row_buffer(reinterpret_cast<const std::uint8_t*>(a.x_scale), m0, m_last + 1, 4 * a.scale_pitch);
  const auto ws_rsrc = row_buffer(reinterpret_cast<const std::uint8_t*>(a.w_scale), n0,
                                  n_last + 1 + (kGate ? a.outputs : 0), 4 * a.scale_pitch);
  // Loads t0 to t1 - 1 of step kt. Past the last step they are issued all the same, without
  // memory behind them, so that every step counts as many.
  auto load = [&](int kt, int buffer, int t0, int t1) {
    std::uint8_t* const at = lds + buffer * T::kStageBytes;
    const bool any = kt < last;
    const auto x_now = row_buffer(a.x, m0, any ? m_last + 1 : 0, a.pitch), w_now = row_buffer(a.w, w_first, any ? n_last + 1 : 0, a.pitch);
#pragma unroll
    for (int t = t0; t < t1; ++t)
      load_lds16(of_x[t] ? x_now : w_now, at + 8 * (t * kWaves + wave) * 128, offset[t], any ? kt * 128 : 0);
    __builtin_amdgcn_sched_barrier(0);
  };
  auto scale_buffer = [&](int kt, int buffer) { return T::kScales + (kSets == 1 ? (kt >> 2) & 1 : buffer) * T::kScaleBytes; };
  auto load_scales = [&](int kt, int buffer) {  // of four steps, with the first of them; a set's with every step
    if constexpr (kSets == 1) {
      if (kt >= last) return;
#pragma unroll
      for (int t = 0; t < kScaleParts; ++t)
        if (t * kWaves + wave < T::kScaleLoads)
          load_lds4(64 * scale_part(t) < kM ? xs_rsrc : ws_rsrc, lds + scale_buffer(kt, buffer) + 256 * scale_part(t), scale_offset[t], (kt >> 2) * 4);
    } else {
      const auto scales = [&](const std::uint32_t* p, int at, int rows) {
        return row_buffer(reinterpret_cast<const std::uint8_t*>(p), at, kt < last ? rows : 0, 4 * a.scale_pitch);
      };
      const auto x_now = scales(a.x_scale, m0, m_last + 1), w_now = scales(a.w_scale, n0, n_last + 1);
#pragma unroll
      for (int t = 0; t < kScaleParts; ++t) {
        std::uint8_t* const to = lds + scale_buffer(kt, buffer) + 256 * scale_part(t);
        load_lds4(64 * scale_part(t) < T::kScaleX ? x_now : w_now, to, scale_offset[t], kt < last ? (kt >> 2) * 4 : 0);
      }
    }
  };

  const int wm = wave / kWavesN * kWM, wn = wave % kWavesN * kWN;
  acc16_t acc[kI][kJ];
#pragma unroll
  for (int i = 0; i < kI; ++i)
#pragma unroll
    for (int j = 0; j < kJ; ++j) acc[i][j] = acc16_t{};

  // A step is four pairs of sixteen features, a pair's operands read as sixteen-byte
  // pieces of codes. While the matrix instructions of one half of a pair run, the codes
  // of the next half are widened; the next pair's are read during the pair, the next
  // step's first ones during the last, behind the step's one barrier: there every wave
  // has read all of its step, so that the buffer can take the step kStages further on.
  struct Codes {
    int4_t x[kI], w[kJ];
  };
  struct Operands {
    bf8_t x[kI], w[kJ];
  };
  float x_unit[kI], w_unit[kJ];
  auto read = [&](Codes& c, int buffer, int p) {
    const std::uint8_t* const at = lds + buffer * T::kStageBytes + (((2 * p + g) ^ ((r >> 1) & 7)) << 4);
#pragma unroll
    for (int i = 0; i < kI; ++i) c.x[i] = *reinterpret_cast<const int4_t*>(at + (wm + 32 * i + r) * 128);
#pragma unroll
    for (int j = 0; j < kJ; ++j) c.w[j] = *reinterpret_cast<const int4_t*>(at + (kM + wn + 32 * j + r) * 128);
  };
  auto read_units = [&](int kt, int buffer) {
    const std::uint32_t* const scales = reinterpret_cast<const std::uint32_t*>(lds + scale_buffer(kt, buffer));
#pragma unroll
    for (int i = 0; i < kI; ++i) x_unit[i] = unit_of(scales[wm + 32 * i + r], kt);
#pragma unroll
    for (int j = 0; j < kJ; ++j) w_unit[j] = unit_of(scales[T::kScaleX + wn + 32 * j + r], kt);
  };
  auto widen_all = [&]<int h>(Operands& o, const Codes& c) {
#pragma unroll
    for (int i = 0; i < kI; ++i) o.x[i] = widen<h>(c.x[i], x_unit[i]);
#pragma unroll
    for (int j = 0; j < kJ; ++j) o.w[j] = widen<h>(c.w[j], w_unit[j]);
  };
  auto multiply = [&](const Operands& o) {
#pragma unroll
    for (int i = 0; i < kI; ++i)
#pragma unroll
      for (int j = 0; j < kJ; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(o.x[i], o.w[j], acc[i][j], 0, 0, 0);
  };
  // Order: loads, reads of LDS, then matrix instructions with conversions between them, as
  // many to each, the first `alone` without.
  constexpr int kProducts = kI * kJ, kConversions = (kI + kJ) * 4;
  auto order = [&]<int kReads, int kAlone>() {
    if constexpr (kReads > 0) __builtin_amdgcn_sched_group_barrier(0x100, kReads, 0);
    if constexpr (kAlone > 0) __builtin_amdgcn_sched_group_barrier(0x008, kAlone, 0);
#pragma unroll
    for (int t = kAlone; t < kProducts; ++t) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, (kConversions + kProducts - kAlone - 1) / (kProducts - kAlone), 0);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  // A step's loads are issued in four parts: all at once they keep a wave from its matrix
  // instructions for a quarter of a step.
  constexpr int kPart = (kLoads + 3) / 4;
  auto part = [&](int i) { return min(i * kPart, kLoads); };

  auto meet = [&] {
    if constexpr (kSets == 1 || kWaves > 1) block_barrier();
    else wave_lds_done();
  };

#pragma unroll
  for (int t = 0; t < kStages; ++t) {
    const int kt = first + t * kSets;
    if (kSets > 1 || t == 0 || (kt & 3) == 0) load_scales(kt, t);
    load(kt, t, 0, t + 1 < kStages ? kLoads : part(1));  // the rest of the last one's in the first step
  }
  Codes codes;
  Operands low, high;
  wait_loads<(kStages - 2) * (kLoads + kScaled) + kScaled + kPart>();
  meet();
  read(codes, 0, 0);
  read_units(first, 0);
  widen_all.template operator()<0>(low, codes);
  int buffer = 0, before = kStages - 1;  // of this step and the one before
  for (int kt0 = share_first; kt0 < last; kt0 += kSets) {  // as many steps for every set, the last ones perhaps without a block
    const int kt = kt0 + set;
    const bool live = kSets == 1 || kt < last;
    const int next = buffer + 1 == kStages ? 0 : buffer + 1;
    const int behind = kt + (kStages - 1) * kSets, ahead = behind + kSets;  // loads that the step before began; that this one begins
    if (live) {
#pragma unroll
      for (int p = 0; p < 3; ++p) {
        Codes after;
        if (p < 2) load(behind, before, part(1 + 2 * p), part(2 + 2 * p));
        read(after, buffer, p + 1);
        multiply(low);
        widen_all.template operator()<1>(high, codes);
        order.template operator()<kI + kJ, 0>();
        if (p < 1) load(behind, before, part(2), part(3));
        multiply(high);
        widen_all.template operator()<0>(low, after);
        order.template operator()<0, 0>();
        codes = after;
      }
      multiply(low);
      widen_all.template operator()<1>(high, codes);
      order.template operator()<0, 0>();
    }
    wait_loads<(kStages - 2) * (kLoads + kScaled)>();
    meet();
    if (live) {
      if (kSets > 1 || (ahead & 3) == 0) load_scales(ahead, buffer);
      load(ahead, buffer, 0, part(1));
      read(codes, next, 0);
      read_units(kt + kSets, next);
      multiply(high);
      widen_all.template operator()<0>(low, codes);
      order.template operator()<kI + kJ, kProducts / 2>();
    }
    before = buffer;
    buffer = next;
  }
  wait_loads<0>();

  // Lane (r, g) has column r of rows 8 (e / 4) + 4 g + e % 4 of each 32 x 32. They pass
  // through LDS, so that a lane stores four results of a row, and that the activation
  // stands in the code few times, not once for each register (which cost 2.6 us in
  // fetching instructions).
  if constexpr (kGate) {  // 32 rows of both halves at a time: a wave's 32 columns of gate, and of up
    constexpr int kGateStride = kN + 8;
    static_assert(64 * kGateStride * 4 <= T::kScales);
    float* const turn = reinterpret_cast<float*>(lds);
    const int wave_row = wm / kWM, column = wn / 2;
#pragma unroll 1
    for (int i0 = 0; i0 < kI; ++i0) {
      block_barrier();  // the buffers, or the rows before, are done with
#pragma unroll
      for (int i = 0; i < kI; ++i) {
        if (i != i0) continue;
#pragma unroll
        for (int j = 0; j < kJ; ++j)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            turn[(32 * wave_row + 8 * (e / 4) + 4 * g + e % 4) * kGateStride + kN / 2 * j + column + r] = acc[i][j][e];
      }
      block_barrier();
      // Sixteen lanes a row, its block of 128 features as encode_block has it.
#pragma unroll 1
      for (int row = static_cast<int>(threadIdx.x) >> 4; row < 64; row += 32) {
        const int m = m0 + (row >> 5) * kWM + 32 * i0 + (row & 31), lane16 = static_cast<int>(threadIdx.x) & 15;
        float4_t v[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int f = 64 * h + 4 * lane16;
          const float* const at = turn + row * kGateStride + f;
          float4_t gate = *reinterpret_cast<const float4_t*>(at), up = *reinterpret_cast<const float4_t*>(at + kN / 2);
          if (a.bias != nullptr) {
            gate = add4(gate, load_features(a.bias, n0 + f, a.outputs));
            up = add4(up, load_features(a.bias + a.outputs, n0 + f, a.outputs));
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) v[h][e] = f + e <= n_last ? activate8(gate[e], a.gate_activation) * up[e] : 0.0F;
        }
        const Coded8 c = encode_block(v);
        if (m >= a.m) continue;
        std::uint32_t* const codes = a.gate_codes + (static_cast<std::int64_t>(m) * a.gate_blocks + tile.n) * 32;
        codes[lane16] = c.word[0];
        codes[16 + lane16] = c.word[1];
        std::uint8_t* const scale = a.gate_scales + static_cast<std::int64_t>(m) * a.gate_groups * 4 + tile.n;
        if (lane16 == 0) *scale = static_cast<std::uint8_t>(c.byte);
        else if (tile.n + 1 == a.gate_blocks && tile.n + lane16 < a.gate_groups * 4) scale[lane16] = 0;  // the last word filled up
      }
    }
    return;
  }
  const bool whole = a.parts == nullptr;
  float* const out = whole ? a.out : a.parts + static_cast<std::int64_t>(blockIdx.y) * a.m * a.n;
  const std::int64_t stride = whole ? a.out_stride : a.n;
  const float* const bias_row = whole ? a.bias : nullptr;
  const int activation = whole ? a.activation : TCX_ACT_NONE;
  auto give = [&](float* to, int i, int row0) {
#pragma unroll
    for (int j = 0; j < kJ; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) to[(row0 + 8 * (e / 4) + 4 * g + e % 4) * T::kStride + 32 * j + r] = acc[i][j][e];
  };
  auto store = [&](float4_t v, int m, int n, float4_t bias) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = activate8(v[e] + bias[e], activation);
    store_features(out + m * stride, n, a.n, v);
  };
  const float4_t none = {0.0F, 0.0F, 0.0F, 0.0F};
  constexpr int kAcross = (kSets == 1 ? kWN : kN) / 4;  // lanes to a row
  const int column = lane % kAcross * 4;
  if constexpr (kSets == 1) {  // 32 rows at a time, each wave on its own
    float* const turn = reinterpret_cast<float*>(lds) + wave * 32 * T::kStride;
    block_barrier();  // the buffers are done with
    const int n = n0 + wn + column;
    const float4_t bias = bias_row != nullptr ? load_features(bias_row, n, a.n) : none;
#pragma unroll
    for (int i = 0; i < kI; ++i) {
      give(turn, i, 0);
      wave_lds_done();
#pragma unroll 1
      for (int row = lane / kAcross; row < 32; row += 64 / kAcross) {
        const int m = m0 + wm + 32 * i + row;
        if (m >= a.m) break;
        store(*reinterpret_cast<const float4_t*>(turn + row * T::kStride + column), m, n, bias);
      }
      wave_lds_done();
    }
  } else {  // every set its sums of the tile in its own LDS, then all of them rows of the whole
    if constexpr (kWaves > 1) block_barrier();
#pragma unroll
    for (int i = 0; i < kI; ++i) give(reinterpret_cast<float*>(lds) + wn, i, wm + 32 * i);
    block_barrier();
    const int n = n0 + column;
    const float4_t bias = bias_row != nullptr ? load_features(bias_row, n, a.n) : none;
#pragma unroll 1
    for (int row = static_cast<int>(threadIdx.x) / kAcross; row < kM; row += T::kThreads / kAcross) {
      const int m = m0 + row;
      if (m >= a.m) break;
      float4_t v = none;
#pragma unroll
      for (int other = 0; other < kSets; ++other)
        v = add4(v, *reinterpret_cast<const float4_t*>(reinterpret_cast<const float*>(memory + other * T::kSetBytes) + row * T::kStride + column));
      store(v, m, n, bias);
    }
  }
}

// With kHalves the tiles past the last whole round of 256, if they leave half the CUs
// empty, are taken by two blocks each, one for the rows of either half (from tile a.whole
// on): 4096 x 5120 x 4096, 320 tiles, in 155 us, else 193.
constexpr int kHalved = 128;
template <int kM, int kN, int kWM, int kWN, int kSets, int kStages, bool kGate, bool kHalves>
__global__ __launch_bounds__((Tiles8<kM, kN, kWM, kWN, kSets, kStages>::kThreads)) void product_kernel(Product8 a) {
  __shared__ __attribute__((aligned(1024))) std::uint8_t memory[Tiles8<kM, kN, kWM, kWN, kSets, kStages>::kLds];
  const int block = static_cast<int>(blockIdx.x);
  if constexpr (kHalves) {
    if (block >= a.whole) {
      const int rest = a.tiles_m * a.tiles_n - a.whole, second = block - a.whole >= rest ? 1 : 0;
      Tile8 tile = tile_of(a, a.whole + item_of(block - a.whole - second * rest, rest));
      tile.m = 2 * tile.m + second;
      if (tile.m * (kM / 2) < a.m) product_tile<kM / 2, kN, kWM / 2, kWN, kSets, kStages, kGate>(a, tile, memory);
      return;
    }
  }
  product_tile<kM, kN, kWM, kWN, kSets, kStages, kGate>(a, tile_of(a, item_of(block, a.whole)), memory);
}

void share_out(Product8& a, int units, int splits, float* parts) {
  a.parts = parts;
  a.each = units / splits;
  a.extra = units % splits;
}

template <int kM, int kN, int kWM, int kWN, int kSets, int kStages, bool kGate = false, bool kHalves = false>
int launch_product(Product8 a, int splits, float* parts, hipStream_t s) {
  a.tiles_m = (a.m + kM - 1) / kM;
  a.tiles_n = kGate ? a.gate_blocks : (a.n + kN - 1) / kN;
  a.by_group = FastDiv(static_cast<std::uint32_t>(8 * a.tiles_n));
  share_out(a, a.blocks, splits, parts);
  constexpr int kThreads = Tiles8<kM, kN, kWM, kWN, kSets, kStages>::kThreads;
  const std::int64_t tiles = static_cast<std::int64_t>(a.tiles_m) * a.tiles_n;
  const std::int64_t rest = tiles * splits % 256, halved = kHalves && rest > 0 && rest <= kHalved ? tiles % 256 : 0;
  if ((tiles + halved) * splits * kThreads > kMaxLaunchWorkItems || tiles >= (std::int64_t{1} << 30))
    return fail(TCX_INVALID_ARGUMENT, "linear8 has too many results");
  a.whole = static_cast<int>(tiles - halved);
  hipLaunchKernelGGL((product_kernel<kM, kN, kWM, kWN, kSets, kStages, kGate, kHalves>),
                     dim3(static_cast<unsigned>(tiles + halved), static_cast<unsigned>(splits)),
                     dim3(kThreads), 0, s, a);
  return check(hipGetLastError(), "linear8 launch");
}

// Up to sixteen rows: each weight is read once, straight into the registers that multiply
// it. The eight waves of a block share the features of a tile of sixteen weights' rows: wave
// p takes units (four blocks of 128) p, p + 8 and so on, kU of them, whose part of x it
// keeps in registers from tile to tile while the next unit's weights are under way.
// Lane (r, g) holds 16-byte pieces g and 4 + g of each block of row r. The waves' sums
// of a tile meet in LDS.
//
// Bound by reading the weights: 8 x 128256 x 4096 in 95 us, 5.6 TB/s; 1 x 4096 x 4096 in
// 5.8 (4.7 from the cache), of which 2.4 are the launch. Loads that stay out of the caches
// (106), a unit more under way (97) and two (102), 512 blocks (97) and waves with all
// features of a tile of their own (124) were slower for the first.
template <int kU>
__global__ __launch_bounds__(512) void few_rows_kernel(Product8 a) {
  __shared__ float4_t sums[2][8][64];
  constexpr int kStaged = 8;
  __shared__ int4_t stages[kU == 1 ? 8 : 1][kU == 1 ? kStaged * 32 : 1];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4, units = a.scale_pitch;

  // Blocks past the row's end are zeros in x. There w has the codes of the row's last block, or
  // of its last unit for a wave without one of its own, with exponents of zero: such values
  // are finite (with their own exponents they may be infinite, and infinity times zero is
  // NaN), or NaN where that column is NaN anyway. Of up to kStaged rows each is brought once, 512
  // bytes of two rows a load, and spread through the wave's own LDS: 0.7 us less for 1 x 4096 x
  // 4096 than lanes that each load their own pieces.
  int4_t x[kU][8], stage[kStaged / 2];
  std::uint32_t x_word[kU];
  const auto x_rsrc = row_buffer(a.x, 0, a.m, a.pitch);
  const bool staged = kU == 1 && a.m <= kStaged;
  if (staged) {
#pragma unroll
    for (int t = 0; t < kStaged / 2; ++t) {
      const int row = 2 * t + (lane >> 5), at = 16 * (lane & 31);
      if (2 * t < a.m)
        stage[t] = load16(x_rsrc, row < a.m && wave < units && at < (a.blocks - 4 * wave) * 128 ? row * a.pitch + at : kNowhere,
                          wave < units ? wave * 512 : 0);
    }
  }
  const int x_row = min(r, a.m - 1);
#pragma unroll
  for (int u = 0; u < kU; ++u) {
    const int unit = wave + 8 * u;
    x_word[u] = unit < units ? a.x_scale[static_cast<std::int64_t>(x_row) * a.scale_pitch + unit] : 0;
    if (staged) continue;
#pragma unroll
    for (int p = 0; p < 8; ++p)
      x[u][p] = load16(x_rsrc, unit < units && 4 * unit + p / 2 < a.blocks ? x_row * a.pitch + 16 * g + 64 * p : kNowhere,
                       unit < units ? unit * 512 : 0);
  }

  struct Weights {
    int4_t piece[8];
    std::uint32_t word;
  };
  auto load = [&](Weights& w, int tile, int u) {
    const int rows = min(a.n - 16 * tile, 16), own = wave + 8 * u, unit = min(own, units - 1);
    const auto rsrc = row_buffer(a.w, 16 * tile, rows, a.pitch);
    const int row = min(r, rows - 1), at = row * a.pitch + 16 * g;
    w.word = own < units ? a.w_scale[static_cast<std::int64_t>(16 * tile + row) * a.scale_pitch + unit] : 0;
#pragma unroll
    for (int p = 0; p < 8; ++p) w.piece[p] = load16(rsrc, at + 64 * (p & 1), min(4 * unit + p / 2, a.blocks - 1) * 128);
  };
  int tile = static_cast<int>(blockIdx.x);
  Weights now, next;
  load(now, tile, 0);
  if (staged) {
    // Piece q of row m stands at q ^ (m & 7).
    int4_t* const own = stages[wave];
#pragma unroll
    for (int t = 0; t < kStaged / 2; ++t) {
      const int row = 2 * t + (lane >> 5);
      if (2 * t < a.m) own[row * 32 + ((lane & 31) ^ (row & 7))] = stage[t];
    }
#pragma unroll
    for (int p = 0; p < 8; ++p) x[0][p] = own[x_row * 32 + ((4 * p + g) ^ (x_row & 7))];
  }

  float4_t acc;
  auto compute = [&](const Weights& w, int u) {
#pragma unroll
    for (int p = 0; p < 8; ++p) {
      const float w_unit = unit_of(w.word, p / 2), x_unit = unit_of(x_word[u], p / 2);
      int4_t codes = x[u][p];
      if constexpr (kU > 1) asm volatile("" : "+v"(codes));  // kept as codes: widened once they would take twice the registers
      acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen<0>(w.piece[p], w_unit), widen<0>(codes, x_unit), acc, 0, 0, 0);
      acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen<1>(w.piece[p], w_unit), widen<1>(codes, x_unit), acc, 0, 0, 0);
    }
  };
  // Thread i of the first 256 gives result i % 16 of the tile and row i / 16 (lane (m, g)
  // has results 4 g on of row m).
  const int m = static_cast<int>(threadIdx.x) >> 4, column = static_cast<int>(threadIdx.x) & 15;
  auto bias_of = [&](int tile) {  // asked for before the next weights are
    return a.bias != nullptr && threadIdx.x < 256 ? a.bias[min(16 * tile + column, a.n - 1)] : 0.0F;
  };
  auto finish = [&](int tile, int turn, float bias) {
    sums[turn][wave][lane] = acc;
    __syncthreads();
    const int n = 16 * tile + column;
    if (threadIdx.x >= 256 || m >= a.m || n >= a.n) return;
    const float* const at = reinterpret_cast<const float*>(&sums[turn][0][m + 16 * (column >> 2)]) + (column & 3);
    float v = 0.0F;
#pragma unroll
    for (int p = 0; p < 8; ++p) v += at[p * 256];
    a.out[m * a.out_stride + n] = activate8(v + bias, a.activation);
  };

  int turn = 0;
  while (true) {
    const int after = tile + static_cast<int>(gridDim.x);
    const float bias = bias_of(tile);
    acc = float4_t{0.0F, 0.0F, 0.0F, 0.0F};
#pragma unroll
    for (int u = 0; u + 1 < kU; ++u) {
      load(next, tile, u + 1);
      compute(now, u);
      now = next;
    }
    if (after >= a.tiles_n) {
      compute(now, kU - 1);
      finish(tile, turn, bias);
      return;
    }
    load(next, after, 0);
    compute(now, kU - 1);
    finish(tile, turn, bias);
    now = next;
    tile = after;
    turn ^= 1;
  }
}

template <int kU>
int launch_few_rows(Product8 a, float* parts, hipStream_t s) {
  a.tiles_n = (a.n + 15) / 16;
  if (parts != nullptr) {  // the one part of a gated product's results
    a.out = parts;
    a.out_stride = a.n;
    a.bias = nullptr;
    a.activation = TCX_ACT_NONE;
  }
  hipLaunchKernelGGL(few_rows_kernel<kU>, dim3(static_cast<unsigned>(std::min(a.tiles_n, 256))), dim3(512), 0, s, a);
  return check(hipGetLastError(), "linear8 launch");
}

// Sums of shares of the features, [splits][m][n], joined in their order. (Without features
// there are none, and this is the whole product.)
struct Join8 {
  const float* parts;
  const float* bias;
  float* out;
  std::int64_t out_stride, part;  // floats between rows of out; between shares
  int n, splits, activation;
  std::uint32_t items;  // four results of a row each
  FastDiv by_row;
};
__device__ __forceinline__ float4_t sum_parts(const float* parts, std::int64_t row, int n, int width, int splits, std::int64_t part) {
  float4_t v = {0.0F, 0.0F, 0.0F, 0.0F};
  if (splits == 1) return load_features(parts + row, n, width);
  for (int s = 0; s < splits; s += 4) {  // four loads at a time
    float4_t p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = load_features(parts + min(s + i, splits - 1) * part + row, n, width);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (s + i < splits) v = add4(v, p[i]);
  }
  return v;
}
__global__ __launch_bounds__(256) void join_kernel(Join8 a) {
  for (std::uint32_t item = blockIdx.x * 256 + threadIdx.x; item < a.items; item += gridDim.x * 256) {
    const std::uint32_t m = a.by_row(item);
    const int n = static_cast<int>(item - m * a.by_row.divisor) * 4;
    float4_t v = sum_parts(a.parts, static_cast<std::int64_t>(m) * a.n, n, a.n, a.splits, a.part);
    if (a.bias != nullptr) v = add4(v, load_features(a.bias, n, a.n));
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = activate8(v[e], a.activation);
    store_features(a.out + m * a.out_stride, n, a.n, v);
  }
}

// act(gate + bias) * (up + bias) of rows [gate | up], in 8 bits: a wave a group of four blocks.
struct Gate8 {
  const float* parts;  // [splits][rows][2 * width]
  const float* bias;
  std::uint32_t* codes;
  std::uint8_t* scales;
  std::int64_t part;
  int width, blocks, groups, activation, splits;
  std::uint32_t items;
  FastDiv by_groups;
};
__global__ __launch_bounds__(256) void gate_kernel(Gate8 a) {
  const int lane = threadIdx.x & 63;
  const std::uint32_t step = gridDim.x * 4;
  for (std::uint32_t item = blockIdx.x * 4 + (threadIdx.x >> 6); item < a.items; item += step) {
    const std::uint32_t row = a.by_groups(item);
    const Place8 p = place8(lane, static_cast<int>(item - row * a.groups));
    const std::int64_t at = static_cast<std::int64_t>(row) * 2 * a.width;
    float4_t v[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int f = p.feature + 64 * h;
      float4_t gate = sum_parts(a.parts, at, f, a.width, a.splits, a.part);
      float4_t up = sum_parts(a.parts + a.width, at, f, a.width, a.splits, a.part);
      if (a.bias != nullptr) {
        gate = add4(gate, load_features(a.bias, f, a.width));
        up = add4(up, load_features(a.bias + a.width, f, a.width));
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) v[h][e] = f + e < a.width ? activate8(gate[e], a.activation) * up[e] : 0.0F;
    }
    store_group(a.codes + static_cast<std::int64_t>(row) * a.blocks * 32, a.scales + static_cast<std::int64_t>(row) * a.groups * 4, p,
                a.blocks, encode_block(v));
  }
}

// The ways to a product, and what a round of blocks on all 256 CUs took, in us: `fixed`
// (start, first loads, results) and `step` for each block of 128 features, with one
// block a CU and with as many as fit, which rounds before the last have (1024 to 12000
// features, most weights from memory; ways 0 and 2 also 128 to 1024 features and n up to
// 128256). Of 256 x 256: with halves of at most 128 tiles, and with whole ones. Few
// features over many tiles are for way 2, whose four blocks a CU hide one's start and
// results behind another's products: 25 x 126974 x 139 in 13 us, way 0 in 30. Way 3's step
// is bound by what the L2s give (24 KB a CU and step, 11 TB/s of all): half the
// conversions and a third buffer made no difference.
//
// The reading of weights bounds a step only of unsplit tiles here, not of shares nor of the
// gated tiles: for few rows of wide ones the times are told too short. The choice is near the
// bytes' time all the same for 1 and 16 x 2 * 28672 x 8192 (99 to 102 us, 88 reading), 2 * 18432 x
// 7168 (60 to 62, 49) and 1 x 8192 x 28672 (45, 44), not for 1 x 2 * 8192 x 8192 (38, 25: 64 x 64
// tiles in four shares). The gated tiles of 64 rows want more of the L2s than they give: 39 us
// for 512 x 2 * 4096 x 4096, told 30.
struct Way8 {
  int kind, m, n, sets, fit;  // tile, and blocks that a CU holds
  float fixed[2], step[2];
};
constexpr Way8 kWays[] = {
    {0, 32, 64, 4, 1, {1.5F, 2.4F}, {0.23F, 0.23F}},   {1, 64, 64, 4, 1, {2.8F, 2.8F}, {0.30F, 0.30F}},
    {2, 64, 64, 1, 4, {1.4F, 4.2F}, {0.75F, 1.22F}},   {3, 128, 64, 2, 1, {2.7F, 2.7F}, {0.58F, 0.58F}},
    {4, 128, 128, 1, 2, {7.0F, 7.7F}, {1.08F, 1.75F}}, {5, 256, 128, 1, 1, {7.0F, 7.0F}, {1.45F, 1.71F}},
    {6, 256, 256, 1, 1, {9.5F, 13.7F}, {1.50F, 2.75F}},
};
constexpr int kFewRows = 7, kFusedGate = 8, kFusedGate64 = 9;  // from kFusedGate on: gated products in one launch
// A microsecond's reading of weights from memory.
constexpr float kReads = 5.4e6F;
struct Plan8 {
  int kind, splits;
};
std::size_t part_bytes(const Product8& a, int splits) {
  return static_cast<std::size_t>(a.m) * static_cast<std::size_t>(a.n) * static_cast<std::size_t>(splits) * sizeof(float);
}
// What shares of the features cost in a second launch and in bytes at 4.5 TB/s.
float join_cost(const Product8& a, int splits) {
  return splits == 1 ? 0.0F : 4.5F + (splits + 1) * 4.0F * static_cast<float>(a.m) * static_cast<float>(a.n) / 4.5e6F;
}
// Units of the features that a wave holds of few rows.
int few_rows_units(const Product8& a) { return (a.scale_pitch + 7) / 8; }
// `gated`: the results go through float32 and a second launch to 8 bits, unless the tiles
// of 256 x 256 do that themselves.
Plan8 plan_product(const Product8& a, bool gated, std::size_t workspace_bytes) {
  Plan8 best{0, 1};
  float least = 1e30F;
  // Few rows, as far as a wave's registers hold its part of x: a round of 256 tiles takes
  // its weights' bytes or a chain of 1.8 us for 4096 features. 16 x 22528 x 4096 in 22 us (32 x 64 tiles: 26),
  // 1 x 4096 x 4096 in 5.8 (8.9); but 8 x 60000 x 1024 in 30 (64 x 64 tiles: 17).
  if (a.m <= 16 && a.scale_pitch <= 24) {
    const float chain = 1.8F * static_cast<float>(few_rows_units(a)), row = static_cast<float>(a.pitch) / kReads;
    const int rounds = (a.n - 1) / 4096;  // whole ones before the last
    least = static_cast<float>(rounds) * std::max(chain, 4096.0F * row) + std::max(chain, static_cast<float>(a.n - rounds * 4096) * row);
    if (gated) least += join_cost(a, 2);
    best = {kFewRows, 1};
  }
  for (const Way8& w : kWays) {
    const std::int64_t tiles = static_cast<std::int64_t>((a.m + w.m - 1) / w.m) * ((a.n + w.n - 1) / w.n);
    for (int splits = 1; splits <= 16; splits = splits < 4 ? splits + 1 : splits * 3 / 2) {
      const std::int64_t blocks = tiles * splits, fit = 256 * w.fit;
      if (splits > 1 && (blocks > fit || a.blocks < splits * w.sets || part_bytes(a, splits) > workspace_bytes)) break;
      const float steps = static_cast<float>((a.blocks + splits - 1) / splits);
      // `full`: 0 with a block on each CU to 1 with as many as fit. Weights that one row of
      // tiles reads come from memory (split ones, of few outputs, were in the cache when timed).
      auto round = [&](std::int64_t count, float full) {
        const float bytes = a.m <= w.m && splits == 1 ? static_cast<float>(count * w.n * kBlock8) / kReads : 0.0F;
        return w.fixed[0] + full * (w.fixed[1] - w.fixed[0]) + steps * std::max(w.step[0] + full * (w.step[1] - w.step[0]), bytes);
      };
      const std::int64_t rounds = (blocks - 1) / fit, rest = blocks - rounds * fit;  // whole ones, and the last's blocks
      float full = w.fit > 1 ? static_cast<float>((rest - 1) / 256) / static_cast<float>(w.fit - 1) : 0.0F;
      if (w.kind == 6 && rest > kHalved) full = 1.0F;
      float time = static_cast<float>(rounds) * round(fit, 1.0F) + round(rest, full);
      time += gated ? join_cost(a, splits + 1) : join_cost(a, splits);
      if (time < least) {
        least = time;
        best = {w.kind, splits};
      }
    }
  }
  if (gated && (static_cast<std::int64_t>(a.outputs) + 256) * 4 * a.scale_pitch < (std::int64_t{1} << 31)) {
    const auto steps = static_cast<float>(a.blocks);
    auto fused = [&](int kind, float time) {
      if (time >= least) return;
      least = time;
      best = {kind, 1};
    };
    const std::int64_t tiles = static_cast<std::int64_t>((a.m + 255) / 256) * a.gate_blocks, rest = tiles % 256;
    float time = static_cast<float>(tiles / 256 + (rest > kHalved ? 1 : 0)) * (12.0F + steps * 2.75F);
    if (rest > 0 && rest <= kHalved) time += 9.0F + steps * 1.45F;
    fused(kFusedGate, time);
    // Tiles of 64 rows: few features, or too few rows for the others to fill the CUs. 16 x 2 * 256 x
    // 256 in 7.2 us (in two launches 8.8), 512 x 2 * 4096 x 4096 in 39 (49).
    const std::int64_t before = (static_cast<std::int64_t>((a.m + 63) / 64) * a.gate_blocks - 1) / 256;
    fused(kFusedGate64, static_cast<float>(before) * (4.2F + steps * 0.98F) + 3.6F + steps * 0.84F);
  }
  return best;
}
int run_plan(const Product8& a, const Plan8& plan, float* parts, hipStream_t s) {
  switch (plan.kind) {
    case 0: return launch_product<32, 64, 32, 64, 4, 3>(a, plan.splits, parts, s);
    case 1: return launch_product<64, 64, 64, 64, 4, 2>(a, plan.splits, parts, s);
    case 2: return launch_product<64, 64, 32, 32, 1, 2>(a, plan.splits, parts, s);
    case 3: return launch_product<128, 64, 64, 32, 2, 2>(a, plan.splits, parts, s);
    case 4: return launch_product<128, 128, 64, 64, 1, 2>(a, plan.splits, parts, s);
    case 5: return launch_product<256, 128, 64, 64, 1, 3>(a, plan.splits, parts, s);
    case 6: return launch_product<256, 256, 128, 64, 1, 2, false, true>(a, plan.splits, parts, s);
    case kFusedGate: return launch_product<256, 256, 128, 64, 1, 2, true, true>(a, 1, nullptr, s);
    case kFusedGate64: return launch_product<64, 256, 32, 64, 1, 3, true>(a, 1, nullptr, s);
    default: break;
  }
  switch (few_rows_units(a)) {
    case 1: return launch_few_rows<1>(a, parts, s);
    case 2: return launch_few_rows<2>(a, parts, s);
    default: return launch_few_rows<3>(a, parts, s);
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
  if (gated) {
    a.outputs = static_cast<int>(d.outputs);
    a.gate_blocks = static_cast<int>(blocks8(d.outputs));
    a.gate_groups = static_cast<int>(scale_words8(d.outputs));
    a.gate_activation = d.activation;
  }
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

}  // namespace
}  // namespace tcx

extern "C" {

int tcx_hip_linear8_plan(const tcx_hip_linear8_desc_t* desc, int gated, size_t workspace_bytes, tcx_hip_linear8_plan_t* plan) {
  using namespace tcx;
  if (plan == nullptr) return fail(TCX_INVALID_ARGUMENT, "linear8 plan is null");
  Product8 a;
  if (int rc = product_args(desc, gated != 0, a); rc != TCX_OK) return rc;
  if (a.m == 0 || a.n == 0 || a.blocks == 0) return fail(TCX_INVALID_ARGUMENT, "no linear8 product for these extents");
  const Plan8 p = plan_product(a, gated != 0, gated != 0 ? SIZE_MAX : workspace_bytes);
  const bool whole = p.kind >= kFusedGate || (gated == 0 && p.splits == 1);
  *plan = {16, 16, 8, 0, p.splits, whole ? 1 : 2, whole ? 0 : part_bytes(a, p.splits)};
  if (p.kind == kFewRows) {
    plan->units = few_rows_units(a);
  } else if (p.kind >= kFusedGate) {
    plan->tile_rows = p.kind == kFusedGate ? 256 : 64;
    plan->tile_outputs = 128;
    plan->sets = 1;
  } else {
    plan->tile_rows = kWays[p.kind].m;
    plan->tile_outputs = kWays[p.kind].n;
    plan->sets = kWays[p.kind].sets;
  }
  return TCX_OK;
}

size_t tcx_hip_linear8_workspace_bytes(const tcx_hip_linear8_desc_t* desc) {
  using namespace tcx;
  Product8 a;
  if (product_args(desc, false, a) != TCX_OK || a.m == 0 || a.n == 0) return 0;
  const Plan8 plan = plan_product(a, false, SIZE_MAX);
  return plan.splits > 1 ? part_bytes(a, plan.splits) : 0;
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
  const auto s = static_cast<hipStream_t>(stream);
  Plan8 plan{0, 0};
  if (a.blocks > 0) {
    plan = plan_product(a, false, workspace != nullptr ? workspace_bytes : 0);
    if (plan.splits == 1) return run_plan(a, plan, nullptr, s);
    if (int rc = run_plan(a, plan, static_cast<float*>(workspace), s); rc != TCX_OK) return rc;
  }
  Join8 j{};
  j.parts = static_cast<const float*>(workspace);
  j.bias = a.bias;
  j.out = out;
  j.out_stride = a.out_stride;
  j.part = static_cast<std::int64_t>(a.m) * a.n;
  j.n = a.n;
  j.splits = plan.splits;
  j.activation = a.activation;
  j.by_row = FastDiv(static_cast<std::uint32_t>((a.n + 3) / 4));
  if (a.m >= (std::int64_t{1} << 31) / j.by_row.divisor) return fail(TCX_INVALID_ARGUMENT, "linear8 has too many results");
  j.items = static_cast<std::uint32_t>(a.m) * j.by_row.divisor;
  hipLaunchKernelGGL(join_kernel, dim3(grid_for(j.items, 256, kStrideBlocks)), dim3(256), 0, s, j);
  return check(hipGetLastError(), "linear8 join launch");
}

size_t tcx_hip_gated_linear8_workspace_bytes(const tcx_hip_linear8_desc_t* desc) {
  using namespace tcx;
  Product8 a;
  if (product_args(desc, true, a) != TCX_OK || a.m == 0 || a.n == 0 || a.blocks == 0) return 0;
  const Plan8 plan = plan_product(a, true, SIZE_MAX);
  return plan.kind >= kFusedGate ? 0 : part_bytes(a, plan.splits);
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
  if (!aligned8(workspace, 16)) return fail(TCX_INVALID_ARGUMENT, "linear8 workspace must be 16-byte aligned");
  if (a.m >= (std::int64_t{1} << 31) / a.gate_groups) return fail(TCX_INVALID_ARGUMENT, "linear8 has too many results");
  Plan8 plan{0, 0};
  if (a.blocks > 0) {
    plan = plan_product(a, true, SIZE_MAX);
    if (plan.kind < kFusedGate && (workspace == nullptr || workspace_bytes < part_bytes(a, plan.splits)))
      return fail(TCX_INVALID_ARGUMENT, "gated_linear8 needs a workspace of the query's size");
  }
  if (int rc = ready(); rc != TCX_OK) return rc;
  const auto s = static_cast<hipStream_t>(stream);
  a.gate_codes = reinterpret_cast<std::uint32_t*>(codes);
  a.gate_scales = reinterpret_cast<std::uint8_t*>(scales);
  if (plan.kind >= kFusedGate) return run_plan(a, plan, nullptr, s);
  if (a.blocks > 0)
    if (int rc = run_plan(a, plan, static_cast<float*>(workspace), s); rc != TCX_OK) return rc;
  Gate8 t{};
  t.parts = static_cast<const float*>(workspace);
  t.bias = a.bias;
  t.part = static_cast<std::int64_t>(a.m) * a.n;
  t.splits = plan.splits;
  t.width = a.outputs;
  t.blocks = a.gate_blocks;
  t.groups = a.gate_groups;
  t.codes = a.gate_codes;
  t.scales = a.gate_scales;
  t.activation = a.gate_activation;
  t.items = static_cast<std::uint32_t>(static_cast<std::int64_t>(a.m) * t.groups);
  t.by_groups = FastDiv(static_cast<std::uint32_t>(t.groups));
  hipLaunchKernelGGL(gate_kernel, dim3(grid_for(t.items, 4, kStrideBlocks)), dim3(256), 0, s, t);
  return check(hipGetLastError(), "gated_linear8 launch");
}

}  // extern "C"
