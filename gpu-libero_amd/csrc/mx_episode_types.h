// Element types, matrix instructions and 8-bit conversions of the episode memory's kernels (gfx950),
// and what the kernels share: arguments, chunk lookup, row limits.
//
// Lane layouts used below (l = lane; checked by running them against plain products):
//   16x16x32: A row l % 16, k = 8 (l / 16) + j; B column l % 16, same k; C column l % 16, rows 4 (l / 16) + i.
//   32x32x16: A row l % 32, k = 8 (l / 32) + j; B column l % 32, same k; C column l % 32,
//             rows 8 (i / 4) + 4 (l / 32) + i % 4.
//   ds_read_tr16_b64: the 16 lanes of a group each address 8 bytes, four lanes to a row of 16 values;
//             lane i of the group receives column i of the four rows.
#pragma once
#include <hip/hip_runtime.h>
#include <cfloat>
#include <cstdint>
#include "../../include/mx_physics.h"
#include "../../include/mx_episode.h"

namespace mxe {

typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
typedef _Float16 hf8 __attribute__((ext_vector_type(8)));
typedef _Float16 hf2 __attribute__((ext_vector_type(2)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef short s8 __attribute__((ext_vector_type(8)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef unsigned u2 __attribute__((ext_vector_type(2)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// Tables, lengths and starts do not change while a kernel runs: where an index is a wave's own, its load goes
// through the scalar cache
typedef __attribute__((address_space(4))) const int32_t Fixed;
__device__ inline Fixed* fixed(const int32_t* p) { return (Fixed*)(uintptr_t)p; }

// Weights are 2^(score - reference), 16-bit operands of the second product.  A reference is set so that the
// largest weight then is 2^kTop; attend_few keeps it until a lane's sum of a step passes kSumHolds, attend_many
// until a weight would pass 2^kHolds.  In bfloat16, which has the range of 32 bits, any reference does.  float16
// ends at 65504 and has full precision down to 2^-14, steps of 2^-24 below: with its largest weights from 2^12 on, those down
// to 2^-26 of the largest (18 nats) are as exact as any, and those below 2^-37 (25 nats) are lost to the product,
// though not to the sum of weights, which is in 32 bits.  (Largest weights of 1 lost all below 2^-25: 4095 values
// 15 nats under one of zero were 2.6 % off.)
template <int kType> struct Elem;
template <> struct Elem<MX_TYPE_BF16> {
  typedef __bf16 T;
  typedef bf8 V8;
  typedef bf2 V2;
  static constexpr unsigned kExponent = 0x7f80;   // all ones in an infinity or NaN
  static constexpr float kTop = 0.f, kSumHolds = 4096.f, kHolds = 8.f;   // see above
  static __device__ f4 mfma16(V8 a, V8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
  static __device__ f16v mfma32(V8 a, V8 b, f16v c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
  // two e4m3 codes (low or high half of w) times a power of two; exact: three fraction bits
  template <bool kHigh> static __device__ V2 from_fp8(unsigned w, float scale) {
    return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, kHigh);
  }
};
template <> struct Elem<MX_TYPE_F16> {
  typedef _Float16 T;
  typedef hf8 V8;
  typedef hf2 V2;
  static constexpr unsigned kExponent = 0x7c00;
  static constexpr float kTop = 12.f, kSumHolds = 65504.f, kHolds = 15.9f;
  static __device__ f4 mfma16(V8 a, V8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
  static __device__ f16v mfma32(V8 a, V8 b, f16v c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
  // exact from 2^-24 up to 65504, as any value of the queries' type
  template <bool kHigh> static __device__ V2 from_fp8(unsigned w, float scale) {
    return __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, kHigh);
  }
};

// Two 16-bit values in a word: the top bit of each half is set if it is an infinity or NaN (an exponent of
// all ones carries into the sign's place when its last bit is added; other bits mean nothing)
template <class E> __device__ inline unsigned not_finite(unsigned w) {
  constexpr unsigned e = E::kExponent | E::kExponent << 16, last = E::kExponent & -E::kExponent;
  return (w & e) + (last | last << 16);
}

template <class E> __device__ inline unsigned finite_or_zero(unsigned w) {
  const unsigned off = not_finite<E>(w);
  return w & ~((off & 0x8000u ? 0xffffu : 0u) | (off & 0x80000000u ? 0xffff0000u : 0u));
}

// A sum of weighted values, its weights made smaller: where the factor is 0 an infinity stays what it is, as its weight
// is not zero but only beyond the range of 32 bits
__device__ inline float rescaled(float x, float by) {
  const float y = x * by;
  return y == y ? y : x;
}
__device__ inline f4 rescaled(f4 x, float by) {
  return f4{rescaled(x[0], by), rescaled(x[1], by), rescaled(x[2], by), rescaled(x[3], by)};
}

// Sums that are made anew from the values that are not finite: where none of those is found (finite ones have passed 32
// bits) an infinity has to come out again.  It is kept as the largest finite number, to which they can be added.
__device__ inline float set_aside(float x) { return fabsf(x) < INFINITY ? x : copysignf(FLT_MAX, x); }
__device__ inline float brought_back(float x) { return fabsf(x) == FLT_MAX ? copysignf(INFINITY, x) : x; }

// E8M0: byte b stands for 2^(b - 127), 255 for NaN.  The scaled conversions take the exponent of their scale in
// this sense, with 255 giving NaN whatever the code and 0 giving 2^-127 (run over all of these).
__device__ inline float scale_of(unsigned byte) { return __uint_as_float(byte << 23); }

template <class E> __device__ inline typename E::V8 from_fp8(u2 w, unsigned byte) {
  const float s = scale_of(byte);
  const auto a = E::template from_fp8<false>(w.x, s), b = E::template from_fp8<true>(w.x, s);
  const auto c = E::template from_fp8<false>(w.y, s), d = E::template from_fp8<true>(w.y, s);
  return typename E::V8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// The kernels' arguments, by value.  `rows` are (token, head of the group) pairs of one key head, in
// the order token * group + head, in tiles of a kernel's own number of rows.
struct Attend {
  const uint8_t *k, *v, *k_scale, *v_scale;
  const int32_t *table, *length, *start;
  const void* q;
  void* out;
  float *lse, *part, *part_ml;       // part: [split][row][D]; part_ml: [split][row][2]; rows: see part_row()
  int64_t q_token, q_head, o_token, o_head;
  int nworld, npage, width, kv_heads, page_shift, tokens, count, max_count, heads, group;
  int causal, window, tiles, splits;
  int part_rows;                     // of one split
  float scale2;                      // |scale| * log2(e), not 0: probabilities are powers of two
  bool negate;                       // scale < 0: the queries change their sign
  bool q_vector, o_vector;           // q's rows are 16-byte aligned, out's 8-byte
};

// A kernel's only argument, read where it is used: as a by-value parameter all of it would be in scalar
// registers from the first instruction to the last, and the loops' own values would be spilled for it.
__device__ __forceinline__ const Attend& arguments() {
  return *(const Attend*)(__attribute__((address_space(4))) const Attend*)__builtin_amdgcn_kernarg_segment_ptr();
}

// Eight values of a query
template <class E> __device__ inline typename E::V8 load_query(const Attend& a, const typename E::T* from) {
  typename E::V8 x;
  if (a.q_vector) {
    x = *(const typename E::V8*)from;
  } else {
#pragma unroll
    for (int j = 0; j < 8; j++) x[j] = from[j];
  }
  return a.negate ? -x : x;
}

// Four values of V from d on (a multiple of 4), of the row at `row` with its scales at `scale`
template <class E, bool kFp8> __device__ inline f4 values_at(const uint8_t* row, const uint8_t* scale, int d) {
  if constexpr (kFp8) {
    const unsigned w = *(const unsigned*)(row + d);
    const float s = scale_of(scale[d / MX_SCALE_BLOCK]);
    const auto a = E::template from_fp8<false>(w, s), b = E::template from_fp8<true>(w, s);
    return f4{(float)a[0], (float)a[1], (float)b[0], (float)b[1]};
  } else {
    typedef typename E::T T4 __attribute__((ext_vector_type(4)));
    return __builtin_convertvector(*(const T4*)((const typename E::T*)row + d), f4);
  }
}

// Whether there is an infinity or NaN among the first `pieces` of 16 bytes, by the lanes of a wave together
template <class E, bool kFp8> __device__ inline bool any_wild(const uint8_t* from, const uint8_t* scale, int pieces) {
  unsigned wild = 0;
  for (int j = threadIdx.x & 63; j < pieces; j += 64) {
    const u4 w = *(const u4*)(from + 16 * j);
    if constexpr (kFp8) {
      const u4 x = __builtin_bit_cast(u4, from_fp8<E>(u2{w.x, w.y}, scale[j / 2]));
      const u4 y = __builtin_bit_cast(u4, from_fp8<E>(u2{w.z, w.w}, scale[j / 2]));
#pragma unroll
      for (int i = 0; i < 4; i++) wild |= not_finite<E>(x[i]) | not_finite<E>(y[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++) wild |= not_finite<E>(w[i]);
    }
  }
  return __ballot((wild & 0x80008000u) != 0) != 0;
}

// The world of a tile.  Ragged chunks: world w has the tile numbers from start[w] group / rows + w on,
// at least as many as its rows need, so that the tile of a block follows from `start` by a search,
// 64 probes at a time, and the number of tiles from sizes that the host knows.
struct Tile {
  int world, row, rows, token, length, position;   // first row, rows in all, first packed token, tokens
                                                   // in reach, position of the chunk's first token
};

__device__ inline long long tile_base(const Attend& a, int w, int rows_per_tile) {
  return (long long)a.start[w] * a.group / rows_per_tile + w;
}

__device__ inline bool find_tile(const Attend& a, int tile, int rows_per_tile, Tile& t) {
  int count, token;
  if (!a.start) {
    const int per = (a.max_count * a.group + rows_per_tile - 1) / rows_per_tile;
    t.world = tile / per;
    t.row = (tile - t.world * per) * rows_per_tile;
    token = t.world * a.count;
    count = a.count;
  } else {
    const int lane = threadIdx.x & 63;
    int low = 0, high = a.nworld;
    while (high - low > 1) {
      const int step = (high - low + 63) >> 6, probe = low + lane * step;
      const bool below = probe < high && tile_base(a, probe, rows_per_tile) <= tile;
      const int passed = max(1, (int)__popcll(__ballot(below)));
      low += (passed - 1) * step;
      high = min(high, low + step);
    }
    low = __builtin_amdgcn_readfirstlane(low);
    t.world = low;
    const long long row = (tile - tile_base(a, low, rows_per_tile)) * rows_per_tile;
    token = fixed(a.start)[low];
    const int stop = fixed(a.start)[low + 1], end = min(stop, a.tokens);
    if (token < 0 || end <= token || row < 0 || row >= (long long)(end - token) * a.group) return false;
    t.row = (int)row;
    count = stop - token;
    t.rows = (int)min((long long)min(end - token, a.max_count) * a.group, (long long)INT32_MAX);
  }
  if (!a.start) t.rows = a.max_count * a.group;
  if (t.row >= t.rows) return false;
  t.token = token;
  const int length = max(fixed(a.length)[t.world], 0);
  t.position = length - count;
  t.length = (int)min((long long)length, (long long)a.width << a.page_shift);
  return true;
}

// The row among the parts of query head h of the chunk's token i: chunks of one size have rows for max_count tokens
// of each world, ragged ones for all packed tokens
__device__ inline int64_t part_row(const Attend& a, const Tile& t, int i, int h) {
  return (a.start ? t.token + i : t.world * a.max_count + i) * (int64_t)a.heads + h;
}

// The part of the keys [low, high) of a tile that a split takes: the same number for each, in steps of 128
// keys, and no fewer than kLeastKeys (the last ones may have none).  By the world's own keys and not by
// the most that the table can hold, so that long and short worlds both keep all splits at work.
constexpr int kLeastKeys = 256;
__device__ inline void split_range(const Attend& a, int split, int low, int high, int& begin, int& end) {
  // rows that see nothing may have a low beyond the table's reach, and up to 2^31 - 2: key numbers counted on from
  // there would pass 32 bits, so that no range starts after its end (at most 2^30)
  begin = min(low & ~63, max(high, 0));
  end = high;
  if (a.splits == 1) return;
  const int each = max(kLeastKeys, (int)(((unsigned)max(high - begin, 0) / (unsigned)a.splits + 128u) & ~127u));
  const long long from = begin + (long long)split * each;
  begin = (int)min(from, (long long)max(high, 0));
  end = (int)min(from + each, (long long)high);
}

// The keys [low, high) that the chunk's token i sees
__device__ inline void limits(const Attend& a, const Tile& t, int i, int& low, int& high) {
  const int position = t.position + i;
  high = position < 0 ? 0 : a.causal ? min(position + 1, t.length) : t.length;
  low = a.window > 0 && position >= a.window ? position - a.window + 1 : 0;
}

}  // namespace mxe
