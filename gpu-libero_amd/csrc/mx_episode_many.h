// Attention of many rows: a workgroup takes 128 rows of one world's key head (new tokens times the query
// heads that share the key head), each of its four waves 32 of them, and 64 keys at a time, which all four
// read from LDS.  The mathematics is that of attend_few (one pass, running maximum, scores transposed so
// that probabilities stay in their lanes), with 32x32 products and one 16-bit part of each probability:
// here the matrix instructions are what bounds the kernel, and its error is that of the result's own rounding.
//
// The running maximum follows the scores only when one passes it by more than 2^8: until then the sums
// are exact multiples of what they would be, and the output need not be rescaled.
#pragma once
#include "mx_episode_types.h"
#include "mx_episode_launch.h"

namespace mxe {

constexpr int kManyKeys = 64;

template <class E, int D>
struct ManyShared {
  static constexpr int kStrideK = D + 8;      // rows of 16-byte reads by 16 lanes fall into all banks once
  // transposing reads take 64 bytes of each of four rows at once: rows 16 banks apart
  static constexpr int kStrideV = D + (D == 128 || D == 64 ? 32 : 0);
  typename E::T k[2][kManyKeys * kStrideK];
  typename E::T v[2][kManyKeys * kStrideV];
  int wild[2][4];                             // by wave: an infinity or NaN among the values it brought
};

__device__ inline float both_halves_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ inline float both_halves_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

template <int kType, bool kFp8, int D>
__global__ __launch_bounds__(256, 2) void attend_many(const Attend a) {
  typedef Elem<kType> E;
  typedef typename E::T T;
  typedef typename E::V8 V8;
  typedef ManyShared<E, D> Shared;
  constexpr int kC = D / 16, kTiles = D / 32;
  constexpr int kPer = kFp8 ? 16 : 8, kChunks = D / kPer, kLoads = (kManyKeys * kChunks + 255) / 256;
  constexpr bool kWhole = kManyKeys * kChunks % 256 == 0, kOneGroup = 16 * kChunks % 64 == 0;
  __shared__ __attribute__((aligned(16))) Shared sh;

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int n32 = lane & 31, half = lane >> 5;

  // Blocks go to the XCDs in turn: where the key heads of all worlds divide among the eight, those of one
  // stay on one XCD, whose L2 then holds their keys and values.  Last rows first: under a causal mask they
  // have the most keys.
  int split, head, tile;
  {
    unsigned block = blockIdx.x;
    split = block % a.splits;
    block /= a.splits;
    const int per = a.tiles / a.nworld;
    if (!a.start && (a.nworld * a.kv_heads) % 8 == 0) {
      const int i = block >> 3, pair = (block & 7) + 8 * (i / per);
      head = pair % a.kv_heads;
      tile = pair / a.kv_heads * per + per - 1 - i % per;
    } else {
      head = block % a.kv_heads;
      tile = a.tiles - 1 - block / a.kv_heads;
    }
  }
  Tile t;
  if (!find_tile(a, tile, kManyRows, t)) return;

  const int last_row = min(t.row + kManyRows, t.rows) - 1;
  int first_low, first_high, last_low, last_high;
  limits(a, t, t.row / a.group, first_low, first_high);
  limits(a, t, last_row / a.group, last_low, last_high);
  int begin, end;
  split_range(a, split, first_low, last_high, begin, end);

  // this wave's and lane's rows
  const int wave_row = t.row + 32 * wave, r = wave_row + n32;
  const bool rows_here = wave_row < t.rows, row_here = r < t.rows;
  int wave_all_low = 0, wave_all_high = 0, wave_low = 0, wave_high = 0;
  if (rows_here) {
    limits(a, t, wave_row / a.group, wave_low, wave_all_high);
    limits(a, t, (min(wave_row + 32, t.rows) - 1) / a.group, wave_all_low, wave_high);
  }
  const int token_in = (row_here ? r : t.row) / a.group;
  const int query_head = head * a.group + (row_here ? r : t.row) - token_in * a.group;
  int low_r, high_r;
  limits(a, t, token_in, low_r, high_r);
  if (!row_here) high_r = 0;
  V8 q[kC];
  {
    const T* from = (const T*)a.q + (int64_t)(t.token + token_in) * a.q_token + (int64_t)query_head * a.q_head;
#pragma unroll
    for (int c = 0; c < kC; c++) q[c] = load_query<E>(a, from + 16 * c + 8 * half);
  }

  f16v o[kTiles];
#pragma unroll
  for (int c = 0; c < kTiles; c++)
#pragma unroll
    for (int i = 0; i < 16; i++) o[c][i] = 0.f;
  float m = -INFINITY, l = 0.f;

  // ---- bringing keys and values: each thread a 16-byte piece of kLoads keys and of their values.  16 keys
  // from a multiple of 16 on lie in one page, so that addresses are a wave's own but for an offset of 32 bits.
  Fixed* table = fixed(a.table + (int64_t)t.world * a.width);
  const int page_mask = (1 << a.page_shift) - 1;
  const int64_t row_bytes = kFp8 ? D : 2 * D;
  int page[4];
  u4 kreg[kLoads], vreg[kLoads];
  unsigned kbyte[kFp8 ? kLoads : 1], vbyte[kFp8 ? kLoads : 1];
  const auto key_of = [&](int j) { return (j * 256 + (int)threadIdx.x) / kChunks; };
  const auto piece_of = [&](int j) { return (j * 256 + (int)threadIdx.x) % kChunks; };
  const auto first_of = [&](int key, int g) { return min(key + 16 * g, (end - 1) & ~15); };
  auto look_up = [&](int key) {
#pragma unroll
    for (int g = 0; g < 4; g++) page[g] = table[first_of(key, g) >> a.page_shift];
  };
  auto load = [&](int key) {
    int64_t base[4];
#pragma unroll
    for (int g = 0; g < 4; g++) {
      const int in = (unsigned)page[g] < (unsigned)a.npage ? page[g] : 0;
      base[g] = (((int64_t)in * a.kv_heads + head) << a.page_shift) + (first_of(key, g) & page_mask);
    }
#pragma unroll
    for (int j = 0; j < kLoads; j++) {
      if (!kWhole && key_of(j) >= kManyKeys) continue;
      // the group of 16 keys: the wave's, or where a wave's pieces straddle two, the lane's
      const int group = kOneGroup ? (j * 256 + 64 * wave) / (16 * kChunks) : key_of(j) / 16;
      int64_t at = base[0];
#pragma unroll
      for (int g = 1; g < 4; g++) at = group == g ? base[g] : at;
      const unsigned row = min(key_of(j) % 16, end - 1 - first_of(key, group));
      const unsigned offset = row * (unsigned)row_bytes + piece_of(j) * 16;
      kreg[j] = *(const u4*)(a.k + at * row_bytes + offset);
      vreg[j] = *(const u4*)(a.v + at * row_bytes + offset);
      if constexpr (kFp8) {
        const unsigned byte = row * kTiles + piece_of(j) / 2;
        kbyte[j] = (a.k_scale + at * kTiles)[byte];
        vbyte[j] = (a.v_scale + at * kTiles)[byte];
      }
    }
  };
  // Into LDS: values of keys that are not there as zeros, and, where only some rows of the workgroup see a
  // key, infinities and NaN too (those rows get them added below).  `all`: every key is there.
  auto is_edge = [&](int key) { return key < last_low || key + kManyKeys > first_high; };
  auto store = [&](int buffer, int key, unsigned present) {
    const bool edge = is_edge(key), all = present == 15u && key + kManyKeys <= end;
    unsigned wild = 0;
#pragma unroll
    for (int j = 0; j < kLoads; j++) {
      if (!kWhole && key_of(j) >= kManyKeys) continue;
      const int key_in = key_of(j), d = piece_of(j) * kPer;
      V8 k[kPer / 8], v[kPer / 8];
      if constexpr (kFp8) {
        k[0] = from_fp8<E>(u2{kreg[j].x, kreg[j].y}, kbyte[j]);
        k[1] = from_fp8<E>(u2{kreg[j].z, kreg[j].w}, kbyte[j]);
        v[0] = from_fp8<E>(u2{vreg[j].x, vreg[j].y}, vbyte[j]);
        v[1] = from_fp8<E>(u2{vreg[j].z, vreg[j].w}, vbyte[j]);
      } else {
        k[0] = __builtin_bit_cast(V8, kreg[j]);
        v[0] = __builtin_bit_cast(V8, vreg[j]);
      }
      if (edge || !all) {
        const bool none = key + key_in >= end || !(present >> (key_in / 16) & 1);
#pragma unroll
        for (int e = 0; e < kPer / 8; e++) {
          u4 words = __builtin_bit_cast(u4, v[e]);
#pragma unroll
          for (int y = 0; y < 4; y++) {
            if (none) words[y] = 0;
            wild |= not_finite<E>(words[y]) & 0x80008000u;
            words[y] = finite_or_zero<E>(words[y]);
          }
          v[e] = __builtin_bit_cast(V8, words);
        }
      }
#pragma unroll
      for (int e = 0; e < kPer / 8; e++) {
        *(V8*)&sh.k[buffer][key_in * Shared::kStrideK + d + 8 * e] = k[e];
        *(V8*)&sh.v[buffer][key_in * Shared::kStrideV + d + 8 * e] = v[e];
      }
    }
    if (edge || !all) {
      const int any = __ballot(wild != 0) != 0;
      if (lane == 0) sh.wild[buffer][wave] = any;
    }
  };
  auto pages_there = [&]() {
    unsigned bits = 0;
#pragma unroll
    for (int g = 0; g < 4; g++) bits |= ((unsigned)page[g] < (unsigned)a.npage ? 1u : 0u) << g;
    return bits;
  };

  typedef __attribute__((address_space(3))) s4* TrPtr;
  int key = begin, buffer = 0;
  unsigned present = 0;
  if (key < end) {
    look_up(key);
    load(key);
    present = pages_there();
    if (key + kManyKeys < end) look_up(key + kManyKeys);
    store(0, key, present);
  }
  for (; key < end; key += kManyKeys, buffer ^= 1) {
    const bool more = key + kManyKeys < end;
    __syncthreads();
    unsigned next_present = 0;
    if (more) {
      load(key + kManyKeys);
      next_present = pages_there();
      if (key + 2 * kManyKeys < end) look_up(key + 2 * kManyKeys);
    }
    if (rows_here && key < wave_high && key + kManyKeys > wave_low) {
      const bool there = present == 15u && key + kManyKeys <= end;
      const bool edge = key < wave_all_low || key + kManyKeys > wave_all_high || !there;
      f16v s[2];
#pragma unroll
      for (int u = 0; u < 2; u++) {
#pragma unroll
        for (int i = 0; i < 16; i++) s[u][i] = 0.f;
        const T* from = &sh.k[buffer][(32 * u + n32) * Shared::kStrideK + 8 * half];
#pragma unroll
        for (int c = 0; c < kC; c++) s[u] = E::mfma32(*(const V8*)(from + 16 * c), q[c], s[u]);
      }
      if (edge) {
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
          for (int i = 0; i < 16; i++) {
            const int at = key + 32 * u + 8 * (i / 4) + 4 * half + i % 4;
            if (!((present >> (2 * u + i / 8) & 1) && at >= low_r && at < high_r && at < end)) s[u][i] = -INFINITY;
          }
      }
      float top = -INFINITY;
#pragma unroll
      for (int u = 0; u < 2; u++)
#pragma unroll
        for (int i = 0; i < 16; i++) top = fmaxf(top, s[u][i]);
      top = both_halves_max(top) * a.scale2;
      if (__ballot(top > m + 8.f)) {
        const float next = fmaxf(m, top), shrink = __builtin_amdgcn_exp2f(m - (next == -INFINITY ? 0.f : next));
        m = next;
        l *= shrink;
#pragma unroll
        for (int c = 0; c < kTiles; c++) o[c] *= shrink;
      }
      const float zero = m == -INFINITY ? 0.f : m;
      V8 p[2][2];
      float sum[2] = {0.f, 0.f};
#pragma unroll
      for (int u = 0; u < 2; u++)
#pragma unroll
        for (int i = 0; i < 16; i++) {
          const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][i], a.scale2, -zero));
          sum[u] += x;
          p[u][i / 8][i % 8] = (T)x;
        }
      l += sum[0] + sum[1];
#pragma unroll
      for (int u = 0; u < 2; u++)
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
          for (int c = 0; c < kTiles; c++) {
            const T* at = &sh.v[buffer][(32 * u + 16 * b + 4 * half + ((lane & 15) >> 2)) * Shared::kStrideV + 32 * c +
                                        16 * ((lane >> 4) & 1) + 4 * (lane & 3)];
            const s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((TrPtr)at);
            const s4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((TrPtr)(at + 8 * Shared::kStrideV));
            o[c] = E::mfma32(__builtin_bit_cast(V8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7)), p[u][b], o[c]);
          }
      if ((!there || is_edge(key)) &&
          (sh.wild[buffer][0] | sh.wild[buffer][1] | sh.wild[buffer][2] | sh.wild[buffer][3])) {
        // values that are not finite went in as zeros: the rows that see them get them added
        for (int k = key; k < min(key + kManyKeys, end); k++) {
          const int in = table[k >> a.page_shift];
          if ((unsigned)in >= (unsigned)a.npage || !(k >= low_r && k < high_r)) continue;
          const int64_t at = (((int64_t)in * a.kv_heads + head) << a.page_shift) + (k & page_mask);
#pragma unroll
          for (int c = 0; c < kTiles; c++)
#pragma unroll
            for (int i = 0; i < 16; i++) {
              const float value = value_at<E, kFp8, D>(a, at, 32 * c + 8 * (i / 4) + 4 * half + i % 4);
              if (!(fabsf(value) < INFINITY)) o[c][i] += value;
            }
        }
      }
    }
    if (more) store(buffer ^ 1, key + kManyKeys, next_present);
    present = next_present;
  }

  if (!row_here) return;
  l = both_halves_sum(l);
  const int64_t row_at = (int64_t)(t.token + token_in) * a.heads + query_head;
  if (a.splits > 1) {
    const int64_t at = (int64_t)split * a.tokens * a.heads + row_at;
    if (l != 0.f)
#pragma unroll
      for (int c = 0; c < kTiles; c++)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
          *(f4*)(a.part + at * D + 32 * c + 2 * i + 4 * half) = f4{o[c][i], o[c][i + 1], o[c][i + 2], o[c][i + 3]};
    if (half == 0) *(f2*)(a.part_ml + 2 * at) = f2{m, l};
    return;
  }
  const float inverse = 1.f / l;
  T* to = (T*)a.out + (int64_t)(t.token + token_in) * a.o_token + (int64_t)query_head * a.o_head;
#pragma unroll
  for (int c = 0; c < kTiles; c++)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      T x[4];
#pragma unroll
      for (int e = 0; e < 4; e++) x[e] = (T)(l == 0.f ? 0.f : o[c][i + e] * inverse);
      if (a.o_vector) {
        typedef T T4 __attribute__((ext_vector_type(4)));
        *(T4*)(to + 32 * c + 2 * i + 4 * half) = T4{x[0], x[1], x[2], x[3]};
      } else {
#pragma unroll
        for (int e = 0; e < 4; e++) to[32 * c + 2 * i + 4 * half + e] = x[e];
      }
    }
  if (a.lse && half == 0) a.lse[row_at] = l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * kLn2;
}

}  // namespace mxe
