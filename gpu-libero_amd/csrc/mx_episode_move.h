// What kernels that move rows into and out of the pages share: the slots of a chunk's rows, and pieces of rows and pages
// with their 8-bit conversions.
#pragma once
#include "mx_episode_types.h"

namespace mxe {

struct Copy {
  uint8_t *pages, *scales;       // of k or v
  const uint8_t* rows;
  int64_t token_stride, head_stride;
  bool vector;                   // rows are 16-byte aligned
};
struct Move {
  Copy of[2];
  const int32_t *table, *length, *start;
  int nworld, npage, width, kv_heads, head_dim, page_shift, tokens, count, tokens_each;
};

// The slot of packed row `token` of a world's chunk, as (page * kv_heads * page_tokens + slot) without the
// head; -1: none
__device__ inline int64_t slot_of(const Move& a, int world, int place, int count) {
  if (place < 0 || place >= count) return -1;
  const int position = max(a.length[world], 0) - count + place;
  if (position < 0 || (position >> a.page_shift) >= a.width) return -1;
  const int page = a.table[(int64_t)world * a.width + (position >> a.page_shift)];
  if ((unsigned)page >= (unsigned)a.npage) return -1;
  return (((int64_t)page * a.kv_heads) << a.page_shift) + (position & ((1 << a.page_shift) - 1));
}

// The worlds of `tokens` (at most 64) packed rows from `first` on, by the lanes of one wave: a lane's own, -1 beyond
// the rows.  Ragged chunks: the first row's world by a search with 64 probes at a time, the others' from there, mostly the
// same; rows that no world has get a neighbour's, with a place outside of its chunk.
__device__ inline int world_of(const int32_t* start, int nworld, int count, int first, int tokens) {
  const int lane = threadIdx.x & 63, token = first + lane;
  if (!start) return lane < tokens ? token / count : -1;
  int low = 0, high = nworld;
  while (high - low > 1) {
    const int step = (high - low + 63) >> 6, probe = low + lane * step;
    const int passed = max(1, (int)__popcll(__ballot(probe < high && start[probe] <= first)));
    low += (passed - 1) * step;
    high = min(high, low + step);
  }
  if (lane >= tokens) return -1;
  if (start[low + 1] <= token) {
    high = nworld;
    while (high - low > 1) {
      const int middle = (low + high) >> 1;
      if (start[middle] <= token) low = middle; else high = middle;
    }
  }
  return low;
}

// The slots of `tokens` (at most 64) packed rows from `first` on, by the lanes of one wave
__device__ inline void find_slots(const Move& a, int first, int tokens, int64_t* slots) {
  const int lane = threadIdx.x, token = first + lane;
  const int world = world_of(a.start, a.nworld, a.count, first, tokens);
  if (world < 0) return;
  const int begin = a.start ? a.start[world] : world * a.count, count = a.start ? a.start[world + 1] - begin : a.count;
  slots[lane] = slot_of(a, world, token - begin, count);
}

// A thread's piece of a row in bytes, and how many pieces of keys and of values it has under way.  8-bit pages: 32
// bytes, so that a thread's codes are 8 or 16 at once, except for reads into single precision, which are bound
// by their own stores.  us, measured with 16 and 32 bytes: 500 histories of 8-bit pages into bf16 180 and 152, 67 chunks of
// single precision written to 8-bit pages and read back 61 and 69 (16 for the read alone 59); one and two under way:
// 500 histories of bf16 173 and 185, the 67 chunks 61 and 59.
constexpr int piece_bytes(bool fp8, bool write, int size) { return fp8 && (write || size < 4) ? 32 : 16; }
constexpr int pieces_ahead(int size) { return size == 4 ? 2 : 1; }

template <class T, int N> __device__ inline void load_row(const T* from, bool vector, float (&x)[N]) {
  constexpr int kEach = 16 / sizeof(T) < N ? 16 / sizeof(T) : N;
  typedef T V __attribute__((ext_vector_type(kEach)));
  if (vector) {
#pragma unroll
    for (int j = 0; j < N; j += kEach) {
      const V v = *(const V*)(from + j);
#pragma unroll
      for (int e = 0; e < kEach; e++) x[j + e] = (float)v[e];
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; j++) x[j] = (float)from[j];
  }
}

// kPast: past the caches.  Rows that were read out are many; 262 MB of 8-bit pages into 524 MB of rows 183 us
// through the caches, 152 past them, and 69 or 61 for 34 + 137 MB.
template <bool kPast, class T, int N> __device__ inline void store_row(T* to, bool vector, const float (&x)[N]) {
  constexpr int kEach = 16 / sizeof(T) < N ? 16 / sizeof(T) : N;
  typedef T V __attribute__((ext_vector_type(kEach)));
  if (vector) {
#pragma unroll
    for (int j = 0; j < N; j += kEach) {
      V v;
#pragma unroll
      for (int e = 0; e < kEach; e++) v[e] = (T)x[j + e];
      if constexpr (kPast) __builtin_nontemporal_store(v, (V*)(to + j));
      else *(V*)(to + j) = v;
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; j++) to[j] = (T)x[j];
  }
}

// `at`: element in the pages; at / 32 is the scale's place, as head_dim is a multiple of 32
template <int kStore, int N> __device__ inline void load_page(const Copy& c, int64_t at, float (&x)[N]) {
  if constexpr (kStore == MX_TYPE_FP8) {
    typedef unsigned W __attribute__((ext_vector_type(N / 4)));
    const W w = *(const W*)(c.pages + at);
    const float scale = scale_of(c.scales[at / MX_SCALE_BLOCK]);
#pragma unroll
    for (int j = 0; j < N / 4; j++) {
      const f2 p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w[j], scale, false);
      const f2 q = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w[j], scale, true);
      x[4 * j] = p[0];
      x[4 * j + 1] = p[1];
      x[4 * j + 2] = q[0];
      x[4 * j + 3] = q[1];
    }
  } else {
    load_row((const typename Elem<kStore>::T*)c.pages + at, true, x);
  }
}

// All threads take part, with at < 0 where there is nothing to store: neighbours share a scale
template <int kStore, int N> __device__ inline void store_page(const Copy& c, int64_t at, const float (&x)[N]) {
  if constexpr (kStore == MX_TYPE_FP8) {
    // the largest magnitude of the block, as the bits of a float that is not negative: they order
    // like integers, infinities and NaN above all numbers
    unsigned top = 0;
#pragma unroll
    for (int j = 0; j < N; j++) top = max(top, __float_as_uint(x[j]) & 0x7fffffffu);
#pragma unroll
    for (int lanes = 1; lanes < MX_SCALE_BLOCK / N; lanes *= 2) top = max(top, (unsigned)__shfl_xor((int)top, lanes));
    // 448 = 1.75 * 2^8: the exponent less 8, and one more above a fraction of 1.75
    const bool finite = top < 0x7f800000u;
    const int e = max((int)(top >> 23) - 127 - 8 + ((top & 0x7fffffu) > 0x600000u), -117);
    const float inverse = __uint_as_float((unsigned)(127 - e) << 23);
    if (at < 0) return;
    typedef unsigned W __attribute__((ext_vector_type(N / 4)));
    W w;
#pragma unroll
    for (int j = 0; j < N / 4; j++) {
      float y[4];
#pragma unroll
      for (int i = 0; i < 4; i++) y[i] = finite ? x[4 * j + i] * inverse : 0.f;
      const unsigned half = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
      w[j] = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], half, true);
    }
    *(W*)(c.pages + at) = w;
    if (at % MX_SCALE_BLOCK == 0) c.scales[at / MX_SCALE_BLOCK] = finite ? (uint8_t)(e + 127) : 255;
  } else {
    if (at >= 0) store_row<false>((typename Elem<kStore>::T*)c.pages + at, true, x);
  }
}

}  // namespace mxe
