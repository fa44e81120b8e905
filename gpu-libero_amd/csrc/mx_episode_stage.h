// Bringing kKeys keys and their values at a time into LDS, for workgroups of 256 threads.
//
// 16-bit pages go from memory to LDS without passing registers (each wave 1 KB at a time, lane after lane), so
// the rows in LDS are as long as in the pages; what keeps the reads off each other's banks is the order of a row's
// 16-byte pieces, which each row has its own of: reads of one piece of 16 rows, and transposing reads of
// four pieces of four rows, fall into all 64 banks once.  8-bit pages are converted on the way.
#pragma once
#include <cstddef>
#include "mx_episode_types.h"

namespace mxe {

template <class E, int kKeys, int D>
struct Staged {
  static constexpr int kPieces = D / 8;       // of a row; 16 of them pass over all banks
  typename E::T k[kKeys * D], v[kKeys * D];
  int wild[4];                                // by wave: an infinity or NaN among the values it brought

  // the place of piece p of a row, and (they are pairs) the piece at a place
  static __device__ __forceinline__ int place_k(int row, int p) {
    if constexpr (D == 96) return p + (row >> 2 & 3) < 12 ? p + (row >> 2 & 3) : p + (row >> 2 & 3) - 12;
    else if constexpr (D < 128) return p ^ (row / (16 / kPieces) & (kPieces - 1));
    else return p ^ (row & 15);
  }
  static __device__ __forceinline__ int piece_k(int row, int at) {
    if constexpr (D == 96) return at - (row >> 2 & 3) >= 0 ? at - (row >> 2 & 3) : at - (row >> 2 & 3) + 12;
    else return place_k(row, at);
  }
  static __device__ __forceinline__ int place_v(int row, int p) {
    if constexpr (D >= 128) return p ^ 4 * (row & 3);
    else if constexpr (D == 64) return p ^ 4 * (row >> 1 & 1);
    else return p;
  }
};

// The keys of a step start at a multiple of their number: pages of 64 tokens and more (kLarge) hold them all,
// smaller ones a multiple of 16 of them, so that addresses are a wave's own but for an offset of 32 bits.  Page numbers are
// asked for a step before the loads that need them.
template <class E, bool kFp8, bool kLarge, int kKeys, int D>
struct Stage {
  typedef typename E::T T;
  typedef typename E::V8 V8;
  typedef Staged<E, kKeys, D> Shared;
  static constexpr int kPer = kFp8 ? 16 : 8, kChunks = D / kPer, kLoads = (kKeys * kChunks + 255) / 256;
  static constexpr bool kWhole = kKeys * kChunks % 256 == 0, kOneGroup = 16 * kChunks % 64 == 0;
  static constexpr int kPages = kLarge ? 1 : kKeys / 16;
  static constexpr unsigned kAll = (1u << kKeys / 16) - 1;
  static constexpr int kRowBytes = kFp8 ? D : 2 * D, kScales = D / MX_SCALE_BLOCK;

  // what a step needs of the arguments, kept in registers
  Fixed* table;
  const uint8_t *k, *v, *k_scale, *v_scale;   // of this head in page 0
  unsigned page_bytes, scale_bytes;           // from page to page
  int page_shift, npage, end;
  int page[kPages];                           // of all keys, or of each 16 of them
  unsigned from_k[kLoads], from_v[kLoads];    // this thread's pieces, from the first key's row
  u4 kreg[kFp8 ? kLoads : 1], vreg[kFp8 ? kLoads : 1];
  unsigned kbyte[kFp8 ? kLoads : 1], vbyte[kFp8 ? kLoads : 1];

  __device__ __forceinline__ Stage(const Attend& a, int world, int head, int end)
      : table(fixed(a.table + (int64_t)world * a.width)), page_shift(a.page_shift), npage(a.npage), end(end) {
    const int64_t rows = (int64_t)head << page_shift;
    k = a.k + rows * kRowBytes;
    v = a.v + rows * kRowBytes;
    k_scale = a.k_scale + rows * kScales;
    v_scale = a.v_scale + rows * kScales;
    page_bytes = ((unsigned)a.kv_heads << page_shift) * kRowBytes;      // at most 1024 heads of 4096 tokens of 512 bytes
    scale_bytes = ((unsigned)a.kv_heads << page_shift) * kScales;
#pragma unroll
    for (int j = 0; j < kLoads; j++) {
      const int row = key_of(j), at = piece_of(j);
      from_k[j] = row * kRowBytes + (kFp8 ? at : Shared::piece_k(row, at)) * 16;
      from_v[j] = row * kRowBytes + (kFp8 ? at : Shared::place_v(row, at)) * 16;
    }
  }

  // Each thread has kLoads pieces of kPer values: of which key, and the how manieth of its row
  static __device__ __forceinline__ int key_of(int j) { return (j * 256 + (int)threadIdx.x) / kChunks; }
  static __device__ __forceinline__ int piece_of(int j) { return (j * 256 + (int)threadIdx.x) % kChunks; }
  static __device__ __forceinline__ int wave() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }
  __device__ __forceinline__ int first_of(int key, int g) const { return min(key + 16 * g, (end - 1) & ~15); }
  __device__ __forceinline__ void look_up(int key) {
#pragma unroll
    for (int g = 0; g < kPages; g++) page[g] = table[(kLarge ? key : first_of(key, g)) >> page_shift];
  }

  // The pages that are there, a bit for each 16 keys
  __device__ __forceinline__ unsigned present() const {
    unsigned bits = 0;
#pragma unroll
    for (int g = 0; g < kPages; g++) bits |= ((unsigned)page[g] < (unsigned)npage ? kLarge ? kAll : 1u : 0u) << g;
    return bits;
  }

  // From memory into LDS, a wave's 64 pieces one after the other from `to` on.  As the builtin, but for the
  // waits that the compiler would put before every LDS read that follows, whatever it reads: arrived() waits.
  // The place goes in as m0 itself (the compiler sets it), one wait state before its use.
  static __device__ __forceinline__ void into_lds(const uint8_t* base, unsigned offset, unsigned place) {
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"{m0}"(place), "v"(offset), "s"(base) : "memory");
  }
  static __device__ __forceinline__ void arrived() {
    if constexpr (!kFp8) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  }

  // `to`: the LDS address of the buffer; `first`: the key in page `in` that the offsets start from
  __device__ __forceinline__ void bring(unsigned to, int j, int in, int first, unsigned at_k, unsigned at_v, unsigned at_scale) {
    const unsigned page = (unsigned)in < (unsigned)npage ? in : 0, row = first & ((1 << page_shift) - 1);
    const uint64_t at = (uint64_t)page * page_bytes + row * (unsigned)kRowBytes;
    if constexpr (kFp8) {
      kreg[j] = *(const u4*)(k + at + at_k);
      vreg[j] = *(const u4*)(v + at + at_v);
      const uint64_t scale = (uint64_t)page * scale_bytes + row * (unsigned)kScales;
      kbyte[j] = (k_scale + scale)[at_scale];
      vbyte[j] = (v_scale + scale)[at_scale];
    } else {
      to += (j * 256 + 64 * wave()) * 16;
      into_lds(k + at, at_k, to + offsetof(Shared, k));
      into_lds(v + at, at_v, to + offsetof(Shared, v));
    }
  }

  // Starts the loads of the keys from `key` on; keys at and beyond `end` repeat the last one's address
  __device__ __forceinline__ void load(unsigned to, int key) {
    if (kLarge && key + kKeys <= end) {
#pragma unroll
      for (int j = 0; j < kLoads; j++)
        if (kWhole || key_of(j) < kKeys)
          bring(to, j, page[0], key, from_k[j], from_v[j], key_of(j) * kScales + piece_of(j) / 2);
      return;
    }
#pragma unroll
    for (int j = 0; j < kLoads; j++) {
      if (!kWhole && key_of(j) >= kKeys) continue;
      // rows beyond the last: that one's piece instead
      int in = page[0], first = key, row = min(key_of(j), end - 1 - key);
      if constexpr (!kLarge) {
        // the group of 16 keys: the wave's, or where a wave's pieces straddle two, the lane's
        const int group = kOneGroup ? (j * 256 + 64 * wave()) / (16 * kChunks) : key_of(j) / 16;
#pragma unroll
        for (int g = 1; g < kPages; g++) in = group == g ? page[g] : in;
        if constexpr (kOneGroup) in = __builtin_amdgcn_readfirstlane(in);
        first = first_of(key, group);
        row = min(key_of(j) % 16, end - 1 - first);
      }
      const unsigned back = (key_of(j) - row) * kRowBytes;
      bring(to, j, in, first, from_k[j] - back, from_v[j] - back, row * kScales + piece_of(j) / 2);
    }
  }

  // 8-bit pages: what load() brought into registers, converted, into LDS.  `careful`: see clean().
  __device__ __forceinline__ void store(Shared& to, int key, unsigned there, bool careful) {
    if constexpr (kFp8) {
      unsigned wild = 0;
#pragma unroll
      for (int j = 0; j < kLoads; j++) {
        if (!kWhole && key_of(j) >= kKeys) continue;
        const int row = key_of(j);
        const bool none = careful && (key + row >= end || !(there >> (row / 16) & 1));
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const int p = 2 * piece_of(j) + e;
          *(V8*)&to.k[row * D + Shared::place_k(row, p) * 8] =
              from_fp8<E>(e ? u2{kreg[j].z, kreg[j].w} : u2{kreg[j].x, kreg[j].y}, kbyte[j]);
          u4 v = __builtin_bit_cast(u4, from_fp8<E>(e ? u2{vreg[j].z, vreg[j].w} : u2{vreg[j].x, vreg[j].y}, vbyte[j]));
          if (careful) wild |= cleaned(v, none);
          *(u4*)&to.v[row * D + Shared::place_v(row, p) * 8] = v;
        }
      }
      if (careful) flag(to, wild);
    }
  }

  // Some of the keys are not there, or not seen by all rows: values of the former become zeros, and infinities and
  // NaN too (the rows that see them get them added, by add_wild()).  16-bit pages: in LDS, each thread what
  // it brought, after its loads are done and before a barrier.
  __device__ __forceinline__ void clean(Shared& to, int key, unsigned there) {
    unsigned wild = 0;
#pragma unroll
    for (int j = 0; j < kLoads; j++) {
      if (!kWhole && key_of(j) >= kKeys) continue;
      const int row = key_of(j);
      u4* at = (u4*)&to.v[(j * 256 + threadIdx.x) * 8];
      u4 v = *at;
      wild |= cleaned(v, key + row >= end || !(there >> (row / 16) & 1));
      *at = v;
    }
    flag(to, wild);
  }

  static __device__ __forceinline__ unsigned cleaned(u4& v, bool none) {
    unsigned wild = 0;
#pragma unroll
    for (int y = 0; y < 4; y++) {
      if (none) v[y] = 0;
      wild |= not_finite<E>(v[y]) & 0x80008000u;
      v[y] = finite_or_zero<E>(v[y]);
    }
    return wild;
  }
  __device__ __forceinline__ void flag(Shared& to, unsigned wild) const {
    const int any = __ballot(wild != 0) != 0;
    if ((threadIdx.x & 63) == 0) to.wild[threadIdx.x >> 6] = any;
  }

  // Values of the keys [key, stop) that are not finite, added to the output of a lane's row if it sees the key
  // (o in the layout of 32x32 products).  Sixteen keys, which lie in one page, are looked through together; it ends early
  // when all is NaN.  (A prompt with one NaN 5.4 ms key by key.)
  __device__ __forceinline__ void add_wild(int key, int stop, int low_r, int high_r, f16v (&o)[D / 32]) const {
    const int half = (threadIdx.x & 63) >> 5;
    for (; key < min(stop, end); key += 16) {
      const int in = table[key >> page_shift], keys = min(16, end - key);
      if ((unsigned)in >= (unsigned)npage) continue;
      const int row = key & ((1 << page_shift) - 1);
      const uint8_t* from = v + (uint64_t)in * page_bytes + row * (unsigned)kRowBytes;
      const uint8_t* scale = v_scale + (uint64_t)in * scale_bytes + row * (unsigned)kScales;
      if (!any_wild<E, kFp8>(from, scale, keys * kChunks)) continue;
      bool open = false;
      for (int j = 0; j < keys; j++) {
        const bool sees = key + j >= low_r && key + j < high_r;
#pragma unroll
        for (int c = 0; c < D / 32; c++)
#pragma unroll
          for (int i = 0; i < 16; i += 4) {
            const f4 x = values_at<E, kFp8>(from + j * kRowBytes, scale + j * kScales, 32 * c + 2 * i + 4 * half);
#pragma unroll
            for (int e = 0; e < 4; e++) o[c][i + e] += sees && !(fabsf(x[e]) < INFINITY) ? x[e] : 0.f;
          }
      }
#pragma unroll
      for (int c = 0; c < D / 32; c++)
#pragma unroll
        for (int i = 0; i < 16; i++) open |= o[c][i] == o[c][i];
      if (!__ballot(open && low_r < high_r)) return;
    }
  }
};

__device__ __forceinline__ float both_halves_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float both_halves_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Where the 32 rows of a wave end up: their parts, or the output.  o, m, l as the kernels keep them (m and l
// in powers of two; l of this lane's half of the keys).
template <class E, int D>
__device__ __forceinline__ void finish_row(const Attend& a, const Tile& t, int split, int token_in, int query_head, float m, float l,
                                  const f16v (&o)[D / 32]) {
  typedef typename E::T T;
  const int half = (threadIdx.x & 63) >> 5;
  l = both_halves_sum(l);
  if (a.splits > 1) {
    const int64_t at = (int64_t)split * a.part_rows + part_row(a, t, token_in, query_head);
    if (l != 0.f)
#pragma unroll
      for (int c = 0; c < D / 32; c++)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
          *(f4*)(a.part + at * D + 32 * c + 2 * i + 4 * half) = f4{o[c][i], o[c][i + 1], o[c][i + 2], o[c][i + 3]};
    if (half == 0) *(f2*)(a.part_ml + 2 * at) = f2{m, l};
    return;
  }
  const float inverse = 1.f / l;
  const int64_t token = t.token + token_in;
  T* to = (T*)a.out + token * a.o_token + (int64_t)query_head * a.o_head;
#pragma unroll
  for (int c = 0; c < D / 32; c++)
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
  if (a.lse && half == 0) a.lse[token * a.heads + query_head] = l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * kLn2;
}

// Blocks go to the XCDs in turn: where the key heads of all worlds divide among the eight, those of one
// stay on one XCD, whose L2 then holds their keys and values.  Last rows first: under a causal mask they
// have the most keys.
__device__ __forceinline__ void place(const Attend& a, int& split, int& head, int& tile) {
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

}  // namespace mxe
