// Attention of many rows: a workgroup takes 128 rows of one world's key head (new tokens times the query
// heads that share the key head), each of its four waves 32 of them, and 64 keys at a time (32 of 256 values), which all four
// read from LDS.  The mathematics is that of attend_few (one pass, running maximum, scores transposed so
// that probabilities stay in their lanes), with 32x32 products and one 16-bit part of each probability:
// here the matrix instructions are part of what bounds the kernel, and a second product for the remainders would add
// half of them again.  The rounding of the probabilities (2^-9 of each in bfloat16, 2^-12 in float16, at random) is of the size
// of the result's own: against 64 bits the error is 1.3 times that of exact probabilities on a prompt, 1.4 times in a window of 2000
// (0.0021 and 0.0016 of the norm, 0.0023 and 0.0017; float16 2.7e-4 and 2.1e-4).
//
// The reference follows the scores only when one passes it by more than 2^8, in float16 2^15.9 (see Weights in
// mx_episode_types.h): until then the sums are exact multiples of what they would be, and the output need not be rescaled.
//
// An infinity or NaN among the values: steps that not all rows see take it out, and after the loop it is added to the rows
// that see it.  The other steps multiply it, which gives the same unless its weight is 0 in 16 bits, or a later
// rescale 0 in 32; so where there are outputs that are not finite, those are made anew from all values.
//
// Two buffers: the next keys and values are on their way while these are weighed, one barrier a step.  Two
// waves per SIMD (three up to 96 values a head, where that took 300 ragged chunks from 52 to 47 us,
// but not for 96 in 8-bit pages, whose conversions then spill: 126 chunks 394 and 201 us, now 196), of
// two workgroups, so that one's products run beside the other's softmax.
// A prompt of 4 x 4096 tokens, 32 heads on 8 of 128 values, bfloat16: 560 us, 980 TFLOP/s (554 to 613 on cards at other
// clocks), matrix instructions 49 % and VALU 49 % busy; on a card at 554 to 566, in copies of the kernel without the softmax's VALU
// work 501 to 507, without the loads 490 to 495, without reading keys and values from LDS 454, with the matrix instructions alone
// 313: no one of them bounds it.  (With the scan for values that are not finite inside the loop 20 to 30 us more: the
// compiler kept its addresses in scalar registers that it then spilled.)
// Tried and not kept, beside a kernel of 597: 64 rows to a wave (the compiler moves the outputs between the two halves of the register
// file at every branch, 1100 us; heads of 64 values hold them, and fewer workgroups run side by side: 8 x 4096 tokens 342 to 354,
// 300 x 150 tokens 120 to 143, the window below 102 to 93), 32 keys a step (700), eight waves to a workgroup (612), a wave's priority raised
// around its products (591 to 615), reads of keys grouped ahead of the products (-1 %), the next step's scores
// computed beside this one's softmax (650), the reference kept without a maximum (617).
// 300 ragged chunks of up to 41 tokens over up to 701, 12 heads on 4 of 96 values, float16 (161 MB): 52 us; the loads alone
// 47, the rest alone 39, neither 21: what a workgroup waits for until its first keys are there, and that in two rounds of
// workgroups (queries asked for after the first keys 55.6 instead of 57.4 before, but 59.3 instead of 58.5 in heads of 128; rows dealt to
// other waves by block, the same).
// 16 worlds' 512 tokens over a window of 2000 in 8-bit pages, 16 heads on 2 of 64 values: 98 us, 610 TFLOP/s; a
// head of 64 values has half the products to each power of two, and the VALU is 62 % busy.  With pages of 16 or 32 tokens
// 121: heads of 32 and 64 values then keep their page numbers in scratch memory (160 bytes a lane), as the compiler indexes
// them at run time (heads of 128: 158 and 164).
// Heads of 256 values: the outputs and queries of 32 rows are 192 registers, so one wave per SIMD, whose
// products nothing runs beside, and which moves values between the halves of the register file: 4 x 2048 tokens, 16 heads on 4,
// bfloat16: 233 us, 590 TFLOP/s (64 keys a step, as many rows as attend_few takes at a time: 397 and 915, beside 295 then).
#pragma once
#include "mx_episode_launch.h"
#include "mx_episode_stage.h"

namespace mxe {

// Keys of a step
constexpr int many_keys(int D) { return D <= 128 ? 64 : 32; }
constexpr int many_waves(int D, bool fp8) { return D <= 32 ? 4 : D <= (fp8 ? 64 : 96) ? 3 : D <= 128 ? 2 : 1; }

template <int kType, bool kFp8, bool kLarge, int D>
__global__ __launch_bounds__(256, many_waves(D, kFp8)) void attend_many(const Attend) {
  const Attend& a = arguments();
  typedef Elem<kType> E;
  typedef typename E::T T;
  typedef typename E::V8 V8;
  constexpr int kKeys = many_keys(D), kC = D / 16, kTiles = D / 32, kU = kKeys / 32;
  typedef Staged<E, kKeys, D> Shared;
  typedef Stage<E, kFp8, kLarge, kKeys, D> Bring;
  constexpr unsigned kAll = Bring::kAll;
  __shared__ __attribute__((aligned(1024))) Shared sh[2];

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int n32 = lane & 31, half = lane >> 5;
  int split, head, tile;
  place(a, split, head, tile);
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

  const float scale2 = a.scale2;
  Bring stage(a, t.world, head, end);
  // keys that are not there, or that only some rows of the workgroup see
  const auto careful = [&](int key, unsigned there) {
    return key < last_low || key + kKeys > first_high || there != kAll || key + kKeys > end;
  };
  // where this lane reads: a key's pieces, and for V^T the four keys and 4 of 16 values of its 16 lanes
  int from_k[kC], from_v[kTiles];
#pragma unroll
  for (int c = 0; c < kC; c++) from_k[c] = n32 * D + Shared::place_k(n32, 2 * c + half) * 8;
  const int v_row = 4 * half + ((lane & 15) >> 2), v_piece = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
#pragma unroll
  for (int c = 0; c < kTiles; c++) from_v[c] = v_row * D + Shared::place_v(v_row, 4 * c + v_piece) * 8 + 4 * (lane & 1);

  typedef __attribute__((address_space(3))) s4* TrPtr;
  typedef __attribute__((address_space(3))) Shared* LocalPtr;
  const unsigned at_lds = (unsigned)(uintptr_t)(LocalPtr)&sh[0];
  int key = begin, buffer = 0, wild_from = end, wild_to = begin;       // steps whose values that are not finite were taken out
  unsigned present = 0;
  if (key < end) {
    stage.look_up(key);
    stage.load(at_lds, key);
    present = stage.present();
    if (key + kKeys < end) stage.look_up(key + kKeys);
    stage.store(sh[0], key, present, careful(key, present));
  }
  for (; key < end; key += kKeys, buffer ^= 1) {
    const bool more = key + kKeys < end, mind = careful(key, present);
    stage.arrived();
    if (!kFp8 && mind) stage.clean(sh[buffer], key, present);
    __syncthreads();
    unsigned next_present = 0;
    if (more) {
      stage.load(at_lds + (buffer ? 0 : (unsigned)sizeof(Shared)), key + kKeys);
      next_present = stage.present();
      if (key + 2 * kKeys < end) stage.look_up(key + 2 * kKeys);
    }
    if (rows_here && key < wave_high && key + kKeys > wave_low) {
      const T *ks = sh[buffer].k, *vs = sh[buffer].v;
      f16v s[kU];
#pragma unroll
      for (int u = 0; u < kU; u++) {
#pragma unroll
        for (int i = 0; i < 16; i++) s[u][i] = 0.f;
#pragma unroll
        for (int c = 0; c < kC; c++) s[u] = E::mfma32(*(const V8*)(ks + from_k[c] + 32 * u * D), q[c], s[u]);
      }
      if (mind && (key < wave_all_low || key + kKeys > wave_all_high || present != kAll || key + kKeys > end)) {
#pragma unroll
        for (int u = 0; u < kU; u++)
#pragma unroll
          for (int i = 0; i < 16; i++) {
            const int at = key + 32 * u + 8 * (i / 4) + 4 * half + i % 4;
            if (!((present >> (2 * u + i / 8) & 1) && at >= low_r && at < high_r && at < end)) s[u][i] = -INFINITY;
          }
      }
      float top = -INFINITY;
#pragma unroll
      for (int u = 0; u < kU; u++)
#pragma unroll
        for (int i = 0; i < 16; i++) top = fmaxf(top, s[u][i]);
      top = both_halves_max(top) * scale2;
      if (__ballot(top > m + E::kHolds)) {
        const float next = fmaxf(m, top - E::kTop), shrink = __builtin_amdgcn_exp2f(m - (next == -INFINITY ? 0.f : next));
        m = next;
        l *= shrink;
#pragma unroll
        for (int c = 0; c < kTiles; c++) o[c] *= shrink;
      }
      const float zero = m == -INFINITY ? 0.f : m;
      V8 p[kU][2];
      float sum[2] = {0.f, 0.f};
#pragma unroll
      for (int u = 0; u < kU; u++)
#pragma unroll
        for (int i = 0; i < 16; i++) {
          const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][i], scale2, -zero));
          sum[i & 1] += x;
          p[u][i / 8][i % 8] = (T)x;
        }
      l += sum[0] + sum[1];
#pragma unroll
      for (int u = 0; u < kU; u++)
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
          for (int c = 0; c < kTiles; c++) {
            const T* at = vs + from_v[c] + (32 * u + 16 * b) * D;
            const s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((TrPtr)at);
            const s4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((TrPtr)(at + 8 * D));
            o[c] = E::mfma32(__builtin_bit_cast(V8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7)), p[u][b], o[c]);
          }
      if (mind && (sh[buffer].wild[0] | sh[buffer].wild[1] | sh[buffer].wild[2] | sh[buffer].wild[3])) {
        wild_from = min(wild_from, key);
        wild_to = key + kKeys;
      }
    }
    if (more) stage.store(sh[buffer ^ 1], key + kKeys, next_present, careful(key + kKeys, next_present));
    present = next_present;
  }

  const float sum = both_halves_sum(l);
  float off = 0.f;
#pragma unroll
  for (int c = 0; c < kTiles; c++)
#pragma unroll
    for (int i = 0; i < 16; i++) off = __builtin_fmaf(o[c][i], 0.f, off);
  if (__ballot(off != off && sum == sum)) {           // not because of the scores: left in
#pragma unroll
    for (int c = 0; c < kTiles; c++)
#pragma unroll
      for (int i = 0; i < 16; i++) o[c][i] = set_aside(o[c][i]);
    wild_from = begin;
    wild_to = end;
  }
  if (wild_from < wild_to) {
    stage.add_wild(wild_from, wild_to, low_r, high_r, o);
#pragma unroll
    for (int c = 0; c < kTiles; c++)
#pragma unroll
      for (int i = 0; i < 16; i++) o[c][i] = brought_back(o[c][i]);
  }
  if (row_here) finish_row<E, D>(a, t, split, token_in, query_head, m, l, o);
}

}  // namespace mxe
