// Attention of few rows: the kTeam waves of a workgroup each take 32 keys at a time of one world's key
// head, for up to 16 * kBlocks rows (new tokens times the query heads that share the key head).  kTeam is 4, or 1 for
// many short histories, in which most of four waves would have no keys (see choose()).
//
// One pass over the keys with a reference m, sum l and output O per row (in 32 bits):
//   S^T = K Q^T (scores of 32 keys in two products' results, a row of the chunk per lane column),
//   p = 2^(S - m), l = l + sum p, O^T = O^T + V^T P^T.
// The maximum is not looked for: the first step's stays the reference m until a lane's sum of a step passes
// 2^12, in float16 65504 (or is no number); then the step's maximum is found, l and O are rescaled and the step is weighed again (see
// Weights in mx_episode_types.h; 210 -> 205 us for
// the 4096 worlds below; attend_many, whose products run beside the powers of two, lost 2 % by it).
// With the scores transposed, a lane holds eight keys of its own row, which is the operand that the
// second product wants if its keys are numbered 4 q + (0..3), 16 + 4 q + (0..3) for lane quarter q; V's
// columns come in that order out of LDS by transposing reads, so probabilities never cross lanes.
// They enter the product as two 16-bit parts, value and remainder, which costs matrix instructions
// that a kernel bound by reading K and V has to spare, and keeps 16 bits of them in bfloat16 and up to 20 in float16, whose
// steps are never below 2^-24 (see Weights).
//
// Bound by memory, with a step's keys and values under way while the last one's are weighed: a wave reads keys as
// the first product's operand straight from memory (a key to a lane, 16 bytes at a time), values through
// LDS of its own without a barrier, and the waves' results are joined once.  What counts is how many
// waves a SIMD holds: keeping the values' words for the rare infinities below took 130 registers and three
// waves at 64 values a head, reading them again 120 and four (249 -> 216 us for 4096 worlds of up to
// 1024 quantised tokens).  Single tokens, alternating inputs: those worlds (4 key heads of 64, 1.13 GB) 205 us, 5.5 TB/s, its
// VALU 57 % busy with conversions and softmax; 500 worlds of up to 2048 tokens in bfloat16 (8 key heads of 128, 2.1 GB) 364 us, 5.8 TB/s;
// two worlds, 131072 quantised tokens in all (277 MB), 48 us and 5 to join the parts.
#pragma once
#include "mx_episode_types.h"

namespace mxe {

// Waves of a SIMD to leave registers for
constexpr int few_waves(int D, int blocks) { return blocks == 1 && D <= 64 ? 4 : blocks <= 2 && D <= 128 ? 2 : 1; }

// kListed: not over all keys of the world, but over those of the blocks that a token's list names (mx_episode_recall).  Keys
// are then counted along the list; 16 of them lie in one block, and are where its number says.
template <int kType, bool kFp8, int D, int kBlocks, int kTeam, bool kListed = false>
__global__ __launch_bounds__(64 * kTeam, few_waves(D, kBlocks)) void attend_few(const Attend a) {
  typedef Elem<kType> E;
  typedef typename E::T T;
  typedef typename E::V8 V8;
  constexpr int kRows = 16 * kBlocks, kC = D / 32;            // products along head_dim
  constexpr int kStride = D + 16;                             // V's row in LDS: transposing reads of 16 rows hit all banks once
  constexpr int kVPer = kFp8 ? 16 : 8, kVLoads = 32 * D / kVPer / 64;
  constexpr bool kTakeOut = !kFp8 || kType == MX_TYPE_F16;      // of every step, not only of those that some rows do not see
  constexpr int kPairs = kFp8 ? D / 64 : 0;                   // 8-bit keys: 16 bytes are the operands of two products
  constexpr int kOStride = D + 4, kStep = 32 * kTeam;
  __shared__ __attribute__((aligned(16))) union Shared {
    T v[kTeam][32 * kStride];
    float o[kTeam][16 * kOStride];
  } sh;
  __shared__ float sh_m[kTeam][kRows], sh_l[kTeam][kRows];

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int n16 = lane & 15, quarter = lane >> 4;
  unsigned block = blockIdx.x;
  const int split = block % a.splits;
  block /= a.splits;
  const int head = block % a.kv_heads, tile = block / a.kv_heads;
  Tile t;
  if (!(kListed ? find_listed_tile(a, tile, kRows, t) : find_tile(a, tile, kRows, t))) return;

  // keys that any row of the tile sees, and keys that all its rows see
  const int last_row = min(t.row + kRows, t.rows) - 1;
  int first_low, first_high, last_low, last_high;
  limits(a, t, t.row / a.group, first_low, first_high);
  limits(a, t, last_row / a.group, last_low, last_high);
  const int all_low = last_low, all_high = first_high;
  int begin, end;
  Fixed* table = fixed(a.table + (int64_t)t.world * a.width);
  // listed blocks: the lanes hold 64 entries of the list and their pages (-1: none), so that a step finds its keys without a
  // load (72 us instead of 73 for 1024 worlds' 11 blocks of 64 8-bit tokens)
  int list_block = -1, list_page = -1, list_held = 0;
  const auto hold = [&](int group) {
    const int32_t* list = a.blocks + ((int64_t)(t.token + t.row / a.group) * a.kv_heads + head) * a.lists;
    const int entry = 64 * group + lane;
    list_block = entry < a.lists ? list[entry] : -1;
    if ((unsigned)list_block >= (unsigned)a.width << (a.page_shift - a.block_shift)) list_block = -1;
    const int page = a.table[(int64_t)t.world * a.width + (max(list_block, 0) >> (a.page_shift - a.block_shift))];
    list_page = list_block >= 0 && (unsigned)page < (unsigned)a.npage ? page : -1;
    list_held = group;
  };
  if constexpr (kListed) {
    int named = 0;                                            // up to the last entry that names a block
    for (int group = (a.lists - 1) >> 6; group >= 0 && !named; group--) {
      hold(group);
      const uint64_t names = __ballot(list_block >= 0);
      if (names) named = 64 * group + 64 - __builtin_clzll(names);
    }
    split_range(a, split, 0, last_high > 0 ? named << a.block_shift : 0, begin, end);
  } else {
    split_range(a, split, first_low, last_high, begin, end);
  }

  // this lane's rows
  int low_r[kBlocks], high_r[kBlocks];
  V8 q[kBlocks][kC];
#pragma unroll
  for (int b = 0; b < kBlocks; b++) {
    const int r = t.row + 16 * b + n16;
    const bool is = r < t.rows;
    const int i = (is ? r : t.row) / a.group, h = (is ? r : t.row) - i * a.group;
    limits(a, t, i, low_r[b], high_r[b]);
    if (!is) high_r[b] = 0;
    const T* from = (const T*)a.q + (int64_t)(t.token + i) * a.q_token + (int64_t)(head * a.group + h) * a.q_head;
#pragma unroll
    for (int c = 0; c < kC; c++) {
      const int d = c < 2 * kPairs ? 64 * (c / 2) + 16 * quarter + 8 * (c & 1) : 32 * c + 8 * quarter;
      q[b][c] = load_query<E>(a, from + d);
    }
  }

  f4 o[kBlocks][D / 16];
  float m[kBlocks], l[kBlocks];
#pragma unroll
  for (int b = 0; b < kBlocks; b++) {
    m[b] = t.row + 16 * b + n16 < t.rows ? -INFINITY : 0.f;
    l[b] = 0.f;
#pragma unroll
    for (int c = 0; c < D / 16; c++) o[b][c] = f4{0.f, 0.f, 0.f, 0.f};
  }

  const int page_mask = (1 << a.page_shift) - 1;

  // The 16 keys from `key` on lie in one page: its number, or 0 with the keys marked absent
  struct Keys {
    int64_t at;           // first key's element / D
    int left;             // keys up to `end`, less one (lanes beyond repeat the last)
    int first;            // number of the first key in its world
    bool is;
  };
  auto locate = [&](int key) {
    Keys s;
    int from = min(key, (end - 1) & ~15), page;
    s.left = end - 1 - from;
    if constexpr (kListed) {
      const int entry = from >> a.block_shift;
      if (entry >> 6 != list_held) hold(entry >> 6);
      const int block = __builtin_amdgcn_readlane(list_block, entry & 63);
      page = __builtin_amdgcn_readlane(list_page, entry & 63);
      from = (max(block, 0) << a.block_shift) + (from & ((1 << a.block_shift) - 1));
      s.is = key < end && page >= 0 && from < last_high;
    } else {
      page = table[from >> a.page_shift];
      s.is = (unsigned)page < (unsigned)a.npage;
    }
    s.first = from;
    s.at = (((int64_t)(s.is ? page : 0) * a.kv_heads + head) << a.page_shift) + (from & page_mask);
    return s;
  };

  u4 kreg[2][kFp8 ? kPairs + 1 : kC];
  unsigned kbyte[2][kFp8 ? kPairs + 1 : 1];
  u4 vreg[kVLoads];
  unsigned vbyte[kFp8 ? kVLoads : 1];
  Keys keys[2];

  auto load = [&](int key) {
    keys[0] = locate(key);
    keys[1] = locate(key + 16);
#pragma unroll
    for (int s = 0; s < 2; s++) {
      const int64_t at = keys[s].at + min(n16, keys[s].left);
      if constexpr (kFp8) {
        const uint8_t* from = a.k + at * D;
        const uint8_t* scale = a.k_scale + at * kC;
#pragma unroll
        for (int c = 0; c < kPairs; c++) {
          kreg[s][c] = *(const u4*)(from + 64 * c + 16 * quarter);
          kbyte[s][c] = scale[2 * c + (quarter >> 1)];
        }
        if constexpr (kC & 1) {
          const u2 w = *(const u2*)(from + 32 * (kC - 1) + 8 * quarter);
          kreg[s][kPairs] = u4{w.x, w.y, 0, 0};
          kbyte[s][kPairs] = scale[kC - 1];
        }
      } else {
        const T* from = (const T*)a.k + at * D;
#pragma unroll
        for (int c = 0; c < kC; c++) kreg[s][c] = *(const u4*)(from + 32 * c + 8 * quarter);
      }
    }
#pragma unroll
    for (int j = 0; j < kVLoads; j++) {
      const int x = j * 64 + lane, key_in = x / (D / kVPer), d = (x - key_in * (D / kVPer)) * kVPer;
      const int64_t at = key_in < 16 ? keys[0].at + min(key_in, keys[0].left) : keys[1].at + min(key_in - 16, keys[1].left);
      if constexpr (kFp8) {
        vreg[j] = *(const u4*)(a.v + at * D + d);
        vbyte[j] = a.v_scale[at * kC + d / 32];
      } else {
        vreg[j] = *(const u4*)((const T*)a.v + at * D + d);
      }
    }
  };

  T* vs = sh.v[wave];
  typedef __attribute__((address_space(3))) s4* TrPtr;
  int key = begin + 32 * wave;
  int wild_from = end, wild_to = begin;       // steps whose values that are not finite were taken out
  if (key < end) load(key);
  for (; key < end; key += kStep) {
    // scores
    f4 s[kBlocks][2];
    const bool is0 = keys[0].is, is1 = keys[1].is;
    const int at0 = kListed ? keys[0].first : key, at1 = kListed ? keys[1].first : key + 16;   // keys' numbers
#pragma unroll
    for (int b = 0; b < kBlocks; b++) s[b][0] = s[b][1] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < 2; u++) {
#pragma unroll
      for (int c = 0; c < kC; c++) {
        V8 x;
        if constexpr (kFp8) {
          if (c < 2 * kPairs) {
            const u4 w = kreg[u][c / 2];
            x = from_fp8<E>(c & 1 ? u2{w.z, w.w} : u2{w.x, w.y}, kbyte[u][c / 2]);
          } else {
            x = from_fp8<E>(u2{kreg[u][kPairs].x, kreg[u][kPairs].y}, kbyte[u][kPairs]);
          }
        } else {
          x = __builtin_bit_cast(V8, kreg[u][c]);
        }
#pragma unroll
        for (int b = 0; b < kBlocks; b++) s[b][u] = E::mfma16(x, q[b][c], s[b][u]);
      }
    }
    // values into LDS, those of keys that do not exist as zeros
    const bool edge = kListed ? at0 + 16 > all_high || at1 + 16 > all_high || !is0 || !is1
                              : key < all_low || key + 32 > all_high || key + 32 > end || !is0 || !is1;
    // an infinity or NaN among the values: taken out, and added after the loop to the rows that see it (a remainder of a
    // probability times an infinity is no remainder).  8-bit values have no infinity in bfloat16 but in blocks of
    // the largest scales (in float16 beyond 65504): there the steps that all rows see leave them in, to be found
    // in the outputs (4096 worlds: 206 us; 210 with a look at each scale).
    unsigned wild = 0;
#pragma unroll
    for (int j = 0; j < kVLoads; j++) {
      const int x = j * 64 + lane, key_in = x / (D / kVPer), d = (x - key_in * (D / kVPer)) * kVPer;
      V8 v[kVPer / 8];
      if constexpr (kFp8) {
        v[0] = from_fp8<E>(u2{vreg[j].x, vreg[j].y}, vbyte[j]);
        v[1] = from_fp8<E>(u2{vreg[j].z, vreg[j].w}, vbyte[j]);
      } else {
        v[0] = __builtin_bit_cast(V8, vreg[j]);
      }
#pragma unroll
      for (int e = 0; e < kVPer / 8; e++) {
        u4 words = __builtin_bit_cast(u4, v[e]);
        const bool beyond = kListed ? (key_in < 16 ? at0 + key_in : at1 + key_in - 16) >= last_high : key + key_in >= end;
        if (edge && (beyond || !(key_in < 16 ? is0 : is1))) words = u4{0, 0, 0, 0};
        if (kTakeOut || edge) {
          unsigned off = 0;
#pragma unroll
          for (int y = 0; y < 4; y++) off |= not_finite<E>(words[y]);
          off &= 0x80008000u;
          if (off)
#pragma unroll
            for (int y = 0; y < 4; y++) words[y] = finite_or_zero<E>(words[y]);
          wild |= off;
        }
        *(u4*)(vs + key_in * kStride + d + 8 * e) = words;
      }
    }
    const bool repair = __ballot(wild != 0) != 0;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    // the next keys are on their way while these are weighed
    const int now = key;
    if (key + kStep < end) load(key + kStep);

    V8 p_high[kBlocks], p_low[kBlocks];
#pragma unroll
    for (int b = 0; b < kBlocks; b++) {
      if (edge) {
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const int at = (kListed ? (u ? at1 : at0) : now + 16 * u) + 4 * quarter + i;
            if (!(at >= low_r[b] && at < high_r[b] && (kListed || at < end) && (u ? is1 : is0))) s[b][u][i] = -INFINITY;
          }
      }
      float sum;
      const auto weigh = [&](float reference) __attribute__((always_inline)) {
        sum = 0.f;
#pragma unroll
        for (int j = 0; j < 8; j++) {
          const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][j / 4][j % 4], a.scale2, -reference));
          sum += p;
          const T h = (T)p;
          p_high[b][j] = h;
          p_low[b][j] = (T)(p - (float)h);
        }
      };
      weigh(m[b]);
      if (__ballot(!(sum <= E::kSumHolds))) {      // a new reference
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < 8; j++) top = fmaxf(top, s[b][j / 4][j % 4]);
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const float before = m[b];
        m[b] = fmaxf(m[b], top * a.scale2 - E::kTop);
        const float next = m[b] == -INFINITY ? 0.f : m[b], shrink = __builtin_amdgcn_exp2f(before - next);
        l[b] *= shrink;
#pragma unroll
        for (int c = 0; c < D / 16; c++) o[b][c] *= shrink;
        weigh(next);
      }
      l[b] += sum;
    }
#pragma unroll
    for (int c = 0; c < D / 16; c++) {
      const T* at = vs + (4 * quarter + (n16 >> 2)) * kStride + 16 * c + 4 * (n16 & 3);
      const s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((TrPtr)at);
      const s4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((TrPtr)(at + 16 * kStride));
      const V8 vt = __builtin_bit_cast(V8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
      for (int b = 0; b < kBlocks; b++) {
        o[b][c] = E::mfma16(vt, p_high[b], o[b][c]);
        o[b][c] = E::mfma16(vt, p_low[b], o[b][c]);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (repair) {
      wild_from = min(wild_from, now);
      wild_to = now + 32;
    }
  }

  // join the waves, 16 rows at a time
#pragma unroll
  for (int b = 0; b < kBlocks; b++) {
    l[b] += __shfl_xor(l[b], 16);
    l[b] += __shfl_xor(l[b], 32);
    if (quarter == 0) {
      sh_m[wave][16 * b + n16] = m[b];
      sh_l[wave][16 * b + n16] = l[b];
    }
  }
  if constexpr (!kTakeOut) {
    // left in, it may have met a weight of 0 or a remainder of the other sign: then the sum is made anew
    bool left = false;
#pragma unroll
    for (int b = 0; b < kBlocks; b++) {
      float off = 0.f;
#pragma unroll
      for (int c = 0; c < D / 16; c++)
#pragma unroll
        for (int i = 0; i < 4; i++) off = __builtin_fmaf(o[b][c][i], 0.f, off);
      left |= off != off && l[b] == l[b];             // and not because of the scores
    }
    if (__ballot(left)) {
#pragma unroll
      for (int b = 0; b < kBlocks; b++)
#pragma unroll
        for (int c = 0; c < D / 16; c++)
#pragma unroll
          for (int i = 0; i < 4; i++) o[b][c][i] = set_aside(o[b][c][i]);
      wild_from = begin + 32 * wave;
      wild_to = end;
    }
  }
  // the values that were taken out, added to the rows that see them; 16 keys are looked through together
  const bool wild_out = wild_from < wild_to;      // rare
  for (key = wild_from; key < wild_to; key += kStep)
    for (int first = key; first < min(key + 32, end); first += 16) {     // 16 keys lie in one page
      const Keys at = locate(first);
      const uint8_t *from = a.v + at.at * (kFp8 ? D : 2 * D), *scale = a.v_scale + at.at * kC;
      const int keys = min(16, kListed ? last_high - at.first : end - first);
      if (!at.is || !any_wild<E, kFp8>(from, scale, keys * (D / kVPer))) continue;
      for (int j = 0; j < keys; j++)
#pragma unroll
        for (int c = 0; c < D / 16; c++) {
          const f4 x = values_at<E, kFp8>(from + j * (kFp8 ? D : 2 * D), scale + j * kC, 16 * c + 4 * quarter);
#pragma unroll
          for (int b = 0; b < kBlocks; b++) {
            const int number = (kListed ? at.first : first) + j;
            const bool sees = number >= low_r[b] && number < high_r[b];
#pragma unroll
            for (int i = 0; i < 4; i++) o[b][c][i] += sees && !(fabsf(x[i]) < INFINITY) ? x[i] : 0.f;
          }
        }
      bool open = false;                               // until all is NaN
#pragma unroll
      for (int b = 0; b < kBlocks; b++)
#pragma unroll
        for (int c = 0; c < D / 16; c++)
#pragma unroll
          for (int i = 0; i < 4; i++) open |= o[b][c][i] == o[b][c][i] && low_r[b] < high_r[b];
      if (!__ballot(open)) wild_to = first;
    }
  if (wild_out)
#pragma unroll
    for (int b = 0; b < kBlocks; b++)
#pragma unroll
      for (int c = 0; c < D / 16; c++)
#pragma unroll
        for (int i = 0; i < 4; i++) o[b][c][i] = brought_back(o[b][c][i]);
#pragma unroll
  for (int b = 0; b < kBlocks; b++) {
    __syncthreads();
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kTeam; w++) top = fmaxf(top, sh_m[w][16 * b + n16]);
    if (top == -INFINITY) top = 0.f;
    const float shrink = __builtin_amdgcn_exp2f(m[b] - top);
#pragma unroll
    for (int c = 0; c < D / 16; c++)
      *(f4*)&sh.o[wave][n16 * kOStride + 16 * c + 4 * quarter] = wild_out ? rescaled(o[b][c], shrink) : o[b][c] * shrink;
    __syncthreads();
    for (int x = threadIdx.x; x < 16 * (D / 4); x += 64 * kTeam) {
      const int row = x / (D / 4), d = (x - row * (D / 4)) * 4, r = t.row + 16 * b + row;
      if (r >= t.rows) continue;
      f4 sum = f4{0.f, 0.f, 0.f, 0.f};
      float most = -INFINITY, total = 0.f;
#pragma unroll
      for (int w = 0; w < kTeam; w++) most = fmaxf(most, sh_m[w][16 * b + row]);
#pragma unroll
      for (int w = 0; w < kTeam; w++) {
        sum += *(const f4*)&sh.o[w][row * kOStride + d];
        total += sh_l[w][16 * b + row] * __builtin_amdgcn_exp2f(sh_m[w][16 * b + row] - (most == -INFINITY ? 0.f : most));
      }
      const int i = r / a.group, h = head * a.group + (r - i * a.group);
      const int64_t row_at = (int64_t)(t.token + i) * a.heads + h;
      if (a.splits > 1) {
        const int64_t at = (int64_t)split * a.part_rows + part_row(a, t, i, h);
        if (total != 0.f) *(f4*)(a.part + at * D + d) = sum;
        if (d == 0) *(f2*)(a.part_ml + 2 * at) = f2{most, total};
      } else {
        const float inverse = 1.f / total;
        T* to = (T*)a.out + (int64_t)(t.token + i) * a.o_token + (int64_t)h * a.o_head + d;
#pragma unroll
        for (int e = 0; e < 4; e++) to[e] = (T)(total == 0.f ? 0.f : sum[e] * inverse);
        if (a.lse && d == 0) a.lse[row_at] = total == 0.f ? -INFINITY : (most + __builtin_amdgcn_logf(total)) * kLn2;
      }
    }
  }
}

}  // namespace mxe
