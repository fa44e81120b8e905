// Recall: the summaries of blocks of keys, the choice of blocks for each query, and the host side of the attention over
// the chosen ones (attend_few with kListed, mx_episode_few.h).
//
// A summary is the mean of a block's keys in 8-bit whole numbers with a power of two, and queries are taken the same way,
// so that a score is a product of whole numbers: exact, whatever the order of its sum, and the choice between two blocks
// is the same on any machine.  It costs one byte to a value, a 2 block_tokens-th of the block's keys in 16 bits.
#include <type_traits>
#include "mx_episode_move.h"
#include "mx_episode_launch.h"

namespace mxe {

typedef int i4 __attribute__((ext_vector_type(4)));

constexpr int kMostCode = 127, kMostPower = 40, kNoNumber = 255;

// The least power of two, from 2^-40 to 2^40, at which the codes of values up to `most` do not pass 127
__device__ inline int power_of(double most) {
  int e;
  const double fraction = frexp(most, &e);                 // most = fraction 2^e, 1/2 <= fraction < 1
  if (!(most > 0.0)) return -kMostPower;
  if (!(most < INFINITY)) return kMostPower;
  return min(max(e - 7 + (fraction > kMostCode / 128.0 ? 1 : 0), -kMostPower), kMostPower);
}

__device__ inline int power_of(float most) {               // most >= 0, its fraction and exponent as bits
  const unsigned bits = __float_as_uint(most);
  return min(max((int)(bits >> 23) - 126 - 7 + ((bits & 0x7fffffu) > 0x7e0000u ? 1 : 0), -kMostPower), kMostPower);
}

// ---------------------------------------------------------------------------- summaries
struct Summarise {
  const uint8_t *k, *k_scale;
  const int32_t *table, *length, *start;
  int8_t* codes;
  uint8_t* exponent;
  int nworld, npage, width, kv_heads, page_shift, block_shift, tokens, count, per;   // per: blocks of a world's chunk at most
};

// A workgroup takes a block and a wave its heads in turn (2048 tokens' 32 blocks, 8 heads of 128 values: 9.5 us; a step
// in which few of 1024 worlds complete one: 4.7): lanes side by side along a key, as many keys as fit beside each
// other, sums in 64 bits joined through LDS.  World w of ragged chunks has the items from start[w] / block_tokens + w
// on.
template <int kStore, int D>
__global__ __launch_bounds__(256) void summarise_blocks(const Summarise a) {
  constexpr int kAcross = D / 8, kDown = 64 / kAcross, kPer = (D + 63) / 64;
  __shared__ double sh[4][kDown][D];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  int world, j, count;
  if (!a.start) {
    world = blockIdx.x / a.per;
    j = blockIdx.x - world * a.per;
    count = a.count;
  } else {
    const int item = blockIdx.x;
    int low = 0, high = a.nworld;
    while (high - low > 1) {
      const int step = (high - low + 63) >> 6, probe = low + lane * step;
      const bool below = probe < high && (max(a.start[probe], 0) >> a.block_shift) + (long long)probe <= item;
      const int passed = max(1, (int)__popcll(__ballot(below)));
      low += (passed - 1) * step;
      high = min(high, low + step);
    }
    world = __builtin_amdgcn_readfirstlane(low);
    const int begin = a.start[world];
    count = a.start[world + 1] - begin;
    j = (int)(item - (begin >> a.block_shift) - (long long)world);
    if (begin < 0 || j < 0) return;
  }
  if (count < 1 || j > (count - 1) >> a.block_shift) return;
  const int length = max(a.length[world], 0);
  const long long block = (max(length - count, 0) >> a.block_shift) + (long long)j;
  if ((block + 1) << a.block_shift > min((long long)length, (long long)a.width << a.page_shift)) return;
  const long long token = block << a.block_shift;
  const int page = a.table[(int64_t)world * a.width + (token >> a.page_shift)];
  if ((unsigned)page >= (unsigned)a.npage) return;
  const int inside = (int)(token & ((1 << a.page_shift) - 1));

  const int down = lane / kAcross, across = lane - down * kAcross;
  const bool takes = down < kDown;
  for (int head = wave; head < a.kv_heads; head += 4) {
    const int64_t first = (((int64_t)page * a.kv_heads + head) << a.page_shift) + inside;
    double sum[8];
#pragma unroll
    for (int i = 0; i < 8; i++) sum[i] = 0.0;
    if (takes)
#pragma unroll 4
      for (int t = down; t < 1 << a.block_shift; t += kDown) {
        const int64_t at = (first + t) * D + 8 * across;
        float x[8];
        if constexpr (kStore == MX_TYPE_FP8) {
          const u2 w = *(const u2*)(a.k + at);
          const float scale = scale_of(a.k_scale[at / MX_SCALE_BLOCK]);
#pragma unroll
          for (int i = 0; i < 2; i++) {
            const f2 p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w[i], scale, false);
            const f2 q = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w[i], scale, true);
            x[4 * i] = p[0];
            x[4 * i + 1] = p[1];
            x[4 * i + 2] = q[0];
            x[4 * i + 3] = q[1];
          }
        } else {
          const auto w = *(const typename Elem<kStore>::V8*)((const typename Elem<kStore>::T*)a.k + at);
#pragma unroll
          for (int i = 0; i < 8; i++) x[i] = (float)w[i];
        }
#pragma unroll
        for (int i = 0; i < 8; i++) sum[i] += (double)x[i];
      }
    if (takes)
#pragma unroll
      for (int i = 0; i < 8; i++) sh[wave][down][8 * across + i] = sum[i];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    double mean[kPer], most = 0.0;
    bool finite = true;
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      const int d = lane + 64 * i;
      double x = 0.0;
      if (d < D)
        for (int r = 0; r < kDown; r++) x += sh[wave][r][d];
      mean[i] = ldexp(x, -a.block_shift);
      finite = finite && fabs(x) < INFINITY;
      most = fmax(most, fabs(mean[i]));
    }
    finite = __ballot(!finite) == 0;
#pragma unroll
    for (int x = 1; x < 64; x *= 2) most = fmax(most, __shfl_xor(most, x));
    const int e = power_of(most);
    const int64_t entry = first >> a.block_shift;             // blocks do not cross pages
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      const int d = lane + 64 * i;
      const double code = fmin(fmax(__builtin_rint(ldexp(mean[i], -e)), -(double)kMostCode), (double)kMostCode);
      if (d < D) a.codes[entry * D + d] = finite ? (int8_t)code : 0;
    }
    if (lane == 0) a.exponent[entry] = finite ? (uint8_t)(e + 127) : kNoNumber;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

// ---------------------------------------------------------------------------- selection
struct Select {
  const int32_t *table, *length, *start;
  const void* q;
  const int8_t* codes;
  const uint8_t* exponent;
  int32_t* blocks;
  int64_t q_token, q_head;
  int nworld, npage, width, kv_heads, page_shift, block_shift, tokens, count, max_count, group;
  int lists, top, near, first;
  int units, tile;               // tiles of `tile` rows, times key heads
  int pieces;                    // of 64 scores that a token has room for in LDS
  bool causal, q_vector;
};

constexpr int kMostTop = 1024;
constexpr int kMostPieces = 32;  // of 64 scores: a wave has them in registers when it chooses
constexpr int kMostTile = 4;     // tokens
constexpr int kShare = 32;       // blocks that each wave of 16 may choose for the last to choose from

__device__ inline unsigned sortable(float x) {
  const unsigned u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// 16 queries of a key head (rows beyond the group are zeros) in codes, as operands of products of 64 values, the last
// of them zeros where D is no multiple of 64; and of the four rows that a lane has in a result the scales, and
// -infinity where there is no row. (One product of 32 values in the place of the zeros: sums that went from a product
// of 64 into one of 32 were wrong now and then in 96 values a head, in this loop and not by themselves.)
template <int D> struct Queries {
  i4 codes[(D + 63) / 64];
  float scale[4], none[4];
};

// Of four lanes, 16 apart
__device__ inline float quarters_max(float x) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// The rows from 16 * `part` on of `tokens` tokens times the group
template <class T, int D>
__device__ inline void load_queries(const Select& a, const T* rows, int tokens, int part, Queries<D>& q) {
  const int lane = threadIdx.x & 63, n16 = lane & 15, quarter = lane >> 4, r = 16 * part + n16;
  constexpr int kValues = 16 * ((D + 63) / 64);
  float x[kValues];
  const bool is = r < tokens * a.group;
  const int token = is ? r / a.group : 0, h = is ? r - token * a.group : 0;
  const T* row = rows + (int64_t)token * a.q_token + (int64_t)h * a.q_head;
#pragma unroll
  for (int i = 0; i < kValues; i += 8) {
    const int d = 64 * (i / 16) + 16 * quarter + i % 16;
    const bool inside = is && d < D;
    float y[8];
    load_row<T, 8>(row + (inside ? d : 0), a.q_vector, y);
#pragma unroll
    for (int j = 0; j < 8; j++) x[i + j] = inside && y[j] == y[j] ? y[j] : 0.f;
  }
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < kValues; i++) most = fmaxf(most, fabsf(x[i]));
  const int e = power_of(quarters_max(most));
  const float by = __uint_as_float((unsigned)(127 - e) << 23);
  unsigned words[kValues / 4];
#pragma unroll
  for (int i = 0; i < kValues / 4; i++) {
    unsigned w = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      // the sum's last bits are the nearest whole number's, of ties the even one's
      const float code = __builtin_amdgcn_fmed3f(x[4 * i + j] * by, -(float)kMostCode, (float)kMostCode) + 12582912.f;
      w |= (__float_as_uint(code) & 0xffu) << (8 * j);
    }
    words[i] = w;
  }
#pragma unroll
  for (int c = 0; c < kValues / 16; c++)
    q.codes[c] = i4{(int)words[4 * c], (int)words[4 * c + 1], (int)words[4 * c + 2], (int)words[4 * c + 3]};
  const float scale = __uint_as_float((unsigned)(127 + e) << 23), none = is ? 0.f : -INFINITY;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    q.scale[i] = __shfl(scale, 4 * quarter + i);
    q.none[i] = __shfl(none, 4 * quarter + i);
  }
}

// What a token may see: blocks up to `blocks`, of which those from near_from on and those before `from` are listed in any
// case, and `chosen` of those between
struct Seen {
  int from, near_from, blocks, chosen;
};

__device__ inline Seen seen_by(const Select& a, bool is, int position, int reach) {
  Seen s;
  const int high = !is || position < 0 ? 0 : a.causal ? min(position + 1, reach) : reach;
  s.blocks = (high + (1 << a.block_shift) - 1) >> a.block_shift;
  s.near_from = min(max((max(position, 0) >> a.block_shift) - a.near + 1, 0), s.blocks);
  s.from = min(a.first, s.near_from);
  s.chosen = min(a.top, s.near_from - s.from);
  return s;
}

// One wave: of `rows` rows of 64 keys (0: none) the `want` largest, of equal ones the first, in their order: put(which, row,
// key) by the lane that has it.  The key of the last one chosen is found bit by bit, counting with ballots, until as many as
// are wanted are above.  (A search among the lanes' largest keys first, and then among the few that are left, in one row:
// 106 us instead of 101 for the prompt below; it is a chain of counts, however many rows each has.)
template <int kRows, class Put>
__device__ inline void choose_rows(const unsigned* keys, int rows, int want, Put put) {
  const int lane = threadIdx.x & 63;
  unsigned key[kRows];
#pragma unroll
  for (int j = 0; j < kRows; j++) key[j] = j < rows ? keys[64 * j + lane] : 0;
  const auto count = [&](unsigned least) {
    int n = 0;
#pragma unroll
    for (int j = 0; j < kRows; j++) n += (int)__popcll(__ballot(key[j] >= least));
    return n;
  };
  unsigned bound = 0;                              // keys above are chosen, and the first ones equal to it
  int above = 0;
  for (int bit = 31; bit >= 0; bit--) {
    const unsigned trial = bound | 1u << bit;
    const int n = count(trial);
    if (n == want) {
      bound = trial - 1;
      above = n;
      break;
    }
    if (n > want) bound = trial;
    else above = n;                                // those with a larger key than `bound` may become
  }
  const unsigned long long before = (1ull << lane) - 1;
  int ties = want - above, at = 0;
#pragma unroll
  for (int j = 0; j < kRows; j++) {
    if (j >= rows) break;
    const unsigned long long x = __ballot(key[j] > bound), y = __ballot(key[j] == bound);
    const int equal_before = (int)__popcll(y & before), taken = min((int)__popcll(y), ties);
    if (key[j] > bound || (key[j] == bound && equal_before < ties))
      put(at + (int)__popcll(x & before) + min(equal_before, ties), j, key[j]);
    at += (int)__popcll(x) + taken;
    ties -= taken;
  }
}

// kTeam waves choose the blocks of up to kMostTile tokens of a world and a key head (1: four such units to a workgroup,
// of one token each).  They score 64 blocks at a time for all of them, by products of 16 rows (tokens times query
// heads) with 16 summaries, into LDS; then a wave chooses for each token.  More blocks than LDS has room for go in
// segments, the chosen ones of those before among the next.
//
// What bounds it: for a step's tokens a chain of loads that depend on each other (length, table, summaries), for
// prompts the instructions of scoring and counting (VALU 50 % busy).  1024 worlds' single tokens, 4 key heads of 64
// values, up to 128 blocks: 14.6 us (the bytes 4); two worlds of 2048 blocks, 8 key heads of 128 values: 18.4; 2048
// tokens over 1024 blocks: 98 (343 with a team to each token, whose waves counted together).
template <int kType, int D, int kTeam>
__global__ __launch_bounds__(kTeam == 1 ? 256 : 64 * kTeam) void select_blocks(const Select) {
  // read where they are used: as a parameter they would be in scalar registers throughout, and those of the loops spilled
  const Select& a = *(const Select*)(__attribute__((address_space(4))) const Select*)__builtin_amdgcn_kernarg_segment_ptr();
  typedef typename Elem<kType>::T T;
  constexpr int kParts = (D + 63) / 64, kTile = kTeam == 4 ? kMostTile : 1;
  extern __shared__ unsigned scores[];            // [token][64 * pieces], then, where there are segments, the kept
                                                  // blocks' numbers [token][kMostTop]
  const int wave = kTeam == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int n16 = lane & 15, quarter = lane >> 4;
  const int team = kTeam == 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
  const int unit = kTeam == 1 ? blockIdx.x * 4 + team : blockIdx.x;
  if (unit >= a.units) return;
  const int head = unit % a.kv_heads, tile = unit / a.kv_heads, room = 64 * a.pieces;
  unsigned* mine = scores + team * room;
  int* kept_block = (int*)(scores + (kTeam == 1 ? 4 : a.tile) * room) + team * kMostTop;
  const auto meet = [] {
    if constexpr (kTeam == 1) {
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    } else {
      __syncthreads();
    }
  };
  // the tile's rows, those of one world at a time
  const int tile_end = min((tile + 1) * a.tile, a.tokens);
  for (int token = tile * a.tile, next; token < tile_end; token = next) {
    const int world = a.start ? world_at(a.start, a.nworld, token) : token / a.count;
    const int begin = a.start ? a.start[world] : world * a.count, stop = a.start ? a.start[world + 1] : begin + a.count;
    const bool is = begin >= 0 && token >= begin && token < stop;
    next = is ? min(stop, tile_end) : token + 1;
    const int tokens = next - token, count = stop - begin, length = max(a.length[world], 0);
    const int position = length - count + token - begin;
    const int reach = (int)min((long long)length, (long long)a.width << a.page_shift);
    int from[kTile], near_from[kTile];             // of each token
    int low = INT32_MAX, high = 0;                 // of the blocks between which to choose
#pragma unroll
    for (int t = 0; t < kTile; t++) {
      const Seen s = seen_by(a, is && t < tokens && token + t - begin < a.max_count, position + t, reach);
      from[t] = s.from;
      near_from[t] = s.near_from;
      if (t >= tokens) continue;
      // what is listed in any case, and what lies behind
      int32_t* list = a.blocks + ((int64_t)(token + t) * a.kv_heads + head) * a.lists;
      const bool all = s.chosen == s.near_from - s.from;
      for (int i = 64 * wave + lane; i < a.lists; i += 64 * kTeam) {
        if (i < s.from || (all && i < s.from + s.chosen)) list[i] = i;
        else if (i >= s.from + s.chosen) {
          const int block = s.near_from + i - s.from - s.chosen;
          list[i] = block < s.blocks ? block : -1;
        }
      }
      if (all || !s.chosen) continue;
      low = min(low, s.from);
      high = max(high, s.near_from);
    }
    if (low >= high) continue;
    const int my_from = quarter == 0 ? from[0] : quarter == 1 ? from[kTile > 1] : quarter == 2 ? from[kTile / 2] : from[kTile - 1];
    const int my_near_from = quarter == 0 ? near_from[0] : quarter == 1 ? near_from[kTile > 1] : quarter == 2 ? near_from[kTile / 2]
                                                                                            : near_from[kTile - 1];

    const T* rows = (const T*)a.q + (int64_t)token * a.q_token + (int64_t)head * a.group * a.q_head;
    const int32_t* table = a.table + (int64_t)world * a.width;
    const int per_shift = a.page_shift - a.block_shift, parts = (tokens * a.group + 15) / 16;
    Queries<D> q;
    if (parts == 1) load_queries<T, D>(a, rows, tokens, 0, q);
    int kept = 0;
    for (int segment = low; segment < high;) {
      const bool segment_before = segment > low;
      const int kept_rows = (kept + 63) >> 6, last = min(segment + 64 * (a.pieces - kept_rows), high);
      const int rows_new = (last - segment + 63) >> 6;
      // few of many: each wave chooses from neighbouring rows of its own first, so that one wave is left with a share
      // of all (32 of 2048 blocks 26 -> 19 us)
      const bool shared = kTeam == 16 && !segment_before && last == high && a.top <= kShare;
      const int each = (rows_new + kTeam - 1) / kTeam;
      // one piece at a time: with the next one's summaries under way a wave has half as many beside it (two pieces of 64
      // values 15.5 -> 22.5 us)
      const int step = shared ? 1 : kTeam, rows_end = shared ? min((wave + 1) * each, rows_new) : rows_new;
      int pages[4];                                // of the next piece's blocks
      const auto look_up = [&](int row) {
#pragma unroll
        for (int u = 0; u < 4; u++) pages[u] = table[min(segment + 64 * row + 16 * u + n16, last - 1) >> per_shift];
      };
      look_up(shared ? wave * each : wave);
#pragma unroll 1
      for (int row = shared ? wave * each : wave; row < rows_end; row += step) {
        const int base = segment + 64 * row;
        i4 part[4][kParts];
        unsigned byte[4];
        bool there[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
          const int block = min(base + 16 * u + n16, last - 1), page = pages[u];
          there[u] = (unsigned)page < (unsigned)a.npage;
          const int64_t entry = (((int64_t)(there[u] ? page : 0) * a.kv_heads + head) << per_shift) + (block & ((1 << per_shift) - 1));
          const int8_t* codes = a.codes + entry * D;
#pragma unroll
          for (int c = 0; c < kParts; c++) {
            const bool inside = 64 * c + 16 * quarter < D;
            part[u][c] = *(const i4*)(codes + (inside ? 64 * c + 16 * quarter : 0));
            if (!inside) part[u][c] = i4{0, 0, 0, 0};
          }
          byte[u] = a.exponent[entry];
        }
        look_up(row + step);
        float best[4];                             // of the first token, where it has more rows than one product
#pragma unroll
        for (int u = 0; u < 4; u++) best[u] = -INFINITY;
        for (int p = 0; p < parts; p++) {
          if (parts > 1) load_queries<T, D>(a, rows, tokens, p, q);
#pragma unroll
          for (int u = 0; u < 4; u++) {
            i4 sum = i4{0, 0, 0, 0};
#pragma unroll
            for (int c = 0; c < kParts; c++) sum = __builtin_amdgcn_mfma_i32_16x16x64_i8(q.codes[c], part[u][c], sum, 0, 0, 0);
            float row[4];
#pragma unroll
            for (int i = 0; i < 4; i++) row[i] = __builtin_fmaf((float)sum[i], q.scale[i], q.none[i]);
            const int at = base + 16 * u + n16;
            const auto store = [&](int from, int near_from, int t, float most) {
              const float score = !there[u] ? -INFINITY : byte[u] == kNoNumber ? INFINITY : most * scale_of(byte[u]);
              mine[t * room + 64 * kept_rows + at - segment] = at < last && at >= from && at < near_from ? sortable(score) : 0;
            };
            if (kTile > 1 && a.group == 4) {       // a quarter of the lanes has a token's rows
              if (quarter < tokens) store(my_from, my_near_from, quarter, fmaxf(fmaxf(row[0], row[1]), fmaxf(row[2], row[3])));
            } else {
#pragma unroll
              for (int t = 0; t < kTile; t++) {
                if (t >= tokens) continue;
                float most = -INFINITY;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                  const int r = 4 * quarter + i;
                  most = fmaxf(most, tokens == 1 || (r >= t * a.group && r < (t + 1) * a.group) ? row[i] : -INFINITY);
                }
                most = quarters_max(most);
                if (parts > 1) most = best[u] = fmaxf(best[u], most);
                if (quarter == 0 && p == parts - 1) store(from[t], near_from[t], t, most);
              }
            }
          }
        }
      }
      unsigned* share = scores + room;             // (only teams of 16, which have one token)
      int* share_block = (int*)(share + kTeam * kShare);
      if (shared) {
        unsigned* keys = mine + 64 * wave * each;
        const int own = max(min(each, rows_new - wave * each), 0);
        if (lane < kShare) share[kShare * wave + lane] = 0;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (own)
          choose_rows<2>(keys, own, a.top, [&](int at, int j, unsigned key) {
            share[kShare * wave + at] = key;
            share_block[kShare * wave + at] = segment + 64 * (wave * each + j) + lane;
          });
      }
      meet();
      const bool done = last == high;
      const int t = kTile > 1 ? wave : 0;          // a wave's own token
      const Seen s = seen_by(a, is && t < tokens && token + t - begin < a.max_count, position + t, reach);
      if (t < tokens && (kTile > 1 || wave == 0) && s.chosen && s.chosen < s.near_from - s.from) {
        unsigned* keys = mine + t * room;
        int* held = kept_block + t * kMostTop;
        int32_t* list = a.blocks + ((int64_t)(token + t) * a.kv_heads + head) * a.lists + s.from;
        const int listed = a.lists - s.from, used = kept_rows + (last - segment + 63) / 64;
        const auto put = [&](int at, int j, unsigned key) {
          const int block = shared ? share_block[64 * j + lane] : j < kept_rows ? held[64 * j + lane]
                                                                               : segment + 64 * (j - kept_rows) + lane;
          if (done) {
            if (at < listed) list[at] = block;
          } else {
            keys[at] = key;
            held[at] = block;
          }
        };
        // a segment may not have as many yet as are wanted: keys of 0 are chosen then, and are no blocks' in the next
        if (shared) choose_rows<(kTeam * kShare + 63) / 64>(share, kTeam * kShare / 64, s.chosen, put);
        else if (used <= 2) choose_rows<2>(keys, used, s.chosen, put);
        else if (used <= 8) choose_rows<8>(keys, used, s.chosen, put);
        else if (used <= 16) choose_rows<16>(keys, used, s.chosen, put);
        else choose_rows<kMostPieces>(keys, used, s.chosen, put);
      }
      segment = last;
      kept = a.top;
      if (!done) {
        meet();
        // behind the kept ones of a row nothing
        for (int t = 0; t < min(tokens, kTile); t++)
          for (int i = kept + 64 * wave + lane; i < ((kept + 63) & ~63); i += 64 * kTeam) mine[t * room + i] = 0;
      }
    }
    meet();                                        // before the next world's scores
  }
}

// ---------------------------------------------------------------------------- rows gathered by their blocks
// The first word of a world's marks: ragged chunks of n tokens have n / 32 + 1 at most, so that the places of all follow from
// `start` and their number from what the host knows, however large a chunk may be
__device__ inline int first_word(const Attend& a, int world) {
  return a.start ? (max(a.start[world], 0) >> 5) + world : world * a.words;
}

// Tokens of a world's chunk whose rows are computed, and its first packed one
__device__ inline int marked_tokens(const Attend& a, int world, int& begin) {
  begin = a.start ? a.start[world] : world * a.count;
  const int stop = a.start ? min(a.start[world + 1], a.tokens) : begin + a.count;
  return begin < 0 ? 0 : max(min(stop - begin, a.max_count), 0);
}

// Blocks of a world that have tokens: none behind them are marked
__device__ inline int blocks_held(const Attend& a, int world) {
  return min((int)((max(a.length[world], 0) + (1LL << a.block_shift) - 1) >> a.block_shift), a.world_blocks);
}

// A workgroup takes 32 tokens of a world's chunk and a key head (2048 tokens' 19 blocks, 8 heads: 5 us; with atomics in
// memory 28): the bits of all blocks that their lists name, collected in LDS (so many blocks at a time), and written
// side by side: marks[key head][word][block], as far as the world has tokens.  Entries of whose keys the row sees none get
// empty parts.
constexpr int kMarked = 8192;
__global__ __launch_bounds__(256) void mark_rows(const Attend a) {
  __shared__ unsigned bits[kMarked];
  const int item = blockIdx.x % a.words_all, head = blockIdx.x / a.words_all;
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i * a.batch_heads < a.kv_heads; i += 256) a.gathered_tiles[i] = 0;
  int world = 0;
  if (a.start) {                                  // the last one whose words begin at or before this
    for (int high = a.nworld; high - world > 1;) {
      const int step = (high - world + 63) >> 6, probe = world + (threadIdx.x & 63) * step;
      const int passed = max(1, (int)__popcll(__ballot(probe < high && first_word(a, probe) <= item)));
      world += (passed - 1) * step;
      high = min(high, world + step);
    }
    world = __builtin_amdgcn_readfirstlane(world);
  } else {
    world = item / a.words;
  }
  int begin;
  const int word = item - first_word(a, world), tokens = min(marked_tokens(a, world, begin) - 32 * word, 32);
  if (word < 0 || tokens <= 0) return;
  const int count = a.start ? a.start[world + 1] - begin : a.count, length = max(a.length[world], 0);
  const int reach = (int)min((long long)length, (long long)a.width << a.page_shift), blocks = blocks_held(a, world);
  unsigned* marks = a.marks + ((int64_t)head * a.words_all + item) * a.world_blocks;
  for (int first = 0; first == 0 || first < blocks; first += kMarked) {
    const int many = min(blocks - first, kMarked);
    for (int i = threadIdx.x; i < many; i += 256) bits[i] = 0;
    __syncthreads();
    for (int at = threadIdx.x; at < tokens * a.lists; at += 256) {
      const int which = at / a.lists, entry = at - which * a.lists, i = 32 * word + which, position = length - count + i;
      const int high = position < 0 ? 0 : a.causal ? min(position + 1, reach) : reach;
      const int block = a.blocks[((int64_t)(begin + i) * a.kv_heads + head) * a.lists + entry];
      if ((unsigned)block < (unsigned)a.world_blocks && block << a.block_shift < high) {
        if ((unsigned)(block - first) < (unsigned)many) atomicOr(&bits[block - first], 1u << which);
      } else if (!first) {
        const int64_t row = (a.start ? begin + i : (int64_t)world * a.max_count + i) * a.heads + head * a.group;
        for (int h = 0; h < a.group; h++) *(f2*)(a.part_ml + 2 * (entry * (int64_t)a.part_rows + row + h)) = f2{-INFINITY, 0.f};
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < many; i += 256) marks[first + i] = bits[i];
  }
}

// A workgroup takes 16 blocks of a world's key head, a wave four of them in turn: how many tiles their tokens are,
// places for those in any order among the others' of the batch, as each row's part is its own, and the tokens in their
// order.
constexpr int kCounted = 16;
__global__ __launch_bounds__(256) void list_tiles(const Attend a) {
  __shared__ int sh_tokens[kCounted], sh_from[kCounted];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, many = kManyRows / a.group;
  const int per = (a.world_blocks + kCounted - 1) / kCounted, pair = blockIdx.x / per, first = (blockIdx.x - pair * per) * kCounted;
  const int world = pair / a.kv_heads, head = pair - world * a.kv_heads, batch = head / a.batch_heads;
  const int blocks = blocks_held(a, world);
  if (first >= blocks) return;
  int begin;
  const int in_all = marked_tokens(a, world, begin), words = (in_all + 31) >> 5;
  const unsigned* marks = a.marks + ((int64_t)head * a.words_all + first_word(a, world)) * a.world_blocks;
  // tokens that the chunk does not have are in no word, whatever is in the memory of one that no workgroup wrote
  const auto word_of = [&](int w, int block) {
    const int tokens = in_all - 32 * w;
    return marks[(int64_t)w * a.world_blocks + block] & (tokens >= 32 ? ~0u : (1u << tokens) - 1);
  };
  // the tokens of a block, by 16 threads
  {
    const int block = first + (threadIdx.x >> 4);
    int tokens = 0;
    if (block < blocks)
      for (int w = threadIdx.x & 15; w < words; w += 16) tokens += __popc(word_of(w, block));
#pragma unroll
    for (int by = 1; by < 16; by *= 2) tokens += __shfl_xor(tokens, by);
    if ((threadIdx.x & 15) == 0) sh_tokens[threadIdx.x >> 4] = tokens;
  }
  __syncthreads();
  if (wave == 0) {
    const int tiles = lane < kCounted ? (sh_tokens[lane] + many - 1) / many : 0;
    int sum = tiles;
#pragma unroll
    for (int by = 1; by < kCounted; by *= 2) {
      const int y = __shfl_up(sum, by);
      if (lane >= by) sum += y;
    }
    int from = 0;
    if (lane == kCounted - 1 && sum) from = atomicAdd(a.gathered_tiles + batch, sum);
    from = __shfl(from, kCounted - 1) + sum - tiles;
    if (lane < kCounted) sh_from[lane] = from;
  }
  __syncthreads();
  for (int i = wave; i < kCounted; i += 4) {
    const int tokens = sh_tokens[i], tiles = (tokens + many - 1) / many;
    if (!tokens) continue;
    // (there is room for all where `start` is as it has to be; tiles of a block without are empty)
    const bool fits = sh_from[i] + tiles <= a.tiles_most;
    const int64_t from = (int64_t)batch * a.tiles_most + sh_from[i];
    for (int j = lane; j < min(tiles, a.tiles_most - sh_from[i]); j += 64)
      a.gathered[from + j] = int4{pair, first + i, fits ? min(tokens - j * many, many) : 0, 0};
    if (!fits) continue;
    int* rows = a.gathered_rows + from * many;
    int before = 0;                               // marked in the words before
    for (int base = 0; base < words; base += 64) {
      unsigned word = base + lane < words ? word_of(base + lane, first + i) : 0;
      int sum = __popc(word);
#pragma unroll
      for (int by = 1; by < 64; by *= 2) {
        const int y = __shfl_up(sum, by);
        if (lane >= by) sum += y;
      }
      for (int place = before + sum - __popc(word); word; word &= word - 1, place++)
        rows[place] = 32 * (base + lane) + __builtin_ctz(word);
      before += __shfl(sum, 63);
    }
  }
}

int gather_rows(Attend& a, const Launch& launch, void* stream) {
  const hipStream_t s = (hipStream_t)stream;
  const unsigned pairs = a.nworld * a.kv_heads, per = (a.world_blocks + kCounted - 1) / kCounted;
  hipLaunchKernelGGL(mark_rows, dim3((unsigned)a.words_all * a.kv_heads), dim3(256), 0, s, a);
  hipLaunchKernelGGL(list_tiles, dim3(pairs * per), dim3(256), 0, s, a);
  return (int)hipGetLastError();
}

// ---------------------------------------------------------------------------- host side
int summaries_check(const MxPages* p, const MxSummaries* s) {
  if (!s || !s->codes || !s->exponent || ((uintptr_t)s->codes & 15)) return MX_ERR_INVALID;
  const int b = s->block_tokens;
  if (b < 16 || b > p->page_tokens || (b & (b - 1))) return MX_ERR_DOMAIN;
  return 0;
}

template <int D> void launch_summarise(const Summarise& a, int type, unsigned groups, void* stream) {
  const auto go = [&](auto store) {
    hipLaunchKernelGGL((summarise_blocks<decltype(store)::value, D>), dim3(groups), dim3(256), 0, (hipStream_t)stream, a);
  };
  if (type == MX_TYPE_FP8) go(std::integral_constant<int, MX_TYPE_FP8>());
  else if (type == MX_TYPE_BF16) go(std::integral_constant<int, MX_TYPE_BF16>());
  else go(std::integral_constant<int, MX_TYPE_F16>());
}

template <int D> void launch_select(const Select& a, int type, int team, unsigned groups, size_t lds, void* stream) {
  const auto go = [&](auto t, auto n) {
    constexpr int kTeam = decltype(n)::value;
    hipLaunchKernelGGL((select_blocks<decltype(t)::value, D, kTeam>), dim3(groups), dim3(kTeam == 1 ? 256 : 64 * kTeam), lds,
                       (hipStream_t)stream, a);
  };
  const auto by_team = [&](auto t) {
    if (team == 1) go(t, std::integral_constant<int, 1>());
    else if (team == 4) go(t, std::integral_constant<int, 4>());
    else if constexpr (D <= 128) go(t, std::integral_constant<int, 16>());
  };
  if (type == MX_TYPE_BF16) by_team(std::integral_constant<int, MX_TYPE_BF16>());
  else by_team(std::integral_constant<int, MX_TYPE_F16>());
}

template <class F> void by_head_dim(int dim, F f) {
  switch (dim) {
    case 32: f(std::integral_constant<int, 32>()); break;
    case 64: f(std::integral_constant<int, 64>()); break;
    case 96: f(std::integral_constant<int, 96>()); break;
    case 128: f(std::integral_constant<int, 128>()); break;
    default: f(std::integral_constant<int, 256>());
  }
}

int recall_plan(const MxPages* p, const MxChunk* c, const MxAttention* m, const MxSelection* s, int block_tokens, Attend& a,
                Launch& launch, bool pointers) {
  if (!s || (m && m->window)) return MX_ERR_INVALID;
  if (pointers && c && c->tokens > 0 && !s->blocks) return MX_ERR_INVALID;
  if (s->width < 1 || s->width > 4096) return MX_ERR_DOMAIN;
  const int rc = pages_check(p);
  if (rc) return rc;
  if (block_tokens < 16 || block_tokens > p->page_tokens || (block_tokens & (block_tokens - 1))) return MX_ERR_DOMAIN;
  return plan(p, c, m, a, launch, pointers, s, __builtin_ctz(block_tokens));
}

}  // namespace mxe

extern "C" {

size_t mx_summaries_bytes(void) { return sizeof(MxSummaries); }
size_t mx_selection_bytes(void) { return sizeof(MxSelection); }

int mx_episode_summarise(const MxPages* p, const MxChunk* c, const MxSummaries* s, void* stream) {
  using namespace mxe;
  int rc = pages_check(p);
  if (rc || (rc = chunk_check(p, c)) || (rc = summaries_check(p, s))) return rc;
  if (!c->tokens) return 0;
  Summarise a{};
  a.k = (const uint8_t*)p->k; a.k_scale = p->k_scale;
  a.table = p->table; a.length = p->length; a.start = c->start;
  a.codes = s->codes; a.exponent = s->exponent;
  a.nworld = p->nworld; a.npage = p->npage; a.width = p->width; a.kv_heads = p->kv_heads;
  a.page_shift = page_shift(p); a.block_shift = __builtin_ctz(s->block_tokens);
  a.tokens = c->tokens; a.count = c->count;
  a.per = c->start ? 0 : ((c->count - 1) >> a.block_shift) + 1;
  const int64_t groups = c->start ? (int64_t)(c->tokens >> a.block_shift) + p->nworld : (int64_t)a.per * p->nworld;
  if (groups > kMostGroups) return MX_ERR_DOMAIN;
  by_head_dim(p->head_dim, [&](auto d) { launch_summarise<decltype(d)::value>(a, p->type, (unsigned)groups, stream); });
  return (int)hipGetLastError();
}

int mx_episode_select(const MxPages* p, const MxChunk* c, const MxSummaries* s, const MxRows* q, const MxSelection* m, void* stream) {
  using namespace mxe;
  int rc = pages_check(p);
  if (rc || (rc = chunk_check(p, c)) || (rc = summaries_check(p, s))) return rc;
  if (!m || !q || q->heads < 1 || q->heads % p->kv_heads) return MX_ERR_INVALID;
  if ((rc = rows_check(q, q->heads, c->tokens > 0))) return rc;
  if (q->type != MX_TYPE_BF16 && q->type != MX_TYPE_F16) return MX_ERR_INVALID;
  if (p->type != MX_TYPE_FP8 && p->type != q->type) return MX_ERR_INVALID;
  if (m->top < 0 || m->near < 1 || m->first < 0 || m->max_count < 0 || m->width < 1) return MX_ERR_INVALID;
  if (m->top > kMostTop || m->width > 4096 || q->heads / p->kv_heads > 1024) return MX_ERR_DOMAIN;
  if ((int64_t)m->first + m->near + m->top > m->width) return MX_ERR_INVALID;
  if (!c->tokens) return 0;
  if (!m->blocks) return MX_ERR_INVALID;
  Select a{};
  a.table = p->table; a.length = p->length; a.start = c->start;
  a.q = q->data; a.q_token = q->token_stride; a.q_head = q->head_stride;
  a.codes = s->codes; a.exponent = s->exponent; a.blocks = m->blocks;
  a.nworld = p->nworld; a.npage = p->npage; a.width = p->width; a.kv_heads = p->kv_heads;
  a.page_shift = page_shift(p); a.block_shift = __builtin_ctz(s->block_tokens);
  a.tokens = c->tokens; a.count = c->count; a.max_count = m->max_count;
  a.group = q->heads / p->kv_heads;
  a.lists = m->width; a.top = m->top; a.near = m->near; a.first = m->first;
  a.causal = m->causal != 0;
  a.q_vector = rows_aligned(q, 16);
  // tokens side by side where worlds have many, so that they share the summaries' loads
  const int64_t pieces = (((int64_t)p->width << (a.page_shift - a.block_shift)) + 63) / 64;
  const int side = a.group > 8 ? 1 : 16 / a.group < kMostTile ? 16 / a.group : kMostTile;
  a.tile = c->tokens >= (int64_t)2 * side * p->nworld ? side : 1;
  a.pieces = (int)(pieces < kMostPieces ? pieces : kMostPieces);
  const int64_t units = ((int64_t)c->tokens + a.tile - 1) / a.tile * p->kv_heads;
  const int team = a.tile > 1 ? 4 : pieces <= 2 || units >= 4096 ? 1 : pieces < 16 || units >= 512 || p->head_dim > 128 ? 4 : 16;
  const int64_t groups = team == 1 ? (units + 3) / 4 : units;
  // threads are counted in 32 bits
  if (groups > (team == 16 ? kMostGroups / 4 : kMostGroups)) return MX_ERR_DOMAIN;
  a.units = (int)units;
  const size_t lds = sizeof(int) * (team == 1 ? 4 : a.tile) * (64 * a.pieces + (pieces > kMostPieces ? kMostTop : 0))
                     + (team == 16 ? sizeof(int) * 2 * 16 * kShare : 0);
  by_head_dim(p->head_dim, [&](auto d) { launch_select<decltype(d)::value>(a, q->type, team, (unsigned)groups, lds, stream); });
  return (int)hipGetLastError();
}

int mx_episode_recall(const MxPages* pages, const MxChunk* chunk, const MxAttention* m, const MxSelection* s,
                      int32_t block_tokens, void* stream) {
  mxe::Attend a{};
  mxe::Launch launch{};
  const int rc = mxe::recall_plan(pages, chunk, m, s, block_tokens, a, launch, true);
  return rc || !launch.tiles ? rc : mxe::attend_planned(a, launch, m, stream);
}

size_t mx_recall_workspace(const MxPages* pages, const MxChunk* chunk, const MxAttention* m, const MxSelection* s,
                           int32_t block_tokens) {
  mxe::Attend a{};
  mxe::Launch launch{};
  return mxe::recall_plan(pages, chunk, m, s, block_tokens, a, launch, false) ? 0 : mxe::workspace_of(a, launch);
}

}
