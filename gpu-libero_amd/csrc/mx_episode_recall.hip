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

// ---------------------------------------------------------------------------- summaries
struct Summarise {
  const uint8_t *k, *k_scale;
  const int32_t *table, *length, *start;
  int8_t* codes;
  uint8_t* exponent;
  int nworld, npage, width, kv_heads, page_shift, block_shift, tokens, count, per;   // per: blocks of a world's chunk at most
};

// A workgroup takes a block and a wave its heads in turn: lanes side by side along a key, as many keys as fit beside each other, sums in 64 bits
// joined through LDS.  World w of ragged chunks has the items from start[w] / block_tokens + w on.
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
  int units;                     // rows times key heads
  bool causal, q_vector;
};

constexpr int kRegisters = 8;    // scores of a lane, through LDS so that the loop over them is short
constexpr int kMostTop = 1024;

__device__ inline unsigned sortable(float x) {
  const unsigned u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// 16 queries of a key head (rows beyond the group are zeros) in codes, as operands of products of 64 values, the last of them
// zeros where D is no multiple of 64; and the scales of the four rows that a lane has in a result, -1 for rows that are none.
// (One product of 32 values in the place of the zeros: sums that went from a product of 64 into one of 32 were wrong now
// and then in 96 values a head, in this loop and not by themselves.)
template <int D> struct Queries {
  i4 codes[(D + 63) / 64];
  float scale[4];
};

template <class T, int D>
__device__ inline void load_queries(const Select& a, const T* rows, int tile, Queries<D>& q) {
  const int lane = threadIdx.x & 63, n16 = lane & 15, quarter = lane >> 4, h = 16 * tile + n16;
  constexpr int kValues = 16 * ((D + 63) / 64);
  float x[kValues];
  const bool is = h < a.group;
  const T* row = rows + (int64_t)(is ? h : 0) * a.q_head;
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
  most = fmaxf(most, __shfl_xor(most, 16));
  most = fmaxf(most, __shfl_xor(most, 32));
  const int e = power_of(most);
  unsigned words[kValues / 4];
#pragma unroll
  for (int i = 0; i < kValues / 4; i++) {
    unsigned w = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const float code = fminf(fmaxf(__builtin_rintf(ldexpf(x[4 * i + j], -e)), -(float)kMostCode), (float)kMostCode);
      w |= ((unsigned)(int)code & 0xffu) << (8 * j);
    }
    words[i] = w;
  }
#pragma unroll
  for (int c = 0; c < kValues / 16; c++)
    q.codes[c] = i4{(int)words[4 * c], (int)words[4 * c + 1], (int)words[4 * c + 2], (int)words[4 * c + 3]};
  const float scale = is ? ldexpf(1.f, e) : -1.f;
#pragma unroll
  for (int i = 0; i < 4; i++) q.scale[i] = __shfl(scale, 4 * quarter + i);
}

// kTeam waves choose the blocks of a row and a key head (1: four such units to a workgroup).  They score 64 blocks at a time, by products of
// 16 queries with 16 blocks, keep a score of each block, find the score of the last block chosen bit by
// bit, counting with ballots, and write the blocks from there on in their order.  More blocks than registers hold
// (only teams of 16) go in segments, the chosen ones of those before among the next.
template <int kType, int D, int kTeam>
__global__ __launch_bounds__(kTeam == 1 ? 256 : 64 * kTeam) void select_blocks(const Select a) {
  typedef typename Elem<kType>::T T;
  constexpr int kSegment = 64 * kRegisters * kTeam, kParts = (D + 63) / 64;
  constexpr bool kKeeps = kTeam == 16;
  __shared__ unsigned scores[kTeam == 1 ? 4 : kTeam][kRegisters][64];
  __shared__ int counts[2][kTeam], sh_above[2 * kTeam], sh_equal[2 * kTeam];
  __shared__ unsigned kept_key[kKeeps ? kMostTop : 1];
  __shared__ int kept_block[kKeeps ? kMostTop : 1];
  const int wave = kTeam == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int team_wave = threadIdx.x >> 6, n16 = lane & 15, quarter = lane >> 4, thread = 64 * wave + lane;
  const int unit = kTeam == 1 ? __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6)) : blockIdx.x;
  if (unit >= a.units) return;
  const int head = unit % a.kv_heads, token = unit / a.kv_heads;
  int32_t* list = a.blocks + (int64_t)unit * a.lists;
  const int world = a.start ? world_at(a.start, a.nworld, token) : token / a.count;
  const int begin = a.start ? a.start[world] : world * a.count, count = a.start ? a.start[world + 1] - begin : a.count;
  const int place = token - begin, length = max(a.length[world], 0), position = length - count + place;
  const int reach = (int)min((long long)length, (long long)a.width << a.page_shift);
  const bool is = begin >= 0 && place >= 0 && place < min(count, a.max_count) && position >= 0;
  const int high = !is ? 0 : a.causal ? min(position + 1, reach) : reach;      // of the keys that are seen
  const int blocks = (high + (1 << a.block_shift) - 1) >> a.block_shift;
  const int near_from = min(max((is ? position >> a.block_shift : 0) - a.near + 1, 0), blocks);
  const int from = min(a.first, near_from), candidates = near_from - from;
  const int chosen = min(a.top, candidates);
  // what is always listed, and what lies behind
  for (int i = thread; i < a.lists; i += 64 * kTeam) {
    if (i < from) list[i] = i;
    else if (i >= from + chosen) list[i] = i - from - chosen < blocks - near_from ? near_from + i - from - chosen : -1;
    else if (chosen == candidates) list[i] = i;
  }
  if (chosen == candidates || !chosen) return;

  const T* rows = (const T*)a.q + (int64_t)token * a.q_token + (int64_t)head * a.group * a.q_head;
  const int32_t* table = a.table + (int64_t)world * a.width;
  const int per_shift = a.page_shift - a.block_shift, tiles = (a.group + 15) / 16;
  Queries<D> q;
  if (tiles == 1) load_queries<T, D>(a, rows, 0, q);
  int kept = 0;
  for (int segment = 0; segment < candidates; segment += kSegment) {
    const int last = min(segment + kSegment, candidates);
#pragma unroll 1
    for (int j = 0; j < kRegisters; j++) {
      const int base = segment + (wave * kRegisters + j) * 64;
      if (base >= last) break;
      i4 part[4][kParts];
      int64_t entry[4];
      bool there[4];
#pragma unroll
      for (int t = 0; t < 4; t++) {
        const int block = from + min(base + 16 * t + n16, last - 1);
        const int page = table[block >> per_shift];
        there[t] = (unsigned)page < (unsigned)a.npage;
        entry[t] = (((int64_t)(there[t] ? page : 0) * a.kv_heads + head) << per_shift) + (block & ((1 << per_shift) - 1));
      }
#pragma unroll
      for (int t = 0; t < 4; t++) {
        const int8_t* codes = a.codes + entry[t] * D;
#pragma unroll
        for (int c = 0; c < kParts; c++) {
          const bool inside = 64 * c + 16 * quarter < D;
          part[t][c] = *(const i4*)(codes + (inside ? 64 * c + 16 * quarter : 0));
          if (!inside) part[t][c] = i4{0, 0, 0, 0};
        }
      }
      // a lane's own block is that of its quarter's product
      const int64_t mine = quarter == 0 ? entry[0] : quarter == 1 ? entry[1] : quarter == 2 ? entry[2] : entry[3];
      const bool is_there = quarter == 0 ? there[0] : quarter == 1 ? there[1] : quarter == 2 ? there[2] : there[3];
      const unsigned byte = a.exponent[mine];
      float best = -INFINITY;
      for (int tile = 0; tile < tiles; tile++) {
        if (tiles > 1) load_queries<T, D>(a, rows, tile, q);
#pragma unroll
        for (int t = 0; t < 4; t++) {
          i4 sum = i4{0, 0, 0, 0};
#pragma unroll
          for (int c = 0; c < kParts; c++) sum = __builtin_amdgcn_mfma_i32_16x16x64_i8(q.codes[c], part[t][c], sum, 0, 0, 0);
          float most = -INFINITY;
#pragma unroll
          for (int i = 0; i < 4; i++) most = q.scale[i] < 0.f ? most : fmaxf(most, (float)sum[i] * q.scale[i]);
          most = fmaxf(most, __shfl_xor(most, 16));
          most = fmaxf(most, __shfl_xor(most, 32));
          best = t == quarter ? fmaxf(best, most) : best;
        }
      }
      const float score = !is_there ? -INFINITY : byte == kNoNumber ? INFINITY : best * scale_of(byte);
      scores[team_wave][j][lane] = base + lane < last ? sortable(score) : 0;
    }
    unsigned key[kRegisters];
#pragma unroll
    for (int j = 0; j < kRegisters; j++)        // a lane reads what it has written
      key[j] = segment + (wave * kRegisters + j) * 64 < last ? scores[team_wave][j][lane] : 0;
    unsigned old_key = 0;
    int old_block = 0;
    if constexpr (kKeeps) {
      if (segment) __syncthreads();
      if (thread < kept) {
        old_key = kept_key[thread];
        old_block = kept_block[thread];
      }
    }
    const int want = min(a.top, last);            // of those seen so far

    unsigned bound = 0;                           // the smallest key that is chosen
    for (int bit = 31; bit >= 0; bit--) {
      const unsigned trial = bound | 1u << bit;
      int n = 0;
#pragma unroll
      for (int j = 0; j < kRegisters; j++) n += (int)__popcll(__ballot(key[j] >= trial));
      if constexpr (kKeeps) n += (int)__popcll(__ballot(old_key >= trial));
      if constexpr (kTeam > 1) {
        if (lane == 0) counts[bit & 1][wave] = n;
        __syncthreads();
        n = 0;
#pragma unroll
        for (int w = 0; w < kTeam; w++) n += counts[bit & 1][w];
      }
      if (n >= want) bound = trial;
    }
    // how many are above it and equal to it: in the kept ones of each wave, then in the new ones
    int above = 0, equal = 0;
#pragma unroll
    for (int j = 0; j < kRegisters; j++) {
      above += (int)__popcll(__ballot(key[j] > bound));
      equal += (int)__popcll(__ballot(key[j] == bound));
    }
    const unsigned long long old_above = kKeeps ? __ballot(old_key > bound) : 0;
    const unsigned long long old_equal = kKeeps ? __ballot(old_key == bound && old_key) : 0;
    int above_old = 0, equal_old = 0, above_new = 0, equal_new = 0, ties = want - above;
    if constexpr (kTeam > 1) {
      if (lane == 0) {
        sh_above[wave] = (int)__popcll(old_above);
        sh_equal[wave] = (int)__popcll(old_equal);
        sh_above[kTeam + wave] = above;
        sh_equal[kTeam + wave] = equal;
      }
      __syncthreads();
      int all = 0;
      for (int w = 0; w < 2 * kTeam; w++) {
        const int x = sh_above[w], y = sh_equal[w];
        all += x;
        above_old += w < wave ? x : 0;
        equal_old += w < wave ? y : 0;
        above_new += w < kTeam + wave ? x : 0;
        equal_new += w < kTeam + wave ? y : 0;
      }
      ties = want - all;
    }
    const bool done = last == candidates;
    const unsigned long long before = (1ull << lane) - 1;
    const auto put = [&](bool above_it, bool equal_to_it, int above_before, int equal_before, unsigned value, int block) {
      if (!(above_it || (equal_to_it && equal_before < ties))) return;
      const int at = above_before + min(equal_before, ties);
      if (done) {
        if (from + at < a.lists) list[from + at] = block;
      } else if constexpr (kKeeps) {
        kept_key[at] = value;
        kept_block[at] = block;
      }
    };
    if constexpr (kKeeps)
      put(old_key > bound, old_key == bound && old_key, above_old + (int)__popcll(old_above & before),
          equal_old + (int)__popcll(old_equal & before), old_key, old_block);
#pragma unroll
    for (int j = 0; j < kRegisters; j++) {
      const unsigned long long x = __ballot(key[j] > bound), y = __ballot(key[j] == bound);
      put(key[j] > bound, key[j] == bound, above_new + (int)__popcll(x & before), equal_new + (int)__popcll(y & before), key[j],
          from + segment + (wave * kRegisters + j) * 64 + lane);
      above_new += (int)__popcll(x);
      equal_new += (int)__popcll(y);
    }
    kept = want;
  }
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

// Waves of a team, by the blocks that a world's table has room for
int team_of(int64_t blocks) { return blocks <= 64 * kRegisters ? 1 : blocks <= 256 * kRegisters ? 4 : 16; }

template <int D> void launch_select(const Select& a, int type, int team, unsigned groups, void* stream) {
  const auto go = [&](auto t, auto n) {
    constexpr int kTeam = decltype(n)::value;
    hipLaunchKernelGGL((select_blocks<decltype(t)::value, D, kTeam>), dim3(groups), dim3(kTeam == 1 ? 256 : 64 * kTeam), 0,
                       (hipStream_t)stream, a);
  };
  const auto by_team = [&](auto t) {
    if (team == 1) go(t, std::integral_constant<int, 1>());
    else if (team == 4) go(t, std::integral_constant<int, 4>());
    else go(t, std::integral_constant<int, 16>());
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
  const int64_t units = (int64_t)c->tokens * p->kv_heads;
  const int team = team_of((int64_t)p->width << (a.page_shift - a.block_shift));
  const int64_t groups = team == 1 ? (units + 3) / 4 : units;
  // threads are counted in 32 bits
  if (groups > (team == 16 ? kMostGroups / 4 : kMostGroups)) return MX_ERR_DOMAIN;
  a.units = (int)units;
  by_head_dim(p->head_dim, [&](auto d) { launch_select<decltype(d)::value>(a, q->type, team, (unsigned)groups, stream); });
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
