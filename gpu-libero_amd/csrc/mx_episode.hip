// The episode memory's entry points: writing to and reading from the pages, joining the parts of a
// split attention, and the host side of all calls.  The attention itself: mx_episode_few.h, mx_episode_many.h.
#include <cmath>
#include <type_traits>
#include "mx_episode_move.h"
#include "mx_episode_launch.h"

namespace mxe {

// ---------------------------------------------------------------------------- write and read
// A workgroup moves `tokens_each` packed tokens of all heads, keys and values: its first threads find
// their slots, then every thread moves pieces in the order of the rows.  Nothing is computed but the scales: bound by memory.
constexpr int kMostTokens = 64;                         // of a workgroup: their slots are kept in LDS

template <class T, int kStore, bool kWrite>
__global__ __launch_bounds__(256) void move_rows(const Move a) {
  constexpr int kPer = piece_bytes(kStore == MX_TYPE_FP8, kWrite, sizeof(T)) / sizeof(T), kItems = pieces_ahead(sizeof(T));
  __shared__ int64_t slots[kMostTokens];
  const int first = blockIdx.x * a.tokens_each, tokens = min(a.tokens - first, a.tokens_each);
  if (threadIdx.x < 64) find_slots(a, first, tokens, slots);
  __syncthreads();
  const int per = a.head_dim / kPer, row = a.kv_heads * per, items = tokens * row;
  for (int base = threadIdx.x; base < items; base += 256 * kItems) {
    float x[kItems][2][kPer];
    int64_t at[kItems], to[2][kItems];
    bool is[kItems];
#pragma unroll
    for (int i = 0; i < kItems; i++) {
      const int item = base + 256 * i;
      is[i] = item < items;
      const int token = (is[i] ? item : 0) / row, rest = (is[i] ? item : 0) - token * row;
      const int head = rest / per, d = (rest - head * per) * kPer;
      const int64_t slot = slots[token];
      at[i] = slot < 0 ? -1 : (slot + ((int64_t)head << a.page_shift)) * a.head_dim + d;
#pragma unroll
      for (int y = 0; y < 2; y++)
        to[y][i] = (int64_t)(first + token) * a.of[y].token_stride + head * a.of[y].head_stride + d;
    }
#pragma unroll
    for (int i = 0; i < kItems; i++)
#pragma unroll
      for (int y = 0; y < 2; y++) {
        if (kWrite ? is[i] : is[i] && at[i] >= 0) {
          if constexpr (kWrite) load_row<T, kPer>((const T*)a.of[y].rows + to[y][i], a.of[y].vector, x[i][y]);
          else load_page<kStore, kPer>(a.of[y], at[i], x[i][y]);
        } else {
#pragma unroll
          for (int j = 0; j < kPer; j++) x[i][y][j] = 0.f;
        }
      }
#pragma unroll
    for (int i = 0; i < kItems; i++)
#pragma unroll
      for (int y = 0; y < 2; y++) {
        if constexpr (kWrite) store_page<kStore, kPer>(a.of[y], is[i] ? at[i] : -1, x[i][y]);
        else if (is[i]) store_row<true>((T*)a.of[y].rows + to[y][i], a.of[y].vector, x[i][y]);
      }
  }
}

// ---------------------------------------------------------------------------- joining the parts
constexpr int kMostSplits = 256;

// Whether a packed row of ragged chunks belongs to a world's, and is not beyond max_count in it
__device__ inline bool covered(const Attend& a, int token) {
  int low = 0, high = a.nworld;
  while (high - low > 1) {
    const int middle = (low + high) >> 1;
    if (a.start[middle] <= token) low = middle; else high = middle;
  }
  const int place = token - a.start[low];
  return a.start[low] >= 0 && place >= 0 && token < a.start[low + 1] && place < a.max_count;
}

// A row's parts in the order of their keys, whatever order they were computed in.  kWaves of a workgroup's four take a
// row: they find the parts' maximum and shares together, then each thread adds up every kLanes-th part of four
// neighbouring values, and the threads' sums are joined in turn.  Four waves for the parts of a few rows; one
// where there are rows enough for all waves (us for whole calls, with four and with one: 19632 rows of 32 values in
// 7 parts 59 and 43, 60000 of 64 in 2 parts 170 and 124, 26880 of 128 in 3 parts 218 and 202).
constexpr int kRowsForWaves = 4096;
template <class T, int D, int kWaves>
__global__ __launch_bounds__(256) void join_parts(const Attend a) {
  constexpr int kQuads = D / 4, kLanes = 64 * kWaves / kQuads, kTeams = 4 / kWaves;
  constexpr int kMost = kWaves == 1 ? 64 : kMostSplits;
  __shared__ float sh_share[kTeams][kMost];
  __shared__ __attribute__((aligned(16))) f4 sh_o[kTeams][kLanes][kQuads];
  const int team = kWaves == 1 ? threadIdx.x >> 6 : 0, thread = kWaves == 1 ? threadIdx.x & 63 : threadIdx.x;
  const auto meet = [] {
    if constexpr (kWaves == 1) {
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    } else {
      __syncthreads();
    }
  };
  float* share = sh_share[team];
  f4(*o)[kQuads] = sh_o[team];
  const int64_t at = (int64_t)blockIdx.x * kTeams + team, sums = (int64_t)a.part_rows / a.heads * a.part_heads;
  if (at >= sums) return;
  int token = (int)(at / a.part_heads);                 // see part_row()
  const int h = (int)(at - (int64_t)token * a.part_heads) + a.part_first;
  const int64_t row = (int64_t)token * a.heads + h, rows = a.part_rows;
  if (!a.start) token += token / a.max_count * (a.count - a.max_count);
  else if (!covered(a, token)) return;                  // has no parts
  const int lane = threadIdx.x & 63;
  f2 ml[kMost / 64];
  float most = -INFINITY;
#pragma unroll
  for (int i = 0; i < kMost / 64; i++) {                // every wave, all parts
    const int s = lane + 64 * i;
    ml[i] = s < a.splits ? *(const f2*)(a.part_ml + 2 * (s * rows + row)) : f2{-INFINITY, 0.f};
    most = fmaxf(most, ml[i][0]);
  }
#pragma unroll
  for (int x = 1; x < 64; x *= 2) most = fmaxf(most, __shfl_xor(most, x));
  const float zero = most == -INFINITY ? 0.f : most;
  float l = 0.f;
#pragma unroll
  for (int i = 0; i < kMost / 64; i++) {
    // a part without a key of its own has no sums: they were not written
    const float w = ml[i][1] == 0.f ? 0.f : __builtin_amdgcn_exp2f(ml[i][0] - zero);
    l += ml[i][1] * w;
    if (thread < 64) share[lane + 64 * i] = ml[i][1] == 0.f ? -1.f : w;
  }
#pragma unroll
  for (int x = 1; x < 64; x *= 2) l += __shfl_xor(l, x);
  meet();
  const int quad = thread % kQuads, first = thread / kQuads;
  f4 sum = f4{0.f, 0.f, 0.f, 0.f};
  if (first < kLanes)
#pragma unroll 4
    for (int s = first; s < a.splits; s += kLanes) {
      const float w = share[s];
      if (w != -1.f) sum += rescaled(*(const f4*)(a.part + (s * sums + at) * D + 4 * quad), w);
    }
  if (first < kLanes) o[first][quad] = sum;
  meet();
  if (thread < kQuads) {
#pragma unroll
    for (int i = 1; i < kLanes; i++) sum += o[i][quad];
    const float inverse = 1.f / l;
    T* to = (T*)a.out + (int64_t)token * a.o_token + (int64_t)h * a.o_head + 4 * quad;
#pragma unroll
    for (int e = 0; e < 4; e++) to[e] = (T)(l == 0.f ? 0.f : sum[e] * inverse);
  }
  if (a.lse && thread == 0) a.lse[(int64_t)token * a.heads + h] = l == 0.f ? -INFINITY : (most + __builtin_amdgcn_logf(l)) * kLn2;
}

// ---------------------------------------------------------------------------- host side
int size_of(int type) { return type == MX_TYPE_F32 ? 4 : type == MX_TYPE_FP8 ? 1 : 2; }

int pages_check(const MxPages* p) {
  if (!p || !p->k || !p->v || !p->table || !p->length) return MX_ERR_INVALID;
  if (p->nworld < 1 || p->npage < 1 || p->width < 1 || p->kv_heads < 1) return MX_ERR_INVALID;
  if (p->type != MX_TYPE_BF16 && p->type != MX_TYPE_F16 && p->type != MX_TYPE_FP8) return MX_ERR_INVALID;
  if (p->type == MX_TYPE_FP8 && (!p->k_scale || !p->v_scale)) return MX_ERR_INVALID;
  const int d = p->head_dim, t = p->page_tokens;
  if (d != 32 && d != 64 && d != 96 && d != 128 && d != 256) return MX_ERR_DOMAIN;
  if (t < 16 || t > 4096 || (t & (t - 1)) || p->kv_heads > 1024) return MX_ERR_DOMAIN;
  if ((int64_t)p->npage * t > INT32_MAX || (int64_t)p->width * t > 1 << 30) return MX_ERR_DOMAIN;
  if (((uintptr_t)p->k | (uintptr_t)p->v) & 15) return MX_ERR_INVALID;
  return 0;
}

int chunk_check(const MxPages* p, const MxChunk* c) {
  if (!c || c->tokens < 0) return MX_ERR_INVALID;
  if (!c->start && (c->count < 0 || (int64_t)c->count * p->nworld != c->tokens)) return MX_ERR_INVALID;
  return 0;
}

bool rows_aligned(const MxRows* r, int bytes) {
  const int64_t s = size_of(r->type);
  return !(((uintptr_t)r->data | (uintptr_t)(r->token_stride * s) | (uintptr_t)(r->head_stride * s)) & (bytes - 1));
}

int rows_check(const MxRows* r, int heads, bool any) {
  if (!r || r->heads != heads) return MX_ERR_INVALID;
  if (any && (!r->data || ((uintptr_t)r->data & (size_of(r->type) - 1)))) return MX_ERR_INVALID;
  return 0;
}

int page_shift(const MxPages* p) { return __builtin_ctz(p->page_tokens); }

template <bool kWrite>
int move(const MxPages* p, const MxChunk* c, const MxRows* k, const MxRows* v, void* stream) {
  int rc = pages_check(p);
  if (rc || (rc = chunk_check(p, c))) return rc;
  const MxRows* rows[2] = {k, v};
  for (const MxRows* r : rows) {
    if ((rc = rows_check(r, p->kv_heads, c->tokens > 0))) return rc;
    if (r->type != MX_TYPE_F32 && r->type != MX_TYPE_BF16 && r->type != MX_TYPE_F16) return MX_ERR_INVALID;
  }
  if (k->type != v->type) return MX_ERR_INVALID;
  if (!c->tokens) return 0;
  // pieces of a token, and tokens of a workgroup
  const int size = size_of(k->type), pieces = p->kv_heads * p->head_dim * size / piece_bytes(p->type == MX_TYPE_FP8, kWrite, size);
  int each = 256 * pieces_ahead(size) / pieces;
  each = each < 1 ? 1 : each > kMostTokens || c->tokens / each >= kMostGroups ? kMostTokens : each;
  const int64_t groups = (c->tokens + (int64_t)each - 1) / each;
  if (groups > kMostGroups) return MX_ERR_DOMAIN;
  Move a{};
  uint8_t *pages[2] = {(uint8_t*)p->k, (uint8_t*)p->v}, *scales[2] = {p->k_scale, p->v_scale};
  for (int i = 0; i < 2; i++)
    a.of[i] = Copy{pages[i], scales[i], (const uint8_t*)rows[i]->data, rows[i]->token_stride, rows[i]->head_stride,
                   rows_aligned(rows[i], 16)};
  a.table = p->table; a.length = p->length; a.start = c->start;
  a.nworld = p->nworld; a.npage = p->npage; a.width = p->width; a.kv_heads = p->kv_heads;
  a.page_shift = page_shift(p); a.tokens = c->tokens; a.count = c->count;
  a.head_dim = p->head_dim; a.tokens_each = each;
  const dim3 grid((unsigned)groups);
  auto go = [&](auto t, auto store) {
    typedef decltype(t) T;
    constexpr int kStore = decltype(store)::value;
    hipLaunchKernelGGL((move_rows<T, kStore, kWrite>), grid, dim3(256), 0, (hipStream_t)stream, a);
  };
  auto by_store = [&](auto t) {
    if (p->type == MX_TYPE_FP8) go(t, std::integral_constant<int, MX_TYPE_FP8>());
    else if (p->type == MX_TYPE_BF16) go(t, std::integral_constant<int, MX_TYPE_BF16>());
    else go(t, std::integral_constant<int, MX_TYPE_F16>());
  };
  if (k->type == MX_TYPE_F32) by_store(0.f);
  else if (k->type == MX_TYPE_BF16) by_store((__bf16)0.f);
  else by_store((_Float16)0.f);
  return (int)hipGetLastError();
}

// Checks, and the launch: which kernel, how many tiles, how the keys are split
int choose(Attend& a, Launch& launch);
int plan(const MxPages* p, const MxChunk* c, const MxAttention* m, Attend& a, Launch& launch, bool pointers,
         const MxSelection* s, int block_shift) {
  int rc = pages_check(p);
  if (rc || (rc = chunk_check(p, c))) return rc;
  if (!m) return MX_ERR_INVALID;
  const int heads = m->q.heads;
  if (heads < 1 || heads % p->kv_heads || m->max_count < 0 || m->window < 0 || m->longest < 0) return MX_ERR_INVALID;
  if (heads / p->kv_heads > 1024) return MX_ERR_DOMAIN;
  if ((rc = rows_check(&m->q, heads, pointers && c->tokens > 0)) || (rc = rows_check(&m->out, heads, pointers && c->tokens > 0)))
    return rc;
  if (m->q.type != MX_TYPE_BF16 && m->q.type != MX_TYPE_F16) return MX_ERR_INVALID;
  if (m->out.type != m->q.type || (p->type != MX_TYPE_FP8 && p->type != m->q.type)) return MX_ERR_INVALID;
  if (!(fabsf(m->scale) * kLog2e < INFINITY)) return MX_ERR_INVALID;    // not finite, or not in base two
  a.k = (const uint8_t*)p->k; a.v = (const uint8_t*)p->v; a.k_scale = p->k_scale; a.v_scale = p->v_scale;
  a.table = p->table; a.length = p->length; a.start = c->start;
  a.q = m->q.data; a.out = m->out.data; a.lse = m->lse;
  a.q_token = m->q.token_stride; a.q_head = m->q.head_stride;
  a.o_token = m->out.token_stride; a.o_head = m->out.head_stride;
  a.nworld = p->nworld; a.npage = p->npage; a.width = p->width; a.kv_heads = p->kv_heads;
  a.page_shift = page_shift(p); a.tokens = c->tokens; a.count = c->count;
  a.heads = heads; a.group = heads / p->kv_heads;
  a.causal = m->causal != 0; a.window = m->window;
  // a scale of 0 becomes one that no score is noticed under: a hidden key's -infinity has to stay
  a.scale2 = fmaxf(fabsf(m->scale) * kLog2e, 1e-37f);
  a.negate = m->scale < 0.f;
  a.q_vector = rows_aligned(&m->q, 16);
  a.o_vector = rows_aligned(&m->out, 8);
  const int most = c->start ? m->max_count : (m->max_count < c->count ? m->max_count : c->count);
  a.max_count = most < c->tokens ? most : c->tokens;
  launch.tiles = 0;
  if (!c->tokens || !a.max_count) return 0;
  if ((int64_t)a.max_count * a.group > INT32_MAX || (int64_t)c->tokens * heads > INT32_MAX) return MX_ERR_DOMAIN;
  launch.type = m->q.type;
  launch.fp8 = p->type == MX_TYPE_FP8;
  launch.head_dim = p->head_dim;
  launch.keys = (int64_t)p->width << a.page_shift;
  if (m->longest && m->longest < launch.keys) launch.keys = m->longest;
  launch.held = launch.keys;
  if (s) {
    launch.listed = true;
    a.blocks = s->blocks; a.lists = s->width; a.block_shift = block_shift;
    launch.keys = (int64_t)s->width << block_shift;
  }
  return choose(a, launch);
}

// Whether rows are gathered by the blocks that they share, so that a block's keys and values are read for up to 128
// rows at once and each row has as many parts as its list has entries, which are written and read again in 32 bits.  By
// what either way takes to an entry of a token and key head, in ns: 0.3 and 0.075 (8 bits: 0.095) for each KB of the
// block's keys and values, or 0.45 for each KB of the parts and 10 for each tile, a tenth more for marking and listing.
// us, gathered and not, of 128 values in bfloat16 but where said, 19 blocks of 64 tokens listed: 2048 tokens over
// 65536, 32 heads on 8, 475 and 911 (8-bit pages 443 and 555), 512 tokens 171 and 234, 256 tokens 124 and 123; 4 x 1024
// over 8192, 8 heads on 8, 265 and 1482, 32 on 4, 858 and 758, 32 on 8 of 256 values 1171 and 3808; 16 x 256 over 8192,
// 16 on 4 of 64 values, 172 and 262 (163 and 201); 64 x 64 over 4096 205 and 240; 300 x 41 over 1024, 12 on 4 of 96
// values, blocks of 32, 631 and 533.  How many tokens share a block goes by the tokens that worlds have, as far as the caller
// knows, not by what the table could hold: 4 x 1024 tokens over 8192, 8 heads on 8, in tables for 524288: 434 and 1518.
constexpr int64_t kMostParts = 1 << 25, kMostBytes = 1 << 30, kBatchBytes = 192 << 20;
bool choose_gathered(Attend& a, Launch& launch) {
  const int64_t blocks = (int64_t)a.width << (a.page_shift - a.block_shift), block = 1LL << a.block_shift;
  const int64_t tokens = a.start ? a.tokens : (int64_t)a.nworld * a.max_count, rows = tokens * a.heads;
  if (a.lists < 2 || a.lists > kMostSplits || a.group > kManyRows || rows > INT32_MAX) return false;
  const int many = kManyRows / a.group;
  const int64_t held = (launch.held + block - 1) >> a.block_shift;                  // blocks that a world has
  const double share = (double)tokens * a.lists / ((double)a.nworld * held);        // tokens to a block
  const double kb = 2.0 * block * launch.head_dim * (launch.fp8 ? 1 : 2) / 1024, part_kb = 4.0 * a.group * launch.head_dim / 1024;
  // the marks, written and read once: 32 tokens of a world to a word, whatever is known of the chunks' sizes
  const int64_t words = a.start ? tokens / 32 + a.nworld : a.nworld * ((a.max_count + 31LL) / 32);
  const double marks_kb = 4.0 * words * blocks * a.kv_heads / 1024, marked_kb = 2.0 * marks_kb / ((double)tokens * a.lists * a.kv_heads);
  // a tile for each full set of rows of a key head, and one that is not full for each block that is listed; as the table may
  // hold more blocks than the worlds are known to have, there are workgroups for tiles that never are (0.7 ns each)
  const int64_t entries = tokens * a.lists;
  const auto tiles_of = [&](int64_t blocks) { return entries / many + (a.nworld * blocks < entries ? a.nworld * blocks : entries); };
  const int64_t head_tiles = tiles_of(blocks), tiles = head_tiles * a.kv_heads;
  const double gathered = 1.1 * (0.45 * part_kb + 10.0 * ceil(share / many) / share) + 0.25 * marked_kb
                          + 0.7 * (head_tiles - tiles_of(held)) / entries;
  if (gathered > 0.3 + (launch.fp8 ? 0.095 : 0.075) * kb) return false;
  const int64_t head_bytes = tokens * a.group * a.lists * launch.head_dim * 4;      // of a key head's sums
  if (rows * a.lists > kMostParts || head_bytes > kMostBytes || marks_kb > kMostBytes / 1024) return false;
  if (tiles * many > kMostBytes / 4) return false;                                  // their tokens
  if (tiles > kMostGroups || words * a.kv_heads > kMostGroups || a.nworld * (blocks / 16 + 1) * a.kv_heads > kMostGroups) return false;
  launch.gathered = true;
  launch.rows = kManyRows;
  launch.tiles = (int)tiles;
  a.splits = a.lists;
  a.part_rows = (int)rows;
  // so many key heads at a time that their parts are still in the last cache when they are joined
  const int64_t batches = (head_bytes * a.kv_heads + kBatchBytes - 1) / kBatchBytes;
  a.batch_heads = batches >= a.kv_heads ? 1 : (int)((a.kv_heads + batches - 1) / batches);
  a.words = (a.max_count + 31) / 32;
  a.words_all = (int)words;
  a.world_blocks = (int)blocks;
  a.tiles_most = (int)head_tiles * a.batch_heads;
  a.tiles = a.tiles_most;
  launch.grid = (unsigned)a.tiles_most;
  return true;
}

// Which kernel, by the rows that share a key head's keys and values.  us for 300 worlds of up to 700 tokens, 4 key
// heads of 128 values, with 12, 24, 48 rows: attend_few of 16 rows 52, 75, 101 in bfloat16 and 32, 48, 66 with 8-bit
// pages, of 32 rows (8-bit pages only) 42, 44, 77, attend_many 57, 59, 63 and 54, 55, 60;
// worlds of up to 512 tokens and heads of 256 values, with 12, 24, 48 rows: attend_few of 16 rows 106, 183, 265
// and 75, 140, 204, of 32 rows 129, 137, 240, attend_many 122, 124, 131 and 136, 137, 143.
//
// Into how many parts each tile's keys are split: where the tiles leave room, as many as the card holds
// workgroups at once (two per CU, four where heads of up to 64 values leave the registers), unless one
// workgroup is done with its keys in about the time that a second launch to join the parts takes.  Two
// worlds of up to 131072 quantised tokens, 8 key heads of 128 values: 256 workgroups 77.9 us, 512 54.0, 1024
// 55.5, 2048 63.1; heads of 64: 512 35.4, 1024 30.7, 2048 33.1.
//
// How many waves of attend_few share a tile: four, but one where there are waves' worth of tiles and their keys are few
// (most of four waves would have none, and wait for each other).  us with four and one, up to 64, 256 and 400 keys:
// 16384 tiles of 64 values, 8 bits, 66 and 27, 88 and 63, 109 and 94; 4096 tiles of 128 values, bfloat16, 43 and 20,
// 70 and 60, 92 and 90; 2048 of those 23 and 12, 39 and 36, 50 and 53; 512 of them 10.8 and 10.9, 11.4 and 16.7, 15 and 23.
constexpr int kShort = 256, kPlenty = 2048;
int choose(Attend& a, Launch& launch) {
  if (launch.listed && choose_gathered(a, launch)) return 0;
  const int64_t rows = launch.listed ? a.group : (int64_t)a.max_count * a.group;
  const bool few = rows <= (launch.fp8 ? 32 : 16);
  launch.blocks = rows <= 16 || (launch.listed && !launch.fp8) ? 1 : 2;
  launch.rows = few || launch.listed ? 16 * launch.blocks : kManyRows;
  const int64_t tiles = launch.listed ? ((rows + launch.rows - 1) / launch.rows) * (a.start ? a.tokens : (int64_t)a.nworld * a.max_count)
                      : a.start ? (int64_t)a.tokens * a.group / launch.rows + a.nworld
                                : ((rows + launch.rows - 1) / launch.rows) * a.nworld;
  int64_t keys = launch.keys;
  if (a.window > 0 && a.causal) {
    const int64_t spanned = (int64_t)a.window + launch.rows / a.group + 1;
    keys = keys < spanned ? keys : spanned;
  }
  const int64_t groups = tiles * a.kv_heads;
  const int room = launch.head_dim <= 64 ? 1024 : 512;
  int64_t splits = keys * (launch.head_dim > 64 ? launch.head_dim : 64) <= 131072 ? 1 : (room + groups - 1) / groups;
  const int64_t most = (keys + 63) / kLeastKeys + 1;     // the first key goes down to a multiple of 64
  splits = splits < most ? splits : most;
  if (splits > kMostSplits) splits = kMostSplits;
  if (groups * splits > kMostGroups) return MX_ERR_DOMAIN;
  launch.team = splits == 1 && keys <= kShort && groups >= kPlenty ? 1 : 4;
  a.tiles = (int)tiles;
  a.splits = (int)splits;
  a.part_heads = a.heads;
  // with parts there are fewer tiles than `room`, so at most 1024 of 128 rows
  a.part_rows = splits > 1 ? (a.start ? a.tokens : a.nworld * a.max_count) * a.heads : 0;
  launch.tiles = a.tiles;
  launch.grid = (unsigned)(groups * splits);
  return 0;
}

// Batches of key heads whose rows are gathered one after the other
int batches_of(const Attend& a) { return (a.kv_heads + a.batch_heads - 1) / a.batch_heads; }

// The workspace: sums, (maximum, sum of weights) of each part, and for gathered rows the tiles' numbers, tiles, their
// rows and marks.  Of a chunk whose sizes the host does not know it is as large as of one that it knows.
struct Workspace {
  size_t ml, counts, tiles, rows, marks, bytes;
};
Workspace workspace_for(const Attend& a, const Launch& launch) {
  Workspace w{};
  const size_t parts = (size_t)a.splits * a.part_rows;
  if (!launch.gathered) {
    w.ml = parts * launch.head_dim * sizeof(float);
    w.bytes = w.ml + parts * 2 * sizeof(float);
    return w;
  }
  const auto after = [](size_t at, size_t bytes) { return (at + bytes + 15) & ~(size_t)15; };
  const size_t batches = batches_of(a), tiles = batches * a.tiles_most;
  w.ml = after(0, (size_t)a.splits * (a.part_rows / a.heads) * a.batch_heads * a.group * launch.head_dim * sizeof(float));
  w.counts = after(w.ml, parts * 2 * sizeof(float));
  w.tiles = after(w.counts, batches * sizeof(int));
  w.rows = after(w.tiles, tiles * sizeof(int4));
  w.marks = after(w.rows, tiles * (kManyRows / a.group) * sizeof(int));
  w.bytes = after(w.marks, (size_t)a.kv_heads * a.words_all * a.world_blocks * sizeof(unsigned));
  return w;
}

size_t workspace_of(const Attend& a, const Launch& launch) {
  return !launch.tiles || a.splits < 2 ? 0 : workspace_for(a, launch).bytes;
}

int launch_attend(const Attend& a, const Launch& launch, void* stream) {
  return launch.head_dim == 32 ? attend32(a, launch, stream)
       : launch.head_dim == 64 ? attend64(a, launch, stream)
       : launch.head_dim == 96 ? attend96(a, launch, stream)
       : launch.head_dim == 128 ? attend128(a, launch, stream)
                                : attend256(a, launch, stream);
}

// The attention's launches, and those which join the parts
int launch_join(const Attend& a, const Launch& launch, void* stream) {
  const int64_t rows = (int64_t)a.part_rows / a.heads * a.part_heads;
  const bool one = rows >= kRowsForWaves && a.splits <= 64;
  const dim3 grid((unsigned)(one ? (rows + 3) / 4 : rows));
  const auto join = [&](auto d) {
    constexpr int D = decltype(d)::value;
    const auto go = [&](auto t, auto waves) {
      hipLaunchKernelGGL((join_parts<decltype(t), D, decltype(waves)::value>), grid, dim3(256), 0, (hipStream_t)stream, a);
    };
    const auto by_rows = [&](auto t) {
      if (one) go(t, std::integral_constant<int, 1>());
      else go(t, std::integral_constant<int, 4>());
    };
    if (launch.type == MX_TYPE_BF16) by_rows((__bf16)0.f);
    else by_rows((_Float16)0.f);
  };
  switch (launch.head_dim) {
    case 32: join(std::integral_constant<int, 32>()); break;
    case 64: join(std::integral_constant<int, 64>()); break;
    case 96: join(std::integral_constant<int, 96>()); break;
    case 128: join(std::integral_constant<int, 128>()); break;
    default: join(std::integral_constant<int, 256>());
  }
  return (int)hipGetLastError();
}

int attend_planned(Attend& a, const Launch& launch, const MxAttention* m, void* stream) {
  const size_t bytes = workspace_of(a, launch);
  if (bytes) {
    if (!m->workspace || m->workspace_bytes < bytes || ((uintptr_t)m->workspace & 15)) return MX_ERR_WORKSPACE;
    const Workspace w = workspace_for(a, launch);
    uint8_t* at = (uint8_t*)m->workspace;
    a.part = (float*)at;
    a.part_ml = (float*)(at + w.ml);
    a.gathered_tiles = (int*)(at + w.counts);
    a.gathered = (int4*)(at + w.tiles);
    a.gathered_rows = (int*)(at + w.rows);
    a.marks = (unsigned*)(at + w.marks);
  }
  if (!launch.gathered) {
    const int rc = launch_attend(a, launch, stream);
    return rc || a.splits < 2 ? rc : launch_join(a, launch, stream);
  }
  int rc = gather_rows(a, launch, stream);
  for (a.batch = 0; !rc && a.batch < batches_of(a); a.batch++) {
    const int first = a.batch * a.batch_heads, heads = a.kv_heads - first < a.batch_heads ? a.kv_heads - first : a.batch_heads;
    a.part_first = first * a.group;
    a.part_heads = heads * a.group;
    rc = launch_attend(a, launch, stream);
    if (!rc) rc = launch_join(a, launch, stream);
  }
  return rc;
}

}  // namespace mxe

extern "C" {

size_t mx_pages_bytes(void) { return sizeof(MxPages); }
size_t mx_chunk_bytes(void) { return sizeof(MxChunk); }
size_t mx_rows_bytes(void) { return sizeof(MxRows); }
size_t mx_attention_bytes(void) { return sizeof(MxAttention); }

int mx_episode_write(const MxPages* pages, const MxChunk* chunk, const MxRows* k, const MxRows* v, void* stream) {
  return mxe::move<true>(pages, chunk, k, v, stream);
}

int mx_episode_read(const MxPages* pages, const MxChunk* chunk, const MxRows* k, const MxRows* v, void* stream) {
  return mxe::move<false>(pages, chunk, k, v, stream);
}

size_t mx_episode_workspace(const MxPages* pages, const MxChunk* chunk, const MxAttention* m) {
  mxe::Attend a{};
  mxe::Launch launch{};
  return mxe::plan(pages, chunk, m, a, launch, false) ? 0 : mxe::workspace_of(a, launch);
}

int mx_episode_attend(const MxPages* pages, const MxChunk* chunk, const MxAttention* m, void* stream) {
  mxe::Attend a{};
  mxe::Launch launch{};
  const int rc = mxe::plan(pages, chunk, m, a, launch, true);
  return rc || !launch.tiles ? rc : mxe::attend_planned(a, launch, m, stream);
}

}
