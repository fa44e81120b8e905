// The episode memory's entry points: writing to and reading from the pages, joining the parts of a
// split attention, and the host side of all calls.  The attention itself: mx_episode_few.h, mx_episode_many.h.
#include <cmath>
#include <type_traits>
#include "mx_episode_types.h"
#include "mx_episode_launch.h"

namespace mxe {

// ---------------------------------------------------------------------------- write and read
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

// The slots of `tokens` (at most 64) packed rows from `first` on, by the lanes of one wave.  Ragged chunks:
// the first row's world by a search with 64 probes at a time, the others' from there, mostly the same.
__device__ inline void find_slots(const Move& a, int first, int tokens, int64_t* slots) {
  const int lane = threadIdx.x, token = first + lane;
  if (!a.start) {
    if (lane < tokens) {
      const int world = token / a.count;
      slots[lane] = slot_of(a, world, token - world * a.count, a.count);
    }
    return;
  }
  int low = 0, high = a.nworld;
  while (high - low > 1) {
    const int step = (high - low + 63) >> 6, probe = low + lane * step;
    const int passed = max(1, (int)__popcll(__ballot(probe < high && a.start[probe] <= first)));
    low += (passed - 1) * step;
    high = min(high, low + step);
  }
  if (lane < tokens) {
    if (a.start[low + 1] <= token) {
      high = a.nworld;
      while (high - low > 1) {
        const int middle = (low + high) >> 1;
        if (a.start[middle] <= token) low = middle; else high = middle;
      }
    }
    slots[lane] = slot_of(a, low, token - a.start[low], a.start[low + 1] - a.start[low]);
  }
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
  const int64_t row = (int64_t)blockIdx.x * kTeams + team, rows = a.part_rows;
  if (row >= rows) return;
  int token = (int)(row / a.heads);                     // see part_row()
  const int h = (int)(row - (int64_t)token * a.heads);
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
      if (w != -1.f) sum += rescaled(*(const f4*)(a.part + (s * rows + row) * D + 4 * quad), w);
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
int plan(const MxPages* p, const MxChunk* c, const MxAttention* m, Attend& a, Launch& launch, bool pointers) {
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
  return choose(a, launch);
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
  const int64_t rows = (int64_t)a.max_count * a.group;
  const bool few = rows <= (launch.fp8 ? 32 : 16);
  launch.blocks = rows <= 16 ? 1 : 2;
  launch.rows = few ? 16 * launch.blocks : kManyRows;
  const int64_t tiles = a.start ? (int64_t)a.tokens * a.group / launch.rows + a.nworld
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
  // with parts there are fewer tiles than `room`, so at most 1024 of 128 rows
  a.part_rows = splits > 1 ? (a.start ? a.tokens : a.nworld * a.max_count) * a.heads : 0;
  launch.tiles = a.tiles;
  launch.grid = (unsigned)(groups * splits);
  return 0;
}

size_t workspace_of(const Attend& a, const Launch& launch) {
  if (!launch.tiles || a.splits < 2) return 0;
  return (size_t)a.splits * a.part_rows * (launch.head_dim + 2) * sizeof(float);
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
  if (rc || !launch.tiles) return rc;
  const size_t bytes = mxe::workspace_of(a, launch);
  if (bytes) {
    if (!m->workspace || m->workspace_bytes < bytes || ((uintptr_t)m->workspace & 15)) return MX_ERR_WORKSPACE;
    a.part = (float*)m->workspace;
    a.part_ml = a.part + (size_t)a.splits * a.part_rows * launch.head_dim;
  }
  const int started = launch.head_dim == 32 ? mxe::attend32(a, launch, stream)
                    : launch.head_dim == 64 ? mxe::attend64(a, launch, stream)
                    : launch.head_dim == 96 ? mxe::attend96(a, launch, stream)
                    : launch.head_dim == 128 ? mxe::attend128(a, launch, stream)
                                             : mxe::attend256(a, launch, stream);
  if (started || a.splits < 2) return started;
  const int64_t rows = a.part_rows;
  const bool one = rows >= mxe::kRowsForWaves && a.splits <= 64;
  const dim3 grid((unsigned)(one ? (rows + 3) / 4 : rows));
  const auto join = [&](auto d) {
    constexpr int D = decltype(d)::value;
    const auto go = [&](auto t, auto waves) {
      hipLaunchKernelGGL((mxe::join_parts<decltype(t), D, decltype(waves)::value>), grid, dim3(256), 0, (hipStream_t)stream, a);
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

}
