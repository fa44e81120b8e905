// The episode memory's entry points: writing to and reading from the pages, joining the parts of a
// split attention, and the host side of all four calls.
#include <cmath>
#include <type_traits>
#include "mx_episode_types.h"
#include "mx_episode_launch.h"

namespace mxe {

// ---------------------------------------------------------------------------- write and read
struct Copy {
  uint8_t *pages, *scales;       // of k (blockIdx.y = 0) or v
  const uint8_t* rows;
  int64_t token_stride, head_stride;
  bool vector;                   // rows are 16-byte aligned
};
struct Move {
  Copy of[2];
  const int32_t *table, *length, *start;
  int nworld, npage, width, kv_heads, page_shift, tokens, count;
};

// The slot of packed row `token`, as (page * kv_heads * page_tokens + slot) without the head; -1: none
__device__ inline int64_t slot_of(const Move& a, int token) {
  int world, place, count;
  if (!a.start) {
    world = token / a.count;
    place = token - world * a.count;
    count = a.count;
  } else {
    int low = 0, high = a.nworld;
    while (high - low > 1) {
      const int middle = (low + high) >> 1;
      if (a.start[middle] <= token) low = middle; else high = middle;
    }
    world = low;
    place = token - a.start[low];
    count = a.start[low + 1] - a.start[low];
    if (place < 0 || place >= count) return -1;
  }
  const int position = max(a.length[world], 0) - count + place;
  if (position < 0 || (position >> a.page_shift) >= a.width) return -1;
  const int page = a.table[(int64_t)world * a.width + (position >> a.page_shift)];
  if ((unsigned)page >= (unsigned)a.npage) return -1;
  return (((int64_t)page * a.kv_heads) << a.page_shift) + (position & ((1 << a.page_shift) - 1));
}

template <class T> __device__ inline void load8(const T* from, bool vector, float (&x)[8]) {
  if (vector) {
    if constexpr (sizeof(T) == 4) {
      const f4 a = *(const f4*)from, b = *(const f4*)(from + 4);
#pragma unroll
      for (int j = 0; j < 4; j++) x[j] = a[j], x[4 + j] = b[j];
    } else {
      typedef T T8 __attribute__((ext_vector_type(8)));
      const T8 a = *(const T8*)from;
#pragma unroll
      for (int j = 0; j < 8; j++) x[j] = (float)a[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; j++) x[j] = (float)from[j];
  }
}

// One thread moves eight values of one head of one token; the four threads of a scale's block are
// neighbours.  Bound by memory; nothing is shared, so threads go in the order of the rows.
template <class T, int kStore>
__global__ __launch_bounds__(256) void write_rows(const Move a, int head_dim) {
  const Copy c = a.of[blockIdx.y];
  const int per = head_dim / 8;
  const int64_t item = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = item / per;
  const int d = (int)(item - row * per) * 8;
  const int64_t token = row / a.kv_heads;
  const int head = (int)(row - token * a.kv_heads);
  if (token >= a.tokens) return;                        // whole blocks of four threads leave together
  const int64_t slot = slot_of(a, (int)token);
  if (slot < 0) return;
  float x[8];
  load8((const T*)c.rows + token * c.token_stride + head * c.head_stride + d, c.vector, x);
  const int64_t at = slot + ((int64_t)head << a.page_shift);
  if constexpr (kStore == MX_TYPE_FP8) {
    // the largest magnitude of the block, as the bits of a float that is not negative: they order
    // like integers, infinities and NaN above all numbers
    unsigned top = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) top = max(top, __float_as_uint(x[j]) & 0x7fffffffu);
    top = max(top, (unsigned)__shfl_xor((int)top, 1));
    top = max(top, (unsigned)__shfl_xor((int)top, 2));
    // 448 = 1.75 * 2^8: the exponent less 8, and one more above a fraction of 1.75
    const bool finite = top < 0x7f800000u;
    const int e = max((int)(top >> 23) - 127 - 8 + ((top & 0x7fffffu) > 0x600000u), -117);
    const float inverse = __uint_as_float((unsigned)(127 - e) << 23);
    if (!finite)
#pragma unroll
      for (int j = 0; j < 8; j++) x[j] = 0.f;
    u2 w;
    unsigned y = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * inverse, x[1] * inverse, 0, false);
    w.x = __builtin_amdgcn_cvt_pk_fp8_f32(x[2] * inverse, x[3] * inverse, y, true);
    y = __builtin_amdgcn_cvt_pk_fp8_f32(x[4] * inverse, x[5] * inverse, 0, false);
    w.y = __builtin_amdgcn_cvt_pk_fp8_f32(x[6] * inverse, x[7] * inverse, y, true);
    *(u2*)(c.pages + at * head_dim + d) = w;
    if ((d & 31) == 0) c.scales[at * (head_dim / 32) + d / 32] = finite ? (uint8_t)(e + 127) : 255;
  } else {
    typedef typename Elem<kStore>::T S;
    typename Elem<kStore>::V8 y;
#pragma unroll
    for (int j = 0; j < 8; j++) y[j] = (S)x[j];
    *(typename Elem<kStore>::V8*)((S*)c.pages + at * head_dim + d) = y;
  }
}

template <class T, int kStore>
__global__ __launch_bounds__(256) void read_rows(const Move a, int head_dim) {
  const Copy c = a.of[blockIdx.y];
  const int per = head_dim / 8;
  const int64_t item = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = item / per;
  const int d = (int)(item - row * per) * 8;
  const int64_t token = row / a.kv_heads;
  const int head = (int)(row - token * a.kv_heads);
  if (token >= a.tokens) return;
  const int64_t slot = slot_of(a, (int)token);
  float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (slot >= 0) {
    const int64_t at = slot + ((int64_t)head << a.page_shift);
    if constexpr (kStore == MX_TYPE_FP8) {
      const u2 w = *(const u2*)(c.pages + at * head_dim + d);
      const unsigned byte = c.scales[at * (head_dim / 32) + d / 32];
      const float scale = byte == 255 ? NAN : __uint_as_float(byte ? byte << 23 : 0x400000u);
      const f2 p = __builtin_amdgcn_cvt_pk_f32_fp8(w.x, false), q = __builtin_amdgcn_cvt_pk_f32_fp8(w.x, true);
      const f2 r = __builtin_amdgcn_cvt_pk_f32_fp8(w.y, false), s = __builtin_amdgcn_cvt_pk_f32_fp8(w.y, true);
      x[0] = p[0] * scale; x[1] = p[1] * scale; x[2] = q[0] * scale; x[3] = q[1] * scale;
      x[4] = r[0] * scale; x[5] = r[1] * scale; x[6] = s[0] * scale; x[7] = s[1] * scale;
    } else {
      load8((const typename Elem<kStore>::T*)c.pages + at * head_dim + d, true, x);
    }
  }
  T* to = (T*)c.rows + token * c.token_stride + head * c.head_stride + d;
  if (c.vector) {
    if constexpr (sizeof(T) == 4) {
      *(f4*)to = f4{x[0], x[1], x[2], x[3]};
      *(f4*)(to + 4) = f4{x[4], x[5], x[6], x[7]};
    } else {
      typedef T T8 __attribute__((ext_vector_type(8)));
      T8 y;
#pragma unroll
      for (int j = 0; j < 8; j++) y[j] = (T)x[j];
      *(T8*)to = y;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; j++) to[j] = (T)x[j];
  }
}

// ---------------------------------------------------------------------------- joining the parts
// Whether a packed row belongs to a world's chunk, and is not beyond max_count in it
__device__ inline bool covered(const Attend& a, int token) {
  if (!a.start) return token % a.count < a.max_count;
  int low = 0, high = a.nworld;
  while (high - low > 1) {
    const int middle = (low + high) >> 1;
    if (a.start[middle] <= token) low = middle; else high = middle;
  }
  const int place = token - a.start[low];
  return a.start[low] >= 0 && place >= 0 && token < a.start[low + 1] && place < a.max_count;
}

// A row's parts in the order of their keys, whatever order they were computed in: a wave takes every
// fourth part of a row with its lanes along head_dim, then the four waves' sums are joined.
template <class T>
__global__ __launch_bounds__(256) void join_parts(const Attend a, int head_dim) {
  __shared__ float o[4][256], ls[4];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t row = blockIdx.x, rows = (int64_t)a.tokens * a.heads;
  // rows that no tile covers (no world's chunk, or beyond max_count) have no parts
  const int64_t token = row / a.heads;
  const int h = (int)(row - token * a.heads);
  if (!covered(a, (int)token)) return;
  float most = -INFINITY;
  for (int s = 0; s < a.splits; s++) most = fmaxf(most, a.part_ml[2 * (s * rows + row)]);
  const float zero = most == -INFINITY ? 0.f : most;
  float sum[4] = {0.f, 0.f, 0.f, 0.f}, l = 0.f;
  for (int s = wave; s < a.splits; s += 4) {
    const int64_t at = s * rows + row;
    const f2 ml = *(const f2*)(a.part_ml + 2 * at);
    if (ml[1] == 0.f) continue;                         // no key of its own: its sums were not written
    const float share = __builtin_amdgcn_exp2f(ml[0] - zero);
    l += ml[1] * share;
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (lane + 64 * j < head_dim) sum[j] += a.part[at * head_dim + lane + 64 * j] * share;
  }
#pragma unroll
  for (int j = 0; j < 4; j++) o[wave][lane + 64 * j] = sum[j];
  if (lane == 0) ls[wave] = l;
  __syncthreads();
  const int d = threadIdx.x;
  l = (ls[0] + ls[1]) + (ls[2] + ls[3]);
  if (d < head_dim) {
    const float x = (o[0][d] + o[1][d]) + (o[2][d] + o[3][d]);
    ((T*)a.out)[token * a.o_token + (int64_t)h * a.o_head + d] = (T)(l == 0.f ? 0.f : x * (1.f / l));
  }
  if (a.lse && d == 0) a.lse[row] = l == 0.f ? -INFINITY : (most + __builtin_amdgcn_logf(l)) * kLn2;
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
  if ((int64_t)p->npage * t > INT32_MAX || (int64_t)p->width * t > INT32_MAX) return MX_ERR_DOMAIN;
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
  const int64_t items = (int64_t)c->tokens * p->kv_heads * (p->head_dim / 8);
  if ((items + 255) / 256 > INT32_MAX) return MX_ERR_DOMAIN;
  Move a{};
  uint8_t *pages[2] = {(uint8_t*)p->k, (uint8_t*)p->v}, *scales[2] = {p->k_scale, p->v_scale};
  for (int i = 0; i < 2; i++)
    a.of[i] = Copy{pages[i], scales[i], (const uint8_t*)rows[i]->data, rows[i]->token_stride, rows[i]->head_stride,
                   rows_aligned(rows[i], 16)};
  a.table = p->table; a.length = p->length; a.start = c->start;
  a.nworld = p->nworld; a.npage = p->npage; a.width = p->width; a.kv_heads = p->kv_heads;
  a.page_shift = page_shift(p); a.tokens = c->tokens; a.count = c->count;
  const dim3 grid((unsigned)((items + 255) / 256), 2);
  auto go = [&](auto t, auto store) {
    typedef decltype(t) T;
    if constexpr (kWrite)
      hipLaunchKernelGGL((write_rows<T, decltype(store)::value>), grid, dim3(256), 0, (hipStream_t)stream, a, p->head_dim);
    else
      hipLaunchKernelGGL((read_rows<T, decltype(store)::value>), grid, dim3(256), 0, (hipStream_t)stream, a, p->head_dim);
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
  if (heads < 1 || heads % p->kv_heads || m->max_count < 0 || m->window < 0) return MX_ERR_INVALID;
  if (heads / p->kv_heads > 1024) return MX_ERR_DOMAIN;
  if ((rc = rows_check(&m->q, heads, pointers && c->tokens > 0)) || (rc = rows_check(&m->out, heads, pointers && c->tokens > 0)))
    return rc;
  if (m->q.type != MX_TYPE_BF16 && m->q.type != MX_TYPE_F16) return MX_ERR_INVALID;
  if (m->out.type != m->q.type || (p->type != MX_TYPE_FP8 && p->type != m->q.type)) return MX_ERR_INVALID;
  if (!(m->scale - m->scale == 0.f)) return MX_ERR_INVALID;    // not finite
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
  return choose(a, launch);
}

// Keys that one row of tiles can see at most, and how they are split: enough workgroups for every CU
// to hold several, in shares of at least 256 keys.
int choose(Attend& a, Launch& launch) {
  const int64_t rows = (int64_t)a.max_count * a.group;
  launch.blocks = rows <= 16 ? 1 : rows <= 32 || launch.head_dim == 256 ? 2 : 4;
  launch.rows = 16 * launch.blocks;
  if (rows > 64 && launch.head_dim <= 128) launch.rows = kManyRows;
  const int64_t tiles = a.start ? (int64_t)a.tokens * a.group / launch.rows + a.nworld
                                : ((rows + launch.rows - 1) / launch.rows) * a.nworld;
  int64_t keys = (int64_t)a.width << a.page_shift;
  if (a.window > 0 && a.causal) {
    const int64_t spanned = (int64_t)a.window + launch.rows / a.group + 1;
    keys = keys < spanned ? keys : spanned;
  }
  keys += 31;                                            // the first key goes down to a multiple of 32
  const int64_t groups = tiles * a.kv_heads;
  int64_t splits = (1024 + groups - 1) / groups;
  const int64_t most = (keys + 255) / 256;
  splits = splits < most ? splits : most;
  const int64_t each = ((keys + splits - 1) / splits + 127) / 128 * 128;
  splits = (keys + each - 1) / each;
  if (groups * splits > INT32_MAX) return MX_ERR_DOMAIN;
  a.tiles = (int)tiles;
  a.splits = (int)splits;
  a.split_keys = (int)(each < INT32_MAX ? each : INT32_MAX);
  launch.tiles = a.tiles;
  launch.grid = (unsigned)(groups * splits);
  return 0;
}

size_t workspace_of(const Attend& a, const Launch& launch) {
  if (!launch.tiles || a.splits < 2) return 0;
  return (size_t)a.splits * a.tokens * a.heads * (launch.head_dim + 2) * sizeof(float);
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
    a.part_ml = a.part + (size_t)a.splits * a.tokens * a.heads * launch.head_dim;
  }
  const int started = launch.head_dim == 32 ? mxe::attend32(a, launch, stream)
                    : launch.head_dim == 64 ? mxe::attend64(a, launch, stream)
                    : launch.head_dim == 96 ? mxe::attend96(a, launch, stream)
                    : launch.head_dim == 128 ? mxe::attend128(a, launch, stream)
                                             : mxe::attend256(a, launch, stream);
  if (started || a.splits < 2) return started;
  const dim3 grid((unsigned)((int64_t)a.tokens * a.heads));
  if (launch.type == MX_TYPE_BF16)
    hipLaunchKernelGGL(mxe::join_parts<__bf16>, grid, dim3(256), 0, (hipStream_t)stream, a, launch.head_dim);
  else
    hipLaunchKernelGGL(mxe::join_parts<_Float16>, grid, dim3(256), 0, (hipStream_t)stream, a, launch.head_dim);
  return (int)hipGetLastError();
}

}
