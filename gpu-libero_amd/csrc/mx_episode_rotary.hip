// Rotary positions: rows turned by given positions, and a chunk's queries and keys turned by their places in their
// worlds, the keys on their way into the pages.
//
// A pair (x_a, x_b) of a row at position p turns by the angle p * turn: y_a = c x_a - s x_b, y_b = s x_a + c x_b.
// Three operations to a value that is read and written once: bound by memory, or, for a step's few rows, by the launch.
// A workgroup first computes cosines and sines of its tokens' pairs into LDS, once for all heads; then a thread takes
// 16 bytes of either half of a head (of a key its own 16 or 32 bytes, as the pages' scales want them, and reads the
// others beside).
//
// Prompts of 4 x 4096 tokens, 32 and 8 heads of 128 values, bfloat16 (403 MB): 72 us, 5.6 TB/s; float32 rows (738 MB): 132
// for the call.  67 prompts of up to 501 tokens, float16 into 8-bit pages, half of each head turned (116 MB): 28.7 us,
// 4.0 TB/s.  4096 single tokens into 8-bit pages (25 MB): 10.3 us, which is a chain: starts, lengths, table and angles come
// before the first row is asked for.  16 x 1024 tokens of 16 heads of 64 values turned (67 MB, out of the last cache): 12.4
// us.
#include <type_traits>
#include "mx_episode_move.h"
#include "mx_episode_launch.h"

namespace mxe {

// Rows to be turned
struct Turned {
  const void* x;
  void* out;
  const double* turn;
  double amplitude;
  int64_t x_token, x_head, o_token, o_head;
  int heads, head_dim, half, tokens, each;      // half: pairs; each: tokens of a workgroup
  bool interleaved, back, pieces;               // pieces: of 16 bytes, that no pair's end cuts
};
struct Rotate {
  Turned t;
  const void* positions;
  int period;
  bool wide;
};
struct Enter {
  Turned t;
  Move m;
  int kv_groups;
};

constexpr int kMostTokens = 64;                 // of a workgroup: their positions are kept in LDS
constexpr int kMostAngles = 4096;               // of a workgroup, 8 bytes of LDS each

// Cosine and sine of `position` times `turn` radians, times `amplitude`, each rounded once from 64 bits: it then has no part
// in the error of what it turns.  In revolutions the angle is brought within an eighth of one, where six and seven terms of
// Taylor's series are off by less than 2^-36.
__device__ inline f2 cos_sin(double position, double turn, double amplitude) {
  const double t = position * (turn * 0.15915494309189535);
  const double quarters = __builtin_rint(t * 4.0);
  const double x = __builtin_fma(quarters, -0.25, t) * 6.283185307179586, y = x * x;
  const auto to = [&](double sum, double next) { return __builtin_fma(y, sum, next); };
  const double s = x * to(to(to(to(to(-1. / 39916800., 1. / 362880.), -1. / 5040.), 1. / 120.), -1. / 6.), 1.);
  const double c = to(to(to(to(to(to(1. / 479001600., -1. / 3628800.), 1. / 40320.), -1. / 720.), 1. / 24.), -0.5), 1.);
  const int quarter = (int)(quarters - 4.0 * __builtin_floor(quarters * 0.25)) & 3;
  const float a = (float)(amplitude * (quarter & 1 ? s : c)), b = (float)(amplitude * (quarter & 1 ? c : s));
  return f2{quarter == 1 || quarter == 2 ? -a : a, quarter & 2 ? -b : b};
}

// Those of all pairs of a workgroup's tokens
__device__ inline void angles(const Turned& t, int tokens, const double* position, f2* cs) {
  for (int i = threadIdx.x; i < tokens * t.half; i += 256) {
    const int token = i / t.half, pair = i - token * t.half;
    f2 x = cos_sin(position[token], t.turn[pair], t.amplitude);
    if (t.back) x.y = -x.y;
    cs[i] = x;
  }
}

// Each product and the sum are rounded to 32 bits by themselves: fused, a quarter of the sums would have another last
// bit than the same formula has elsewhere, and of float32 keys one in 50000 another neighbour in bfloat16 pages (in float16
// one in 8700).  Two instructions more to a pair are not seen beside the memory: 4 x 4096 tokens' 32 and 8 heads of 128
// values, whole calls, bfloat16 74.3 us fused and not, float32 132.1 and 132.3.
__device__ inline f2 turned(f2 x, f2 cs) {
#pragma clang fp contract(off)
  return f2{x.x * cs.x - x.y * cs.y, x.x * cs.y + x.y * cs.x};
}

// The workgroup's tokens from `first` on, of which those whose position is no number are left out
template <class T>
__device__ inline void turn_rows(const Turned& a, int first, int tokens, const double* position, const f2* cs) {
  constexpr int N = 16 / sizeof(T);
  const int half = a.half, rest = a.head_dim - 2 * half;
  const int pairs = a.pieces ? (a.interleaved ? 0 : half / N) : half;             // of a head, then its single pieces
  const int per = pairs + (a.pieces ? (a.interleaved ? a.head_dim : rest) / N : rest);
  const int row = a.heads * per, items = tokens * row;
  for (int item = threadIdx.x; item < items; item += 256) {
    const int token = item / row, in_row = item - token * row, head = in_row / per, piece = in_row - head * per;
    if (position[token] != position[token]) continue;
    const T* x = (const T*)a.x + (int64_t)(first + token) * a.x_token + (int64_t)head * a.x_head;
    T* out = (T*)a.out + (int64_t)(first + token) * a.o_token + (int64_t)head * a.o_head;
    const f2* angle = cs + token * half;
    if (a.pieces) {
      if (piece < pairs) {                                  // of both halves
        const int d = piece * N;
        float u[N], v[N];
        load_row<T, N>(x + d, true, u);
        load_row<T, N>(x + half + d, true, v);
#pragma unroll
        for (int j = 0; j < N; j++) {
          const f2 y = turned(f2{u[j], v[j]}, angle[d + j]);
          u[j] = y.x;
          v[j] = y.y;
        }
        store_row<false, T, N>(out + d, true, u);
        store_row<false, T, N>(out + half + d, true, v);
      } else {
        const int d = (a.interleaved ? 0 : 2 * half) + (piece - pairs) * N;
        float u[N];
        load_row<T, N>(x + d, true, u);
        if (a.interleaved) {
#pragma unroll
          for (int j = 0; j < N; j += 2)
            if (d + j < 2 * half) {
              const f2 y = turned(f2{u[j], u[j + 1]}, angle[(d + j) / 2]);
              u[j] = y.x;
              u[j + 1] = y.y;
            }
        }
        store_row<false, T, N>(out + d, true, u);
      }
    } else if (piece < pairs) {
      const int i = a.interleaved ? 2 * piece : piece, j = a.interleaved ? i + 1 : i + half;
      const f2 y = turned(f2{(float)x[i], (float)x[j]}, angle[piece]);
      out[i] = (T)y.x;
      out[j] = (T)y.y;
    } else {
      out[half + piece] = x[half + piece];
    }
  }
}

template <class T>
__global__ __launch_bounds__(256) void rotate_rows(const Rotate a) {
  extern __shared__ __attribute__((aligned(16))) f2 cs[];
  __shared__ double position[kMostTokens];
  const int first = blockIdx.x * a.t.each, tokens = min(a.t.tokens - first, a.t.each);
  if (threadIdx.x < tokens) {
    const int at = (first + threadIdx.x) % a.period;
    position[threadIdx.x] = a.wide ? (double)((const int64_t*)a.positions)[at] : (double)((const int32_t*)a.positions)[at];
  }
  __syncthreads();
  angles(a.t, tokens, position, cs);
  __syncthreads();
  turn_rows<T>(a.t, first, tokens, position, cs);
}

// N values of a key from d on, turned: those that they turn with are read beside them
template <class T, int N>
__device__ inline void turn_piece(const Turned& a, const T* row, int d, bool vector, const f2* angle, float (&x)[N]) {
  const int half = a.half;
  if (a.interleaved) {
#pragma unroll
    for (int j = 0; j < N; j += 2)
      if (d + j < 2 * half) {
        const f2 y = turned(f2{x[j], x[j + 1]}, angle[(d + j) / 2]);
        x[j] = y.x;
        x[j + 1] = y.y;
      }
  } else if (half % N == 0) {
    if (d >= 2 * half) return;
    const bool low = d < half;
    const int pair = low ? d : d - half;
    float other[N];
    load_row<T, N>(row + (low ? d + half : pair), vector, other);
#pragma unroll
    for (int j = 0; j < N; j++) {
      const f2 y = turned(low ? f2{x[j], other[j]} : f2{other[j], x[j]}, angle[pair + j]);
      x[j] = low ? y.x : y.y;
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; j++) {
      const int at = d + j;
      if (at >= 2 * half) continue;
      const bool low = at < half;
      const int pair = low ? at : at - half;
      const float other = (float)row[low ? at + half : pair];
      const f2 y = turned(low ? f2{x[j], other} : f2{other, x[j]}, angle[pair]);
      x[j] = low ? y.x : y.y;
    }
  }
}

// The first workgroups take keys and values, the others queries: one launch for a step's rows
template <class T, int kStore>
__global__ __launch_bounds__(256) void enter_rows(const Enter a) {
  constexpr int N = piece_bytes(kStore == MX_TYPE_FP8, true, sizeof(T)) / sizeof(T);
  extern __shared__ __attribute__((aligned(16))) f2 cs[];
  __shared__ double position[kMostTokens];
  __shared__ int64_t slots[kMostTokens];
  const bool keys = (int)blockIdx.x < a.kv_groups;
  const int each = keys ? a.m.tokens_each : a.t.each;
  const int first = ((int)blockIdx.x - (keys ? 0 : a.kv_groups)) * each, tokens = min(a.m.tokens - first, each);
  if (threadIdx.x < 64) {
    const int world = world_of(a.m.start, a.m.nworld, a.m.count, first, tokens);
    if (world >= 0) {
      const int begin = a.m.start ? a.m.start[world] : world * a.m.count;
      const int count = a.m.start ? a.m.start[world + 1] - begin : a.m.count, place = first + (int)threadIdx.x - begin;
      const bool is = begin >= 0 && place >= 0 && place < count;
      position[threadIdx.x] = is ? (double)(max(a.m.length[world], 0) - count + place) : NAN;
      slots[threadIdx.x] = keys && is ? slot_of(a.m, world, place, count) : -1;
    }
  }
  __syncthreads();
  angles(a.t, tokens, position, cs);
  __syncthreads();
  if (!keys) {
    turn_rows<T>(a.t, first, tokens, position, cs);
    return;
  }
  const int per = a.m.head_dim / N, row = a.m.kv_heads * per, items = tokens * row;
  // all threads of a block of 32 values take part in storing it
  for (int item = threadIdx.x; item < items; item += 256) {
    const int token = item / row, in_row = item - token * row, head = in_row / per, d = (in_row - head * per) * N;
    const int64_t slot = slots[token];
    if (slot < 0) continue;
    const int64_t at = (slot + ((int64_t)head << a.m.page_shift)) * a.m.head_dim + d;
    float x[2][N];
    const T* from[2];
#pragma unroll
    for (int y = 0; y < 2; y++) {
      const Copy& c = a.m.of[y];
      from[y] = (const T*)c.rows + (int64_t)(first + token) * c.token_stride + head * c.head_stride;
      load_row<T, N>(from[y] + d, c.vector, x[y]);
    }
    turn_piece<T, N>(a.t, from[0], d, a.m.of[0].vector, cs + token * a.t.half, x[0]);
#pragma unroll
    for (int y = 0; y < 2; y++) store_page<kStore, N>(a.m.of[y], at, x[y]);
  }
}

// ---------------------------------------------------------------------------- host side
int rotary_check(const MxRotary* r, int head_dim) {
  if (!r || !r->turn || ((uintptr_t)r->turn & 7)) return MX_ERR_INVALID;
  if (head_dim < 2 || head_dim > 1024) return MX_ERR_DOMAIN;
  if (r->width < 2 || r->width > head_dim || r->width % 2) return MX_ERR_INVALID;
  return 0;
}

// Rows' part of the arguments
Turned turned_rows(const MxRotary* r, const MxRows* x, const MxRows* out, int head_dim, int tokens, bool back) {
  Turned t{};
  const int size = size_of(x->type), piece = 16 / size;
  t.x = x->data; t.out = out->data; t.turn = r->turn;
  t.x_token = x->token_stride; t.x_head = x->head_stride; t.o_token = out->token_stride; t.o_head = out->head_stride;
  t.heads = x->heads; t.head_dim = head_dim; t.half = r->width / 2; t.tokens = tokens;
  t.amplitude = r->amplitude;
  t.interleaved = r->interleaved != 0;
  t.back = back;
  t.pieces = rows_aligned(x, 16) && rows_aligned(out, 16) && head_dim % piece == 0
             && (t.interleaved || (t.half % piece == 0 && (head_dim - r->width) % piece == 0));
  return t;
}

// Tokens of a workgroup, for `pieces` of a token that its threads take one at a time: 256 to 1024 pieces, the more the
// less often the angles' latency is waited for, if there are so many workgroups of them (67 prompts of up to 501 tokens
// with 256, 512, 1024 and 2048 pieces 57, 33, 27 and 27 us, 4096 single tokens 10.0, 10.3, 15.0 and 14.7).
int tokens_each(int64_t pieces, int half, int64_t tokens, int groups) {
  const int64_t angles = kMostAngles / half < kMostTokens ? kMostAngles / half : kMostTokens;
  int64_t most = tokens * pieces / groups;
  most = most < 256 ? 256 : most > 1024 ? 1024 : most;
  int64_t each = most / pieces;
  each = each < 1 ? 1 : each;
  if (tokens / each >= kMostGroups / 2) each = kMostTokens;
  return (int)(each < angles ? each : angles);
}

bool rows_type(int type) { return type == MX_TYPE_F32 || type == MX_TYPE_BF16 || type == MX_TYPE_F16; }

}  // namespace mxe

extern "C" {

size_t mx_rotary_bytes(void) { return sizeof(MxRotary); }

int mx_rotate(const MxRotary* rotary, const MxRows* x, const MxRows* out, int32_t head_dim, int32_t tokens,
              const void* positions, int32_t period, int32_t wide, int32_t back, void* stream) {
  using namespace mxe;
  int rc = rotary_check(rotary, head_dim);
  if (rc) return rc;
  if (!x || !out || tokens < 0 || x->heads < 1 || !rows_type(x->type) || out->type != x->type) return MX_ERR_INVALID;
  if ((rc = rows_check(x, x->heads, tokens > 0)) || (rc = rows_check(out, x->heads, tokens > 0))) return rc;
  if (!tokens) return 0;
  if (!positions || period < 1 || ((uintptr_t)positions & (wide ? 7 : 3))) return MX_ERR_INVALID;
  if ((int64_t)x->heads * head_dim > 1 << 24) return MX_ERR_DOMAIN;
  Rotate a{};
  a.t = turned_rows(rotary, x, out, head_dim, tokens, back != 0);
  a.positions = positions; a.period = period; a.wide = wide != 0;
  const int piece = a.t.pieces ? 16 / size_of(x->type) : 1;
  a.t.each = tokens_each(((int64_t)x->heads * head_dim + piece - 1) / piece, a.t.half, tokens, 2048);
  const int64_t groups = (tokens + (int64_t)a.t.each - 1) / a.t.each;
  if (groups > kMostGroups) return MX_ERR_DOMAIN;
  const size_t lds = (size_t)a.t.each * a.t.half * sizeof(f2);
  const auto go = [&](auto t) {
    hipLaunchKernelGGL((rotate_rows<decltype(t)>), dim3((unsigned)groups), dim3(256), lds, (hipStream_t)stream, a);
  };
  if (x->type == MX_TYPE_F32) go(0.f);
  else if (x->type == MX_TYPE_BF16) go((__bf16)0.f);
  else go((_Float16)0.f);
  return (int)hipGetLastError();
}

int mx_episode_enter(const MxPages* p, const MxChunk* c, const MxRotary* rotary, const MxRows* q, const MxRows* out,
                     const MxRows* k, const MxRows* v, void* stream) {
  using namespace mxe;
  int rc = pages_check(p);
  if (rc || (rc = chunk_check(p, c)) || (rc = rotary_check(rotary, p->head_dim))) return rc;
  const bool any = c->tokens > 0;
  if ((rc = rows_check(k, p->kv_heads, any)) || (rc = rows_check(v, p->kv_heads, any))) return rc;
  if (!q || !out || q->heads < 1) return MX_ERR_INVALID;
  if ((rc = rows_check(q, q->heads, any)) || (rc = rows_check(out, q->heads, any))) return rc;
  if (!rows_type(k->type) || v->type != k->type || q->type != k->type || out->type != k->type) return MX_ERR_INVALID;
  if (!any) return 0;
  if ((int64_t)q->heads * p->head_dim > 1 << 24) return MX_ERR_DOMAIN;
  Enter a{};
  a.t = turned_rows(rotary, q, out, p->head_dim, c->tokens, false);
  const int size = size_of(k->type), piece = piece_bytes(p->type == MX_TYPE_FP8, true, size) / size;
  const int q_piece = a.t.pieces ? 16 / size : 1;
  a.t.each = tokens_each(((int64_t)q->heads * p->head_dim + q_piece - 1) / q_piece, a.t.half, c->tokens, 2048);
  a.m.tokens_each = tokens_each((int64_t)p->kv_heads * p->head_dim / piece, a.t.half, c->tokens, 512);
  uint8_t *pages[2] = {(uint8_t*)p->k, (uint8_t*)p->v}, *scales[2] = {p->k_scale, p->v_scale};
  const MxRows* rows[2] = {k, v};
  for (int i = 0; i < 2; i++)
    a.m.of[i] = Copy{pages[i], scales[i], (const uint8_t*)rows[i]->data, rows[i]->token_stride, rows[i]->head_stride,
                     rows_aligned(rows[i], 16)};
  a.m.table = p->table; a.m.length = p->length; a.m.start = c->start;
  a.m.nworld = p->nworld; a.m.npage = p->npage; a.m.width = p->width; a.m.kv_heads = p->kv_heads;
  a.m.page_shift = page_shift(p); a.m.tokens = c->tokens; a.m.count = c->count;
  a.m.head_dim = p->head_dim;
  const int64_t kv_groups = (c->tokens + (int64_t)a.m.tokens_each - 1) / a.m.tokens_each;
  const int64_t groups = kv_groups + (c->tokens + (int64_t)a.t.each - 1) / a.t.each;
  if (groups > kMostGroups) return MX_ERR_DOMAIN;
  a.kv_groups = (int)kv_groups;
  const int most = a.t.each > a.m.tokens_each ? a.t.each : a.m.tokens_each;
  const size_t lds = (size_t)most * a.t.half * sizeof(f2);
  auto go = [&](auto t, auto store) {
    typedef decltype(t) T;
    constexpr int kStore = decltype(store)::value;
    hipLaunchKernelGGL((enter_rows<T, kStore>), dim3((unsigned)groups), dim3(256), lds, (hipStream_t)stream, a);
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

}
