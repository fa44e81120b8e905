// Room for tokens: the worlds' tables and lengths and the stack of free pages change on the GPU, and a chunk's rows learn
// their worlds, positions and slots.
//
// Where a world's pages come off the stack follows from the needs of all worlds before it, and whether they do at all
// from everyone's.  One workgroup does all for up to 1024 worlds with few pages.  For more there are two launches:
// there are few numbers to a world, so each workgroup reads all of them again for its prefix and the totals instead of
// waiting for its neighbours; lengths then change in the second launch, which also hands out the pages that the first
// has put on the stack. Bound by launches and by a few dependent loads: 67 worlds 3.6 us; 4096 worlds that all restart
// 11 and 4 us, of which the reading of all worlds is most (with sums in 64 bits 13, with 1024 threads to a workgroup
// 13); it grows with them, 31 us for a change of 16384 and 185 of 131072.  The places of the 4096 worlds' 2.1 million rows
// (25 MB): 13 us, 9 where all worlds have the same number.
#include "mx_episode_move.h"
#include "mx_episode_launch.h"

namespace mxe {

struct Room {
  int32_t *table, *length, *free, *state;
  const int32_t* count;
  const uint8_t* over;
  int32_t* start;
  int4* found;                   // of each workgroup of update_count(), for update_tables()
  int nworld, width, npage, page_shift, tokens, each, rows, worlds_each;
};

// What a change does to a world: its tokens before (of which `base` stay at most) and after, its pages that stay, that
// it has, and that it then has
struct Change {
  int base, after, kept, held, need, rows;
  bool refused;
};

__device__ inline Change change_of(const Room& a, int has, int by, bool over) {
  Change c;
  const int pages = (1 << a.page_shift) - 1, reach = a.width << a.page_shift;      // at most 2^30
  const int length = min(max(has, 0), reach);
  c.base = over ? 0 : length;
  const unsigned after = (unsigned)c.base + (unsigned)by;                          // of no fewer than 0: below 2^32
  c.refused = by < -c.base || (by > 0 && after > (unsigned)min(a.tokens, reach));
  c.after = c.refused ? c.base : (int)after;
  c.held = (length + pages) >> a.page_shift;
  c.kept = (min(c.base, c.after) + pages) >> a.page_shift;
  c.need = (c.after + pages) >> a.page_shift;
  c.rows = max(by, 0);
  return c;
}

__device__ inline Change change_of(const Room& a, int w) {
  return change_of(a, a.length[w], a.count ? a.count[w] : a.each, a.over && a.over[w]);
}

// Sums over a workgroup of kMany values to a thread: those before the thread's, in place, and all of them
template <int kThreads, int kMany>
__device__ inline void sums_before(long long (&x)[kMany], long long (&sh)[kThreads / 64][kMany], long long (&all)[kMany]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  long long sum[kMany];
#pragma unroll
  for (int i = 0; i < kMany; i++) sum[i] = x[i];
#pragma unroll
  for (int by = 1; by < 64; by *= 2)
#pragma unroll
    for (int i = 0; i < kMany; i++) {
      const long long y = __shfl_up(sum[i], by);
      if (lane >= by) sum[i] += y;
    }
  if (lane == 63)
#pragma unroll
    for (int i = 0; i < kMany; i++) sh[wave][i] = sum[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kMany; i++) {
    x[i] = sum[i] - x[i];
    all[i] = 0;
  }
#pragma unroll
  for (int w = 0; w < kThreads / 64; w++)
#pragma unroll
    for (int i = 0; i < kMany; i++) {
      const long long y = sh[w][i];
      x[i] += w < wave ? y : 0;
      all[i] += y;
    }
  __syncthreads();
}

// Which of a workgroup's worlds a piece of work belongs to: the last w with before[w] <= i
__device__ inline int owner(const long long* before, int worlds, long long i) {
  int low = 0, high = worlds;
  while (high - low > 1) {
    const int middle = (low + high) >> 1;
    if (before[middle] <= i) low = middle; else high = middle;
  }
  return low;
}

// Why a change is refused, from the sums over all worlds
__device__ inline int why_not(const Room& a, bool refused, long long left, long long back, long long need, long long rows) {
  return (refused ? MX_ROOM_TOKENS : 0) | (need > min(left + back, (long long)a.npage) ? MX_ROOM_PAGES : 0)
         | (rows > a.rows ? MX_ROOM_ROWS : 0);
}

// Of a world in a refused change only what has to go, goes
__device__ inline void refuse(Change& c, bool over) {
  c.after = c.base;
  c.kept = over ? 0 : c.held;
  c.need = c.kept;
}

// Pieces of work, `many` of them, that belong to a workgroup's worlds from before[o] on: their table entries count on from
// from[o], and are moved in turn
template <int kThreads, class Move>
__device__ inline void each_entry(const Room& a, int first, int worlds, const long long* before, const int* from, long long many,
                                  Move move) {
  for (long long i = threadIdx.x; i < many; i += kThreads) {
    const int o = owner(before, worlds, i);
    const long long slot = from[o] + i - before[o];
    if (slot < a.width) move(a.table + (int64_t)(first + o) * a.width + slot, i);
  }
}

// One workgroup, a world to a thread
constexpr int kAlone = 1024;
template <int kThreads>
__global__ __launch_bounds__(kThreads) void update_alone(const Room a) {
  __shared__ long long sh[kThreads / 64][4], before[kThreads];
  __shared__ int from[kThreads];
  const int w = threadIdx.x;
  const bool mine = w < a.nworld, over = mine && a.over && a.over[w];
  const long long left = min(max(a.state[0], 0), a.npage);
  Change c{};
  if (mine) c = change_of(a, w);
  // pages back (of emptied worlds alone, and all), pages needed, rows
  long long x[4] = {over ? c.held : 0, c.held - min(c.kept, c.held), c.need - c.kept, c.rows}, all[4];
  sums_before<kThreads, 4>(x, sh, all);
  const int why = why_not(a, __syncthreads_or(c.refused), left, all[1], all[2], all[3]);
  if (why) refuse(c, over);
  const long long back = why ? all[0] : all[1];
  before[w] = why ? x[0] : x[1];
  from[w] = min(c.kept, c.held);
  if (a.start && mine) {
    a.start[w] = why ? 0 : (int)x[3];
    if (w == a.nworld - 1) a.start[a.nworld] = why ? 0 : (int)all[3];
  }
  const long long top = min(left + back, (long long)a.npage);
  if (back) {                                     // the first page that comes back lies highest on the stack
    __syncthreads();
    each_entry<kThreads>(a, 0, a.nworld, before, from, back, [&](int32_t* entry, long long i) {
      const long long at = left + back - 1 - i;
      if (at >= 0 && at < a.npage) a.free[at] = *entry;
      *entry = -1;
    });
    __syncthreads();
  }
  if (!why && all[2]) {
    before[w] = x[2];
    __syncthreads();
    each_entry<kThreads>(a, 0, a.nworld, before, from, all[2], [&](int32_t* entry, long long i) {
      if (top - 1 - i >= 0) *entry = a.free[top - 1 - i];
    });
  }
  if (mine) a.length[w] = c.after;
  if (w == 0) {
    a.state[0] = (int)(why ? top : top - all[2]);
    if (why) a.state[1] |= why;
  }
}

constexpr int kMostWorlds = 256;                // of a workgroup

// Totals, the pages that come back, and the rows' starts
__global__ __launch_bounds__(256) void update_count(const Room a) {
  __shared__ long long sums[4][2], sh[4][2], before[kMostWorlds];
  __shared__ int from[kMostWorlds], parts[4][6];
  const int first = blockIdx.x * a.worlds_each, worlds = min(a.nworld - first, a.worlds_each);
  // sums over all worlds: pages needed and rows, in 64 bits as there may be any number of them; pages back (of emptied
  // worlds alone, and all); and over those before this workgroup's: pages back, needed, and rows, which are right if
  // the change is not refused
  long long wide[2] = {0, 0};
  int x[6] = {0, 0, 0, 0, 0, 0}, refused = 0;
  constexpr int kAhead = 8;                       // worlds of a thread whose numbers are under way together
  for (int base = threadIdx.x; base < a.nworld; base += kAhead * 256) {
    int length[kAhead], count[kAhead];
    bool over[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; u++) {
      const int w = base + u * 256;
      const bool is = w < a.nworld;
      length[u] = is ? a.length[w] : 0;
      count[u] = !is ? 0 : a.count ? a.count[w] : a.each;
      over[u] = is && a.over && a.over[w];
    }
#pragma unroll
    for (int u = 0; u < kAhead; u++) {
      const Change c = change_of(a, length[u], count[u], over[u]);
      const int gone = over[u] ? c.held : 0, back = c.held - min(c.kept, c.held), need = c.need - c.kept;
      const bool earlier = base + u * 256 < first;
      refused |= c.refused;
      wide[0] += need;
      wide[1] += c.rows;
      x[0] += gone;
      x[1] += back;
      x[2] += earlier ? gone : 0;
      x[3] += earlier ? back : 0;
      x[4] += earlier ? need : 0;
      x[5] += earlier ? c.rows : 0;
    }
  }
#pragma unroll
  for (int by = 1; by < 64; by *= 2) {
#pragma unroll
    for (int i = 0; i < 2; i++) wide[i] += __shfl_xor(wide[i], by);
#pragma unroll
    for (int i = 0; i < 6; i++) x[i] += __shfl_xor(x[i], by);
  }
  if ((threadIdx.x & 63) == 0) {
#pragma unroll
    for (int i = 0; i < 2; i++) sums[threadIdx.x >> 6][i] = wide[i];
#pragma unroll
    for (int i = 0; i < 6; i++) parts[threadIdx.x >> 6][i] = x[i];
  }
  refused = __syncthreads_or(refused);
#pragma unroll
  for (int i = 0; i < 2; i++) wide[i] = sums[0][i] + sums[1][i] + sums[2][i] + sums[3][i];
#pragma unroll
  for (int i = 0; i < 6; i++) x[i] = parts[0][i] + parts[1][i] + parts[2][i] + parts[3][i];
  const long long left = min(max(a.state[0], 0), a.npage);
  const int why = why_not(a, refused, left, x[1], wide[0], wide[1]);
  const long long back_in_all = why ? x[0] : x[1];

  // this workgroup's worlds, one to a thread
  const int w = first + threadIdx.x;
  const bool mine = (int)threadIdx.x < worlds;
  Change c{};
  if (mine) c = change_of(a, w);
  if (mine && why) refuse(c, a.over && a.over[w]);
  const int kept = min(c.kept, c.held);
  long long y[2] = {c.held - kept, c.rows}, total[2];
  sums_before<256, 2>(y, sh, total);
  if (a.start && mine) {
    a.start[w] = why ? 0 : (int)(x[5] + y[1]);
    if (w == a.nworld - 1) a.start[a.nworld] = why ? 0 : (int)wide[1];
  }
  before[threadIdx.x] = y[0];
  from[threadIdx.x] = kept;
  __syncthreads();
  // the first page that comes back lies highest on the stack
  const long long top = left + back_in_all - 1 - (why ? x[2] : x[3]);
  each_entry<256>(a, first, worlds, before, from, total[0], [&](const int32_t* entry, long long i) {
    if (top - i >= 0 && top - i < a.npage) a.free[top - i] = *entry;
  });
  if (threadIdx.x == 0)
    a.found[blockIdx.x] = int4{(int)max(min(left + back_in_all, (long long)a.npage), 0LL), x[4], why, (int)wide[0]};
}

// Tables and lengths
__global__ __launch_bounds__(256) void update_tables(const Room a) {
  __shared__ long long sh[4][2], before[kMostWorlds], given[kMostWorlds];
  __shared__ int from[kMostWorlds], to[kMostWorlds];
  const int first = blockIdx.x * a.worlds_each, worlds = min(a.nworld - first, a.worlds_each);
  const int4 found = a.found[blockIdx.x];
  const int left = found.x, why = found.z, w = first + threadIdx.x;
  const bool mine = (int)threadIdx.x < worlds;
  Change c{};
  if (mine) c = change_of(a, w);
  if (mine && why) refuse(c, a.over && a.over[w]);
  // entries that get a page, and those that name none any more
  long long x[2] = {max(c.need - c.kept, 0), max(c.held - max(c.kept, c.need), 0)}, all[2];
  sums_before<256, 2>(x, sh, all);
  before[threadIdx.x] = x[0];
  given[threadIdx.x] = x[1];
  from[threadIdx.x] = c.kept;
  to[threadIdx.x] = max(c.kept, c.need);
  __syncthreads();
  each_entry<256>(a, first, worlds, before, from, all[0], [&](int32_t* entry, long long i) {
    const long long at = left - 1LL - found.y - i;
    if (at >= 0) *entry = a.free[at];
  });
  each_entry<256>(a, first, worlds, given, to, all[1], [&](int32_t* entry, long long i) { *entry = -1; });
  if (mine) a.length[w] = c.after;
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    a.state[0] = why ? left : left - found.w;
    if (why) a.state[1] |= why;
  }
}

// Four neighbouring rows to a lane: they are mostly of one world and in one page
struct Places {
  Move m;
  int32_t *world, *position, *slot;
  bool vector;                   // the results are 16-byte aligned
};

// The starts in LDS: of as many worlds as a workgroup's rows have where each has one token, the commonest large step (4096
// worlds 9.1 us, 9.5 searched for in memory)
constexpr int kRowsEach = 4, kStarts = 256 * kRowsEach + 1;
__global__ __launch_bounds__(256) void find_places(const Places a) {
  const Move& m = a.m;
  __shared__ int starts[kStarts];
  const int rows_each = 256 * kRowsEach;
  const int block = (int)((long long)blockIdx.x * rows_each), in_block = min(m.tokens - block, rows_each);
  // the worlds of the workgroup's rows, and where their rows begin
  int low = 0, high = m.nworld;
  if (m.start && m.nworld + 1 > kStarts) {
    low = world_at(m.start, m.nworld, block);
    high = world_at(m.start, m.nworld, block + in_block - 1) + 1;
  }
  const int many = high - low + 1;
  const bool held = m.start && many <= kStarts;
  if (held) {
    for (int i = threadIdx.x; i < many; i += 256) starts[i] = m.start[low + i];
    __syncthreads();
  }
  const auto start_of = [&](int world) { return held ? starts[world - low] : m.start[world]; };
  const int in = kRowsEach * (int)threadIdx.x;
  if (in >= in_block) return;
  const int first = block + in;
  int world = low, begin = 0, stop = 0, length = 0, page = -1, entry = -1;
  const auto find = [&](int token) {               // from an earlier row's world on: mostly the same
    if (m.start) {
      int below = high;
      if (start_of(world + 1) <= token)
        while (below - world > 1) {
          const int middle = (world + below) >> 1;
          if (start_of(middle) <= token) world = middle; else below = middle;
        }
      begin = start_of(world);
      stop = start_of(world + 1);
    } else {
      world = token / m.count;
      begin = world * m.count;
      stop = begin + m.count;
    }
    length = max(m.length[world], 0);
    entry = -1;
  };
  find(first);
  int32_t out[3][kRowsEach];
  const int rows = min(kRowsEach, in_block - in);
#pragma unroll
  for (int i = 0; i < kRowsEach; i++) {
    const int token = first + i;
    if (i >= rows) continue;
    if (token >= stop && world + 1 < high) find(token);
    const bool is = begin >= 0 && token >= begin && token < stop;
    const int position = length - (stop - begin) + token - begin;
    int slot = -1;
    if (is && position >= 0 && position >> m.page_shift < m.width) {
      if (position >> m.page_shift != entry) {
        entry = position >> m.page_shift;
        page = m.table[(int64_t)world * m.width + entry];
      }
      if ((unsigned)page < (unsigned)m.npage) slot = (page << m.page_shift) + (position & ((1 << m.page_shift) - 1));
    }
    out[0][i] = is ? world : -1;
    out[1][i] = is ? max(position, -1) : -1;
    out[2][i] = slot;
  }
  int32_t* to[3] = {a.world + first, a.position + first, a.slot + first};
#pragma unroll
  for (int x = 0; x < 3; x++) {
    if (a.vector && rows == kRowsEach) {
      *(int4*)to[x] = int4{out[x][0], out[x][1], out[x][2], out[x][3]};
    } else {
#pragma unroll
      for (int i = 0; i < kRowsEach; i++)
        if (i < rows) to[x][i] = out[x][i];
    }
  }
}

// ---------------------------------------------------------------------------- host side
int room_check(const MxRoom* r) {
  if (!r || !r->table || !r->length || r->nworld < 1 || r->width < 1 || r->npage < 1 || r->tokens < 0) return MX_ERR_INVALID;
  const int t = r->page_tokens;
  if (t < 16 || t > 4096 || (t & (t - 1))) return MX_ERR_DOMAIN;
  if ((int64_t)r->npage * t > INT32_MAX || (int64_t)r->width * t > 1 << 30) return MX_ERR_DOMAIN;
  return 0;
}

// Worlds of a workgroup: every workgroup reads all worlds, so no more than 512 of them if there are worlds enough
int worlds_each(int nworld) {
  const int each = (nworld + 511) / 512;
  return each < 16 ? 16 : each;
}

// Whether one workgroup does all: its threads move all pages of all worlds at worst
bool alone(const MxRoom* r) { return r->nworld <= kAlone && (int64_t)r->nworld * r->width <= 65536; }

}  // namespace mxe

extern "C" {

size_t mx_room_bytes(void) { return sizeof(MxRoom); }
size_t mx_room_change_bytes(void) { return sizeof(MxRoomChange); }

size_t mx_room_workspace(const MxRoom* room) {
  if (mxe::room_check(room) || mxe::alone(room)) return 0;
  const int each = mxe::worlds_each(room->nworld);
  return (size_t)((room->nworld + each - 1) / each) * sizeof(int4);
}

int mx_room_update(const MxRoom* room, const MxRoomChange* change, void* stream) {
  using namespace mxe;
  const int rc = room_check(room);
  if (rc) return rc;
  if (!change || !room->free || !room->state || change->rows < 0) return MX_ERR_INVALID;
  if (room->nworld > kMostWorlds * 512) return MX_ERR_DOMAIN;
  const size_t bytes = mx_room_workspace(room);
  if (bytes && (!change->workspace || change->workspace_bytes < bytes || ((uintptr_t)change->workspace & 15))) return MX_ERR_WORKSPACE;
  Room a{};
  a.table = room->table; a.length = room->length; a.free = room->free; a.state = room->state;
  a.count = change->count; a.over = change->over; a.start = change->start;
  a.found = (int4*)change->workspace;
  a.nworld = room->nworld; a.width = room->width; a.npage = room->npage;
  a.page_shift = __builtin_ctz(room->page_tokens);
  a.tokens = room->tokens; a.each = change->each; a.rows = change->rows;
  a.worlds_each = worlds_each(room->nworld);
  if (!bytes) {
    if (room->nworld <= 256) hipLaunchKernelGGL(update_alone<256>, dim3(1), dim3(256), 0, (hipStream_t)stream, a);
    else hipLaunchKernelGGL(update_alone<kAlone>, dim3(1), dim3(kAlone), 0, (hipStream_t)stream, a);
    return (int)hipGetLastError();
  }
  const dim3 grid((unsigned)((room->nworld + a.worlds_each - 1) / a.worlds_each));
  hipLaunchKernelGGL(update_count, grid, dim3(256), 0, (hipStream_t)stream, a);
  hipLaunchKernelGGL(update_tables, grid, dim3(256), 0, (hipStream_t)stream, a);
  return (int)hipGetLastError();
}

int mx_room_places(const MxRoom* room, const MxChunk* c, int32_t* world, int32_t* position, int32_t* slot, void* stream) {
  using namespace mxe;
  const int rc = room_check(room);
  if (rc) return rc;
  if (!c || c->tokens < 0) return MX_ERR_INVALID;
  if (!c->start && (c->count < 0 || (int64_t)c->count * room->nworld != c->tokens)) return MX_ERR_INVALID;
  if (!c->tokens) return 0;
  if (!world || !position || !slot) return MX_ERR_INVALID;
  Places a{};
  a.m.table = room->table; a.m.length = room->length; a.m.start = c->start;
  a.m.nworld = room->nworld; a.m.npage = room->npage; a.m.width = room->width; a.m.kv_heads = 1;
  a.m.page_shift = __builtin_ctz(room->page_tokens); a.m.tokens = c->tokens; a.m.count = c->count;
  a.world = world; a.position = position; a.slot = slot;
  a.vector = !(((uintptr_t)world | (uintptr_t)position | (uintptr_t)slot) & 15);
  const unsigned groups = (unsigned)((c->tokens + 256LL * kRowsEach - 1) / (256 * kRowsEach));
  hipLaunchKernelGGL(find_places, dim3(groups), dim3(256), 0, (hipStream_t)stream, a);
  return (int)hipGetLastError();
}

}
