// Room for tokens: the worlds' tables and lengths and the stack of free pages change on the GPU, and a chunk's rows learn
// their worlds, positions and slots.
//
// Where a world's pages come off the stack follows from the needs of all worlds before it, and whether they do at all from
// everyone's.  There are few numbers to a world, so each workgroup reads all of them again for its prefix and the totals
// instead of waiting for its neighbours; lengths then change in a second launch, which also hands out the pages that the
// first has put on the stack.  Both are bound by their launches and by a few dependent loads.
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

// What a change does to a world: its tokens before (of which `base` stay at most) and after, its pages that stay, that it has,
// and that it then has
struct Change {
  int base, after, kept, held, need, rows;
  bool refused;
};

__device__ inline Change change_of(const Room& a, int w) {
  Change c;
  const int pages = (1 << a.page_shift) - 1;
  const long long reach = (long long)a.width << a.page_shift;
  const int length = (int)min((long long)max(a.length[w], 0), reach);
  c.base = a.over && a.over[w] ? 0 : length;
  const int by = a.count ? a.count[w] : a.each;
  const long long after = (long long)c.base + by;
  c.refused = after < 0 || (by > 0 && after > min((long long)a.tokens, reach));
  c.after = c.refused ? c.base : (int)after;
  c.held = (int)(((long long)length + pages) >> a.page_shift);
  c.kept = (min(c.base, c.after) + pages) >> a.page_shift;
  c.need = (c.after + pages) >> a.page_shift;
  c.rows = max(by, 0);
  return c;
}

// Sums over a workgroup of 256: those before the thread's and all of them
template <class T> __device__ inline T sums_before(T x, T* sh, T& all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  T sum = x;
#pragma unroll
  for (int by = 1; by < 64; by *= 2) {
    const T y = __shfl_up(sum, by);
    if (lane >= by) sum += y;
  }
  if (lane == 63) sh[wave] = sum;
  __syncthreads();
  T before = sum - x;
  all = 0;
#pragma unroll
  for (int w = 0; w < 4; w++) {
    if (w < wave) before += sh[w];
    all += sh[w];
  }
  __syncthreads();
  return before;
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

constexpr int kMostWorlds = 256;                // of a workgroup

// Totals, the pages that come back, and the rows' starts.  Whether tokens are refused decides which pages come back: those of
// emptied worlds always, those of tokens given back only then.
__global__ __launch_bounds__(256) void update_count(const Room a) {
  __shared__ long long sh[4], before[kMostWorlds];
  __shared__ int from[kMostWorlds];
  const int first = blockIdx.x * a.worlds_each, worlds = min(a.nworld - first, a.worlds_each);
  // sums over all worlds, and over those before this workgroup's: pages back (without and with tokens given back), pages
  // needed, rows
  long long all_over = 0, all_back = 0, all_need = 0, all_rows = 0, my_over = 0, my_back = 0, my_need = 0, my_rows = 0;
  int refused = 0;
  for (int w = threadIdx.x; w < a.nworld; w += 256) {
    const Change c = change_of(a, w);
    const int over = a.over && a.over[w] ? c.held : 0, back = c.held - min(c.kept, c.held), need = c.need - c.kept;
    refused |= c.refused;
    all_over += over;
    all_back += back;
    all_need += need;
    all_rows += c.rows;
    if (w < first) {
      my_over += over;
      my_back += back;
      my_need += need;
      my_rows += c.rows;
    }
  }
  long long none;
  sums_before(all_over, sh, all_over);
  sums_before(all_back, sh, all_back);
  sums_before(all_need, sh, all_need);
  sums_before(all_rows, sh, all_rows);
  sums_before(my_over, sh, my_over);
  sums_before(my_back, sh, my_back);
  sums_before(my_need, sh, my_need);
  sums_before(my_rows, sh, my_rows);
  const long long left = min(max(a.state[0], 0), a.npage);
  int why = __syncthreads_or(refused) ? MX_ROOM_TOKENS : 0;
  if (all_need > min(left + all_back, (long long)a.npage)) why |= MX_ROOM_PAGES;
  if (all_rows > a.rows) why |= MX_ROOM_ROWS;
  const long long back_in_all = why ? all_over : all_back;

  // this workgroup's worlds, one to a thread
  const int w = first + threadIdx.x;
  const bool mine = (int)threadIdx.x < worlds;
  Change c{};
  if (mine) c = change_of(a, w);
  const int kept = !mine ? 0 : why ? (a.over && a.over[w] ? 0 : c.held) : min(c.kept, c.held);
  const long long back = mine ? c.held - kept : 0, rows = mine && !why ? c.rows : 0;
  long long total;
  const long long back_before = sums_before(back, sh, total), rows_before = sums_before(rows, sh, none);
  if (a.start && mine) {
    a.start[w] = why ? 0 : (int)(my_rows + rows_before);
    if (w == a.nworld - 1) a.start[a.nworld] = why ? 0 : (int)all_rows;
  }
  before[threadIdx.x] = back_before;
  from[threadIdx.x] = kept;
  __syncthreads();
  // the first page that comes back lies highest on the stack
  const long long top = left + back_in_all - 1 - (why ? my_over : my_back);
  for (long long i = threadIdx.x; i < total; i += 256) {
    const int o = owner(before, worlds, i);
    const long long slot = from[o] + i - before[o], at = top - i;
    if (at >= 0 && at < a.npage && slot < a.width) a.free[at] = a.table[(int64_t)(first + o) * a.width + slot];
  }
  if (threadIdx.x == 0) {
    a.found[blockIdx.x] = int4{(int)min(left + back_in_all, (long long)a.npage), (int)my_need, why, (int)all_need};
  }
}

// Tables and lengths
__global__ __launch_bounds__(256) void update_tables(const Room a) {
  __shared__ long long sh[4], before[kMostWorlds];
  __shared__ int from[kMostWorlds];
  const int first = blockIdx.x * a.worlds_each, worlds = min(a.nworld - first, a.worlds_each);
  const int4 found = a.found[blockIdx.x];
  const int left = found.x, why = found.z, w = first + threadIdx.x;
  const bool mine = (int)threadIdx.x < worlds;
  Change c{};
  if (mine) c = change_of(a, w);
  const bool over = mine && a.over && a.over[w];
  if (why) {
    c.after = c.base;
    c.kept = over ? 0 : c.held;
    c.need = c.kept;
  }
  const long long given = mine ? max(c.held - max(c.kept, c.need), 0) : 0;      // entries that name no page any more
  const long long taken = mine ? max(c.need - c.kept, 0) : 0;
  long long all;
  const long long taken_before = sums_before(taken, sh, all);
  before[threadIdx.x] = taken_before;
  from[threadIdx.x] = c.kept;
  __syncthreads();
  for (long long i = threadIdx.x; i < all; i += 256) {
    const int o = owner(before, worlds, i);
    const long long slot = from[o] + i - before[o], at = left - 1 - found.y - i;
    if (at >= 0 && slot < a.width) a.table[(int64_t)(first + o) * a.width + slot] = a.free[at];
  }
  __syncthreads();
  const long long given_before = sums_before(given, sh, all);
  before[threadIdx.x] = given_before;
  from[threadIdx.x] = max(c.kept, c.need);
  __syncthreads();
  for (long long i = threadIdx.x; i < all; i += 256) {
    const int o = owner(before, worlds, i);
    const long long slot = from[o] + i - before[o];
    if (slot < a.width) a.table[(int64_t)(first + o) * a.width + slot] = -1;
  }
  if (mine) a.length[w] = c.after;
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    a.state[0] = why ? left : left - found.w;
    if (why) a.state[1] |= why;
  }
}

// A row to a lane
struct Places {
  Move m;
  int32_t *world, *position, *slot;
};

__global__ __launch_bounds__(256) void find_places(const Places a) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long long first = blockIdx.x * 256LL + 64 * wave;
  if (first >= a.m.tokens) return;
  const int lane = threadIdx.x & 63, tokens = (int)min(64LL, a.m.tokens - first), token = (int)first + lane;
  const int world = world_of(a.m.start, a.m.nworld, a.m.count, (int)first, tokens);
  if (world < 0) return;
  const int begin = a.m.start ? a.m.start[world] : world * a.m.count, count = a.m.start ? a.m.start[world + 1] - begin : a.m.count;
  const int place = token - begin;
  const bool is = begin >= 0 && place >= 0 && place < count;
  const int position = max(a.m.length[world], 0) - count + place;
  a.world[token] = is ? world : -1;
  a.position[token] = is ? max(position, -1) : -1;
  a.slot[token] = is ? (int)slot_of(a.m, world, place, count) : -1;
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

}  // namespace mxe

extern "C" {

size_t mx_room_bytes(void) { return sizeof(MxRoom); }
size_t mx_room_change_bytes(void) { return sizeof(MxRoomChange); }

size_t mx_room_workspace(const MxRoom* room) {
  if (mxe::room_check(room)) return 0;
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
  if (!change->workspace || change->workspace_bytes < bytes || ((uintptr_t)change->workspace & 15)) return MX_ERR_WORKSPACE;
  Room a{};
  a.table = room->table; a.length = room->length; a.free = room->free; a.state = room->state;
  a.count = change->count; a.over = change->over; a.start = change->start;
  a.found = (int4*)change->workspace;
  a.nworld = room->nworld; a.width = room->width; a.npage = room->npage;
  a.page_shift = __builtin_ctz(room->page_tokens);
  a.tokens = room->tokens; a.each = change->each; a.rows = change->rows;
  a.worlds_each = worlds_each(room->nworld);
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
  hipLaunchKernelGGL(find_places, dim3((unsigned)((c->tokens + 255LL) / 256)), dim3(256), 0, (hipStream_t)stream, a);
  return (int)hipGetLastError();
}

}
