// What the host side of the episode memory's attention has decided, and the launchers, one for each head_dim
// (mx_episode_d*.hip: a translation unit each, so that they compile side by side).
#pragma once
#include "mx_episode_types.h"

namespace mxe {

constexpr int kManyRows = 128;              // rows of a tile of attend_many

constexpr int64_t kMostGroups = (1 << 24) - 1;   // workgroups of 256 of a launch: threads are counted in 32 bits

struct Launch {
  int type, head_dim, blocks, rows, tiles;    // blocks of 16 rows to a tile
  int team;                                   // waves of attend_few that share a tile
  int64_t keys, held;                         // the most that a row sees, and that a world has, as far as the host knows
  bool fp8, listed, gathered;                 // listed: attention to listed blocks; gathered: of rows that share one
  unsigned grid;
};

// Checks and what a launch needs of an attention, all keys or (blocks, of 2^block_shift tokens) listed ones; its workspace;
// and the launches (mx_episode.hip)
int plan(const MxPages* p, const MxChunk* c, const MxAttention* m, Attend& a, Launch& launch, bool pointers,
         const MxSelection* s = nullptr, int block_shift = 0);
size_t workspace_of(const Attend& a, const Launch& launch);
int gather_rows(Attend& a, const Launch& launch, void* stream);    // (mx_episode_recall.hip)
int attend_planned(Attend& a, const Launch& launch, const MxAttention* m, void* stream);

// Checks that all entry points share (mx_episode.hip)
int size_of(int type);
int pages_check(const MxPages* p);
int chunk_check(const MxPages* p, const MxChunk* c);
bool rows_aligned(const MxRows* r, int bytes);
int rows_check(const MxRows* r, int heads, bool any);
int page_shift(const MxPages* p);

int attend32(const Attend& a, const Launch& launch, void* stream);
int attend64(const Attend& a, const Launch& launch, void* stream);
int attend96(const Attend& a, const Launch& launch, void* stream);
int attend128(const Attend& a, const Launch& launch, void* stream);
int attend256(const Attend& a, const Launch& launch, void* stream);

}  // namespace mxe
