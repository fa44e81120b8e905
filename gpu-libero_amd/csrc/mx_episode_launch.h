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
  int64_t keys;                               // the most that a world has, as far as the host knows
  bool fp8;
  unsigned grid;
};

int choose(Attend& a, Launch& launch);

int attend32(const Attend& a, const Launch& launch, void* stream);
int attend64(const Attend& a, const Launch& launch, void* stream);
int attend96(const Attend& a, const Launch& launch, void* stream);
int attend128(const Attend& a, const Launch& launch, void* stream);
int attend256(const Attend& a, const Launch& launch, void* stream);

}  // namespace mxe
