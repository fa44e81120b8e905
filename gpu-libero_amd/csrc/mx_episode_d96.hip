// Episode memory: the attention kernels for heads of 96 values.
#include "mx_episode_dim.h"

namespace mxe {
int attend96(const Attend& a, const Launch& launch, void* stream) { return attend_dim<96>(a, launch, stream); }
}  // namespace mxe
