// Episode memory: the attention kernels for heads of 256 values.
#include "mx_episode_dim.h"

namespace mxe {
int attend256(const Attend& a, const Launch& launch, void* stream) { return attend_dim<256>(a, launch, stream); }
}  // namespace mxe
