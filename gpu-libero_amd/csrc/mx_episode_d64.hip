// Episode memory: the attention kernels for heads of 64 values.
#include "mx_episode_dim.h"

namespace mxe {
int attend64(const Attend& a, const Launch& launch, void* stream) { return attend_dim<64>(a, launch, stream); }
}  // namespace mxe
