// Episode memory: the attention kernels for heads of 128 values.
#include "mx_episode_dim.h"

namespace mxe {
int attend128(const Attend& a, const Launch& launch, void* stream) { return attend_dim<128>(a, launch, stream); }
}  // namespace mxe
