// Episode memory: the attention kernels for heads of 32 values.
#include "mx_episode_dim.h"

namespace mxe {
int attend32(const Attend& a, const Launch& launch, void* stream) { return attend_dim<32>(a, launch, stream); }
}  // namespace mxe
