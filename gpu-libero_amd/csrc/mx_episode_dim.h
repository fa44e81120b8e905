// The attention kernels of one head_dim, and their launcher.
#pragma once
#include "mx_episode_few.h"
#include "mx_episode_many.h"
#include "mx_episode_launch.h"

namespace mxe {

template <int D, int kType, bool kFp8>
int attend_typed(const Attend& a, const Launch& launch, void* stream) {
  const dim3 grid(launch.grid), block(256);
  const hipStream_t s = (hipStream_t)stream;
  if (launch.gathered) {
    if (a.page_shift >= 6) hipLaunchKernelGGL((attend_many<kType, kFp8, true, D, true>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((attend_many<kType, kFp8, false, D, true>), grid, block, 0, s, a);
    return (int)hipGetLastError();
  }
  if (launch.listed) {
    if (launch.blocks == 1) {
      if (launch.team == 1) hipLaunchKernelGGL((attend_few<kType, kFp8, D, 1, 1, true>), grid, dim3(64), 0, s, a);
      else hipLaunchKernelGGL((attend_few<kType, kFp8, D, 1, 4, true>), grid, block, 0, s, a);
    } else if constexpr (kFp8) {
      if (launch.team == 1) hipLaunchKernelGGL((attend_few<kType, kFp8, D, 2, 1, true>), grid, dim3(64), 0, s, a);
      else hipLaunchKernelGGL((attend_few<kType, kFp8, D, 2, 4, true>), grid, block, 0, s, a);
    }
    return (int)hipGetLastError();
  }
  if (launch.rows == kManyRows) {
    if (a.page_shift >= 6) hipLaunchKernelGGL((attend_many<kType, kFp8, true, D>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((attend_many<kType, kFp8, false, D>), grid, block, 0, s, a);
    return (int)hipGetLastError();
  }
  if (launch.blocks == 1) {
    if (launch.team == 1) hipLaunchKernelGGL((attend_few<kType, kFp8, D, 1, 1>), grid, dim3(64), 0, s, a);
    else hipLaunchKernelGGL((attend_few<kType, kFp8, D, 1, 4>), grid, block, 0, s, a);
  } else if constexpr (kFp8) {
    if (launch.team == 1) hipLaunchKernelGGL((attend_few<kType, kFp8, D, 2, 1>), grid, dim3(64), 0, s, a);
    else hipLaunchKernelGGL((attend_few<kType, kFp8, D, 2, 4>), grid, block, 0, s, a);
  }
  return (int)hipGetLastError();
}

template <int D>
int attend_dim(const Attend& a, const Launch& launch, void* stream) {
  if (launch.type == MX_TYPE_BF16)
    return launch.fp8 ? attend_typed<D, MX_TYPE_BF16, true>(a, launch, stream)
                      : attend_typed<D, MX_TYPE_BF16, false>(a, launch, stream);
  return launch.fp8 ? attend_typed<D, MX_TYPE_F16, true>(a, launch, stream)
                    : attend_typed<D, MX_TYPE_F16, false>(a, launch, stream);
}

}  // namespace mxe
