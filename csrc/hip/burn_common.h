// What the burns share.
#pragma once

#include <hip/hip_runtime.h>

namespace gpumon_hip {

// run(count) twice, `iters` in all, so that a burn's waves keep their slots to its end. Eight waves share a
// SIMD's matrix pipe, which any one of them fills. Left alone they are either done one after the other, and 55 %
// of the slots are held over the launch, or take turns, and 95 % are: which of the two has changed with
// nothing but the instructions after the loop. With the last 16th at a lower priority a wave that gets there
// waits until all have. Held, without and with it: bf16 54 and 92 %, fp8 57 and 95, mxfp8 55 and 96, mxfp4 56 and
// 94, at the same rates (a 64th, through which waves slip while they wait, 90 % of bf16).
template <typename F>
__device__ __forceinline__ void hold_slots(int iters, F run) {
  const int tail = iters / 16;
  __builtin_amdgcn_s_setprio(1);
  run(iters - tail);
  __builtin_amdgcn_s_setprio(0);
  run(tail);
}

}  // namespace gpumon_hip
