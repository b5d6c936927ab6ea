// Order among the lanes of one wave that exchange values through LDS.
#pragma once
#include <hip/hip_runtime.h>

namespace m26g {

// What this wave's lanes have written to LDS and read from it so far comes before what any of them reads or writes next. No
// instruction: the LDS serves a wave's accesses in order, and the compiler is kept from moving them past each other.
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

}  // namespace m26g
