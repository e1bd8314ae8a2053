// mf_launch.cuh -- the device side of launch_overlapped() (mf_runtime.h).
#pragma once

namespace mf {

// Wait until all that is before this kernel in its stream is done and visible.
// Until then the kernel may not read or write global memory, and what it reads
// afterwards it reads with plain loads: the read-only path (ld.global.nc) takes
// its data to be constant for as long as the kernel lives, which here begins
// while the kernel before it still writes.
__device__ __forceinline__ void after_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// From here on (in every CTA, or when it ends) the next kernel of the stream
// may be set up, if it was launched with launch_overlapped().
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

}  // namespace mf
