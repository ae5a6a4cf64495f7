// How the classes of a row are shared out, and which components of the logits a share lies in. Plain C++, so that it can be checked without a GPU.
#pragma once

#ifndef PCB_HOST_DEVICE
#ifdef __CUDACC__
#define PCB_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define PCB_HOST_DEVICE inline
#endif
#endif

namespace pcb {

// Where share `share` of `shares` nearly equal ones starts (share == shares: where the last one ends). Up to 2^31 - 1 classes.
PCB_HOST_DEVICE int share_start(int classes, int share, int shares) { return (int)((long long)classes * share / shares); }

// The first component behind those with classes below `hi` (1 at least), `units` classes to a component. The sum may pass 2^31 (where a component has more than 2^30 classes), not 2^32. (As
// (hi - 1) / units + 1 the kernels of long rows, which are at the limit of their registers, kept more of them in memory: 4096 x 131072 bf16 186 us forward and 345 backward, 178 and 337 so.)
PCB_HOST_DEVICE int components_below(int hi, int units) { return (int)(((unsigned)hi + (unsigned)units - 1u) / (unsigned)units); }

}  // namespace pcb
