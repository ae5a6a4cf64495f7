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

// The first component behind those with classes below `hi` (1 at least), `units` classes to a component. (As (hi + units - 1) / units the sum passes 2^31 where a component has more
// than 2^30 classes: the last shares of such a row were empty.)
PCB_HOST_DEVICE int components_below(int hi, int units) { return (hi - 1) / units + 1; }

}  // namespace pcb
