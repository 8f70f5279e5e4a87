// The compositing of rays, for the entry points of the recurrence.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/svox_b200.h"

namespace svoxb {

// Rays of at most this many samples on average: beyond, a ray is split among blocks instead.
constexpr int64_t kRayLongest = 4096;
// Up to this many a ray gets 8 lanes instead of 32.
constexpr int64_t kRayShort = 12;

// Lanes of a ray; 0: not a call for these kernels.
int ray_group(const svoxb_scan* s);
int64_t ray_kept(const svoxb_scan* s, int group);
int ray_forward(const svoxb_scan* s, int group, float* last, float* kept, cudaStream_t stream);
int ray_backward(const svoxb_scan* s, int group, const float* kept, const float* d_last, void* dx,
                 void* dg, float* dh0, cudaStream_t stream);

}  // namespace svoxb
