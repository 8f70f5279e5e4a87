// The compositing of rays, for the entry points of the recurrence.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/svox_b200.h"

namespace svoxb {


// How a call goes to these kernels: lanes of a ray (0: not at all), whether a lane takes four
// neighbouring samples, and where there are more channels, lanes of a sample and channels of a lane.
struct RayPlan {
    int lanes = 0;
    bool quads = false, fits = true;    // (fits: the arrays lie as that takes them)
    int width = 0, share = 0;
    int window = 0;             // rays that a warp orders by length (quads)
};
RayPlan ray_plan(const svoxb_scan* s);
int64_t ray_kept(const svoxb_scan* s, RayPlan plan);
int ray_forward(const svoxb_scan* s, RayPlan plan, float* last, float* kept, cudaStream_t stream);
int ray_backward(const svoxb_scan* s, RayPlan plan, const float* kept, const float* d_last, void* dx,
                 void* dg, float* dh0, cudaStream_t stream);

}  // namespace svoxb
