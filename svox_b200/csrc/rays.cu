// Dispatch of the compositing of rays (rays.cuh) from sizes and types to its kernels.
#include "rays.cuh"

#include <type_traits>

#include "rays.h"
#include "status.h"

namespace svoxb {

int status_of_rays(int clear, int* word) {
    SVOXB_CUDA(cudaMemcpyFromSymbol(word, g_status, sizeof(int)));
    if (clear && *word != 0) {
        const int zero = 0;
        SVOXB_CUDA(cudaMemcpyToSymbol(g_status, &zero, sizeof(int)));
    }
    return SVOXB_OK;
}

int ray_group(const svoxb_scan* s) {
    if (!s->last_only || !s->reverse || s->H != 1 || s->C > kRayChannels) return 0;
    const int64_t mean = s->offsets ? (s->B > 0 ? s->T / s->B : 0) : s->T;
    // (their lengths are counted in 32 bits)
    if (mean > kRayLongest || (s->offsets && s->T > 0x7fffffff)) return 0;
    return mean <= kRayShort ? 8 : 32;
}

int64_t ray_kept(const svoxb_scan* s, int group) {
    return s->offsets ? s->T / group + s->B : s->B * ((s->T + group - 1) / group);
}

namespace {

ScanArgs ray_args(const svoxb_scan* s) {
    ScanArgs p{};
    p.x = s->values; p.g = s->thickness; p.h0 = s->initial; p.offsets = s->offsets;
    p.B = s->B; p.T = s->T; p.C = s->C; p.H = 1; p.D = s->C;
    p.xb = s->values_row; p.xs = s->values_step; p.gb = s->thickness_row; p.gs = s->thickness_step;
    p.hb = s->initial_row;
    p.reverse = 1;
    p.weighted = s->weighted;
    return p;
}

// Calls f with the types, the channels and the lanes of a ray.
template <class VT, class GT> struct Types { using V = VT; using G = GT; };
template <int N> using Int = std::integral_constant<int, N>;
template <class F>
void with_kernel(const svoxb_scan* s, int group, F f) {
    auto lanes = [&](auto t, auto c) {
        if (group == 8) f(t, c, Int<8>{});
        else f(t, c, Int<32>{});
    };
    auto types = [&](auto t) {
        switch (s->C) {
            case 1: return lanes(t, Int<1>{});
            case 2: return lanes(t, Int<2>{});
            case 3: return lanes(t, Int<3>{});
            default: return lanes(t, Int<4>{});
        }
    };
    const bool same = s->thickness_type == s->values_type;
    if (s->values_type == SVOXB_TYPE_F32) types(Types<float, float>{});
    else if (s->values_type == SVOXB_TYPE_BF16 && same) types(Types<__nv_bfloat16, __nv_bfloat16>{});
    else if (s->values_type == SVOXB_TYPE_BF16) types(Types<__nv_bfloat16, float>{});
    else if (same) types(Types<__half, __half>{});
    else types(Types<__half, float>{});
}

unsigned blocks_of(const svoxb_scan* s, int group) {
    return (unsigned)((s->B * group + kRayBlock - 1) / kRayBlock);
}

}  // namespace

int ray_forward(const svoxb_scan* s, int group, float* last, float* kept, cudaStream_t stream) {
    with_kernel(s, group, [&](auto t, auto c, auto g) {
        using K = decltype(t);
        ray_kernel<typename K::V, typename K::G, decltype(c)::value, decltype(g)::value>
            <<<blocks_of(s, group), kRayBlock, 0, stream>>>(ray_args(s), last, kept);
    });
    SVOXB_CUDA(cudaGetLastError());
    return SVOXB_OK;
}

int ray_backward(const svoxb_scan* s, int group, const float* kept, const float* d_last, void* dx,
                 void* dg, float* dh0, cudaStream_t stream) {
    with_kernel(s, group, [&](auto t, auto c, auto g) {
        using K = decltype(t);
        using VT = typename K::V;
        using GT = typename K::G;
        ray_back_kernel<VT, GT, decltype(c)::value, decltype(g)::value>
            <<<blocks_of(s, group), kRayBlock, 0, stream>>>(ray_args(s), kept, d_last,
                                                            static_cast<VT*>(dx),
                                                            static_cast<GT*>(dg), dh0);
    });
    SVOXB_CUDA(cudaGetLastError());
    return SVOXB_OK;
}

}  // namespace svoxb
