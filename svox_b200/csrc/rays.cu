// Dispatch of the compositing of rays (rays.cuh) from sizes and types to its kernels.
#include "rays.cuh"

#include <type_traits>

#include "rays.h"
#include "status.h"

namespace svoxb {

// Rays of at most this many samples on average: beyond, a ray is split among blocks instead.
constexpr int64_t kRayLongest = 4096;
// Up to this many a ray gets 8 lanes instead of 32, a sample each.
constexpr int64_t kRayShort = 12;
// By quads a ray gets 4 lanes, and twice as many beyond each of these averages; a warp's window is four
// times as many rays as it has groups of lanes (none for 32 lanes).  Rays of 3 channels of exponentially
// distributed lengths, forward and backward, us with 4 / 8 / 16 lanes, and 32:
//   2^20 rays of 4: 145 / 238 / 439 / 1189, of 20: 323 / 356 / 515 / 1262, of 42: 598 / 547 / 648 / 1344;
//   2^16 of 84: 146 / 111 / 95 / 118; 2^17 of 160: 504 / 377 / 271 / 292; 2^15 of 600: 822 / 491 / 326 / 266
// and without windows: of 42, 725 / 726 / 860.
constexpr int64_t kQuadsMean[] = {28, 60, 240};
// Features of 136 to 256 channels (in 16 bits, whole 16-byte pieces): a warp to a ray from so many rays
// on, and from half as many where they are of no more samples than this; tiles before.  200 channels,
// forward and backward, us, a warp to a ray / tiles, on 16-byte boundaries: 512 rays of 64 samples
// 51 / 77, of 300 304 / 242; 256 of 64 51 / 45; 64 of 2000 1664 / 200; and off them: 1024 of 200 389 / 505,
// 512 of 300 484 / 314, 4096 of 64 168 / 688.
constexpr int64_t kWideRays = 1024, kWideShort = 128;
// Lanes that all rays together can have at once; 4096 rays of 21, forward: 9.1 / 6.0 / 4.3 / 4.0 us.
constexpr int64_t kQuadsFew = 1 << 17;
// Warps that a window of rays has to leave.
constexpr int64_t kWarpsBusy = 148 * 24;

int status_of_rays(int clear, int* word) {
    SVOXB_CUDA(cudaMemcpyFromSymbol(word, g_status, sizeof(int)));
    if (clear && *word != 0) {
        const int zero = 0;
        SVOXB_CUDA(cudaMemcpyToSymbol(g_status, &zero, sizeof(int)));
    }
    return SVOXB_OK;
}

RayPlan ray_plan(const svoxb_scan* s) {
    RayPlan plan;
    if (!s->last_only || !s->reverse || s->H != 1) return plan;
    const int64_t mean = s->offsets ? (s->B > 0 ? s->T / s->B : 0) : s->T;
    // (their lengths are counted in 32 bits)
    if (mean > kRayLongest || (s->offsets && s->T > 0x7fffffff - 256)) return plan;
    if (s->C > kRayChannels) {
        // (sizes and types alone choose between these kernels and the tiles, which keep other things
        // for the backward pass; where the rows lie, only how these read them)
        const int size = s->values_type == SVOXB_TYPE_F32 ? 4 : 2, piece = 16 / size;
        const bool pieces = s->C % piece == 0;
        const int64_t rays = mean <= kWideShort ? kWideRays / 2 : kWideRays;
        if (s->C > 128 && !(pieces && s->C / piece <= 32 && s->B >= rays)) return plan;
        const bool whole = reinterpret_cast<uintptr_t>(s->values) % 16 == 0 && pieces &&
                           s->values_step % piece == 0 && s->values_row % piece == 0;
        plan.share = whole ? piece : 1;
        const int shares = s->C / plan.share;
        plan.width = 1;
        while (plan.width < shares && plan.width < 32) plan.width *= 2;
        plan.lanes = 32;
        return plan;
    }
    const bool dense = s->values_step == s->C && s->thickness_step == 1 &&
                       (s->offsets || ((s->values_row == s->T * s->C || s->B == 1) &&
                                       (s->thickness_row == s->T || s->B == 1)));
    const auto on = [](const void* ptr, int type) {
        return reinterpret_cast<uintptr_t>(ptr) % (type == SVOXB_TYPE_F32 ? 16 : 8) == 0;
    };
    plan.fits = dense && on(s->values, s->values_type) && on(s->thickness, s->thickness_type);
    plan.quads = s->layout == 0 ? plan.fits : s->layout == 1;
    if (!plan.quads) {
        plan.lanes = mean <= kRayShort ? 8 : 32;
        return plan;
    }
    plan.lanes = 4;
    for (const int64_t upto : kQuadsMean)
        if (mean > upto) plan.lanes *= 2;
    // few rays: as many lanes as leave none of them without a place
    while (plan.lanes < 32 && s->B * plan.lanes * 2 <= kQuadsFew) plan.lanes *= 2;
    // (a ray to a warp ends when it ends)
    const int groups = 32 / plan.lanes;
    plan.window = groups > 1 && s->B / (4 * groups) >= kWarpsBusy ? 4 * groups : groups;
    return plan;
}

// Floats that the forward keeps: what reaches every chunk.  The chunks of quads begin
// with the ray's first quad, up to three samples in front of it, so that a ray may have one more:
// two rays never share an entry where ray b begins at first / chunk + 2 b.
int64_t ray_kept(const svoxb_scan* s, RayPlan plan) {
    const int chunk = plan.lanes * (plan.quads ? 4 : 1), more = plan.quads ? 1 : 0;
    return s->offsets ? s->T / chunk + s->B * (1 + more)
                      : s->B * ((s->T + chunk - 1) / chunk + more);
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
void with_kernel(const svoxb_scan* s, RayPlan plan, F f) {
    auto lanes = [&](auto t, auto c) {
        if (plan.quads && plan.lanes == 4) f(t, c, Int<4>{}, std::true_type{});
        else if (plan.quads && plan.lanes == 8) f(t, c, Int<8>{}, std::true_type{});
        else if (plan.quads && plan.lanes == 16) f(t, c, Int<16>{}, std::true_type{});
        else if (plan.quads) f(t, c, Int<32>{}, std::true_type{});
        else if (plan.lanes == 8) f(t, c, Int<8>{}, std::false_type{});
        else f(t, c, Int<32>{}, std::false_type{});
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

// The same for more channels: the types, the channels of a lane, and how often it has them.
template <class F>
void with_rows(const svoxb_scan* s, RayPlan plan, F f) {
    auto types = [&](auto t) {
        constexpr int piece = 16 / (int)sizeof(typename decltype(t)::V);
        if (plan.share > 1) f(t, Int<piece>{}, Int<1>{});
        else if (s->C <= 32) f(t, Int<1>{}, Int<1>{});
        else if (s->C <= 128 || piece == 4) f(t, Int<1>{}, Int<4>{});
        else if constexpr (piece == 8) f(t, Int<1>{}, Int<8>{});
    };
    const bool same = s->thickness_type == s->values_type;
    if (s->values_type == SVOXB_TYPE_F32) types(Types<float, float>{});
    else if (s->values_type == SVOXB_TYPE_BF16 && same) types(Types<__nv_bfloat16, __nv_bfloat16>{});
    else if (s->values_type == SVOXB_TYPE_BF16) types(Types<__nv_bfloat16, float>{});
    else if (same) types(Types<__half, __half>{});
    else types(Types<__half, float>{});
}

unsigned blocks_of(const svoxb_scan* s, RayPlan plan) {
    if (plan.quads) {
        const int64_t warps = (s->B + plan.window - 1) / plan.window;
        return (unsigned)((warps * 32 + kRayBlock - 1) / kRayBlock);
    }
    return (unsigned)((s->B * plan.lanes + kRayBlock - 1) / kRayBlock);
}

}  // namespace

int ray_forward(const svoxb_scan* s, RayPlan plan, float* last, float* kept, cudaStream_t stream) {
    ScanArgs p = ray_args(s);
    p.tile = plan.window;
    if (plan.width) {
        p.lanes = plan.width;
        with_rows(s, plan, [&](auto t, auto v, auto n) {
            row_kernel<typename decltype(t)::V, typename decltype(t)::G, decltype(v)::value,
                       decltype(n)::value>
                <<<blocks_of(s, plan), kRayBlock, 0, stream>>>(p, last, kept);
        });
        SVOXB_CUDA(cudaGetLastError());
        return SVOXB_OK;
    }
    with_kernel(s, plan, [&](auto t, auto c, auto g, auto quads) {
        using VT = typename decltype(t)::V;
        using GT = typename decltype(t)::G;
        constexpr int C = decltype(c)::value, G = decltype(g)::value;
        if constexpr (decltype(quads)::value)
            quad_kernel<VT, GT, C, G><<<blocks_of(s, plan), kRayBlock, 0, stream>>>(p, last, kept);
        else
            ray_kernel<VT, GT, C, G><<<blocks_of(s, plan), kRayBlock, 0, stream>>>(p, last, kept);
    });
    SVOXB_CUDA(cudaGetLastError());
    return SVOXB_OK;
}

int ray_backward(const svoxb_scan* s, RayPlan plan, const float* kept, const float* d_last, void* dx,
                 void* dg, float* dh0, cudaStream_t stream) {
    ScanArgs p = ray_args(s);
    p.tile = plan.window;
    if (plan.width) {
        p.lanes = plan.width;
        p.paired = reinterpret_cast<uintptr_t>(dx) % 16 == 0;
        with_rows(s, plan, [&](auto t, auto v, auto n) {
            using VT = typename decltype(t)::V;
            using GT = typename decltype(t)::G;
            row_back_kernel<VT, GT, decltype(v)::value, decltype(n)::value>
                <<<blocks_of(s, plan), kRayBlock, 0, stream>>>(
                    p, kept, d_last, static_cast<VT*>(dx), static_cast<GT*>(dg), dh0);
        });
        SVOXB_CUDA(cudaGetLastError());
        return SVOXB_OK;
    }
    with_kernel(s, plan, [&](auto t, auto c, auto g, auto quads) {
        using VT = typename decltype(t)::V;
        using GT = typename decltype(t)::G;
        constexpr int C = decltype(c)::value, G = decltype(g)::value;
        VT* x = static_cast<VT*>(dx);
        GT* gates = static_cast<GT*>(dg);
        p.paired = reinterpret_cast<uintptr_t>(x) % (4 * sizeof(VT)) == 0 &&
                   reinterpret_cast<uintptr_t>(gates) % (4 * sizeof(GT)) == 0;
        if constexpr (decltype(quads)::value)
            quad_back_kernel<VT, GT, C, G><<<blocks_of(s, plan), kRayBlock, 0, stream>>>(
                p, kept, d_last, x, gates, dh0);
        else
            ray_back_kernel<VT, GT, C, G><<<blocks_of(s, plan), kRayBlock, 0, stream>>>(
                p, kept, d_last, x, gates, dh0);
    });
    SVOXB_CUDA(cudaGetLastError());
    return SVOXB_OK;
}

}  // namespace svoxb
