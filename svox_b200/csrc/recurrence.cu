// C-ABI entry points of the gated recurrence (see include/svox_b200.h) and the choice of its
// kernels.
#include "recurrence.cuh"

#include <initializer_list>
#include <type_traits>

#include "rays.h"
#include "status.h"

namespace svoxb {

int status_of_recurrence(int clear, int* word) {
    SVOXB_CUDA(cudaMemcpyFromSymbol(word, g_status, sizeof(int)));
    if (clear && *word != 0) {
        const int zero = 0;
        SVOXB_CUDA(cudaMemcpyToSymbol(g_status, &zero, sizeof(int)));
    }
    return SVOXB_OK;
}

namespace {

size_t type_size(int type) { return type == SVOXB_TYPE_F32 ? 4 : 2; }

int validate(const svoxb_scan* s) {
    if (!s) return SVOXB_ERR_NULL;
    if (s->B < 0 || s->T < 0 || s->C < 1 || s->H < 1 || s->C % s->H != 0) return SVOXB_ERR_SHAPE;
    for (int t : {s->values_type, s->thickness_type})
        if (t != SVOXB_TYPE_F32 && t != SVOXB_TYPE_BF16 && t != SVOXB_TYPE_F16)
            return SVOXB_ERR_FORMAT;
    // gates in 32 bits or in the values' type
    if (s->thickness_type != SVOXB_TYPE_F32 && s->thickness_type != s->values_type)
        return SVOXB_ERR_FORMAT;
    if (s->layout < 0 || s->layout > 2) return SVOXB_ERR_OPTION;
    const bool any = s->B > 0 && s->T > 0;
    if (any && (!s->values || !s->thickness)) return SVOXB_ERR_NULL;
    if (s->B > 0x7fffffff || s->T > (1LL << 40) || s->C > (1 << 24)) return SVOXB_ERR_TOO_LARGE;
    return SVOXB_OK;
}

struct Plan {
    ScanArgs p{};
    bool channel_gates = false;     // a lane's two channels have a gate each
    int chunk = 1;                  // steps of a tile
    int64_t steps = 0;              // of all rows
    int64_t blocks = 0;
    int64_t kept() const {          // states kept for the backward pass
        if (p.B == 0) return 0;
        return (p.offsets ? p.T / chunk + p.B : p.B * ((p.T + chunk - 1) / chunk)) * p.C;
    }
    int64_t pair_bytes() const { return p.splits > 1 ? p.B * p.splits * p.C * 8 : 0; }
    int64_t part_bytes() const { return p.parts > 1 ? (int64_t)p.parts * steps * p.H * 4 : 0; }
};

// The largest of 16, 4 and `size` bytes that the address, the strides and the width of a tile's rows
// (`counts`, in elements) are multiples of.
int copied_at_once(const void* ptr, size_t size, std::initializer_list<int64_t> counts) {
    for (const size_t n : {(size_t)16, (size_t)4}) {
        bool fits = reinterpret_cast<uintptr_t>(ptr) % n == 0;
        for (const int64_t c : counts) fits = fits && c * (int64_t)size % (int64_t)n == 0;
        if (fits) return (int)n;
    }
    return (int)size;
}

// The tiles of a call.  Nothing that decides the layout of the kept states (tile, chunk) looks at
// more than the sizes: the forward and the backward pass have to agree on it.
Plan make_plan(const svoxb_scan* s) {
    Plan plan;
    ScanArgs& p = plan.p;
    p.x = s->values; p.g = s->thickness; p.h0 = s->initial; p.offsets = s->offsets;
    p.B = s->B; p.T = s->T; p.C = s->C; p.H = s->H; p.D = s->C / s->H;
    p.xb = s->values_row; p.xs = s->values_step; p.gb = s->thickness_row; p.gs = s->thickness_step;
    p.hb = s->initial_row;
    p.reverse = s->reverse; p.weighted = s->weighted;
    plan.steps = p.offsets ? p.T : p.B * p.T;
    const size_t vs = type_size(s->values_type), gs = type_size(s->thickness_type);
    // (a lane's two channels share a gate, or have one each, of their own or of their groups)
    plan.channel_gates = p.D == 1 || p.D % 2 != 0;
    // (rows of a packed call: as long as twice the average)
    const int64_t len = p.offsets ? (p.B > 0 ? (2 * p.T + p.B - 1) / p.B : 0) : p.T;
    auto tile = [&](int W) {
        p.parts = 1;
        if (p.D == 1) p.tile = p.C < W ? p.C : W;
        else if (p.D <= W) p.tile = p.C < W ? p.C : W / p.D * p.D;
        else { p.parts = (p.D + W - 1) / W; p.tile = W; }
        p.lanes = 1;
        while (p.lanes * 2 < p.tile) p.lanes *= 2;
        p.tiles = p.parts > 1 ? p.H * p.parts : (p.C + p.tile - 1) / p.tile;
        p.units = p.B * p.tiles;
        p.warps = 1;
        while (p.warps < kScanWarps && p.warps * (32 / p.lanes) * kSteps < len) p.warps *= 2;
        plan.chunk = p.warps * (32 / p.lanes) * kSteps;
        const int per = kScanWarps / p.warps;
        plan.blocks = (p.units + per - 1) / per;
        return (len + plan.chunk - 1) / plan.chunk;
    };
    // As wide tiles as give every multiprocessor a block and some a second one (160 blocks: 137 us wide
    // and 126 narrow, 88 and 74 with shared gates; 192: 138 and 143); narrow ones, which have more steps to
    // them, while a row is a few of them; else wide ones, and ranges of a row to several blocks,
    // which costs a pass over the inputs beforehand.  Forward and backward together, us, wide tiles
    // in ranges / narrow tiles without: 7 rows of 1001 steps of 333 channels 72 / 40, 16 of 512 of 256
    // (4 groups) 34 / 19, 4 of 2048 of 512 39 / 32 (8 groups: 41 / 38); with 64 narrow tiles instead of
    // 148, 1 of 4096 of 1024, 57 / 88 (before whole tiles had kernels of their own).
    const int sms = sm_count();
    int64_t chunks = 0;
    for (const int W : {64, 16}) {
        chunks = tile(W);
        if (plan.blocks * 8 >= sms * 9) break;
    }
    p.splits = 1;
    if (plan.blocks > 0 && plan.blocks < sms && (plan.blocks * 2 < sms || chunks > 8)) {
        const int64_t wide = tile(64);
        if (wide >= 8) {
            chunks = wide;
            int64_t n = 2 * (int64_t)sms / plan.blocks;
            if (n > chunks / 4) n = chunks / 4;
            if (n > 256) n = 256;
            p.splits = (int)n;
        } else {
            chunks = tile(16);
        }
    }
    const int64_t tiles_of = (chunks + p.splits - 1) / p.splits;
    // (of 32-bit values two tiles under way fill as much of the shared memory)
    const int most = vs == 2 ? kScanStages : 2;
    p.stages = tiles_of < 1 ? 1 : tiles_of < most ? (int)tiles_of : most;
    const int64_t last = p.parts > 1 ? p.D % p.tile : p.C % p.tile;
    const int64_t start = p.parts > 1 ? p.D : p.tile;       // distances of the tiles' starts
    p.x_bytes = copied_at_once(p.x, vs, {p.xb, p.xs, p.tile, last, start});
    p.d_bytes = (int)vs;
    p.g_bytes = copied_at_once(p.g, gs, {p.gb, p.gs, p.tile, last, start});
    return plan;
}

// Rows of C elements of `ptr` lie on boundaries of two, tile by tile.
bool in_twos(const Plan& plan, const void* ptr, int type) {
    const ScanArgs& p = plan.p;
    return reinterpret_cast<uintptr_t>(ptr) % (2 * type_size(type)) == 0 && p.C % 2 == 0 &&
           p.tile % 2 == 0 && (p.parts == 1 || p.D % 2 == 0);
}

template <class Kernel>
int ready(Kernel kernel, size_t smem) {
    int per_sm = 0;
    return blocks_per_sm(reinterpret_cast<const void*>(kernel), kScanBlock, smem, &per_sm);
}

// Calls f with the lanes of a row where every tile of the call is whole (see ScanThread), else 0.
template <class F>
int with_lanes(const Plan& plan, int d_bytes, F f) {
    const ScanArgs& p = plan.p;
    const bool whole = p.warps == kScanWarps && p.tile == 2 * p.lanes && p.x_bytes == 16 &&
                       d_bytes == 16 && p.paired &&
                       (p.parts > 1 ? p.D : p.C) % p.tile == 0 &&
                       (plan.channel_gates ? p.D == 1 && p.g_bytes == 16 : true);
    if (whole && p.lanes == 32) return f(std::integral_constant<int, 32>{});
    if (whole && p.lanes == 8) return f(std::integral_constant<int, 8>{});
    return f(std::integral_constant<int, 0>{});
}

template <class VT, class GT, bool PC, int MODE>
int launch_scan(const Plan& plan, const void* x, float2* pairs, void* states, float* last,
                float* kept, cudaStream_t stream) {
    using S = ScanShape<VT, GT, PC>;
    const size_t smem = (size_t)kScanWarps * plan.p.stages * (S::kX + S::kG);
    return with_lanes(plan, 16, [&](auto lanes) {
        auto kernel = scan_kernel<VT, GT, PC, MODE, decltype(lanes)::value>;
        const int st = ready(kernel, smem);
        if (st) return st;
        kernel<<<dim3((unsigned)plan.blocks, plan.p.splits), kScanBlock, smem, stream>>>(
            plan.p, static_cast<const VT*>(x), pairs, static_cast<VT*>(states), last, kept);
        SVOXB_CUDA(cudaGetLastError());
        return (int)SVOXB_OK;
    });
}

template <class VT, class GT, bool PC>
int run_forward(const Plan& plan, void* states, float* last, float* kept, void* workspace,
                cudaStream_t stream) {
    const ScanArgs& p = plan.p;
    float2* pairs = static_cast<float2*>(workspace);
    if (p.offsets == nullptr && p.T <= kFewSteps && p.B * p.C < (1LL << 37)) {
        auto few = [&](auto w) {
            constexpr int W = decltype(w)::value;
            const int64_t n = p.B * (p.C / W);
            scan_few_kernel<VT, GT, W><<<(unsigned)((n + 127) / 128), 128, 0, stream>>>(
                p, static_cast<VT*>(states), last, kept);
        };
        if (p.paired && p.x_bytes >= 2 * (int)sizeof(VT)) few(std::integral_constant<int, 2>{});
        else few(std::integral_constant<int, 1>{});
        SVOXB_CUDA(cudaGetLastError());
        return SVOXB_OK;
    }
    if (p.splits > 1) {
        const int st = launch_scan<VT, GT, PC, 1>(plan, p.x, pairs, nullptr, nullptr, nullptr,
                                                  stream);
        if (st) return st;
        if (states == nullptr && kept == nullptr) {
            scan_last_kernel<<<(unsigned)((p.B * p.C + 255) / 256), 256, 0, stream>>>(p, pairs,
                                                                                    last);
            SVOXB_CUDA(cudaGetLastError());
            return SVOXB_OK;
        }
    }
    return launch_scan<VT, GT, PC, 0>(plan, p.x, pairs, states, last, kept, stream);
}

template <class VT, class GT, bool PC>
int run_backward(const Plan& plan, const float* kept, const void* d, const float* d_last,
                 void* dx, void* dg, float* dh0, void* workspace, cudaStream_t stream) {
    using S = ScanShape<VT, GT, PC>;
    const ScanArgs& p = plan.p;
    float2* pairs = static_cast<float2*>(workspace);
    float* parted = reinterpret_cast<float*>(static_cast<char*>(workspace) + plan.pair_bytes());
    if (p.splits > 1) {
        // the gradients of the states in the values' place
        Plan back = plan;
        back.p.xb = 0;
        back.p.xs = p.C;
        back.p.x_bytes = p.d_bytes;
        if (!p.offsets) back.p.xb = p.T * p.C;
        const int st = launch_scan<VT, GT, PC, 2>(back, d, pairs, nullptr, nullptr, nullptr, stream);
        if (st) return st;
    }
    Plan two = plan;                    // three arrays: two tiles of each are as much as fits twice
    if (two.p.stages > 2) two.p.stages = 2;
    const size_t smem = (size_t)kScanWarps * (two.p.stages * (2 * S::kX + S::kG) +
                                              (p.D > 1 ? S::kSum : 0));
    const int st = with_lanes(two, d == nullptr ? 16 : p.d_bytes, [&](auto lanes) {
        auto kernel = scan_back_kernel<VT, GT, PC, decltype(lanes)::value>;
        const int bad = ready(kernel, smem);
        if (bad) return bad;
        kernel<<<dim3((unsigned)plan.blocks, p.splits), kScanBlock, smem, stream>>>(
            two.p, static_cast<const VT*>(p.x), pairs, kept, static_cast<const VT*>(d), d_last,
            static_cast<VT*>(dx), static_cast<GT*>(dg), parted, dh0);
        SVOXB_CUDA(cudaGetLastError());
        return (int)SVOXB_OK;
    });
    if (st) return st;
    if (p.parts > 1 && dg != nullptr) {
        scan_parts_kernel<GT><<<(unsigned)((plan.steps * p.H + 255) / 256), 256, 0, stream>>>(
            p, parted, static_cast<GT*>(dg));
        SVOXB_CUDA(cudaGetLastError());
    }
    return SVOXB_OK;
}

// Calls f with the values' and the gates' type, and whether each channel has a gate of its own.
template <class VT, class GT> struct Types { using V = VT; using G = GT; };
template <class F>
int with_kernel(const svoxb_scan* s, const Plan& plan, F f) {
    auto types = [&](auto t) {
        return plan.channel_gates ? f(t, std::true_type{}) : f(t, std::false_type{});
    };
    const bool same = s->thickness_type == s->values_type;
    switch (s->values_type) {
        // (a lane has one channel: gates that are shared stay shared)
        case SVOXB_TYPE_F32: return types(Types<float, float>{});
        case SVOXB_TYPE_BF16:
            return same ? types(Types<__nv_bfloat16, __nv_bfloat16>{})
                        : types(Types<__nv_bfloat16, float>{});
        default:
            return same ? types(Types<__half, __half>{}) : types(Types<__half, float>{});
    }
}

int too_many(const Plan& plan) {
    return plan.blocks > 0x7fffffffLL ||
           (plan.p.parts > 1 && plan.steps * plan.p.H > (0x7fffffffLL << 8));
}

}  // namespace
}  // namespace svoxb

using namespace svoxb;

extern "C" {

int32_t svoxb_gated_scan_layout(const svoxb_scan* s) {
    if (validate(s) != SVOXB_OK) return -1;
    return ray_plan(s).quads ? 1 : 2;
}

int64_t svoxb_gated_scan_kept(const svoxb_scan* s) {
    if (validate(s) != SVOXB_OK) return -1;
    if (const RayPlan rays = ray_plan(s); rays.lanes) return ray_kept(s, rays);
    return make_plan(s).kept();
}

int64_t svoxb_gated_scan_workspace(const svoxb_scan* s, int backward) {
    if (validate(s) != SVOXB_OK) return -1;
    if (ray_plan(s).lanes) return 0;
    const Plan plan = make_plan(s);
    return plan.pair_bytes() + (backward ? plan.part_bytes() : 0);
}

int svoxb_gated_scan(const svoxb_scan* s, void* states, float* last, float* kept, void* workspace,
                     void* stream) {
    const int st = validate(s);
    if (st) return st;
    const auto str = static_cast<cudaStream_t>(stream);
    if (s->B == 0) {
        if (s->offsets && states && s->T > 0)
            SVOXB_CUDA(cudaMemsetAsync(states, 0, s->T * s->C * type_size(s->values_type), str));
        return SVOXB_OK;
    }
    const bool any_states = s->offsets ? s->T > 0 : s->B * s->T > 0;
    if (!last || (any_states && (states == nullptr) != (s->last_only != 0))) return SVOXB_ERR_NULL;
    if (const RayPlan rays = ray_plan(s); rays.quads && !rays.fits) return SVOXB_ERR_OPTION;
    else if (rays.lanes)
        return ray_forward(s, rays, last, kept, str);
    Plan plan = make_plan(s);
    plan.p.paired = in_twos(plan, states, s->values_type);
    if (plan.pair_bytes() > 0 && !workspace) return SVOXB_ERR_NULL;
    if (too_many(plan)) return SVOXB_ERR_TOO_LARGE;
    return with_kernel(s, plan, [&](auto t, auto pc) {
        using K = decltype(t);
        return run_forward<typename K::V, typename K::G, decltype(pc)::value>(
            plan, states, last, kept, workspace, str);
    });
}

int svoxb_gated_scan_backward(const svoxb_scan* s, const float* kept, const void* d_states,
                              const float* d_last, void* d_values, void* d_thickness,
                              float* d_initial, void* workspace, void* stream) {
    const int st = validate(s);
    if (st) return st;
    const auto str = static_cast<cudaStream_t>(stream);
    if (s->B == 0) {
        if (s->offsets && s->T > 0) {
            if (d_values)
                SVOXB_CUDA(cudaMemsetAsync(d_values, 0, s->T * s->C * type_size(s->values_type), str));
            if (d_thickness)
                SVOXB_CUDA(cudaMemsetAsync(d_thickness, 0, s->T * s->H * type_size(s->thickness_type),
                                           str));
        }
        return SVOXB_OK;
    }
    if (s->last_only && d_states) return SVOXB_ERR_OPTION;
    if (const RayPlan rays = ray_plan(s); rays.lanes) {
        if (rays.quads && !rays.fits) return SVOXB_ERR_OPTION;
        if (ray_kept(s, rays) > 0 && !kept) return SVOXB_ERR_NULL;
        return ray_backward(s, rays, kept, d_last, d_values, d_thickness, d_initial, str);
    }
    Plan plan = make_plan(s);
    plan.p.paired = in_twos(plan, d_values, s->values_type) &&
                    (s->H != s->C || in_twos(plan, d_thickness, s->thickness_type));
    plan.p.d_bytes = copied_at_once(d_states, type_size(s->values_type),
                                    {s->C, plan.p.tile, plan.p.C % plan.p.tile,
                                     plan.p.parts > 1 ? plan.p.D : 0,
                                     plan.p.parts > 1 ? plan.p.D % plan.p.tile : 0});
    if ((plan.kept() > 0 && !kept) || (plan.pair_bytes() + plan.part_bytes() > 0 && !workspace))
        return SVOXB_ERR_NULL;
    if (too_many(plan)) return SVOXB_ERR_TOO_LARGE;
    return with_kernel(s, plan, [&](auto t, auto pc) {
        using K = decltype(t);
        return run_backward<typename K::V, typename K::G, decltype(pc)::value>(
            plan, kept, d_states, d_last, d_values, d_thickness, d_initial, workspace, str);
    });
}

}  // extern "C"
