// C-ABI entry points of the gated recurrence (see include/svox_b200.h) and the choice of its
// kernels.
#include "recurrence.cuh"

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

constexpr int kSteps = 8;           // steps of a thread's stretch

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
    const bool any = s->B > 0 && s->T > 0;
    if (any && (!s->values || !s->thickness)) return SVOXB_ERR_NULL;
    if (s->B > 0x7fffffff || s->T > (1LL << 40) || s->C > (1 << 24)) return SVOXB_ERR_TOO_LARGE;
    return SVOXB_OK;
}

struct Plan {
    ScanArgs p{};
    int wide = 1;               // channels of a thread
    int64_t steps = 0;          // of all rows
    int64_t blocks = 0;
    int chunk() const { return p.segs * kSteps; }
    int64_t kept() const {      // states kept for the backward pass
        if (p.B == 0) return 0;
        return (p.offsets ? p.T / chunk() + p.B : p.B * ((p.T + chunk() - 1) / chunk())) * p.C;
    }
    int64_t pair_bytes() const { return p.splits > 1 ? p.B * p.splits * p.C * 8 : 0; }
    int64_t part_bytes() const { return p.parts > 1 ? (int64_t)p.parts * steps * p.H * 4 : 0; }
};

// What decides the layout of the kept states comes from the sizes alone: the forward and the
// backward pass have to agree on it.  `pairs`: whether a thread may take two channels.
Plan make_plan(const svoxb_scan* s, bool pairs = true) {
    Plan plan;
    ScanArgs& p = plan.p;
    p.x = s->values; p.g = s->thickness; p.h0 = s->initial; p.offsets = s->offsets;
    p.B = s->B; p.T = s->T; p.C = s->C; p.H = s->H; p.D = s->C / s->H;
    p.xb = s->values_row; p.xs = s->values_step; p.gb = s->thickness_row; p.gs = s->thickness_step;
    p.hb = s->initial_row;
    p.reverse = s->reverse; p.weighted = s->weighted;
    plan.steps = p.offsets ? p.T : p.B * p.T;
    // two channels to a thread where every row of them lies on a boundary of two
    auto even = [](const void* ptr, int64_t row, int64_t step, size_t size) {
        return reinterpret_cast<uintptr_t>(ptr) % (2 * size) == 0 && row % 2 == 0 && step % 2 == 0;
    };
    const size_t vs = type_size(s->values_type), gs = type_size(s->thickness_type);
    if (pairs && p.C % 2 == 0 && (p.D == 1 || p.D % 2 == 0) && even(p.x, p.xb, p.xs, vs) &&
        (p.D > 1 || even(p.g, p.gb, p.gs, gs)) && p.C > 32)
        plan.wide = 2;
    const int W = 32 * plan.wide;
    p.parts = 1;
    if (p.D == 1) {
        p.tile = W;
        p.tiles = (p.C + W - 1) / W;
    } else if (p.D <= W) {
        p.tile = W / p.D * p.D;
        p.tiles = (p.C + p.tile - 1) / p.tile;
    } else {
        p.parts = (p.D + W - 1) / W;
        p.tile = W;
        p.tiles = p.H * p.parts;
    }
    p.units = p.B * p.tiles;
    // (rows of a packed call: as long as twice the average)
    const int64_t len = p.offsets ? (p.B > 0 ? (2 * p.T + p.B - 1) / p.B : 0) : p.T;
    p.segs = 1;
    while (p.segs < kScanWarps && p.segs * kSteps < len) p.segs *= 2;
    const int per = kScanWarps / p.segs;
    plan.blocks = (p.units + per - 1) / per;
    p.splits = 1;
    const int64_t chunks = (len + plan.chunk() - 1) / plan.chunk(), want = 4 * (int64_t)sm_count();
    if (plan.blocks > 0 && plan.blocks * 2 < want && chunks >= 8) {
        int64_t n = want / plan.blocks;
        if (n > chunks / 4) n = chunks / 4;
        if (n > 256) n = 256;
        p.splits = (int)n;
    }
    return plan;
}

template <class VT, class GT, int V, bool PC>
int run_forward(const Plan& plan, void* states, float* last, float* kept, void* workspace,
                cudaStream_t stream) {
    const ScanArgs& p = plan.p;
    const dim3 grid((unsigned)plan.blocks, p.splits);
    float2* pairs = static_cast<float2*>(workspace);
    if (p.splits > 1) {
        scan_pairs_kernel<VT, GT, V, PC, kSteps, false><<<grid, kScanBlock, 0, stream>>>(
            p, nullptr, pairs);
        SVOXB_CUDA(cudaGetLastError());
        if (states == nullptr && kept == nullptr) {
            scan_last_kernel<<<(unsigned)((p.B * p.C + 255) / 256), 256, 0, stream>>>(p, pairs,
                                                                                    last);
            SVOXB_CUDA(cudaGetLastError());
            return SVOXB_OK;
        }
    }
    scan_kernel<VT, GT, V, PC, kSteps><<<grid, kScanBlock, 0, stream>>>(
        p, pairs, static_cast<VT*>(states), last, kept);
    SVOXB_CUDA(cudaGetLastError());
    return SVOXB_OK;
}

template <class VT, class GT, int V, bool PC>
int run_backward(const Plan& plan, const float* kept, const void* d, const float* d_last,
                 void* dx, void* dg, float* dh0, void* workspace, cudaStream_t stream) {
    const ScanArgs& p = plan.p;
    const dim3 grid((unsigned)plan.blocks, p.splits);
    float2* pairs = static_cast<float2*>(workspace);
    float* parted = reinterpret_cast<float*>(static_cast<char*>(workspace) + plan.pair_bytes());
    const VT* dv = static_cast<const VT*>(d);
    if (p.splits > 1) {
        scan_pairs_kernel<VT, GT, V, PC, kSteps, true><<<grid, kScanBlock, 0, stream>>>(p, dv,
                                                                                      pairs);
        SVOXB_CUDA(cudaGetLastError());
    }
    scan_back_kernel<VT, GT, V, PC, kSteps><<<grid, kScanBlock, 0, stream>>>(
        p, pairs, kept, dv, d_last, static_cast<VT*>(dx), static_cast<GT*>(dg), parted, dh0);
    SVOXB_CUDA(cudaGetLastError());
    if (p.parts > 1 && dg != nullptr) {
        scan_parts_kernel<GT><<<(unsigned)((plan.steps * p.H + 255) / 256), 256, 0, stream>>>(
            p, parted, static_cast<GT*>(dg));
        SVOXB_CUDA(cudaGetLastError());
    }
    return SVOXB_OK;
}

// Calls f with the values' and the gates' type, the channels of a thread, and whether each channel
// has a gate of its own.
template <class VT, class GT> struct Types { using V = VT; using G = GT; };
template <int N> struct Int { static constexpr int value = N; };
template <bool B> struct Bool { static constexpr bool value = B; };
template <class F>
int with_kernel(const svoxb_scan* s, const Plan& plan, F f) {
    auto types = [&](auto t) {
        const bool pc = plan.p.D == 1;
        if (plan.wide == 2) return pc ? f(t, Int<2>{}, Bool<true>{}) : f(t, Int<2>{}, Bool<false>{});
        return pc ? f(t, Int<1>{}, Bool<true>{}) : f(t, Int<1>{}, Bool<false>{});
    };
    const bool same = s->thickness_type == s->values_type;
    switch (s->values_type) {
        case SVOXB_TYPE_F32: return types(Types<float, float>{});
        case SVOXB_TYPE_BF16:
            return same ? types(Types<__nv_bfloat16, __nv_bfloat16>{})
                        : types(Types<__nv_bfloat16, float>{});
        default:
            return same ? types(Types<__half, __half>{}) : types(Types<__half, float>{});
    }
}

bool on_pairs(const void* ptr, int type) {
    return reinterpret_cast<uintptr_t>(ptr) % (2 * type_size(type)) == 0;
}

int too_many(const Plan& plan) {
    return plan.blocks > 0x7fffffffLL ||
           (plan.p.parts > 1 && plan.steps * plan.p.H > (0x7fffffffLL << 8));
}

}  // namespace
}  // namespace svoxb

using namespace svoxb;

extern "C" {

int64_t svoxb_gated_scan_kept(const svoxb_scan* s) {
    if (validate(s) != SVOXB_OK) return -1;
    return make_plan(s).kept();
}

int64_t svoxb_gated_scan_workspace(const svoxb_scan* s, int backward) {
    if (validate(s) != SVOXB_OK) return -1;
    int64_t most = 0;
    for (const bool pairs : {false, true}) {
        const Plan plan = make_plan(s, pairs);
        const int64_t bytes = plan.pair_bytes() + (backward ? plan.part_bytes() : 0);
        if (bytes > most) most = bytes;
    }
    return most;
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
    const Plan plan = make_plan(s, on_pairs(states, s->values_type));
    if (!last || (plan.pair_bytes() > 0 && !workspace)) return SVOXB_ERR_NULL;
    if (too_many(plan)) return SVOXB_ERR_TOO_LARGE;
    return with_kernel(s, plan, [&](auto t, auto v, auto pc) {
        using K = decltype(t);
        return run_forward<typename K::V, typename K::G, decltype(v)::value, decltype(pc)::value>(
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
    const Plan plan = make_plan(s, on_pairs(d_states, s->values_type) &&
                                       on_pairs(d_values, s->values_type) &&
                                       (s->H != s->C || on_pairs(d_thickness, s->thickness_type)));
    if ((plan.kept() > 0 && !kept) || (plan.pair_bytes() + plan.part_bytes() > 0 && !workspace))
        return SVOXB_ERR_NULL;
    if (too_many(plan)) return SVOXB_ERR_TOO_LARGE;
    return with_kernel(s, plan, [&](auto t, auto v, auto pc) {
        using K = decltype(t);
        return run_backward<typename K::V, typename K::G, decltype(v)::value, decltype(pc)::value>(
            plan, kept, d_states, d_last, d_values, d_thickness, d_initial, workspace, str);
    });
}

}  // extern "C"
