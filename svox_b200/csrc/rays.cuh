// Compositing of samples with few channels that share their thickness: the colours of rays.
//
// The last state of the recurrence (recurrence.cuh), back to front, is a sum from the front,
//   out = sum of W[i] x[i] + T[n] background,   T[i] = a[0] ... a[i-1],   W[i] = T[i] w[i]
// so a group of G lanes walks a ray, a sample to a lane, and scans nothing but what reaches a sample
// (its products: exp of a sum of thicknesses would be off by the sum's rounding, 4e-6 of a background
// behind a thickness of 70); the channels are summed in each lane and over the lanes at the end.
// With d the upstream gradient and c[i] = d . x[i] the backward pass is
//   dx[i] = W[i] d,   dg[i] = T[i+1] c[i] - (sum over j > i of W[j] c[j] + T[n] d . background)
// one more scan of plain sums, from the far end, whatever the number of channels.  The forward keeps
// what reaches every G-th sample for it.
//
// Where the samples lie densely and on 16-byte boundaries (`quads`), a lane takes four neighbouring
// ones, whose four thicknesses are one request and their 4 C values C more.  The quads are those of
// the array, so that a ray's first and last one may have samples of its neighbours, which count as
// nothing.  That leaves a scan over the lanes for every four samples, and lets four rays share a
// warp without more requests to the L1 than one ray a warp made.
//
// In the tiles of recurrence.cuh, whose lanes are channels first, 2^20 rays of 42 samples of 3
// channels took 5.19 ms, and 9.25 ms backwards.
#pragma once

#include "recurrence.cuh"

namespace svoxb {

constexpr int kRayBlock = 64;       // (rays differ in length: blocks of few wait for few)
constexpr int kRayChannels = 4;     // of those whose channels are summed in every lane

// What reaches beyond each lane's N samples, and `reach` what reaches the group.  Behind an opaque
// sample nothing counts, a thickness that is not a number neither, and behind such a thickness nothing
// is known up to the next opaque sample.  `careful`: some product here is not a number, so that the
// lanes tell what is in front of what (and the gates of samples that nothing reaches are closed).
template <int G, int N>
__device__ __forceinline__ float reach_beyond(int lane, float reach, Gate (&gate)[N], bool& careful) {
    float v = gate[0].a;
    if (N == 4) v = (gate[0].a * gate[1 % N].a) * (gate[2 % N].a * gate[3 % N].a);
#pragma unroll
    for (int d = 1; d < G; d *= 2) {
        const float o = __shfl_up_sync(~0u, v, d, G);
        if (lane >= d) v *= o;
    }
    v *= reach;
    careful = __any_sync(~0u, v != v);
    if (careful) {
        // of the lane's samples, then of all up to them: what is left of 1, and whether one is opaque
        float left = 1.f;
        bool opaque = false;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            opaque |= gate[i].a == 0.f;
            left = left == 0.f || gate[i].a == 0.f ? 0.f : left * gate[i].a;
        }
#pragma unroll
        for (int d = 1; d < G; d *= 2) {
            const float o = __shfl_up_sync(~0u, left, d, G);
            const bool shut = __shfl_up_sync(~0u, opaque, d, G);
            if (lane < d) continue;
            left = o == 0.f || (o != o && opaque) ? 0.f : o * left;
            opaque |= shut;
        }
        if (v != v) v = reach == 0.f || (reach != reach && opaque) ? 0.f : reach * left;
        float front = __shfl_up_sync(~0u, v, 1, G);
        if (lane == 0) front = reach;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (front == 0.f) gate[i] = Gate{0.f, 0.f};
            front = gate[i].a == 0.f ? 0.f : front * gate[i].a;
        }
    }
    return v;
}

template <class VT, class GT, int C, int G>
struct RayThread {
    int lane;                       // in the group
    int64_t b, first;
    bool there;
    int len;                        // (a call for these kernels has fewer than 2^31 samples)
    int chunks, most;               // of G samples: of this ray, of the warp's longest
    const VT* x;
    const GT* g;

    __device__ __forceinline__ void init(const ScanArgs& p) {
        lane = threadIdx.x % G;
        b = ((int64_t)blockIdx.x * kRayBlock + threadIdx.x) / G;
        there = b < p.B;
        if (!there) b = p.B - 1;
        const ScanRow row = scan_row(p, b);
        first = row.first;
        len = there ? (int)row.len : 0;
        x = static_cast<const VT*>(p.x) + (p.offsets ? first * p.xs : b * p.xb) + lane * p.xs;
        g = static_cast<const GT*>(p.g) + (p.offsets ? first * p.gs : b * p.gb) + lane * p.gs;
        chunks = (len + G - 1) / G;
        most = G == 32 ? chunks : __reduce_max_sync(~0u, chunks);
    }
    __device__ __forceinline__ int64_t kept_at(const ScanArgs& p) const {
        return p.offsets ? first / G + b : b * ((p.T + G - 1) / G);
    }
    // Sum over this lane and the ones behind it.
    __device__ __forceinline__ float from(float v) const {
#pragma unroll
        for (int d = 1; d < G; d *= 2) {
            const float o = __shfl_down_sync(~0u, v, d, G);
            if (lane + d < G) v += o;
        }
        return v;
    }
};

template <class VT, class GT, int C, int G>
__global__ void __launch_bounds__(kRayBlock)
ray_kernel(ScanArgs p, float* __restrict__ last, float* __restrict__ kept) {
    RayThread<VT, GT, C, G> th;
    th.init(p);
    float reach = 1.f, acc[C];          // what reaches the chunk
#pragma unroll
    for (int c = 0; c < C; ++c) acc[c] = 0.f;
    const int64_t dx = G * p.xs, dg = G * p.gs;
    float* keep = kept != nullptr && th.lane == 0 ? kept + th.kept_at(p) : nullptr;
    int left = th.len - th.lane;            // samples from this lane's one on
    for (int k = 0; k < th.most; ++k) {
        const bool in = left > 0;
        float xv[C];
        const float gi = in ? to_float(*th.g) : 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c) xv[c] = in ? to_float(th.x[c]) : 0.f;
        left -= G;
        th.x += dx;
        th.g += dg;
        if (keep != nullptr && in) *keep++ = reach;
        Gate gates[1] = {gate_of(gi)};
        bool careful;
        const float v = reach_beyond<G>(th.lane, reach, gates, careful);
        const Gate gate = gates[0];
        float T = __shfl_up_sync(~0u, v, 1, G);
        if (th.lane == 0) T = reach;
        reach = __shfl_sync(~0u, v, G - 1, G);
        const float W = p.weighted ? T : T * gate.w;
        if (W != 0.f)
#pragma unroll
            for (int c = 0; c < C; ++c) acc[c] = fmaf(W, xv[c], acc[c]);
    }
#pragma unroll
    for (int d = G / 2; d > 0; d /= 2)
#pragma unroll
        for (int c = 0; c < C; ++c) acc[c] += __shfl_xor_sync(~0u, acc[c], d);
    if (!th.there) return;
#pragma unroll
    for (int c = 0; c < C; ++c)
        if (th.lane == c) {
            const float bg = p.h0 != nullptr ? __ldg(p.h0 + th.b * p.hb + c) : 0.f;
            last[th.b * C + c] = past(reach, bg, acc[c]);
        }
}

template <class VT, class GT, int C, int G>
__global__ void __launch_bounds__(kRayBlock)
ray_back_kernel(ScanArgs p, const float* __restrict__ kept, const float* __restrict__ d_last,
                VT* __restrict__ dx, GT* __restrict__ dg, float* __restrict__ dh0) {
    clear_uncovered(p, C, dx);
    clear_uncovered(p, 1, dg);
    RayThread<VT, GT, C, G> th;
    th.init(p);
    float d[C], bg = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        d[c] = d_last != nullptr && th.there ? __ldg(d_last + th.b * C + c) : 0.f;
        if (p.h0 != nullptr && th.there) bg = fmaf(d[c], __ldg(p.h0 + th.b * p.hb + c), bg);
    }
    // The values' gradients leave as one stretch: in its j-th store a lane has element j * G + lane,
    // of sample `whose[j]`.
    int whose[C];
    float scale[C];
#pragma unroll
    for (int j = 0; j < C; ++j) {
        const int e = j * G + th.lane;
        whose[j] = e / C;
#pragma unroll
        for (int c = 0; c < C; ++c)
            if (e % C == c) scale[j] = d[c];
    }
    const float* const keep = kept + th.kept_at(p);
    float T_end = 1.f, behind = 0.f;        // what the samples behind the chunk bring
    const int64_t step_x = G * p.xs, step_g = G * p.gs;
    th.x += (int64_t)(th.most - 1) * step_x;
    th.g += (int64_t)(th.most - 1) * step_g;
    GT* to_g = dg == nullptr ? nullptr : dg + th.first + (int64_t)(th.most - 1) * G + th.lane;
    VT* to_x = dx == nullptr ? nullptr
                             : dx + (th.first + (int64_t)(th.most - 1) * G) * C + th.lane;
    int left = th.len - (th.most - 1) * G;  // samples from the chunk's first on
    for (int k = th.most - 1; k >= 0; --k, left += G) {
        const bool in = th.lane < left;
        const float reach = left > 0 ? keep[k] : 1.f;
        const float gi = in ? to_float(*th.g) : 0.f;
        float xv[C], c = 0.f;
#pragma unroll
        for (int q = 0; q < C; ++q) xv[q] = in ? to_float(th.x[q]) : 0.f;
#pragma unroll
        for (int q = 0; q < C; ++q) c = fmaf(d[q], xv[q], c);
        th.x -= step_x;
        th.g -= step_g;
        Gate gates[1] = {gate_of(gi)};
        bool careful;
        const float v = reach_beyond<G>(th.lane, reach, gates, careful);
        const Gate gate = gates[0];
        float T = __shfl_up_sync(~0u, v, 1, G);
        if (th.lane == 0) T = reach;
        const float total = __shfl_sync(~0u, v, G - 1, G);
        if (left > 0 && left <= G) {        // the ray's last chunk
            T_end = total;
            behind = past(T_end, bg, 0.f);
        }
        const float Tn = T * gate.a;
        const float w = p.weighted ? (in ? 1.f : 0.f) : gate.w, W = T * w;
        const float here = th.from(times(W, c)) + behind;       // of this sample and all behind it
        float rest = __shfl_down_sync(~0u, here, 1, G);
        if (th.lane == G - 1) rest = behind;
        behind = __shfl_sync(~0u, here, 0, G);
        if (to_g != nullptr) {
            // (a value that is not finite in a place of no thickness is no sample)
            const float own = p.weighted || Tn == 0.f ? 0.f : Tn * c;
            if (in) *to_g = from_float<GT>(w == 0.f && !finite(c) ? 0.f : own - rest);
            to_g -= G;
        }
        if (to_x != nullptr) {
#pragma unroll
            for (int j = 0; j < C; ++j) {
                const float Wj = __shfl_sync(~0u, W, whose[j], G);
                if (whose[j] < left) to_x[j * G] = from_float<VT>(Wj * scale[j]);
            }
            to_x -= G * C;
        }
    }
    if (!th.there) return;
    if (dh0 != nullptr)
#pragma unroll
        for (int c = 0; c < C; ++c)
            if (th.lane == c) dh0[th.b * C + c] = past(T_end, d[c], 0.f);
}

// ---------------------------------------------------------------------------
// The same by quads.  The rays of a warp's groups end together only if they are as long; so a warp
// takes `window` rays, orders them by their lengths and goes through them, as many at a time as it
// has groups.  For exponentially distributed lengths of 48 samples on average, four rays at a time
// take 3.4 rounds of 32 samples as they come and 2.5 out of 16 (2^20 such rays with gradients: 726 ->
// 547 us).

template <class VT, class GT, int C, int G>
struct RayQuads {
    static constexpr int kChunk = 4 * G;
    int lane;
    int64_t b, first;
    bool there;
    int len, lead;                  // samples; those of the first quad that are not this ray's
    int chunks, most;
    int64_t rest;                   // samples of the array from the lane's first one on

    // The warp's rays, by falling length.
    struct Ray { int64_t first; int len, from; };
    int64_t base;
    const Ray* rays;
    __device__ __forceinline__ void init(const ScanArgs& p, Ray (&shared)[kRayBlock]) {
        const int me = threadIdx.x & 31;
        lane = threadIdx.x % G;
        base = ((int64_t)blockIdx.x * (kRayBlock / 32) + threadIdx.x / 32) * p.tile;
        const bool here = me < p.tile && base + me < p.B;
        const ScanRow row = scan_row(p, here ? base + me : p.B - 1);
        const int len = here ? (int)row.len : -1;
        int rank = me;
        if (p.offsets != nullptr && p.tile > 32 / G) {
            rank = 0;
            for (int j = 0; j < p.tile; ++j) {
                const int o = __shfl_sync(~0u, len, j);
                rank += o > len || (o == len && j < me);
            }
        }
        Ray* const all = shared + (threadIdx.x & ~31);
        if (me < p.tile) all[rank] = Ray{row.first, len, me};
        rays = all + (threadIdx.x & 31) / G;
        __syncwarp();
    }
    // The group's ray of round r.
    __device__ __forceinline__ void take(const ScanArgs& p, int r) {
        const Ray ray = rays[r * (32 / G)];
        b = base + ray.from;
        first = ray.first;
        len = ray.len;
        there = len >= 0;
        if (!there) len = 0;
        lead = (int)(first & 3);
        chunks = len > 0 ? (int)(((int64_t)lead + len + kChunk - 1) / kChunk) : 0;
        most = G == 32 ? chunks : __reduce_max_sync(~0u, chunks);
        rest = (p.offsets ? p.T : p.B * p.T) - (first - lead) - 4 * lane;
    }
    // (see svoxb_gated_scan_kept)
    __device__ __forceinline__ int64_t kept_at(const ScanArgs& p) const {
        return p.offsets ? first / kChunk + 2 * b : b * ((p.T + kChunk - 1) / kChunk + 1);
    }
    // Place of the lane's quad of chunk k in the ray: samples pos .. pos + 3.
    __device__ __forceinline__ int pos(int k) const { return k * kChunk + 4 * lane - lead; }
    __device__ __forceinline__ bool in(int at) const { return (unsigned)at < (unsigned)len; }
    template <class T, int N>
    __device__ __forceinline__ void load(const T* all, int at, int64_t left, float (&v)[4 * N]) const {
        const T* from = all + (first + at) * N;
        if (left >= 4) {
#pragma unroll
            for (int j = 0; j < N; ++j) {
                float q[4];
                load_some<4>(from + 4 * j, q);
#pragma unroll
                for (int i = 0; i < 4; ++i) v[4 * j + i] = q[i];
            }
        } else {            // the array ends within the quad
#pragma unroll
            for (int i = 0; i < 4 * N; ++i) v[i] = i < left * N ? to_float(from[i]) : 0.f;
        }
    }
    __device__ __forceinline__ float from(float v) const {
#pragma unroll
        for (int d = 1; d < G; d *= 2) {
            const float o = __shfl_down_sync(~0u, v, d, G);
            if (lane + d < G) v += o;
        }
        return v;
    }
};

template <class VT, class GT, int C, int G>
__global__ void __launch_bounds__(kRayBlock, 20)
quad_kernel(ScanArgs p, float* __restrict__ last, float* __restrict__ kept) {
    __shared__ typename RayQuads<VT, GT, C, G>::Ray s_rays[kRayBlock];
    RayQuads<VT, GT, C, G> th;
    th.init(p, s_rays);
    const VT* const x = static_cast<const VT*>(p.x);
    const GT* const g = static_cast<const GT*>(p.g);
    for (int r = 0; r < p.tile / (32 / G); ++r) {
        th.take(p, r);
        float reach = 1.f, acc[C];
#pragma unroll
        for (int c = 0; c < C; ++c) acc[c] = 0.f;
        float* const keep = kept != nullptr && th.lane == 0 ? kept + th.kept_at(p) : nullptr;
        for (int k = 0; k < th.most; ++k) {
            const int at = th.pos(k);
            float gv[4] = {0.f, 0.f, 0.f, 0.f}, xv[4 * C];
            if (at < th.len) {
                const int64_t left = th.rest - (int64_t)k * th.kChunk;
                th.template load<GT, 1>(g, at, left, gv);
                th.template load<VT, C>(x, at, left, xv);
            } else {
#pragma unroll
                for (int i = 0; i < 4 * C; ++i) xv[i] = 0.f;
            }
            if (keep != nullptr && k < th.chunks) keep[k] = reach;
            Gate gate[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                gv[i] = th.in(at + i) ? gv[i] : 0.f;
                gate[i] = gate_of(gv[i]);
            }
            bool careful;
            const float v = reach_beyond<G>(th.lane, reach, gate, careful);
            float T = __shfl_up_sync(~0u, v, 1, G);
            if (th.lane == 0) T = reach;
            reach = __shfl_sync(~0u, v, G - 1, G);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float W = p.weighted ? (th.in(at + i) ? T : 0.f) : T * gate[i].w;
                if (W != 0.f)
#pragma unroll
                    for (int c = 0; c < C; ++c) acc[c] = fmaf(W, xv[i * C + c], acc[c]);
                T *= gate[i].a;
                if (careful && gate[i].a == 0.f) T = 0.f;
            }
        }
#pragma unroll
        for (int d = G / 2; d > 0; d /= 2)
#pragma unroll
            for (int c = 0; c < C; ++c) acc[c] += __shfl_xor_sync(~0u, acc[c], d);
#pragma unroll
        for (int c = 0; c < C; ++c)
            if (th.lane == c && th.there) {
                const float bg = p.h0 != nullptr ? __ldg(p.h0 + th.b * p.hb + c) : 0.f;
                last[th.b * C + c] = past(reach, bg, acc[c]);
            }
    }
}

template <class VT, class GT, int C, int G>
__global__ void __launch_bounds__(kRayBlock, 16)
quad_back_kernel(ScanArgs p, const float* __restrict__ kept, const float* __restrict__ d_last,
                 VT* __restrict__ dx, GT* __restrict__ dg, float* __restrict__ dh0) {
    clear_uncovered(p, C, dx);
    clear_uncovered(p, 1, dg);
    __shared__ typename RayQuads<VT, GT, C, G>::Ray s_rays[kRayBlock];
    RayQuads<VT, GT, C, G> th;
    th.init(p, s_rays);
    const VT* const x = static_cast<const VT*>(p.x);
    const GT* const g = static_cast<const GT*>(p.g);
    for (int r = 0; r < p.tile / (32 / G); ++r) {
        th.take(p, r);
        float d[C], bg = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            d[c] = d_last != nullptr && th.there ? __ldg(d_last + th.b * C + c) : 0.f;
            if (p.h0 != nullptr && th.there) bg = fmaf(d[c], __ldg(p.h0 + th.b * p.hb + c), bg);
        }
        const float* const keep = kept + th.kept_at(p);
        float T_end = 1.f, behind = 0.f;        // what the samples behind the chunk bring
        for (int k = th.most - 1; k >= 0; --k) {
            const int at = th.pos(k);
            const float reach = k < th.chunks ? keep[k] : 1.f;
            float gv[4] = {0.f, 0.f, 0.f, 0.f}, xv[4 * C];
            if (at < th.len) {
                const int64_t left = th.rest - (int64_t)k * th.kChunk;
                th.template load<GT, 1>(g, at, left, gv);
                th.template load<VT, C>(x, at, left, xv);
            } else {
#pragma unroll
                for (int i = 0; i < 4 * C; ++i) xv[i] = 0.f;
            }
            Gate gate[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                gv[i] = th.in(at + i) ? gv[i] : 0.f;
                gate[i] = gate_of(gv[i]);
            }
            bool careful;
            const float v = reach_beyond<G>(th.lane, reach, gate, careful);
            float T = __shfl_up_sync(~0u, v, 1, G);
            if (th.lane == 0) T = reach;
            const float total = __shfl_sync(~0u, v, G - 1, G);
            if (k == th.chunks - 1) {
                T_end = total;
                behind = past(T_end, bg, 0.f);
            }
            const float front = T;
            float W[4], c[4], Wc[4], own[4];
            unsigned none = 0;          // samples that have no gradient of their thickness
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                c[i] = 0.f;
#pragma unroll
                for (int q = 0; q < C; ++q) c[i] = fmaf(d[q], xv[i * C + q], c[i]);
                W[i] = T * (p.weighted ? (th.in(at + i) ? 1.f : 0.f) : gate[i].w);
                Wc[i] = W[i] * c[i];
                T *= gate[i].a;
                if (careful && gate[i].a == 0.f) T = 0.f;
                own[i] = p.weighted ? 0.f : T * c[i];
            }
            if (!finite((c[0] + c[1]) + (c[2] + c[3]))) {
                // What is not finite counts only where it has weight, and past its sample only what
                // that lets through; where there is no thickness it is no sample.
                float past_it = front;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    Wc[i] = times(W[i], c[i]);
                    past_it = gate[i].a == 0.f ? 0.f : past_it * gate[i].a;
                    if (!p.weighted) own[i] = times(past_it, c[i]);
                    if (!finite(c[i]) && !p.weighted && gate[i].w == 0.f) none |= 1u << i;
                }
            }
            const float here = th.from((Wc[0] + Wc[1]) + (Wc[2] + Wc[3])) + behind;
            float rest = __shfl_down_sync(~0u, here, 1, G);     // what all behind the quad bring
            if (th.lane == G - 1) rest = behind;
            behind = __shfl_sync(~0u, here, 0, G);
            if (at < th.len) {
                float out[4];
#pragma unroll
                for (int i = 3; i >= 0; --i) {
                    out[i] = own[i] - rest;
                    rest += Wc[i];
                }
                if (none)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (none >> i & 1) out[i] = 0.f;
                const bool whole = at >= 0 && at + 3 < th.len;
                const int64_t to = th.first + at;
                if (dg != nullptr) {
                    if (whole && p.paired) store_some<4>(dg + to, out);
                    else
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (th.in(at + i)) dg[to + i] = from_float<GT>(out[i]);
                }
                if (dx != nullptr) {
                    if (whole && p.paired) {
#pragma unroll
                        for (int j = 0; j < C; ++j) {
                            float q[4];
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                q[i] = W[(4 * j + i) / C] * d[(4 * j + i) % C];
                            store_some<4>(dx + to * C + 4 * j, q);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (th.in(at + i))
#pragma unroll
                                for (int c = 0; c < C; ++c)
                                    dx[(to + i) * C + c] = from_float<VT>(W[i] * d[c]);
                    }
                }
            }
        }
        if (!th.there) continue;
        if (dh0 != nullptr)
#pragma unroll
            for (int c = 0; c < C; ++c)
                if (th.lane == c) dh0[th.b * C + c] = past(T_end, d[c], 0.f);
    }
}

// ---------------------------------------------------------------------------
// Values of more channels (features): 32 samples are weighted at a time, one to a lane, and then
// their values go by, `width` lanes to a sample with V channels each (16 bytes where rows lie on
// 16-byte boundaries), NT times over where a lane's share is one channel and there are more than 32.
// The exponentials are those of the samples, not of their channels.
template <class VT, class GT, int V, int NT>
struct RayRows {
    int width, per;             // lanes of a sample; samples that go by at once
    int sub, cl;                // which of those is this lane's; its share
    int have;                   // lanes' shares of a row that exist: cl + t * 32 < have

    __device__ __forceinline__ void init(const ScanArgs& p) {
        const int lane = threadIdx.x & 31;
        width = p.lanes;
        per = 32 / width;
        sub = lane / width;
        cl = lane - sub * width;
        have = p.C / V;
    }
    __device__ __forceinline__ bool on(int t) const { return cl + 32 * t < have; }
    __device__ __forceinline__ int ch(int t) const { return (cl + 32 * t) * V; }
};

template <class VT, class GT, int V, int NT>
__global__ void __launch_bounds__(kRayBlock)
row_kernel(ScanArgs p, float* __restrict__ last, float* __restrict__ kept) {
    RayThread<VT, GT, 1, 32> th;
    RayRows<VT, GT, V, NT> rows;
    th.init(p);
    rows.init(p);
    float reach = 1.f, acc[NT][V];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int v = 0; v < V; ++v) acc[t][v] = 0.f;
    float* keep = kept != nullptr && th.lane == 0 ? kept + th.kept_at(p) : nullptr;
    const VT* x = th.x + ((int64_t)rows.sub - th.lane) * p.xs;      // this lane's row of the chunk
    float g_next = th.lane < th.len ? to_float(*th.g) : 0.f;
    for (int k = 0; k < th.chunks; ++k) {
        const int left = th.len - 32 * k;
        const float gi = g_next;
        th.g += 32 * p.gs;
        g_next = th.lane + 32 < left ? to_float(*th.g) : 0.f;
        if (keep != nullptr) keep[k] = reach;
        Gate gates[1] = {gate_of(gi)};
        bool careful;
        const float v = reach_beyond<32>(th.lane, reach, gates, careful);
        const Gate gate = gates[0];
        float T = __shfl_up_sync(~0u, v, 1);
        if (th.lane == 0) T = reach;
        reach = __shfl_sync(~0u, v, 31);
        const float W = p.weighted ? T : T * gate.w;
        const int n = left < 32 ? (left + rows.per - 1) / rows.per : rows.width;
#pragma unroll 4
        for (int j = 0; j < n; ++j) {
            const int s = j * rows.per + rows.sub;
            const VT* const row = x + (int64_t)(j * rows.per) * p.xs;
            const float w = __shfl_sync(~0u, W, s);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                float xv[V];
#pragma unroll
                for (int q = 0; q < V; ++q) xv[q] = 0.f;
                if (s < left && rows.on(t)) load_some<V>(row + rows.ch(t), xv);
                if (w != 0.f)
#pragma unroll
                    for (int q = 0; q < V; ++q) acc[t][q] = fmaf(w, xv[q], acc[t][q]);
            }
        }
        x += 32 * p.xs;
    }
    if (!th.there) return;
    for (int d = rows.width; d < 32; d *= 2)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int q = 0; q < V; ++q) acc[t][q] += __shfl_xor_sync(~0u, acc[t][q], d);
    if (rows.sub == 0)
#pragma unroll
        for (int t = 0; t < NT; ++t)
            if (rows.on(t))
#pragma unroll
                for (int q = 0; q < V; ++q) {
                    const int c = rows.ch(t) + q;
                    const float bg = p.h0 != nullptr ? __ldg(p.h0 + th.b * p.hb + c) : 0.f;
                    last[th.b * p.C + c] = past(reach, bg, acc[t][q]);
                }
}

template <class VT, class GT, int V, int NT>
__global__ void __launch_bounds__(kRayBlock)
row_back_kernel(ScanArgs p, const float* __restrict__ kept, const float* __restrict__ d_last,
                VT* __restrict__ dx, GT* __restrict__ dg, float* __restrict__ dh0) {
    clear_uncovered(p, p.C, dx);
    clear_uncovered(p, 1, dg);
    RayThread<VT, GT, 1, 32> th;
    RayRows<VT, GT, V, NT> rows;
    th.init(p);
    rows.init(p);
    if (!th.there) return;
    float d[NT][V], bg = 0.f;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int q = 0; q < V; ++q) {
            const int c = rows.ch(t) + q;
            d[t][q] = d_last != nullptr && rows.on(t) ? __ldg(d_last + th.b * p.C + c) : 0.f;
            if (p.h0 != nullptr && rows.on(t))
                bg = fmaf(d[t][q], __ldg(p.h0 + th.b * p.hb + c), bg);
        }
    for (int o = 1; o < rows.width; o *= 2) bg += __shfl_xor_sync(~0u, bg, o);
    const float* const keep = kept + th.kept_at(p);
    float T_end = 1.f, behind = 0.f;
    for (int k = th.chunks - 1; k >= 0; --k) {
        const int left = th.len - 32 * k;
        const bool in = th.lane < left;
        const float reach = keep[k];
        const float gi = in ? to_float(th.g[(int64_t)k * 32 * p.gs]) : 0.f;
        const int n = left < 32 ? (left + rows.per - 1) / rows.per : rows.width;
        const VT* const x = th.x + ((int64_t)k * 32 + rows.sub - th.lane) * p.xs;
        // d . x of each sample, to its lane
        float c = 0.f;
#pragma unroll 4
        for (int j = 0; j < n; ++j) {
            const int s = j * rows.per + rows.sub;
            float part = 0.f;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                float xv[V];
#pragma unroll
                for (int q = 0; q < V; ++q) xv[q] = 0.f;
                if (s < left && rows.on(t))
                    load_some<V>(x + (int64_t)(j * rows.per) * p.xs + rows.ch(t), xv);
#pragma unroll
                for (int q = 0; q < V; ++q) part = fmaf(d[t][q], xv[q], part);
            }
            for (int o = 1; o < rows.width; o *= 2) part += __shfl_xor_sync(~0u, part, o);
            part = __shfl_sync(~0u, part, (th.lane & (rows.per - 1)) * rows.width);
            if (th.lane / rows.per == j) c = part;
        }
        Gate gates[1] = {gate_of(gi)};
        bool careful;
        const float v = reach_beyond<32>(th.lane, reach, gates, careful);
        const Gate gate = gates[0];
        float T = __shfl_up_sync(~0u, v, 1);
        if (th.lane == 0) T = reach;
        if (k == th.chunks - 1) {
            T_end = __shfl_sync(~0u, v, 31);
            behind = past(T_end, bg, 0.f);
        }
        const float Tn = T * gate.a;
        const float w = p.weighted ? (in ? 1.f : 0.f) : gate.w, W = T * w;
        const float here = th.from(times(W, c)) + behind;
        float rest = __shfl_down_sync(~0u, here, 1);
        if (th.lane == 31) rest = behind;
        behind = __shfl_sync(~0u, here, 0);
        if (dg != nullptr && in) {
            // (a value that is not finite in a place of no thickness is no sample)
            const float own = p.weighted || Tn == 0.f ? 0.f : Tn * c;
            dg[th.first + (int64_t)k * 32 + th.lane] =
                from_float<GT>(w == 0.f && !finite(c) ? 0.f : own - rest);
        }
        if (dx != nullptr) {
            VT* const to = dx + (th.first + (int64_t)k * 32 + rows.sub) * p.C;
#pragma unroll 4
            for (int j = 0; j < n; ++j) {
                const int s = j * rows.per + rows.sub;
                const float Ws = __shfl_sync(~0u, W, s);
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    float out[V];
#pragma unroll
                    for (int q = 0; q < V; ++q) out[q] = Ws * d[t][q];
                    if (s >= left || !rows.on(t)) continue;
                    VT* const row = to + (int64_t)(j * rows.per) * p.C + rows.ch(t);
                    if (p.paired) store_some<V>(row, out);
                    else
#pragma unroll
                        for (int q = 0; q < V; ++q) row[q] = from_float<VT>(out[q]);
                }
            }
        }
    }
    if (dh0 != nullptr && rows.sub == 0)
#pragma unroll
        for (int t = 0; t < NT; ++t)
            if (rows.on(t))
#pragma unroll
                for (int q = 0; q < V; ++q)
                    dh0[th.b * p.C + rows.ch(t) + q] = past(T_end, d[t][q], 0.f);
}

}  // namespace svoxb
