// Compositing of samples with few channels that share their thickness: the colours of rays.
//
// The last state of the recurrence (recurrence.cuh), back to front, is a sum from the front,
//   out = sum of T[i] w[i] x[i] + T[n] background,   T[i] = exp(-(g[0] + ... + g[i-1]))
// so a group of G lanes walks a ray from the front, a sample to a lane, and scans nothing but the
// thickness; the channels are summed in each lane and over the lanes at the end.  The gradient needs
// the state behind each sample only in its product with the upstream gradient d,
//   D[i] = d . h[i] = a[i] D[i+1] + w[i] (d . x[i]),   dg[i] = T[i+1] (d . x[i] - D[i+1])
// one scan of pairs whatever the number of channels, from the far end, and dx[i] = T[i] w[i] d.  The
// forward keeps the thickness in front of every G samples for it.
//
// In the tiles of recurrence.cuh, whose lanes are channels first, 2^20 rays of 42 samples of 3
// channels took 5.19 ms, and 9.25 ms backwards.
#pragma once

#include "recurrence.cuh"

namespace svoxb {

constexpr int kRayBlock = 256;
constexpr int kRayChannels = 4;     // at most

template <class VT, class GT, int C, int G>
struct RayThread {
    int lane;                       // in the group
    int64_t b;
    bool there;
    ScanRow row;
    const VT* x;
    const GT* g;
    int64_t chunks, most;           // of G samples: of this ray, of the warp's longest

    __device__ __forceinline__ void init(const ScanArgs& p) {
        lane = threadIdx.x % G;
        b = ((int64_t)blockIdx.x * kRayBlock + threadIdx.x) / G;
        there = b < p.B;
        if (!there) b = p.B - 1;
        row = scan_row(p, b);
        x = static_cast<const VT*>(p.x) + (p.offsets ? row.first * p.xs : b * p.xb);
        g = static_cast<const GT*>(p.g) + (p.offsets ? row.first * p.gs : b * p.gb);
        chunks = there ? (row.len + G - 1) / G : 0;
        most = chunks;
        if (G < 32)
#pragma unroll
            for (int d = G; d < 32; d *= 2) {
                const int64_t o = __shfl_xor_sync(~0u, most, d);
                most = o > most ? o : most;
            }
    }
    __device__ __forceinline__ int64_t kept_at(const ScanArgs& p) const {
        return p.offsets ? row.first / G + b : b * ((p.T + G - 1) / G);
    }
    // Thickness in front of this lane's sample within the chunk; `all`: of the chunk.
    __device__ __forceinline__ float before(float gi, float* all) const {
        float v = gi;
#pragma unroll
        for (int d = 1; d < G; d *= 2) {
            const float o = __shfl_up_sync(~0u, v, d, G);
            if (lane >= d) v += o;
        }
        *all = __shfl_sync(~0u, v, G - 1, G);
        const float o = __shfl_up_sync(~0u, v, 1, G);
        return lane > 0 ? o : 0.f;
    }
};

template <class VT, class GT, int C, int G>
__global__ void __launch_bounds__(kRayBlock)
ray_kernel(ScanArgs p, float* __restrict__ last, float* __restrict__ kept) {
    RayThread<VT, GT, C, G> th;
    th.init(p);
    float S = 0.f, acc[C];
#pragma unroll
    for (int c = 0; c < C; ++c) acc[c] = 0.f;
    const VT* x = th.x + th.lane * p.xs;
    const GT* g = th.g + th.lane * p.gs;
    float* const keep = kept != nullptr && th.lane == 0 ? kept + th.kept_at(p) : nullptr;
    for (int64_t k = 0; k < th.most; ++k, x += G * p.xs, g += G * p.gs) {
        const bool in = k < th.chunks && k * G + th.lane < th.row.len;
        float xv[C];
        const float gi = in ? to_float(*g) : 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c) xv[c] = in ? to_float(x[c]) : 0.f;
        if (keep != nullptr && k < th.chunks) keep[k] = S;
        float all;
        const float T = decay_of(S + th.before(gi, &all));
        const float W = p.weighted ? T : T * weight_of(gi, decay_of(gi));
        if (W != 0.f)
#pragma unroll
            for (int c = 0; c < C; ++c) acc[c] = fmaf(W, xv[c], acc[c]);
        S += all;
    }
#pragma unroll
    for (int d = G / 2; d > 0; d /= 2)
#pragma unroll
        for (int c = 0; c < C; ++c) acc[c] += __shfl_xor_sync(~0u, acc[c], d);
    if (!th.there) return;
    const float T = decay_of(S);
#pragma unroll
    for (int c = 0; c < C; ++c)
        if (th.lane == c) {
            const float bg = p.h0 != nullptr ? __ldg(p.h0 + th.b * p.hb + c) : 0.f;
            last[th.b * C + c] = past(T, bg, acc[c]);
        }
}

template <class VT, class GT, int C, int G>
__global__ void __launch_bounds__(kRayBlock)
ray_back_kernel(ScanArgs p, const float* __restrict__ kept, const float* __restrict__ d_last,
                VT* __restrict__ dx, GT* __restrict__ dg, float* __restrict__ dh0) {
    RayThread<VT, GT, C, G> th;
    th.init(p);
    float d[C], D = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        d[c] = d_last != nullptr ? __ldg(d_last + th.b * C + c) : 0.f;
        if (p.h0 != nullptr) D = fmaf(d[c], __ldg(p.h0 + th.b * p.hb + c), D);
    }
    // The values' gradients leave as one stretch: in its j-th store a lane has element j * G + lane,
    // of sample `from[j]` and channel `ch`.
    int from[C];
    float scale[C];
#pragma unroll
    for (int j = 0; j < C; ++j) {
        const int e = j * G + th.lane;
        from[j] = e / C;
#pragma unroll
        for (int c = 0; c < C; ++c)
            if (e % C == c) scale[j] = d[c];
    }
    const float* const keep = kept + th.kept_at(p);
    float end = 0.f;                // thickness of the whole ray
    float S_next = th.most > 0 && th.most <= th.chunks ? keep[th.most - 1] : 0.f;
    for (int64_t k = th.most - 1; k >= 0; --k) {
        const int64_t i = k * G + th.lane;
        const bool in = k < th.chunks && i < th.row.len;
        const float gi = in ? to_float(th.g[i * p.gs]) : 0.f;
        float xv[C], c = 0.f;
#pragma unroll
        for (int q = 0; q < C; ++q) xv[q] = in ? to_float(th.x[i * p.xs + q]) : 0.f;
#pragma unroll
        for (int q = 0; q < C; ++q) c = fmaf(d[q], xv[q], c);
        const float S = S_next;
        S_next = k > 0 && k <= th.chunks ? keep[k - 1] : 0.f;
        float all;
        const float T = decay_of(S + th.before(gi, &all));
        if (k == th.chunks - 1) end = S + all;
        const float a = decay_of(gi), w = p.weighted ? (in ? 1.f : 0.f) : weight_of(gi, a);
        // D at every sample of the chunk, from its end
        float A = a, B = times(w, c);
#pragma unroll
        for (int s = 1; s < G; s *= 2) {
            const float oa = __shfl_down_sync(~0u, A, s, G), ob = __shfl_down_sync(~0u, B, s, G);
            if (th.lane + s < G) {
                B = past(A, ob, B);
                A *= oa;
            }
        }
        const float mine = past(A, D, B);
        float behind = __shfl_down_sync(~0u, mine, 1, G);
        if (th.lane == G - 1) behind = D;
        D = __shfl_sync(~0u, mine, 0, G);
        const float Tn = T * a, W = T * w;
        // (a value that is not finite in a place of no thickness is no sample)
        const float own = p.weighted ? 0.f : w == 0.f && !finite(c) ? behind : c;
        if (in && dg != nullptr)
            dg[th.row.first + i] = from_float<GT>(Tn == 0.f ? 0.f : Tn * (own - behind));
        if (dx != nullptr) {
            const int64_t left = (th.row.len - k * G) * C;      // elements of this and later chunks
#pragma unroll
            for (int j = 0; j < C; ++j) {
                const float Wj = __shfl_sync(~0u, W, from[j], G);
                if (k < th.chunks && j * G + th.lane < left)
                    dx[(th.row.first + k * G) * C + j * G + th.lane] = from_float<VT>(Wj * scale[j]);
            }
        }
    }
    if (!th.there) return;
    if (dh0 != nullptr)
#pragma unroll
        for (int c = 0; c < C; ++c)
            if (th.lane == c) dh0[th.b * C + c] = past(decay_of(end), d[c], 0.f);
    clear_uncovered(p, th.b, 0, C, (int64_t)C, dx, th.lane, G);
    clear_uncovered(p, th.b, 0, 1, (int64_t)1, dg, th.lane, G);
}

}  // namespace svoxb
