// The gated linear recurrence along a sequence of samples, and its backward pass.
//
//   h[t] = a[t] h[t-1] + w[t] x[t],   a = exp(-g),  w = 1 - a  (w = 1 for weighted inputs)
//
// with one g >= 0 (the thickness of a sample) for each group of D neighbouring channels.  Front
// to back along a ray that is emission and absorption; run from the far end, its last state is
// the colour that is seen.  Two neighbouring stretches of steps combine as
//   (A, B) then (A', B')  ->  (A' A, A' B + B')
// so a stretch is scanned from registers: every thread takes kSteps steps of its channels, the
// warps of a unit take consecutive stretches, and what comes before a stretch is folded from the
// stretches' pairs in shared memory, always in the order of the steps (one result, whatever the
// launch).  The backward pass runs the same from the other end over
//   G[t] = d[t] + a[t+1] G[t+1],   dx = w G,   dg = sum over the group of a (x - h[t-1]) G
// (-a h[t-1] G for weighted inputs) and finds h[t-1] again from x and g and the state at the start
// of each stretch, which the forward kept in 32 bits: 10 instead of 12 bytes per 16-bit element,
// and no rounded state in a gradient.
//
// A sample whose weight is 0 adds nothing whatever its value (0 times NaN included), and nothing
// from before a sample with a = 0 gets past it.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace svoxb {

constexpr int kScanWarps = 8;
constexpr int kScanBlock = 32 * kScanWarps;

struct ScanArgs {
    const void* x;           // (rows, T, C) or (N, C)
    const void* g;           // the same with H in C's place
    const float* h0;         // (rows, C); null: zeros
    const int64_t* offsets;  // packed rows
    int64_t B, T;            // rows; steps of a row, or of all rows together (packed)
    int32_t C, H, D;
    int64_t xb, xs, gb, gs, hb;
    int32_t reverse, weighted;
    // tiles of channels: whole groups, or a part of one
    int32_t tile, tiles, parts;
    int32_t segs;            // warps of a unit, a power of two
    int32_t splits;          // stretches of a row that different blocks take
    int64_t units;           // B * tiles
};

// (of the tile of a unit)
struct ScanTile { int first, width, head; };
__device__ __forceinline__ ScanTile scan_tile(const ScanArgs& p, int t) {
    if (p.parts > 1) {
        const int h = t / p.parts, part = t - h * p.parts;
        const int left = p.D - part * p.tile;
        return {h * p.D + part * p.tile, left < p.tile ? left : p.tile, h};
    }
    const int first = t * p.tile, left = p.C - first;
    return {first, left < p.tile ? left : p.tile, first / p.D};
}

struct ScanRow { int64_t first, len; };      // in steps of all rows
__device__ __forceinline__ ScanRow scan_row(const ScanArgs& p, int64_t b) {
    if (p.offsets == nullptr) return {b * p.T, p.T};
    const int64_t lo = __ldg(p.offsets + b), hi = __ldg(p.offsets + b + 1);
    const int64_t from = lo < 0 ? 0 : lo > p.T ? p.T : lo;
    const int64_t to = hi < from ? from : hi > p.T ? p.T : hi;
    if (from != lo || to != hi) report(SVOXB_ERR_INDEX);
    return {from, to - from};
}

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <class T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}
template <> __device__ __forceinline__ __half from_float<__half>(float v) {
    return __float2half_rn(v);
}

// V neighbouring elements, in one request.
template <class T, int V> struct __align__(sizeof(T) * V) Some { T v[V]; };
template <int V, class T>
__device__ __forceinline__ void load_some(const T* from, float (&to)[V]) {
    const Some<T, V> s = *reinterpret_cast<const Some<T, V>*>(from);
#pragma unroll
    for (int v = 0; v < V; ++v) to[v] = to_float(s.v[v]);
}
template <int V, class T>
__device__ __forceinline__ void store_some(T* to, const float (&from)[V]) {
    Some<T, V> s;
#pragma unroll
    for (int v = 0; v < V; ++v) s.v[v] = from_float<T>(from[v]);
    *reinterpret_cast<Some<T, V>*>(to) = s;
}

// w = 1 - exp(-g): near 0, where the difference would cancel, by its Taylor series (the first term
// left out is below 2^-24 of the sum).
__device__ __forceinline__ float weight_of(float g, float a) {
    const float s = g * (1.f - g * (1.f / 2) * (1.f - g * (1.f / 3) * (1.f - g * (1.f / 4) *
                    (1.f - g * (1.f / 5) * (1.f - g * (1.f / 6))))));
    return fabsf(g) < 0.25f ? s : 1.f - a;
}
__device__ __forceinline__ float times(float w, float x) { return w == 0.f ? 0.f : w * x; }
// a h + b, with nothing of h where a is 0
__device__ __forceinline__ float past(float a, float h, float b) {
    return a == 0.f ? b : fmaf(a, h, b);
}

// The warps of a unit wait for each other (a unit of one warp, for its lanes).
__device__ __forceinline__ void unit_sync(int group, int segs) {
    if (segs == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(segs * 32) : "memory");
}

// Steps of a packed call that no row covers, before the first row and behind the last, get zeros.
template <class T>
__device__ __forceinline__ void clear_uncovered(const ScanArgs& p, int64_t b, const ScanTile& tile,
                                                int64_t row_len, T* out, int thread, int threads) {
    if (p.offsets == nullptr || out == nullptr) return;
    for (int end = 0; end < 2; ++end) {
        if (b != (end ? p.B - 1 : 0)) continue;
        const int64_t at = __ldg(p.offsets + (end ? p.B : 0));
        const int64_t cut = at < 0 ? 0 : at > p.T ? p.T : at;
        const int64_t from = end ? cut : 0, to = end ? p.T : cut;
        for (int64_t i = thread; i < (to - from) * tile.width; i += threads)
            out[(from + i / tile.width) * row_len + tile.first + i % tile.width] =
                from_float<T>(0.f);
    }
}

// Which steps of a row belong to a split: whole stretches of a unit.
__device__ __forceinline__ void split_range(int64_t len, int chunk, int splits, int split,
                                            int64_t* from, int64_t* to) {
    const int64_t chunks = (len + chunk - 1) / chunk;
    const int64_t per = (chunks + splits - 1) / splits;
    const int64_t a = per * split < chunks ? per * split : chunks;
    const int64_t b = per * (split + 1) < chunks ? per * (split + 1) : chunks;
    *from = a;
    *to = b;
}

// Index of the kept state at the start of stretch k of a row.
__device__ __forceinline__ int64_t kept_index(const ScanArgs& p, const ScanRow& row, int64_t b,
                                              int chunk, int64_t k) {
    return p.offsets == nullptr ? b * ((p.T + chunk - 1) / chunk) + k : row.first / chunk + b + k;
}

template <class VT, class GT, int V, bool PC, int L>
struct ScanThread {
    static constexpr int GV = PC ? V : 1;
    int lane, group, seg, split;
    int64_t b;
    ScanTile tile;
    ScanRow row;
    bool on;                 // this lane has channels
    int ch, head;            // its first channel, its group
    const VT* x;
    const GT* g;
    int chunk;

    __device__ __forceinline__ bool init(const ScanArgs& p) {
        lane = threadIdx.x & 31;
        const int warp = threadIdx.x >> 5;
        group = warp / p.segs;
        seg = warp - group * p.segs;
        split = blockIdx.y;
        const int64_t unit = (int64_t)blockIdx.x * (kScanWarps / p.segs) + group;
        if (unit >= p.units) return false;
        b = unit / p.tiles;
        tile = scan_tile(p, (int)(unit - b * p.tiles));
        row = scan_row(p, b);
        on = lane * V < tile.width;
        ch = tile.first + (on ? lane * V : 0);
        head = PC ? ch : ch / p.D;
        const int64_t xo = p.offsets ? row.first * p.xs : b * p.xb;
        const int64_t go = p.offsets ? row.first * p.gs : b * p.gb;
        x = static_cast<const VT*>(p.x) + xo + ch;
        g = static_cast<const GT*>(p.g) + go + head;
        chunk = p.segs * L;
        return true;
    }
    __device__ __forceinline__ int64_t place(const ScanArgs& p, int64_t t) const {
        return p.reverse ? row.len - 1 - t : t;
    }
    __device__ __forceinline__ void gates(const ScanArgs& p, int64_t t0, float (&to)[L][GV]) const {
#pragma unroll
        for (int l = 0; l < L; ++l) {
#pragma unroll
            for (int v = 0; v < GV; ++v) to[l][v] = 0.f;
            if (on && t0 + l < row.len) load_some<GV>(g + place(p, t0 + l) * p.gs, to[l]);
        }
    }
    template <class T>
    __device__ __forceinline__ void rows(const ScanArgs& p, int64_t t0, const T* from,
                                         int64_t step, float (&to)[L][V]) const {
#pragma unroll
        for (int l = 0; l < L; ++l) {
#pragma unroll
            for (int v = 0; v < V; ++v) to[l][v] = 0.f;
            if (on && t0 + l < row.len) load_some<V>(from + place(p, t0 + l) * step, to[l]);
        }
    }
    // state before the row
    __device__ __forceinline__ void start(const ScanArgs& p, float (&h)[V]) const {
#pragma unroll
        for (int v = 0; v < V; ++v)
            h[v] = on && p.h0 != nullptr && ch + v < tile.first + tile.width
                       ? __ldg(p.h0 + b * p.hb + ch + v) : 0.f;
    }
};

// Pairs of whole splits, (B, splits, C): of the forward (A, B), of the backward (A, E) where E is
// what the split's own gradients send back past its first step.
template <class VT, class GT, int V, bool PC, int L, bool BACK>
__global__ void __launch_bounds__(kScanBlock)
scan_pairs_kernel(ScanArgs p, const VT* __restrict__ d, float2* __restrict__ pairs) {
    using Thread = ScanThread<VT, GT, V, PC, L>;
    __shared__ float2 s_pair[kScanWarps][32 * V];
    Thread th;
    if (!th.init(p)) return;
    int64_t k0, k1;
    split_range(th.row.len, th.chunk, p.splits, th.split, &k0, &k1);
    // the warps share the split's steps in consecutive parts of whole L
    const int64_t per = (k1 - k0) * L;      // (k1 - k0 stretches of segs * L steps)
    const int64_t from = k0 * th.chunk + th.seg * per;
    float A[V], B[V];
#pragma unroll
    for (int v = 0; v < V; ++v) { A[v] = 1.f; B[v] = 0.f; }
    for (int64_t i = 0; i < per; i += L) {
        const int64_t t0 = BACK ? from + per - L - i : from + i;
        float g[L][Thread::GV], x[L][V];
        th.gates(p, t0, g);
        if (BACK) {
            if (d != nullptr) th.rows(p, t0, d + th.row.first * p.C + th.ch, p.C, x);
        } else {
            th.rows(p, t0, th.x, p.xs, x);
        }
#pragma unroll
        for (int i2 = 0; i2 < L; ++i2) {
            const int l = BACK ? L - 1 - i2 : i2;
            const bool in = t0 + l < th.row.len;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float gt = g[l][PC ? v : 0];
                const float a = expf(-gt);
                if (BACK) {
                    if (in) B[v] = past(a, B[v] + (d != nullptr ? x[l][v] : 0.f), 0.f);
                } else {
                    const float w = p.weighted ? (in ? 1.f : 0.f) : weight_of(gt, a);
                    B[v] = past(a, B[v], times(w, x[l][v]));
                }
                A[v] *= a;
            }
        }
    }
#pragma unroll
    for (int v = 0; v < V; ++v)
        s_pair[threadIdx.x >> 5][th.lane * V + v] = make_float2(A[v], B[v]);
    unit_sync(th.group, p.segs);
    if (th.seg != 0 || !th.on) return;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        float At = 1.f, Bt = 0.f;
        for (int i = 0; i < p.segs; ++i) {
            const int s = BACK ? p.segs - 1 - i : i;
            const float2 q = s_pair[th.group * p.segs + s][th.lane * V + v];
            Bt = past(q.x, Bt, q.y);
            At *= q.x;
        }
        pairs[(th.b * p.splits + th.split) * p.C + th.ch + v] = make_float2(At, Bt);
    }
}

// The last state from the pairs of all splits.
static __global__ void scan_last_kernel(ScanArgs p, const float2* __restrict__ pairs,
                                        float* __restrict__ last) {
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= p.B * p.C) return;
    const int64_t b = i / p.C, c = i - b * p.C;
    float h = p.h0 != nullptr ? __ldg(p.h0 + b * p.hb + c) : 0.f;
    for (int s = 0; s < p.splits; ++s) {
        const float2 q = pairs[(b * p.splits + s) * p.C + c];
        h = past(q.x, h, q.y);
    }
    last[i] = h;
}

// states: null, or (steps, C); kept: null, or the state at the start of every stretch.
template <class VT, class GT, int V, bool PC, int L>
__global__ void __launch_bounds__(kScanBlock)
scan_kernel(ScanArgs p, const float2* __restrict__ pairs, VT* __restrict__ states,
            float* __restrict__ last, float* __restrict__ kept) {
    using Thread = ScanThread<VT, GT, V, PC, L>;
    __shared__ float2 s_pair[2][kScanWarps][32 * V];
    Thread th;
    if (!th.init(p)) return;
    int64_t k0, k1;
    split_range(th.row.len, th.chunk, p.splits, th.split, &k0, &k1);
    float carry[V];
    th.start(p, carry);
    if (th.split > 0 && th.on) {
        for (int s = 0; s < th.split; ++s)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float2 q = pairs[(th.b * p.splits + s) * p.C + th.ch + v];
                carry[v] = past(q.x, carry[v], q.y);
            }
    }
    VT* out = states == nullptr ? nullptr : states + th.row.first * p.C + th.ch;
    int buf = 0;
    for (int64_t k = k0; k < k1; ++k, buf ^= 1) {
        const int64_t t0 = k * th.chunk + th.seg * L;
        float a[L][V], u[L][V];
        {
            float g[L][Thread::GV];
            th.gates(p, t0, g);
            th.rows(p, t0, th.x, p.xs, u);
#pragma unroll
            for (int l = 0; l < L; ++l) {
                const bool in = t0 + l < th.row.len;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const float gt = g[l][PC ? v : 0];
                    a[l][v] = expf(-gt);
                    const float w = p.weighted ? (in ? 1.f : 0.f) : weight_of(gt, a[l][v]);
                    u[l][v] = times(w, u[l][v]);
                }
            }
        }
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float A = 1.f, B = 0.f;
#pragma unroll
            for (int l = 0; l < L; ++l) {
                A *= a[l][v];
                B = past(a[l][v], B, u[l][v]);
            }
            s_pair[buf][threadIdx.x >> 5][th.lane * V + v] = make_float2(A, B);
        }
        unit_sync(th.group, p.segs);
        float h[V];
        if (kept != nullptr && th.seg == 0 && th.on) {
            float* to = kept + kept_index(p, th.row, th.b, th.chunk, k) * p.C + th.ch;
#pragma unroll
            for (int v = 0; v < V; ++v) to[v] = carry[v];
        }
        for (int s = 0; s < p.segs; ++s)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                if (s == th.seg) h[v] = carry[v];
                const float2 q = s_pair[buf][th.group * p.segs + s][th.lane * V + v];
                carry[v] = past(q.x, carry[v], q.y);
            }
        if (out != nullptr) {
#pragma unroll
            for (int l = 0; l < L; ++l) {
#pragma unroll
                for (int v = 0; v < V; ++v) h[v] = past(a[l][v], h[v], u[l][v]);
                if (th.on && t0 + l < th.row.len)
                    store_some<V>(out + th.place(p, t0 + l) * p.C, h);
            }
        }
    }
    if (th.split == p.splits - 1 && th.seg == 0 && th.on)
#pragma unroll
        for (int v = 0; v < V; ++v) last[th.b * p.C + th.ch + v] = carry[v];
    if (th.split == 0)
        clear_uncovered(p, th.b, th.tile, (int64_t)p.C, states, th.seg * 32 + th.lane, p.segs * 32);
}

// dg of a group that several tiles share goes to `parted` (parts, steps, H) floats.
template <class VT, class GT, int V, bool PC, int L>
__global__ void __launch_bounds__(kScanBlock)
scan_back_kernel(ScanArgs p, const float2* __restrict__ pairs, const float* __restrict__ kept,
                 const VT* __restrict__ d, const float* __restrict__ d_last, VT* __restrict__ dx,
                 GT* __restrict__ dg, float* __restrict__ parted, float* __restrict__ dh0) {
    using Thread = ScanThread<VT, GT, V, PC, L>;
    __shared__ float s_pair[2][kScanWarps][3][32 * V];
    __shared__ float s_sum[PC ? 1 : kScanWarps][PC ? 1 : L][PC ? 1 : 33];
    Thread th;
    if (!th.init(p)) return;
    const int warp = threadIdx.x >> 5;
    int64_t k0, k1;
    split_range(th.row.len, th.chunk, p.splits, th.split, &k0, &k1);
    float R[V];         // what flows back into the last state of the stretch
#pragma unroll
    for (int v = 0; v < V; ++v)
        R[v] = th.on && d_last != nullptr ? __ldg(d_last + th.b * p.C + th.ch + v) : 0.f;
    if (th.on)
        for (int s = p.splits - 1; s > th.split; --s)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float2 q = pairs[(th.b * p.splits + s) * p.C + th.ch + v];
                R[v] = past(q.x, R[v], q.y);
            }
    int buf = 0;
    for (int64_t k = k1 - 1; k >= k0; --k, buf ^= 1) {
        const int64_t t0 = k * th.chunk + th.seg * L;
        float g[L][Thread::GV], a[L][V], x[L][V], e[L][V], h[V];
        th.gates(p, t0, g);
        th.rows(p, t0, th.x, p.xs, x);
        if (d != nullptr)
            th.rows(p, t0, d + th.row.first * p.C + th.ch, p.C, e);
        else
#pragma unroll
            for (int l = 0; l < L; ++l)
#pragma unroll
                for (int v = 0; v < V; ++v) e[l][v] = 0.f;
        {
            const float* from = kept + kept_index(p, th.row, th.b, th.chunk, k) * p.C + th.ch;
#pragma unroll
            for (int v = 0; v < V; ++v) h[v] = th.on ? from[v] : 0.f;
        }
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float A = 1.f, B = 0.f, E = 0.f;
#pragma unroll
            for (int l = 0; l < L; ++l) {
                const float gt = g[l][PC ? v : 0];
                a[l][v] = expf(-gt);
                const bool in = t0 + l < th.row.len;
                const float w = p.weighted ? (in ? 1.f : 0.f) : weight_of(gt, a[l][v]);
                A *= a[l][v];
                B = past(a[l][v], B, times(w, x[l][v]));
            }
#pragma unroll
            for (int l = L - 1; l >= 0; --l) E = past(a[l][v], E + e[l][v], 0.f);
            s_pair[buf][warp][0][th.lane * V + v] = A;
            s_pair[buf][warp][1][th.lane * V + v] = B;
            s_pair[buf][warp][2][th.lane * V + v] = E;
        }
        unit_sync(th.group, p.segs);
        float G[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int at = th.lane * V + v;
            for (int s = 0; s < th.seg; ++s) {
                const auto& q = s_pair[buf][th.group * p.segs + s];
                h[v] = past(q[0][at], h[v], q[1][at]);
            }
            for (int s = p.segs - 1; s >= 0; --s) {
                if (s == th.seg) G[v] = R[v];
                const auto& q = s_pair[buf][th.group * p.segs + s];
                R[v] = past(q[0][at], R[v], q[2][at]);
            }
        }
        // the states before each step, in x's place: what dg needs of both
        float q[L][V];
#pragma unroll
        for (int l = 0; l < L; ++l)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float gt = g[l][PC ? v : 0];
                const bool in = t0 + l < th.row.len;
                const float w = p.weighted ? (in ? 1.f : 0.f) : weight_of(gt, a[l][v]);
                const float u = times(w, x[l][v]);
                // (a value that is not finite in a place of no thickness is no sample)
                const float xv = w == 0.f && !isfinite(x[l][v]) ? h[v] : x[l][v];
                q[l][v] = a[l][v] == 0.f ? 0.f : a[l][v] * (p.weighted ? -h[v] : xv - h[v]);
                x[l][v] = w;
                h[v] = past(a[l][v], h[v], u);
            }
#pragma unroll
        for (int l = L - 1; l >= 0; --l) {
            const bool in = th.on && t0 + l < th.row.len;
            float sum = 0.f, dxv[V], dgv[Thread::GV];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                G[v] += e[l][v];
                dxv[v] = x[l][v] * G[v];
                const float one = q[l][v] * G[v];
                if (PC) dgv[PC ? v : 0] = one;
                else sum += one;
                G[v] = past(a[l][v], G[v], 0.f);
            }
            const int64_t at = th.row.first + th.place(p, t0 + l);
            if (in && dx != nullptr) store_some<V>(dx + at * p.C + th.ch, dxv);
            if (PC) {
                if (in && dg != nullptr) store_some<Thread::GV>(dg + at * p.H + th.head, dgv);
            } else {
                s_sum[PC ? 0 : warp][PC ? 0 : l][PC ? 0 : th.lane] = th.on ? sum : 0.f;
            }
        }
        if (!PC && dg != nullptr) {
            __syncwarp();
            const int groups = p.parts > 1 ? 1 : th.tile.width / p.D;
            const int lanes = p.parts > 1 ? 32 : p.D / V;
            for (int i = th.lane; i < L * groups; i += 32) {
                const int l = i / groups, j = i - l * groups;
                float sum = 0.f;
                for (int c = 0; c < lanes; ++c)
                    sum += s_sum[PC ? 0 : warp][PC ? 0 : l][PC ? 0 : j * lanes + c];
                if (t0 + l < th.row.len) {
                    const int64_t at = th.row.first + th.place(p, t0 + l);
                    if (p.parts > 1) {
                        const int part = (th.tile.first - th.tile.head * p.D) / p.tile;
                        const int64_t steps = p.offsets ? p.T : p.B * p.T;
                        parted[(part * steps + at) * p.H + th.tile.head] = sum;
                    } else {
                        dg[at * p.H + th.tile.head + j] = from_float<GT>(sum);
                    }
                }
            }
            __syncwarp();
        }
    }
    if (th.split == 0) {
        if (th.seg == 0 && th.on && dh0 != nullptr)
#pragma unroll
            for (int v = 0; v < V; ++v) dh0[th.b * p.C + th.ch + v] = R[v];
        clear_uncovered(p, th.b, th.tile, (int64_t)p.C, dx, th.seg * 32 + th.lane, p.segs * 32);
        ScanTile heads = th.tile;
        heads.first = PC ? th.tile.first : th.tile.head;
        heads.width = PC ? th.tile.width : p.parts > 1 ? 1 : th.tile.width / p.D;
        if (p.parts == 1 || th.tile.first == th.tile.head * p.D)
            clear_uncovered(p, th.b, heads, (int64_t)p.H, dg, th.seg * 32 + th.lane, p.segs * 32);
    }
}

// dg from the sums of the parts of each group.
template <class GT>
__global__ void scan_parts_kernel(ScanArgs p, const float* __restrict__ parted,
                                  GT* __restrict__ dg) {
    const int64_t n = (p.offsets ? p.T : p.B * p.T) * p.H;
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= n) return;
    if (p.offsets != nullptr) {
        // (the steps of no row have no sums: they have been cleared)
        const int64_t step = i / p.H;
        if (step < __ldg(p.offsets) || step >= __ldg(p.offsets + p.B)) return;
    }
    float sum = 0.f;
    for (int part = 0; part < p.parts; ++part) sum += parted[part * n + i];
    dg[i] = from_float<GT>(sum);
}

}  // namespace svoxb
