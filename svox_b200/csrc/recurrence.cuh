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

#include <type_traits>

#include "common.cuh"

namespace svoxb {

constexpr int kScanWarps = 8;
constexpr int kScanBlock = 32 * kScanWarps;
constexpr int kScanStages = 3;      // tiles of a warp that are under way at most

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
    int32_t lanes;           // lanes of a row of channels, a power of two (the others: later steps)
    int32_t warps;           // of a unit, a power of two
    int32_t splits;          // ranges of a row that different blocks take
    int32_t stages;          // tiles a warp has under way
    int32_t x_bytes, g_bytes, d_bytes;   // how much of a row is copied at once: 16, 4 or 2 bytes
    int32_t paired;          // rows of the outputs lie on boundaries of two elements
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

__device__ __forceinline__ bool finite(float v) { return fabsf(v) <= 3.402823466e38f; }

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

// a = exp(-g) by the hardware's power of two: 2 ulp of its own and g * 2^-24 from the product, an
// error that a itself outweighs (g exp(-g) < 0.4).
__device__ __forceinline__ float decay_of(float g) {
    float a;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(a) : "f"(g * -1.4426950408889634f));
    return a;
}
// w = 1 - exp(-g): near 0, where the difference would cancel, by its Taylor series (the first term
// left out is below 2^-24 of the sum).
__device__ __forceinline__ float weight_of(float g, float a) {
    const float s = g * fmaf(g, fmaf(g, fmaf(g, fmaf(g, fmaf(g, -1.f / 720, 1.f / 120), -1.f / 24),
                                            1.f / 6), -0.5f), 1.f);
    return fabsf(g) < 0.25f ? s : 1.f - a;
}
__device__ __forceinline__ float times(float w, float x) { return w == 0.f ? 0.f : w * x; }
// a h + b, with nothing of h where a is 0
__device__ __forceinline__ float past(float a, float h, float b) {
    return a == 0.f ? b : fmaf(a, h, b);
}

// Steps of a packed call that no row covers, before the first row and behind the last, get zeros.
template <class T>
__device__ __forceinline__ void clear_uncovered(const ScanArgs& p, int64_t b, int first, int width,
                                                int64_t row_len, T* out, int thread, int threads) {
    if (p.offsets == nullptr || out == nullptr) return;
    for (int end = 0; end < 2; ++end) {
        if (b != (end ? p.B - 1 : 0)) continue;
        const int64_t at = __ldg(p.offsets + (end ? p.B : 0));
        const int64_t cut = at < 0 ? 0 : at > p.T ? p.T : at;
        const int64_t from = end ? cut : 0, to = end ? p.T : cut;
        for (int64_t i = thread; i < (to - from) * width; i += threads)
            out[(from + i / width) * row_len + first + i % width] = from_float<T>(0.f);
    }
}

// Index of the kept state at the start of stretch k of a row.
__device__ __forceinline__ int64_t kept_index(const ScanArgs& p, const ScanRow& row, int64_t b,
                                              int chunk, int64_t k) {
    return p.offsets == nullptr ? b * ((p.T + chunk - 1) / chunk) + k : row.first / chunk + b + k;
}

// ---------------------------------------------------------------------------
// Tiles.  A unit (a row's tile of up to `lanes` * V channels) is scanned by `warps` warps; of a warp,
// each group of `lanes` lanes takes L steps, so that a tile has warps * (32 / lanes) * L steps.  Each
// warp copies its own part of the tiles to shared memory, asynchronously and up to kScanStages ahead:
// row l holds what the lanes need for their l-th step, whatever the width of a channel row.
template <class VT, class GT, bool PC>
struct ScanShape {
    static constexpr int V = sizeof(VT) == 2 ? 2 : 1;      // channels of a lane
    static constexpr int L = 16 / V;                       // steps of a lane
    static constexpr int GV = PC ? V : 1;
    static constexpr int kX = L * 32 * V * sizeof(VT);     // bytes of a warp's tile of values,
    static constexpr int kG = L * 32 * GV * sizeof(GT);    // of gates
    static constexpr int kSum = L * (32 * V + 1) * 4;      // of a warp's products for dg
};

__device__ __forceinline__ void copy_async(void* to, const void* from, int bytes, bool in) {
    const unsigned a = (unsigned)__cvta_generic_to_shared(to);
    const int n = in ? bytes : 0;           // (the rest is filled with zeros)
    if (bytes == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(a), "l"(from), "r"(n)
                     : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(a), "l"(from), "r"(n)
                     : "memory");
}
__device__ __forceinline__ void copies_issued() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Waits until at most `younger` groups of copies are under way.
__device__ __forceinline__ void copies_wait(int younger) {
    if (younger == 2) asm volatile("cp.async.wait_group 2;" ::: "memory");
    else if (younger == 1) asm volatile("cp.async.wait_group 1;" ::: "memory");
    else asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// A thread's place: its unit, its steps within a tile, its channels.
template <class VT, class GT, bool PC>
struct ScanThread {
    using S = ScanShape<VT, GT, PC>;
    int lane, warp, group, wseg;    // wseg: the warp's number in its unit
    int sub, cl, chunk;
    int64_t b;
    ScanTile tile;
    ScanRow row;
    int have;                // channels of this lane
    bool on;                 // it has some
    int ch;                  // its first channel
    int gate;                // where its gate is in a row of a shared tile of gates
    int split;
    int64_t k0, k1;          // tiles of this block's range

    __device__ __forceinline__ bool init(const ScanArgs& p) {
        lane = threadIdx.x & 31;
        warp = threadIdx.x >> 5;
        group = warp / p.warps;
        wseg = warp - group * p.warps;
        split = blockIdx.y;
        const int64_t unit = (int64_t)blockIdx.x * (kScanWarps / p.warps) + group;
        if (unit >= p.units) return false;
        b = unit / p.tiles;
        tile = scan_tile(p, (int)(unit - b * p.tiles));
        row = scan_row(p, b);
        sub = lane / p.lanes;
        cl = lane - sub * p.lanes;
        have = tile.width - cl * S::V;
        have = have < 0 ? 0 : have < S::V ? have : S::V;
        on = have > 0;
        ch = tile.first + (on ? cl * S::V : 0);
        const int heads = p.parts > 1 ? 1 : p.D > 1 ? tile.width / p.D : 0;
        gate = PC ? 0 : sub * heads + (p.parts > 1 ? 0 : on ? cl * S::V / p.D : 0);
        chunk = p.warps * (32 / p.lanes) * S::L;
        const int64_t chunks = (row.len + chunk - 1) / chunk;
        const int64_t per = (chunks + p.splits - 1) / p.splits;
        k0 = per * split < chunks ? per * split : chunks;
        k1 = per * (split + 1) < chunks ? per * (split + 1) : chunks;
        return true;
    }
    __device__ __forceinline__ int64_t first_step(const ScanArgs& p, int64_t k, int s) const {
        return k * chunk + (wseg * (32 / p.lanes) + s) * S::L;
    }
    __device__ __forceinline__ int64_t place(const ScanArgs& p, int64_t t) const {
        return p.reverse ? row.len - 1 - t : t;
    }
    // The warp's part of tile k of an array, BYTES at a time.  A lane's pieces lie in one column,
    // so many rows apart.
    template <class T, int W, int BYTES>
    __device__ __forceinline__ void copy_pieces(const ScanArgs& p, int64_t k, T* to, const T* from,
                                                int64_t step) const {
        constexpr int n = BYTES / (int)sizeof(T);           // elements of a piece
        constexpr int P = 32 * W / n, COLS = P < 32 ? P : 32, ROWS = 32 / COLS;
        const int each = p.lanes * W;                       // elements of a row of channels
#pragma unroll
        for (int half = 0; half < P; half += COLS) {
            const int j = (half + lane % COLS) * n;
            const int s = j >> (31 - __clz(each)), c = j & (each - 1);
            if (c >= tile.width) continue;
            int64_t t = first_step(p, k, s) + lane / COLS;
            const T* src = from + place(p, t) * step + c;
            const int64_t down = (p.reverse ? -ROWS : ROWS) * step;
            T* dst = to + lane / COLS * 32 * W + j;
#pragma unroll
            for (int l = 0; l < S::L; l += ROWS) {
                const bool in = t < row.len;
                if (BYTES >= 4) copy_async(dst, in ? src : from, BYTES, in);
                else *dst = in ? *src : from_float<T>(0.f);
                t += ROWS;
                src += down;
                dst += ROWS * 32 * W;
            }
        }
    }
    template <class T, int W>
    __device__ __forceinline__ void copy_rows(const ScanArgs& p, int64_t k, T* to, const T* from,
                                              int64_t step, int at_once) const {
        if (at_once == 16) copy_pieces<T, W, 16>(p, k, to, from, step);
        else if (at_once == 4) copy_pieces<T, W, 4>(p, k, to, from, step);
        else copy_pieces<T, W, (int)sizeof(T)>(p, k, to, from, step);
    }
    __device__ __forceinline__ void copy_values(const ScanArgs& p, int64_t k, VT* to,
                                                const VT* from, int64_t step, int at_once) const {
        copy_rows<VT, S::V>(p, k, to, from, step, at_once);
    }
    __device__ __forceinline__ void copy_gates(const ScanArgs& p, int64_t k, GT* to) const {
        const GT* from = static_cast<const GT*>(p.g) + (p.offsets ? row.first * p.gs : b * p.gb);
        if (PC && p.D == 1) {
            copy_rows<GT, S::V>(p, k, to, from + tile.first, p.gs, p.g_bytes);
            return;
        }
        // one gate for several channels: once each, or (PC) for every channel of the group
        const int heads = p.parts > 1 ? 1 : tile.width / p.D;
        const int width = PC ? tile.width : heads, subs = 32 / p.lanes;
        const int pitch = PC ? p.lanes * S::V : heads;
        if (!PC && heads * subs == 1) {
            const int64_t t = first_step(p, k, 0) + lane;
            if (lane >= S::L) return;
            const bool in = t < row.len;
            const GT* src = from + (in ? place(p, t) : 0) * p.gs + tile.head;
            if (sizeof(GT) == 4) copy_async(to + lane * 32, src, 4, in);
            else to[lane * 32] = in ? *src : from_float<GT>(0.f);
            return;
        }
        for (int i = lane; i < S::L * subs * width; i += 32) {
            const int l = i / (subs * width), j = i - l * (subs * width);
            const int s = j / width, c = j - s * width;
            const int64_t t = first_step(p, k, s) + l;
            const bool in = t < row.len;
            const GT* src = from + (in ? place(p, t) : 0) * p.gs +
                            (PC ? (tile.first + c) / p.D : tile.head + c);
            GT* dst = to + l * 32 * S::GV + s * pitch + c;
            if (sizeof(GT) == 4) copy_async(dst, src, 4, in);
            else *dst = in ? *src : from_float<GT>(0.f);
        }
    }
    __device__ __forceinline__ void load_gates(const GT* tile_g, int l, float (&g)[S::GV]) const {
        if (PC) load_some<S::GV>(tile_g + (l * 32 + lane) * S::GV, g);
        else g[0] = to_float(tile_g[l * 32 + gate]);
    }
    // state before the row
    __device__ __forceinline__ void start(const ScanArgs& p, float (&h)[S::V]) const {
#pragma unroll
        for (int v = 0; v < S::V; ++v)
            h[v] = p.h0 != nullptr && v < have
                       ? __ldg(p.h0 + b * p.hb + ch + v) : 0.f;
    }
    // V neighbouring elements of an output row, as far as the tile goes
    template <class T, int W>
    __device__ __forceinline__ void put(const ScanArgs& p, T* to, const float (&v)[W]) const {
        if (W == 1 || p.paired) {
            store_some<W>(to, v);
        } else {
#pragma unroll
            for (int i = 0; i < W; ++i)
                if (i < have) to[i] = from_float<T>(v[i]);
        }
    }
    template <class T>
    __device__ __forceinline__ void get(const T* from, float (&v)[S::V]) const {
#pragma unroll
        for (int i = 0; i < S::V; ++i)
            v[i] = i < have ? (float)from[i] : 0.f;
    }
    __device__ __forceinline__ void unit_sync(const ScanArgs& p) const {
        if (p.warps == 1) __syncwarp();
        else asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(p.warps * 32) : "memory");
    }
};

// Pairs of the stretches of a unit's lanes, joined.  In: (A, B) of this lane's L steps.  Out: what
// the steps before it in the tile do to the state (A, B), and the tile's own pair (TA, TB).  BACK:
// the steps behind it, from the other end.
template <int V, bool BACK>
__device__ __forceinline__ void join_lanes(int lanes, int lane, float (&A)[V], float (&B)[V]) {
    for (int d = lanes; d < 32; d *= 2) {
        const bool any = BACK ? lane + d < 32 : lane >= d;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const float a = BACK ? __shfl_down_sync(~0u, A[v], d) : __shfl_up_sync(~0u, A[v], d);
            const float b = BACK ? __shfl_down_sync(~0u, B[v], d) : __shfl_up_sync(~0u, B[v], d);
            if (any) {
                B[v] = past(A[v], b, B[v]);
                A[v] *= a;
            }
        }
    }
}

// MODE 0: states and the last one; 1: the pair (A, B) of the block's range; 2: the pair (A, E) of it
// backwards, where E is what the range's own gradients `x` send back past its first step.
template <class VT, class GT, bool PC, int MODE>
__global__ void __launch_bounds__(kScanBlock, MODE == 0 ? 2 : 3)
scan_kernel(ScanArgs p, const VT* __restrict__ x, float2* __restrict__ pairs,
            VT* __restrict__ states, float* __restrict__ last, float* __restrict__ kept) {
    using Th = ScanThread<VT, GT, PC>;
    using S = typename Th::S;
    constexpr int V = S::V, L = S::L;
    constexpr bool BACK = MODE == 2;
    extern __shared__ __align__(16) unsigned char s_tiles[];
    __shared__ float2 s_pair[2][kScanWarps][32 * V];
    Th th;
    if (!th.init(p)) return;
    const int64_t n = th.k1 - th.k0;
    // (a range backwards has its tiles from the last to the first)
    auto tile_at = [&](int64_t i) { return BACK ? th.k1 - 1 - i : th.k0 + i; };
    unsigned char* const mine = s_tiles + (size_t)th.warp * p.stages * (S::kX + S::kG);
    const VT* const from = x == nullptr ? nullptr
        : x + (p.offsets ? th.row.first * p.xs : th.b * p.xb) + th.tile.first;
    auto issue = [&](int64_t i) {
        if (i < n) {
            unsigned char* at = mine + (int)(i % p.stages) * (S::kX + S::kG);
            if (from != nullptr)
                th.copy_values(p, tile_at(i), reinterpret_cast<VT*>(at), from, p.xs, p.x_bytes);
            th.copy_gates(p, tile_at(i), reinterpret_cast<GT*>(at + S::kX));
        }
        copies_issued();
    };
    float carry[V], through[V];          // MODE 1, 2: the pair so far
#pragma unroll
    for (int v = 0; v < V; ++v) { carry[v] = 0.f; through[v] = 1.f; }
    for (int i = 0; i < p.stages - 1; ++i) issue(i);
    if (MODE == 0) {
        th.start(p, carry);
        if (th.on)
            for (int s = 0; s < th.split; ++s)
#pragma unroll
                for (int v = 0; v < V; ++v)
                    if (v < th.have) {
                        const float2 q = pairs[(th.b * p.splits + s) * p.C + th.ch + v];
                        carry[v] = past(q.x, carry[v], q.y);
                    }
    }
    VT* const out = states == nullptr ? nullptr : states + th.row.first * p.C + th.ch;
    const int64_t out_step = p.reverse ? -(int64_t)p.C : p.C;
    for (int64_t i = 0; i < n; ++i) {
        const int64_t k = tile_at(i), t0 = th.first_step(p, k, th.sub);
        issue(i + p.stages - 1);
        copies_wait(p.stages - 1);
        __syncwarp();
        const unsigned char* at = mine + (int)(i % p.stages) * (S::kX + S::kG);
        const VT* const tx = reinterpret_cast<const VT*>(at);
        const GT* const tg = reinterpret_cast<const GT*>(at + S::kX);
        float a[L][V], u[L][V], A[V], B[V];
        // (a step beyond the row has no thickness and no value: it changes nothing)
        auto scan = [&](auto safe) {
            constexpr bool SAFE = decltype(safe)::value;
#pragma unroll
            for (int v = 0; v < V; ++v) { A[v] = 1.f; B[v] = 0.f; }
#pragma unroll
            for (int j = 0; j < L; ++j) {
                const int l = BACK ? L - 1 - j : j;
                float g[S::GV];
                th.load_gates(tg, l, g);
#pragma unroll
                for (int v = 0; v < V; ++v) u[l][v] = 0.f;
                if (!BACK || from != nullptr) load_some<V>(tx + (l * 32 + th.lane) * V, u[l]);
                float one_a = 0.f, one_w = 0.f;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    if (v < S::GV) {
                        one_a = decay_of(g[v < S::GV ? v : 0]);
                        one_w = p.weighted ? 1.f : weight_of(g[v < S::GV ? v : 0], one_a);
                    }
                    a[l][v] = one_a;
                    if (BACK) {
                        B[v] = SAFE ? past(one_a, B[v] + u[l][v], 0.f) : one_a * (B[v] + u[l][v]);
                    } else {
                        u[l][v] = SAFE ? times(one_w, u[l][v]) : one_w * u[l][v];
                        B[v] = SAFE ? past(one_a, B[v], u[l][v]) : fmaf(one_a, B[v], u[l][v]);
                    }
                    A[v] *= one_a;
                }
            }
        };
        scan(std::false_type{});
        // What is not finite stays so to the end of the stretch; then the steps that do not count
        // are told from those that do.
        bool odd = false;
#pragma unroll
        for (int v = 0; v < V; ++v) odd |= v < th.have && !(finite(B[v]) && finite(A[v]));
        if (odd) scan(std::true_type{});
        float TA[V], TB[V];     // the lane's place in the warp
        join_lanes<V, BACK>(p.lanes, th.lane, A, B);
        const int edge = BACK ? th.cl : 32 - p.lanes + th.cl;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            TA[v] = __shfl_sync(~0u, A[v], edge);
            TB[v] = __shfl_sync(~0u, B[v], edge);
        }
        if (p.lanes < 32) {     // what lies before the lane
            const int by = BACK ? th.lane + p.lanes : th.lane - p.lanes;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float pa = __shfl_sync(~0u, A[v], by & 31);
                const float pb = __shfl_sync(~0u, B[v], by & 31);
                const bool some = BACK ? by < 32 : by >= 0;
                A[v] = some ? pa : 1.f;
                B[v] = some ? pb : 0.f;
            }
        } else {
#pragma unroll
            for (int v = 0; v < V; ++v) { A[v] = 1.f; B[v] = 0.f; }
        }
        if (kept != nullptr && th.wseg == 0 && th.sub == 0 && th.on) {
            float* to = kept + kept_index(p, th.row, th.b, th.chunk, k) * p.C + th.ch;
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (v < th.have) to[v] = carry[v];
        }
        float h[V];
        if (p.warps == 1) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                h[v] = past(A[v], carry[v], B[v]);
                carry[v] = past(TA[v], carry[v], TB[v]);
                through[v] *= TA[v];
            }
        } else {
            auto& pair = s_pair[i & 1];
            if (th.sub == 0)
#pragma unroll
                for (int v = 0; v < V; ++v)
                    pair[th.warp][th.cl * V + v] = make_float2(TA[v], TB[v]);
            th.unit_sync(p);
            for (int j = 0; j < p.warps; ++j) {
                const int w = BACK ? p.warps - 1 - j : j;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    if (w == th.wseg) h[v] = past(A[v], carry[v], B[v]);
                    const float2 q = pair[th.group * p.warps + w][th.cl * V + v];
                    carry[v] = past(q.x, carry[v], q.y);
                    if (MODE != 0) through[v] *= q.x;
                }
            }
        }
        if (MODE == 0 && out != nullptr && th.on) {
            VT* to = out + th.place(p, t0) * p.C;
#pragma unroll
            for (int v = 0; v < V; ++v) odd |= v < th.have && !finite(h[v]);
            if (t0 + L <= th.row.len && !odd) {
#pragma unroll
                for (int l = 0; l < L; ++l, to += out_step) {
#pragma unroll
                    for (int v = 0; v < V; ++v) h[v] = fmaf(a[l][v], h[v], u[l][v]);
                    th.put(p, to, h);
                }
            } else {
#pragma unroll
                for (int l = 0; l < L; ++l, to += out_step) {
#pragma unroll
                    for (int v = 0; v < V; ++v) h[v] = past(a[l][v], h[v], u[l][v]);
                    if (t0 + l < th.row.len) th.put(p, to, h);
                }
            }
        }
        __syncwarp();
    }
    if (th.wseg == 0 && th.sub == 0 && th.on)
#pragma unroll
        for (int v = 0; v < V; ++v) {
            if (v >= th.have) continue;
            if (MODE != 0)
                pairs[(th.b * p.splits + th.split) * p.C + th.ch + v] =
                    make_float2(through[v], carry[v]);
            else if (th.split == p.splits - 1)
                last[th.b * p.C + th.ch + v] = carry[v];
        }
    if (MODE == 0 && th.split == 0)
        clear_uncovered(p, th.b, th.tile.first, th.tile.width, (int64_t)p.C, states,
                        th.wseg * 32 + th.lane, p.warps * 32);
}

// Rows of a few steps (a sequence that goes on one step at a time): a thread for every W channels,
// step by step.  In tiles the step of 64 rows of 1024 channels took 4.3 us.
constexpr int kFewSteps = 8;
template <class VT, class GT, int W>
__global__ void __launch_bounds__(128)
scan_few_kernel(ScanArgs p, VT* __restrict__ states, float* __restrict__ last,
                float* __restrict__ kept) {
    const int64_t i = (int64_t)blockIdx.x * 128 + threadIdx.x;
    const int per = p.C / W;
    if (i >= p.B * per) return;
    const int64_t b = i / per;
    const int c = (int)(i - b * per) * W;
    const VT* const x = static_cast<const VT*>(p.x) + b * p.xb + c;
    const GT* const g = static_cast<const GT*>(p.g) + b * p.gb;
    float h[W];
#pragma unroll
    for (int v = 0; v < W; ++v) {
        h[v] = p.h0 != nullptr ? __ldg(p.h0 + b * p.hb + c + v) : 0.f;
        if (kept != nullptr && p.T > 0) kept[b * p.C + c + v] = h[v];
    }
    for (int t = 0; t < (int)p.T; ++t) {
        const int64_t at = p.reverse ? p.T - 1 - t : t;
        float xv[W];
        load_some<W>(x + at * p.xs, xv);
#pragma unroll
        for (int v = 0; v < W; ++v) {
            const float gv = to_float(g[at * p.gs + (c + v) / p.D]);
            const float a = decay_of(gv);
            h[v] = past(a, h[v], times(p.weighted ? 1.f : weight_of(gv, a), xv[v]));
        }
        if (states != nullptr) store_some<W>(states + (b * p.T + at) * p.C + c, h);
    }
#pragma unroll
    for (int v = 0; v < W; ++v) last[b * p.C + c + v] = h[v];
}

// The last state from the pairs of all ranges.
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

// The backward pass of a tile.  `parted`: (parts, steps, H) floats for the sums of a group that
// several tiles share.
template <class VT, class GT, bool PC>
__global__ void __launch_bounds__(kScanBlock, 2)
scan_back_kernel(ScanArgs p, const VT* __restrict__ x, const float2* __restrict__ pairs,
                 const float* __restrict__ kept, const VT* __restrict__ d,
                 const float* __restrict__ d_last, VT* __restrict__ dx, GT* __restrict__ dg,
                 float* __restrict__ parted, float* __restrict__ dh0) {
    using Th = ScanThread<VT, GT, PC>;
    using S = typename Th::S;
    constexpr int V = S::V, L = S::L;
    extern __shared__ __align__(16) unsigned char s_tiles[];
    __shared__ float s_pair[2][kScanWarps][3][32 * V];
    Th th;
    if (!th.init(p)) return;
    const int64_t n = th.k1 - th.k0;
    const int stage = 2 * S::kX + S::kG;
    unsigned char* const mine = s_tiles + (size_t)th.warp * p.stages * stage;
    float* const sums = reinterpret_cast<float*>(s_tiles + (size_t)kScanWarps * p.stages * stage +
                                                 th.warp * S::kSum);
    const VT* const from_x = x + (p.offsets ? th.row.first * p.xs : th.b * p.xb) + th.tile.first;
    const VT* const from_d = d == nullptr ? nullptr : d + th.row.first * p.C + th.tile.first;
    float h_next[V];
    auto issue = [&](int64_t i) {
        if (i < n) {
            const int64_t k = th.k1 - 1 - i;
            unsigned char* at = mine + (int)(i % p.stages) * stage;
            th.copy_values(p, k, reinterpret_cast<VT*>(at), from_x, p.xs, p.x_bytes);
            if (from_d != nullptr)
                th.copy_values(p, k, reinterpret_cast<VT*>(at + S::kX), from_d, p.C, p.d_bytes);
            th.copy_gates(p, k, reinterpret_cast<GT*>(at + 2 * S::kX));
        }
        copies_issued();
    };
    auto kept_at = [&](int64_t i, float (&to)[V]) {
        if (i < n)
            th.get(kept + kept_index(p, th.row, th.b, th.chunk, th.k1 - 1 - i) * p.C + th.ch, to);
    };
    for (int i = 0; i < p.stages - 1; ++i) issue(i);
    kept_at(0, h_next);
    float R[V];         // what flows back into the last state of the tile
#pragma unroll
    for (int v = 0; v < V; ++v) R[v] = 0.f;
    if (d_last != nullptr) th.get(d_last + th.b * p.C + th.ch, R);
    if (th.on)
        for (int s = p.splits - 1; s > th.split; --s)
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (v < th.have) {
                    const float2 q = pairs[(th.b * p.splits + s) * p.C + th.ch + v];
                    R[v] = past(q.x, R[v], q.y);
                }
    const int64_t dx_step = p.reverse ? -(int64_t)p.C : p.C;
    const int64_t dg_step = p.reverse ? -(int64_t)p.H : p.H;
    for (int64_t i = 0; i < n; ++i) {
        const int64_t k = th.k1 - 1 - i, t0 = th.first_step(p, k, th.sub);
        issue(i + p.stages - 1);
        copies_wait(p.stages - 1);
        __syncwarp();
        const unsigned char* at = mine + (int)(i % p.stages) * stage;
        const VT* const tx = reinterpret_cast<const VT*>(at) + th.lane * V;
        const VT* const td = reinterpret_cast<const VT*>(at + S::kX) + th.lane * V;
        const GT* const tg = reinterpret_cast<const GT*>(at + 2 * S::kX);
        float h[V];
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = h_next[v];
        kept_at(i + 1, h_next);
        float a[L][V], w[L][V], A[V], B[V], EA[V], E[V];
        auto scan = [&](auto safe) {
            constexpr bool SAFE = decltype(safe)::value;
#pragma unroll
            for (int v = 0; v < V; ++v) { A[v] = 1.f; B[v] = 0.f; E[v] = 0.f; }
#pragma unroll
            for (int l = 0; l < L; ++l) {
                float g[S::GV], xv[V], one_a = 0.f, one_w = 0.f;
                th.load_gates(tg, l, g);
                load_some<V>(tx + l * 32 * V, xv);
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    if (v < S::GV) {
                        one_a = decay_of(g[v < S::GV ? v : 0]);
                        one_w = p.weighted ? 1.f : weight_of(g[v < S::GV ? v : 0], one_a);
                    }
                    a[l][v] = one_a;
                    w[l][v] = one_w;
                    A[v] *= one_a;
                    B[v] = SAFE ? past(one_a, B[v], times(one_w, xv[v]))
                                : fmaf(one_a, B[v], one_w * xv[v]);
                }
            }
            if (from_d != nullptr) {
#pragma unroll
                for (int l = L - 1; l >= 0; --l) {
                    float e[V];
                    load_some<V>(td + l * 32 * V, e);
#pragma unroll
                    for (int v = 0; v < V; ++v)
                        E[v] = SAFE ? past(a[l][v], E[v] + e[v], 0.f) : a[l][v] * (E[v] + e[v]);
                }
            }
        };
        scan(std::false_type{});
        bool odd = false;
#pragma unroll
        for (int v = 0; v < V; ++v)
            odd |= v < th.have && !(finite(A[v]) && finite(B[v]) && finite(E[v]));
        if (odd) scan(std::true_type{});
#pragma unroll
        for (int v = 0; v < V; ++v) EA[v] = A[v];
        float TA[V], TB[V], TE[V];
        join_lanes<V, false>(p.lanes, th.lane, A, B);
        join_lanes<V, true>(p.lanes, th.lane, EA, E);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            TA[v] = __shfl_sync(~0u, EA[v], th.cl);
            TB[v] = __shfl_sync(~0u, B[v], 32 - p.lanes + th.cl);
            TE[v] = __shfl_sync(~0u, E[v], th.cl);
        }
        if (p.lanes < 32) {
            const int lo = th.lane - p.lanes, hi = th.lane + p.lanes;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float pa = __shfl_sync(~0u, A[v], lo & 31), pb = __shfl_sync(~0u, B[v], lo & 31);
                const float na = __shfl_sync(~0u, EA[v], hi & 31), ne = __shfl_sync(~0u, E[v], hi & 31);
                A[v] = lo >= 0 ? pa : 1.f;
                B[v] = lo >= 0 ? pb : 0.f;
                EA[v] = hi < 32 ? na : 1.f;
                E[v] = hi < 32 ? ne : 0.f;
            }
        } else {
#pragma unroll
            for (int v = 0; v < V; ++v) { A[v] = EA[v] = 1.f; B[v] = E[v] = 0.f; }
        }
        float G[V];
        if (p.warps == 1) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                h[v] = past(A[v], h[v], B[v]);
                G[v] = past(EA[v], R[v], E[v]);
                R[v] = past(TA[v], R[v], TE[v]);
            }
        } else {
            auto& pair = s_pair[i & 1];
            if (th.sub == 0)
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    pair[th.warp][0][th.cl * V + v] = TA[v];
                    pair[th.warp][1][th.cl * V + v] = TB[v];
                    pair[th.warp][2][th.cl * V + v] = TE[v];
                }
            th.unit_sync(p);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const int c = th.cl * V + v;
                for (int j = 0; j < th.wseg; ++j) {
                    const auto& q = pair[th.group * p.warps + j];
                    h[v] = past(q[0][c], h[v], q[1][c]);
                }
                h[v] = past(A[v], h[v], B[v]);
                for (int j = p.warps - 1; j >= 0; --j) {
                    if (j == th.wseg) G[v] = past(EA[v], R[v], E[v]);
                    const auto& q = pair[th.group * p.warps + j];
                    R[v] = past(q[0][c], R[v], q[2][c]);
                }
            }
        }
        const bool whole = t0 + L <= th.row.len;
        VT* to_x = dx == nullptr ? nullptr
                                 : dx + (th.row.first + th.place(p, t0 + L - 1)) * p.C + th.ch;
        GT* to_g = dg == nullptr || p.D > 1
                       ? nullptr : dg + (th.row.first + th.place(p, t0 + L - 1)) * p.H + th.ch;
        auto unwind = [&](auto safe) {
            constexpr bool SAFE = decltype(safe)::value;
            // forwards: what dg has besides the adjoint
            float q[L][V];
#pragma unroll
            for (int l = 0; l < L; ++l) {
                float xv[V];
                load_some<V>(tx + l * 32 * V, xv);
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const float wv = w[l][v], av = a[l][v];
                    if (SAFE) {
                        // (a value that is not finite in a place of no thickness is no sample)
                        const float xs = wv == 0.f && !finite(xv[v]) ? h[v] : xv[v];
                        q[l][v] = av == 0.f ? 0.f : av * (p.weighted ? -h[v] : xs - h[v]);
                        h[v] = past(av, h[v], times(wv, xv[v]));
                    } else {
                        q[l][v] = av * (p.weighted ? -h[v] : xv[v] - h[v]);
                        h[v] = fmaf(av, h[v], wv * xv[v]);
                    }
                }
            }
            // and back
#pragma unroll
            for (int l = L - 1; l >= 0; --l) {
                const bool in = th.on && (whole || t0 + l < th.row.len);
                float e[V], dxv[V], dgv[V];
#pragma unroll
                for (int v = 0; v < V; ++v) e[v] = 0.f;
                if (from_d != nullptr) load_some<V>(td + l * 32 * V, e);
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    G[v] += e[v];
                    dxv[v] = w[l][v] * G[v];
                    dgv[v] = q[l][v] * G[v];
                    G[v] = SAFE ? past(a[l][v], G[v], 0.f) : a[l][v] * G[v];
                }
                if (in && dx != nullptr) th.put(p, to_x - (L - 1 - l) * dx_step, dxv);
                if (to_g != nullptr) {
                    if (in) th.put(p, to_g - (L - 1 - l) * dg_step, dgv);
                } else if (p.D > 1 && dg != nullptr) {
#pragma unroll
                    for (int v = 0; v < V; ++v) sums[l * (32 * V + 1) + th.lane * V + v] = dgv[v];
                }
            }
        };
#pragma unroll
        for (int v = 0; v < V; ++v) odd |= v < th.have && !(finite(h[v]) && finite(G[v]));
        if (odd) unwind(std::true_type{});
        else unwind(std::false_type{});
        if (p.D > 1 && dg != nullptr) {
            __syncwarp();
            const int heads = p.parts > 1 ? 1 : th.tile.width / p.D, subs = 32 / p.lanes;
            const int width = p.parts > 1 ? th.tile.width : p.D;
            for (int j = th.lane; j < L * subs * heads; j += 32) {
                const int l = j / (subs * heads), r = j - l * (subs * heads);
                const int s = r / heads, hd = r - s * heads;
                const float* from = sums + l * (32 * V + 1) + s * p.lanes * V + hd * p.D;
                float sum = 0.f;
                for (int c = 0; c < width; ++c) sum += from[c];
                const int64_t t = th.first_step(p, k, s) + l;
                if (t >= th.row.len) continue;
                const int64_t where = th.row.first + th.place(p, t);
                if (p.parts > 1) {
                    const int part = (th.tile.first - th.tile.head * p.D) / p.tile;
                    const int64_t steps = p.offsets ? p.T : p.B * p.T;
                    parted[(part * steps + where) * p.H + th.tile.head] = sum;
                } else {
                    dg[where * p.H + th.tile.head + hd] = from_float<GT>(sum);
                }
            }
        }
        __syncwarp();
    }
    if (th.split == 0) {
        if (th.wseg == 0 && th.sub == 0 && th.on && dh0 != nullptr)
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (v < th.have) dh0[th.b * p.C + th.ch + v] = R[v];
        const int thread = th.wseg * 32 + th.lane, threads = p.warps * 32;
        clear_uncovered(p, th.b, th.tile.first, th.tile.width, (int64_t)p.C, dx, thread, threads);
        const bool own_head = p.parts == 1 || th.tile.first == th.tile.head * p.D;
        if (own_head)
            clear_uncovered(p, th.b, p.D == 1 ? th.tile.first : th.tile.head,
                            p.D == 1 ? th.tile.width : p.parts > 1 ? 1 : th.tile.width / p.D,
                            (int64_t)p.H, dg, thread, threads);
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
