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
// stretches' pairs in shared memory, always in the order of the steps, so that a call repeats to the
// bit.  The backward pass runs the same from the other end over
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
    // tiles of channels: whole groups, or a part of one (`tile` of rays by quads: a warp's window)
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

// a = exp(-g) and w = 1 - a.  Up to kThin, where the difference would cancel, w comes from a
// polynomial g (1 + c1 g + ... + c4 g^4), the best of its degree there (off by 2.7e-9 of w, and by
// 1.6 u with its rounding, u = 2^-24), and a from w, rounded to nearest: the hardware's power of two is
// off to one side near 1, by about 1e-8, and so is the nearest float to log2(e).  That made 2e-6 of what
// reaches a background behind 200 samples, and 4e-4 of a state behind 2^17 thin steps, now 2e-5.
// Beyond, where few steps leave nothing, a is off by 2 ulp of the power of two and g u from its
// argument, an error that a itself outweighs (g exp(-g) < 0.4).
constexpr float kThin = 0.25f;
constexpr float kThin1 = -0.49999964f, kThin2 = 0.16665322f, kThin3 = -0.041502316f,
                kThin4 = 0.0075347046f;
struct Gate { float a, w; };
__device__ __forceinline__ Gate gate_of(float g) {
    const float s = g * fmaf(g, fmaf(g, fmaf(g, fmaf(g, kThin4, kThin3), kThin2), kThin1), 1.f);
    constexpr double log2e = 1.4426950408889634;
    constexpr float most = (float)log2e, rest = (float)(log2e - most);
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(fmaf(g, -most, g * -rest)));
    return fabsf(g) < kThin ? Gate{1.f - s, s} : Gate{e, 1.f - e};
}
__device__ __forceinline__ float times(float w, float x) { return w == 0.f ? 0.f : w * x; }
// a h + b, with nothing of h where a is 0
__device__ __forceinline__ float past(float a, float h, float b) {
    return a == 0.f ? b : fmaf(a, h, b);
}

// Two channels at once: sm_100's packed 32-bit arithmetic, one instruction for both.
struct F2 { float x, y; };
__device__ __forceinline__ F2 two(float v) { return {v, v}; }
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
    F2 r;
    asm("{.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
        "mov.b64 c, {%6, %7};\n\tfma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
    F2 r;
    asm("{.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
        "mul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
    F2 r;
    asm("{.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
        "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ F2 past2(F2 a, F2 h, F2 b) {
    return {past(a.x, h.x, b.x), past(a.y, h.y, b.y)};
}
// The product of the gates of two neighbouring stretches.  It is 0 where one of them is, whatever the
// other, and only there: a product of many gates that rounds to 0 is held as the smallest float, so
// that a stretch of 0 has an opaque step, which nothing gets past, while a state that is not a number
// gets past any other.  (It need not be a number where a gate is not: what its stretch adds is not
// either.)
constexpr float kLeast = 1.4e-45f;
__device__ __forceinline__ float min3(float a, float b, float c) {
    float r;
    asm("min.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ F2 gates2(F2 a, F2 before) {
    const F2 r = mul2(a, before);
    return {fmaxf(r.x, min3(a.x, before.x, kLeast)), fmaxf(r.y, min3(a.y, before.y, kLeast))};
}
// The same of the product A of a stretch's steps (without a gate for each channel both are the same).
__device__ __forceinline__ float least8(float a, float b, float c, float d, float e, float f, float g,
                                        float h) {
    return min3(min3(a, b, c), min3(d, e, f), min3(g, h, kLeast));
}
template <bool PC>
__device__ __forceinline__ void keep_open(F2& A, const F2 (&a)[8]) {
    A.x = fmaxf(A.x, least8(a[0].x, a[1].x, a[2].x, a[3].x, a[4].x, a[5].x, a[6].x, a[7].x));
    A.y = !PC ? A.x : fmaxf(A.y, least8(a[0].y, a[1].y, a[2].y, a[3].y, a[4].y, a[5].y, a[6].y,
                                        a[7].y));
}
__device__ __forceinline__ F2 shfl2(F2 v, int lane) {
    return {__shfl_sync(~0u, v.x, lane), __shfl_sync(~0u, v.y, lane)};
}
// 0 where all is finite, NaN otherwise.
__device__ __forceinline__ float spoilt(F2 a, F2 b) {
    const F2 r = fma2(a, two(0.f), mul2(b, two(0.f)));
    return r.x + r.y;
}
// gate_of of two channels (with log2(e) in one part: an argument's own rounding is as large).
__device__ __forceinline__ void gates_of(F2 g, F2& a, F2& w) {
    const F2 t = mul2(g, two(-1.4426950408889634f));
    F2 e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(t.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(t.y));
    F2 s = fma2(g, two(kThin4), two(kThin3));
    s = fma2(g, s, two(kThin2));
    s = fma2(g, s, two(kThin1));
    s = mul2(g, fma2(g, s, two(1.f)));
    const F2 c = fma2(s, two(-1.f), two(1.f)), d = fma2(e, two(-1.f), two(1.f));
    const bool x = fabsf(g.x) < kThin, y = fabsf(g.y) < kThin;
    a = {x ? c.x : e.x, y ? c.y : e.y};
    w = {x ? s.x : d.x, y ? s.y : d.y};
}

// Steps of a packed call that no row covers, before the first row and behind the last (a buffer that
// is not full), get zeros: from all threads of the launch.
template <class T>
__device__ __forceinline__ void clear_uncovered(const ScanArgs& p, int64_t row_len, T* out) {
    if (p.offsets == nullptr || out == nullptr) return;
    const int64_t first = __ldg(p.offsets), end = __ldg(p.offsets + p.B);
    const int64_t lo = first < 0 ? 0 : first > p.T ? p.T : first;
    const int64_t hi = end < 0 ? 0 : end > p.T ? p.T : end;
    const int64_t before = lo * row_len, all = before + (p.T - hi) * row_len;
    const int64_t stride = (int64_t)gridDim.x * gridDim.y * blockDim.x;
    int64_t i = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * blockDim.x + threadIdx.x;
    for (; i < all; i += stride)
        out[i < before ? i : hi * row_len + (i - before)] = from_float<T>(0.f);
}

// Index of the kept state at the start of stretch k of a row.
__device__ __forceinline__ int64_t kept_index(const ScanArgs& p, const ScanRow& row, int64_t b,
                                              int chunk, int64_t k) {
    return p.offsets == nullptr ? b * ((p.T + chunk - 1) / chunk) + k : row.first / chunk + b + k;
}

// ---------------------------------------------------------------------------
// Tiles.  A lane has two channels; a unit (a row's tile of up to 2 * `lanes` channels) is scanned by
// `warps` warps; of a warp, each group of `lanes` lanes takes kSteps steps, so that a tile has
// warps * (32 / lanes) * kSteps steps.  Each warp copies its own part of the tiles to shared memory,
// asynchronously and up to kScanStages ahead: row l holds what the lanes need for their l-th step,
// whatever the width of a channel row.
constexpr int kSteps = 8;
template <class VT, class GT, bool PC>
struct ScanShape {
    static constexpr int GV = PC ? 2 : 1;
    static constexpr int kX = kSteps * 64 * sizeof(VT);         // bytes of a warp's tile of values,
    static constexpr int kG = kSteps * 32 * GV * sizeof(GT);    // of gates
    static constexpr int kPitch = PC ? 65 : 36;                 // of its products for dg
    static constexpr int kSum = kSteps * kPitch * 4;
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
// LN: 0, or the lanes of a row of channels where every tile is whole, its rows are copied 16 bytes at
// a time and its unit has all warps: what every large call of plain arrays is, without the
// arithmetic on its shape ((8, 4096, 2048) bf16, forward and backward: 123 and 272 -> 98 and 176 us; 101 and 175
// with the products and the gates as they are now).
template <class VT, class GT, bool PC, int LN>
struct ScanThread {
    using S = ScanShape<VT, GT, PC>;
    static __device__ __forceinline__ int lanes_of(const ScanArgs& p) { return LN ? LN : p.lanes; }
    static __device__ __forceinline__ int warps_of(const ScanArgs& p) {
        return LN ? kScanWarps : p.warps;
    }
    int lane, warp, group, wseg;    // wseg: the warp's number in its unit
    int sub, cl, chunk;
    int64_t b;
    ScanTile tile;
    ScanRow row;
    int have;                // channels of this lane
    int ch;                  // its first channel
    int gate, gate2;         // where the gates of its two are in a row of a tile of shared gates
    int step0;               // its first step within a tile
    int split;
    bool one_each;           // a gate for each channel
    int64_t k0, k1;          // tiles of this block's range

    __device__ __forceinline__ bool init(const ScanArgs& p) {
        lane = threadIdx.x & 31;
        warp = threadIdx.x >> 5;
        group = warp / warps_of(p);
        wseg = warp - group * warps_of(p);
        split = blockIdx.y;
        one_each = p.D == 1;
        const int64_t unit = (int64_t)blockIdx.x * (kScanWarps / warps_of(p)) + group;
        if (unit >= p.units) return false;
        b = unit / p.tiles;
        tile = scan_tile(p, (int)(unit - b * p.tiles));
        row = scan_row(p, b);
        sub = lane / lanes_of(p);
        cl = lane - sub * lanes_of(p);
        have = tile.width - cl * 2;
        have = LN || have >= 2 ? 2 : have < 0 ? 0 : have;
        ch = tile.first + (have ? cl * 2 : 0);
        const int heads = p.parts > 1 ? 1 : p.D > 1 ? tile.width / p.D : 0;
        gate = sub * heads + (p.parts > 1 || !have ? 0 : cl * 2 / p.D);
        gate2 = sub * heads + (p.parts > 1 || have < 2 ? 0 : (cl * 2 + 1) / p.D);
        step0 = (wseg * (32 / lanes_of(p)) + sub) * kSteps;
        chunk = warps_of(p) * (32 / lanes_of(p)) * kSteps;
        const int64_t chunks = (row.len + chunk - 1) / chunk;
        const int64_t per = (chunks + p.splits - 1) / p.splits;
        k0 = per * split < chunks ? per * split : chunks;
        k1 = per * (split + 1) < chunks ? per * (split + 1) : chunks;
        return true;
    }
    __device__ __forceinline__ int64_t place(const ScanArgs& p, int64_t t) const {
        return p.reverse ? row.len - 1 - t : t;
    }
    // Steps of tile k that the row has.
    __device__ __forceinline__ int room(int64_t k) const {
        const int64_t left = row.len - k * chunk;
        return left < chunk ? (int)left : chunk;
    }
    // The warp's part of a tile, BYTES at a time.  `from`: the row's first step in the tile; a lane's
    // pieces lie in one column, so many rows apart.
    template <class T, int W, int BYTES>
    __device__ __forceinline__ void copy_pieces(const ScanArgs& p, T* to, const T* from,
                                                int64_t step, int room) const {
        constexpr int n = BYTES / (int)sizeof(T);           // elements of a piece
        constexpr int P = 32 * W / n, COLS = P < 32 ? P : 32, ROWS = 32 / COLS;
        const int each = lanes_of(p) * W;                       // elements of a row of channels
#pragma unroll
        for (int half = 0; half < P; half += COLS) {
            const int j = (half + lane % COLS) * n;
            const int s = j >> (31 - __clz(each)), c = j & (each - 1);
            if (c >= tile.width) continue;
            int t = (wseg * (32 / lanes_of(p)) + s) * kSteps + lane / COLS;
            const T* src = from + t * step + c;
            T* dst = to + lane / COLS * 32 * W + j;
#pragma unroll
            for (int l = 0; l < kSteps; l += ROWS) {
                const bool in = t < room;
                if (BYTES >= 4) copy_async(dst, in ? src : from, BYTES, in);
                else *dst = in ? *src : from_float<T>(0.f);
                t += ROWS;
                src += ROWS * step;
                dst += ROWS * 32 * W;
            }
        }
    }
    template <class T, int W>
    __device__ __forceinline__ void copy_rows(const ScanArgs& p, T* to, const T* from, int64_t step,
                                              int room, int at_once) const {
        if (at_once == 16) copy_pieces<T, W, 16>(p, to, from, step, room);
        else if (at_once == 4) copy_pieces<T, W, 4>(p, to, from, step, room);
        else copy_pieces<T, W, (int)sizeof(T)>(p, to, from, step, room);
    }
    // The same 16 bytes at a time with what a lane needs for it at hand.
    template <class T>
    struct Pieces {
        static constexpr int n = 16 / (int)sizeof(T), COLS = 64 / n, ROWS = 32 / COLS;
        int64_t off, down;      // its first piece, from there to the next
        int t;                  // the step of its first piece; none: none
        unsigned dst;
        __device__ __forceinline__ void init(const ScanArgs& p, const ScanThread& th, int64_t step) {
            const int each = lanes_of(p) * 2, j = th.lane % COLS * n;
            const int s = j >> (31 - __clz(each)), c = j & (each - 1);
            const int t0 = (th.wseg * (32 / lanes_of(p)) + s) * kSteps + th.lane / COLS;
            off = t0 * step + c;
            down = ROWS * step;
            t = c < th.tile.width ? t0 : 1 << 30;
            dst = (unsigned)((th.lane / COLS * 64 + j) * sizeof(T));
        }
        __device__ __forceinline__ void copy(unsigned tile, const T* from, int room) const {
            if (!LN && t >= 1 << 30) return;
            const T* src = from + off;
#pragma unroll
            for (int l = 0; l < kSteps; l += ROWS, src += down) {
                const bool in = t + l < room;
                const int bytes = in ? 16 : 0;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::
                             "r"(tile + dst + (unsigned)(l * 64 * sizeof(T))), "l"(in ? src : from),
                             "r"(bytes) : "memory");
            }
        }
    };
    // The same of the gates, of a row from `from` (its first gate of the tile in the first step).
    __device__ __forceinline__ void copy_gates(const ScanArgs& p, GT* to, const GT* from,
                                               int64_t step, int room) const {
        if (PC && p.D == 1) {
            copy_rows<GT, 2>(p, to, from, step, room, p.g_bytes);
            return;
        }
        // one gate for several channels: once each
        const int heads = p.parts > 1 ? 1 : tile.width / p.D, subs = 32 / lanes_of(p);
        if (heads == 1) {
            for (int i = lane; i < kSteps * subs; i += 32) {
                const int t = wseg * subs * kSteps + i;     // step of sub i / kSteps
                const bool in = t < room;
                const GT* src = in ? from + t * step : from;
                GT* dst = to + (i % kSteps) * 32 * S::GV + i / kSteps;
                if (sizeof(GT) == 4) copy_async(dst, src, 4, in);
                else *dst = in ? *src : from_float<GT>(0.f);
            }
            return;
        }
        for (int i = lane; i < kSteps * subs * heads; i += 32) {
            const int l = i / (subs * heads), j = i - l * (subs * heads);
            const int s = j / heads, t = (wseg * subs + s) * kSteps + l;
            const bool in = t < room;
            const GT* src = in ? from + t * step + (j - s * heads) : from;
            GT* dst = to + l * 32 * S::GV + j;
            if (sizeof(GT) == 4) copy_async(dst, src, 4, in);
            else *dst = in ? *src : from_float<GT>(0.f);
        }
    }
    // What a tile never fills holds zeros: no thickness, no value.
    __device__ __forceinline__ void clear(const ScanArgs& p, unsigned char* mine, int bytes) const {
        if (!LN && tile.width < lanes_of(p) * 2)
            for (int i = lane * 16; i < bytes; i += 512)
                *reinterpret_cast<uint4*>(mine + i) = make_uint4(0, 0, 0, 0);
        __syncwarp();
    }
    // a and w of the lane's two channels in step l
    template <bool WEIGHTED>
    __device__ __forceinline__ void gates(const GT* g, int l, F2& a, F2& w) const {
        if (PC) {
            float v[2];
            if (LN || one_each) {
                load_some<2>(g + (l * 32 + lane) * 2, v);
            } else {
                v[0] = to_float(g[l * 64 + gate]);
                v[1] = to_float(g[l * 64 + gate2]);
            }
            gates_of({v[0], v[1]}, a, w);
        } else {
            const Gate t = gate_of(to_float(g[l * 32 + gate]));
            a = two(t.a);
            w = two(t.w);
        }
        if (WEIGHTED) w = two(1.f);
    }
    __device__ __forceinline__ F2 at(const VT* tile_x, int l) const {
        float v[2];
        load_some<2>(tile_x + (l * 32 + lane) * 2, v);
        return {v[0], v[1]};
    }
    // a and what step l adds (raw: its value as it is), for the careful loops
    __device__ __forceinline__ void step(const ScanArgs& p, const VT* x, const GT* g, int l, F2& a,
                                         F2& u, bool raw) const {
        F2 w;
        gates<false>(g, l, a, w);
        u = x == nullptr ? two(0.f) : at(x, l);
        if (!p.weighted && !raw) u = {times(w.x, u.x), times(w.y, u.y)};
    }
    __device__ __forceinline__ F2 get(const float* from) const {
        return {have > 0 ? __ldg(from) : 0.f, have > 1 ? __ldg(from + 1) : 0.f};
    }
    __device__ __forceinline__ void put(const ScanArgs& p, float* to, F2 v) const {
        if (have > 0) to[0] = v.x;
        if (have > 1) to[1] = v.y;
    }
    // state before the row
    __device__ __forceinline__ F2 start(const ScanArgs& p) const {
        return p.h0 != nullptr ? get(p.h0 + b * p.hb + ch) : two(0.f);
    }
    // two neighbouring elements of an output row, as far as the tile goes
    template <class T>
    __device__ __forceinline__ void store(const ScanArgs& p, T* to, F2 v) const {
        if (LN || p.paired) {
            const float w[2] = {v.x, v.y};
            store_some<2>(to, w);
        } else {
            to[0] = from_float<T>(v.x);
            if (have > 1) to[1] = from_float<T>(v.y);
        }
    }
    // What the row's other ranges, before this one or (back) behind it, do to `h`.  The unit's groups
    // of lanes fold a part of them each, in the order of the steps (folded by every thread, up to 255
    // pairs took 30 of the 45 us of a sequence of 131072 steps of 64 channels).
    __device__ __forceinline__ F2 ranges(const ScanArgs& p, const float2* pairs, F2 h, bool back,
                                         float4* shared) const {
        if (p.splits == 1) return h;
        const int n = back ? p.splits - 1 - split : split;
        const int subs = 32 / lanes_of(p), workers = warps_of(p) * subs, me = wseg * subs + sub;
        const int per = (n + workers - 1) / workers;
        const int from = per * me < n ? per * me : n, to = from + per < n ? from + per : n;
        const float2* at = pairs + (b * p.splits + (back ? p.splits - 1 - from : from)) * p.C + ch;
        const int step = back ? -p.C : p.C;
        F2 A = two(1.f), B = two(0.f);
        if (have > 0) {
            const int second = have - 1;
#pragma unroll 8
            for (int s = from; s < to; ++s, at += step) {
                const float2 q = __ldcg(at), r = __ldcg(at + second);
                B = past2({q.x, r.x}, B, {q.y, r.y});
                A = gates2({q.x, r.x}, A);
            }
        }
        shared += group * warps_of(p) * 32;
        shared[me * lanes_of(p) + cl] = make_float4(A.x, A.y, B.x, B.y);
        unit_sync(p);
        for (int w = 0; w < workers && w * per < n; ++w) {
            const float4 q = shared[w * lanes_of(p) + cl];
            h = past2({q.x, q.y}, h, {q.z, q.w});
        }
        unit_sync(p);
        return h;
    }
    __device__ __forceinline__ void unit_sync(const ScanArgs& p) const {
        if (warps_of(p) == 1) __syncwarp();
        else asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(warps_of(p) * 32) : "memory");
    }
};

// Joins the pairs of a warp's groups of lanes.  In: (A, B) of this lane's steps.  Out: what the
// warp's steps before them (BACK: behind them, from the other end) do to the state, and the pair of
// all (TA only if ALL).
template <bool BACK, bool PC, bool ALL = true>
__device__ __forceinline__ void join_lanes(int lanes, int lane, F2& A, F2& B, F2& TA, F2& TB) {
    if (lanes == 32) {
        TA = A;
        TB = B;
        A = two(1.f);
        B = two(0.f);
        return;
    }
    // (without a gate for each channel both are the same)
    auto shfl_a = [&](int from) {
        return PC ? shfl2(A, from) : two(__shfl_sync(~0u, A.x, from));
    };
    for (int d = lanes; d < 32; d *= 2) {
        const int from = BACK ? lane + d : lane - d;
        const F2 a = shfl_a(from & 31), b = shfl2(B, from & 31);
        if (from >= 0 && from < 32) {
            B = past2(A, b, B);
            A = gates2(A, a);
        }
    }
    const int edge = BACK ? lane & (lanes - 1) : 32 - lanes + (lane & (lanes - 1));
    if (ALL) TA = shfl_a(edge);
    TB = shfl2(B, edge);
    const int by = BACK ? lane + lanes : lane - lanes;
    A = shfl_a(by & 31);
    B = shfl2(B, by & 31);
    if (by < 0 || by >= 32) {
        A = two(1.f);
        B = two(0.f);
    }
}

// MODE 0: states and the last one; 1: the pair (A, B) of the block's range; 2: the pair (A, E) of it
// backwards, where E is what the range's own gradients `x` send back past its first step.
template <class VT, class GT, bool PC, int MODE, int LN>
__global__ void __launch_bounds__(kScanBlock, MODE == 0 ? 2 : 3)
scan_kernel(ScanArgs p, const VT* __restrict__ x, float2* __restrict__ pairs,
            VT* __restrict__ states, float* __restrict__ last, float* __restrict__ kept) {
    using Th = ScanThread<VT, GT, PC, LN>;
    using S = typename Th::S;
    constexpr int L = kSteps;
    constexpr bool BACK = MODE == 2;
    extern __shared__ __align__(16) unsigned char s_tiles[];
    __shared__ float4 s_pair[2][kScanWarps][32];
    if (MODE == 0) clear_uncovered(p, p.C, states);
    Th th;
    if (!th.init(p)) return;
    const int n = (int)(th.k1 - th.k0);
    const int stage = S::kX + S::kG;
    unsigned char* const mine = s_tiles + (size_t)th.warp * p.stages * stage;
    th.clear(p, mine, p.stages * stage);
    // (a range backwards has its tiles from the last to the first)
    const int64_t first = BACK ? th.k1 - 1 : th.k0;
    const int64_t step_x = p.reverse ? -p.xs : p.xs, step_g = p.reverse ? -p.gs : p.gs;
    const int64_t at0 = th.place(p, first * th.chunk);
    const VT* from_x = x + (p.offsets ? th.row.first * p.xs : th.b * p.xb) + at0 * p.xs +
                       th.tile.first;
    const GT* from_g = static_cast<const GT*>(p.g) +
        (p.offsets ? th.row.first * p.gs : th.b * p.gb) + at0 * p.gs + th.tile.head;
    typename Th::template Pieces<VT> px;
    typename Th::template Pieces<GT> pg;
    px.init(p, th, step_x);
    pg.init(p, th, step_g);
    const bool whole_x = LN || p.x_bytes == 16;
    const bool whole_g = PC && (LN || (p.D == 1 && p.g_bytes == 16));
    const unsigned shared = (unsigned)__cvta_generic_to_shared(mine);
    const int64_t next_x = (BACK ? -th.chunk : th.chunk) * step_x;
    const int64_t next_g = (BACK ? -th.chunk : th.chunk) * step_g;
    int issued = 0, slot_in = 0, slot = 0;      // (offsets of the tiles' places)
    auto issue = [&] {
        if (issued < n) {
            const int room = th.room(BACK ? first - issued : first + issued);
            if (BACK && x == nullptr) {
            } else if (whole_x) {
                px.copy(shared + slot_in, from_x, room);
            } else {
                th.template copy_rows<VT, 2>(p, reinterpret_cast<VT*>(mine + slot_in), from_x, step_x,
                                             room, p.x_bytes);
            }
            if (whole_g) pg.copy(shared + slot_in + S::kX, from_g, room);
            else th.copy_gates(p, reinterpret_cast<GT*>(mine + slot_in + S::kX), from_g, step_g, room);
            from_x += next_x;
            from_g += next_g;
            slot_in = slot_in + stage == p.stages * stage ? 0 : slot_in + stage;
        }
        ++issued;
        copies_issued();
    };
    for (int i = 0; i < p.stages - 1; ++i) issue();
    F2 carry = MODE == 0 ? th.ranges(p, pairs, th.start(p), false, &s_pair[0][0][0]) : two(0.f);
    F2 through = two(1.f);              // MODE 1, 2: with carry, the pair so far (of the first warp)
    VT* out = states == nullptr ? nullptr
        : states + (th.row.first + th.place(p, first * th.chunk + th.step0)) * p.C + th.ch;
    float* keep = kept == nullptr || th.wseg != 0 || th.sub != 0 ? nullptr
        : kept + kept_index(p, th.row, th.b, th.chunk, first) * p.C + th.ch;
    const int out_step = p.reverse ? -p.C : p.C;
    const int64_t out_next = (int64_t)th.chunk * out_step;
    for (int i = 0; i < n; ++i) {
        issue();
        copies_wait(p.stages - 1);
        __syncwarp();
        const unsigned char* at = mine + slot;
        slot = slot + stage == p.stages * stage ? 0 : slot + stage;
        const VT* const tx = reinterpret_cast<const VT*>(at);
        const GT* const tg = reinterpret_cast<const GT*>(at + S::kX);
        F2 a[L], u[L], A, B;
        // (a step beyond the row has no thickness and no value: it changes nothing)
        auto scan = [&](auto weighted) {
            A = two(1.f);
            B = two(0.f);
#pragma unroll
            for (int j = 0; j < L; ++j) {
                const int l = BACK ? L - 1 - j : j;
                F2 w;
                th.template gates<BACK || decltype(weighted)::value>(tg, l, a[l], w);
                const F2 v = BACK && x == nullptr ? two(0.f) : th.at(tx, l);
                if (BACK) {
                    B = mul2(a[l], add2(B, v));
                } else {
                    u[l] = decltype(weighted)::value ? v : mul2(w, v);
                    B = fma2(a[l], B, u[l]);
                }
                A = mul2(A, a[l]);
            }
        };
        if (p.weighted) scan(std::true_type{});
        else scan(std::false_type{});
        // What is not finite stays so to the end of the stretch; then the steps that do not count
        // are told from those that do, in a loop of its own.
        bool odd = spoilt(A, B) != 0.f;
        keep_open<PC>(A, a);
        if (odd) {
            A = two(1.f);
            B = two(0.f);
#pragma unroll 1
            for (int j = 0; j < L; ++j) {
                F2 al, ul;
                if (BACK) {
                    th.step(p, x == nullptr ? nullptr : tx, tg, L - 1 - j, al, ul, true);
                    B = past2(al, add2(B, ul), two(0.f));
                } else {
                    th.step(p, tx, tg, j, al, ul, false);
                    B = past2(al, B, ul);
                }
                A = gates2(al, A);
            }
        }
        if (keep != nullptr) {
            th.put(p, keep, carry);
            keep += p.C;
        }
        F2 TA, TB;
        join_lanes<BACK, PC>(Th::lanes_of(p), th.lane, A, B, TA, TB);
        F2 h = carry;
        if (Th::warps_of(p) == 1) {
            carry = past2(TA, carry, TB);
            if (MODE != 0) through = gates2(TA, through);
        } else {
            auto& pair = s_pair[i & 1];
            if (th.sub == 0) pair[th.warp][th.cl] = make_float4(TA.x, TA.y, TB.x, TB.y);
            th.unit_sync(p);
            const F2 before = carry;
            const float4* const all = &pair[th.group * Th::warps_of(p)][th.cl];
#pragma unroll 8
            for (int j = 0; j < Th::warps_of(p); ++j) {
                const int w = BACK ? Th::warps_of(p) - 1 - j : j;
                if (w == th.wseg) h = carry;
                const float4 q = all[w * 32];
                carry = fma2({q.x, q.y}, carry, {q.z, q.w});
            }
            if (MODE != 0 && th.wseg == 0)
#pragma unroll 8
                for (int w = 0; w < Th::warps_of(p); ++w) {
                    const float2 q = *reinterpret_cast<const float2*>(&all[w * 32]);
                    through = gates2({q.x, q.y}, through);
                }
            if (spoilt(carry, carry) != 0.f) {
                carry = before;
                for (int j = 0; j < Th::warps_of(p); ++j) {
                    const int w = BACK ? Th::warps_of(p) - 1 - j : j;
                    if (w == th.wseg) h = carry;
                    const float4 q = all[w * 32];
                    carry = past2({q.x, q.y}, carry, {q.z, q.w});
                }
            }
        }
        if (MODE == 0 && out != nullptr) {
            if (Th::lanes_of(p) < 32) h = past2(A, h, B);
            odd |= spoilt(h, h) != 0.f;
            const int64_t t0 = (first + i) * th.chunk + th.step0;
            VT* to = out;
            out += out_next;
            if (th.have && t0 + L <= th.row.len && !odd) {
#pragma unroll
                for (int l = 0; l < L; ++l, to += out_step) {
                    h = fma2(a[l], h, u[l]);
                    th.store(p, to, h);
                }
            } else if (th.have) {
#pragma unroll 1
                for (int l = 0; l < L && t0 + l < th.row.len; ++l, to += out_step) {
                    F2 al, ul;
                    th.step(p, tx, tg, l, al, ul, false);
                    h = past2(al, h, ul);
                    th.store(p, to, h);
                }
            }
        }
        __syncwarp();
    }
    if (th.wseg == 0 && th.sub == 0) {
        if (MODE != 0) {
            float2* to = pairs + (th.b * p.splits + th.split) * p.C + th.ch;
            if (th.have > 0) to[0] = make_float2(through.x, carry.x);
            if (th.have > 1) to[1] = make_float2(through.y, carry.y);
        } else if (th.split == p.splits - 1) {
            th.put(p, last + th.b * p.C + th.ch, carry);
        }
    }
}

// The backward pass of a tile.  `parted`: (parts, steps, H) floats for the sums of a group that
// several tiles share.
template <class VT, class GT, bool PC, int LN>
__global__ void __launch_bounds__(kScanBlock, 2)
scan_back_kernel(ScanArgs p, const VT* __restrict__ x, const float2* __restrict__ pairs,
                 const float* __restrict__ kept, const VT* __restrict__ d,
                 const float* __restrict__ d_last, VT* __restrict__ dx, GT* __restrict__ dg,
                 float* __restrict__ parted, float* __restrict__ dh0) {
    using Th = ScanThread<VT, GT, PC, LN>;
    using S = typename Th::S;
    constexpr int L = kSteps;
    extern __shared__ __align__(16) unsigned char s_tiles[];
    __shared__ float4 s_pair[2][kScanWarps][32];
    __shared__ float2 s_flow[2][kScanWarps][32];
    clear_uncovered(p, p.C, dx);
    clear_uncovered(p, p.H, dg);
    Th th;
    if (!th.init(p)) return;
    const int n = (int)(th.k1 - th.k0);
    const int stage = 2 * S::kX + S::kG;
    unsigned char* const mine = s_tiles + (size_t)th.warp * p.stages * stage;
    float* const sums = reinterpret_cast<float*>(s_tiles + (size_t)kScanWarps * p.stages * stage +
                                                 th.warp * S::kSum);
    th.clear(p, mine, p.stages * stage);
    const int64_t first = th.k1 - 1;
    const int64_t step_x = p.reverse ? -p.xs : p.xs, step_g = p.reverse ? -p.gs : p.gs;
    const int step_c = p.reverse ? -p.C : p.C, step_h = p.reverse ? -p.H : p.H;
    const int64_t at0 = th.place(p, first * th.chunk);
    const VT* from_x = x + (p.offsets ? th.row.first * p.xs : th.b * p.xb) + at0 * p.xs +
                       th.tile.first;
    const GT* from_g = static_cast<const GT*>(p.g) +
        (p.offsets ? th.row.first * p.gs : th.b * p.gb) + at0 * p.gs + th.tile.head;
    const VT* from_d = d + (th.row.first + at0) * p.C + th.tile.first;
    typename Th::template Pieces<VT> px, pd;
    typename Th::template Pieces<GT> pg;
    px.init(p, th, step_x);
    pd.init(p, th, step_c);
    pg.init(p, th, step_g);
    const bool whole_x = LN || p.x_bytes == 16, whole_d = LN || p.d_bytes == 16;
    const bool whole_g = PC && (LN || (p.D == 1 && p.g_bytes == 16));
    const unsigned shared = (unsigned)__cvta_generic_to_shared(mine);
    int issued = 0, slot_in = 0, slot = 0;      // (offsets of the tiles' places)
    auto issue = [&] {
        if (issued < n) {
            const int room = th.room(first - issued);
            if (whole_x) px.copy(shared + slot_in, from_x, room);
            else
                th.template copy_rows<VT, 2>(p, reinterpret_cast<VT*>(mine + slot_in), from_x, step_x,
                                             room, p.x_bytes);
            if (d != nullptr) {
                if (whole_d) pd.copy(shared + slot_in + S::kX, from_d, room);
                else
                    th.template copy_rows<VT, 2>(p, reinterpret_cast<VT*>(mine + slot_in + S::kX),
                                                 from_d, step_c, room, p.d_bytes);
            }
            if (whole_g) pg.copy(shared + slot_in + 2 * S::kX, from_g, room);
            else
                th.copy_gates(p, reinterpret_cast<GT*>(mine + slot_in + 2 * S::kX), from_g, step_g,
                              room);
            from_x -= th.chunk * step_x;
            from_d -= (int64_t)th.chunk * step_c;
            from_g -= th.chunk * step_g;
            slot_in = slot_in + stage == p.stages * stage ? 0 : slot_in + stage;
        }
        ++issued;
        copies_issued();
    };
    for (int i = 0; i < p.stages - 1; ++i) issue();
    const float* keep = kept + kept_index(p, th.row, th.b, th.chunk, first) * p.C + th.ch;
    F2 h_next = n > 0 ? th.get(keep) : two(0.f);
    F2 R = d_last != nullptr ? th.get(d_last + th.b * p.C + th.ch) : two(0.f);
    // what flows back into the last state of the tile
    R = th.ranges(p, pairs, R, true, &s_pair[0][0][0]);
    // (outputs are written from a stretch's last step to its first)
    const int64_t out0 = th.row.first + th.place(p, first * th.chunk + th.step0 + L - 1);
    VT* to_x = dx == nullptr ? nullptr : dx + out0 * p.C + th.ch;
    GT* to_g = dg == nullptr || (!(LN && PC) && p.D > 1) ? nullptr : dg + out0 * p.H + th.ch;
    const bool summed = !(LN && PC) && dg != nullptr && p.D > 1;
    for (int i = 0; i < n; ++i) {
        const int64_t k = first - i;
        issue();
        copies_wait(p.stages - 1);
        __syncwarp();
        const unsigned char* at = mine + slot;
        slot = slot + stage == p.stages * stage ? 0 : slot + stage;
        const VT* const tx = reinterpret_cast<const VT*>(at);
        const VT* const td = reinterpret_cast<const VT*>(at + S::kX);
        const GT* const tg = reinterpret_cast<const GT*>(at + 2 * S::kX);
        F2 h = h_next;
        keep -= p.C;
        if (i + 1 < n) h_next = th.get(keep);
        F2 a[L], w[L], A = two(1.f), B = two(0.f), E = two(0.f);
        auto scan = [&](auto weighted) {
#pragma unroll
            for (int l = 0; l < L; ++l) {
                th.template gates<decltype(weighted)::value>(tg, l, a[l], w[l]);
                const F2 v = th.at(tx, l);
                B = fma2(a[l], B, decltype(weighted)::value ? v : mul2(w[l], v));
                A = mul2(A, a[l]);
            }
        };
        if (p.weighted) scan(std::true_type{});
        else scan(std::false_type{});
        if (d != nullptr)
#pragma unroll
            for (int l = L - 1; l >= 0; --l) E = mul2(a[l], add2(E, th.at(td, l)));
        bool odd = spoilt(A, B) != 0.f || spoilt(E, E) != 0.f;
        keep_open<PC>(A, a);
        if (odd) {
            F2 al, ul;
            A = two(1.f);
            B = E = two(0.f);
#pragma unroll 1
            for (int l = 0; l < L; ++l) {
                th.step(p, tx, tg, l, al, ul, false);
                B = past2(al, B, ul);
                A = gates2(al, A);
            }
#pragma unroll 1
            for (int l = L - 1; l >= 0; --l) {
                th.step(p, d == nullptr ? nullptr : td, tg, l, al, ul, true);
                E = past2(al, add2(E, ul), two(0.f));
            }
        }
        F2 EA = A, TA, TB, TE, all_a;
        join_lanes<false, PC>(Th::lanes_of(p), th.lane, A, B, TA, TB);
        join_lanes<true, PC, false>(Th::lanes_of(p), th.lane, EA, E, all_a, TE);
        F2 G = R;
        if (Th::warps_of(p) == 1) {
            R = past2(TA, R, TE);
        } else {
            if (th.sub == 0) {
                s_pair[i & 1][th.warp][th.cl] = make_float4(TA.x, TA.y, TB.x, TB.y);
                s_flow[i & 1][th.warp][th.cl] = make_float2(TE.x, TE.y);
            }
            th.unit_sync(p);
            const float4* const all = &s_pair[i & 1][th.group * Th::warps_of(p)][th.cl];
            const float2* const flow = &s_flow[i & 1][th.group * Th::warps_of(p)][th.cl];
            const F2 h_before = h, R_before = R;
#pragma unroll 8
            for (int j = 0; j < Th::warps_of(p); ++j) {
                if (j >= th.wseg) break;
                const float4 q = all[j * 32];
                h = fma2({q.x, q.y}, h, {q.z, q.w});
            }
#pragma unroll 8
            for (int j = Th::warps_of(p) - 1; j >= 0; --j) {
                if (j == th.wseg) G = R;
                const float2 a2 = *reinterpret_cast<const float2*>(&all[j * 32]), e2 = flow[j * 32];
                R = fma2({a2.x, a2.y}, R, {e2.x, e2.y});
            }
            if (spoilt(h, R) != 0.f) {
                h = h_before;
                R = R_before;
                for (int j = 0; j < th.wseg; ++j) {
                    const float4 q = all[j * 32];
                    h = past2({q.x, q.y}, h, {q.z, q.w});
                }
                for (int j = Th::warps_of(p) - 1; j >= 0; --j) {
                    if (j == th.wseg) G = R;
                    const float4 q = all[j * 32];
                    const float2 e2 = flow[j * 32];
                    R = past2({q.x, q.y}, R, {e2.x, e2.y});
                }
            }
        }
        if (Th::lanes_of(p) < 32) {
            h = past2(A, h, B);
            G = past2(EA, G, E);
        }
        odd |= spoilt(h, G) != 0.f;
        const int64_t t0 = k * th.chunk + th.step0;
        const int mine = th.have == 0 || t0 >= th.row.len ? 0      // steps that this lane has
                         : t0 + L <= th.row.len ? L : (int)(th.row.len - t0);
        // (dg of a step goes where it belongs, or to the sums of its group)
        auto give = [&](int l, bool in, F2 wG, F2 one) {
            if (dx != nullptr && in) th.store(p, to_x - (int64_t)(L - 1 - l) * step_c, wG);
            if (to_g != nullptr) {
                if (in) th.store(p, to_g - (int64_t)(L - 1 - l) * step_h, one);
            } else if (!summed) {
            } else if (PC) {
                sums[l * S::kPitch + th.lane * 2] = one.x;
                sums[l * S::kPitch + th.lane * 2 + 1] = one.y;
            } else {
                sums[l * S::kPitch + th.lane] = one.x + one.y;
            }
        };
        auto unwind = [&](auto weighted) {
            constexpr bool WEIGHTED = decltype(weighted)::value;
            // forwards: what dg has besides the adjoint
            F2 q[L];
#pragma unroll
            for (int l = 0; l < L; ++l) {
                const F2 v = th.at(tx, l);
                q[l] = mul2(a[l], fma2(h, two(-1.f), WEIGHTED ? two(0.f) : v));
                h = fma2(a[l], h, WEIGHTED ? v : mul2(w[l], v));
            }
            // and back
#pragma unroll
            for (int l = L - 1; l >= 0; --l) {
                if (d != nullptr) G = add2(G, th.at(td, l));
                give(l, l < mine, WEIGHTED ? G : mul2(w[l], G),
                     mul2(q[l], G));
                G = mul2(a[l], G);
            }
        };
        if (odd) {
            F2 before[L], al, ul;
#pragma unroll 1
            for (int l = 0; l < L; ++l) {
                before[l] = h;
                th.step(p, tx, tg, l, al, ul, false);
                h = past2(al, h, ul);
            }
#pragma unroll 1
            for (int l = L - 1; l >= 0; --l) {
                F2 wl, v = th.at(tx, l), q;
                th.template gates<false>(tg, l, al, wl);
                if (p.weighted) wl = two(1.f);
                if (d != nullptr) G = add2(G, th.at(td, l));
                const F2 hb = before[l];
                // (a value that is not finite in a place of no thickness is no sample)
                if (wl.x == 0.f && !finite(v.x)) v.x = hb.x;
                if (wl.y == 0.f && !finite(v.y)) v.y = hb.y;
                q.x = al.x == 0.f ? 0.f : al.x * (p.weighted ? -hb.x : v.x - hb.x);
                q.y = al.y == 0.f ? 0.f : al.y * (p.weighted ? -hb.y : v.y - hb.y);
                // (nor has anything a gradient whose state has none)
                give(l, l < mine, mul2(wl, G), {times(G.x, q.x), times(G.y, q.y)});
                G = past2(al, G, two(0.f));
            }
        } else if (p.weighted) {
            unwind(std::true_type{});
        } else {
            unwind(std::false_type{});
        }
        if (to_x != nullptr) to_x -= (int64_t)th.chunk * step_c;
        if (to_g != nullptr) to_g -= (int64_t)th.chunk * step_h;
        if (summed) {
            __syncwarp();
            const int heads = p.parts > 1 ? 1 : th.tile.width / p.D, subs = 32 / Th::lanes_of(p);
            const int tasks = L * subs * heads;
            // a sum's terms: channels (PC), or pairs of them
            const int width = (p.parts > 1 ? th.tile.width : p.D) / (PC ? 1 : 2);
            const int row_of = PC ? Th::lanes_of(p) * 2 : Th::lanes_of(p);
            // few sums: several lanes to each
            const int share = tasks < 32 && (tasks & (tasks - 1)) == 0 ? 32 / tasks : 1;
            for (int j0 = 0; j0 < tasks; j0 += 32 / share) {
                const int j = j0 + th.lane / share;
                const int l = j / (subs * heads), r = j - l * (subs * heads);
                const int s = r / heads, hd = r - s * heads;
                float sum = 0.f;
                if (j < tasks) {
                    const float* from = sums + l * S::kPitch + s * row_of + hd * width;
                    for (int c = th.lane % share; c < width; c += share) sum += from[c];
                }
                for (int o = 1; o < share; o *= 2) sum += __shfl_xor_sync(~0u, sum, o);
                const int64_t t = k * th.chunk + (th.wseg * subs + s) * L + l;
                if (j >= tasks || t >= th.row.len || th.lane % share != 0) continue;
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
        if (th.wseg == 0 && th.sub == 0 && dh0 != nullptr)
            th.put(p, dh0 + th.b * p.C + th.ch, R);
    }
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
            const Gate gate = gate_of(to_float(g[at * p.gs + (c + v) / p.D]));
            h[v] = past(gate.a, h[v], times(p.weighted ? 1.f : gate.w, xv[v]));
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
