// Leaf records held in 8 bits: quantised as they are written, scaled back as they are read.
//
// A record of K floats becomes K - 1 codes, one exponent for every `group` neighbouring ones (a
// colour channel's coefficients), and the last float, the density, as fp16:
//   value = code * 2^(exponent - 127)
// The scale is the smallest power of two that leaves the group's largest magnitude at most 127 after
// rounding (int8), or at most 448 (e4m3): every product with it is exact, so a code is off by at most
// half a step of its own type and nothing else, and reading into 16-bit floats loses nothing.  What
// that costs against a scale with a mantissa is at most one of int8's seven bits.  An exponent of
// 255 with codes of 0 stands for a group with a value that is not finite: it reads as NaN.  The
// density keeps 11 bits, those a checkpoint file keeps of every value.
//
// Records are as long as their sectors: 32 bytes for SH9 (27 + 3 + 2 to the byte), 64 for SH16, 80
// for SH25 where floats take 112, 196 and 304.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"

namespace svoxb {

constexpr int kRecordsBlock = 256;
constexpr int kRecordStage = 4096;      // bytes of records a warp has under way
constexpr int kValueStage = 8192;       // bytes of values it has

// Groups of a record, and its length: codes, exponents, then the density in its last two bytes.
__host__ __device__ constexpr int record_groups(int K, int group) {
    return (K - 1 + group - 1) / group;
}
__host__ __device__ constexpr int record_bytes(int K, int group) {
    const int raw = K - 1 + record_groups(K, group) + 2;
    return raw <= 8 ? 8 : (raw + 15) / 16 * 16;
}

struct RecordArgs {
    uint8_t* records;
    uint32_t* owner;            // row + 1 of the last row for a slot, while a write is under way
    const int32_t* child;
    const float* offset;
    const float* scaling;
    int64_t M, slots;
    int32_t N, K, group, bytes;
};

__device__ __forceinline__ int64_t locate(const RecordArgs& r, const TopTable& top,
                                          const float* __restrict__ points,
                                          const int64_t* __restrict__ ids, int64_t i) {
    if (points == nullptr) {
        if (ids == nullptr) return i;
        const int64_t s = __ldg(ids + i);
        if (s >= 0 && s < r.slots) return s;
        report(SVOXB_ERR_INDEX);
        return -1;
    }
    const float px = to_tree(__ldg(points + 3 * i), __ldg(r.offset), __ldg(r.scaling));
    const float py = to_tree(__ldg(points + 3 * i + 1), __ldg(r.offset + 1), __ldg(r.scaling + 1));
    const float pz = to_tree(__ldg(points + 3 * i + 2), __ldg(r.offset + 2), __ldg(r.scaling + 2));
    LeafHit hit;
    const bool ok = r.N == 2 ? descend2(r.child, r.M, top, px, py, pz, hit)
                             : descendN(r.child, r.M, r.N, px, py, pz, hit);
    return ok ? hit.slot : -1;
}

template <class T> __device__ __forceinline__ T as_type(float v);
template <> __device__ __forceinline__ float as_type<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 as_type<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}
template <> __device__ __forceinline__ __half as_type<__half>(float v) {
    return __float2half_rn(v);
}
__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }

template <bool E4M3>
__device__ __forceinline__ float code_value(uint8_t code) {
    if (!E4M3) return (float)(int8_t)code;
    __nv_fp8_e4m3 c;
    c.__x = code;
    return (float)c;
}
template <bool E4M3>
__device__ __forceinline__ uint8_t code_of(float v) {
    if (!E4M3) return (uint8_t)(int8_t)__float2int_rn(v);
    return __nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
}
// Exponent of a group from the bits of its largest magnitude (those of floats order like integers).
template <bool E4M3>
__device__ __forceinline__ int exponent_of(uint32_t most) {
    if (most >= 0x7f800000u) return 255;
    const int m = (int)(most & 0x7fffffu);
    const int e = (int)(most >> 23) - (E4M3 ? 8 : 6) + (E4M3 ? m > 0x600000 : m >= 0x7f0000);
    return e < 1 ? 1 : e;
}

// Copies `until` records between their places and the warp's stage, 16 bytes a lane (8 where a
// record is no longer).
template <bool IN>
__device__ __forceinline__ void move_records(const RecordArgs& r, uint8_t* stage, int64_t slot,
                                             bool there, int first, int until, int lane) {
    const int piece = r.bytes < 16 ? 8 : 16, pieces = r.bytes / piece;
    const int all = until * pieces;
    for (int base = 0; base < all; base += 32) {
        const int j = base + lane;
        const int k = j < all ? j / pieces : 0;
        const int64_t s = __shfl_sync(0xffffffffu, slot, first + k);
        const bool t = __shfl_sync(0xffffffffu, there, first + k);
        if (j >= all || !t) continue;
        uint8_t* const here = stage + j * piece;
        uint8_t* const far = r.records + s * r.bytes + (j - k * pieces) * piece;
        if (IN) {
            const unsigned a = (unsigned)__cvta_generic_to_shared(here);
            if (piece == 16)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(a), "l"(far)
                             : "memory");
            else
                asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(a), "l"(far)
                             : "memory");
        } else if (piece == 16) {
            *reinterpret_cast<uint4*>(far) = *reinterpret_cast<const uint4*>(here);
        } else {
            *reinterpret_cast<uint2*>(far) = *reinterpret_cast<const uint2*>(here);
        }
    }
    if (IN) asm volatile("cp.async.wait_all;" ::: "memory");
    __syncwarp();
}

// Records of any layout: a code to a lane.
template <class T, bool E4M3>
__global__ void __launch_bounds__(kRecordsBlock)
records_read_kernel(RecordArgs r, TopTable top, const float* __restrict__ points,
                    const int64_t* __restrict__ ids, int64_t Q, T* __restrict__ out, int per) {
    extern __shared__ __align__(16) uint8_t s_stage[];
    const int64_t i = (int64_t)blockIdx.x * kRecordsBlock + threadIdx.x;
    const int lane = threadIdx.x & 31;
    const int64_t slot = i < Q ? locate(r, top, points, ids, i) : -1;
    const int64_t wb = i - lane;
    if (wb >= Q) return;
    const int K = r.K, group = r.group;
    uint8_t* const mine = s_stage + (threadIdx.x >> 5) * per * r.bytes;
    const int n = (int)(Q - wb < 32 ? Q - wb : 32);
    const unsigned found = __ballot_sync(0xffffffffu, slot >= 0);
    for (int first = 0; first < n; first += per) {
        const int until = n - first < per ? n - first : per;
        move_records<true>(r, mine, slot, slot >= 0, first, until, lane);
        T* const to = out + (wb + first) * K;
        for (int f = lane; f < until * K; f += 32) {
            const int k = f / K, c = f - k * K;
            const uint8_t* const rec = mine + k * r.bytes;
            float v;
            if (c == K - 1)
                v = __half2float(*reinterpret_cast<const __half*>(rec + r.bytes - 2));
            else
                v = code_value<E4M3>(rec[c]) *
                    __uint_as_float((uint32_t)rec[K - 1 + c / group] << 23);
            // (no such record: not a number)
            if (!(found >> (first + k) & 1)) v = __uint_as_float(0x7fc00000u);
            to[f] = as_type<T>(v);
        }
        __syncwarp();
    }
}

// First half of a write: the leaf of each row, and the last row of each leaf.
static __global__ void __launch_bounds__(kRecordsBlock)
records_claim_kernel(RecordArgs r, TopTable top, const float* __restrict__ points,
                     const int64_t* __restrict__ ids, int64_t Q, int64_t* __restrict__ found) {
    const int64_t i = (int64_t)blockIdx.x * kRecordsBlock + threadIdx.x;
    if (i >= Q) return;
    const int64_t s = locate(r, top, points, ids, i);
    found[i] = s;
    if (s >= 0) atomicMax(r.owner + s, (uint32_t)(i + 1));
}

// Second half: the rows that are their leaves' last are quantised and written, and their claims
// withdrawn (a row that finds no claim any more is not its leaf's last either).
template <class T, bool E4M3>
__global__ void __launch_bounds__(kRecordsBlock)
records_write_kernel(RecordArgs r, const int64_t* __restrict__ found, int64_t Q,
                     const T* __restrict__ values, int per) {
    extern __shared__ __align__(16) uint8_t s_stage[];
    const int64_t i = (int64_t)blockIdx.x * kRecordsBlock + threadIdx.x;
    const int lane = threadIdx.x & 31;
    // (without `found` row q is record q)
    const int64_t slot = i >= Q ? -1 : found != nullptr ? found[i] : i;
    const bool wins = slot >= 0 && (found == nullptr || r.owner[slot] == (uint32_t)(i + 1));
    const int64_t wb = i - lane;
    if (wb >= Q) return;
    const int K = r.K, groups = record_groups(K, r.group);
    const int values_bytes = (per * K * (int)sizeof(T) + 15) / 16 * 16;
    uint8_t* const stage = s_stage + (threadIdx.x >> 5) * (per * r.bytes + values_bytes);
    T* const rows = reinterpret_cast<T*>(stage + per * r.bytes);
    const int n = (int)(Q - wb < 32 ? Q - wb : 32);
    const unsigned winners = __ballot_sync(0xffffffffu, wins);
    for (int first = 0; first < n; first += per) {
        const int until = n - first < per ? n - first : per;
        for (int f = lane; f < until * K; f += 32)
            if (winners >> (first + f / K) & 1) rows[f] = values[(wb + first) * K + f];
        __syncwarp();
        for (int task = lane; task < until * groups; task += 32) {
            const int k = task / groups, j = task - k * groups;
            const int c0 = j * r.group, c1 = c0 + r.group < K - 1 ? c0 + r.group : K - 1;
            const T* const row = rows + k * K;
            uint8_t* const rec = stage + k * r.bytes;
            uint32_t most = 0;
            for (int c = c0; c < c1; ++c) {
                const uint32_t m = __float_as_uint(as_float(row[c])) & 0x7fffffffu;
                most = m > most ? m : most;
            }
            const int e = exponent_of<E4M3>(most);
            const float scale = __uint_as_float((uint32_t)(254 - e) << 23);
            for (int c = c0; c < c1; ++c)
                rec[c] = e == 255 ? 0 : code_of<E4M3>(as_float(row[c]) * scale);
            rec[K - 1 + j] = (uint8_t)e;
            if (j == 0) {
                for (int b = K - 1 + groups; b < r.bytes - 2; ++b) rec[b] = 0;
                *reinterpret_cast<__half*>(rec + r.bytes - 2) =
                    __float2half_rn(as_float(row[K - 1]));
            }
        }
        __syncwarp();
        move_records<false>(r, stage, slot, wins, first, until, lane);
    }
    if (wins && found != nullptr) r.owner[slot] = 0;
}

// ---------------------------------------------------------------------------
// Records whose layout the compiler knows (those of the colour bases, and plain colours): a lane has
// a whole record in its registers, where every code finds its exponent without an index, and rows of
// floats pass through shared memory only to meet memory as one stretch per warp.  Rows begin K words
// apart there: for odd K lanes never meet in a bank, for K of whole 16-byte words the eight lanes of
// a request do not.  Before, with a code to a lane, index arithmetic made 55 instructions of every 32
// values read and 64 of those written: 2^20 SH9 records in 61 and 76 us, 2^22 SH16 records in 356.
template <int K, int G, bool E4M3>
struct Record {
    static constexpr int NG = record_groups(K, G), R = record_bytes(K, G), WORDS = R / 4;
    uint32_t w[WORDS];

    // Bytes between records in shared memory: eight lanes that load 16 bytes each meet in no bank.
    static constexpr int kPitch = R == 32 || R == 64 ? R + 16 : R;

    __device__ __forceinline__ void load(const uint8_t* from) {
        if constexpr (R == 8) {
            const uint2 q = *reinterpret_cast<const uint2*>(from);
            w[0] = q.x, w[1 % WORDS] = q.y;
        } else
#pragma unroll
        for (int i = 0; i < R / 16; ++i) {
            const uint4 q = *(reinterpret_cast<const uint4*>(from) + i);
            w[4 * i] = q.x, w[(4 * i + 1) % WORDS] = q.y;
            w[(4 * i + 2) % WORDS] = q.z, w[(4 * i + 3) % WORDS] = q.w;
        }
    }
    __device__ __forceinline__ void store(uint8_t* to) const {
        if constexpr (R == 8)
            *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1 % WORDS]);
        else
#pragma unroll
        for (int i = 0; i < R / 16; ++i)
            reinterpret_cast<uint4*>(to)[i] = make_uint4(w[4 * i], w[(4 * i + 1) % WORDS],
                                                         w[(4 * i + 2) % WORDS],
                                                         w[(4 * i + 3) % WORDS]);
    }
    __device__ __forceinline__ uint32_t byte(int i) const { return w[i / 4] >> (i % 4 * 8) & 0xff; }
    __device__ __forceinline__ float scale(int g) const {
        return __uint_as_float(byte(K - 1 + g) << 23);
    }
    // Codes c and c + 1 as floats (c even).
    __device__ __forceinline__ float2 codes(int c) const {
        const uint32_t v = w[c / 4];
        if (E4M3) {
            const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(
                (__nv_fp8x2_storage_t)(c % 4 ? v >> 16 : v & 0xffff), __NV_E4M3);
            return __half22float2(*reinterpret_cast<const __half2*>(&h));
        }
        // (2^23 + code + 128) - (2^23 + 128)
        const uint32_t u = v ^ 0x80808080u;
        const float a = __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7650 | c % 4));
        const float b = __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7650 | c % 4 + 1));
        return make_float2(a - 8388736.f, b - 8388736.f);
    }
    __device__ __forceinline__ float density() const {
        return __half2float(__ushort_as_half((unsigned short)(w[WORDS - 1] >> 16)));
    }
};

// Four neighbouring elements at once where rows are of whole 16-byte words.
template <class T> struct __align__(4 * sizeof(T)) Quad { T v[4]; };

// Shared memory of a reading warp: its records, then half of its rows.
template <class T, int K, int G>
__host__ __device__ constexpr int read_stage() {
    const int in = 32 * Record<K, G, false>::kPitch, out = 16 * K * (int)sizeof(T);
    return in > out ? in : out;
}

template <class T, bool E4M3, int K, int G>
__global__ void __launch_bounds__(kRecordsBlock, K <= 49 ? 6 : 5)
records_read_known(RecordArgs r, TopTable top, const float* __restrict__ points,
                   const int64_t* __restrict__ ids, int64_t Q, T* __restrict__ out) {
    extern __shared__ __align__(16) uint8_t s_stage[];
    const int64_t i = (int64_t)blockIdx.x * kRecordsBlock + threadIdx.x;
    const int lane = threadIdx.x & 31;
    const int64_t wb = i - lane;
    if (wb >= Q) return;
    using Rec = Record<K, G, E4M3>;
    Rec rec;
    const int64_t slot = i < Q ? locate(r, top, points, ids, i) : -1;
    uint8_t* const stage = s_stage + (threadIdx.x >> 5) * read_stage<T, K, G>();
    if constexpr (Rec::R == 8) {
        rec.load(r.records + (slot < 0 ? 0 : slot) * 8);
    } else {
        // The records come by the warp, a few whole lines to a request, and then to their lanes (from
        // the lanes themselves, every request touched 32 lines: 310 -> 270 us for 2^22 SH16 records).
        constexpr int PIECES = Rec::R / 16;
#pragma unroll
        for (int j = 0; j < PIECES; ++j) {
            const int k = (lane + 32 * j) / PIECES, piece = (lane + 32 * j) % PIECES;
            const int64_t s = __shfl_sync(0xffffffffu, slot, k);
            if (s >= 0)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                                 (unsigned)__cvta_generic_to_shared(stage + k * Rec::kPitch +
                                                                    16 * piece)),
                             "l"(r.records + s * Rec::R + 16 * piece) : "memory");
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncwarp();
        rec.load(stage + lane * Rec::kPitch);
        __syncwarp();
    }
    // (half of the warp's rows at a time: what they take of the shared memory decides how many warps
    // wait for their points side by side)
    constexpr int ROWS = 16, PER = 16 / sizeof(T), WHOLE = ROWS * K / PER;
    T* const rows = reinterpret_cast<T*>(stage);
    T* const mine = rows + (lane % ROWS) * K;
    const int n = (int)(Q - wb < 32 ? Q - wb : 32);
    const bool aligned = (reinterpret_cast<uintptr_t>(out) & 15) == 0;
#pragma unroll 1
    for (int first = 0; first < n; first += ROWS) {
        // (decoded in either round anew: kept for both, K floats a lane would fill the registers)
#pragma unroll
        for (int j = 0; j < rec.WORDS; ++j) asm volatile("" : "+r"(rec.w[j]));
        if (lane / ROWS == first / ROWS) {
            float v[4];
#pragma unroll
            for (int c = 0; c < K; ++c) {
                if (c == K - 1) {
                    v[c % 4] = rec.density();
                } else {
                    const float2 q = rec.codes(c & ~1);
                    v[c % 4] = (c % 2 ? q.y : q.x) * rec.scale(c / G);
                }
                if (K % 4 != 0) {
                    mine[c] = as_type<T>(slot < 0 ? __uint_as_float(0x7fc00000u) : v[c % 4]);
                } else if (c % 4 == 3) {
                    Quad<T> four;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        four.v[j] = as_type<T>(slot < 0 ? __uint_as_float(0x7fc00000u) : v[j]);
                    *reinterpret_cast<Quad<T>*>(mine + c - 3) = four;
                }
            }
        }
        __syncwarp();
        // (16 rows are a whole number of 16-byte words)
        T* const to = out + (wb + first) * K;
        const int left = (n - first < ROWS ? n - first : ROWS) * K;
        if (aligned && left == ROWS * K) {
#pragma unroll
            for (int f = 0; f < WHOLE; f += 32)
                if (f + lane < WHOLE)
                    reinterpret_cast<uint4*>(to)[f + lane] =
                        reinterpret_cast<const uint4*>(rows)[f + lane];
        } else {
            for (int f = lane; f < left; f += 32) to[f] = rows[f];
        }
        __syncwarp();
    }
}

constexpr int kWriteBlock = 128;
template <class T, bool E4M3, int K, int G>
__global__ void __launch_bounds__(kWriteBlock)
records_write_known(RecordArgs r, const int64_t* __restrict__ found, int64_t Q,
                    const T* __restrict__ values) {
    extern __shared__ __align__(16) uint8_t s_stage[];
    const int64_t i = (int64_t)blockIdx.x * kWriteBlock + threadIdx.x;
    const int lane = threadIdx.x & 31;
    const int64_t wb = i - lane;
    if (wb >= Q) return;
    T* const rows = reinterpret_cast<T*>(s_stage) + (threadIdx.x >> 5) * 32 * K;
    const T* const from = values + wb * K;
    const int n = (int)(Q - wb < 32 ? Q - wb : 32) * K;
    constexpr int PER = 16 / sizeof(T);
    if ((reinterpret_cast<uintptr_t>(values) & 15) == 0) {
#pragma unroll 4
        for (int f = lane; f < n / PER; f += 32)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                             (unsigned)__cvta_generic_to_shared(rows + f * PER)),
                         "l"(from + f * PER) : "memory");
        if (lane < n % PER) rows[n / PER * PER + lane] = from[n / PER * PER + lane];
    } else {
        for (int f = lane; f < n; f += 32) rows[f] = from[f];
    }
    // (without `found` row q is record q)
    const int64_t slot = i >= Q ? -1 : found != nullptr ? found[i] : i;
    const bool wins = slot >= 0 && (found == nullptr ||
                                    atomicCAS(r.owner + slot, (uint32_t)(i + 1), 0u) ==
                                        (uint32_t)(i + 1));
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncwarp();
    if (!wins) return;
    const T* const mine = rows + lane * K;
    auto value = [&](int c) { return as_float(mine[c]); };
    Record<K, G, E4M3> rec;
#pragma unroll
    for (int j = 0; j < rec.WORDS; ++j) rec.w[j] = 0;
#pragma unroll
    for (int g = 0; g < rec.NG; ++g) {
        const int c0 = g * G, c1 = c0 + G < K - 1 ? c0 + G : K - 1;
        uint32_t most = 0;
#pragma unroll
        for (int c = c0; c < c1; ++c) {
            const uint32_t m = __float_as_uint(value(c)) & 0x7fffffffu;
            most = m > most ? m : most;
        }
        const int e = exponent_of<E4M3>(most);
        // (a group with a value that is not finite: codes of 0)
        const float scale = e == 255 ? 0.f : __uint_as_float((uint32_t)(254 - e) << 23);
        const uint32_t keep = e == 255 ? 0 : 0xff;
#pragma unroll
        for (int c = c0; c < c1; ++c) {
            uint32_t code;
            if (E4M3)
                code = __nv_cvt_float_to_fp8(value(c) * scale, __NV_SATFINITE, __NV_E4M3);
            else        // rounded to an integer by a sum whose last place is 1
                code = __float_as_uint(fmaf(value(c), scale, 12582912.f));
            rec.w[c / 4] |= (code & keep) << (c % 4 * 8);
        }
        rec.w[(K - 1 + g) / 4] |= (uint32_t)e << ((K - 1 + g) % 4 * 8);
    }
    rec.w[rec.WORDS - 1] |= (uint32_t)__half_as_ushort(__float2half_rn(value(K - 1))) << 16;
    rec.store(r.records + slot * rec.R);
}

}  // namespace svoxb
