// C-ABI entry points of the quantised leaf records (see include/svox_b200.h).
#include "records.cuh"

#include <type_traits>

#include "status.h"

namespace svoxb {

int status_of_records(int clear, int* word) {
    SVOXB_CUDA(cudaMemcpyFromSymbol(word, g_status, sizeof(int)));
    if (clear && *word != 0) {
        const int zero = 0;
        SVOXB_CUDA(cudaMemcpyToSymbol(g_status, &zero, sizeof(int)));
    }
    return SVOXB_OK;
}

namespace {

int validate(const svoxb_records* r, const float* points, const int64_t* ids, int64_t Q, int type) {
    if (!r || !r->records) return SVOXB_ERR_NULL;
    if (r->K < 2 || r->group < 1 || r->M < 1 || r->N < 2 || r->N > 16 || Q < 0)
        return SVOXB_ERR_SHAPE;
    if (r->code_type != SVOXB_CODE_INT8 && r->code_type != SVOXB_CODE_E4M3)
        return SVOXB_ERR_FORMAT;
    if (type != SVOXB_TYPE_F32 && type != SVOXB_TYPE_BF16 && type != SVOXB_TYPE_F16)
        return SVOXB_ERR_FORMAT;
    if (r->K > SVOXB_RECORDS_MAX_K || Q >= 0xffffffffLL) return SVOXB_ERR_TOO_LARGE;
    if (Q == 0) return SVOXB_OK;
    if (points && ids) return SVOXB_ERR_OPTION;
    if (!points && !ids && Q > r->M * r->N * r->N * r->N) return SVOXB_ERR_SHAPE;
    if (points && (!r->child || !r->offset || !r->scaling)) return SVOXB_ERR_NULL;
    return SVOXB_OK;
}

RecordArgs args_of(const svoxb_records* r) {
    RecordArgs a{};
    a.records = static_cast<uint8_t*>(r->records);
    a.owner = r->owner;
    a.child = r->child;
    a.offset = r->offset;
    a.scaling = r->scaling;
    a.M = r->M;
    a.N = r->N;
    a.slots = r->M * r->N * r->N * r->N;
    a.K = r->K;
    a.group = r->group;
    a.bytes = record_bytes(r->K, r->group);
    return a;
}

// The jump table of the query (see launch_query): a quarter as many cells as there are points.
int build_top(const svoxb_records* r, int64_t Q, TopScratch* top, cudaStream_t stream) {
    int level = 0;
    while (level < 7 && Q >= (int64_t)4 << (3 * (level + 1))) ++level;
    if (level < 5) return SVOXB_OK;
    svoxb_tree t{};
    t.child = r->child;
    t.M = r->M;
    t.N = r->N;
    return top->build(&t, level, stream);
}

template <class T> struct Of { using type = T; };
template <class F>
int with_type(int type, F f) {
    switch (type) {
        case SVOXB_TYPE_F32: return f(Of<float>{});
        case SVOXB_TYPE_BF16: return f(Of<__nv_bfloat16>{});
        default: return f(Of<__half>{});
    }
}

// Calls f with the floats of a record and its group, if the compiler knows that layout.
template <int N> using Int = std::integral_constant<int, N>;
template <class F>
bool with_layout(const RecordArgs& a, F f) {
    if (a.K == 4 && a.group == 1) f(Int<4>{}, Int<1>{});
    else if (a.K == 4 && a.group == 3) f(Int<4>{}, Int<3>{});
    else if (a.K == 13 && a.group == 4) f(Int<13>{}, Int<4>{});
    else if (a.K == 28 && a.group == 9) f(Int<28>{}, Int<9>{});
    else if (a.K == 49 && a.group == 16) f(Int<49>{}, Int<16>{});
    else if (a.K == 76 && a.group == 25) f(Int<76>{}, Int<25>{});
    else return false;
    return true;
}

template <class Kernel>
int ready(Kernel kernel, int block, size_t smem) {
    int per_sm = 0;
    return blocks_per_sm(reinterpret_cast<const void*>(kernel), block, smem, &per_sm);
}

template <class T, bool E4M3>
int launch_read(const RecordArgs& a, const TopTable& top, const float* points, const int64_t* ids,
                int64_t Q, T* out, cudaStream_t stream) {
    const unsigned grid = (unsigned)((Q + kRecordsBlock - 1) / kRecordsBlock);
    int st = SVOXB_OK;
    const bool known = with_layout(a, [&](auto k, auto g) {
        auto kernel = records_read_known<T, E4M3, decltype(k)::value, decltype(g)::value>;
        constexpr size_t smem = (size_t)kRecordsBlock / 32 *
                                read_stage<T, decltype(k)::value, decltype(g)::value>();
        if ((st = ready(kernel, kRecordsBlock, smem))) return;
        kernel<<<grid, kRecordsBlock, smem, stream>>>(a, top, points, ids, Q, out);
    });
    if (st) return st;
    if (!known) {
        int per = 32;
        while (per * a.bytes > kRecordStage && per > 1) per /= 2;
        const size_t smem = (size_t)kRecordsBlock / 32 * per * a.bytes;
        records_read_kernel<T, E4M3><<<grid, kRecordsBlock, smem, stream>>>(a, top, points, ids, Q,
                                                                           out, per);
    }
    SVOXB_CUDA(cudaGetLastError());
    return SVOXB_OK;
}

template <class T, bool E4M3>
int launch_write(const RecordArgs& a, const int64_t* found, int64_t Q, const T* values,
                 cudaStream_t stream) {
    int st = SVOXB_OK;
    const bool known = with_layout(a, [&](auto k, auto g) {
        auto kernel = records_write_known<T, E4M3, decltype(k)::value, decltype(g)::value>;
        const size_t smem = (size_t)kWriteBlock * a.K * sizeof(T);
        if ((st = ready(kernel, kWriteBlock, smem))) return;
        kernel<<<(unsigned)((Q + kWriteBlock - 1) / kWriteBlock), kWriteBlock, smem, stream>>>(
            a, found, Q, values);
    });
    if (st) return st;
    if (!known) {
        int per = 32;
        while ((per * a.bytes > kRecordStage || per * a.K * (int)sizeof(T) > kValueStage) && per > 1)
            per /= 2;
        const unsigned grid = (unsigned)((Q + kRecordsBlock - 1) / kRecordsBlock);
        const size_t warp = per * a.bytes + stepped((size_t)per * a.K * sizeof(T), 16);
        auto kernel = records_write_kernel<T, E4M3>;
        const size_t smem = kRecordsBlock / 32 * warp;
        if ((st = ready(kernel, kRecordsBlock, smem))) return st;
        kernel<<<grid, kRecordsBlock, smem, stream>>>(a, found, Q, values, per);
    }
    SVOXB_CUDA(cudaGetLastError());
    return SVOXB_OK;
}

}  // namespace
}  // namespace svoxb

using namespace svoxb;

extern "C" {

int svoxb_record_bytes(int32_t K, int32_t group) {
    if (K < 2 || group < 1 || K > SVOXB_RECORDS_MAX_K) return -1;
    return record_bytes(K, group);
}

int svoxb_records_read(const svoxb_records* r, const float* points, const int64_t* ids, int64_t Q,
                       void* out, int32_t out_type, void* stream) {
    int st = validate(r, points, ids, Q, out_type);
    if (st || Q == 0) return st;
    if (!out) return SVOXB_ERR_NULL;
    const auto str = static_cast<cudaStream_t>(stream);
    TopScratch top;
    if (points && (st = build_top(r, Q, &top, str))) return st;
    const TopTable tt{top.cells, top.level};
    const RecordArgs a = args_of(r);
    return with_type(out_type, [&](auto t) {
        using T = typename decltype(t)::type;
        return r->code_type == SVOXB_CODE_E4M3
                   ? launch_read<T, true>(a, tt, points, ids, Q, static_cast<T*>(out), str)
                   : launch_read<T, false>(a, tt, points, ids, Q, static_cast<T*>(out), str);
    });
}

int svoxb_records_write(const svoxb_records* r, const float* points, const int64_t* ids, int64_t Q,
                        const void* values, int32_t values_type, int64_t* found, void* stream) {
    int st = validate(r, points, ids, Q, values_type);
    if (st || Q == 0) return st;
    const bool all = !points && !ids;           // row q is record q: nothing to find or claim
    if (!values || (!all && (!found || !r->owner))) return SVOXB_ERR_NULL;
    const auto str = static_cast<cudaStream_t>(stream);
    TopScratch top;
    if (points && (st = build_top(r, Q, &top, str))) return st;
    const RecordArgs a = args_of(r);
    if (all) found = nullptr;
    else
        records_claim_kernel<<<(unsigned)((Q + kRecordsBlock - 1) / kRecordsBlock), kRecordsBlock,
                               0, str>>>(a, TopTable{top.cells, top.level}, points, ids, Q, found);
    SVOXB_CUDA(cudaGetLastError());
    return with_type(values_type, [&](auto t) {
        using T = typename decltype(t)::type;
        const T* v = static_cast<const T*>(values);
        return r->code_type == SVOXB_CODE_E4M3 ? launch_write<T, true>(a, found, Q, v, str)
                                               : launch_write<T, false>(a, found, Q, v, str);
    });
}

}  // extern "C"
