// Rows sorted by class and back (the dispatch and combination around per-class
// work: each class's projections, or any per-expert product).
//
//   sort     a stable counting sort of N = T k slots by class id.  Ids outside [0, E) come after all
//            others.  A slot's place is its class's offset plus the earlier slots of its class; within a
//            wavefront "earlier" is a population count over the lanes with the same id (found by one
//            ballot per id bit), between wavefronts and workgroups a prefix sum of counts, so the result
//            does not depend on any order of execution.
//   spread   sorted[slot[t, j]] = w[t, j] x[t]
//   gather   out[t] = sum_j w[t, j] rows[slot[t, j]], j ascending in fp32, rounded once
//
// spread and gather are each other's adjoints, and both can add the gradient of the weights,
// <x[t], rows[slot[t, j]]>, for rows that they read anyway.
#include "../../../include/torch_projectors_hip.h"
#include "tp_match.hh"

namespace tp {
namespace {

// ------------------------------------------------------------------ sort
constexpr int kSortWaves = 4;

template <class I> __device__ __forceinline__ int class_of(const I* ids, int64_t i, int E) {
    const I c = ids[i];
    return c >= 0 && c < I(E) ? int(c) : E;
}

// One workgroup sorts all slots: counts per wavefront, their prefix sums in (class, wavefront) order, places.
template <class I>
__global__ __launch_bounds__(64 * kSortWaves) void k_sort_one(const I* __restrict__ ids, int n, int E,
                                                              int* __restrict__ order, int* __restrict__ slot,
                                                              int* __restrict__ offsets) {
    extern __shared__ int cnt[];  // [kSortWaves][E + 1], then [E + 1] of totals
    int* total = cnt + kSortWaves * (E + 1);
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int groups = (n + 63) / 64, per = (groups + kSortWaves - 1) / kSortWaves;
    const int g0 = wave * per, g1 = min(g0 + per, groups);
    int* mine = cnt + wave * (E + 1);
    for (int i = tid; i < kSortWaves * (E + 1); i += 64 * kSortWaves) cnt[i] = 0;
    __syncthreads();
    for (int g = g0; g < g1; ++g) {
        const int i = g * 64 + lane;
        if (i < n) atomicAdd(&mine[class_of(ids, i, E)], 1);
    }
    __syncthreads();
    for (int c = tid; c <= E; c += 64 * kSortWaves) {
        int t = 0;
        for (int w = 0; w < kSortWaves; ++w) t += cnt[w * (E + 1) + c];
        total[c] = t;
    }
    __syncthreads();
    if (tid == 0) {
        int at = 0;
        for (int c = 0; c <= E; ++c) {
            const int t = total[c];
            total[c] = at;
            at += t;
        }
    }
    __syncthreads();
    for (int c = tid; c <= E; c += 64 * kSortWaves) {
        int at = total[c];
        offsets[c] = at;
        for (int w = 0; w < kSortWaves; ++w) {
            const int t = cnt[w * (E + 1) + c];
            cnt[w * (E + 1) + c] = at;
            at += t;
        }
    }
    __syncthreads();
    const int bits = 32 - __clz(E);
    for (int g = g0; g < g1; ++g) {
        const int i = g * 64 + lane;
        const bool in = i < n;
        const int c = in ? class_of(ids, i, E) : -1;
        uint64_t same = __ballot(in);
        for (int b = 0; b < bits; ++b) {
            const uint64_t set = __ballot((c >> b) & 1);
            same &= (c >> b) & 1 ? set : ~set;
        }
        if (in) {
            const int place = mine[c] + __popcll(same & ((uint64_t(1) << lane) - 1));
            order[place] = i;
            slot[i] = place;
            // the last lane of each class moves its counter on, after all lanes have read it
            __builtin_amdgcn_wave_barrier();
            if (lane == 63 - __clzll(same)) mine[c] = place + 1;
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// ------------------------------------------------------------------ rows
constexpr int kRowBlock = 256;

__device__ __forceinline__ float block_sum(float v, float* lds) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    float t = 0;
    for (int w = 0; w < kRowBlock / 64; ++w) t += lds[w];
    return t;
}

// One workgroup per row.
template <class S, bool DOT>
__global__ __launch_bounds__(kRowBlock) void k_spread_rows(RouteArgs a, const typename S::Bits* __restrict__ x,
                                                           typename S::Bits* __restrict__ sorted,
                                                           const typename S::Bits* __restrict__ rows,
                                                           float* __restrict__ d_weights) {
    __shared__ float lds[kRowBlock / 64];
    const int kept = *a.kept;
    for (int64_t t = blockIdx.x; t < a.T; t += gridDim.x)
    for (int j = 0; j < a.k; ++j) {
        const int at = a.slot[t * a.k + j];
        const bool in = at < kept;
        const float w = a.weights ? a.weights[t * a.k + j] : 1.0f;
        float dot = 0;
        for (int64_t d = threadIdx.x; d < a.D; d += kRowBlock) {
            const float v = S::widen(x[t * a.D + d]);
            sorted[int64_t(at) * a.D + d] = S::round(in ? w * v : 0.0f);
            if (DOT) dot += in ? v * S::widen(rows[int64_t(at) * a.D + d]) : 0.0f;
        }
        if (DOT) {
            dot = block_sum(dot, lds);
            if (threadIdx.x == 0) d_weights[t * a.k + j] = dot;
        }
    }
}

template <class S, bool DOT>
__global__ __launch_bounds__(kRowBlock) void k_gather_rows(RouteArgs a, const typename S::Bits* __restrict__ rows,
                                                           typename S::Bits* __restrict__ out,
                                                           const typename S::Bits* __restrict__ x,
                                                           float* __restrict__ d_weights) {
    __shared__ float lds[kRowBlock / 64];
    const int kept = a.k ? *a.kept : 0;
    for (int64_t t = blockIdx.x; t < a.T; t += gridDim.x) {
    for (int64_t d = threadIdx.x; d < a.D; d += kRowBlock) {
        float sum = 0;
        for (int j = 0; j < a.k; ++j) {
            const int at = a.slot[t * a.k + j];
            if (at >= kept) continue;
            const float w = a.weights ? a.weights[t * a.k + j] : 1.0f;
            sum += w * S::widen(rows[int64_t(at) * a.D + d]);
        }
        out[t * a.D + d] = S::round(sum);
    }
    if (DOT)
        for (int j = 0; j < a.k; ++j) {
            const int at = a.slot[t * a.k + j];
            float dot = 0;
            if (at < kept)
                for (int64_t d = threadIdx.x; d < a.D; d += kRowBlock)
                    dot += S::widen(x[t * a.D + d]) * S::widen(rows[int64_t(at) * a.D + d]);
            dot = block_sum(dot, lds);
            if (threadIdx.x == 0) d_weights[t * a.k + j] = dot;
        }
    }
}

template <class S>
hipError_t spread(const RouteArgs& a, const void* x, void* sorted, const void* rows, float* d_weights, hipStream_t s) {
    using B = typename S::Bits;
    const dim3 grid(match_grid(a.T));
    if (d_weights)
        k_spread_rows<S, true><<<grid, kRowBlock, 0, s>>>(a, static_cast<const B*>(x), static_cast<B*>(sorted),
                                                          static_cast<const B*>(rows), d_weights);
    else
        k_spread_rows<S, false><<<grid, kRowBlock, 0, s>>>(a, static_cast<const B*>(x), static_cast<B*>(sorted),
                                                           nullptr, nullptr);
    return hipGetLastError();
}

template <class S>
hipError_t gather(const RouteArgs& a, const void* rows, void* out, const void* x, float* d_weights, hipStream_t s) {
    using B = typename S::Bits;
    const dim3 grid(match_grid(a.T));
    if (d_weights)
        k_gather_rows<S, true><<<grid, kRowBlock, 0, s>>>(a, static_cast<const B*>(rows), static_cast<B*>(out),
                                                          static_cast<const B*>(x), d_weights);
    else
        k_gather_rows<S, false><<<grid, kRowBlock, 0, s>>>(a, static_cast<const B*>(rows), static_cast<B*>(out),
                                                           nullptr, nullptr);
    return hipGetLastError();
}

}  // namespace

int64_t sort_by_class_work(int64_t, int64_t) { return 0; }

hipError_t launch_sort_by_class(int id_bytes, const void* ids, int64_t slots, int E, int* order, int* slot,
                                int* offsets, void*, hipStream_t s) {
    const size_t lds = size_t(kSortWaves + 1) * (E + 1) * sizeof(int);
    const void* f = id_bytes == 4 ? reinterpret_cast<const void*>(&k_sort_one<int32_t>)
                                  : reinterpret_cast<const void*>(&k_sort_one<int64_t>);
    if (lds > 65536)
        if (hipError_t e = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, int(lds))) return e;
    if (id_bytes == 4)
        k_sort_one<int32_t><<<1, 64 * kSortWaves, lds, s>>>(static_cast<const int32_t*>(ids), int(slots), E, order,
                                                            slot, offsets);
    else
        k_sort_one<int64_t><<<1, 64 * kSortWaves, lds, s>>>(static_cast<const int64_t*>(ids), int(slots), E, order,
                                                            slot, offsets);
    return hipGetLastError();
}

hipError_t launch_spread_rows(const RouteArgs& a, const void* x, void* sorted, const void* rows, float* d_weights,
                              hipStream_t s) {
    switch (a.dt) {
        case TP_F32: return spread<F32>(a, x, sorted, rows, d_weights, s);
        case TP_F16: return spread<F16>(a, x, sorted, rows, d_weights, s);
        default: return spread<BF16>(a, x, sorted, rows, d_weights, s);
    }
}

hipError_t launch_gather_rows(const RouteArgs& a, const void* rows, void* out, const void* x, float* d_weights,
                              hipStream_t s) {
    switch (a.dt) {
        case TP_F32: return gather<F32>(a, rows, out, x, d_weights, s);
        case TP_F16: return gather<F16>(a, rows, out, x, d_weights, s);
        default: return gather<BF16>(a, rows, out, x, d_weights, s);
    }
}

}  // namespace tp
