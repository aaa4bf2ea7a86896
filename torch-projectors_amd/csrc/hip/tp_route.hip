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

#include <algorithm>

namespace tp {
namespace {

// ------------------------------------------------------------------ sort
// A workgroup of W wavefronts sorts up to 64 W kGroups slots: each wavefront takes consecutive groups of 64, keeps
// their classes and their ranks among its own slots of that class in registers, and its counts per class in
// LDS.  Few slots are one workgroup's; of more, a first kernel counts each workgroup's stretch, and the last,
// knowing every stretch's counts, places it.  Up to some 10^5 slots bound by the chain of launches, counts and scans:
// 4096 slots 7 us, 65536 12.  Millions are bound by their bytes' way, not their number (1048576 24 us, 8388608 112,
// where 8 bytes in and 8 out are 20): ids are read twice, and `order` is written four bytes at a time.  (Loops over wavefronts' counts are not unrolled: instructions are fetched once
// per launch, and 4096 slots took 8.3 us with more loads on their way at once.)
constexpr int kGroups = 8, kMaxSortWaves = 16;

template <class I> __device__ __forceinline__ int class_of(const I* ids, int64_t i, int E) {
    const I c = ids[i];
    return c >= 0 && c < I(E) ? int(c) : E;
}

// Inclusive sum over the lanes up to this one.
__device__ __forceinline__ int wave_scan(int v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int u = __shfl_up(v, d);
        v += lane >= d ? u : 0;
    }
    return v;
}

// Places slots [i0, i1) (i1 - i0 at most 64 waves kGroups a turn; several turns where there are more).
// before: for each class the slots of earlier stretches, all: those of all stretches (null: there is one).
template <class I>
__global__ __launch_bounds__(64 * kMaxSortWaves) void k_sort_place(const I* __restrict__ ids, int64_t n, int64_t stretch,
                                                                   int E, const int* __restrict__ counts, int stretches,
                                                                   bool summed, int* __restrict__ order,
                                                                   int* __restrict__ slot, int* __restrict__ offsets) {
    extern __shared__ int lds[];
    const int C = E + 1, waves = blockDim.x >> 6, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    int* cnt = lds;               // [waves][C]: counts, then places of the wavefront's next slots
    int* base = lds + waves * C;  // [C]: place of the workgroup's next slot of a class
    __shared__ int wave_total[kMaxSortWaves];
    __shared__ int carry;
    const int64_t i0 = int64_t(blockIdx.x) * stretch, i1 = min(i0 + stretch, n);
    const int bits = 32 - __clz(E);

    // base: an exclusive scan of the classes' totals, plus what earlier stretches hold (one stretch: the scan
    // follows the counting below)
    auto scan_classes = [&](auto total, auto done) {
        if (tid == 0) carry = 0;
        for (int c0 = 0; c0 < C; c0 += int(blockDim.x)) {
            const int c = c0 + tid, t = c < C ? total(c) : 0, s = wave_scan(t);
            if (lane == 63) wave_total[wave] = s;
            __syncthreads();
            int at = carry + s - t;
            for (int w = 0; w < wave; ++w) at += wave_total[w];
            if (c < C) done(c, at);
            __syncthreads();
            if (tid == int(blockDim.x) - 1) carry = at + t;
            __syncthreads();
        }
    };
    if (counts) {
        scan_classes(
            [&](int c) {
                if (summed) {  // counts: [stretch][C] of earlier stretches' slots, then the totals
                    base[c] = counts[int64_t(blockIdx.x) * C + c];
                    return counts[int64_t(stretches) * C + c];
                }
                int earlier = 0, all = 0;
#pragma unroll 16
                for (int b = 0; b < stretches; ++b) {
                    const int v = counts[int64_t(b) * C + c];
                    all += v;
                    earlier += b < int(blockIdx.x) ? v : 0;
                }
                base[c] = earlier;
                return all;
            },
            [&](int c, int at) {
                base[c] += at;
                if (blockIdx.x == 0) offsets[c] = at;
            });
    }
    for (int64_t turn = i0; turn < i1 || turn == i0; turn += int64_t(waves) * 64 * kGroups) {
        for (int i = tid; i < waves * C; i += blockDim.x) cnt[i] = 0;
        __syncthreads();
        int cls[kGroups], rank[kGroups];
        int* mine = cnt + wave * C;
        const int64_t first = turn + int64_t(wave) * 64 * kGroups;
        // a short stretch is dealt to the wavefronts in equal shares
        const int groups = int(min(int64_t(kGroups), (i1 - turn + 64 * waves - 1) / (64 * waves)));
        const int64_t start = groups == kGroups ? first : turn + int64_t(wave) * 64 * groups;
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            const int64_t i = start + g * 64 + lane;
            cls[g] = g < groups && i < i1 ? class_of(ids, i, E) : -1;
        }
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            if (g >= groups) break;
            const int c = cls[g];
            uint64_t same = __ballot(c >= 0);
            if (c >= 0) {
                for (int b = 0; b < bits; ++b) {
                    const uint64_t set = __ballot((c >> b) & 1);
                    same &= (c >> b) & 1 ? set : ~set;
                }
                const int old = mine[c];
                rank[g] = old + __popcll(same & ((uint64_t(1) << lane) - 1));
                // the last lane of each class counts on, after all lanes have read
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                if (lane == 63 - __clzll(same)) mine[c] = rank[g] + 1;
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            }
        }
        __syncthreads();
        auto to_places = [&](int c, int at) {  // wavefronts' counts of class c to their first places
            for (int w = 0; w < waves; ++w) {
                const int t = cnt[w * C + c];
                cnt[w * C + c] = at;
                at += t;
            }
            return at;
        };
        if (counts) {
            for (int c = tid; c < C; c += blockDim.x) base[c] = to_places(c, base[c]);
            __syncthreads();
        } else {
            scan_classes(
                [&](int c) {
                    int t = 0;
                    for (int w = 0; w < waves; ++w) t += cnt[w * C + c];
                    return t;
                },
                [&](int c, int at) {
                    offsets[c] = at;
                    to_places(c, at);
                });
        }
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            if (g >= groups || cls[g] < 0) continue;
            const int64_t i = start + g * 64 + lane;
            const int place = mine[cls[g]] + rank[g];
            order[place] = int(i);
            slot[i] = place;
        }
        __syncthreads();
    }
}

// counts[b][c]: slots of class c in stretch b.
template <class I>
__global__ __launch_bounds__(1024) void k_sort_count(const I* __restrict__ ids, int64_t n, int64_t stretch, int E,
                                                     int* __restrict__ counts) {
    extern __shared__ int lds[];
    const int C = E + 1;
    for (int c = threadIdx.x; c < C; c += blockDim.x) lds[c] = 0;
    __syncthreads();
    const int64_t i1 = min(int64_t(blockIdx.x + 1) * stretch, n);
    for (int64_t i = int64_t(blockIdx.x) * stretch + threadIdx.x; i < i1; i += blockDim.x)
        atomicAdd(&lds[class_of(ids, i, E)], 1);  // (a count: in any order the same)
    __syncthreads();
    for (int c = threadIdx.x; c < C; c += blockDim.x) counts[int64_t(blockIdx.x) * C + c] = lds[c];
}

// Many stretches: their counts to the sums of earlier ones, and the totals after them.  64 classes a workgroup, whose
// wavefronts take consecutive stretches.
__global__ __launch_bounds__(1024) void k_sort_sum(int* __restrict__ counts, int stretches, int C) {
    __shared__ int part[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;
    const int b0 = int(int64_t(stretches) * wave / 16), b1 = int(int64_t(stretches) * (wave + 1) / 16);
    int sum = 0;
    if (c < C)
        for (int b = b0; b < b1; ++b) sum += counts[int64_t(b) * C + c];
    part[wave][lane] = sum;
    __syncthreads();
    if (c >= C) return;
    int at = 0;
    for (int w = 0; w < wave; ++w) at += part[w][lane];
    for (int b = b0; b < b1; ++b) {
        const int v = counts[int64_t(b) * C + c];
        counts[int64_t(b) * C + c] = at;
        at += v;
    }
    if (wave == 15) counts[int64_t(stretches) * C + c] = at;
}

// Wavefronts of the placing workgroups (LDS holds a count per class for each), the slots of each workgroup, and
// whether the counts are summed by a kernel of their own or by every workgroup for itself.  Measured: one workgroup
// or several, 4096 slots of 16 classes 7.6 and 8.0 us, 6000 of 64 10.4 and 9.2, 8192 of 1000 16.4 and 11.6; 16
// stretches with their own sums or 64 summed, 16384 slots of 64 classes 10.2 and 10.5, 32768 11.1 and 10.9, 65536
// 13.4 and 11.8, 131072 of 4096 classes (64 stretches) 157 and 35.
struct SortPlan {
    int waves, stretches;
    int64_t stretch;
    bool summed;
};
SortPlan sort_plan(int64_t n, int E) {
    int waves = E <= 1024 ? kMaxSortWaves : 4;
    const int64_t group = int64_t(waves) * 64, hold = group * kGroups;
    if (n <= std::min<int64_t>(hold, 4096)) {
        while (waves > 1 && int64_t(waves / 2) * 64 >= n) waves /= 2;
        return {waves, 1, std::max<int64_t>(n, 1), false};
    }
    const bool summed = n > 32768 || E > 1024;
    // equal stretches, or as many of a whole turn as there are, or 2048 of several turns
    const int64_t count = summed ? 64 : 16, turns = (n + hold - 1) / hold, each = (turns + 2047) / 2048;
    const int64_t stretch = turns <= count ? ((n + count - 1) / count + group - 1) / group * group : each * hold;
    return {waves, int((n + stretch - 1) / stretch), stretch, summed};
}

template <class I>
hipError_t sort(const I* ids, int64_t n, int E, int* order, int* slot, int* offsets, int* counts, hipStream_t s) {
    const SortPlan p = sort_plan(n, E);
    const int C = E + 1;
    if (p.stretches > 1) {
        k_sort_count<I><<<p.stretches, 1024, C * sizeof(int), s>>>(ids, n, p.stretch, E, counts);
        if (p.summed) k_sort_sum<<<(C + 63) / 64, 1024, 0, s>>>(counts, p.stretches, C);
        if (hipError_t e = hipGetLastError()) return e;
    }
    const size_t lds = size_t(p.waves + 1) * C * sizeof(int);
    if (lds > 65536)
        if (hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&k_sort_place<I>),
                                               hipFuncAttributeMaxDynamicSharedMemorySize, int(lds)))
            return e;
    k_sort_place<I><<<p.stretches, 64 * p.waves, lds, s>>>(ids, n, p.stretch, E, p.stretches > 1 ? counts : nullptr,
                                                           p.stretches, p.summed, order, slot, offsets);
    return hipGetLastError();
}

// ------------------------------------------------------------------ rows
// Both directions go by rows, not places: W wavefronts take a row (or a stretch of it), whose k places they know,
// so that the row is read (spread) or written (gather) once whatever k is.  Memory bound: 16384 x 4 rows of 4096
// bfloat16 spread in 120 us (5.6 TB/s), gathered in 114 (5.9).  Values move 16 bytes a
// lane at a time, whatever the rows' alignment; of up to KB choices the loads are in flight together, and the
// products for the weights' gradient stay in registers.  More than KB choices: spread goes over the row again for
// each KB of them (four at once are faster than eight: 16384 x 8 rows of 512 bfloat16 65 against 84 us with the
// weights' gradient), gather reads KB at a time and does the products in a second look (so there KB is up to eight:
// 48 against 69 us).  Spread without that gradient has two stretches of the row on their way, gather where a row has one or
// two choices (2048 x 2 rows of 4224 fp32 23.1 and 23.4 us, so 21.7 and 21.0; 65536 x 2 of 300 58 and 53, so 51 and 42; but
// gathers of four choices, 16384 x 4 of 4096 bfloat16, 120 us and 126).
template <class S> struct Values {
    static constexpr int n = Pack<S>::n;
    float v[n];
};
template <class S> __device__ __forceinline__ Values<S> load_values(const typename S::Bits* p, int64_t left, bool stream) {
    Values<S> r;
    if (left >= Values<S>::n) {
        const Pack<S> w = stream ? stream_pack<S>(p) : load_pack<S>(p);
#pragma unroll
        for (int i = 0; i < Values<S>::n; ++i) r.v[i] = S::widen(w.v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < Values<S>::n; ++i) r.v[i] = i < left ? S::widen(p[i]) : 0.0f;
    }
    return r;
}
template <class S>
__device__ __forceinline__ void store_values(typename S::Bits* p, int64_t left, const Values<S>& r, bool stream) {
    Pack<S> w;
#pragma unroll
    for (int i = 0; i < Values<S>::n; ++i) w.v[i] = S::round(r.v[i]);
    if (left >= Values<S>::n) {
        if (stream) stream_pack<S>(p, w);
        else store_pack<S>(p, w);
    } else {
#pragma unroll
        for (int i = 0; i < Values<S>::n; ++i)
            if (i < left) p[i] = w.v[i];
    }
}

// The places of KB choices of a row and what they weigh.
template <int KB> struct Places {
    int64_t at[KB];  // first value of the row there
    float w[KB];
    bool in[KB], real[KB];  // is not dropped; is a choice at all
    bool held[KB];          // is a choice with a place among the sorted rows
};
template <int KB>
__device__ __forceinline__ Places<KB> places_of(const RouteArgs& a, int64_t t, int j0, int kept) {
    Places<KB> p;
#pragma unroll
    for (int u = 0; u < KB; ++u) {
        const int64_t s = t * a.k + j0 + u;
        p.real[u] = j0 + u < a.k;
        const uint32_t at = p.real[u] ? uint32_t(a.slot[s]) : 0u, last = uint32_t(a.T * a.k) - 1u;
        p.held[u] = p.real[u] && at <= last;
        p.in[u] = p.held[u] && at < uint32_t(kept);
        p.at[u] = int64_t(min(at, last)) * a.D;  // (read where `in`)
        p.w[u] = p.real[u] && a.weights ? a.weights[s] : 1.0f;
    }
    return p;
}
// For writing: a choice without a place, of an order from elsewhere, writes what another one of these writes, to the
// same place (zeros at the last place would meet the row that has it; a branch for each store makes the loads ahead wait
// for the stores, 16384 x 4 rows of 4096 bfloat16 141 us, so 120; a path of its own takes registers from the other one,
// 16384 x 8 of 512 with the weights' gradient 72 us, so 59; what it costs, 2048 x 2 of 4224 fp32 with that gradient 37.1
// us, 35.8 without it, otherwise at most 2 %).  False where none has a place.
template <int KB> __device__ __forceinline__ bool placed(Places<KB>& p) {
    bool any = true;
#pragma unroll
    for (int u = 0; u < KB; ++u) any = any && p.held[u] == p.real[u];
    if (any) return true;  // (the weights are not waited for)
    bool in = false;
    int64_t at = 0;
    float w = 0.0f;
#pragma unroll
    for (int u = 0; u < KB; ++u)
        if (p.held[u]) any = true, in = p.in[u], at = p.at[u], w = p.w[u];
#pragma unroll
    for (int u = 0; u < KB; ++u)
        if (!p.held[u]) p.in[u] = in, p.at[u] = at, p.w[u] = w;
    return any;
}

// Sums of the W wavefronts of a row, the same in all of them.
template <int W, int KB> __device__ __forceinline__ void row_sums(float (&v)[KB], float (*lds)[KB]) {
#pragma unroll
    for (int u = 0; u < KB; ++u) v[u] = wave_sum(v[u]);
    if (W == 1) return;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
        for (int u = 0; u < KB; ++u) lds[threadIdx.x >> 6][u] = v[u];
    __syncthreads();
#pragma unroll
    for (int u = 0; u < KB; ++u) {
        v[u] = lds[0][u];
#pragma unroll
        for (int w = 1; w < W; ++w) v[u] += lds[w][u];
    }
    __syncthreads();
}

// W wavefronts per item: a workgroup of 256 with four items (W = 1), or one item of W wavefronts.  An item is a
// stretch of `span` values of a row; `parts` of them are a row (one with DOT).
template <int W> constexpr int row_block() { return W == 1 ? 256 : 64 * W; }
struct RowItem {
    int64_t t, d0, d1;
};
template <int W> __device__ __forceinline__ bool row_item(const RouteArgs& a, int64_t item0, int64_t span, int parts, RowItem& r) {
    const int64_t item = item0 + (W == 1 ? __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6)) : 0);
    if (item >= a.T * parts) return false;
    r.t = parts == 1 ? item : over(item, parts);
    r.d0 = (item - r.t * parts) * span;
    r.d1 = min(r.d0 + span, a.D);
    return true;
}

template <class S, int W, int KB, bool DOT>
__global__ __launch_bounds__(row_block<W>()) void k_spread_rows(RouteArgs a, int64_t span, int parts, bool stream,
                                                                const typename S::Bits* __restrict__ x,
                                                                typename S::Bits* __restrict__ sorted,
                                                                const typename S::Bits* __restrict__ rows,
                                                                float* __restrict__ d_weights) {
    constexpr int n = Values<S>::n, items = W == 1 ? 4 : 1, step = W * 64 * n, U = DOT ? 1 : 2;
    __shared__ float lds[W][KB];
    const int kept = *a.kept, lane = W == 1 ? threadIdx.x & 63 : threadIdx.x;
    for (int64_t item0 = int64_t(blockIdx.x) * items; item0 < a.T * parts; item0 += int64_t(gridDim.x) * items) {
        RowItem r;
        if (!row_item<W>(a, item0, span, parts, r)) break;
        for (int j0 = 0; j0 < a.k; j0 += KB) {
            Places<KB> p = places_of<KB>(a, r.t, j0, kept);
            const int64_t end = placed(p) ? r.d1 : r.d0;
            float dot[KB] = {};
            for (int64_t d0 = r.d0 + lane * n; d0 < end; d0 += U * step) {
                Values<S> v[U];
#pragma unroll
                for (int e = 0; e < U; ++e)
                    v[e] = load_values<S>(x + r.t * a.D + d0 + e * step, r.d1 - d0 - e * step, stream && a.k <= KB);
#pragma unroll
                for (int e = 0; e < U; ++e) {
                    const int64_t d = d0 + e * step, left = r.d1 - d;
                    if (left <= 0) break;
                    Values<S> o[KB];
                    if (DOT) {
#pragma unroll
                        for (int u = 0; u < KB; ++u) {
                            if (p.in[u]) o[u] = load_values<S>(rows + p.at[u] + d, left, stream);
                            else o[u] = Values<S>{};
                        }
#pragma unroll
                        for (int u = 0; u < KB; ++u)
                            if (p.in[u])
#pragma unroll
                                for (int i = 0; i < n; ++i) dot[u] = __builtin_fmaf(v[e].v[i], o[u].v[i], dot[u]);
                    }
#pragma unroll
                    for (int u = 0; u < KB; ++u) {
                        if (!p.real[u]) continue;
#pragma unroll
                        for (int i = 0; i < n; ++i) o[u].v[i] = p.in[u] ? p.w[u] * v[e].v[i] : 0.0f;
                        store_values<S>(sorted + p.at[u] + d, left, o[u], stream);
                    }
                }
            }
            if (DOT) {
                row_sums<W, KB>(dot, lds);
                if (lane == 0)
#pragma unroll
                    for (int u = 0; u < KB; ++u)
                        if (p.real[u]) d_weights[r.t * a.k + j0 + u] = p.held[u] ? dot[u] : 0.0f;
            }
        }
    }
}

template <class S, int W, int KB, bool DOT>
__global__ __launch_bounds__(row_block<W>()) void k_gather_rows(RouteArgs a, int64_t span, int parts, bool stream,
                                                                const typename S::Bits* __restrict__ rows,
                                                                typename S::Bits* __restrict__ out,
                                                                const typename S::Bits* __restrict__ x,
                                                                float* __restrict__ d_weights) {
    constexpr int n = Values<S>::n, items = W == 1 ? 4 : 1, step = W * 64 * n, U = 2;
    __shared__ float lds[W][KB];
    const int kept = a.k ? *a.kept : 0, lane = W == 1 ? threadIdx.x & 63 : threadIdx.x;
    for (int64_t item0 = int64_t(blockIdx.x) * items; item0 < a.T * parts; item0 += int64_t(gridDim.x) * items) {
        RowItem r;
        if (!row_item<W>(a, item0, span, parts, r)) break;
        Places<KB> p = places_of<KB>(a, r.t, 0, kept);
        float dot[KB] = {};
        constexpr bool two = !DOT && KB == 2;  // stretches at once (the row has no more choices then)
        if (two)
            for (int64_t d0 = r.d0 + lane * n; d0 < r.d1; d0 += U * step) {
                Values<S> o[U][KB];
#pragma unroll
                for (int e = 0; e < U; ++e)
#pragma unroll
                    for (int u = 0; u < KB; ++u) {
                        if (p.in[u]) o[e][u] = load_values<S>(rows + p.at[u] + d0 + e * step, r.d1 - d0 - e * step, stream);
                        else o[e][u] = Values<S>{};
                    }
#pragma unroll
                for (int e = 0; e < U; ++e) {
                    const int64_t d = d0 + e * step, left = r.d1 - d;
                    if (left <= 0) break;
                    Values<S> sum{};
#pragma unroll
                    for (int u = 0; u < KB; ++u)
                        if (p.in[u])
#pragma unroll
                            for (int i = 0; i < n; ++i) sum.v[i] += p.w[u] * o[e][u].v[i];
                    store_values<S>(out + r.t * a.D + d, left, sum, stream);
                }
            }
        for (int64_t d = two ? r.d1 : r.d0 + lane * n; d < r.d1; d += step) {
            const int64_t left = r.d1 - d;
            Values<S> sum{}, v{}, o[KB];
            for (int j0 = 0; j0 < a.k; j0 += KB) {
                if (a.k > KB) p = places_of<KB>(a, r.t, j0, kept);
#pragma unroll
                for (int u = 0; u < KB; ++u) {
                    if (p.in[u]) o[u] = load_values<S>(rows + p.at[u] + d, left, stream);
                    else o[u] = Values<S>{};
                }
                if (DOT && a.k <= KB) v = load_values<S>(x + r.t * a.D + d, left, stream);
#pragma unroll
                for (int u = 0; u < KB; ++u)
                    if (p.in[u])
#pragma unroll
                        for (int i = 0; i < n; ++i) {
                            sum.v[i] += p.w[u] * o[u].v[i];
                            if (DOT) dot[u] = __builtin_fmaf(v.v[i], o[u].v[i], dot[u]);
                        }
            }
            store_values<S>(out + r.t * a.D + d, left, sum, stream);
        }
        if (!DOT) continue;
        for (int j0 = 0; j0 < a.k; j0 += KB) {
            if (a.k > KB) {
                p = places_of<KB>(a, r.t, j0, kept);
#pragma unroll
                for (int u = 0; u < KB; ++u) dot[u] = 0.0f;
                for (int64_t d = r.d0 + lane * n; d < r.d1; d += step) {
                    const int64_t left = r.d1 - d;
                    const Values<S> v = load_values<S>(x + r.t * a.D + d, left, stream);
#pragma unroll
                    for (int u = 0; u < KB; ++u) {
                        if (!p.in[u]) continue;
                        const Values<S> o = load_values<S>(rows + p.at[u] + d, left, stream);
#pragma unroll
                        for (int i = 0; i < n; ++i) dot[u] = __builtin_fmaf(v.v[i], o.v[i], dot[u]);
                    }
                }
            }
            row_sums<W, KB>(dot, lds);
            if (lane == 0)
#pragma unroll
                for (int u = 0; u < KB; ++u)
                    if (j0 + u < a.k) d_weights[r.t * a.k + j0 + u] = dot[u];
        }
    }
}

// Sorted rows of at least this size, what the XCDs' L2s hold together, are streamed past the caches.  Which side is the
// faster one depends on what a program does around the call, too.  Measured, streamed and through the caches, us: inputs
// and outputs that were not in the caches (many in turn), weighted spread and gather of 2048 x 2 rows of 2112 fp32 (35
// MB) 13.4 and 14.8, 11.7 and 13.1, of 4224 (69 MB) 24 and 27, 20 and 24, 16384 x 4 of 1024 bfloat16 (134 MB) 33.5 and
// 34.5, 34 and 39, 9000 x 2 of 2560 fp32 (184 MB) 52 and 54, 47 and 53; the same input again and again, 69 MB 23 and 17,
// 18 and 17, 184 MB 51 and 49, 45 and 43, 268 MB and more: streamed or equal; a spread, a pass over the sorted rows and a
// gather, 35 MB 36.4 and 36.2, 69 MB 65 and 63, 105 MB 101 and 97, 134 MB 100 and 105, 268 MB 204 and 214, 537 MB 430 and
// 450.  Against it: 65536 x 2 rows of 300 fp32 (157 MB), spread 59 and 54 (of 200, 33 and 38).
constexpr int64_t kStreamBytes = int64_t(32) << 20;

// Wavefronts of a row: one while a row is at most 2.5 KB, else 4 (16384 x 2 rows of 2560 bytes: spread 25.3 us by one,
// 26.1 by four, with the weights' gradient 38 and 44; of 4096 bytes 45 and 35, 66 and 58).
// With fewer than 2048 of them a row is cut into stretches for 2048 (100 x 2 rows of 66560 bytes, spread, whole and cut: 13.3
// and 6.4 us; 500 x 2 of 8448 5.0 and 4.7, 1000 x 4 of 2500 7.2 and 6.3, but 2000 x 2 of 8448, already 8000
// wavefronts, 12.8 and 14.1).
// The weights' gradient needs whole rows.  It takes 4 wavefronts for short rows that are fewer than 1024 (spread by one
// and four: 512 x 2 of 2500 bytes 5.3 and 4.1 us, 1024 4.8 and 5.1 of 1800, 6.1 and 5.6 of 2500, 2000 6.3 and 8.1, 7.8 and
// 8.5), and 16 for long rows of which each has a CU of its own (by four and 16: 64 x 2 of 4400 bytes 4.3 and 4.0, of
// 2800 3.6 and 3.8; 256 x 2 of 8448 5.8 and 5.2, 300 6.2 and 8.3), beyond 32 KB up to two a CU (512 x 2 of 33280 21.8
// and 20.1, of 24000 13.2 and 14.4; 700 of 33280 26.7 and 27.3).  Gathering more than four choices, which 16 wavefronts
// do four at a time and fewer eight, pays for 16 beyond 16 KB only (64 x 8 of 8448 12.7 and 13.1, of 16896 23.7 and 20.4;
// 300 of 66560 104 and 154).
struct RowPlan {
    int waves, parts;
    int64_t span;
};
RowPlan row_plan(const RouteArgs& a, int size, bool spread, bool dot) {
    const int64_t bytes = a.D * size;
    RowPlan p{bytes <= 2560 ? 1 : 4, 1, a.D};
    if (bytes <= 1024) return p;
    if (dot) {
        const int64_t long_row = spread || a.k <= 4 ? (a.T <= 256 ? 4096 : 32768) : 16384;
        if (bytes <= 2560) p.waves = a.T < 1024 ? 4 : 1;
        else if (a.T <= (spread || a.k <= 4 ? 512 : 256) && bytes > long_row) p.waves = 16;
        return p;
    }
    if (a.T * p.waves >= 2048) return p;
    p.waves = 1;
    const int64_t want = (2048 + a.T - 1) / a.T, step = 1024 / size;  // a wavefront's values at once
    p.span = ((a.D + want - 1) / want + step - 1) / step * step;
    p.parts = int((a.D + p.span - 1) / p.span);
    return p;
}

#define TP_ROWS_DOT(kernel, W, KB) \
    kernel<S, W, KB, true><<<grid, row_block<W>(), 0, s>>>(a, p.span, p.parts, stream, in, to, other, d_weights)
#define TP_ROWS(kernel, W, KB)                                                                                       \
    (dot ? TP_ROWS_DOT(kernel, W, KB)                                                                                \
         : kernel<S, W, KB, false><<<grid, row_block<W>(), 0, s>>>(a, p.span, p.parts, stream, in, to, nullptr, nullptr))
#define TP_ROWS_16(kernel) (a.k <= 2 ? TP_ROWS_DOT(kernel, 16, 2) : TP_ROWS_DOT(kernel, 16, 4))  // (by the gradient only)
#define TP_ROWS_BY_K(kernel, W) (a.k <= 2 ? TP_ROWS(kernel, W, 2) : TP_ROWS(kernel, W, 4))

template <class S, bool SPREAD>
hipError_t move_rows(const RouteArgs& a, const void* in_, void* to_, const void* other_, float* d_weights, hipStream_t s) {
    using B = typename S::Bits;
    const auto* in = static_cast<const B*>(in_);
    auto* to = static_cast<B*>(to_);
    const auto* other = static_cast<const B*>(other_);
    const bool dot = d_weights != nullptr;
    const RowPlan p = row_plan(a, sizeof(B), SPREAD, dot);
    const int64_t items = a.T * p.parts;
    const bool stream = a.T * a.k * a.D * int64_t(sizeof(B)) >= kStreamBytes;
    const unsigned grid = match_grid(p.waves == 1 ? (items + 3) / 4 : items);
    if (SPREAD) {
        if (p.waves == 1) TP_ROWS_BY_K(k_spread_rows, 1);
        else if (p.waves == 4) TP_ROWS_BY_K(k_spread_rows, 4);
        else TP_ROWS_16(k_spread_rows);
    } else if (dot && a.k > 4) {
        if (p.waves == 1) TP_ROWS_DOT(k_gather_rows, 1, 8);
        else if (p.waves == 4) TP_ROWS_DOT(k_gather_rows, 4, 8);
        else TP_ROWS_DOT(k_gather_rows, 16, 4);  // (8 do not fit its registers)
    } else {
        if (p.waves == 1) TP_ROWS_BY_K(k_gather_rows, 1);
        else if (p.waves == 4) TP_ROWS_BY_K(k_gather_rows, 4);
        else TP_ROWS_16(k_gather_rows);
    }
    return hipGetLastError();
}
#undef TP_ROWS
#undef TP_ROWS_DOT
#undef TP_ROWS_16
#undef TP_ROWS_BY_K

}  // namespace

int64_t sort_by_class_work(int64_t slots, int64_t classes) {
    const SortPlan p = sort_plan(slots, int(classes));
    return p.stretches > 1 ? (int64_t(p.stretches) + 1) * (classes + 1) * int64_t(sizeof(int)) : 0;
}

hipError_t launch_sort_by_class(int id_bytes, const void* ids, int64_t slots, int E, int* order, int* slot,
                                int* offsets, void* work, hipStream_t s) {
    auto* counts = static_cast<int*>(work);
    return id_bytes == 4 ? sort(static_cast<const int32_t*>(ids), slots, E, order, slot, offsets, counts, s)
                         : sort(static_cast<const int64_t*>(ids), slots, E, order, slot, offsets, counts, s);
}

hipError_t launch_spread_rows(const RouteArgs& a, const void* x, void* sorted, const void* rows, float* d_weights,
                              hipStream_t s) {
    switch (a.dt) {
        case TP_F32: return move_rows<F32, true>(a, x, sorted, rows, d_weights, s);
        case TP_F16: return move_rows<F16, true>(a, x, sorted, rows, d_weights, s);
        default: return move_rows<BF16, true>(a, x, sorted, rows, d_weights, s);
    }
}

hipError_t launch_gather_rows(const RouteArgs& a, const void* rows, void* out, const void* x, float* d_weights,
                              hipStream_t s) {
    switch (a.dt) {
        case TP_F32: return move_rows<F32, false>(a, rows, out, x, d_weights, s);
        case TP_F16: return move_rows<F16, false>(a, rows, out, x, d_weights, s);
        default: return move_rows<BF16, false>(a, rows, out, x, d_weights, s);
    }
}

}  // namespace tp
