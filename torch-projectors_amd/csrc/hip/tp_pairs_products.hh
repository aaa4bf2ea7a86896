// The tiled products of the pair log probabilities for one storage type (included by tp_pairs_*.hip).
//
// 4096 x 36864 bfloat16 pairs of 4224 values: 1230 us for the scores and their statistics (1.04 PFLOP/s), 1440 formed again for G in five pieces, 2880
// for the references' gradients and 3220 for the images' (0.89 and 0.79 PFLOP/s, each with both pieces of G).  The matrix units are 36 to 50 % busy;
// wavefronts wait 35 to 45 % of their time at a step's barrier, for loads and for each other, and nothing else is on the CU to fill that.
// 2048 x 8192 float32 pairs of 4224: 720, 717, 816 and 797 us (174 to 198 TFLOP/s of six products each).  Matrix instructions (52 to 61 %) and
// those that cut values into pieces (34 %) take nearly all of the SIMDs' time between them.
// A product has both its operands in one type: G goes through 16-bit units in two pieces, what rounding it leaves being the second.  With the first alone
// bfloat16 gradients are 2.3e-3 off, and 1.7e-3 with both, which is their own rounding.
#pragma once

#include "tp_pairs.hh"
#include "tp_tile.hh"

#include <type_traits>

namespace tp {
namespace {

// What a reference adds to its scores, in LDS: score = min(sum c + add, limit), where the limit of one that is ruled out
// is -inf, whatever its sum is (the minimum with a NaN is the other), and that of the others +inf (a NaN becomes
// +inf, which makes its image's results NaN all the same).  -inf is no score of an allowed reference: max(sum c + add, -limit) is -inf
// for those that are -inf or NaN, and for no other.
struct alignas(8) Offset {
    float add, limit;
};
__device__ __forceinline__ bool ruled_out(const PairOff& o, int64_t n) {
    return (o.mask && !o.mask[n]) || (o.bias && o.bias[n] == -INFINITY);
}
template <class T> __device__ __forceinline__ void tile_offsets(const PairOff& o, int64_t first, Offset* off) {
    for (int i = threadIdx.x; i < T::BM; i += T::NT) {
        const int64_t n = first + i;
        const float b = n >= o.N || ruled_out(o, n) ? -INFINITY : o.bias ? o.bias[n] : 0.0f;
        off[i] = b == -INFINITY ? Offset{0.0f, -INFINITY} : Offset{times(b, o.c), INFINITY};
    }
}
__device__ __forceinline__ float score(float sum, const Offset& o, float c) { return fminf(fmaf(sum, c, o.add), o.limit); }
__device__ __forceinline__ float lowest_of(float sum, const Offset& o, float c) { return fmaxf(fmaf(sum, c, o.add), -o.limit); }
__device__ __forceinline__ float exp_of(float z) { return __builtin_amdgcn_exp2f(z * kLog2e); }
__device__ __forceinline__ float base_of(float most) { return most == -INFINITY ? 0.0f : most; }

// A lane holds 16 FM references of each of its FN images: their maximum and sum in registers, then over the two
// halves of the wavefront and the WM wavefronts.
struct StatsEpi {
    using Args = StatsOut;
    template <class S> static constexpr bool kTwice = false;
    template <class S, class T>
    static __device__ __forceinline__ void run(const Args& g, Acc<T>& acc, uint32_t im, uint32_t in, char* lds) {
        const int tid = threadIdx.x;
        const Place<T> place(tid);
        const int64_t n0 = int64_t(im) * T::BM, m0 = int64_t(in) * T::BN;
        Offset* off = reinterpret_cast<Offset*>(lds);
        ScorePart* part = reinterpret_cast<ScorePart*>(off + T::BM);  // [WM][BN]
        tile_offsets<T>(g.off, n0, off);
        float most[T::FN], least[T::FN], sum[T::FN];
        int at[T::FN];  // the given reference, relative to the lane's first row as at() counts
#pragma unroll
        for (int j = 0; j < T::FN; ++j) {
            const int64_t m = m0 + place.col(j);
            const int64_t given = g.given && m < g.M ? g.given[m] : -1;
            at[j] = given >= n0 && given < n0 + T::BM && given < g.off.N ? int(given - n0) - place.first() : -1;
            most[j] = -INFINITY;
            least[j] = INFINITY;
            sum[j] = 0.0f;
        }
        __syncthreads();
        const Offset* mine = off + place.first();
        // (the scores are formed twice: kept, they would need the registers of the sums once more)
#pragma unroll
        for (int i = 0; i < T::FM; ++i) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const Offset o = mine[place.at(i, e)];
#pragma unroll
                for (int j = 0; j < T::FN; ++j) most[j] = fmaxf(most[j], score(acc[i][j][e], o, g.off.c));
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        float base[T::FN];
#pragma unroll
        for (int j = 0; j < T::FN; ++j) {
            most[j] = fmaxf(most[j], __shfl_xor(most[j], 32));
            base[j] = base_of(most[j]);
        }
        asm volatile("" ::: "memory");  // (the offsets are read again)
#pragma unroll
        for (int i = 0; i < T::FM; ++i) {
#pragma unroll
            for (int j = 0; j < T::FN; ++j) {
                const int here = at[j] - i * 32;
                const bool any = here >= 0 && here < 32 && !(here & 4);
                if (__builtin_amdgcn_ballot_w64(any) == 0) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const Offset o = mine[place.at(i, e)];
                        sum[j] += exp_of(score(acc[i][j][e], o, g.off.c) - base[j]);
                        least[j] = fminf(least[j], lowest_of(acc[i][j][e], o, g.off.c));
                    }
                } else {  // the given reference's score goes out, and is not among the others
                    float given = 0.0f;
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const bool is = here == place.at(0, e);
                        const Offset o = mine[place.at(i, e)];
                        const float z = score(acc[i][j][e], o, g.off.c);
                        const float p = exp_of(z - base[j]);
                        least[j] = fminf(least[j], lowest_of(acc[i][j][e], o, g.off.c));
                        given = is ? z : given;
                        sum[j] += is ? 0.0f : p;
                    }
                    if (any) g.given_score[m0 + place.col(j)] = given;
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
#pragma unroll
        for (int j = 0; j < T::FN; ++j) {
            if (least[j] == -INFINITY) sum[j] = NAN;
            sum[j] += __shfl_xor(sum[j], 32);
            if (place.q == 0) part[place.wm * T::BN + place.col(j)] = ScorePart{most[j], sum[j]};
        }
        __syncthreads();
        for (int i = tid; i < T::BN; i += T::NT) {
            if (m0 + i >= g.M) continue;
            ScorePart all = part[i];
#pragma unroll
            for (int w = 1; w < T::WM; ++w) {
                const ScorePart p = part[w * T::BN + i];
                const float both = fmaxf(all.most, p.most), base = base_of(both);
                all.sum = all.sum * exp_of(all.most - base) + p.sum * exp_of(p.most - base);
                all.most = both;
            }
            g.parts[int64_t(im) * g.M + m0 + i] = all;
        }
    }
};

// Sum over 16 (or 8) neighbouring lanes, in each of them: adds whose second operand comes from another lane.
template <int LANES> __device__ __forceinline__ float lanes_sum(float v) {
    auto plus = [&](auto ctrl) {
        v += __uint_as_float(__builtin_amdgcn_update_dpp(0, int(__float_as_uint(v)), decltype(ctrl)::value, 0xf, 0xf, true));
    };
    static_assert(LANES == 16 || LANES == 8, "a row of DPP lanes or half of one");
    if (LANES == 16) plus(std::integral_constant<int, 0x140>{});  // mirrored row
    plus(std::integral_constant<int, 0x141>{});                   // mirrored half row
    plus(std::integral_constant<int, 0x4e>{});                    // pairs of four swapped
    plus(std::integral_constant<int, 0xb1>{});                    // neighbours swapped
    return v;
}

// Pieces of G (as g_pieces says on the host), and what rounding left of a value for the second.
template <class S> constexpr int kPieces = Units<S>::planes == 1 ? 2 : 1;
template <class S> __device__ __forceinline__ float left_of(float v, typename S::Bits rounded) {
    const float w = S::widen(rounded);
    return fabsf(w) < INFINITY ? v - w : 0.0f;
}

struct GradEpi {
    using Args = GradOut;
    template <class S> static constexpr bool kTwice = false;
    template <class S, class T>
    static __device__ __forceinline__ void run(const Args& g, Acc<T>& acc, uint32_t im, uint32_t in, char* lds) {
        const int tid = threadIdx.x;
        const Place<T> place(tid);
        const int64_t n0 = int64_t(im) * T::BM, m0 = int64_t(in) * T::BN;
        char* rows = lds;
        Offset* off = reinterpret_cast<Offset*>(lds + (T::NT / 64) * Rows4<T>::kBytes);
        float* sums = reinterpret_cast<float*>(off + T::BM);  // [WN][BM]
        static_assert((T::NT / 64) * Rows4<T>::kBytes + 4 * T::BM * (2 + T::WN) <= tile_lds<S, T>(), "LDS of the products");
        tile_offsets<T>(g.off, n0, off);
        float most[T::FN], a[T::FN], at_given[T::FN];
        int at[T::FN];
#pragma unroll
        for (int j = 0; j < T::FN; ++j) {
            const int64_t m = m0 + place.col(j);
            PairCoef k{0.0f, 0.0f, 0.0f, -1};
            if (m < g.M) k = g.coef[m];
            const int64_t given = k.given - g.first;
            at[j] = k.given >= 0 && given >= n0 && given < n0 + T::BM ? int(given - n0) - place.first() : -1;
            most[j] = k.most;
            a[j] = k.a;
            at_given[j] = k.at_given;
        }
        __syncthreads();
        const Offset* mine = off + place.first();
        // What a reference that is ruled out holds is not used: a product that is not finite says that it may hold what a factor
        // of zero would not take out of the images' gradients, which then look at who is.
        bool ruled = false;
        for (int i = tid & 63; i < T::FM * 32; i += 64) {
            const int row = place.wm * T::FM * 32 + i;
            ruled |= n0 + row < g.off.N && off[row].limit == -INFINITY;
        }
        if (__builtin_amdgcn_ballot_w64(ruled) != 0) {
            bool bad = false;
#pragma unroll
            for (int i = 0; i < T::FM; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const bool out = mine[place.at(i, e)].limit == -INFINITY;
#pragma unroll
                    for (int j = 0; j < T::FN; ++j) bad |= out && !(fabsf(acc[i][j][e]) < INFINITY);
                }
            if (bad) *g.look = 1;
        }
        auto* out = static_cast<typename S::Bits*>(g.g);
#pragma unroll
        for (int i = 0; i < T::FM; ++i) {
            v16f row[T::FN];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const Offset o = mine[place.at(i, e)];
#pragma unroll
                for (int j = 0; j < T::FN; ++j) {
                    const float z = score(acc[i][j][e], o, g.off.c);
                    const float v = a[j] * exp_of(z - most[j]);
                    row[j][e] = o.limit == -INFINITY ? 0.0f : v;  // (a may be NaN)
                }
            }
#pragma unroll
            for (int j = 0; j < T::FN; ++j) {
                const int here = at[j] - i * 32;
                if (__builtin_amdgcn_ballot_w64(here >= 0 && here < 32) != 0)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const bool is = here == place.at(0, e) && mine[place.at(i, e)].limit != -INFINITY;
                        row[j][e] = is ? at_given[j] : row[j][e];
                    }
                if (m0 + place.col(j) >= g.M)
#pragma unroll
                    for (int e = 0; e < 16; ++e) row[j][e] = 0.0f;
            }
            Rows4<T>::run(row, i, rows, [&](int row, int col, float4 v) {
                const float sum = lanes_sum<Rows4<T>::kLanes>((v.x + v.y) + (v.z + v.w));
                if ((tid & (Rows4<T>::kLanes - 1)) == 0) sums[place.wn * T::BM + row] = sum;
                const int64_t n = n0 + row, m = m0 + col;
                if (n >= g.off.N || m >= g.ldg) return;  // (ldg is a multiple of 8)
                auto* to = out + n * (kPieces<S> * g.ldg) + m;
                typename S::Bits b[4] = {S::round(v.x), S::round(v.y), S::round(v.z), S::round(v.w)};
                __builtin_memcpy(__builtin_assume_aligned(to, sizeof b), b, sizeof b);
                if constexpr (kPieces<S> > 1) {
                    b[0] = S::round(left_of<S>(v.x, b[0]));
                    b[1] = S::round(left_of<S>(v.y, b[1]));
                    b[2] = S::round(left_of<S>(v.z, b[2]));
                    b[3] = S::round(left_of<S>(v.w, b[3]));
                    __builtin_memcpy(__builtin_assume_aligned(to + g.ldg, sizeof b), b, sizeof b);
                }
            });
        }
        if (!g.sums) return;
        __syncthreads();
        for (int i = tid; i < T::BM; i += T::NT) {
            if (n0 + i >= g.off.N) continue;
            float sum = 0.0f;
#pragma unroll
            for (int w = 0; w < T::WN; ++w) sum += sums[w * T::BM + i];
            g.sums[int64_t(in) * g.off.N + n0 + i] = sum;
        }
    }
};

struct MatrixEpi {
    using Args = MatrixOut;
    template <class S> static constexpr bool kTwice = kPieces<S> > 1;  // (with each of G's pieces)
    template <class S, class T>
    static __device__ __forceinline__ void run(const Args& g, Acc<T>& acc, uint32_t im, uint32_t in, char* lds) {
        const int64_t i0 = int64_t(im) * T::BM, j0 = int64_t(in) * T::BN;
        const float scale = g.scale ? *g.scale : 1.0f;
        auto* out = static_cast<typename S::Bits*>(g.out);
#pragma unroll
        for (int i = 0; i < T::FM; ++i)
            Rows4<T>::run(acc[i], i, lds, [&](int row, int col, float4 v) {
                const int64_t at = i0 + row, c = j0 + col;
                if (at >= g.rows || c >= g.cols) return;
                const int n = int(min(g.cols - c, int64_t(4)));
                float f[4] = {v.x, v.y, v.z, v.w};
                if (g.ruled.N && ruled_out(g.ruled, at)) f[0] = f[1] = f[2] = f[3] = 0.0f;  // (what images hold does not matter)
                if (g.before)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (k < n) f[k] += g.before[at * g.cols + c + k];
                if (g.after) {
                    if (n == 4) {
                        __builtin_memcpy(g.after + at * g.cols + c, f, sizeof f);
                    } else {
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (k < n) g.after[at * g.cols + c + k] = f[k];
                    }
                    return;
                }
                const typename S::Bits b[4] = {S::round(f[0] * scale), S::round(f[1] * scale), S::round(f[2] * scale),
                                               S::round(f[3] * scale)};
                if (n == 4) {
                    __builtin_memcpy(out + at * g.ld + c, b, sizeof b);
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (k < n) out[at * g.ld + c + k] = b[k];
                }
            });
    }
};

}  // namespace

template <class S> hipError_t PairProducts<S>::stats(const PairArgs& a, const TilePlan& t, const StatsOut& o, float* part, hipStream_t s) {
    const Product g{{a.r, a.ldr, a.K, nullptr, nullptr, nullptr}, {a.x, a.ldx, a.K, nullptr, nullptr, nullptr}, a.N, a.M, a.K, 0, 0, 0, t.whole, t.splits, part};
    return product<S, false, false, StatsEpi>(g, t, o, s);
}
template <class S>
hipError_t PairProducts<S>::grad(const PairArgs& a, const void* r, int64_t n, const TilePlan& t, const GradOut& o, float* part, hipStream_t s) {
    const Product g{{r, a.ldr, a.K, nullptr, nullptr, nullptr}, {a.x, a.ldx, a.K, nullptr, nullptr, nullptr}, n, a.M, a.K, 0, 0, 0, t.whole, t.splits, part};
    return product<S, false, false, GradEpi>(g, t, o, s);
}
template <class S>
hipError_t PairProducts<S>::d_references(const PairArgs& a, const void* gr, int64_t ldg, int64_t n, const TilePlan& t,
                                         const MatrixOut& o, float* part, hipStream_t s) {
    // (g holds zeros from M to ldg: whole chunks)
    const Product g{{gr, kPieces<S> * ldg, ldg, nullptr, nullptr, nullptr}, {a.x, a.ldx, a.M, nullptr, nullptr, nullptr}, n, a.K, a.M, ldg, 0, 0, t.whole, t.splits, part};
    return product<S, false, true, MatrixEpi>(g, t, o, s);
}
template <class S>
hipError_t PairProducts<S>::d_images(const PairArgs& a, const void* gr, int64_t ldg, const void* r, const PairOff& off,
                                     const int* look, const TilePlan& t, const MatrixOut& o, float* part, hipStream_t s) {
    const Product g{{gr, kPieces<S> * ldg, off.N, nullptr, nullptr, nullptr}, {r, a.ldr, off.N, look, off.mask, off.bias}, a.M, a.K, off.N, ldg, 0, 0, t.whole, t.splits, part};
    return product<S, true, true, MatrixEpi>(g, t, o, s);
}

}  // namespace tp
