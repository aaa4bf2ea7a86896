// The tiled products of the pair log probabilities for one storage type (included by tp_pairs_*.hip).
#pragma once

#include "tp_pairs.hh"
#include "tp_tile.hh"

namespace tp {
namespace {

constexpr float kLog2e = 1.44269504088896340736f;

// LDS behind what the epilogue's other parts use: a tile's offsets, -inf where the reference is ruled out.
template <class T> __device__ __forceinline__ void tile_offsets(const PairOff& o, int64_t first, float* off) {
    for (int i = threadIdx.x; i < T::BM; i += T::NT) {
        const int64_t n = first + i;
        off[i] = n < o.N && (!o.mask || o.mask[n]) ? (o.bias ? o.bias[n] : 0.0f) : -INFINITY;
    }
}
// (what the product of a reference that is ruled out came to does not matter)
__device__ __forceinline__ float score(float sum, float off, float c) { return off == -INFINITY ? -INFINITY : (sum + off) * c; }

// A lane holds 16 FM references of each of its FN images: their maximum and sum in registers, then over the two
// halves of the wavefront and the WM wavefronts.
struct StatsEpi {
    using Args = StatsOut;
    template <class S, class T>
    static __device__ __forceinline__ void run(const Args& g, Acc<T>& acc, uint32_t im, uint32_t in, char* lds) {
        const int tid = threadIdx.x;
        const Place<T> place(tid);
        const int64_t n0 = int64_t(im) * T::BM, m0 = int64_t(in) * T::BN;
        float* off = reinterpret_cast<float*>(lds);
        ScorePart* part = reinterpret_cast<ScorePart*>(off + T::BM);  // [WM][BN]
        tile_offsets<T>(g.off, n0, off);
        __syncthreads();
#pragma unroll
        for (int j = 0; j < T::FN; ++j) {
            const int64_t m = m0 + place.col(j);
            const int64_t given = g.given && m < g.M ? g.given[m] - n0 : -1;
            const int at = given >= 0 && given < T::BM && given + n0 < g.off.N ? int(given) : -1;
            float most = -INFINITY, sum = 0.0f, z_given = 0.0f;
            asm volatile("" ::: "memory");  // (the offsets are read again: kept for the next column they would fill the registers)
#pragma unroll
            for (int i = 0; i < T::FM; ++i) {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    acc[i][j][e] = score(acc[i][j][e], off[place.row(i, e)], g.off.c);
                    most = fmaxf(most, acc[i][j][e]);
                }
                __builtin_amdgcn_sched_barrier(0);  // (else all offsets of the tile wait in registers)
            }
            most = fmaxf(most, __shfl_xor(most, 32));
            const float base = most == -INFINITY ? 0.0f : most;
#pragma unroll
            for (int i = 0; i < T::FM; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float z = acc[i][j][e];
                    const bool is = place.row(i, e) == at;
                    const float p = __builtin_amdgcn_exp2f((z - base) * kLog2e);
                    sum += is ? 0.0f : p;
                    z_given = is ? z : z_given;
                }
            if (at >= 0 && at / (T::FM * 32) == place.wm && ((at >> 2) & 1) == place.q) g.given_score[m] = z_given;
            sum += __shfl_xor(sum, 32);
            if (place.q == 0) part[place.wm * T::BN + place.col(j)] = ScorePart{most, sum};
        }
        __syncthreads();
        for (int i = tid; i < T::BN; i += T::NT) {
            if (m0 + i >= g.M) continue;
            ScorePart all = part[i];
#pragma unroll
            for (int w = 1; w < T::WM; ++w) {
                const ScorePart p = part[w * T::BN + i];
                const float most = fmaxf(all.most, p.most), base = most == -INFINITY ? 0.0f : most;
                all.sum = all.sum * __builtin_amdgcn_exp2f((all.most - base) * kLog2e) +
                          p.sum * __builtin_amdgcn_exp2f((p.most - base) * kLog2e);
                all.most = most;
            }
            g.parts[int64_t(im) * g.M + m0 + i] = all;
        }
    }
};

struct GradEpi {
    using Args = GradOut;
    template <class S, class T>
    static __device__ __forceinline__ void run(const Args& g, Acc<T>& acc, uint32_t im, uint32_t in, char* lds) {
        const int tid = threadIdx.x;
        const Place<T> place(tid);
        const int64_t n0 = int64_t(im) * T::BM, m0 = int64_t(in) * T::BN;
        char* rows = lds;
        float* off = reinterpret_cast<float*>(lds + (T::NT / 64) * Rows4<T>::kBytes);
        float* sums = off + T::BM;  // [WN][BM]
        static_assert((T::NT / 64) * Rows4<T>::kBytes + 4 * T::BM * (1 + T::WN) <= tile_lds<S, T>(), "LDS of the products");
        tile_offsets<T>(g.off, n0, off);
        __syncthreads();
#pragma unroll
        for (int j = 0; j < T::FN; ++j) {
            const int64_t m = m0 + place.col(j);
            PairCoef k{0.0f, 0.0f, 0.0f, -1};
            if (m < g.M) k = g.coef[m];
            const int64_t given = k.given - g.first - n0;
            const int at = k.given >= 0 && given >= 0 && given < T::BM ? int(given) : -1;
            asm volatile("" ::: "memory");
#pragma unroll
            for (int i = 0; i < T::FM; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int row = place.row(i, e);
                    const float z = score(acc[i][j][e], off[row], g.off.c);
                    float v = k.a * __builtin_amdgcn_exp2f((z - k.most) * kLog2e);
                    v = row == at ? k.at_given : v;
                    acc[i][j][e] = m < g.M && off[row] != -INFINITY ? v : 0.0f;
                    if (e == 15) __builtin_amdgcn_sched_barrier(0);
                }
        }
        auto* out = static_cast<typename S::Bits*>(g.g);
#pragma unroll
        for (int i = 0; i < T::FM; ++i)
            Rows4<T>::run(acc[i], i, rows, [&](int row, int col, float4 v) {
                float sum = (v.x + v.y) + (v.z + v.w);
#pragma unroll
                for (int d = Rows4<T>::kLanes / 2; d; d >>= 1) sum += __shfl_xor(sum, d);
                if ((tid & (Rows4<T>::kLanes - 1)) == 0) sums[place.wn * T::BM + row] = sum;
                const int64_t n = n0 + row, m = m0 + col;
                if (n >= g.off.N || m >= g.ldg) return;  // (ldg is a multiple of 8)
                const typename S::Bits b[4] = {S::round(v.x), S::round(v.y), S::round(v.z), S::round(v.w)};
                __builtin_memcpy(__builtin_assume_aligned(out + n * g.ldg + m, sizeof b), b, sizeof b);
            });
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

template <class S> struct Shapes {
    using Small = TileShape<64, 64, 2, 2>;
    using Middle = TileShape<128, 128, 2, 4>;
    using Large = TileShape<256, 256, 2, 4>;
};
template <> struct Shapes<F32> {  // (three planes of 256 x 128 are 144 KB in two stages)
    using Small = TileShape<64, 64, 2, 2>;
    using Middle = TileShape<128, 128, 2, 4>;
    using Large = TileShape<256, 128, 4, 2>;
};

template <class S, class T, bool ATR, bool BTR, class Epi>
hipError_t product_of(Product g, const typename Epi::Args& ea, hipStream_t s) {
    g.tm = uint32_t((g.rows + T::BM - 1) / T::BM);
    g.tn = uint32_t((g.cols + T::BN - 1) / T::BN);
    k_tile<S, T, ATR, BTR, Epi><<<dim3(g.tm * g.tn * g.splits), T::NT, 0, s>>>(g, ea);
    if (hipError_t e = hipGetLastError()) return e;
    if (g.splits > 1) k_tile_join<S, T, Epi><<<dim3(g.tm * g.tn), T::NT, 0, s>>>(g, ea);
    return hipGetLastError();
}
template <class S, bool ATR, bool BTR, class Epi>
hipError_t product(const Product& g, int tile, const typename Epi::Args& ea, hipStream_t s) {
    switch (tile) {
        case 0: return product_of<S, typename Shapes<S>::Small, ATR, BTR, Epi>(g, ea, s);
        case 1: return product_of<S, typename Shapes<S>::Middle, ATR, BTR, Epi>(g, ea, s);
        default: return product_of<S, typename Shapes<S>::Large, ATR, BTR, Epi>(g, ea, s);
    }
}

}  // namespace

template <class S> hipError_t PairProducts<S>::stats(const PairArgs& a, const PairTile& t, const StatsOut& o, float* part, hipStream_t s) {
    const Product g{{a.r, a.ldr, nullptr}, {a.x, a.ldx, nullptr}, a.N, a.M, a.K, t.splits, part, 0, 0};
    return product<S, false, false, StatsEpi>(g, t.tile, o, s);
}
template <class S>
hipError_t PairProducts<S>::grad(const PairArgs& a, const void* r, int64_t n, const PairTile& t, const GradOut& o, float* part, hipStream_t s) {
    const Product g{{r, a.ldr, nullptr}, {a.x, a.ldx, nullptr}, n, a.M, a.K, t.splits, part, 0, 0};
    return product<S, false, false, GradEpi>(g, t.tile, o, s);
}
template <class S>
hipError_t PairProducts<S>::d_references(const PairArgs& a, const void* gr, int64_t ldg, int64_t n, const PairTile& t,
                                         const MatrixOut& o, float* part, hipStream_t s) {
    const Product g{{gr, ldg, nullptr}, {a.x, a.ldx, nullptr}, n, a.K, a.M, t.splits, part, 0, 0};
    return product<S, false, true, MatrixEpi>(g, t.tile, o, s);
}
template <class S>
hipError_t PairProducts<S>::d_images(const PairArgs& a, const void* gr, int64_t ldg, const void* r, const uint8_t* mask,
                                     int64_t n, const PairTile& t, const MatrixOut& o, float* part, hipStream_t s) {
    const Product g{{gr, ldg, nullptr}, {r, a.ldr, mask}, a.M, a.K, n, t.splits, part, 0, 0};
    return product<S, true, true, MatrixEpi>(g, t.tile, o, s);
}

}  // namespace tp
