// Log probabilities of pairs (image, reference) without their scores in memory, and their gradient.
//
//   score    z[m, n] = (<x_m, r_n> + bias_n) c, c = 1 / temperature, over the allowed references
//   results  log_sum[m] = ln sum_n exp(z[m, n]),  given[m] = z[m, g] - log_sum[m] of the given reference g
//   gradient G[m, n] = c (p[m, n] (d_log_sum[m] - d_given[m]) + d_given[m] [n = g]), p = exp(z - log_sum)
//            d_x = G r,  d_r = G^T x,  d_bias = the sums of G over the images
//
// Many images: the scores are formed in tiles (tp_tile.hh), a tile's references reduced at once to their largest score and
// sum per image, and these joined.  The gradient forms the scores again, piece after piece of the references and the images,
// turns them into G in the products' type, and multiplies it with both sides; a piece's G is all that is kept of M x N.
// Few images: the references stream past them once, as fast as they can be read; the scores (at most 8 rows) are kept for the
// gradient, which streams the references and their gradient.
//
// The given reference is kept out of the sums, as next to a probability of one the logarithm of all of them would
// lose what the others hold: given = -ln(1 + others / own).
#include "../../../include/torch_projectors_hip.h"
#include "tp_pairs.hh"

#include <algorithm>

namespace tp {
namespace {

constexpr int kStats = 4;  // largest, others' sum, own, and one to spare: an image's stand in 16 bytes

__device__ __forceinline__ float exp_of(float z) { return __builtin_amdgcn_exp2f(z * kLog2e); }
// (largest, sum of exp(z - largest)) of two sets of scores
__device__ __forceinline__ void join(float& most, float& sum, float most2, float sum2) {
    const float both = fmaxf(most, most2), base = both == -INFINITY ? 0.0f : both;
    sum = sum * exp_of(most - base) + sum2 * exp_of(most2 - base);
    most = both;
}

// Results of an image from its largest score, the others' sum and the given reference's score.
__device__ __forceinline__ void finish(const PairArgs& a, int64_t m, float most, float others, float z, float* given_out,
                                       float* log_sum, float* state) {
    const int64_t g = a.given ? a.given[m] : -1;
    const bool valid = g >= 0 && g < a.N;
    const float base = most == -INFINITY ? 0.0f : most;
    const float own = valid ? exp_of(z - base) : 0.0f, total = others + own;
    // (1 + x) - 1 is what logf sees of a sum near one: the others by themselves
    const float log_total = own == 1.0f && others < 0.5f ? log1pf(others) : logf(total);
    log_sum[m] = base + log_total;
    if (total == 0.0f) log_sum[m] = -INFINITY;
    if (given_out) {
        float v = own > others ? -log1pf(others / own) : (z - base) - log_total;
        if (total == 0.0f) v = -INFINITY;
        given_out[m] = valid ? v : g == -1 ? 0.0f : NAN;
    }
    if (state) {
        float* st = state + m * kStats;
        st[0] = base;
        st[1] = others;
        st[2] = own;
    }
}

// ------------------------------------------------------------------ many images: the tiles' parts joined
// 16 images by 16 lanes, which share the parts (128 neighbouring bytes of each): 6 us for 4096 images of 144 parts, a launch's length.
__global__ __launch_bounds__(256) void k_pairs_join(PairArgs a, const ScorePart* __restrict__ parts, int tiles,
                                                    const float* __restrict__ given_score, float* given_out,
                                                    float* log_sum, float* state) {
    __shared__ ScorePart all[16][17];
    const int x = threadIdx.x & 15, y = threadIdx.x >> 4;
    const int64_t m = int64_t(blockIdx.x) * 16 + x;
    float most = -INFINITY, sum = 0.0f;
    if (m < a.M) {
#pragma unroll 4
        for (int t = y; t < tiles; t += 16) {
            const ScorePart p = parts[int64_t(t) * a.M + m];
            join(most, sum, p.most, p.sum);
        }
    }
    all[y][x] = ScorePart{most, sum};
    __syncthreads();
    if (y || m >= a.M) return;
#pragma unroll
    for (int i = 1; i < 16; ++i) join(most, sum, all[i][x].most, all[i][x].sum);
    const bool valid = a.given && a.given[m] >= 0 && a.given[m] < a.N;
    finish(a, m, most, sum, valid ? given_score[m] : -INFINITY, given_out, log_sum, state);
}

// ------------------------------------------------------------------ the gradient's coefficients
// An image's upstream gradients as they are used.
struct Upstream {
    float log_sum, given;
    int at;  // the given reference, -1: none
};
__device__ __forceinline__ Upstream upstream(const PairArgs& a, int64_t m, const float* d_given, const float* d_log_sum) {
    const int64_t g = a.given ? a.given[m] : -1;
    const bool valid = g >= 0 && g < a.N;
    Upstream u{d_log_sum ? d_log_sum[m] : 0.0f, d_given && a.given && g != -1 ? d_given[m] : 0.0f, valid ? int(g) : -1};
    if (!valid && u.given != 0.0f) u.given = NAN;
    return u;
}
__device__ __forceinline__ PairCoef coefficients(const PairArgs& a, const float* state, int64_t m, const float* d_given,
                                                 const float* d_log_sum) {
    const float* st = state + m * kStats;
    const float others = st[1], own = st[2], total = others + own;
    const Upstream u = upstream(a, m, d_given, d_log_sum);
    const float dl = u.log_sum, dg = u.given;
    PairCoef k{st[0], a.c * (dl - dg) / total, a.c * (dl * own + dg * others) / total, u.at};
    if (total == 0.0f) k.a = k.at_given = 0.0f;  // a row that allows nothing
    return k;
}

// Half precision: G is scaled by a power of two that brings its largest possible value to 2^13 to 2^14 (its normal
// numbers start at 2^-14: what is 2^-28 of the largest, or more, keeps all bits), and back by scale[0].  Images that have no finite gradient,
// or none, have no say in it.
__global__ __launch_bounds__(1024) void k_pairs_coef(PairArgs a, const float* __restrict__ state, const float* d_given,
                                                     const float* d_log_sum, bool half, PairCoef* coef, float* scale, int* look) {
    __shared__ float room[16];
    float up = 1.0f;
    if (half) {
        float most = 0.0f;
        for (int64_t m = threadIdx.x; m < a.M; m += 1024) {
            const Upstream u = upstream(a, m, d_given, d_log_sum);
            const float v = a.c * (fabsf(u.log_sum) + fabsf(u.given)), total = state[m * kStats + 1] + state[m * kStats + 2];
            if (v < INFINITY && total > 0.0f) most = fmaxf(most, v);
        }
#pragma unroll
        for (int d = 32; d; d >>= 1) most = fmaxf(most, __shfl_xor(most, d));
        if ((threadIdx.x & 63) == 0) room[threadIdx.x >> 6] = most;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 16; ++i) most = fmaxf(most, room[i]);
        int e = 0;
        frexpf(most, &e);  // most < 2^e
        up = most > 0.0f ? ldexpf(1.0f, max(min(14 - e, 100), -100)) : 1.0f;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        scale[0] = 1.0f / up;
        *look = 0;
    }
    for (int64_t m = int64_t(blockIdx.x) * 1024 + threadIdx.x; m < a.M; m += int64_t(gridDim.x) * 1024) {
        PairCoef k = coefficients(a, state, m, d_given, d_log_sum);
        k.a *= up;
        k.at_given *= up;
        coef[m] = k;
    }
}

// d_bias of a piece's references from the image tiles' sums, those of the images' further pieces on top.
__global__ __launch_bounds__(256) void k_pairs_bias(const float* __restrict__ sums, int tiles, int64_t n,
                                                    const float* __restrict__ scale, bool more, float* d_bias) {
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < n; i += int64_t(gridDim.x) * 256) {
        float v = 0.0f;
#pragma unroll 4
        for (int t = 0; t < tiles; ++t) v += sums[int64_t(t) * n + i];
        v *= scale[0];
        d_bias[i] = more ? d_bias[i] + v : v;
    }
}

// ------------------------------------------------------------------ few images: scores
using v4f = __attribute__((ext_vector_type(4))) float;
using v8bf = __attribute__((ext_vector_type(8))) __bf16;
using v8h = __attribute__((ext_vector_type(8))) _Float16;

// 16 bytes of 16 rows each, lanes r + 16 q: float32 through the float32 units (which are not what bounds this).
template <class S> __device__ __forceinline__ v4f few_product(const Pack<S>& a, const Pack<S>& b, v4f c);
template <> __device__ __forceinline__ v4f few_product<BF16>(const Pack<BF16>& a, const Pack<BF16>& b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ v4f few_product<F16>(const Pack<F16>& a, const Pack<F16>& b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ v4f few_product<F32>(const Pack<F32>& a, const Pack<F32>& b, v4f c) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
        c = __builtin_amdgcn_mfma_f32_16x16x4f32(F32::widen(a.v[i]), F32::widen(b.v[i]), c, 0, 0, 0);
    return c;
}

// n of a pack's values from p on, zeros behind them
template <class S> __device__ __forceinline__ Pack<S> load_some(const typename S::Bits* p, int64_t n) {
    if (n >= Pack<S>::n) return load_pack<S>(p);
    Pack<S> r;
#pragma unroll
    for (int i = 0; i < Pack<S>::n; ++i) r.v[i] = i < n ? p[i] : typename S::Bits(0);
    return r;
}

// A workgroup takes 16 references, each of its wavefronts every eighth 128 bytes of their rows (of its range of the
// rows), straight from memory into operands: kAhead such units' loads are in flight at once.  Bytes bound it: 4096 references of 16640
// bfloat16 values take 23 us, 5.9 TB/s.  (A ring of loads that never drains is 4 us slower there, more registers for fewer
// wavefronts, though 8 us faster for float32, 58 with the join.)

template <class S>
__global__ __launch_bounds__(64 * kFewWaves) void k_pairs_few(PairArgs a, int splits, float* __restrict__ out) {
    using Bits = typename S::Bits;
    constexpr int U = kUnit / int(sizeof(Bits)), P = Pack<S>::n;
    __shared__ float sums[kFewWaves][16][kFewImages];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, r = lane & 15, q = lane >> 4;
    const int64_t n0 = int64_t(blockIdx.x) * 16;
    const int split = blockIdx.y;
    // rows past the end read the last one's values and are not stored
    const Bits* pr = static_cast<const Bits*>(a.r) + min(n0 + r, a.N - 1) * a.ldr + q * P;
    const Bits* px = static_cast<const Bits*>(a.x) + min(int64_t(r), a.M - 1) * a.ldx + q * P;
    const int units = int((a.K + U - 1) / U);
    const int u0 = int(int64_t(units) * split / splits), u1 = int(int64_t(units) * (split + 1) / splits);
    v4f acc[2] = {v4f{0, 0, 0, 0}, v4f{0, 0, 0, 0}};
    for (int u = u0 + wave; u < u1; u += kFewWaves * kAhead) {
        Pack<S> vr[kAhead][2], vx[kAhead][2];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            if (u + k * kFewWaves >= u1) break;
            const int64_t at = int64_t(u + k * kFewWaves) * U;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (at + U <= a.K) {
                    vr[k][h] = load_pack<S>(pr + at + h * 4 * P);
                    vx[k][h] = load_pack<S>(px + at + h * 4 * P);
                } else {
                    vr[k][h] = load_some<S>(pr + at + h * 4 * P, a.K - at - h * 4 * P - q * P);
                    vx[k][h] = load_some<S>(px + at + h * 4 * P, a.K - at - h * 4 * P - q * P);
                }
            }
        }
        __builtin_amdgcn_sched_barrier(0);  // all loads before the first use
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            if (u + k * kFewWaves >= u1) break;
#pragma unroll
            for (int h = 0; h < 2; ++h) acc[h] = few_product<S>(vr[k][h], vx[k][h], acc[h]);
        }
    }
    // (lane: image r, references 4 q + j)
    if (r < kFewImages)
#pragma unroll
        for (int j = 0; j < 4; ++j) sums[wave][4 * q + j][r] = acc[0][j] + acc[1][j];
    __syncthreads();
    const int i = tid & 15, m = tid >> 4;
    if (m >= a.M || n0 + i >= a.N) return;
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < kFewWaves; ++w) v += sums[w][i][m];
    out[(int64_t(split) * a.M + m) * a.N + n0 + i] = v;
}

// One image's scores from the ranges' sums, reduced by one workgroup, or by several, each of which leaves a part for
// k_pairs_join; kept in `scores` where the gradient will read them.  (4096 references of one image: 5 us, a chain of start, loads and two
// reductions.)
__global__ __launch_bounds__(1024) void k_pairs_few_join(PairArgs a, const float* part, int splits, float* scores,
                                                         float* given_out, float* log_sum, float* state, int64_t each,
                                                         ScorePart* parts, float* given_score) {
    __shared__ ScorePart all[16];
    __shared__ float z_given;
    const int64_t m = blockIdx.x, first = int64_t(blockIdx.y) * each, end = min(first + each, a.N);
    const int64_t g = a.given ? a.given[m] : -1;
    float most = -INFINITY, sum = 0.0f;
    constexpr int V = 4;
    for (int64_t n0 = first + threadIdx.x; n0 < end; n0 += 1024 * V) {
        // (all of a step's loads, then what they mean)
        float add[V], s[V];
        bool counts[V];
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const int64_t n = min(n0 + k * 1024, end - 1);
            add[k] = a.bias ? a.bias[n] : 0.0f;
            counts[k] = !a.mask || a.mask[n];
            s[k] = part[m * a.N + n];
        }
#pragma unroll 4
        for (int t = 1; t < splits; ++t)
#pragma unroll
            for (int k = 0; k < V; ++k) s[k] += part[(int64_t(t) * a.M + m) * a.N + min(n0 + k * 1024, end - 1)];
        float z[V], here = most;
#pragma unroll
        for (int k = 0; k < V; ++k) {
            z[k] = fmaf(s[k], a.c, times(add[k], a.c));
            if (!(fabsf(z[k]) < INFINITY)) z[k] = NAN;  // (-inf is what is ruled out, and no score)
            if (!counts[k] || add[k] == -INFINITY || n0 + k * 1024 >= end) z[k] = -INFINITY;
            here = fmaxf(here, z[k]);
        }
        const float base = here == -INFINITY ? 0.0f : here;
        sum *= exp_of(most - base);
        most = here;
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const int64_t n = n0 + k * 1024;
            if (n >= end) continue;
            if (scores) scores[m * a.N + n] = z[k];
            if (n == g)
                z_given = z[k];
            else
                sum += exp_of(z[k] - base);
        }
    }
    auto shuffled = [&](int from) {
#pragma unroll
        for (int d = from; d; d >>= 1) {
            const float most2 = __shfl_xor(most, d), sum2 = __shfl_xor(sum, d);
            join(most, sum, most2, sum2);
        }
    };
    shuffled(32);
    if ((threadIdx.x & 63) == 0) all[threadIdx.x >> 6] = ScorePart{most, sum};
    __syncthreads();
    if (threadIdx.x >= 16) return;
    most = all[threadIdx.x].most;
    sum = all[threadIdx.x].sum;
    shuffled(8);
    if (threadIdx.x) return;
    if (!parts) return finish(a, m, most, sum, g >= 0 && g < a.N ? z_given : -INFINITY, given_out, log_sum, state);
    parts[int64_t(blockIdx.y) * a.M + m] = ScorePart{most, sum};
    if (g >= first && g < end) given_score[m] = z_given;
}

// ------------------------------------------------------------------ few images: gradient
// A workgroup takes 4 x 256 columns and a range of the references, 64 at a time: their G of every image in LDS, then
// each reference's row read once, added to the images' gradients in registers (G r) while its own gradient (G^T x) is
// written.  Bytes bound it: 4096 float32 references of 16640 values and their gradients take about 100 us, 5.3 TB/s read and written (122
// where the gradient's stores were not streamed past the caches).

// Four values as one access, at any address that a value may have.
template <class B> struct Streamed {
    using Any = B __attribute__((ext_vector_type(kBackCols)));
    using At = B __attribute__((ext_vector_type(kBackCols), aligned(sizeof(B))));
};

template <class S, int MB>
__global__ __launch_bounds__(256) void k_pairs_few_back(PairArgs a, const float* __restrict__ state, const float* d_given,
                                                        const float* d_log_sum, int64_t per, float* __restrict__ dx_part,
                                                        void* d_r, float* d_bias) {
    using Bits = typename S::Bits;
    __shared__ float G[kBackRows][MB];
    __shared__ bool counts[kBackRows];
    __shared__ PairCoef coef[MB];
    const int tid = threadIdx.x;
    const int64_t first = int64_t(blockIdx.y) * per, last = min(first + per, a.N);
    const int64_t c = (int64_t(blockIdx.x) * 256 + tid) * kBackCols;
    const int have = c < a.K ? int(min(a.K - c, int64_t(kBackCols))) : 0;
    const float* scores = state + a.M * kStats;
    if (tid < MB) coef[tid] = tid < a.M ? coefficients(a, state, tid, d_given, d_log_sum) : PairCoef{0, 0, 0, -1};
    float x[MB][kBackCols], dx[MB][kBackCols];
#pragma unroll
    for (int m = 0; m < MB; ++m)
#pragma unroll
        for (int k = 0; k < kBackCols; ++k) {
            dx[m][k] = 0.0f;
            x[m][k] = d_r && m < a.M && k < have ? S::widen(static_cast<const Bits*>(a.x)[m * a.ldx + c + k]) : 0.0f;
        }
    constexpr int W = 8;  // rows on their way
    Bits next[W][kBackCols];
    for (int64_t n0 = first; n0 < last; n0 += kBackRows) {
        const int rows = int(min(last - n0, int64_t(kBackRows)));
        const Bits* r = static_cast<const Bits*>(a.r) + n0 * a.ldr + c;
        auto fetch = [&](int row) {
            if (!dx_part) return;
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const Bits* p = r + min(row + w, rows - 1) * a.ldr;
                if (have == kBackCols) {
                    __builtin_memcpy(next[w], p, sizeof next[w]);
                } else {
#pragma unroll
                    for (int k = 0; k < kBackCols; ++k) next[w][k] = k < have ? p[k] : Bits(0);
                }
            }
        };
        fetch(0);
        __syncthreads();
        for (int i = tid; i < kBackRows * MB; i += 256) {
            const int m = i / kBackRows, row = i % kBackRows;
            float v = 0.0f;
            if (m < a.M && row < rows) {
                const float z = scores[m * a.N + n0 + row];
                if (z != -INFINITY) v = n0 + row == coef[m].given ? coef[m].at_given : coef[m].a * exp_of(z - coef[m].most);
            }
            G[row][m] = v;
        }
        if (tid < rows) counts[tid] = (!a.mask || a.mask[n0 + tid]) && (!a.bias || a.bias[n0 + tid] != -INFINITY);
        __syncthreads();
        if (blockIdx.x == 0 && d_bias && tid < rows) {
            float v = 0.0f;
#pragma unroll
            for (int m = 0; m < MB; ++m) v += G[tid][m];
            d_bias[n0 + tid] = v;
        }
        if (!have) continue;
        Bits* o = static_cast<Bits*>(d_r) + (d_r ? n0 * a.K + c : 0);
        for (int row0 = 0; row0 < rows; row0 += W) {
            Bits now[W][kBackCols];
#pragma unroll
            for (int w = 0; w < W; ++w)
#pragma unroll
                for (int k = 0; k < kBackCols; ++k) now[w][k] = dx_part ? next[w][k] : Bits(0);
            if (row0 + W < rows) fetch(row0 + W);
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const int row = row0 + w;
                if (row >= rows) break;
                // (what a reference that is ruled out holds is not used, and it has no gradient, whatever images hold)
                const bool use = counts[row];
                float up[kBackCols] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int m = 0; m < MB; ++m) {
                    const float g = G[row][m];
#pragma unroll
                    for (int k = 0; k < kBackCols; ++k) {
                        dx[m][k] += g * (use ? S::widen(now[w][k]) : 0.0f);
                        up[k] += g * x[m][k];
                    }
                }
                if (!d_r) continue;
                Bits b[kBackCols];
#pragma unroll
                for (int k = 0; k < kBackCols; ++k) b[k] = S::round(use ? up[k] : 0.0f);
                if (have == kBackCols) {
                    using At = typename Streamed<Bits>::At;
                    __builtin_nontemporal_store(__builtin_bit_cast(typename Streamed<Bits>::Any, b), reinterpret_cast<At*>(o + row * a.K));
                } else {
#pragma unroll
                    for (int k = 0; k < kBackCols; ++k)
                        if (k < have) o[row * a.K + k] = b[k];
                }
            }
        }
    }
    if (!dx_part) return;
#pragma unroll
    for (int m = 0; m < MB; ++m) {
        if (m >= a.M) break;
#pragma unroll
        for (int k = 0; k < kBackCols; ++k)
            if (k < have) dx_part[(int64_t(blockIdx.y) * a.M + m) * a.K + c + k] = dx[m][k];
    }
}

// The ranges' sums, rounded.
template <class S>
__global__ __launch_bounds__(256) void k_pairs_sum(const float* __restrict__ part, int ranges, int64_t n, void* out) {
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < n; i += int64_t(gridDim.x) * 256) {
        float v = 0.0f;
#pragma unroll 8
        for (int t = 0; t < ranges; ++t) v += part[int64_t(t) * n + i];
        static_cast<typename S::Bits*>(out)[i] = S::round(v);
    }
}

// ------------------------------------------------------------------ launches
// Whether all products' operands of these images and references go straight to LDS.
bool pair_direct(const PairArgs& a) {
    auto fits = [](const void* p, int64_t ld) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0; };
    return a.dt != TP_F32 && a.K % 8 == 0 && fits(a.x, a.ldx) && fits(a.r, a.ldr);
}

template <class F> hipError_t by_type(int dt, F f) {
    switch (dt) {
        case TP_F32: return f(F32{});
        case TP_F16: return f(F16{});
        default: return f(BF16{});
    }
}

// Zeros where there is nothing to sum (a memset would not do in a captured graph).
__global__ __launch_bounds__(256) void k_pairs_zero(uint8_t* p, int64_t bytes) {
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < bytes; i += int64_t(gridDim.x) * 256) p[i] = 0;
}
void zero(void* p, int64_t bytes, hipStream_t s) {
    if (p && bytes) k_pairs_zero<<<match_grid((bytes + 255) / 256), 256, 0, s>>>(static_cast<uint8_t*>(p), bytes);
}

// No reference at all.
__global__ __launch_bounds__(256) void k_pairs_none(PairArgs a, float* given_out, float* log_sum, float* state) {
    for (int64_t m = int64_t(blockIdx.x) * 256 + threadIdx.x; m < a.M; m += int64_t(gridDim.x) * 256)
        finish(a, m, -INFINITY, 0.0f, -INFINITY, given_out, log_sum, state);
}

}  // namespace

// (rows may turn out not to start at 16-byte boundaries: room for either plan)
template <class F> int64_t either_plan(int dt, int64_t K, F bytes) {
    const int64_t staged = bytes(false);
    if (dt == TP_F32 || K % 8) return staged;
    const int64_t straight = bytes(true);
    return staged > straight ? staged : straight;
}
int64_t pair_work(int dt, int64_t M, int64_t N, int64_t K) {
    if (M == 0 || N == 0) return 0;
    if (pair_few(M)) return up16(few_splits(dt, N, K) * M * N * 4) + up16(few_parts(N) * M * int64_t(sizeof(ScorePart))) + up16(M * 4);
    return either_plan(dt, K, [&](bool direct) {
        const TilePlan t = tile_plan(dt, direct, N, M, K);
        return up16(M * 4) + up16(tile_count(dt, t, N, true) * M * int64_t(sizeof(ScorePart))) + tile_part_bytes(dt, t, N, M);
    });
}

hipError_t launch_pair_log_probs(const PairArgs& a, float* given_out, float* log_sum, float* state, void* work,
                                 hipStream_t s) {
    if (a.M == 0) return hipSuccess;
    if (a.N == 0) {
        k_pairs_none<<<match_grid((a.M + 255) / 256), 256, 0, s>>>(a, given_out, log_sum, state);
        return hipGetLastError();
    }
    if (pair_few(a.M)) {
        const int splits = few_splits(a.dt, a.N, a.K);
        auto* part = static_cast<float*>(work);
        const dim3 grid(unsigned((a.N + 15) / 16), unsigned(splits));
        const hipError_t e = by_type(a.dt, [&](auto S) {
            k_pairs_few<decltype(S)><<<grid, 64 * kFewWaves, 0, s>>>(a, splits, part);
            return hipGetLastError();
        });
        if (e) return e;
        const int64_t n = few_parts(a.N);
        auto* parts = reinterpret_cast<ScorePart*>(static_cast<char*>(work) + up16(int64_t(splits) * a.M * a.N * 4));
        auto* given_score = reinterpret_cast<float*>(reinterpret_cast<char*>(parts) + up16(n * a.M * int64_t(sizeof(ScorePart))));
        k_pairs_few_join<<<dim3(unsigned(a.M), unsigned(n)), 1024, 0, s>>>(a, part, splits, state ? state + a.M * kStats : nullptr, given_out,
                                                                          log_sum, state, few_each(a.N), n > 1 ? parts : nullptr, given_score);
        if (hipError_t f = hipGetLastError()) return f;
        if (n > 1) k_pairs_join<<<dim3(1), 256, 0, s>>>(a, parts, int(n), given_score, given_out, log_sum, state);
        return hipGetLastError();
    }
    const TilePlan t = tile_plan(a.dt, pair_direct(a), a.N, a.M, a.K);
    const int64_t tiles = tile_count(a.dt, t, a.N, true);
    auto* given_score = static_cast<float*>(work);
    auto* parts = reinterpret_cast<ScorePart*>(static_cast<char*>(work) + up16(a.M * 4));
    auto* part = reinterpret_cast<float*>(reinterpret_cast<char*>(parts) + up16(tiles * a.M * int64_t(sizeof(ScorePart))));
    const StatsOut o{{a.bias, a.mask, a.N, a.c}, a.given, a.M, parts, given_score};
    const hipError_t e = by_type(a.dt, [&](auto S) { return PairProducts<decltype(S)>::stats(a, t, o, part, s); });
    if (e) return e;
    k_pairs_join<<<dim3(unsigned((a.M + 15) / 16)), 256, 0, s>>>(a, parts, int(tiles), given_score, given_out, log_sum, state);
    return hipGetLastError();
}

int64_t pair_back_work(int dt, int64_t M, int64_t N, int64_t K, bool d_x, bool d_r) {
    if (M == 0 || N == 0) return 0;
    if (pair_few(M)) return d_x ? up16((N + few_per(N, K) - 1) / few_per(N, K) * M * K * 4) : 0;
    return either_plan(dt, K, [&](bool direct) { return back_layout(dt, direct, M, N, K, d_x, d_r).bytes; });
}

hipError_t launch_pair_log_probs_back(const PairArgs& a, const float* state, const float* d_given,
                                      const float* d_log_sum, void* d_x, void* d_r, float* d_bias, void* work,
                                      hipStream_t s) {
    const int size = size_of(a.dt);
    if (a.M == 0 || a.N == 0) {
        zero(d_x, a.M * a.K * size, s);
        zero(d_r, a.N * a.K * size, s);
        zero(d_bias, a.N * 4, s);
        return hipGetLastError();
    }
    if (pair_few(a.M)) {
        const int64_t per = few_per(a.N, a.K);
        const int ranges = int((a.N + per - 1) / per);
        auto* part = d_x ? static_cast<float*>(work) : nullptr;
        const dim3 grid(unsigned((a.K + 256 * kBackCols - 1) / (256 * kBackCols)), unsigned(ranges));
        return by_type(a.dt, [&](auto S) {
            using T = decltype(S);
            if (a.M == 1)
                k_pairs_few_back<T, 1><<<grid, 256, 0, s>>>(a, state, d_given, d_log_sum, per, part, d_r, d_bias);
            else if (a.M <= 4)
                k_pairs_few_back<T, 4><<<grid, 256, 0, s>>>(a, state, d_given, d_log_sum, per, part, d_r, d_bias);
            else
                k_pairs_few_back<T, 8><<<grid, 256, 0, s>>>(a, state, d_given, d_log_sum, per, part, d_r, d_bias);
            if (d_x) k_pairs_sum<T><<<match_grid((a.M * a.K + 255) / 256), 256, 0, s>>>(part, ranges, a.M * a.K, d_x);
            return hipGetLastError();
        });
    }
    const BackLayout b = back_layout(a.dt, pair_direct(a), a.M, a.N, a.K, d_x, d_r);
    char* w = static_cast<char*>(work);
    auto* coef = reinterpret_cast<PairCoef*>(w + b.coef);
    auto* scale = reinterpret_cast<float*>(w + b.scale);
    auto* look = reinterpret_cast<int*>(scale + 1);
    auto* sums = reinterpret_cast<float*>(w + b.sums);
    auto* part = reinterpret_cast<float*>(w + b.part);
    auto* dr = reinterpret_cast<float*>(w + b.dr);
    const bool half = a.dt == TP_F16;
    const int64_t blocks = (a.M + 1023) / 1024;
    k_pairs_coef<<<dim3(unsigned(blocks < 64 ? blocks : 64)), 1024, 0, s>>>(a, state, d_given, d_log_sum, half, coef, scale, look);
    if (hipError_t e = hipGetLastError()) return e;
    const PairOff none{nullptr, nullptr, 0, 0.0f};
    for (int64_t first = 0; first < a.N; first += b.references) {
        const int64_t n = std::min(a.N - first, b.references);
        const char* r = static_cast<const char*>(a.r) + first * a.ldr * size;
        const PairOff off{a.bias ? a.bias + first : nullptr, a.mask ? a.mask + first : nullptr, n, a.c};
        for (int64_t image = 0; image < a.M; image += b.images) {
            PairArgs p = a;  // (of this piece's images)
            p.M = std::min(a.M - image, b.images);
            p.x = static_cast<const char*>(a.x) + image * a.ldx * size;
            auto* dx = reinterpret_cast<float*>(w + b.dx) + image * a.K;
            const GradOut go{off, coef + image, p.M, first, w + b.g, b.ldg, d_bias ? sums : nullptr, look};
            const MatrixOut ro{off, scale, n, a.K, image ? dr : nullptr, image + p.M < a.M ? dr : nullptr,
                               d_r ? static_cast<char*>(d_r) + first * a.K * size : nullptr, a.K};
            const MatrixOut xo{none, scale, p.M, a.K, first ? dx : nullptr, first + n < a.N ? dx : nullptr,
                               d_x ? static_cast<char*>(d_x) + image * a.K * size : nullptr, a.K};
            const hipError_t e = by_type(a.dt, [&](auto S) {
                using P = PairProducts<decltype(S)>;
                if (hipError_t f = P::grad(p, r, n, b.grad, go, part, s)) return f;
                if (d_r)
                    if (hipError_t f = P::d_references(p, w + b.g, b.ldg, n, b.refs, ro, part, s)) return f;
                return d_x ? P::d_images(p, w + b.g, b.ldg, r, off, look, b.imgs, xo, part, s) : hipSuccess;
            });
            if (e) return e;
            if (d_bias) {
                k_pairs_bias<<<match_grid((n + 255) / 256), 256, 0, s>>>(sums, int(tile_count(a.dt, b.grad, p.M, false)), n,
                                                                         scale, image != 0, d_bias + first);
                if (hipError_t f = hipGetLastError()) return f;
            }
        }
    }
    return hipSuccess;
}

}  // namespace tp
