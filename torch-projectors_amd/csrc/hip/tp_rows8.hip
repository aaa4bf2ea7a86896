// Scores of images against references in 8-bit integers with a scale for each row.
//
//   quantize  scale = max |x| / 127 of a row (2^-126 at least), code = x / scale to the nearest integer, half to even;
//             both quotients rounded to fp32.  A row with a value that is not finite has scale NaN and codes 0.
//   scores    out[m, n] = (float(sum_k a[m, k] b[n, k]) sa[m]) sb[n] + bias[n], the sum in int32: exact in any order,
//             as 127^2 times 131072 values is below 2^31.
//
// Codes are evenly spaced, so a row keeps 1 / 254 of its largest value: for whitened images, whose values are all of a size,
// that is finer than 8-bit floating point's 3-bit mantissa.  Products run at 2.0 to 2.4 POP/s, 1.6 times a bfloat16 library product's rate.
#include "../../../include/torch_projectors_hip.h"
#include "tp_match.hh"
#include "tp_tile.hh"

#include <type_traits>

namespace tp {
namespace {

constexpr int kRow = kRowPad;  // bytes of a row that a step of the products takes

// ------------------------------------------------------------------ quantize
__device__ __forceinline__ uint32_t magnitude_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ float row_scale(uint32_t most) {
    return most >= 0x7f800000u ? NAN : fmaxf(__uint_as_float(most) / 127.0f, 0x1p-126f);
}
__device__ __forceinline__ uint32_t code_of(float x, float scale) {
    const float v = rintf(x / scale);
    return v == v ? uint32_t(int(fminf(fmaxf(v, -127.0f), 127.0f))) & 255u : 0u;
}
template <class S> __device__ __forceinline__ void load8(const typename S::Bits* p, int64_t n, float (&v)[8]) {
    if (n >= 8) {
#pragma unroll
        for (int i = 0; i < 8 / Pack<S>::n; ++i) {
            const Pack<S> w = load_pack<S>(p + i * Pack<S>::n);
#pragma unroll
            for (int j = 0; j < Pack<S>::n; ++j) v[i * Pack<S>::n + j] = S::widen(w.v[j]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? S::widen(p[i]) : 0.0f;
    }
}
__device__ __forceinline__ uint32_t max8(const float (&v)[8], uint32_t most) {
#pragma unroll
    for (int i = 0; i < 8; ++i) most = max(most, magnitude_bits(v[i]));
    return most;
}
__device__ __forceinline__ uint2 codes8(const float (&v)[8], float scale) {
    uint32_t c[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i / 4] |= code_of(v[i], scale) << (i % 4 * 8);
    return uint2{c[0], c[1]};
}
__device__ __forceinline__ uint32_t wave_most(uint32_t v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v = max(v, uint32_t(__shfl_xor(int(v), d)));
    return v;
}

// Eight codes.  The quotient by the reciprocal is within 2^-15 of the right one (three roundings of numbers up to 127): where it is
// not that close to a border between two codes both have the same, and the right quotient, some ten instructions, is not formed.
__device__ __forceinline__ uint2 codes8(const float (&v)[8], float scale, float inverse) {
    float c[8];
    bool close = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float q = v[i] * inverse;
        c[i] = rintf(q);
        close = close || !(fabsf(q - c[i]) < 0.5f - 0x1p-14f);
    }
    if (__builtin_amdgcn_ballot_w64(close) != 0) return codes8(v, scale);
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i / 4] |= (uint32_t(int(c[i])) & 255u) << (i % 4 * 8);
    return uint2{w[0], w[1]};
}
__device__ __forceinline__ float row_inverse(float scale) { return 1.0f / scale; }

// W wavefronts per row.  A row of at most 2048 W values stays in registers between its largest and its codes; a longer one is
// read twice.  Bytes bound it: 4096 float32 rows of 16640 values take 85 us, 4.0 TB/s read and written (105 read twice).
constexpr int kHeld = 4;  // chunks of eight values that a lane holds
template <class S, int W, bool HELD>
__global__ __launch_bounds__(W > 4 ? 64 * W : 256) void k_quantize_rows(const typename S::Bits* __restrict__ x, int64_t rows, int64_t cols,
                                                                        int64_t stride, int64_t padded, uint8_t* __restrict__ codes,
                                                                        float* __restrict__ scales) {
    constexpr int kWaves = W > 4 ? W : 4, kRows = kWaves / W;
    __shared__ uint32_t room[kWaves];
    const int wave = threadIdx.x >> 6, t = threadIdx.x % (64 * W);
    for (int64_t r0 = int64_t(blockIdx.x) * kRows; r0 < rows; r0 += int64_t(gridDim.x) * kRows) {
        const int64_t r = r0 + wave / W;
        const bool there = r < rows;
        const typename S::Bits* p = x + (there ? r : 0) * stride;
        uint32_t most = 0;
        float held[HELD ? kHeld : 1][8];
        if (there) {
            if constexpr (HELD) {
#pragma unroll
                for (int k = 0; k < kHeld; ++k) load8<S>(p + 8 * t + k * 512 * W, cols - 8 * t - k * 512 * W, held[k]);
#pragma unroll
                for (int k = 0; k < kHeld; ++k) most = max8(held[k], most);
            } else {
#pragma unroll 4
                for (int64_t c = 8 * t; c < cols; c += 512 * W) {
                    load8<S>(p + c, cols - c, held[0]);
                    most = max8(held[0], most);
                }
            }
        }
        most = wave_most(most);
        if (W > 1) {
            __syncthreads();
            if ((threadIdx.x & 63) == 0) room[wave] = most;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < W; ++i) most = max(most, room[wave / W * W + i]);
        }
        if (!there) continue;
        const float scale = row_scale(most), inverse = row_inverse(scale);
        if (t == 0) scales[r] = scale;
        uint8_t* out = codes + r * padded;
        if constexpr (HELD) {
#pragma unroll
            for (int k = 0; k < kHeld; ++k) {
                const int64_t c = 8 * t + k * 512 * W;
                if (c < padded) *reinterpret_cast<uint2*>(out + c) = codes8(held[k], scale, inverse);
            }
        } else {
            for (int64_t c = 8 * t; c < padded; c += 512 * W) {
                load8<S>(p + c, cols - c, held[0]);
                *reinterpret_cast<uint2*>(out + c) = codes8(held[0], scale, inverse);
            }
        }
    }
}

// ------------------------------------------------------------------ scores
// Few images: [splits] ranges of the rows' steps are one workgroup each, and where there are several their sums go to
// part [splits][M][N], which k_rows8_join adds up.
struct Rows8Args {
    const uint8_t* a;
    const float* sa;
    const uint8_t* b;
    const float* sb;
    int64_t M, N;
    int steps, splits;
    const float* bias;
    void* out;
    int* part;
    __device__ __forceinline__ int first(uint32_t split) const { return int(int64_t(steps) * split / splits); }
};
__device__ __forceinline__ float scaled(int sum, float sa, float sb, float bias) { return float(sum) * sa * sb + bias; }

template <class O> __global__ __launch_bounds__(256) void k_rows8_join(Rows8Args g) {
    const int64_t MN = g.M * g.N;
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < MN; i += int64_t(gridDim.x) * 256) {
        int v = 0;
#pragma unroll 4
        for (int s = 0; s < g.splits; ++s) v += g.part[s * MN + i];
        const int64_t m = over(i, uint32_t(g.N)), n = i - m * g.N;
        static_cast<typename O::Bits*>(g.out)[i] = O::round(scaled(v, g.sa[m], g.sb[n], g.bias ? g.bias[n] : 0.0f));
    }
}

// Few images: as fast as the references' codes can be read.  A workgroup takes 16 references, each of its wavefronts
// every eighth step of them, straight from memory into operands: kAhead steps' loads are in flight at once.  S: one image of
// that type, which every workgroup rounds itself (its row's largest value needs the whole row), else void and up to 16 FM images'
// codes.  (4096 references of 16640 codes: 14.3 us against 2 images' codes, 16.9 a call with the one image's rounding, 4 TB/s of the
// references; a ring of loads that never drains 15.7.)
constexpr int kFewWaves = 8, kAhead = 4;
struct OneRow {
    const void* x;
    int64_t cols;
};
constexpr int kOneMost = 32768;  // values of a row that is rounded this way (they stand in LDS)

template <int FM, class O, class S>
__global__ __launch_bounds__(64 * kFewWaves) void k_rows8_few(Rows8Args g, OneRow one) {
    constexpr bool kOne = !std::is_same<S, void>::value;
    extern __shared__ __attribute__((aligned(16))) uint8_t room[];  // the image's codes
    __shared__ int sums[kFewWaves][FM * 16][16];
    __shared__ uint32_t mosts[kFewWaves];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, r = lane & 15, q = lane >> 4;
    const int64_t n0 = int64_t(blockIdx.x) * 16, K = int64_t(g.steps) * kRow;
    const uint32_t split = blockIdx.y;
    const int k0 = g.first(split), k1 = g.first(split + 1);
    // rows past the end read the last one's codes and are not stored
    const uint8_t* pb = g.b + min(n0 + r, g.N - 1) * K + q * 16;
    const uint8_t* pa[FM];
#pragma unroll
    for (int f = 0; f < FM; ++f) pa[f] = kOne ? nullptr : g.a + min(int64_t(f * 16 + r), g.M - 1) * K + q * 16;
    v4i acc[FM];
#pragma unroll
    for (int f = 0; f < FM; ++f) acc[f] = v4i{0, 0, 0, 0};
    v4i cb[kAhead][2], ca[kAhead][FM][2];
    auto fetch = [&](int k) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (k + u * kFewWaves >= k1) break;
            const int64_t at = int64_t(k + u * kFewWaves) * kRow;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                cb[u][h] = *reinterpret_cast<const v4i*>(pb + at + h * 64);
                if constexpr (!kOne)
#pragma unroll
                    for (int f = 0; f < FM; ++f) ca[u][f][h] = *reinterpret_cast<const v4i*>(pa[f] + at + h * 64);
            }
        }
        __builtin_amdgcn_sched_barrier(0);  // all loads before the first use
    };
    fetch(k0 + wave);
    float scale = 0.0f;
    if constexpr (kOne) {
        const auto* x = static_cast<const typename S::Bits*>(one.x);
        // the first kKept x 4096 values stay in registers between their largest and their codes
        constexpr int kKept = 5;
        uint32_t most = 0;
        float kept[kKept][8], v[8];
#pragma unroll
        for (int i = 0; i < kKept; ++i) load8<S>(x + 8 * tid + i * 4096, one.cols - 8 * tid - i * 4096, kept[i]);
#pragma unroll
        for (int i = 0; i < kKept; ++i) most = max8(kept[i], most);
        for (int64_t c = 8 * tid + kKept * 4096; c < one.cols; c += 4096) {
            load8<S>(x + c, one.cols - c, v);
            most = max8(v, most);
        }
        most = wave_most(most);
        if (lane == 0) mosts[wave] = most;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kFewWaves; ++w) most = max(most, mosts[w]);
        scale = row_scale(most);
        const float inverse = row_inverse(scale);
#pragma unroll
        for (int i = 0; i < kKept; ++i)
            if (8 * tid + i * 4096 < K) *reinterpret_cast<uint2*>(room + 8 * tid + i * 4096) = codes8(kept[i], scale, inverse);
        for (int64_t c = 8 * tid + kKept * 4096; c < K; c += 4096) {
            load8<S>(x + c, one.cols - c, v);
            *reinterpret_cast<uint2*>(room + c) = codes8(v, scale, inverse);
        }
        __syncthreads();
    }
    for (int k = k0 + wave; k < k1; k += kFewWaves * kAhead) {
        if (k != k0 + wave) fetch(k);
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int at = k + u * kFewWaves;
            if (at >= k1) break;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int f = 0; f < FM; ++f) {
                    const v4i a = kOne ? *reinterpret_cast<const v4i*>(room + at * kRow + h * 64 + q * 16) : ca[u][f][h];
                    acc[f] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, cb[u][h], acc[f], 0, 0, 0);
                }
        }
    }
#pragma unroll
    for (int f = 0; f < FM; ++f)
#pragma unroll
        for (int j = 0; j < 4; ++j) sums[wave][f * 16 + 4 * q + j][r] = acc[f][j];
    __syncthreads();
    for (int i = tid; i < FM * 256; i += 64 * kFewWaves) {
        const int64_t m = i >> 4, n = n0 + (i & 15);
        if (m >= g.M || n >= g.N) continue;
        int v = 0;
#pragma unroll
        for (int w = 0; w < kFewWaves; ++w) v += sums[w][m][i & 15];
        if (g.splits > 1)
            g.part[(int64_t(split) * g.M + m) * g.N + n] = v;
        else
            static_cast<typename O::Bits*>(g.out)[m * g.N + n] =
                O::round(scaled(v, kOne ? scale : g.sa[m], g.sb[n], g.bias ? g.bias[n] : 0.0f));
    }
}

// Many images: the products in tiles of tp_tile.hh, scaled on their way out.  4096 x 8192 x 16640 takes 470 to 550 us, 2.0 to 2.4 POP/s (a library
// product 2.15 at 8192 each way): matrix units 54 % busy, wavefronts waiting 48 % of their time for a turn at them and 30 % for loads and each other.
struct ScaledOut {
    const float *sa, *sb;  // of the tile's rows (images) and columns (references)
    const float* bias;
    void* out;
    int64_t M, N;
};
template <class O> struct ScaledEpi {
    using Args = ScaledOut;
    template <class S> static constexpr bool kTwice = false;
    template <class S, class T>
    static __device__ __forceinline__ void run(const Args& g, Acc<T>& acc, uint32_t im, uint32_t in, char* lds) {
        const Place<T> place(threadIdx.x);
        const int64_t m0 = int64_t(im) * T::BM, n0 = int64_t(in) * T::BN;
        float sb[T::FN], off[T::FN];
#pragma unroll
        for (int j = 0; j < T::FN; ++j) {
            const int64_t n = n0 + place.col(j);
            sb[j] = n < g.N ? g.sb[n] : 0.0f;
            off[j] = g.bias && n < g.N ? g.bias[n] : 0.0f;
        }
        float* sa = reinterpret_cast<float*>(lds + T::NT / 64 * Rows4<T>::kBytes);  // (behind the fragments' rows)
        static_assert(T::NT / 64 * Rows4<T>::kBytes + T::BM * 4 <= tile_lds<S, T>(), "LDS of the products");
        for (int i = threadIdx.x; i < T::BM; i += T::NT) sa[i] = m0 + i < g.M ? g.sa[m0 + i] : 0.0f;
        __syncthreads();
        const float* mine = sa + place.first();
        auto* out = static_cast<typename O::Bits*>(g.out);
#pragma unroll
        for (int i = 0; i < T::FM; ++i) {
            v16f row[T::FN];
#pragma unroll
            for (int e = 0; e < 16; ++e)
#pragma unroll
                for (int j = 0; j < T::FN; ++j)
                    row[j][e] = scaled(int(__float_as_uint(acc[i][j][e])), mine[place.at(i, e)], sb[j], off[j]);
            Rows4<T>::run(row, i, lds, [&](int at, int col, float4 v) {
                const int64_t m = m0 + at, n = n0 + col;
                if (m >= g.M || n >= g.N) return;
                const typename O::Bits b[4] = {O::round(v.x), O::round(v.y), O::round(v.z), O::round(v.w)};
                if (n + 4 <= g.N) {
                    __builtin_memcpy(out + m * g.N + n, b, sizeof b);
                } else {
#pragma unroll
                    for (int k = 0; k < 3; ++k)
                        if (n + k < g.N) out[m * g.N + n + k] = b[k];
                }
            });
        }
    }
};

// ------------------------------------------------------------------ which kernel
struct Rows8Plan {
    int few, splits;  // FM of k_rows8_few and its ranges, or 0: tiles
};

// The tiles' plan is that of 16-bit products: their steps are as long, as many bytes go through LDS for as many instructions.
TilePlan rows8_tiles(int64_t M, int64_t N, int64_t steps) { return tile_plan(TP_BF16, true, M, N, steps * kRow / 2); }

// One image, and few images of not too many references: k_rows8_few, which reads them at up to 5 TB/s but for every 16 images again.  The
// borders by references and by bytes of their codes, each varied with the other held (us, k_rows8_few / tiles):
//   8 images    8192 references of 1024, 4224, 16640 codes 4.4 / 5.8, 9.7 / 13.8, 28 / 28; 16384: 7.2 / 5.9, 17 / 19, 56 / 52; 36864: 16 / 9.9, 36 / 27, 133 / 129
//   16 images   4096: 3.4 / 5.8, 6.1 / 14.2, 17.7 / 19.6; 8192: 5.0 / 6.0, 11.1 / 14.1, 33 / 29; 16384: 8.1 / 6.1, 19.8 / 19.1, 65 / 53
//   32 images   2048: 4.0 / 6.1, 8.0 / 11.2, 16.3 / 17.0; 4096: 3.9 / 6.0, 7.9 / 14.3, 25 / 20; 8192: 6.3 / 6.1, 15.3 / 14.2, 48 / 29
Rows8Plan rows8_plan(int64_t M, int64_t N, int64_t steps) {
    Rows8Plan p{M <= 16 ? 1 : 2, 1};
    if (M == 1) return p;  // (its image is rounded in the same launch)
    const int64_t groups = (N + 15) / 16, bytes = N * steps * kRow;
    const bool streams = M <= 8 ? N <= 16384 : M <= 16 ? N <= 8192 && bytes <= 80 << 20 : M <= 32 && N <= 4096 && bytes <= 36 << 20;
    if (!streams) return {0, 1};
    const int64_t wanted = (kCus + groups - 1) / groups, most = (steps + kFewWaves * kAhead - 1) / (kFewWaves * kAhead);
    p.splits = int(wanted > most ? most : wanted);
    return p;
}

template <class O> hipError_t row_scores(const Rows8Args& g, const Rows8Plan& p, hipStream_t s) {
    if (!p.few) {
        const int64_t half = int64_t(g.steps) * kRow / 2;  // (pairs of codes)
        const TilePlan t = rows8_tiles(g.M, g.N, g.steps);
        const Product product{{g.a, half, half, nullptr, nullptr, nullptr}, {g.b, half, half, nullptr, nullptr, nullptr}, g.M, g.N, half, 0, 0, 0,
                              t.whole, t.splits, reinterpret_cast<float*>(g.part)};
        return tp::product<I8x2, false, false, ScaledEpi<O>>(product, t, ScaledOut{g.sa, g.sb, g.bias, g.out, g.M, g.N}, s);
    }
    const dim3 grid(unsigned((g.N + 15) / 16), unsigned(p.splits));
    if (p.few == 1)
        k_rows8_few<1, O, void><<<grid, 64 * kFewWaves, 0, s>>>(g, OneRow{});
    else
        k_rows8_few<2, O, void><<<grid, 64 * kFewWaves, 0, s>>>(g, OneRow{});
    if (hipError_t e = hipGetLastError()) return e;
    if (p.splits > 1) k_rows8_join<O><<<match_grid((g.M * g.N + 255) / 256), 256, 0, s>>>(g);
    return hipGetLastError();
}

template <class S> void quantize(const void* x, int64_t rows, int64_t cols, int64_t stride, void* codes, void* scales, hipStream_t s) {
    const auto* p = static_cast<const typename S::Bits*>(x);
    auto* c = static_cast<uint8_t*>(codes);
    auto* f = static_cast<float*>(scales);
    const int64_t padded = row_bytes(cols);
    // (rows of 512, 4096, 16640 float32 values: 1, 2 and 16 wavefronts a row)
    if (cols <= 512 * kHeld)
        k_quantize_rows<S, 1, true><<<match_grid((rows + 3) / 4), 256, 0, s>>>(p, rows, cols, stride, padded, c, f);
    else if (cols <= 1024 * kHeld)
        k_quantize_rows<S, 2, true><<<match_grid((rows + 1) / 2), 256, 0, s>>>(p, rows, cols, stride, padded, c, f);
    else if (cols <= 2048 * kHeld)
        k_quantize_rows<S, 4, true><<<match_grid(rows), 256, 0, s>>>(p, rows, cols, stride, padded, c, f);
    else if (cols <= 4096 * kHeld)
        k_quantize_rows<S, 8, true><<<match_grid(rows), 512, 0, s>>>(p, rows, cols, stride, padded, c, f);
    else if (cols <= 8192 * kHeld)
        k_quantize_rows<S, 16, true><<<match_grid(rows), 1024, 0, s>>>(p, rows, cols, stride, padded, c, f);
    else
        k_quantize_rows<S, 16, false><<<match_grid(rows), 1024, 0, s>>>(p, rows, cols, stride, padded, c, f);
}

// One image is rounded by the product's own kernel where its codes fit LDS beside others.
bool rounds_itself(int64_t M, int64_t cols) { return M == 1 && cols <= kOneMost; }

int64_t up16(int64_t bytes) { return (bytes + 15) / 16 * 16; }

}  // namespace

hipError_t launch_quantize_rows(int dt, const void* x, int64_t rows, int64_t cols, int64_t stride, void* codes,
                                void* scales, hipStream_t s) {
    switch (dt) {
        case TP_F32: quantize<F32>(x, rows, cols, stride, codes, scales, s); break;
        case TP_F16: quantize<F16>(x, rows, cols, stride, codes, scales, s); break;
        default: quantize<BF16>(x, rows, cols, stride, codes, scales, s);
    }
    return hipGetLastError();
}

int64_t row_scores_work(int64_t M, int64_t N, int64_t bytes) {
    const Rows8Plan p = rows8_plan(M, N, bytes / kRow);
    if (!p.few) return tile_part_bytes(TP_BF16, rows8_tiles(M, N, bytes / kRow), M, N);
    return p.splits > 1 ? up16(p.splits * M * N * int64_t(sizeof(int))) : 0;
}

hipError_t launch_row_scores(const void* a, const void* sa, int64_t M, const void* b, const void* sb, int64_t N,
                             int64_t bytes, const void* bias, int out_dt, void* out, void* work, hipStream_t s) {
    const Rows8Plan p = rows8_plan(M, N, bytes / kRow);
    const Rows8Args g{static_cast<const uint8_t*>(a), static_cast<const float*>(sa), static_cast<const uint8_t*>(b),
                      static_cast<const float*>(sb), M, N, int(bytes / kRow), p.splits, static_cast<const float*>(bias),
                      out, static_cast<int*>(work)};
    return out_dt == TP_F32 ? row_scores<F32>(g, p, s) : row_scores<BF16>(g, p, s);
}

// (the sums of the product's ranges, then codes and scales from a 16-byte boundary on)
int64_t row_score_images_work(int64_t M, int64_t N, int64_t cols) {
    const int64_t bytes = row_bytes(cols);
    if (rounds_itself(M, cols)) return 0;
    return row_scores_work(M, N, bytes) + M * bytes + M * int64_t(sizeof(float));
}

template <class S> hipError_t score_one(const Rows8Args& g, const OneRow& one, int out_dt, hipStream_t s) {
    const dim3 grid(unsigned((g.N + 15) / 16));
    const unsigned lds = unsigned(g.steps * kRow);
    if (out_dt == TP_F32)
        k_rows8_few<1, F32, S><<<grid, 64 * kFewWaves, lds, s>>>(g, one);
    else
        k_rows8_few<1, BF16, S><<<grid, 64 * kFewWaves, lds, s>>>(g, one);
    return hipGetLastError();
}

hipError_t launch_row_score_images(int dt, const void* x, int64_t M, int64_t cols, int64_t stride, const void* b,
                                   const void* sb, int64_t N, const void* bias, int out_dt, void* out, void* work,
                                   hipStream_t s) {
    const int64_t bytes = row_bytes(cols);
    if (rounds_itself(M, cols)) {
        const Rows8Args g{nullptr, nullptr, static_cast<const uint8_t*>(b), static_cast<const float*>(sb), 1, N,
                          int(bytes / kRow), 1, static_cast<const float*>(bias), out, nullptr};
        const OneRow one{x, cols};
        return dt == TP_F32 ? score_one<F32>(g, one, out_dt, s) : dt == TP_F16 ? score_one<F16>(g, one, out_dt, s)
                                                                               : score_one<BF16>(g, one, out_dt, s);
    }
    auto* part = static_cast<char*>(work);
    auto* codes = part + row_scores_work(M, N, bytes);
    auto* scales = codes + M * bytes;
    if (hipError_t e = launch_quantize_rows(dt, x, M, cols, stride, codes, scales, s)) return e;
    return launch_row_scores(codes, scales, M, b, sb, N, bytes, bias, out_dt, out, part, s);
}

}  // namespace tp
