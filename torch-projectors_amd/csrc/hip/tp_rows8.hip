// Scores of images against references in 8-bit integers with a scale for each row.
//
//   quantize  scale = max |x| / 127 of a row (2^-126 at least), code = x / scale to the nearest integer, half to even;
//             both quotients rounded to fp32.  A row with a value that is not finite has scale NaN and codes 0.
//   scores    out[m, n] = (float(sum_k a[m, k] b[n, k]) sa[m]) sb[n] + bias[n], the sum in int32: exact in any order,
//             as 127^2 times 131072 values is below 2^31.
//
// Codes are evenly spaced, so a row keeps 1 / 254 of its largest value: for whitened images, whose values are all of a size,
// that is finer than 8-bit floating point's 3-bit mantissa, at twice the rate of the bfloat16 units which those need.
#include "../../../include/torch_projectors_hip.h"
#include "tp_match.hh"
#include "tp_stage.hh"

#include <type_traits>

namespace tp {
namespace {

using v4i = __attribute__((ext_vector_type(4))) int;
using v16i = __attribute__((ext_vector_type(16))) int;
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

// W wavefronts per row, which read it twice: the second time it comes from the caches.
template <class S, int W>
__global__ __launch_bounds__(256) void k_quantize_rows(const typename S::Bits* __restrict__ x, int64_t rows, int64_t cols,
                                                       int64_t stride, int64_t padded, uint8_t* __restrict__ codes,
                                                       float* __restrict__ scales) {
    __shared__ uint32_t room[4];
    const int wave = threadIdx.x >> 6, t = threadIdx.x & (64 * W - 1);
    for (int64_t r0 = int64_t(blockIdx.x) * (4 / W); r0 < rows; r0 += int64_t(gridDim.x) * (4 / W)) {
        const int64_t r = r0 + wave / W;
        const bool there = r < rows;
        const typename S::Bits* p = x + (there ? r : 0) * stride;
        uint32_t most = 0;
        float v[8];
        if (there)
#pragma unroll 4
            for (int64_t c = 8 * t; c < cols; c += 512 * W) {
                load8<S>(p + c, cols - c, v);
                most = max8(v, most);
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
        const float scale = row_scale(most);
        if (t == 0) scales[r] = scale;
#pragma unroll 4
        for (int64_t c = 8 * t; c < padded; c += 512 * W) {
            load8<S>(p + c, cols - c, v);
            *reinterpret_cast<uint2*>(codes + r * padded + c) = codes8(v, scale);
        }
    }
}

// ------------------------------------------------------------------ scores
// [splits] ranges of the rows' steps are one workgroup each, and where there are several their sums go to part
// [splits][M][N], which k_rows8_join adds up.
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
// codes.
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
            const int64_t at = int64_t(min(k + u * kFewWaves, k1 - 1)) * kRow;
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
    fetch(min(k0 + wave, k1 - 1));
    float scale = 0.0f;
    if constexpr (kOne) {
        const auto* x = static_cast<const typename S::Bits*>(one.x);
        uint32_t most = 0;
        float v[8];
        for (int64_t c = 8 * tid; c < one.cols; c += 512 * kFewWaves) {
            load8<S>(x + c, one.cols - c, v);
            most = max8(v, most);
        }
        most = wave_most(most);
        if (lane == 0) mosts[wave] = most;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kFewWaves; ++w) most = max(most, mosts[w]);
        scale = row_scale(most);
        for (int64_t c = int64_t(k0) * kRow + 8 * tid; c < int64_t(k1) * kRow; c += 512 * kFewWaves) {
            load8<S>(x + c, one.cols - c, v);
            *reinterpret_cast<uint2*>(room + (c - int64_t(k0) * kRow)) = codes8(v, scale);
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
                    const v4i a = kOne ? *reinterpret_cast<const v4i*>(room + (at - k0) * kRow + h * 64 + q * 16) : ca[u][f][h];
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

// The product in tiles: a workgroup of WM x WN x KW wavefronts computes BM x BN scores.  One step of a tile's rows in
// LDS is 128 bytes each, fragment after fragment (fragment f of a part of the tile has its rows F r + f, r < 32), and the
// 16-byte chunks of a row permuted among themselves (chunk c of row r of a fragment at place c ^ ((r / 2) & 7)), so
// that the 16 lanes that read one chunk of 16 rows at a time reach each of the 64 banks once.
template <int BM, int BN> struct alignas(16) Stage8 {
    uint8_t a[BM * kRow], b[BN * kRow];
};

template <int BM, int BN, int WM, int WN, int KW, class O>
__global__ __launch_bounds__(64 * WM * WN * KW, BM * BN == 128 * 128 ? 4 : 1) void k_rows8_tile(Rows8Args g, uint32_t tm, uint32_t tn) {
    constexpr int W = WM * WN * KW, FM = BM / WM / 32, FN = BN / WN / 32, NT = 4 / KW;
    constexpr int LA = BM / 8 / W, LB = BN / 8 / W;  // loads of a wavefront for a stage
    static_assert(LA * W * 8 == BM && LB * W * 8 == BN, "whole loads");
    __shared__ Stage8<BM, BN> stages[2];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, r = lane & 31, q = lane >> 5;
    const int kw = wave % KW, wm = wave / KW / WN, wn = wave / KW % WN;
    // workgroups are dealt to the XCDs in turn: each XCD takes a contiguous run of the items, whose tiles
    // share rows and columns in its L2
    const uint32_t items = gridDim.x, x = blockIdx.x & 7, per = items >> 3, more = items & 7;
    uint32_t item = x * per + min(x, more) + (blockIdx.x >> 3);
    const uint32_t split = item / (tm * tn);
    item -= split * tm * tn;
    // tiles in bands of 4 along M, column by column
    const uint32_t band = item / (4 * tn), at = item - band * 4 * tn, height = min(4u, tm - band * 4);
    const int64_t m0 = int64_t(band * 4u + at % height) * BM, n0 = int64_t(at / height) * BN;
    const int k0 = g.first(split), k1 = g.first(split + 1);
    const int64_t K = int64_t(g.steps) * kRow;

    uint32_t oa[LA], ob[LB];
    const int row8 = lane >> 3, place = lane & 7;
    auto offset = [&](int slot, int F) {  // of a row's place in LDS and this lane's chunk there
        const int rr = slot & 31, f = (slot >> 5) % F, part = (slot >> 5) / F;
        return uint32_t(((part * 32 + rr) * F + f) * K) + (place ^ ((rr >> 1) & 7)) * 16;
    };
#pragma unroll
    for (int i = 0; i < LA; ++i) oa[i] = offset((wave * LA + i) * 8 + row8, FM);
#pragma unroll
    for (int i = 0; i < LB; ++i) ob[i] = offset((wave * LB + i) * 8 + row8, FN);
    // rows past the end read zeros
    const auto ga = codes_buffer(g.a + m0 * K, min(int64_t(BM), g.M - m0), K);
    const auto gb = codes_buffer(g.b + n0 * K, min(int64_t(BN), g.N - n0), K);
    v16i acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;
    auto load = [&](Stage8<BM, BN>& st, int k) {
        to_lds(ga, oa, k * kRow, st.a + wave * LA * 1024);
        to_lds(gb, ob, k * kRow, st.b + wave * LB * 1024);
    };
    const int key = (r >> 1) & 7;
    load(stages[0], k0);
#pragma unroll 1
    for (int k = k0; k < k1; ++k) {
        const int cur = (k - k0) & 1;
        stage_ready();
        const uint8_t* sa = stages[cur].a + (wm * 32 * FM + r) * kRow;
        const uint8_t* sb = stages[cur].b + (wn * 32 * FN + r) * kRow;
        v4i fa[2][FM], fb[2][FN];
        auto read = [&](int t) {
            const int c = ((2 * (kw * NT + t) + q) ^ key) * 16;
#pragma unroll
            for (int f = 0; f < FM; ++f) fa[t & 1][f] = *reinterpret_cast<const v4i*>(sa + f * 32 * kRow + c);
#pragma unroll
            for (int f = 0; f < FN; ++f) fb[t & 1][f] = *reinterpret_cast<const v4i*>(sb + f * 32 * kRow + c);
        };
        read(0);
        if (k + 1 < k1) load(stages[cur ^ 1], k + 1);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            if (t + 1 < NT) read(t + 1);
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fa[t & 1][i], fb[t & 1][j], acc[i][j], 0, 0, 0);
        }
    }

    // a wavefront's share of its part's results: elements e0 .. e0 + EN - 1 of each fragment
    constexpr int EN = 16 / KW;
    const int e0 = kw * EN;
    int sum[FM][FN][EN];
    if constexpr (KW == 1) {
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int e = 0; e < EN; ++e) sum[i][j][e] = acc[i][j][e];
    } else {
        int* room = reinterpret_cast<int*>(stages);
        static_assert(sizeof(stages) >= size_t(W) * 4096, "a fragment of every wavefront");
        const int* part = room + (wave - kw) * 1024 + e0 * 64 + lane;
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                __syncthreads();
#pragma unroll
                for (int e = 0; e < 16; ++e) room[wave * 1024 + e * 64 + lane] = acc[i][j][e];
                __syncthreads();
#pragma unroll
                for (int e = 0; e < EN; ++e) {
                    int v = part[e * 64];
#pragma unroll
                    for (int w = 1; w < KW; ++w) v += part[w * 1024 + e * 64];
                    sum[i][j][e] = v;
                }
            }
    }

    const int64_t n = n0 + (wn * 32 + r) * FN;
    const bool whole = n + FN <= g.N;
    float off[FN], sb[FN];
#pragma unroll
    for (int j = 0; j < FN; ++j) {
        const bool there = n + j < g.N;
        off[j] = g.bias && there ? g.bias[n + j] : 0.0f;
        sb[j] = there ? g.sb[n + j] : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int e = 0; e < EN; ++e) {
            const int at_e = e0 + e;
            const int64_t m = m0 + (wm * 32 + (at_e / 4) * 8 + q * 4 + at_e % 4) * FM + i;
            if (m >= g.M) continue;
            if (g.splits > 1) {
                int* p = g.part + (int64_t(split) * g.M + m) * g.N + n;
                if (whole) {
                    int v[FN];
#pragma unroll
                    for (int j = 0; j < FN; ++j) v[j] = sum[i][j][e];
                    __builtin_memcpy(p, v, sizeof v);
                } else {
#pragma unroll
                    for (int j = 0; j < FN; ++j)
                        if (n + j < g.N) p[j] = sum[i][j][e];
                }
                continue;
            }
            const float sa = g.sa[m];
            auto* p = static_cast<typename O::Bits*>(g.out) + m * g.N + n;
            typename O::Bits v[FN];
#pragma unroll
            for (int j = 0; j < FN; ++j) v[j] = O::round(scaled(sum[i][j][e], sa, sb[j], off[j]));
            if (whole) {
                __builtin_memcpy(p, v, sizeof v);
            } else {
#pragma unroll
                for (int j = 0; j < FN; ++j)
                    if (n + j < g.N) p[j] = v[j];
            }
        }
}

// ------------------------------------------------------------------ which kernel
struct Rows8Plan {
    int few, tile, splits;  // few: FM of k_rows8_few, or 0; tile: index of kTiles
};
struct TileKind {
    int bm, bn;
    double step_us, alone_us;
};
constexpr TileKind kTiles[] = {{64, 64, 0.14, 0.40}, {128, 128, 0.45, 0.7}, {256, 256, 1.6, 1.4}};
constexpr int kCus = 256, kMaxSplits = 16;
constexpr int64_t kMaxTiles = int64_t(1) << 22;  // (a launch has fewer than 2^32 lanes)

Rows8Plan rows8_plan(int64_t M, int64_t N, int64_t steps) {
    Rows8Plan best{M <= 16 ? 1 : 2, 0, 1};
    double least = 1e300;
    if (M == 1) return best;  // (its image is rounded in the same launch)
    if (M <= 32) {
        const int64_t groups = (N + 15) / 16;
        int64_t s = (kCus + groups - 1) / groups;
        const int64_t most = (steps + kFewWaves * kAhead - 1) / (kFewWaves * kAhead);
        best.splits = int(s > most ? most : s);
        if (M <= 16) return best;
        least = (2.5 + 0.15 * steps) * double((N + 16 * kCus - 1) / (16 * kCus));
    }
    for (int t = 0; t < 3; ++t) {
        const TileKind& kind = kTiles[t];
        const int64_t tiles = ((M + kind.bm - 1) / kind.bm) * ((N + kind.bn - 1) / kind.bn);
        if (tiles > kMaxTiles) continue;
        for (int s = 1; s <= kMaxSplits && s <= steps; ++s) {
            if (s > 1 && tiles * s > 8 * kCus) break;
            const double each = double((tiles * s + kCus - 1) / kCus);
            double us = 2.0 + ((steps + s - 1) / s + 2) * (each * kind.step_us > kind.alone_us ? each * kind.step_us : kind.alone_us);
            if (s > 1) us += 4.0 + double(M) * N * (8 * s + 4) / 4.5e6;
            if (us < least) {
                least = us;
                best = {0, t, s};
            }
        }
    }
    return best;
}

template <class O> hipError_t row_scores(const Rows8Args& g, const Rows8Plan& p, hipStream_t s) {
    if (p.few) {
        const dim3 grid(unsigned((g.N + 15) / 16), unsigned(p.splits));
        if (p.few == 1)
            k_rows8_few<1, O, void><<<grid, 64 * kFewWaves, 0, s>>>(g, OneRow{});
        else
            k_rows8_few<2, O, void><<<grid, 64 * kFewWaves, 0, s>>>(g, OneRow{});
    } else {
        const TileKind& kind = kTiles[p.tile];
        const uint32_t tm = uint32_t((g.M + kind.bm - 1) / kind.bm), tn = uint32_t((g.N + kind.bn - 1) / kind.bn);
        const dim3 grid(tm * tn * p.splits);
        if (p.tile == 0)
            k_rows8_tile<64, 64, 1, 1, 4, O><<<grid, 256, 0, s>>>(g, tm, tn);
        else if (p.tile == 1)
            k_rows8_tile<128, 128, 2, 2, 2, O><<<grid, 512, 0, s>>>(g, tm, tn);
        else
            k_rows8_tile<256, 256, 2, 4, 1, O><<<grid, 512, 0, s>>>(g, tm, tn);
    }
    if (hipError_t e = hipGetLastError()) return e;
    if (p.splits > 1) k_rows8_join<O><<<match_grid((g.M * g.N + 255) / 256), 256, 0, s>>>(g);
    return hipGetLastError();
}

template <class S> void quantize(const void* x, int64_t rows, int64_t cols, int64_t stride, void* codes, void* scales, hipStream_t s) {
    const auto* p = static_cast<const typename S::Bits*>(x);
    auto* c = static_cast<uint8_t*>(codes);
    auto* f = static_cast<float*>(scales);
    const int64_t padded = row_bytes(cols);
    if (cols <= 2048)
        k_quantize_rows<S, 1><<<match_grid((rows + 3) / 4), 256, 0, s>>>(p, rows, cols, stride, padded, c, f);
    else
        k_quantize_rows<S, 4><<<match_grid(rows), 256, 0, s>>>(p, rows, cols, stride, padded, c, f);
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
