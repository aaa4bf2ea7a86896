// Scores of images against references in 8-bit blocks.
//
//   quantize  each block of 128 values of a row gets the least exponent e with max |x| <= 448 2^e (448
//             being the largest e4m3 value) and the codes round(x 2^-e), to nearest even.  The scale is a
//             power of two, so that scaling is exact and the matrix units apply it themselves.
//   scores    out[m, n] = bias[n] + sum_b 2^(ea + eb) sum_k a[m, k] b[n, k], summed in fp32.
//
// The matrix units' own 8-bit products align each eight of them to about 14 bits before they add them (a
// product of 4 beside one of 65536 is lost; random blocks come out 1.7e-5 off, where the type's sums have
// 24 bits).  So the codes are widened to bfloat16, one v_cvt_scalef32_pk_bf16_fp8 per two values, and multiplied by
// the bfloat16 units, whose products are exact and whose sums are fp32 (7e-9 off on the same blocks).  That is what it
// costs: an 8-bit library product of 8192^3 reaches 3.03 PFLOP/s on this card, a bfloat16 one 1.40.
// bfloat16 holds a code times its scale exactly for scales of 2^-124 to 2^119 (bytes 3 to 246).  Blocks whose largest
// value is below 448 2^-125 = 1.05e-35 (bytes 0 to 2) have theirs rounded to multiples of 2^-133, and values from 248
// 2^120 = 3.297e38 up, whose nearest code stands for 2^128, are infinite.
//
// The order of the values within an instruction's operands does not matter as long as both sides have the
// same.
#include "../../../include/torch_projectors_hip.h"
#include "tp_match.hh"

#include <type_traits>

namespace tp {
namespace {

using v4f = __attribute__((ext_vector_type(4))) float;

// ------------------------------------------------------------------ quantize
// Exponent of a block whose largest finite magnitude has these bits: 448 = 1.75 2^8, so one more where the mantissa
// is past 1.75 (a carry).  Subnormal ones are far below 2^-127 448.
__device__ __forceinline__ int block_exponent(uint32_t most) {
    return most ? max(int((most + 0x1fffffu) >> 23) - 135, -127) : 0;
}
__device__ __forceinline__ float power_of_2(int e) { return __uint_as_float(uint32_t(e + 127) << 23); }  // -126 .. 127
// The bits of a finite value's magnitude (they are in the order of the magnitudes), 0 for others.
__device__ __forceinline__ uint32_t magnitude(float x) {
    const uint32_t m = __float_as_uint(x) & 0x7fffffffu;
    return m < 0x7f800000u ? m : 0u;
}

// Codes of two values: to nearest even, NaN for what is not finite.
__device__ __forceinline__ uint32_t codes2(float x, float y, float f) {
    const uint32_t two = uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(x * f, y * f, 0, false)) & 0xffffu;
    return two | (isfinite(x) ? 0u : 0x7fu) | (isfinite(y) ? 0u : 0x7f00u);
}
// Codes of eight values: to nearest even, NaN for what is not finite.
__device__ __forceinline__ uint2 codes8(const float (&x)[8], int e) {
    const float f = power_of_2(-e);
    uint32_t c[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const float* v = x + 4 * h;
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * f, v[1] * f, 0, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * f, v[3] * f, w, true);
        c[h] = uint32_t(w);
    }
    bool finite = true;
#pragma unroll
    for (int i = 0; i < 8; ++i) finite = finite && isfinite(x[i]);
    if (!finite) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (!isfinite(x[i])) c[i / 4] |= 0x7fu << (i % 4 * 8);
    }
    return uint2{c[0], c[1]};
}

// 16 lanes per block of a row, eight values each.  Memory bound: reads each value once, writes a byte for it
// (4096 x 16640 fp32 in 61 us, 5.6 TB/s; streamed loads take 64).
template <class S>
__global__ __launch_bounds__(256) void k_quantize(const typename S::Bits* __restrict__ x, int64_t rows, int64_t cols,
                                                  int64_t stride, int nb, int64_t srows, uint8_t* __restrict__ codes,
                                                  uint8_t* __restrict__ scales) {
    const int part = threadIdx.x & 15;
    const uint32_t span = (nb + 15) / 16;  // workgroups of a row
    for (int64_t g = blockIdx.x; g < srows * span; g += gridDim.x) {
        const int64_t r = over(g, span), b = (g - r * span) * 16 + (threadIdx.x >> 4);
        if (b >= nb) continue;
        if (r >= rows) {  // the padding rows' scales
            if (part == 0) scales[b * srows + r] = 127;
            continue;
        }
        const int64_t c = b * kScaleBlock + 8 * part;
        const typename S::Bits* p = x + r * stride + c;
        float v[8];
        if (c + 8 <= cols) {
            Pack<S> w[8 / Pack<S>::n];
#pragma unroll
            for (int i = 0; i < 8 / Pack<S>::n; ++i) w[i] = load_pack<S>(p + i * Pack<S>::n);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = S::widen(w[i / Pack<S>::n].v[i % Pack<S>::n]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = c + i < cols ? S::widen(p[i]) : 0.0f;
        }
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) most = max(most, magnitude(v[i]));
#pragma unroll
        for (int d = 8; d; d >>= 1) most = max(most, uint32_t(__shfl_xor(int(most), d)));
        const int e = block_exponent(most);
        if (part == 0) scales[b * srows + r] = uint8_t(e + 127);
        *reinterpret_cast<uint2*>(codes + (r * nb + b) * kScaleBlock + 8 * part) = codes8(v, e);
    }
}

// ------------------------------------------------------------------ scores
using v8bf = __attribute__((ext_vector_type(8))) __bf16;
using v2bf = __attribute__((ext_vector_type(2))) __bf16;

// A scale byte as the power of two it stands for (0: 2^-127, a subnormal).
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(max(byte << 23, 0x00400000u)); }

// Eight codes times their block's scale: exact for scales of 2^-124 to 2^119.
__device__ __forceinline__ v8bf widen8(int lo, int hi, float scale) {
    const v2bf a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false);
    const v2bf b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
    const v2bf c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false);
    const v2bf d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
    return v8bf{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Largest of a wavefront's values, in every lane.
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    // row_shr:1, 2, 4, 8, then row_bcast:15 and 31: lane 63 has seen all (0 where none is brought)
    v = max(v, uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x111, 0xf, 0xf, false)));
    v = max(v, uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x112, 0xf, 0xf, false)));
    v = max(v, uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x114, 0xf, 0xf, false)));
    v = max(v, uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x118, 0xf, 0xf, false)));
    v = max(v, uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x142, 0xf, 0xf, false)));
    v = max(v, uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x143, 0xf, 0xf, false)));
    return uint32_t(__builtin_amdgcn_readlane(int(v), 63));
}

// What the kernels of the product share: [splits] ranges of the nb blocks are one workgroup each, and
// where there are several their sums go to part [splits][M][N], which k_scores_join adds up.
struct ScoreArgs {
    const uint8_t *a, *sa, *b, *sb;
    int64_t M, N, sra, srb;
    int nb, splits;
    const float* bias;
    void* out;
    float* part;
    __device__ __forceinline__ int first(uint32_t split) const { return int(int64_t(nb) * split / splits); }
};

template <class O> __device__ __forceinline__ void store_score(const ScoreArgs& g, uint32_t split, int64_t m, int64_t n, float v) {
    if (g.splits > 1)
        g.part[(int64_t(split) * g.M + m) * g.N + n] = v;
    else
        static_cast<typename O::Bits*>(g.out)[m * g.N + n] = O::round(v + (g.bias ? g.bias[n] : 0.0f));
}

template <class O> __global__ __launch_bounds__(256) void k_scores_join(ScoreArgs g) {
    const int64_t MN = g.M * g.N;
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < MN; i += int64_t(gridDim.x) * 256) {
        float v = 0.0f;
#pragma unroll 4
        for (int s = 0; s < g.splits; ++s) v += g.part[s * MN + i];
        if (g.bias) v += g.bias[uint64_t(i) < (uint64_t(1) << 32) ? uint32_t(i) % uint32_t(g.N) : i % g.N];
        static_cast<typename O::Bits*>(g.out)[i] = O::round(v);
    }
}

// Few images (at most 16 FM): as fast as the references' codes can be read.  A workgroup takes 16 references,
// each of its wavefronts every eighth block of them, straight from memory into operands: kAhead blocks'
// loads are in flight at once (8 KB a wavefront, 64 KB a CU).  One image against 4096 references of 16640
// values: 14.9 us, 4.6 TB/s; against 64 to 2048 12 us, as 16 wavefronts take, too: what a CU can have on its way, the
// other CUs being idle, as a row's blocks are not dealt out over workgroups (the bytes of 1024 references are 2.6 us).
constexpr int kFewWaves = 8, kAhead = 4;

// A row that a wavefront quantises itself, block by block: no launch and no memory for its codes.
struct OneImage {
    const void* x;
    int64_t cols;
};

template <int FM, class O, class S>
__global__ __launch_bounds__(64 * kFewWaves) __attribute__((amdgpu_waves_per_eu(2, 2))) void k_scores_few(ScoreArgs g,
                                                                                                       OneImage one) {
    constexpr bool kOne = !std::is_same<S, void>::value;  // (M is 1; the image's codes and scales are not given)
    __shared__ float sums[kFewWaves][FM * 16][16];
    __shared__ __attribute__((aligned(16))) uint32_t wide[kOne ? kFewWaves : 1][kOne ? kAhead : 1][64];  // pairs of bfloat16
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, r = lane & 15, q = lane >> 4;
    const int64_t n0 = int64_t(blockIdx.x) * 16, K = int64_t(g.nb) * kScaleBlock;
    // rows past the end read the last one's codes and are not stored
    const int64_t bn = min(n0 + r, g.N - 1);
    const uint8_t* pb = g.b + bn * K + q * 16;
    const uint8_t* sb = g.sb + bn;
    const uint8_t* pa[FM];
    const uint8_t* sa[FM];
    v4f acc[FM];
#pragma unroll
    for (int f = 0; f < FM; ++f) {
        const int64_t am = min(int64_t(f * 16 + r), g.M - 1);
        pa[f] = kOne ? nullptr : g.a + am * K + q * 16;
        sa[f] = kOne ? nullptr : g.sa + am;
        acc[f] = v4f{0, 0, 0, 0};
    }
    for (int k = wave; k < g.nb; k += kFewWaves * kAhead) {
        if constexpr (kOne) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        int4 cb[kAhead][2], ca[kAhead][FM][2];
        uint32_t eb[kAhead], ea[kAhead][FM];
        float image[kOne ? kAhead : 1][2];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int64_t at = min(k + u * kFewWaves, g.nb - 1);
#pragma unroll
            for (int h = 0; h < 2; ++h) cb[u][h] = *reinterpret_cast<const int4*>(pb + at * kScaleBlock + h * 64);
            eb[u] = sb[at * g.srb];
            if constexpr (kOne) {
                const auto* x = static_cast<const typename S::Bits*>(one.x) + at * kScaleBlock;
                const int last = int(min(one.cols - at * kScaleBlock, int64_t(kScaleBlock))) - 1;
#pragma unroll
                for (int i = 0; i < 2; ++i) image[u][i] = S::widen(x[min(2 * lane + i, last)]);
#pragma unroll
                for (int i = 0; i < 2; ++i) image[u][i] = 2 * lane + i <= last ? image[u][i] : 0.0f;
                continue;
            }
#pragma unroll
            for (int f = 0; f < FM; ++f) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    ca[u][f][h] = *reinterpret_cast<const int4*>(pa[f] + at * kScaleBlock + h * 64);
                ea[u][f] = sa[f][at * g.sra];
            }
        }
        __builtin_amdgcn_sched_barrier(0);  // all loads before the first use
        if constexpr (kOne) {
            // (the wavefront's own part of LDS, written and read in order)
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const float v = image[u][0], w = image[u][1];
                const int e = block_exponent(wave_max(max(magnitude(v), magnitude(w))));
                wide[wave][u][lane] = __builtin_bit_cast(
                    uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(int(codes2(v, w, power_of_2(-e))),
                                                                        scale_of(uint32_t(e + 127)), false));
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (k + u * kFewWaves >= g.nb) break;
            const float fb = scale_of(eb[u]);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const v8bf b0 = widen8(cb[u][h].x, cb[u][h].y, fb), b1 = widen8(cb[u][h].z, cb[u][h].w, fb);
                if constexpr (kOne) {
                    const auto* a = reinterpret_cast<const v8bf*>(wide[wave][u] + h * 32 + q * 8);
                    acc[0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[0], b0, acc[0], 0, 0, 0);
                    acc[0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[1], b1, acc[0], 0, 0, 0);
                    continue;
                }
#pragma unroll
                for (int f = 0; f < FM; ++f) {
                    const float fa = scale_of(ea[u][f]);
                    const int4 c = ca[u][f][h];
                    acc[f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen8(c.x, c.y, fa), b0, acc[f], 0, 0, 0);
                    acc[f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen8(c.z, c.w, fa), b1, acc[f], 0, 0, 0);
                }
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
        float v = 0;
#pragma unroll
        for (int w = 0; w < kFewWaves; ++w) v += sums[w][m][i & 15];
        store_score<O>(g, 0, m, n, v);
    }
}

// The product in tiles: a workgroup of WM x WN x KW wavefronts computes BM x BN scores.  4096 x 8192 x 16640 by
// tiles of 256 x 256 takes 775 to 855 us (1.31 to 1.44 PFLOP/s; a bfloat16 library product 1.40 on this
// card): the matrix units are busy for two thirds of the cycles, at a clock that the power limit holds at 1.9 GHz.
// Codes of one block of a tile's rows in LDS: 128 bytes a row, fragment after fragment (fragment f of a part of
// the tile has its rows F r + f, r < 32), and the 16-byte chunks of a row permuted among themselves (chunk c of row
// r of a fragment at place c ^ ((r / 2) & 7)), so that the 16 lanes that read one chunk of 16 rows at a time reach
// each of the 64 banks once.
template <int BM, int BN> struct alignas(16) Stage {
    uint8_t a[BM * kScaleBlock], b[BN * kScaleBlock];
    uint32_t sa[64], sb[64];  // scale bytes (the first BM and BN are used)
};

using LocalPtr = __attribute__((address_space(3))) void*;

// The codes of `rows` rows from p on as a buffer: reads past its end give zeros.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t codes_buffer(const uint8_t* p, int64_t rows, int64_t K) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p), 0, int(uint32_t(rows * K)), 0x00027000);
}

// N loads of a wavefront to LDS, 8 rows of 128 bytes each; off: each lane's byte offsets from `at` on.
template <int N>
__device__ __forceinline__ void to_lds(__amdgpu_buffer_rsrc_t src, const uint32_t (&off)[N], int at, uint8_t* dst) {
#pragma unroll
    for (int i = 0; i < N; ++i)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(src, (LocalPtr)(dst + i * 1024), 16, int(off[i]), at, 0, 0);
}

// The scales of rows `first` .. first + F - 1 (F divides first and 4) from the stage's bytes.  They are read
// as words: before a load of single bytes, which may alias anything, the compiler waits for all loads to LDS.
template <int F> __device__ __forceinline__ void scales_of(const uint32_t* words, int first, float (&s)[F]) {
    const uint32_t w = words[first >> 2] >> (8 * (first & 3));
#pragma unroll
    for (int f = 0; f < F; ++f) s[f] = scale_of((w >> (8 * f)) & 255u);
}

using v16f = __attribute__((ext_vector_type(16))) float;

// NT quarters of a block from quarter t0 on.  fill starts the loads of the next block: its instructions go where the
// first operands are on their way from LDS.
template <int FM, int FN, int NT, class Fill>
__device__ __forceinline__ void tile_step(const uint8_t* __restrict__ ca, const uint8_t* __restrict__ cb, int t0, int key,
                                          int q, const uint32_t* __restrict__ sa, const uint32_t* __restrict__ sb,
                                          int ra0, int rb0, v16f (&acc)[FM][FN], Fill fill) {
    float ea[FM], eb[FN];
    scales_of<FM>(sa, ra0, ea);
    scales_of<FN>(sb, rb0, eb);
    // of a whole block the operands of one quarter are read from LDS while the one before is multiplied
    constexpr int D = NT <= 2 ? 1 : 2;
    int4 ra[D][FM], rb[D][FN];
    auto read = [&](int t) {
        const int at = ((2 * (t0 + t) + q) ^ key) * 16;
#pragma unroll
        for (int f = 0; f < FM; ++f) ra[t % D][f] = *reinterpret_cast<const int4*>(ca + f * 32 * kScaleBlock + at);
#pragma unroll
        for (int f = 0; f < FN; ++f) rb[t % D][f] = *reinterpret_cast<const int4*>(cb + f * 32 * kScaleBlock + at);
    };
#pragma unroll
    for (int t = 0; t < D - 1; ++t) read(t);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        if (t + D - 1 < NT) read(t + D - 1);
        if (t == 0) fill();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            v8bf fa[FM], fb[FN];
#pragma unroll
            for (int f = 0; f < FM; ++f) {
                const int4 c = ra[t % D][f];
                fa[f] = h ? widen8(c.z, c.w, ea[f]) : widen8(c.x, c.y, ea[f]);
            }
#pragma unroll
            for (int f = 0; f < FN; ++f) {
                const int4 c = rb[t % D][f];
                fb[f] = h ? widen8(c.z, c.w, eb[f]) : widen8(c.x, c.y, eb[f]);
            }
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[i], fb[j], acc[i][j], 0, 0, 0);
        }
        if (NT > 2) __builtin_amdgcn_sched_barrier(0);
    }
}

// Wait until this wavefront's loads to LDS have arrived, and its reads of the stage that is filled next, then for the
// other wavefronts.
__device__ __forceinline__ void stage_ready() {
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// A wavefront's rows of 32 x 32 fragments lie F apart (fragment f has rows F r + f), so that one load brings
// the scales of a lane's rows and a lane's F columns are neighbours in the output.
// KW > 1: as many wavefronts share a part of the tile, each with its quarters of every block, so that no value is
// widened twice; their sums are added in LDS at the end.
// (tiles of 128 x 128 keep to 128 registers: two workgroups of 8 wavefronts per CU)
template <int BM, int BN, int WM, int WN, int KW, class O>
__global__ __launch_bounds__(64 * WM * WN * KW, BM * BN == 128 * 128 ? 4 : 1) void k_scores_tile(ScoreArgs g, uint32_t tm, uint32_t tn) {
    constexpr int W = WM * WN * KW, FM = BM / WM / 32, FN = BN / WN / 32;
    constexpr int LA = BM / 8 / W, LB = BN / 8 / W;  // loads of a wavefront for a stage
    static_assert(LA * W * 8 == BM && LB * W * 8 == BN, "whole loads");
    __shared__ Stage<BM, BN> stages[2];
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
    const int64_t K = int64_t(g.nb) * kScaleBlock;

    uint32_t oa[LA], ob[LB];
    const int row8 = lane >> 3, place = lane & 7;
    auto offset = [&](int slot, int F) {  // of a row's place in LDS and this lane's chunk there
        const int r = slot & 31, f = (slot >> 5) % F, part = (slot >> 5) / F;
        return uint32_t(((part * 32 + r) * F + f) * K) + (place ^ ((r >> 1) & 7)) * 16;
    };
#pragma unroll
    for (int i = 0; i < LA; ++i) oa[i] = offset((wave * LA + i) * 8 + row8, FM);
#pragma unroll
    for (int i = 0; i < LB; ++i) ob[i] = offset((wave * LB + i) * 8 + row8, FN);
    // rows past the end read zeros
    const auto ga = codes_buffer(g.a + m0 * K, min(int64_t(BM), g.M - m0), K);
    const auto gb = codes_buffer(g.b + n0 * K, min(int64_t(BN), g.N - n0), K);
    const int ra = (wm * 32 + r) * FM, rb = (wn * 32 + r) * FN;  // a lane's first row and column of the tile
    v16f acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;

    // two stages in turn: while one is multiplied the other is filled (333 x 1999 x 8280 by tiles of 64 x 64: two
    // 25.7 us, three 26.0, four 30.8, as the LDS then holds fewer workgroups)
    const int lane4 = lane * 4;
    const uint8_t *sa = g.sa + k0 * g.sra + m0, *sb = g.sb + k0 * g.srb + n0;  // the next block's scales
    auto load = [&](Stage<BM, BN>& st, int k) {
        to_lds(ga, oa, k * kScaleBlock, st.a + wave * LA * 1024);
        to_lds(gb, ob, k * kScaleBlock, st.b + wave * LB * 1024);
        // (every wavefront brings all scales: the same bytes to the same place)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(codes_buffer(sa, 1, g.sra - m0), (LocalPtr)st.sa, 4, lane4, 0, 0, 0);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(codes_buffer(sb, 1, g.srb - n0), (LocalPtr)st.sb, 4, lane4, 0, 0, 0);
        sa += g.sra;
        sb += g.srb;
    };
    load(stages[0], k0);
#pragma unroll 1
    for (int k = k0; k < k1; ++k) {
        const int cur = (k - k0) & 1;
        stage_ready();
        const Stage<BM, BN>& st = stages[cur];
        tile_step<FM, FN, 4 / KW>(st.a + (wm * 32 * FM + r) * kScaleBlock, st.b + (wn * 32 * FN + r) * kScaleBlock,
                                  kw * (4 / KW), (r >> 1) & 7, q, st.sa, st.sb, ra, rb, acc, [&] {
                                      if (k + 1 < k1) load(stages[cur ^ 1], k + 1);
                                  });
    }

    // a wavefront's share of its part's results: elements e0 .. e0 + EN - 1 of each fragment
    constexpr int EN = 16 / KW;
    const int e0 = kw * EN;
    float sum[FM][FN][EN];
    if constexpr (KW == 1) {
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int e = 0; e < EN; ++e) sum[i][j][e] = acc[i][j][e];
    } else {
        float* room = reinterpret_cast<float*>(stages);
        static_assert(sizeof(stages) >= size_t(W) * 4096, "a fragment of every wavefront");
        const float* part = room + (wave - kw) * 1024 + e0 * 64 + lane;
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
                    float v = part[e * 64];
#pragma unroll
                    for (int w = 1; w < KW; ++w) v += part[w * 1024 + e * 64];
                    sum[i][j][e] = v;
                }
            }
    }

    const int64_t n = n0 + rb;
    const bool whole = n + FN <= g.N;
    float off[FN];
#pragma unroll
    for (int j = 0; j < FN; ++j) off[j] = g.bias && n + j < g.N ? g.bias[n + j] : 0.0f;
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int e = 0; e < EN; ++e) {
            const int at_e = e0 + e;
            const int64_t m = m0 + (wm * 32 + (at_e / 4) * 8 + q * 4 + at_e % 4) * FM + i;
            if (m >= g.M) continue;
            if (!whole) {
#pragma unroll
                for (int j = 0; j < FN; ++j)
                    if (n + j < g.N) store_score<O>(g, split, m, n + j, sum[i][j][e]);
            } else if (g.splits > 1) {
                float v[FN];
#pragma unroll
                for (int j = 0; j < FN; ++j) v[j] = sum[i][j][e];
                __builtin_memcpy(g.part + (int64_t(split) * g.M + m) * g.N + n, v, sizeof v);
            } else {
                typename O::Bits v[FN];
#pragma unroll
                for (int j = 0; j < FN; ++j) v[j] = O::round(sum[i][j][e] + off[j]);
                __builtin_memcpy(static_cast<typename O::Bits*>(g.out) + m * g.N + n, v, sizeof v);
            }
        }
}

// ------------------------------------------------------------------ which kernel
// One image: k_scores_few.  Else the tile and the number of ranges of the blocks with the least time by a
// count of steps (one block of K for one tile).  A CU with n workgroups of a tile takes n step_us for a step
// of each, but no less than alone_us: one workgroup alone waits for LDS and for its own products.  Measured:
// 4096 x 8192 x 16640 (full CUs) 64: 1056 us, 128: 857, 256: 775; 2000 x 2000 x 4224 46, 37 and 93; 333 x 1999 x
// 8280 in one range 37, 60 and 174 us, in four 24, 28 and 61.  Several ranges cost a launch and their sums written
// and read.  Up to 32 images k_scores_few may be faster: 16 and 24 x 1000 x 4224 6.3 and 7.6 us (tiles 9.0 and 9.1),
// but 24 x 4096 x 16640 23.6 (18.2).  Against every tile and 1 to 16 ranges on 28 sizes from 17 x 2000 to 4096 x 8192
// the choice is within 8 % of the best.
struct ScorePlan {
    int few, tile, splits;  // few: FM of k_scores_few, or 0; tile: index of kTiles
};
struct TileKind {
    int bm, bn;
    double step_us, alone_us;
};
constexpr TileKind kTiles[] = {{64, 64, 0.28, 0.50}, {128, 128, 0.87, 1.0}, {256, 256, 3.1, 2.6}};
constexpr int kCus = 256, kMaxSplits = 16;

ScorePlan score_plan(int64_t M, int64_t N, int64_t nb) {
    ScorePlan best{M <= 16 ? 1 : 2, 0, 1};
    if (M == 1) return best;
    double least = M > 32 ? 1e300 : (2.5 + (M <= 16 ? 0.12 : 0.15) * nb) * double((N + 16 * kCus - 1) / (16 * kCus));
    for (int t = 0; t < 3; ++t) {
        const TileKind& kind = kTiles[t];
        const int64_t tiles = ((M + kind.bm - 1) / kind.bm) * ((N + kind.bn - 1) / kind.bn);
        for (int s = 1; s <= kMaxSplits && s <= nb; ++s) {
            const double each = double((tiles * s + kCus - 1) / kCus);
            double us = 2.0 + ((nb + s - 1) / s + 2) * (each * kind.step_us > kind.alone_us ? each * kind.step_us : kind.alone_us);
            if (s > 1) us += 4.0 + double(M) * N * (8 * s + 4) / 4.5e6;
            if (us < least) {
                least = us;
                best = {0, t, s};
            }
        }
    }
    return best;
}

}  // namespace

hipError_t launch_quantize_blocks(int dt, const void* x, int64_t rows, int64_t cols, int64_t stride, void* codes,
                                  void* scales, hipStream_t s) {
    const int nb = int(block_count(cols));
    const int64_t sr = scale_rows(rows);
    const dim3 grid(match_grid(sr * ((nb + 15) / 16)));
    auto* c = static_cast<uint8_t*>(codes);
    auto* e = static_cast<uint8_t*>(scales);
    switch (dt) {
        case TP_F32:
            k_quantize<F32><<<grid, 256, 0, s>>>(static_cast<const uint32_t*>(x), rows, cols, stride, nb, sr, c, e);
            break;
        case TP_F16:
            k_quantize<F16><<<grid, 256, 0, s>>>(static_cast<const uint16_t*>(x), rows, cols, stride, nb, sr, c, e);
            break;
        default:
            k_quantize<BF16><<<grid, 256, 0, s>>>(static_cast<const uint16_t*>(x), rows, cols, stride, nb, sr, c, e);
    }
    return hipGetLastError();
}

int64_t block_scores_work(int64_t M, int64_t N, int64_t nb) {
    const ScorePlan p = score_plan(M, N, nb);
    return p.splits > 1 ? p.splits * M * N * int64_t(sizeof(float)) : 0;
}

template <class O> hipError_t scores(const ScoreArgs& g, const ScorePlan& p, hipStream_t s) {
    if (p.few) {
        const dim3 grid(unsigned((g.N + 15) / 16));
        if (p.few == 1)
            k_scores_few<1, O, void><<<grid, 64 * kFewWaves, 0, s>>>(g, OneImage{});
        else
            k_scores_few<2, O, void><<<grid, 64 * kFewWaves, 0, s>>>(g, OneImage{});
    } else {
        const TileKind& kind = kTiles[p.tile];
        const uint32_t tm = uint32_t((g.M + kind.bm - 1) / kind.bm), tn = uint32_t((g.N + kind.bn - 1) / kind.bn);
        const dim3 grid(tm * tn * p.splits);
        if (p.tile == 0)
            k_scores_tile<64, 64, 1, 1, 4, O><<<grid, 256, 0, s>>>(g, tm, tn);
        else if (p.tile == 1)
            k_scores_tile<128, 128, 2, 2, 2, O><<<grid, 512, 0, s>>>(g, tm, tn);
        else
            k_scores_tile<256, 256, 2, 4, 1, O><<<grid, 512, 0, s>>>(g, tm, tn);
    }
    if (hipError_t e = hipGetLastError()) return e;
    if (p.splits > 1) k_scores_join<O><<<match_grid((g.M * g.N + 255) / 256), 256, 0, s>>>(g);
    return hipGetLastError();
}

hipError_t launch_block_scores(const void* a, const void* sa, int64_t M, const void* b, const void* sb, int64_t N,
                               int64_t nb, const void* bias, int out_dt, void* out, void* work, hipStream_t s) {
    const ScorePlan p = score_plan(M, N, nb);
    const ScoreArgs g{static_cast<const uint8_t*>(a), static_cast<const uint8_t*>(sa), static_cast<const uint8_t*>(b),
                      static_cast<const uint8_t*>(sb), M, N, scale_rows(M), scale_rows(N), int(nb), p.splits,
                      static_cast<const float*>(bias), out, static_cast<float*>(work)};
    return out_dt == TP_F32 ? scores<F32>(g, p, s) : scores<BF16>(g, p, s);
}

// One image is quantised by k_scores_few itself: 256 references of 4224 values 7.1 us in two launches, 5.2 in
// one; 4096 of 16640 17.8 and 15.2.
// (the sums of the product's ranges, then codes and scales from a 16-byte boundary on)
int64_t sums_before_codes(int64_t M, int64_t N, int64_t nb) { return (block_scores_work(M, N, nb) + 15) / 16 * 16; }
int64_t score_images_work(int64_t M, int64_t N, int64_t cols) {
    if (M == 1) return 0;
    const int64_t nb = block_count(cols);
    return sums_before_codes(M, N, nb) + M * nb * kScaleBlock + nb * scale_rows(M);
}

template <class S> hipError_t score_one(const ScoreArgs& g, const OneImage& one, int out_dt, hipStream_t s) {
    const dim3 grid(unsigned((g.N + 15) / 16));
    if (out_dt == TP_F32)
        k_scores_few<1, F32, S><<<grid, 64 * kFewWaves, 0, s>>>(g, one);
    else
        k_scores_few<1, BF16, S><<<grid, 64 * kFewWaves, 0, s>>>(g, one);
    return hipGetLastError();
}

hipError_t launch_score_images(int dt, const void* x, int64_t M, int64_t cols, int64_t stride, const void* b,
                               const void* sb, int64_t N, const void* bias, int out_dt, void* out, void* work,
                               hipStream_t s) {
    const int64_t nb = block_count(cols);
    if (M == 1) {
        const ScoreArgs g{nullptr, nullptr, static_cast<const uint8_t*>(b), static_cast<const uint8_t*>(sb), 1, N, 0,
                          scale_rows(N), int(nb), 1, static_cast<const float*>(bias), out, nullptr};
        const OneImage one{x, cols};
        return dt == TP_F32 ? score_one<F32>(g, one, out_dt, s) : dt == TP_F16 ? score_one<F16>(g, one, out_dt, s)
                                                                               : score_one<BF16>(g, one, out_dt, s);
    }
    auto* part = static_cast<char*>(work);
    auto* codes = part + sums_before_codes(M, N, nb);
    auto* scales = codes + M * nb * kScaleBlock;
    if (hipError_t e = launch_quantize_blocks(dt, x, M, cols, stride, codes, scales, s)) return e;
    return launch_block_scores(codes, scales, M, b, sb, N, nb, bias, out_dt, out, part, s);
}

}  // namespace tp
