// Scores of images against references in 8-bit blocks.
//
//   quantize  each block of 128 values of a row gets the least exponent e with max |x| <= 448 2^e (448
//             being the largest e4m3 value) and the codes round(x 2^-e), to nearest even.  The scale is a
//             power of two, so that scaling is exact and the matrix units apply it themselves.
//   scores    out[m, n] = bias[n] + sum_b 2^(ea + eb) sum_k a[m, k] b[n, k], summed in fp32.
//
// The matrix units' own 8-bit products align each eight of them to about 14 bits before they add them (a
// product of 4 beside one of 65536 is lost; random blocks come out 1.7e-5 off, where the type's sums have
// 24 bits).  So the codes are widened to bfloat16, which holds a code times any scale exactly, one
// v_cvt_scalef32_pk_bf16_fp8 per two values, and multiplied by the bfloat16 units, whose products are
// exact and whose sums are fp32 (7e-9 off on the same blocks).
//
// The order of the values within an instruction's operands does not matter as long as both sides have the
// same.
#include "../../../include/torch_projectors_hip.h"
#include "tp_match.hh"

namespace tp {
namespace {

using v4f = __attribute__((ext_vector_type(4))) float;

// ------------------------------------------------------------------ quantize
// Exponent of a block with largest finite magnitude `most`: most = f 2^x with f in [0.5, 1), and
// 448 = 0.875 2^9.
__device__ __forceinline__ int block_exponent(float most) {
    int x;
    const float f = frexpf(most, &x);
    return most == 0.0f ? 0 : max(f > 0.875f ? x - 8 : x - 9, -127);
}

// Codes of two values: to nearest even, NaN for what is not finite.
__device__ __forceinline__ uint32_t codes2(float x, float y, int e) {
    // 2^-e in two factors: e reaches -127, and 2^127 is the largest power of two
    const float f = ldexpf(1.0f, -e);
    const uint32_t two = __builtin_amdgcn_cvt_pk_fp8_f32(x * f, y * f, 0, false) & 0xffffu;
    const uint32_t nx = isfinite(x) ? 0u : 0x7fu, ny = isfinite(y) ? 0u : 0x7f00u;
    return two | nx | ny;
}

// A wavefront per block of a row, two values per lane.
template <class S>
__global__ __launch_bounds__(256) void k_quantize(const typename S::Bits* __restrict__ x, int64_t rows, int64_t cols,
                                                  int64_t stride, int64_t nb, int64_t srows,
                                                  uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    const int lane = threadIdx.x & 63;
    for (int64_t item = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6); item < srows * nb; item += int64_t(gridDim.x) * 4) {
    const int64_t r = item / nb, b = item % nb;
    if (r >= rows) {  // the padding rows' scales
        if (lane == 0) scales[b * srows + r] = 127;
        continue;
    }
    const int64_t c = b * kScaleBlock + 2 * lane;
    const float u = c < cols ? S::widen(x[r * stride + c]) : 0.0f;
    const float v = c + 1 < cols ? S::widen(x[r * stride + c + 1]) : 0.0f;
    float most = fmaxf(isfinite(u) ? fabsf(u) : 0.0f, isfinite(v) ? fabsf(v) : 0.0f);
#pragma unroll
    for (int d = 32; d; d >>= 1) most = fmaxf(most, __shfl_xor(most, d));
    const int e = block_exponent(most);
    if (lane == 0) scales[b * srows + r] = uint8_t(e + 127);
    reinterpret_cast<uint16_t*>(codes + r * nb * kScaleBlock + b * kScaleBlock)[lane] = uint16_t(codes2(u, v, e));
    }
}

// ------------------------------------------------------------------ scores
using v8bf = __attribute__((ext_vector_type(8))) __bf16;
using v2bf = __attribute__((ext_vector_type(2))) __bf16;

// A scale byte as the power of two it stands for (0: 2^-127, a subnormal).
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(max(byte << 23, 0x00400000u)); }

// Eight codes times their block's scale: exact, a bfloat16 holding 4 significant bits at any such exponent.
__device__ __forceinline__ v8bf widen8(int lo, int hi, float scale) {
    const v2bf a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false);
    const v2bf b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
    const v2bf c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false);
    const v2bf d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
    return v8bf{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// A wavefront computes 16 rows x 64 columns, operands straight from memory.  Rows and columns past the
// end read the last one's and are not stored.
template <class O>
__global__ __launch_bounds__(256) void k_scores(const uint8_t* __restrict__ a, const uint8_t* __restrict__ sa,
                                                int64_t M, int64_t sra, const uint8_t* __restrict__ b,
                                                const uint8_t* __restrict__ sb, int64_t N, int64_t srb, int64_t nb,
                                                const float* __restrict__ bias, typename O::Bits* __restrict__ out) {
    const int lane = threadIdx.x & 63, r16 = lane & 15, q = lane >> 4;
    const int64_t tn = (N + 63) / 64, K = nb * kScaleBlock;
    for (int64_t tile = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6); tile < (M + 15) / 16 * tn;
         tile += int64_t(gridDim.x) * 4) {
        const int64_t m0 = tile / tn * 16, n0 = tile % tn * 64, am = min(m0 + r16, M - 1);
        const uint8_t* pa = a + am * K + q * 8;
        const uint8_t* pb[4];
        int64_t bn[4];
        v4f acc[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            bn[i] = min(n0 + 16 * i + r16, N - 1);
            pb[i] = b + bn[i] * K + q * 8;
            acc[i] = v4f{0, 0, 0, 0};
        }
        for (int64_t k = 0; k < nb; ++k) {
            const float ea = scale_of(sa[k * sra + am]);
            float eb[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) eb[i] = scale_of(sb[k * srb + bn[i]]);
#pragma unroll
            for (int h = 0; h < kScaleBlock; h += 32) {
                const int2 ca = *reinterpret_cast<const int2*>(pa + k * kScaleBlock + h);
                const v8bf fa = widen8(ca.x, ca.y, ea);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int2 cb = *reinterpret_cast<const int2*>(pb[i] + k * kScaleBlock + h);
                    acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa, widen8(cb.x, cb.y, eb[i]), acc[i], 0, 0, 0);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t n = n0 + 16 * i + r16;
            if (n >= N) continue;
            const float off = bias ? bias[n] : 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int64_t m = m0 + 4 * q + j;
                if (m < M) out[m * N + n] = O::round(acc[i][j] + off);
            }
        }
    }
}

}  // namespace

hipError_t launch_quantize_blocks(int dt, const void* x, int64_t rows, int64_t cols, int64_t stride, void* codes,
                                  void* scales, hipStream_t s) {
    const int64_t nb = (cols + kScaleBlock - 1) / kScaleBlock, sr = scale_rows(rows);
    const dim3 grid(match_grid((sr * nb + 3) / 4));
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

int64_t block_scores_work(int64_t, int64_t, int64_t) { return 0; }

hipError_t launch_block_scores(const void* a, const void* sa, int64_t M, const void* b, const void* sb, int64_t N,
                               int64_t nb, const void* bias, int out_dt, void* out, void*, hipStream_t s) {
    const int64_t tiles = (M + 15) / 16 * ((N + 63) / 64);
    const dim3 grid(match_grid((tiles + 3) / 4));
    const auto* pa = static_cast<const uint8_t*>(a);
    const auto* pb = static_cast<const uint8_t*>(b);
    const auto* ea = static_cast<const uint8_t*>(sa);
    const auto* eb = static_cast<const uint8_t*>(sb);
    const auto* f = static_cast<const float*>(bias);
    if (out_dt == TP_F32)
        k_scores<F32><<<grid, 256, 0, s>>>(pa, ea, M, scale_rows(M), pb, eb, N, scale_rows(N), nb, f,
                                           static_cast<uint32_t*>(out));
    else
        k_scores<BF16><<<grid, 256, 0, s>>>(pa, ea, M, scale_rows(M), pb, eb, N, scale_rows(N), nb, f,
                                            static_cast<uint16_t*>(out));
    return hipGetLastError();
}

}  // namespace tp
