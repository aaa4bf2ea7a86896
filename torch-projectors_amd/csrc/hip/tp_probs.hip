// Log probabilities of given candidates, the entropy, the log sum and the best alternatives of rows of
// scores, and the gradient of the scores.
//
// With c = 1 / temperature, a row's largest allowed score m, z = c (x - m):
//   s = sum e^z, u = sum z e^z;  log p = z - ln s;  entropy = ln s - u / s;  log_sum = c m + ln s
// Each lane keeps (m, s, u) of the scores that it has read, rescaled when its m grows, so a row is read
// once; m is subtracted before the temperature divides, so rows of the type's lowest value do not overflow.
// Sums are fp32.
//   d x = c ( p (dL - sum dG - sum dT - dH (log p + H)) + what is given or listed at x )
//
// Alternatives: a wavefront keeps its `top` best as sorted keys, one per lane: the score's bits in an order that
// integers have, then the complement of its index, so ties go to the lowest index.  A score above the last
// key's is inserted by the lanes' common effort: its place is a population count, the keys behind it move
// one lane up.  In rows in no particular order that happens about top (1 + ln(n / top)) times for n scores.
//
// Scores of -inf count as not allowed.  A NaN makes the row's results NaN.
#include "../../../include/torch_projectors_hip.h"
#include "tp_match.hh"

namespace tp {
namespace {

constexpr int kProbsBlock = 256, kProbsWaves = kProbsBlock / 64;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.693147180559945309417f;

__device__ __forceinline__ float neg_inf() { return -__builtin_inff(); }

// The larger of two, NaN if either is.
__device__ __forceinline__ float max_or_nan(float a, float b) { return a != a ? a : (b > a || b != b ? b : a); }

// Larger keys are better: the score, then the lower index.  0 is no candidate.
__device__ __forceinline__ uint64_t key_of(float x, uint32_t index) {
    const uint32_t b = __float_as_uint(x + 0.0f);  // -0 and 0 are equal
    return (uint64_t(b & 0x80000000u ? ~b : b | 0x80000000u) << 32) | ~index;
}
__device__ __forceinline__ float score_of(uint64_t key) {
    const uint32_t o = uint32_t(key >> 32);
    return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ uint32_t index_of(uint64_t key) { return ~uint32_t(key); }

// Insert a key (uniform over the wavefront) into the sorted keys, one per lane.
__device__ __forceinline__ void insert(uint64_t& mine, uint64_t key, int lane) {
    const int place = __popcll(__ballot(mine > key));
    const uint64_t before = __shfl_up(mine, 1);
    if (lane >= place) mine = lane == place ? key : before;
}

// Sums over scores relative to their largest: z in units of 1 / (c log2 e), i.e. exponents of 2.
struct Sums {
    float m, s, u;
};
// exp2 of z clamped to where it is 0, so that z exp2(z) is 0 and not NaN for -inf.
__device__ __forceinline__ void add_score(Sums& a, float x, float c2) {
    const float z = fmaxf((x - a.m) * c2, -200.0f), e = __builtin_amdgcn_exp2f(z);
    a.s += e;
    a.u += z * e;
}
// The sums of a relative to m >= a.m.
__device__ __forceinline__ Sums moved(const Sums& a, float m, float c2) {
    if (a.s == 0.0f) return Sums{m, 0.0f, 0.0f};
    const float z = fmaxf((a.m - m) * c2, -200.0f), f = __builtin_amdgcn_exp2f(z);
    return Sums{m, a.s * f, (a.u + a.s * z) * f};
}
__device__ __forceinline__ Sums joined(const Sums& a, const Sums& b, float c2) {
    const float m = max_or_nan(a.m, b.m);
    const Sums p = moved(a, m, c2), q = moved(b, m, c2);
    return Sums{m, p.s + q.s, p.u + q.u};
}

// One workgroup per row.
template <class S>
__global__ __launch_bounds__(kProbsBlock) void k_probs(ProbsArgs a, float* __restrict__ given_out,
                                                       float* __restrict__ entropy, float* __restrict__ log_sum,
                                                       float* __restrict__ top_out, int64_t* __restrict__ top_index,
                                                       float* __restrict__ stats) {
    __shared__ Sums part[kProbsWaves];
    __shared__ uint64_t keys[kProbsWaves][kMaxTop];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int64_t t = blockIdx.x; t < a.T; t += gridDim.x) {
    const auto* x = static_cast<const typename S::Bits*>(a.scores) + t * a.stride;
    const uint8_t* mask = a.mask ? a.mask + t * a.mask_stride : nullptr;
    const float c2 = kLog2e / a.temperature;
    Sums mine{neg_inf(), 0.0f, 0.0f};
    uint64_t key = 0;
    float least = neg_inf();  // the last listed score: only larger ones are listed (they have later indices)
    for (int64_t v0 = wave * 64; v0 < a.V; v0 += kProbsBlock) {
        const int64_t v = v0 + lane;
        float f = neg_inf();
        if (v < a.V && (!mask || mask[v])) f = S::widen(x[v]);
        const float m = max_or_nan(mine.m, f);
        if (m != mine.m) mine = moved(mine, m, c2);
        if (f != neg_inf()) add_score(mine, f, c2);
        if (a.top) {
            uint64_t better = __ballot(f > least);
            while (better) {
                const int from = __ffsll(static_cast<long long>(better)) - 1;
                better &= better - 1;
                insert(key, key_of(__shfl(f, from), uint32_t(v0 + from)), lane);
            }
            const uint64_t last = __shfl(key, a.top - 1);
            least = last ? score_of(last) : neg_inf();
        }
    }
#pragma unroll
    for (int d = 32; d; d >>= 1)
        mine = joined(mine, Sums{__shfl_xor(mine.m, d), __shfl_xor(mine.s, d), __shfl_xor(mine.u, d)}, c2);
    if (lane == 0) part[wave] = mine;
    keys[wave][lane] = lane < a.top ? key : 0;
    __syncthreads();
    if (wave == 0) {
    for (int w = 1; w < kProbsWaves; ++w) {
        mine = joined(mine, part[w], c2);
        for (int j = 0; j < a.top; ++j)
            if (keys[w][j]) insert(key, keys[w][j], lane);
    }
    const bool none = mine.m == neg_inf();
    const float m = mine.m;
    const float ls = m == __builtin_inff() ? __builtin_nanf("") : logf(mine.s);
    if (lane == 0) {
        const float H = none ? 0.0f : !isfinite(m) ? __builtin_nanf("") : ls - mine.u * kLn2 / mine.s;
        entropy[t] = H;
        log_sum[t] = isfinite(m) ? m / a.temperature + ls : m;
        float* st = stats + t * kProbsStats;
        st[0] = m;
        st[1] = ls;
        st[2] = H;
        st[3] = 0.0f;
    }
    for (int64_t g = lane; g < a.G; g += 64) {
        const int64_t v = a.given[t * a.G + g];
        float lp = 0.0f;
        if (v != -1) {
            if (v < 0 || v >= a.V) lp = __builtin_nanf("");
            else if (m != m) lp = m;
            else if (none || (mask && !mask[v])) lp = neg_inf();
            else lp = (S::widen(x[v]) - m) / a.temperature - ls;
        }
        given_out[t * a.G + g] = lp;
    }
    if (lane < a.top) {
        top_out[t * a.top + lane] = m != m ? m : key ? (score_of(key) - m) / a.temperature - ls : neg_inf();
        top_index[t * a.top + lane] = key ? int64_t(index_of(key)) : -1;
    }
    }
    __syncthreads();  // the next row's sums overwrite this one's
    }
}

// One workgroup per row: every score's gradient but that of the given and listed ones, then those.
template <class S>
__global__ __launch_bounds__(kProbsBlock) void k_probs_back(ProbsArgs a, const float* __restrict__ stats,
                                                            const int64_t* __restrict__ top_index,
                                                            const float* __restrict__ d_given,
                                                            const float* __restrict__ d_entropy,
                                                            const float* __restrict__ d_log_sum,
                                                            const float* __restrict__ d_top,
                                                            typename S::Bits* __restrict__ d_scores) {
    for (int64_t t = blockIdx.x; t < a.T; t += gridDim.x) {
    const auto* x = static_cast<const typename S::Bits*>(a.scores) + t * a.stride;
    auto* d = d_scores + t * a.V;
    const uint8_t* mask = a.mask ? a.mask + t * a.mask_stride : nullptr;
    const float m = stats[t * kProbsStats], ls = stats[t * kProbsStats + 1], H = stats[t * kProbsStats + 2];
    const float c = 1.0f / a.temperature, c2 = kLog2e / a.temperature, ls2 = ls * kLog2e;
    const bool none = m == neg_inf();
    const int64_t G = d_given ? a.G : 0;
    const int K = d_top ? a.top : 0;
    float all = d_log_sum ? d_log_sum[t] : 0.0f;
    for (int64_t g = 0; g < G; ++g)
        if (a.given[t * G + g] != -1) all -= d_given[t * G + g];
    for (int j = 0; j < K; ++j)
        if (top_index[t * K + j] >= 0) all -= d_top[t * K + j];
    const float dH = d_entropy ? d_entropy[t] : 0.0f;
    // the gradient of score v without what is given or listed there
    auto smooth = [&](int64_t v) {
        if (none || (mask && !mask[v])) return 0.0f;
        const float lp2 = (S::widen(x[v]) - m) * c2 - ls2, p = __builtin_amdgcn_exp2f(lp2);
        return p * (all - dH * (fmaxf(lp2, -200.0f) * kLn2 + H));
    };
    for (int64_t v = threadIdx.x; v < a.V; v += kProbsBlock) d[v] = S::round(c * smooth(v));
    __syncthreads();
    for (int64_t i = threadIdx.x; i < G + K; i += kProbsBlock) {
        auto at = [&](int64_t j) { return j < G ? a.given[t * G + j] : top_index[t * K + j - G]; };
        const int64_t v = at(i);
        if (none || v < 0 || v >= a.V || (mask && !mask[v])) continue;
        float sum = 0.0f;
        bool first = true;
        for (int64_t j = 0; j < G + K; ++j)
            if (at(j) == v) {
                if (j < i) first = false;
                sum += j < G ? d_given[t * G + j] : d_top[t * K + j - G];
            }
        if (first) d[v] = S::round(c * (smooth(v) + sum));
    }
    }
}

}  // namespace

int64_t log_probs_work(int64_t, int64_t, int) { return 0; }

hipError_t launch_log_probs(const ProbsArgs& a, float* given_out, float* entropy, float* log_sum, float* top_out,
                            int64_t* top_index, float* stats, void*, hipStream_t s) {
    const dim3 grid(match_grid(a.T));
    switch (a.dt) {
        case TP_F32:
            k_probs<F32><<<grid, kProbsBlock, 0, s>>>(a, given_out, entropy, log_sum, top_out, top_index, stats);
            break;
        case TP_F16:
            k_probs<F16><<<grid, kProbsBlock, 0, s>>>(a, given_out, entropy, log_sum, top_out, top_index, stats);
            break;
        default:
            k_probs<BF16><<<grid, kProbsBlock, 0, s>>>(a, given_out, entropy, log_sum, top_out, top_index, stats);
    }
    return hipGetLastError();
}

hipError_t launch_log_probs_back(const ProbsArgs& a, const float* stats, const int64_t* top_index,
                                 const float* d_given, const float* d_entropy, const float* d_log_sum,
                                 const float* d_top, void* d_scores, hipStream_t s) {
    const dim3 grid(match_grid(a.T));
    switch (a.dt) {
        case TP_F32:
            k_probs_back<F32><<<grid, kProbsBlock, 0, s>>>(a, stats, top_index, d_given, d_entropy, d_log_sum, d_top,
                                                           static_cast<uint32_t*>(d_scores));
            break;
        case TP_F16:
            k_probs_back<F16><<<grid, kProbsBlock, 0, s>>>(a, stats, top_index, d_given, d_entropy, d_log_sum, d_top,
                                                           static_cast<uint16_t*>(d_scores));
            break;
        default:
            k_probs_back<BF16><<<grid, kProbsBlock, 0, s>>>(a, stats, top_index, d_given, d_entropy, d_log_sum, d_top,
                                                            static_cast<uint16_t*>(d_scores));
    }
    return hipGetLastError();
}

}  // namespace tp
