// Internal interface of the pair log probabilities (tp_pairs.hip) with the C ABI (tp_capi.hip) and with the tiled products'
// translation units, one per type (tp_pairs_*.hip).
#pragma once

#include "tp_match.hh"
#include "tp_pairs_plan.hh"

namespace tp {

struct PairArgs {
    int dt;  // of images and references (TP_F32, TP_F16, TP_BF16)
    const void* x;
    int64_t M, K, ldx;
    const void* r;
    int64_t N, ldr;
    const int64_t* given;  // [M] or null
    const float* bias;     // [N] or null
    const uint8_t* mask;   // [N], nonzero is allowed, or null
    float c;               // 1 / temperature
};

// Floats of the state that the gradient reads: four of each image (largest score, the others' sum of
// exp(score - largest), the given reference's, and one that is not used), and where there are few images their scores.
inline bool pair_few(int64_t M) { return M <= kFewImages; }
inline int64_t pair_state(int64_t M, int64_t N) { return 4 * M + (pair_few(M) ? M * N : 0); }

int64_t pair_work(int dt, int64_t M, int64_t N, int64_t K);
hipError_t launch_pair_log_probs(const PairArgs& a, float* given_out, float* log_sum, float* state, void* work,
                                 hipStream_t s);
// d_given, d_log_sum: upstream or null; d_x, d_r (of a.dt, contiguous), d_bias: wanted or null
int64_t pair_back_work(int dt, int64_t M, int64_t N, int64_t K, bool d_x, bool d_r);
hipError_t launch_pair_log_probs_back(const PairArgs& a, const float* state, const float* d_given,
                                      const float* d_log_sum, void* d_x, void* d_r, float* d_bias, void* work,
                                      hipStream_t s);

// ------------------------------------------------------------------ tiled products, one type each
// What an image's gradient is made of: G = d score / d(<image, reference> + bias) = a exp(score - most), at_given
// where the reference is the given one.
struct PairCoef {
    float most, a, at_given;
    int given;  // -1: none
};
static_assert(sizeof(PairCoef) == 16, "the gradient's workspace");
constexpr float kLog2e = 1.44269504088896340736f;
#ifdef __HIPCC__
// What a bias adds to a score.  The type's lowest value is a bias like another: no temperature makes -inf of it, which would
// rule its reference out.
__device__ __forceinline__ float times(float bias, float c) {
    const float v = bias * c;
    return v < -3.402823466e38f ? -3.402823466e38f : v;
}
#endif
struct ScorePart {
    float most, sum;  // of a tile's references: the largest score, and sum exp(score - most) without the given one
};
struct PairOff {  // what a tile's references add to their scores
    const float* bias;
    const uint8_t* mask;
    int64_t N;
    float c;  // 1 / temperature
};
// stats: parts [reference tiles][M] and given_score [M]
struct StatsOut {
    PairOff off;
    const int64_t* given;
    int64_t M;
    ScorePart* parts;
    float* given_score;
};
// gradient of the scores: g [references][pieces][ldg] of the type (half precision scaled by the coefficients; of 16 bits the rounded
// values, then what rounding left of them, rounded), and the sums over the images [image tiles][N] (or null)
struct GradOut {
    PairOff off;  // (of this piece's references)
    const PairCoef* coef;
    int64_t M, first;  // first: this piece's first reference
    void* g;
    int64_t ldg;
    float* sums;
    int* look;  // set to 1 where a reference that is ruled out made a product that is not finite
};
// rows x cols times *scale: float32 sums [rows][cols] are added where `before`, and kept where `after`, else out
struct MatrixOut {
    PairOff ruled;  // of the rows: zeros where they are ruled out (N 0: none is)
    const float* scale;
    int64_t rows, cols;
    const float* before;
    float* after;
    void* out;
    int64_t ld;
};
template <class S> struct PairProducts {
    // references x images
    static hipError_t stats(const PairArgs& a, const TilePlan& t, const StatsOut& o, float* part, hipStream_t s);
    static hipError_t grad(const PairArgs& a, const void* r, int64_t n, const TilePlan& t, const GradOut& o, float* part, hipStream_t s);
    // out [n][K] = g x, out [M][K] = g^t r
    static hipError_t d_references(const PairArgs& a, const void* g, int64_t ldg, int64_t n, const TilePlan& t,
                                   const MatrixOut& o, float* part, hipStream_t s);
    static hipError_t d_images(const PairArgs& a, const void* g, int64_t ldg, const void* r, const PairOff& off,
                               const int* look, const TilePlan& t, const MatrixOut& o, float* part, hipStream_t s);
};

}  // namespace tp
