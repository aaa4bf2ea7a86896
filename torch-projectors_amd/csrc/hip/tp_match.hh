// Internal interface of the matching operators (tp_scores.hip, tp_probs.hip,
// tp_route.hip) with the C ABI (tp_capi.hip), and what their kernels share.
#pragma once

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace tp {

// ------------------------------------------------------------------ 8-bit blocks (tp_scores.hip)
constexpr int kScaleBlock = 128;  // values that share a scale
constexpr int kScaleRows = 16;    // rows of the scales are padded to this
constexpr int64_t kMaxScoreRows = int64_t(1) << 26;  // of either side (a launch has fewer than 2^32 lanes)

inline int64_t scale_rows(int64_t rows) { return (rows + kScaleRows - 1) / kScaleRows * kScaleRows; }

inline int64_t block_count(int64_t cols) { return (cols + kScaleBlock - 1) / kScaleBlock; }

// x [rows, cols] of `dt`, rows `stride` elements apart -> codes [rows, 128 nb], scales [nb, scale_rows(rows)].
hipError_t launch_quantize_blocks(int dt, const void* x, int64_t rows, int64_t cols, int64_t stride, void* codes,
                                  void* scales, hipStream_t s);

// Bytes of workspace that launch_block_scores needs for these sizes (0: none).
int64_t block_scores_work(int64_t M, int64_t N, int64_t nb);
// out [M, N] (TP_F32 or TP_BF16) = bias[n] + sum over blocks; bias fp32 or null.
hipError_t launch_block_scores(const void* a, const void* sa, int64_t M, const void* b, const void* sb, int64_t N,
                               int64_t nb, const void* bias, int out_dt, void* out, void* work, hipStream_t s);

// The same for rows x [M, cols] of `dt`, `stride` apart, that are quantised first (one row: by the product's own
// kernel, on its way; bytes of work for codes and scales otherwise, then launch_block_scores').
int64_t score_images_work(int64_t M, int64_t N, int64_t cols);
hipError_t launch_score_images(int dt, const void* x, int64_t M, int64_t cols, int64_t stride, const void* b,
                               const void* sb, int64_t N, const void* bias, int out_dt, void* out, void* work,
                               hipStream_t s);

// ------------------------------------------------------------------ log probabilities (tp_probs.hip)
constexpr int kMaxTop = 64;  // a wavefront keeps one alternative per lane

struct ProbsArgs {
    int dt;                      // of the scores (TP_F32, TP_F16, TP_BF16)
    const void* scores;          // [T, V], rows `stride` elements apart
    int64_t T, V, stride;
    const int64_t* given;        // [T, G] or null
    int64_t G;
    const uint8_t* mask;         // [V] (mask_stride 0) or [T, V]: nonzero is allowed; null: all are
    int64_t mask_stride;
    int top;
    float c, c2;  // 1 and log2 e, over the temperature
};
// Statistics of a row that the gradient reads (null where none will): the largest allowed score, ln of the sum of
// exp((x - largest) / temperature), the entropy, and an unused word.
constexpr int kProbsStats = 4;

int64_t log_probs_work(int64_t T, int64_t V, int top);
hipError_t launch_log_probs(const ProbsArgs& a, float* given_out, float* entropy, float* log_sum, float* top_out,
                            int64_t* top_index, float* stats, void* work, hipStream_t s);
// d_*: upstream gradients or null; d_scores [T, V] contiguous, of a.dt.
hipError_t launch_log_probs_back(const ProbsArgs& a, const float* stats, const int64_t* top_index,
                                 const float* d_given, const float* d_entropy, const float* d_log_sum,
                                 const float* d_top, void* d_scores, hipStream_t s);

// ------------------------------------------------------------------ rows by class (tp_route.hip)
constexpr int kMaxClasses = 4096;

int64_t sort_by_class_work(int64_t slots, int64_t classes);
// ids int32 or int64 [slots] -> order [slots], slot [slots], offsets [classes + 1], all int32.
hipError_t launch_sort_by_class(int id_bytes, const void* ids, int64_t slots, int classes, int* order, int* slot,
                                int* offsets, void* work, hipStream_t s);

struct RouteArgs {
    int dt;                // of the rows
    int64_t T, D;          // rows in row order, and values of each
    int k;                 // classes of each row
    const int* slot;       // [T, k]: places in class order
    const int* kept;       // &offsets[classes]: places from there on hold no row
    const float* weights;  // [T, k] or null (ones)
};
// sorted[slot[t, j]] = w[t, j] x[t] (zero where dropped); with `rows` and `d_weights` (both or none) also
// d_weights[t, j] = <x[t], rows[slot[t, j]]>.
hipError_t launch_spread_rows(const RouteArgs& a, const void* x, void* sorted, const void* rows, float* d_weights,
                              hipStream_t s);
// out[t] = sum_j w[t, j] rows[slot[t, j]]; with `x` and `d_weights` (both or none) also
// d_weights[t, j] = <x[t], rows[slot[t, j]]>.
hipError_t launch_gather_rows(const RouteArgs& a, const void* rows, void* out, const void* x, float* d_weights,
                              hipStream_t s);

// Workgroups of a launch over `items`: the kernels stride over the rest (a launch has fewer than 2^32 lanes).
inline unsigned match_grid(int64_t items) {
    return static_cast<unsigned>(items < (int64_t(1) << 22) ? items : int64_t(1) << 22);
}

#ifdef __HIPCC__
// ------------------------------------------------------------------ device helpers
// Storage types: `Bits` as loaded, widened exactly to fp32, rounded once (to nearest even).
struct F32 {
    using Bits = uint32_t;
    static __device__ __forceinline__ float widen(Bits b) { return __uint_as_float(b); }
    static __device__ __forceinline__ Bits round(float f) { return __float_as_uint(f); }
};
struct BF16 {
    using Bits = uint16_t;
    static __device__ __forceinline__ float widen(Bits b) { return __uint_as_float(uint32_t(b) << 16); }
    static __device__ __forceinline__ Bits round(float f) { return __builtin_bit_cast(Bits, static_cast<__bf16>(f)); }
};
struct F16 {
    using Bits = uint16_t;
    static __device__ __forceinline__ float widen(Bits b) { return float(__builtin_bit_cast(_Float16, b)); }
    static __device__ __forceinline__ Bits round(float f) { return __builtin_bit_cast(Bits, static_cast<_Float16>(f)); }
};

// 16 bytes of a storage type at any address that the type itself may have: gfx950 loads and stores
// them in one instruction whatever their alignment.
template <class S> struct Pack {
    static constexpr int n = 16 / int(sizeof(typename S::Bits));
    typename S::Bits v[n];
};
template <class S> __device__ __forceinline__ Pack<S> load_pack(const typename S::Bits* p) {
    Pack<S> r;
    __builtin_memcpy(&r, p, 16);
    return r;
}
template <class S> __device__ __forceinline__ void store_pack(typename S::Bits* p, const Pack<S>& r) {
    __builtin_memcpy(p, &r, 16);
}
// The same for what will not be used again before the caches have lost it anyway (streaming).
template <class S> struct PackBits {
    using Any = uint32_t __attribute__((ext_vector_type(4)));
    using At = uint32_t __attribute__((ext_vector_type(4), aligned(sizeof(typename S::Bits))));
};
template <class S> __device__ __forceinline__ Pack<S> stream_pack(const typename S::Bits* p) {
    const typename PackBits<S>::Any w = __builtin_nontemporal_load(reinterpret_cast<const typename PackBits<S>::At*>(p));
    return __builtin_bit_cast(Pack<S>, w);
}
template <class S> __device__ __forceinline__ void stream_pack(typename S::Bits* p, const Pack<S>& r) {
    __builtin_nontemporal_store(__builtin_bit_cast(typename PackBits<S>::Any, r),
                                reinterpret_cast<typename PackBits<S>::At*>(p));
}

// n / d for n >= 0: in 32 bits where that will do (a 64-bit division is some 100 instructions).
__device__ __forceinline__ int64_t over(int64_t n, uint32_t d) {
    return uint64_t(n) >> 32 ? int64_t(uint64_t(n) / d) : int64_t(uint32_t(n) / d);
}

// Sum over a wavefront, the same in every lane (fixed order).
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    return v;
}
#endif

}  // namespace tp
