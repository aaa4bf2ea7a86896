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
// Alternatives: a wavefront keeps its best as sorted keys, one per lane: the score's bits in an order that
// integers have, then the complement of its index, so ties go to the lowest index.  Scores above the top-th
// key's are candidates; of a tile with many (the first; rising rows) only those that reach a floor below
// which none can be listed, close to the top-th largest of the lanes' own largest (without it 1 x 4096 with 8
// alternatives takes 26 us instead of 5.3, 4096 x 36864 119 instead of 96).  Candidates go through LDS.  A few are
// inserted one by one, the keys below moving up by a lane; more are merged by counting: a key's place is the
// number of keys above it, which all lanes count at once over broadcast reads (4096 x 36864 bfloat16 with 32
// alternatives: counting from 1 candidate on 84 us, from 13 on 76, never 78; 64 x 294912 fp32 31.4, 30.8 and 33.2).
// More than 32 alternatives leave too few lanes for counting (4096 x 36864 with 64: 116 us, inserted 112).
//
// Split: a row is one wavefront's, or 2, 4 or 8 of a workgroup's, or, where rows are few, several workgroups',
// whose sums and keys k_probs_join joins.  Large calls are bound by memory (4096 x 36864 fp32 with 8 alternatives
// 96 us, 6.3 TB/s; bfloat16 66 to 73 us, 4.1 to 4.6 TB/s, by the instructions of a score), small ones by the chain from launch to result: of
// the 5.3 us of 1 x 4096 a fifth each goes to the start, the loads and sums, and the selection, the rest to the joins.
//
// Scores of -inf count as not allowed.  A NaN makes the row's results NaN.
#include "../../../include/torch_projectors_hip.h"
#include "tp_match.hh"

#include <algorithm>

namespace tp {
namespace {

constexpr int kProbsBlock = 512, kProbsWaves = kProbsBlock / 64;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.693147180559945309417f;

__host__ __device__ __forceinline__ constexpr float neg_inf() { return -__builtin_inff(); }

// The larger of two, NaN if either is (one instruction for two of these).
__device__ __forceinline__ float max_or_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// Larger keys are better: the score's bits in the order of the scores, then the lower index.  0 is no candidate.
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);  // -0 and 0 are equal
    return b ^ (uint32_t(int32_t(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float score_of(uint64_t key) {
    const uint32_t o = uint32_t(key >> 32);
    return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ uint32_t index_of(uint64_t key) { return ~uint32_t(key); }

__device__ __forceinline__ uint32_t read_lane(uint32_t v, int lane) {
    return uint32_t(__builtin_amdgcn_readlane(int(v), lane));
}
__device__ __forceinline__ uint64_t read_lane(uint64_t v, int lane) {
    return uint64_t(read_lane(uint32_t(v >> 32), lane)) << 32 | read_lane(uint32_t(v), lane);
}
// The value that a DPP control brings, `none` where it brings none.
template <int CTRL> __device__ __forceinline__ uint32_t brought(uint32_t v, uint32_t none) {
    return uint32_t(__builtin_amdgcn_update_dpp(int(none), int(v), CTRL, 0xf, 0xf, false));
}
template <int CTRL> __device__ __forceinline__ float brought(float v, float none) {
    return __uint_as_float(brought<CTRL>(__float_as_uint(v), __float_as_uint(none)));
}
// Each lane's f over the lanes up to it (none: f's neutral value): row_shr:1, 2, 4, 8, then row_bcast:15 to
// rows 1 and 3 and row_bcast:31 to rows 2 and 3.
template <class T, class F> __device__ __forceinline__ T scanned(T v, T none, F f) {
    v = f(v, brought<0x111>(v, none));
    v = f(v, brought<0x112>(v, none));
    v = f(v, brought<0x114>(v, none));
    v = f(v, brought<0x118>(v, none));
    const int lane = threadIdx.x & 63;
    const T b = brought<0x142>(v, none);
    v = lane & 16 ? f(v, b) : v;
    const T c = brought<0x143>(v, none);
    return lane & 32 ? f(v, c) : v;
}
// f over all lanes.
template <class F> __device__ __forceinline__ float reduced(float v, float none, F f) {
    return __uint_as_float(read_lane(__float_as_uint(scanned(v, none, f)), 63));
}
template <class F> __device__ __forceinline__ uint32_t reduced(uint32_t v, uint32_t none, F f) {
    return read_lane(scanned(v, none, f), 63);
}

// Number of lanes below this one whose bit is set.
__device__ __forceinline__ int below(uint64_t lanes) {
    return int(__builtin_amdgcn_mbcnt_hi(uint32_t(lanes >> 32), __builtin_amdgcn_mbcnt_lo(uint32_t(lanes), 0)));
}
// A wavefront's LDS.  Only it reads and writes it, in order; the fences keep the compiler to that.
constexpr int kLaneScores = 16;                 // of a tile
constexpr int kTileScores = 64 * kLaneScores;
struct alignas(16) Room {
    uint64_t found[kTileScores + 4];  // candidates, then zeros up to the next multiple of 4
    uint64_t keys[64];
};
__device__ __forceinline__ void lds_order() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

// A value that at least k of the lanes `in` reach, close to the k-th largest: the 12 bits below those that all of
// them share are found one by one, by counting the lanes that reach a value (0 where they are fewer than k).
__device__ __forceinline__ uint32_t floor_of(uint32_t v, bool in, int k) {
    if (__popcll(__ballot(in)) < k) return 0;
    const uint32_t hi = reduced(in ? v : 0u, 0u, [](uint32_t a, uint32_t b) { return max(a, b); });
    const uint32_t lo = reduced(in ? v : ~0u, ~0u, [](uint32_t a, uint32_t b) { return min(a, b); });
    if (hi == lo) return lo;
    uint32_t bit = 0x80000000u >> __clz(hi ^ lo), f = hi & ~(2 * bit - 1);
    v = in ? v : 0u;
#pragma unroll
    for (int i = 0; i < 12; ++i) {
        f = __popcll(__ballot(v >= (f | bit))) >= k ? f | bit : f;
        bit >>= 1;
    }
    return f;
}
// How many of the n keys from p on (zeros after them up to a multiple of 4; p 16-byte aligned) are above `key`; U
// fours of them are on their way at once.
template <int U = 1> __device__ __forceinline__ int above(uint64_t key, const uint64_t* p, int n) {
    int a = 0;
#pragma unroll U
    for (int j = 0; j < n; j += 4) {
        const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(p + j), y = *reinterpret_cast<const ulonglong2*>(p + j + 2);
        a += (x.x > key ? 1 : 0) + (x.y > key ? 1 : 0) + (y.x > key ? 1 : 0) + (y.y > key ? 1 : 0);
    }
    return a;
}

// The same of two sorted lists of n keys, one after the other, by searching them.
__device__ __forceinline__ int above_in_two(uint64_t key, const uint64_t* p, int n) {
    int a[2] = {};
#pragma unroll 1
    for (int b = 1 << (31 - __clz(n)); b; b >>= 1)
#pragma unroll
        for (int l = 0; l < 2; ++l) a[l] += a[l] + b <= n && p[l * n + min(a[l] + b, n) - 1] > key ? b : 0;
    return a[0] + a[1];
}

// The best keys of a wavefront, sorted, one per lane below top, and the score of the top-th (-inf while there are
// fewer).
struct Best {
    uint64_t key = 0;
    float least = neg_inf();

    // Merge room.found[0, n).
    __device__ __forceinline__ void take(int n, int top, Room& room, int lane) {
        if (lane < 4) room.found[n + lane] = 0;
        lds_order();
        int i = 0;
        if (!read_lane(key, 0)) {  // the first ones
            const uint64_t mine = lane < n ? room.found[lane] : 0;
            i = min(n, 64);
            place(mine, above(mine, room.found, i), top, room, lane);
        }
        if (i == n) {
        } else if (n <= 12 || top > 32) {
            for (; i < n; ++i) {
                const uint64_t k = room.found[i], before = uint64_t(brought<0x138>(uint32_t(key >> 32), ~0u)) << 32 |
                                                           brought<0x138>(uint32_t(key), ~0u);  // wave_shr:1
                key = lane >= top ? 0 : key > k ? key : before > k ? k : before;
            }
        } else {
            const int step = (64 - top) & ~3;
            for (; i < n; i += step) {
                const int count = min(step, n - i);
                const uint64_t mine = lane < top ? key : lane - top < count ? room.found[i + lane - top] : 0;
                // (of many equal ones most are below: 64 x 294912 of one value 27 us, 44 without)
                if (!__ballot(lane >= top && mine > read_lane(key, top - 1))) continue;
                room.keys[lane] = key;
                lds_order();
                place(mine, above(mine, room.found + i, count) + above(mine, room.keys, top), top, room, lane);
            }
        }
        const uint64_t last = read_lane(key, top - 1);
        least = last ? score_of(last) : neg_inf();
    }

    // Each lane's key, unless it is 0, to its place in the list.
    __device__ __forceinline__ void place(uint64_t mine, int at, int top, Room& room, int lane) {
        lds_order();
        room.keys[lane] = 0;
        if (mine && at < top) room.keys[at] = mine;
        lds_order();
        key = room.keys[lane];
        lds_order();
    }
};

// Sums over scores relative to their largest: z in units of 1 / (c log2 e), i.e. exponents of 2.
struct Sums {
    float m, s, u;
};
// z is clamped to where its exponential is 0, so that z exp2(z) is 0 and not NaN for -inf.
__device__ __forceinline__ void add_score(Sums& a, float x, float c2) {
    const float z = fmaxf((x - a.m) * c2, -200.0f), e = __builtin_amdgcn_exp2f(z);
    a.s += e;
    a.u = __builtin_fmaf(z, e, a.u);
}
// The sums of a relative to m >= a.m.
__device__ __forceinline__ Sums moved(const Sums& a, float m, float c2) {
    const float z = fmaxf((a.m - m) * c2, -200.0f), f = __builtin_amdgcn_exp2f(z);
    return Sums{m, a.s * f, __builtin_fmaf(a.s, z, a.u) * f};
}
__device__ __forceinline__ Sums joined(const Sums& a, const Sums& b, float c2) {
    const float m = max_or_nan(a.m, b.m);
    const Sums p = moved(a, m, c2), q = moved(b, m, c2);
    return Sums{m, p.s + q.s, p.u + q.u};
}
// All lanes' sums joined: their largest m first, then one rescaling, then plain sums.
__device__ __forceinline__ Sums wave_joined(Sums a, float c2) {
    const float m = reduced(a.m, neg_inf(), [](float x, float y) { return max_or_nan(x, y); });
    a = moved(a, m, c2);
    const auto add = [](float x, float y) { return x + y; };
    return Sums{m, reduced(a.s, 0.0f, add), reduced(a.u, 0.0f, add)};
}

// A lane's scores of the tile at v0: packs of neighbours, lane after lane.  Masked ones and those from v1 on
// are -inf.
template <class S> __device__ __forceinline__ int64_t tile_index(int64_t v0, int lane, int i) {
    return v0 + (i / Pack<S>::n * 64 + lane) * Pack<S>::n + i % Pack<S>::n;
}
template <class S> using Tile = Pack<S>[kLaneScores / Pack<S>::n];
// A tile that is whole, as it is stored: not waited for before it is widened.
template <class S>
__device__ __forceinline__ void load_whole(const typename S::Bits* x, int64_t v0, bool stream, int lane, Tile<S>& w) {
    constexpr int n = Pack<S>::n, P = kLaneScores / n;
    if (stream) {
#pragma unroll
        for (int p = 0; p < P; ++p) w[p] = stream_pack<S>(x + tile_index<S>(v0, lane, p * n));
    } else {
#pragma unroll
        for (int p = 0; p < P; ++p) w[p] = load_pack<S>(x + tile_index<S>(v0, lane, p * n));
    }
}
// The scores of the tile at v0: of w where that is loaded.
template <class S>
__device__ __forceinline__ void tile_scores(const typename S::Bits* x, const uint8_t* mask, int64_t v0, int64_t v1,
                                            bool loaded, const Tile<S>& w, int lane, float (&f)[kLaneScores]) {
    constexpr int n = Pack<S>::n, P = kLaneScores / n;
    if (loaded) {
#pragma unroll
        for (int i = 0; i < kLaneScores; ++i) f[i] = S::widen(w[i / n].v[i % n]);
    } else {
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const int64_t v = tile_index<S>(v0, lane, p * n);
            if (v + n <= v1) {
                const Pack<S> r = load_pack<S>(x + v);
#pragma unroll
                for (int i = 0; i < n; ++i) f[p * n + i] = S::widen(r.v[i]);
            } else {
#pragma unroll
                for (int i = 0; i < n; ++i) f[p * n + i] = v + i < v1 ? S::widen(x[v + i]) : neg_inf();
            }
        }
    }
    if (mask) {
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const int64_t v = tile_index<S>(v0, lane, p * n);
            uint8_t b[n];
            if (v + n <= v1) {
                __builtin_memcpy(b, mask + v, n);
            } else {
#pragma unroll
                for (int i = 0; i < n; ++i) b[i] = v + i < v1 ? mask[v + i] : 0;
            }
#pragma unroll
            for (int i = 0; i < n; ++i)
                if (!b[i]) f[p * n + i] = neg_inf();
        }
    }
}
template <class S>
__device__ __forceinline__ void load_tile(const typename S::Bits* x, const uint8_t* mask, int64_t v0, int64_t v1,
                                          bool stream, int lane, float (&f)[kLaneScores]) {
    Tile<S> w;
    const bool whole = v0 + kTileScores <= v1;
    if (whole) load_whole<S>(x, v0, stream, lane, w);
    tile_scores<S>(x, mask, v0, v1, whole, w, lane, f);
}

// Scores [v0, v1) of a row, by one wavefront.
template <class S>
__device__ __forceinline__ void scan_scores(const typename S::Bits* x, const uint8_t* mask, int64_t v0, int64_t v1,
                                            float c2, int top, bool stream, int lane, Room& room, Sums& sums, Best& best) {
    // 16-bit scores, half as many bytes a tile: the next tile is on its way while one is looked at (4096 x 36864
    // with 8 alternatives 82 -> 73 us; of fp32 other wavefronts' tiles are enough, 8192 x 4300 35.9 against 39.2)
    constexpr bool ahead = sizeof(typename S::Bits) == 2;
    Tile<S> w;
    bool loaded = ahead && v0 + kTileScores <= v1;
    if (loaded) load_whole<S>(x, v0, stream, lane, w);
    for (; v0 < v1; v0 += kTileScores) {
        float f[kLaneScores];
        if (!ahead) {
            loaded = v0 + kTileScores <= v1;
            if (loaded) load_whole<S>(x, v0, stream, lane, w);
        }
        tile_scores<S>(x, mask, v0, v1, loaded, w, lane, f);
        if (ahead) {
            loaded = v0 + 2 * kTileScores <= v1;
            if (loaded) load_whole<S>(x, v0 + kTileScores, stream, lane, w);
        }
        float most = f[0];
#pragma unroll
        for (int i = 1; i < kLaneScores; ++i) most = max_or_nan(most, f[i]);
        sums = moved(sums, max_or_nan(sums.m, most), c2);
#pragma unroll
        for (int i = 0; i < kLaneScores; ++i) add_score(sums, f[i], c2);
        if (!top) continue;
        if (__ballot(most != most)) {  // (the largest without the NaN)
            most = f[0];
#pragma unroll
            for (int i = 1; i < kLaneScores; ++i) most = fmaxf(most, f[i]);
            if (most != most) most = neg_inf();
        }
        const uint64_t lanes = __ballot(most > best.least);
        if (!lanes) continue;
        const uint32_t floor = __popcll(lanes) > 4 ? floor_of(order_of(most), most > best.least, top) : 0;
        const float from = score_of(uint64_t(max(floor, order_of(best.least) + 1)) << 32);  // (past +inf: a NaN)
        int n = 0;
#pragma unroll
        for (int i = 0; i < kLaneScores; ++i) {
            const uint64_t set = __ballot(f[i] >= from);
            if (!set) continue;
            if (f[i] >= from)
                room.found[n + below(set)] =
                    uint64_t(order_of(f[i])) << 32 | uint32_t(~uint32_t(tile_index<S>(v0, lane, i)));
            n += __popcll(set);
        }
        best.take(n, top, room, lane);
    }
}

// Merge the lists of `blocks` parts, `top` keys each, 1024 keys at a time, of which those below a floor are left out:
// the top-th largest of the lists' first 64 keys (of more lists' first keys, of the lanes' largest).
__device__ __forceinline__ void join_keys(Best& best, const uint64_t* p, int blocks, int top, Room& room, int lane) {
    constexpr int N = kLaneScores;
    const int count = blocks * top;
    uint64_t first = 0;
    for (int b = lane; b < max(blocks, 64); b += 64) {
        const int rank = b / blocks;
        first = max(first, rank < top ? p[(b - rank * blocks) * top + rank] : 0);
    }
    uint32_t floor = 0;
    for (int i0 = 0; i0 < count; i0 += 64 * N) {
        uint64_t k[N];
#pragma unroll
        for (int i = 0; i < N; ++i) k[i] = i0 + i * 64 + lane < count ? p[i0 + i * 64 + lane] : 0;
        if (i0 == 0) floor = floor_of(uint32_t(first >> 32), first != 0, top);
        const uint64_t from = max(read_lane(best.key, top - 1) + 1, uint64_t(floor) << 32);
        int n = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (i0 + i * 64 >= count) break;
            const uint64_t set = __ballot(k[i] >= from);
            if (!set) continue;
            if (k[i] >= from) room.found[n + below(set)] = k[i];
            n += __popcll(set);
        }
        best.take(n, top, room, lane);
    }
}

struct ProbsOut {
    float *given, *entropy, *log_sum, *top;
    int64_t* top_index;
    float* stats;
};

// A lane's given candidate of row t: its index, and its score (-inf where masked or out of range).
__device__ __forceinline__ int64_t given_index(const ProbsArgs& a, int64_t t, int64_t g) {
    return g < a.G ? a.given[t * a.G + g] : -1;
}
template <class S> __device__ __forceinline__ float given_score(const ProbsArgs& a, int64_t t, int64_t v) {
    if (v < 0 || v >= a.V || (a.mask && !a.mask[t * a.mask_stride + v])) return neg_inf();
    return S::widen(static_cast<const typename S::Bits*>(a.scores)[t * a.stride + v]);
}

// The results of row t, by one wavefront, from its sums and keys.
template <class S>
__device__ __forceinline__ void write_row(const ProbsArgs& a, const ProbsOut& o, int64_t t, const Sums& sums, uint64_t key,
                                          int64_t given, float given_x, int lane) {
    const float m = sums.m, c = a.c;
    const bool none = m == neg_inf();
    const float ls = m == __builtin_inff() ? __builtin_nanf("") : __builtin_amdgcn_logf(sums.s) * kLn2;  // (s >= 1)
    if (lane == 0) {
        const float H = none ? 0.0f : !isfinite(m) ? __builtin_nanf("") : ls - sums.u * kLn2 / sums.s;
        o.entropy[t] = H;
        o.log_sum[t] = isfinite(m) ? __builtin_fmaf(m, c, ls) : m;
        if (o.stats) *reinterpret_cast<float4*>(o.stats + t * kProbsStats) = float4{m, ls, H, 0.0f};
    }
    for (int64_t g = lane; g < a.G; g += 64) {
        const int64_t v = g < 64 ? given : given_index(a, t, g);
        const float x = g < 64 ? given_x : given_score<S>(a, t, v);
        float lp = 0.0f;
        if (v != -1) {
            if (v < 0 || v >= a.V) lp = __builtin_nanf("");
            else lp = none ? m : x == neg_inf() && m == m ? x : (x - m) * c - ls;
        }
        o.given[t * a.G + g] = lp;
    }
    if (lane < a.top) {
        o.top[t * a.top + lane] = m != m ? m : key ? (score_of(key) - m) * c - ls : neg_inf();
        o.top_index[t * a.top + lane] = key ? int64_t(index_of(key)) : -1;
    }
}

// What the workgroups of a row leave for k_probs_join where there are several: their sums, and their keys.
struct Parts {
    Sums* sums;      // [T][blocks]
    uint64_t* keys;  // [T][blocks][top]
};

// `group` wavefronts of a workgroup per row: 1, 2, 4 or 8, and with 8 `blocks` workgroups, whose parts are joined.
template <class S, int group>
__global__ __launch_bounds__(kProbsBlock, 4) void k_probs(ProbsArgs a, ProbsOut o, int blocks, int64_t span, bool stream,
                                                      Parts parts) {
    constexpr int rows = kProbsWaves / group;  // of a workgroup
    __shared__ Sums sums_of[kProbsWaves];
    __shared__ Room rooms[kProbsWaves];
    __shared__ __attribute__((aligned(16))) uint64_t keys_of[kProbsWaves * kMaxTop], best_of[kMaxTop];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const float c2 = a.c2;
    const int list = max((a.top + 3) & ~3, 8);  // keys and zeros of a wavefront in keys_of
    const int s = 31 - __clz(kProbsBlock / kProbsWaves / list);
    const int64_t items = rows > 1 ? (a.T + rows - 1) / rows : a.T * blocks;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        // wavefront `part` of row t
        const int64_t t = rows > 1 ? item * rows + wave / group : blocks == 1 ? item : over(item, blocks);
        const int64_t part = rows > 1 ? wave % group : (item - t * blocks) * kProbsWaves + wave;
        const bool in = rows == 1 || t < a.T, writes = in && wave % group == 0;
        Sums sums{neg_inf(), 0.0f, 0.0f};
        Best best;
        const int64_t given = writes && blocks == 1 ? given_index(a, t, lane) : -1;
        float given_x = neg_inf();
        if (in) {
            const auto* x = static_cast<const typename S::Bits*>(a.scores) + t * a.stride;
            const int64_t v0 = part * span, v1 = min(v0 + span, a.V);
            scan_scores<S>(x, a.mask ? a.mask + t * a.mask_stride : nullptr, v0, v1, c2, a.top, stream,
                           lane, rooms[wave], sums, best);
            given_x = given_score<S>(a, t, given);
            sums = wave_joined(sums, c2);
        }
        if (group > 1) {
            if (lane == 0) sums_of[wave] = sums;
            if (lane < list) keys_of[wave * list + lane] = best.key;
            if (group == kProbsWaves && threadIdx.x < kMaxTop) best_of[threadIdx.x] = 0;
            __syncthreads();
            if (group == kProbsWaves && a.top) {
                // a key's place is the number of keys above it, of which 2^s lanes count some each (lists of more
                // than 8 are searched)
                const int i = threadIdx.x >> s, p = threadIdx.x & ((1 << s) - 1);
                const uint64_t mine = i < kProbsWaves * list ? keys_of[i] : 0;
                int more = 0;
                if (s == 3)  // (list is 8)
                    more = above<2>(mine, keys_of + 8 * p, 8);
                else if (mine)
                    for (int w = 2 * p; w < kProbsWaves; w += 2 << s) more += above_in_two(mine, keys_of + w * list, list);
                for (int d = 1; d < 1 << s; d <<= 1) more += __shfl_xor(more, d);
                if (mine && p == 0 && more < a.top) best_of[more] = mine;
                __syncthreads();
                best.key = best_of[lane];
            }
            if (writes) {
                sums = wave_joined(lane < group ? sums_of[wave + lane] : Sums{neg_inf(), 0.0f, 0.0f}, c2);
                if (group < kProbsWaves && a.top)
                    for (int w = wave + 1; w < wave + group; ++w) {
                        if (lane < a.top) rooms[wave].found[lane] = keys_of[w * list + lane];
                        best.take(a.top, a.top, rooms[wave], lane);
                    }
            }
            __syncthreads();
        }
        if (!writes) continue;
        if (blocks == 1) {
            write_row<S>(a, o, t, sums, best.key, given, given_x, lane);
        } else {
            if (lane == 0) parts.sums[item] = sums;
            if (lane < a.top) parts.keys[item * a.top + lane] = best.key;
        }
    }
}

// One wavefront per row: its `blocks` parts.
template <class S>
__global__ __launch_bounds__(64) void k_probs_join(ProbsArgs a, ProbsOut o, int blocks, Parts parts) {
    __shared__ Room room;
    const int lane = threadIdx.x;
    const float c2 = a.c2;
    for (int64_t t = blockIdx.x; t < a.T; t += gridDim.x) {
        const int64_t given = given_index(a, t, lane);
        const Sums* of = parts.sums + t * blocks;
        Sums sums = lane < blocks ? of[lane] : Sums{neg_inf(), 0.0f, 0.0f};
        Best best;
        if (a.top) join_keys(best, parts.keys + t * blocks * a.top, blocks, a.top, room, lane);
        const float given_x = given_score<S>(a, t, given);
        for (int b = lane + 64; b < blocks; b += 64) sums = joined(sums, of[b], c2);
        sums = wave_joined(sums, c2);
        write_row<S>(a, o, t, sums, best.key, given, given_x, lane);
    }
}

// Wavefronts of a row, and the scores of each: as many as fill the card (16 on each CU), none with less than a
// tile; a whole workgroup's where each has a CU of its own (its join is the faster one, with half of the wavefronts
// without scores: 1 x 4096 with 8 alternatives 6.3 us by 4 of 8 wavefronts, 5.4 by 8; 100 rows 7.3 and 5.8; but 512
// rows of 2048 6.2 by 2, 6.8 by 8).
struct ProbsPlan {
    int waves;
    int64_t span;
};
ProbsPlan probs_plan(int64_t T, int64_t V) {
    const int64_t tiles = (V + kTileScores - 1) / kTileScores;
    const int64_t most = std::min<int64_t>((4096 + T - 1) / T, tiles);
    int64_t w = 1;
    while (w < most && w < kProbsWaves) w *= 2;
    if (w > 1 && T <= 256) w = kProbsWaves;
    if (most > kProbsWaves) w = (most + kProbsWaves - 1) / kProbsWaves * kProbsWaves;
    const int64_t span = (tiles + w - 1) / w * kTileScores;
    return {int(w), span};
}

// The gradient: a wavefront per stretch of a row.  Every score's share but that of the given and listed ones first,
// then those scores' once more with it, each by one lane.  Memory bound: reads and writes each score once
// (4096 x 36864 fp32 192 us, 6.3 TB/s).
//
// MANY, more than 64 given and listed candidates of a row: each wavefront walks all of them once, 64 at a time, and adds
// what falls into its stretch up in LDS, in the order of the candidates (so that the result is always the same): lanes
// with places of their own at once, of lanes that share a place all of them by one.  Each candidate is so read once for
// each 2048 scores of its row (or fewer, a stretch), and added once: 4096 x 4300 fp32 with 65 given 26 us, 1024 57; 512 x
// 36864 with 65 27, 4096 137, 36864 1250, bound by the walks (18 of each row's candidates).
constexpr int kBackBlock = 256, kBackWaves = kBackBlock / 64;
constexpr int kManySpan = 2048;
struct alignas(16) ManyRoom {
    float added[kManySpan];  // upstream gradients at the places of the stretch
    uint8_t owner[kManySpan];
};

template <class S, bool MANY>
__global__ __launch_bounds__(kBackBlock) void k_probs_back(ProbsArgs a, int64_t span, bool stream, const float* __restrict__ stats,
                                                            const int64_t* __restrict__ top_index,
                                                            const float* __restrict__ d_given,
                                                            const float* __restrict__ d_entropy,
                                                            const float* __restrict__ d_log_sum,
                                                            const float* __restrict__ d_top,
                                                            typename S::Bits* __restrict__ d_scores) {
    __shared__ ManyRoom rooms[MANY ? kBackWaves : 1];
    const int lane = threadIdx.x & 63;
    const float c = a.c, c2 = a.c2;
    const int64_t G = d_given ? a.G : 0;
    const int K = d_top ? a.top : 0;
    const uint32_t spans = uint32_t(over(a.V + span - 1, uint32_t(span)));
    for (int64_t item = int64_t(blockIdx.x) * kBackWaves + (threadIdx.x >> 6); item < a.T * spans;
         item += int64_t(gridDim.x) * kBackWaves) {
        const int64_t t = over(item, spans), first = (item - t * spans) * span, end = min(first + span, a.V);
        const auto* x = static_cast<const typename S::Bits*>(a.scores) + t * a.stride;
        auto* d = d_scores + t * a.V;
        const uint8_t* mask = a.mask ? a.mask + t * a.mask_stride : nullptr;
        const int64_t n = G + K;
        auto index_at = [&](int64_t j) { return j < G ? a.given[t * G + j] : j < n ? top_index[t * K + j - G] : -1; };
        auto up_at = [&](int64_t j) { return j < G ? d_given[t * G + j] : j < n ? d_top[t * K + j - G] : 0.0f; };
        // what a candidate takes from the row's sum: nothing for -1, and of one out of range, whose log probability
        // is NaN, a NaN unless its upstream gradient is 0
        auto share = [&](int64_t v, float up) {
            return v == -1 ? 0.0f : (v >= 0 && v < a.V) || up == 0.0f ? up : __builtin_nanf("");
        };
        // a lane's given or listed candidate and its upstream gradient
        const int64_t mine = MANY ? -1 : index_at(lane);
        const float up = MANY ? 0.0f : up_at(lane);
        const float4 st = *reinterpret_cast<const float4*>(stats + t * kProbsStats);
        const float dL = d_log_sum ? d_log_sum[t] : 0.0f, dH = d_entropy ? d_entropy[t] : 0.0f;
        float f[kLaneScores];
        load_tile<S>(x, mask, first, end, stream, lane, f);
        auto here = [&](int64_t v) { return v >= first && v < end && !(mask && !mask[v]); };
        const bool fix = here(mine);
        const float at_mine = fix ? S::widen(x[mine]) : 0.0f;
        const float m = st.x, ls = st.y, H = st.z, ls2 = ls * kLog2e;
        const bool none = m == neg_inf();
        float all = -share(mine, up);
        if constexpr (MANY) {
            ManyRoom& room = rooms[threadIdx.x >> 6];
            for (int i = 4 * lane; i < kManySpan; i += 256) *reinterpret_cast<float4*>(room.added + i) = float4{};
            lds_order();
            for (int64_t j0 = 0; j0 < n; j0 += 64) {
                const int64_t v = index_at(j0 + lane);
                const float u = up_at(j0 + lane);
                all -= share(v, u);
                const bool in = here(v);
                uint64_t left = __ballot(in);
                if (!left) continue;
                const int place = in ? int(v - first) : 0;
                // one lane's number stays at a place that several share
                if (in) room.owner[place] = uint8_t(lane);
                lds_order();
                uint64_t shared = __ballot(in && room.owner[place] != lane);
                lds_order();
                while (shared) {
                    const int at = int(read_lane(uint32_t(place), __ffsll(static_cast<unsigned long long>(shared)) - 1));
                    const uint64_t same = __ballot(in && place == at);
                    const float sum = wave_sum(in && place == at ? u : 0.0f);
                    if (lane == 0) room.added[at] += sum;
                    lds_order();
                    left &= ~same;
                    shared &= ~same;
                }
                if (left >> lane & 1) room.added[place] += u;
                lds_order();
            }
        }
        all = wave_sum(all) + dL;
        // the gradient of score f without what is given or listed there, c p (all - dH (ln p + H)); 0 where not allowed,
        // and everywhere in a row that allows nothing; NaN where allowed in a row with a NaN or +inf
        const bool plain = !none && ls == ls;
        const float at_0 = plain ? c * __builtin_fmaf(-dH, H, all) : none ? 0.0f : __builtin_nanf("");
        const float slope = plain ? c * -dH * kLn2 : 0.0f;
        // (where a factor is not finite, 0 times it is not 0)
        const bool all_finite = !__ballot(!isfinite(at_0) || !isfinite(slope));
        auto smooth = [&](float f) {
            const float lp2 = fmaxf((f - m) * c2 - ls2, -200.0f);
            return __builtin_amdgcn_exp2f(lp2) * __builtin_fmaf(slope, lp2, at_0);
        };
        for (int64_t v0 = first; v0 < end; v0 += kTileScores) {
            if (v0 != first) load_tile<S>(x, mask, v0, end, stream, lane, f);
            constexpr int P = Pack<S>::n;
#pragma unroll
            for (int p = 0; p < kLaneScores / P; ++p) {
                const int64_t v = tile_index<S>(v0, lane, p * P);
                float g[P];
#pragma unroll
                for (int i = 0; i < P; ++i) g[i] = smooth(f[p * P + i]);
                if (!all_finite)
#pragma unroll
                    for (int i = 0; i < P; ++i)
                        if (f[p * P + i] == neg_inf()) g[i] = 0.0f;
                if constexpr (MANY)
                    if (plain)
#pragma unroll
                        for (int i = 0; i < P; ++i)
                            g[i] = __builtin_fmaf(c, rooms[threadIdx.x >> 6].added[v - first + i], g[i]);
                Pack<S> w;
#pragma unroll
                for (int i = 0; i < P; ++i) w.v[i] = S::round(g[i]);
                if (v + P <= end) {
                    if (stream) stream_pack<S>(d + v, w);
                    else store_pack<S>(d + v, w);
                } else {
#pragma unroll
                    for (int i = 0; i < P; ++i)
                        if (v + i < end) d[v + i] = w.v[i];
                }
            }
        }
        if constexpr (MANY) {
            lds_order();
        } else if (plain) {
            // (the stores above come before those below: one wavefront's, in order)
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            // what is given or listed at the same score is summed by the first lane that holds it
            float sum = 0.0f;
            bool is_first = true;
            for (int l = 0; l < int(n); ++l) {
                const bool same = read_lane(uint64_t(mine), l) == uint64_t(mine);
                if (same) sum += __uint_as_float(read_lane(__float_as_uint(up), l));
                if (same && l < lane) is_first = false;
            }
            if (fix && is_first) d[mine] = S::round(__builtin_fmaf(c, sum, smooth(at_mine)));
        }
    }
}

// Scores of about the last cache's size (256 MB) or more are streamed past the caches.  Measured, forward and gradient:
// 4096 x 36864 bfloat16 (288 MB) 180 us through the caches, 160 streamed, fp32 (576 MB) 351 and 308; but 1000 x 16384
// fp32 (62 MB) 45 and 47.
constexpr int64_t kStreamScores = int64_t(192) << 20;
bool streams(const ProbsArgs& a, size_t size) { return a.T * a.V * int64_t(size) >= kStreamScores; }

// Scores of a stretch of the gradient: 8 KB, but one tile where stretches would be fewer than eight to a CU, and of
// fp32 scores that are streamed.  Measured with 1, 2 and 4 tiles: 4096 x 4300 fp32 30, 25 and 26 us, bfloat16 (8192
// rows) 45, 35 and 31; streamed, 4096 x 36864 fp32 192, 195 and 213, bfloat16 140, 109 and 101; 8 x 294912 fp32
// 6.7, 6.9 and 8.5.
int64_t back_span(const ProbsArgs& a, size_t size) {
    const int64_t tiles = a.T * ((a.V + kTileScores - 1) / kTileScores), most = 8192 / int64_t(size) / kTileScores;
    return (tiles < 2048 * most || (size == 4 && streams(a, size)) ? 1 : most) * int64_t(kTileScores);
}

template <class S, int group>
hipError_t probs(const ProbsArgs& a, const ProbsOut& o, const ProbsPlan& p, void* work, hipStream_t s) {
    constexpr int rows = kProbsWaves / group;
    const int blocks = std::max(p.waves / kProbsWaves, 1);
    auto* keys = static_cast<uint64_t*>(work);
    const Parts parts{reinterpret_cast<Sums*>(keys + a.T * blocks * a.top), keys};
    k_probs<S, group><<<match_grid(rows > 1 ? (a.T + rows - 1) / rows : a.T * blocks), kProbsBlock, 0, s>>>(a, o, blocks,
                                                                                                     p.span, streams(a, sizeof(typename S::Bits)), parts);
    if (hipError_t e = hipGetLastError()) return e;
    if (blocks > 1) k_probs_join<S><<<match_grid(a.T), 64, 0, s>>>(a, o, blocks, parts);
    return hipGetLastError();
}
template <class S> hipError_t probs(const ProbsArgs& a, const ProbsOut& o, void* work, hipStream_t s) {
    const ProbsPlan p = probs_plan(a.T, a.V);
    switch (p.waves) {
        case 1: return probs<S, 1>(a, o, p, work, s);
        case 2: return probs<S, 2>(a, o, p, work, s);
        case 4: return probs<S, 4>(a, o, p, work, s);
        default: return probs<S, 8>(a, o, p, work, s);
    }
}

template <class S>
hipError_t probs_back(const ProbsArgs& a, const float* stats, const int64_t* top_index, const float* d_given,
                      const float* d_entropy, const float* d_log_sum, const float* d_top, void* d_scores,
                      hipStream_t s) {
    const bool many = (d_given ? a.G : 0) + (d_top ? a.top : 0) > 64;
    const int64_t best = back_span(a, sizeof(typename S::Bits)), span = many ? std::min<int64_t>(best, kManySpan) : best;
    const int64_t items = a.T * ((a.V + span - 1) / span);
    (many ? k_probs_back<S, true> : k_probs_back<S, false>)<<<match_grid((items + kBackWaves - 1) / kBackWaves), kBackBlock, 0, s>>>(
        a, span, streams(a, sizeof(typename S::Bits)), stats, top_index, d_given, d_entropy, d_log_sum, d_top, static_cast<typename S::Bits*>(d_scores));
    return hipGetLastError();
}

}  // namespace

int64_t log_probs_work(int64_t T, int64_t V, int top) {
    const ProbsPlan p = probs_plan(T, V);
    return p.waves > kProbsWaves ? T * (p.waves / kProbsWaves) * (int64_t(sizeof(Sums)) + 8 * int64_t(top)) : 0;
}

hipError_t launch_log_probs(const ProbsArgs& a, float* given_out, float* entropy, float* log_sum, float* top_out,
                            int64_t* top_index, float* stats, void* work, hipStream_t s) {
    const ProbsOut o{given_out, entropy, log_sum, top_out, top_index, stats};
    switch (a.dt) {
        case TP_F32: return probs<F32>(a, o, work, s);
        case TP_F16: return probs<F16>(a, o, work, s);
        default: return probs<BF16>(a, o, work, s);
    }
}

hipError_t launch_log_probs_back(const ProbsArgs& a, const float* stats, const int64_t* top_index,
                                 const float* d_given, const float* d_entropy, const float* d_log_sum,
                                 const float* d_top, void* d_scores, hipStream_t s) {
    switch (a.dt) {
        case TP_F32: return probs_back<F32>(a, stats, top_index, d_given, d_entropy, d_log_sum, d_top, d_scores, s);
        case TP_F16: return probs_back<F16>(a, stats, top_index, d_given, d_entropy, d_log_sum, d_top, d_scores, s);
        default: return probs_back<BF16>(a, stats, top_index, d_given, d_entropy, d_log_sum, d_top, d_scores, s);
    }
}

}  // namespace tp
