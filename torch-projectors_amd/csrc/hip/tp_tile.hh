// Tiled matrix products of the pair log probabilities and of the scores in 8-bit integers: operands staged in LDS, multiplied by the matrix units, and
// handed as fragments to an epilogue.
//
//   D[i, j] = sum over k of A(i, k) B(j, k)
//
// An operand lies in memory with its contraction adjacent (row i holds k = 0, 1, ...) or across (row k holds i = 0,
// 1, ...); the latter is transposed on its way from LDS by ds_read_tr16_b64.  16-bit values go through the bfloat16 or
// half precision units as they are.  float32 values x are cut into three bfloat16 pieces, x = h + m + l exactly: h the
// upper 8 bits of the mantissa, m the rest rounded to 8, l what that leaves, of either sign.  (From some 2^-110 down l has fewer bits: multiples of
// 2^-133 are what is left.)  A product is the six largest of the nine products of pieces: what is left out, m l twice and l l, is below 2^-22 of each product
// and has no sign, so that a sum loses little more than its own rounding.  Six products at the bfloat16 rate are
// faster than the float32 units' one: 190 to 210 TFLOP/s of float32 in large products, where a library product reaches 155.
#pragma once

#include "tp_match.hh"
#include "tp_tile_plan.hh"

namespace tp {

using v8bf = __attribute__((ext_vector_type(8))) __bf16;
using v8h = __attribute__((ext_vector_type(8))) _Float16;
using v16f = __attribute__((ext_vector_type(16))) float;
using v4s = __attribute__((ext_vector_type(4))) short;
using v4i = __attribute__((ext_vector_type(4))) int;
using v16i = __attribute__((ext_vector_type(16))) int;
using v4u = __attribute__((ext_vector_type(4))) uint32_t;
using LocalBytes = const __attribute__((address_space(3))) char*;
using LocalTr = __attribute__((address_space(3))) v4s*;

// How values of a storage type go through the matrix units: in `planes` pieces, `bk` of the contraction at a time
// (128 bytes of each row in LDS, 192 in three planes).  whole: the sums are integers, in the bits of the fragments.
template <class S> struct Units;
// Pairs of 8-bit integers: laid out like 16-bit values, half as many as there are integers.
struct I8x2 {
    using Bits = uint16_t;
};
template <> struct Units<I8x2> {
    static constexpr int planes = 1, bk = 64;
    static constexpr bool whole = true;
    static __device__ __forceinline__ v16f mfma(int4 a, int4 b, v16f c) {
        return __builtin_bit_cast(v16f, __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(v4i, a), __builtin_bit_cast(v4i, b),
                                                                              __builtin_bit_cast(v16i, c), 0, 0, 0));
    }
};
template <> struct Units<BF16> {
    static constexpr int planes = 1, bk = 64;
    static constexpr bool whole = false;
    static __device__ __forceinline__ v16f mfma(int4 a, int4 b, v16f c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
    }
};
template <> struct Units<F16> {
    static constexpr int planes = 1, bk = 64;
    static constexpr bool whole = false;
    static __device__ __forceinline__ v16f mfma(int4 a, int4 b, v16f c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
    }
};
template <> struct Units<F32> {
    static constexpr int planes = 3, bk = 32;
    static constexpr bool whole = false;
    static __device__ __forceinline__ v16f mfma(int4 a, int4 b, v16f c) { return Units<BF16>::mfma(a, b, c); }
};

// A workgroup's tile of BM x BN of D, by WM x WN wavefronts.  DEEP: operands that go straight to LDS do so in four stages of 32 of
// the contraction, else in two of 64.
template <int BM_, int BN_, int WM_, int WN_, bool DEEP_ = false> struct TileShape {
    static constexpr bool DEEP = DEEP_;
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, NT = 64 * WM * WN;
    static constexpr int FM = BM / WM / 32, FN = BN / WN / 32;  // fragments of a wavefront
};

// Eight neighbouring values on their way from memory to LDS.
template <class S> struct Eight {
    Pack<S> w[8 / Pack<S>::n];
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < 8; ++i) set(i, 0);
    }
    __device__ __forceinline__ void set(int i, typename S::Bits b) { w[i / Pack<S>::n].v[i % Pack<S>::n] = b; }
    __device__ __forceinline__ typename S::Bits get(int i) const { return w[i / Pack<S>::n].v[i % Pack<S>::n]; }
    __device__ __forceinline__ void read(const typename S::Bits* p) {
#pragma unroll
        for (int i = 0; i < 8 / Pack<S>::n; ++i) w[i] = load_pack<S>(p + i * Pack<S>::n);
    }
    // as the units take them, plane by plane
    __device__ __forceinline__ void planes(int4 (&out)[Units<S>::planes]) const {
        if constexpr (Units<S>::planes == 1) {
            out[0] = __builtin_bit_cast(int4, w[0]);
        } else {
            uint32_t part[3][4];
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                uint32_t lo = get(i), hi = get(i + 1);
                auto left = [&](uint32_t pair) {
                    lo = __float_as_uint(__uint_as_float(lo) - __uint_as_float(pair << 16));
                    hi = __float_as_uint(__uint_as_float(hi) - __uint_as_float(pair & 0xffff0000u));
                };
                part[0][i / 2] = __builtin_amdgcn_perm(hi, lo, 0x07060302u);  // the upper halves of both
                left(part[0][i / 2]);
                const __attribute__((ext_vector_type(2))) float f{__uint_as_float(lo), __uint_as_float(hi)};
                part[1][i / 2] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f, __attribute__((ext_vector_type(2))) __bf16));
                left(part[1][i / 2]);
                part[2][i / 2] = __builtin_amdgcn_perm(hi, lo, 0x07060302u);
            }
#pragma unroll
            for (int p = 0; p < 3; ++p) out[p] = int4{int(part[p][0]), int(part[p][1]), int(part[p][2]), int(part[p][3])};
        }
    }
};

// One operand of a product.
struct Operand {
    const void* p;
    int64_t ld;           // elements between its rows in memory, at most kMaxStride
    int64_t kdim;         // contraction that there is (zeros count as being there)
    // (contraction across only) where *look is not 0, rows whose byte is zero or whose bias is -inf count as zeros, whatever they
    // hold; each may be null
    const int* look;
    const uint8_t* keep;
    const float* bias;
};

// An operand's part of a tile: DIM rows of D's side by bk of the contraction, CH chunks of eight values a thread.
//   adjacent: LDS row i holds its bk values; chunk c of row i at place c ^ (i / rows in 256 bytes), so that 16 lanes
//             reading one chunk of 16 rows reach each of the 64 banks once
//   across:   LDS row k holds DIM values; four rows of 64 bytes, as 32 lanes read them, at places that differ by 64
// DIRECT: from memory straight to LDS, without registers between (16-bit values whose rows start at 16-byte
// boundaries; a row is a whole number of chunks, or is followed by what makes it one).
template <class S, bool ACROSS, int DIM, int NT, bool DIRECT, int BK> struct Side {
    static constexpr int PL = Units<S>::planes;
    static constexpr int CPR = ACROSS ? DIM / 8 : BK / 8, CH = DIM * BK / 8 / NT;
    static constexpr int kPlane = DIM * BK * 2;  // bytes
    static_assert(CH * 8 * NT == DIM * BK, "whole chunks");
    using Bits = typename S::Bits;

    const char* base;  // the tile's first value at contraction 0
    int64_t ld, dim, kdim;
    bool looks;
    const uint8_t* keep;
    const float* bias;
    uint32_t off[CH];  // bytes from base (+ the step) of each chunk
    int tid;

    static __device__ __forceinline__ int row_of(int slot) { return slot / CPR; }
    static __device__ __forceinline__ int chunk_of(int slot) { return slot % CPR; }
    static __device__ __forceinline__ int swizzle(int row) {
        if (ACROSS) return DIM >= 128 ? (row & 3) << 2 : ((row >> 1) & 1) << 2;
        return (row / (128 / BK)) & (CPR - 1);
    }

    // first: of the tile along D's side; dim_all: what there is of that
    __device__ __forceinline__ void init(const Operand& o, int64_t first, int64_t dim_all, int t) {
        tid = t;
        ld = o.ld;
        looks = ACROSS && o.look && *o.look;
        keep = o.keep;
        bias = o.bias;
        dim = min(dim_all - first, int64_t(DIM));
        kdim = o.kdim;
        base = static_cast<const char*>(o.p) + (ACROSS ? first : first * ld) * int64_t(sizeof(Bits));
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int slot = i * NT + tid, row = row_of(slot), c = chunk_of(slot);
            if (DIRECT) {  // (a place in LDS, and the chunk that belongs there)
                // (rows past the end read the last one where the contraction is adjacent)
                const int from = (c ^ swizzle(row)) * 8, at = ACROSS ? row : min(row, int(dim) - 1);
                off[i] = (uint32_t(at) * uint32_t(ld) + from) * uint32_t(sizeof(Bits));
                continue;
            }
            // rows and chunks past the end read the last one: what comes of them is not stored
            const uint32_t at = ACROSS ? uint32_t(row) * uint32_t(ld) + min(c * 8, (int(dim) - 1) & ~7)
                                       : uint32_t(min(row, int(dim) - 1)) * uint32_t(ld) + c * 8;
            off[i] = at * uint32_t(sizeof(Bits));
        }
    }
    // which rows of the step at k0 count (where it looks: nonzero where the chunk's does)
    __device__ __forceinline__ void look(int64_t k0, uint32_t (&kept)[CH]) const {
        if (looks) {
#pragma unroll
            for (int i = 0; i < CH; ++i) {
                const int64_t k = min(k0 + row_of(i * NT + tid), kdim - 1);
                kept[i] = (!keep || keep[k]) && (!bias || bias[k] != -INFINITY);
            }
        }
    }
    // The step at k0 straight to LDS; what lies outside the operand arrives as zeros, and so do rows that do not count.
    // The loads are written out: behind a builtin the compiler waits for all of them before it reads any transposed fragment, of
    // whichever stage.  They have no registers to return to; arrive() waits for them.  (m0 is reserved: the compiler sets it before each
    // use of its own)
    // from: elements from the operand's first value to those meant
    __device__ __forceinline__ void fill(int64_t k0, const char* lds, int64_t from) const {
        constexpr uint32_t kNowhere = 0x80000000u;
        const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        const char* at = base + (from + (ACROSS ? k0 * ld : 0)) * int64_t(sizeof(Bits));
        // (whole chunks: of a 32-bit word that the buffer ends in the middle of neither half arrives)
        const int64_t values = ACROSS ? (kdim - k0 - 1) * ld + ((dim + 7) & ~int64_t(7)) : (dim - 1) * ld + kdim;
        const int64_t bytes = min(values * int64_t(sizeof(Bits)), int64_t(0x7fffffff));
        // a raw buffer: base address, its upper half, size, and the data format of 32-bit words
        const uint64_t address = reinterpret_cast<uint64_t>(at);
        const v4u src{uint32_t(address), uint32_t(address >> 32) & 0xffffu, uint32_t(bytes), 0x00027000u};
        const int step = ACROSS ? 0 : int(k0 * int64_t(sizeof(Bits)));
        const int left = int(min(kdim - k0, int64_t(BK)));
        uint32_t o[CH];
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int slot = i * NT + tid;
            o[i] = ACROSS || (chunk_of(slot) ^ swizzle(row_of(slot))) * 8 < left ? off[i] : kNowhere;
        }
        if (looks) {
            uint32_t kept[CH];
            look(k0, kept);
#pragma unroll
            for (int i = 0; i < CH; ++i) {
                o[i] = kept[i] ? o[i] : kNowhere;
                asm volatile("" : "+v"(o[i]));  // (waited for here, not by those who do not look)
            }
        }
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const uint32_t to = __builtin_amdgcn_readfirstlane(
                uint32_t(reinterpret_cast<uintptr_t>((LocalBytes)(lds + (i * NT + wave * 64) * 16))));
            asm volatile("s_nop 4\n\ts_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                         :
                         : "s"(to), "v"(o[i]), "s"(src), "s"(step)
                         : "memory");
        }
    }
    // The contraction up to here can be read in whole chunks: every row of a step is there, and the last chunk's read
    // ends inside the operand.
    __device__ __forceinline__ int64_t whole() const {
        const int64_t past = ACROSS ? -dim & 7 : 0;  // values that a row's last chunk reads of the next rows
        if (past && ld == 0) return 0;               // (there are none)
        return max(kdim - (past ? (past + ld - 1) / ld : 0), int64_t(0)) / BK * BK;
    }
    using Regs = Eight<S>[CH];
    __device__ __forceinline__ void load(int64_t k0, Regs& reg, uint32_t (&kept)[CH]) const {
        const char* at = base + (ACROSS ? k0 * ld : k0) * int64_t(sizeof(Bits));
#pragma unroll
        for (int i = 0; i < CH; ++i) reg[i].read(reinterpret_cast<const Bits*>(at + off[i]));
        look(k0, kept);
    }
    // The same for a step that is not whole.
    __device__ __forceinline__ void load_some(int64_t k0, Regs& reg, uint32_t (&kept)[CH]) const {
        const char* at = base + (ACROSS ? k0 * ld : k0) * int64_t(sizeof(Bits));
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int slot = i * NT + tid, row = row_of(slot), c = chunk_of(slot);
            reg[i].zero();
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const bool there = ACROSS ? k0 + row < kdim && c * 8 + j < dim : k0 + c * 8 + j < kdim;
                if (there) reg[i].set(j, reinterpret_cast<const Bits*>(at + off[i])[j]);
            }
        }
        look(k0, kept);
    }
    __device__ __forceinline__ void store(char* lds, const Regs& reg, const uint32_t (&kept)[CH]) const {
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int slot = i * NT + tid, row = row_of(slot), c = chunk_of(slot);
            int4 v[PL];
            reg[i].planes(v);
            if (looks && !kept[i]) {
#pragma unroll
                for (int p = 0; p < PL; ++p) v[p] = int4{0, 0, 0, 0};
            }
#pragma unroll
            for (int p = 0; p < PL; ++p)
                *reinterpret_cast<int4*>(lds + p * kPlane + row * (CPR * 16) + (c ^ swizzle(row)) * 16) = v[p];
        }
    }
    // Fragment of rows `first` .. first + 31 of D's side, of the 16 of the contraction from 16 t on: lane r + 32 q has
    // row r and 8 q .. 8 q + 7 of them.
    static __device__ __forceinline__ int4 fragment(const char* lds, int first, int t, int lane) {
        if constexpr (!ACROSS) {
            const int row = first + (lane & 31), c = 2 * t + (lane >> 5);
            return *reinterpret_cast<const int4*>(lds + row * (CPR * 16) + (c ^ swizzle(lane & 31)) * 16);
        } else {
            // 16 lanes bring 4 rows of 16 values; lane i of them is given value i of each row
            const int k = 16 * t + 8 * (lane >> 5) + ((lane & 15) >> 2);
            const int c = first / 8 + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
            const char* at = lds + k * (CPR * 16) + (c ^ swizzle(k)) * 16 + (lane & 1) * 8;
            // (four rows on the swizzle is the same)
            const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LocalTr)(at));
            const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LocalTr)(at + 4 * (CPR * 16)));
            return __builtin_bit_cast(int4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        }
    }
};

// What the products' kernels share: the first `whole` tiles are one workgroup each; of the others [splits] ranges of
// the contraction are one each, and where there are several their fragments go to part, which k_tile_join adds up.
// Where the epilogue says so (kTwice) the contraction is gone through once more, with a's values `again` elements further on.
struct Product {
    Operand a, b;
    int64_t rows, cols, kdim, again;
    uint32_t tm, tn, whole;
    int splits;
    float* part;
};

template <class T> using Acc = v16f[T::FM][T::FN];

// Where a lane's results lie in the tile: element e of fragment (i, j) of its wavefront.
template <class T> struct Place {
    int wm, wn, r, q;
    __device__ __forceinline__ explicit Place(int tid) {
        const int wave = tid >> 6;
        wm = wave / T::WN;
        wn = wave % T::WN;
        r = tid & 31;
        q = (tid >> 5) & 1;
    }
    // the row of the tile is first() + at(i, e), the latter known to the compiler
    __device__ __forceinline__ int first() const { return wm * T::FM * 32 + q * 4; }
    static __device__ constexpr int at(int i, int e) { return i * 32 + (e >> 2) * 8 + (e & 3); }
    __device__ __forceinline__ int col(int j) const { return (wn * T::FN + j) * 32 + r; }
};

// Workgroups are dealt to the XCDs in turn: each XCD takes a contiguous run of the items, whose tiles share rows and
// columns in its L2; tiles in bands of 4 along the rows, column by column.
__device__ __forceinline__ void tile_at(uint32_t item, uint32_t tm, uint32_t tn, uint32_t& im, uint32_t& in) {
    const uint32_t band = item / (4 * tn), at = item - band * 4 * tn, height = min(4u, tm - band * 4);
    im = band * 4 + at % height;
    in = at / height;
}
__device__ __forceinline__ uint32_t xcd_item(uint32_t block, uint32_t items) {
    const uint32_t x = block & 7, per = items >> 3, more = items & 7;
    return x * per + min(x, more) + (block >> 3);
}

// Wait until all but N of this wavefront's loads to LDS have arrived, and its reads of LDS, then for the other wavefronts.
template <int N> __device__ __forceinline__ void arrive() {
    static_assert(N < 64, "vmcnt has six bits");
    __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 0x0070);  // vmcnt(N) lgkmcnt(0)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

template <class S, class T> constexpr int tile_lds() { return 2 * Units<S>::planes * (T::BM + T::BN) * Units<S>::bk * 2; }

// Epi: static void run(const Args&, Acc<T>&, im, in, char* lds) of the tile (im, in).
template <class S, class T, bool ATR, bool BTR, bool DIRECT, class Epi>
__global__ __launch_bounds__(T::NT) void k_tile(Product g, typename Epi::Args ea) {
    constexpr int BK = DIRECT && T::DEEP ? 32 : Units<S>::bk, PL = Units<S>::planes;
    using SA = Side<S, ATR, T::BM, T::NT, DIRECT, BK>;
    using SB = Side<S, BTR, T::BN, T::NT, DIRECT, BK>;
    constexpr int kA = PL * SA::kPlane, kStage = kA + PL * SB::kPlane;
    __shared__ __attribute__((aligned(16))) char lds[tile_lds<S, T>()];
    const int tid = threadIdx.x, lane = tid & 63;
    const Place<T> place(tid);
    const uint32_t rest = g.tm * g.tn - g.whole;
    uint32_t item, split = 0, im, in;
    int splits = 1;
    if (blockIdx.x < g.whole) {
        item = xcd_item(blockIdx.x, g.whole);
    } else {
        item = xcd_item(blockIdx.x - g.whole, rest * g.splits);
        split = item / rest;
        item += g.whole - split * rest;
        splits = g.splits;
    }
    tile_at(item, g.tm, g.tn, im, in);
    SA a;
    SB b;
    a.init(g.a, int64_t(im) * T::BM, g.rows, tid);
    b.init(g.b, int64_t(in) * T::BN, g.cols, tid);
    constexpr bool kTwice = Epi::template kTwice<S>;
    const int64_t turn = (g.kdim + BK - 1) / BK * BK, steps = turn / BK * (kTwice ? 2 : 1);
    const int64_t k0 = steps * split / splits * BK, k1 = steps * (split + 1) / splits * BK;

    Acc<T> acc;
    auto clear = [](Acc<T>& v) {
#pragma unroll
        for (int i = 0; i < T::FM; ++i)
#pragma unroll
            for (int j = 0; j < T::FN; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) v[i][j][e] = 0.0f;
    };
    clear(acc);
    // A sum over thousands of products in one go loses what its own size is to each of them, and the units round towards zero: every
    // kFlush of the contraction it is added to another set of registers and begun anew.  For scores, whose differences count, where
    // there are registers (not in 16-bit tiles of 256 x 256): of 2048 x 8192 float32 pairs of 16640 values log_sum is 4.8e-6 off without and
    // 3.4e-7 with it.  For gradients of float32 rows where there are (not in tiles of 256 x 128; sums of 100000 terms of one sign 2.8e-6 off
    // without and 1.3e-7 with it); those of 16-bit rows are rounded to 2^-11 or less.
    constexpr bool kTwo = !Units<S>::whole && T::FM * T::FN <= 4 && (!BTR || (PL > 1 && T::FM * T::FN <= 2));
    constexpr int kFlush = 512;
    Acc<T> total;
    if constexpr (kTwo) clear(total);
    auto flush = [&] {
#pragma unroll
        for (int i = 0; i < T::FM; ++i)
#pragma unroll
            for (int j = 0; j < T::FN; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) total[i][j][e] += acc[i][j][e];
        clear(acc);
    };

    if constexpr (DIRECT) {
        constexpr int kStages = T::DEEP ? 4 : 2, L = SA::CH + SB::CH;  // L: a wavefront's loads for a stage
        const int n = int((k1 - k0 + BK - 1) / BK);
        int4 fa[2][T::FM], fb[2][T::FN];
        auto stage = [&](int s) { return lds + s % kStages * kStage; };
        auto fill = [&](int s) {
            const int64_t k = k0 + int64_t(s) * BK;
            const bool again = kTwice && k >= turn;
            a.fill(again ? k - turn : k, stage(s), again ? g.again : 0);
            b.fill(again ? k - turn : k, stage(s) + kA, 0);
        };
        auto read = [&](int s, int t) {
            const char *sa = stage(s), *sb = sa + kA;
#pragma unroll
            for (int i = 0; i < T::FM; ++i) fa[t % 2][i] = SA::fragment(sa, (place.wm * T::FM + i) * 32, t, lane);
#pragma unroll
            for (int j = 0; j < T::FN; ++j) fb[t % 2][j] = SB::fragment(sb, (place.wn * T::FN + j) * 32, t, lane);
            __builtin_amdgcn_sched_barrier(0);
        };
        auto multiply = [&](int t) {
#pragma unroll
            for (int i = 0; i < T::FM; ++i)
#pragma unroll
                for (int j = 0; j < T::FN; ++j) acc[i][j] = Units<S>::mfma(fa[t % 2][i], fb[t % 2][j], acc[i][j]);
            __builtin_amdgcn_sched_barrier(0);
        };
        if constexpr (!T::DEEP) {
            // one stage is multiplied while the other is filled
            if (n > 0) fill(0);
#pragma unroll 1
            for (int s = 0; s < n; ++s) {
                if (kTwo && s % (kFlush / BK) == 0) flush();
                arrive<0>();
                read(s, 0);
                if (s + 1 < n) fill(s + 1);
#pragma unroll
                for (int t = 0; t < BK / 16; ++t) {
                    if (t + 1 < BK / 16) read(s, t + 1);
                    multiply(t);
                }
            }
        } else {
            // While one stage is multiplied the next has arrived and two are on their way.  A step's first operands are
            // read behind the barrier of the step before, so that products are at hand while wavefronts wait for each
            // other.  (4096 x 12288 bfloat16 pairs of 4224 values: 384 us for the images' gradients, 429 in two stages;
            // tiles of 128 x 128 are slower that way, 516 and 441 for the scores' gradient: twice the barriers)
            if (n > 0) fill(0);
            if (n > 1) fill(1);
            if (n > 2) fill(2);
            if (n > 2)
                arrive<2 * L>();
            else
                arrive<0>();
            if (n > 0) read(0, 0);
#pragma unroll 1
            for (int s = 0; s < n; ++s) {
                if (kTwo && s % (kFlush / BK) == 0) flush();
                if (s + 3 < n) fill(s + 3);  // (where the stage before this one was)
                read(s, 1);
                multiply(0);
                if (s + 1 < n) {
                    if (s + 3 < n)
                        arrive<2 * L>();
                    else
                        arrive<0>();
                    read(s + 1, 0);
                }
                multiply(1);
            }
        }
    } else {
        // one step's products from a stage: the operands of a sixteenth are read while those of the one before are multiplied
        // (in planes there are no registers for that, and no need: six products for each operand)
        constexpr int D = PL == 1 ? 2 : 1;
        auto multiply = [&](const char* stage) {
            const char *sa = stage, *sb = stage + kA;
            int4 fa[D][PL][T::FM], fb[D][PL][T::FN];
            auto read = [&](int t) {
#pragma unroll
                for (int p = 0; p < PL; ++p) {
#pragma unroll
                    for (int i = 0; i < T::FM; ++i)
                        fa[t % D][p][i] = SA::fragment(sa + p * SA::kPlane, (place.wm * T::FM + i) * 32, t, lane);
#pragma unroll
                    for (int j = 0; j < T::FN; ++j)
                        fb[t % D][p][j] = SB::fragment(sb + p * SB::kPlane, (place.wn * T::FN + j) * 32, t, lane);
                }
            };
            if (D == 2) read(0);
#pragma unroll
            for (int t = 0; t < BK / 16; ++t) {
                if (t + D - 1 < BK / 16) read(t + D - 1);
                // the small products of pieces first
#pragma unroll
                for (int s = PL - 1; s >= 0; --s)
#pragma unroll
                    for (int p = 0; p <= s; ++p)
#pragma unroll
                        for (int i = 0; i < T::FM; ++i)
#pragma unroll
                            for (int j = 0; j < T::FN; ++j)
                                acc[i][j] = Units<S>::mfma(fa[t % D][p][i], fb[t % D][s - p][j], acc[i][j]);
            }
        };
        // two steps are on their way to registers while a third is multiplied
        typename SA::Regs ra[2];
        typename SB::Regs rb[2];
        uint32_t ka[2][SA::CH], kb[2][SB::CH];
        auto load = [&](int64_t k, int r) {
            a.load(k, ra[r], ka[r]);
            b.load(k, rb[r], kb[r]);
        };
        auto store = [&](int r) {
            a.store(lds + r * kStage, ra[r], ka[r]);
            b.store(lds + r * kStage + kA, rb[r], kb[r]);
        };
#pragma unroll 1
        for (int pass = 0; pass < (kTwice ? 2 : 1); ++pass) {
            const int64_t p0 = pass ? max(k0 - turn, int64_t(0)) : k0, p1 = pass ? k1 - turn : kTwice ? min(k1, turn) : k1;
            if (pass) {
                a.base += g.again * int64_t(sizeof(typename S::Bits));
                __syncthreads();
            }
            const int64_t kw = max(p0, min(p1, min(a.whole(), b.whole()))), last = kw - BK;
            if (p0 < kw) {
                load(p0, 0);
                load(min(p0 + BK, last), 1);
                store(0);
            }
#pragma unroll 1
            for (int64_t k = p0; k < kw; k += 2 * BK) {
                if (kTwo && k % kFlush < 2 * BK) flush();
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const int64_t at = k + r * BK;
                    if (at >= kw) break;
                    __syncthreads();
                    load(min(at + 2 * BK, last), r);  // (past the end: the last one again, not used)
                    multiply(lds + r * kStage);
                    if (at + BK < kw) store(r ^ 1);
                }
            }
            // what is left of the contraction
#pragma unroll 1
            for (int64_t k = kw; k < p1; k += BK) {
                a.load_some(k, ra[0], ka[0]);
                b.load_some(k, rb[0], kb[0]);
                __syncthreads();
                store(0);
                __syncthreads();
                multiply(lds);
            }
        }
    }
    if constexpr (kTwo) {
        flush();
#pragma unroll
        for (int i = 0; i < T::FM; ++i)
#pragma unroll
            for (int j = 0; j < T::FN; ++j) acc[i][j] = total[i][j];
    }
    if (splits > 1) {
        float* out = g.part + (int64_t(split) * rest + item - g.whole) * (T::BM * T::BN) + tid * 4;
#pragma unroll
        for (int i = 0; i < T::FM; ++i)
#pragma unroll
            for (int j = 0; j < T::FN; ++j)
#pragma unroll
                for (int e = 0; e < 16; e += 4)
                    *reinterpret_cast<float4*>(out + ((i * T::FN + j) * 4 + e / 4) * (T::NT * 4)) =
                        float4{acc[i][j][e], acc[i][j][e + 1], acc[i][j][e + 2], acc[i][j][e + 3]};
        return;
    }
    __syncthreads();
    Epi::template run<S, T>(ea, acc, im, in, lds);
}

template <class S> __device__ __forceinline__ float plus(float a, float b) {
    return Units<S>::whole ? __uint_as_float(__float_as_uint(a) + __float_as_uint(b)) : a + b;
}

// The ranges' fragments added up, then the epilogue.
template <class S, class T, class Epi>
__global__ __launch_bounds__(T::NT) void k_tile_join(Product g, typename Epi::Args ea) {
    __shared__ __attribute__((aligned(16))) char lds[tile_lds<S, T>()];
    const uint32_t item = xcd_item(blockIdx.x, gridDim.x);
    uint32_t im, in;
    tile_at(g.whole + item, g.tm, g.tn, im, in);
    Acc<T> acc;
#pragma unroll
    for (int i = 0; i < T::FM; ++i)
#pragma unroll
        for (int j = 0; j < T::FN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;
    constexpr int kUnroll = T::FM * T::FN <= 2 ? 4 : 1;  // (ranges on their way; the others have no registers)
#pragma unroll kUnroll
    for (int s = 0; s < g.splits; ++s) {
        const float* p = g.part + (int64_t(s) * gridDim.x + item) * (T::BM * T::BN) + threadIdx.x * 4;
#pragma unroll
        for (int i = 0; i < T::FM; ++i) {
#pragma unroll
            for (int j = 0; j < T::FN; ++j)
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    const float4 v = *reinterpret_cast<const float4*>(p + ((i * T::FN + j) * 4 + e / 4) * (T::NT * 4));
                    acc[i][j][e] = plus<S>(acc[i][j][e], v.x);
                    acc[i][j][e + 1] = plus<S>(acc[i][j][e + 1], v.y);
                    acc[i][j][e + 2] = plus<S>(acc[i][j][e + 2], v.z);
                    acc[i][j][e + 3] = plus<S>(acc[i][j][e + 3], v.w);
                }
            if (kUnroll == 1 && i % 2) __builtin_amdgcn_sched_barrier(0);
        }
    }
    Epi::template run<S, T>(ea, acc, im, in, lds);
}

// A row of fragments of a wavefront through its own part of LDS: use(row in the tile, first column, four neighbouring values)
// for each four of its 32 x 32 FN values, 8 FN lanes a row.  (The workgroup is done with LDS before the first.)
template <class T> struct Rows4 {
    static constexpr int kStride = T::FN * 32 + 4, kLanes = T::FN * 8, kBytes = 32 * kStride * 4;  // bytes of a wavefront
    template <class Use> static __device__ __forceinline__ void run(v16f (&acc)[T::FN], int i, char* lds, Use use) {
        const int tid = threadIdx.x, lane = tid & 63;
        const Place<T> place(tid);
        float* mine = reinterpret_cast<float*>(lds + (tid >> 6) * kBytes);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int j = 0; j < T::FN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) mine[((e >> 2) * 8 + place.q * 4 + (e & 3)) * kStride + j * 32 + place.r] = acc[j][e];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int row = 0; row < 32; row += 64 / kLanes) {
            const int at = row + lane / kLanes, c = lane % kLanes * 4;
            const float4 v = *reinterpret_cast<const float4*>(mine + at * kStride + c);
            use((place.wm * T::FM + i) * 32 + at, place.wn * T::FN * 32 + c, v);
        }
        __builtin_amdgcn_sched_barrier(0);  // (rows of fragments one after the other: registers)
    }
};

template <class S> struct Shapes {
    using Small = TileShape<64, 64, 2, 2>;
    using Middle = TileShape<128, 128, 2, 4>;
    using Large = TileShape<256, 256, 2, 4, true>;  // (straight to LDS only: there are no registers for what is on its way)
};
template <> struct Shapes<I8x2> {
    using Small = TileShape<64, 64, 2, 2>;
    using Middle = TileShape<128, 128, 2, 4>;
    using Large = TileShape<256, 256, 2, 4>;  // (4096 x 8192 x 16640: 470 to 490 us, in four stages 505)
};
template <> struct Shapes<F32> {  // (three planes of 256 x 128 are 144 KB in two stages)
    using Small = TileShape<64, 64, 2, 2>;
    using Middle = TileShape<128, 128, 2, 4>;
    using Large = TileShape<256, 128, 4, 2>;
};

// Whether an operand's chunks of eight 16-bit values can go straight to LDS.
template <bool ACROSS> bool direct(const Operand& o) {
    return reinterpret_cast<uintptr_t>(o.p) % 16 == 0 && o.ld % 8 == 0 && (ACROSS || o.kdim % 8 == 0);
}

template <class S, class T, bool ATR, bool BTR, bool DIRECT, class Epi>
hipError_t product_of(Product g, const typename Epi::Args& ea, hipStream_t s) {
    g.tm = uint32_t((g.rows + T::BM - 1) / T::BM);
    g.tn = uint32_t((g.cols + T::BN - 1) / T::BN);
    if (int64_t(g.tm) * g.tn > kMaxTiles) return hipErrorInvalidValue;
    const uint32_t tiles = g.tm * g.tn, rest = tiles > g.whole ? tiles - g.whole : 0;
    g.whole = tiles - rest;
    k_tile<S, T, ATR, BTR, DIRECT, Epi><<<dim3(g.whole + rest * g.splits), T::NT, 0, s>>>(g, ea);
    if (hipError_t e = hipGetLastError()) return e;
    if (rest && g.splits > 1) k_tile_join<S, T, Epi><<<dim3(rest), T::NT, 0, s>>>(g, ea);
    return hipGetLastError();
}
template <class S, bool ATR, bool BTR, class Epi>
hipError_t product(const Product& g, const TilePlan& t, const typename Epi::Args& ea, hipStream_t s) {
    using Small = typename Shapes<S>::Small;
    using Middle = typename Shapes<S>::Middle;
    using Large = typename Shapes<S>::Large;
    if constexpr (Units<S>::planes == 1) {
        if (t.direct && direct<ATR>(g.a) && direct<BTR>(g.b)) {
            if (t.tile == 0) return product_of<S, Small, ATR, BTR, true, Epi>(g, ea, s);
            if (t.tile == 1) return product_of<S, Middle, ATR, BTR, true, Epi>(g, ea, s);
            return product_of<S, Large, ATR, BTR, true, Epi>(g, ea, s);
        }
    } else if (t.tile == 2) {
        return product_of<S, Large, ATR, BTR, false, Epi>(g, ea, s);
    }
    if constexpr (!Units<S>::whole) {  // (codes are rows of whole chunks)
        if (t.tile == 0) return product_of<S, Small, ATR, BTR, false, Epi>(g, ea, s);
        if (t.tile == 1) return product_of<S, Middle, ATR, BTR, false, Epi>(g, ea, s);
    }
    return hipErrorInvalidValue;
}

}  // namespace tp
