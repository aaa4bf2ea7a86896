// Rows of bytes on their way from memory to LDS, for the tiled products of 8-bit codes (tp_scores.hip, tp_rows8.hip).
#pragma once

#include "tp_match.hh"

namespace tp {

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

// Wait until this wavefront's loads to LDS have arrived, and its reads of the stage that is filled next, then for the
// other wavefronts.
__device__ __forceinline__ void stage_ready() {
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

}  // namespace tp
