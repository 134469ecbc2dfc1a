// What the kernels on paged KV caches share.
#pragma once

#include "attention_device.h"

namespace wick_rocm {

// Pages that rows take.
__host__ __device__ inline uint32_t pages_of(uint64_t rows, uint32_t page_shift) { return (uint32_t)((rows + (1u << page_shift) - 1u) >> page_shift); }

// Sum over a wave's lanes up to this one, without LDS: inside rows of 16 lanes, then the last of a row to the next one, and of a half to the other.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t lane_moved_or_zero(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ uint32_t lanes_upto(uint32_t v) {
    v += lane_moved_or_zero<0x111, 0xf>(v), v += lane_moved_or_zero<0x112, 0xf>(v), v += lane_moved_or_zero<0x114, 0xf>(v), v += lane_moved_or_zero<0x118, 0xf>(v);
    v += lane_moved_or_zero<0x142, 0xa>(v), v += lane_moved_or_zero<0x143, 0xc>(v);
    return v;
}

}  // namespace wick_rocm
