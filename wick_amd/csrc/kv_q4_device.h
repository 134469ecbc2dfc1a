// The layout of a KV cache held in 4 bits, for the kernels that touch one.
//
// A cache of max_seq rows of n_kv_heads heads is two planes: the quants, [n_kv_heads][max_seq][head_dim / 8] words of 8 consecutive
// values, and behind them the scales, [n_kv_heads][max_seq][head_dim / 32] f16, one to a block of 32 values; a value stands for
// (nibble - 8) * scale.  A head's rows lie one behind the other, so that a workgroup, which attends over one head, reads whole
// cache lines of its own head alone and evicts rows of each head on their own.  Value 2 i of a word is nibble i of its lower half and
// value 2 i + 1 nibble i of the upper: (w >> 4 i) & 0x000f000f is a pair of neighbours, which two more instructions turn into halves.
#pragma once

#include "wick_rocm_device.h"

namespace wick_rocm {

// A cache's planes from the buffer that holds both.
struct Q4Cache {
    uint32_t* quants;
    uint16_t* scales;
};
__device__ __forceinline__ Q4Cache q4_planes(void* cache, uint32_t max_seq, uint32_t n_kv_heads, uint32_t head_dim) {
    uint8_t* const p = static_cast<uint8_t*>(cache);
    return {reinterpret_cast<uint32_t*>(p), reinterpret_cast<uint16_t*>(p + (size_t)n_kv_heads * max_seq * (head_dim / 2))};
}

__device__ __forceinline__ float q4_value(uint32_t w, uint32_t i, float scale) {  // value i of a word: exact
    return (float)((int)(w >> (4u * (i >> 1) + 16u * (i & 1u)) & 15u) - 8) * scale;
}

}  // namespace wick_rocm
