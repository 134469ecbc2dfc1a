// What the kernels on paged KV caches share.
#pragma once

#include "attention_device.h"

namespace wick_rocm {

// Pages that rows take.
__host__ __device__ inline uint32_t pages_of(uint64_t rows, uint32_t page_shift) { return (uint32_t)((rows + (1u << page_shift) - 1u) >> page_shift); }

}  // namespace wick_rocm
