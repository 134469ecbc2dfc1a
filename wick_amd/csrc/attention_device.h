// What the attention kernels on the f16 matrix cores share: f32 operands as two halves, reductions over a query's lane groups, and
// the exponential.
#pragma once

#include "wick_rocm_device.h"

namespace wick_rocm {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));

// hi = f16(x), lo = f16(x - hi) of four values x = y * SCALE (a power of two).  The product and the difference are exact, so that each half
// is one fused multiply-add that rounds to f16: two instructions a value (1.5 where nothing is scaled and pairs are converted together)
// instead of four and a half.
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));
template <int SCALE = 1>
__device__ __forceinline__ void split_f16(const v4f& y, h4& hi, h4& lo) {
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
        h2 h;
        if constexpr (SCALE == 1) h = __builtin_convertvector((v2f{y[i], y[i + 1]}), h2);
        else h[0] = (_Float16)(y[i] * (float)SCALE), h[1] = (_Float16)(y[i + 1] * (float)SCALE);
        asm("" : "+v"(h));
        hi[i] = h[0], hi[i + 1] = h[1];
        lo[i] = (_Float16)__builtin_fmaf(y[i], (float)SCALE, -(float)h[0]), lo[i + 1] = (_Float16)__builtin_fmaf(y[i + 1], (float)SCALE, -(float)h[1]);
    }
}

// Reductions over the four lane groups of a query (lanes l, l ^ 16, l ^ 32, l ^ 48) with gfx950's row / half swaps: swapping a
// register with a copy of itself leaves the two partners' values in the pair, so their maximum (or sum) needs no select
// and no trip through the LDS crossbar.  Every lane ends with the result.
__device__ __forceinline__ float groups_max(float v) {
    const uint32_t b = __float_as_uint(v);
    auto r = __builtin_amdgcn_permlane16_swap(b, b, false, false);
    v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    const uint32_t c = __float_as_uint(v);
    auto q = __builtin_amdgcn_permlane32_swap(c, c, false, false);
    return fmaxf(__uint_as_float(q[0]), __uint_as_float(q[1]));
}
__device__ __forceinline__ float groups_sum(float v) {
    const uint32_t b = __float_as_uint(v);
    auto r = __builtin_amdgcn_permlane16_swap(b, b, false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    const uint32_t c = __float_as_uint(v);
    auto q = __builtin_amdgcn_permlane32_swap(c, c, false, false);
    return __uint_as_float(q[0]) + __uint_as_float(q[1]);
}

// exp(x) for x <= 0 (-inf included) on the hardware's exp2 (v_exp_f32, about one ulp): two instructions where the polynomial of
// ggml_expf takes about thirty, and the softmax of a tile is nine of them per lane.  The weights differ from ggml_expf's in the
// last bit or two; the streaming softmax of this kernel differs from the reference's two-pass one at that level anyway.
__device__ __forceinline__ float exp_nonpos_hw(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896340736f); }

}  // namespace wick_rocm
