// The KV cache held in 4 bits (its layout: kv_q4_device.h): rows appended and read back, eviction of the rows that have gathered
// the least attention weight.
#include "kv_q4_device.h"
#include "wick_rocm_internal.h"

namespace wick_rocm {

namespace {

constexpr float kQ4Largest = 65504.0f;  // of a value that a block can hold: eight times its scale is an f16, whatever product takes it

// ---- append, read back ---------------------------------------------------------------------
// A block's scale is its value of largest magnitude over -8 (the positive one of two), so that this value is held as it is up to
// the scale's rounding to f16; the quants come from the unrounded scale: n = min(15, trunc(x * (1 / d) + 8.5)), each step one f32
// operation.  A block without a scale holds zeros (d rounds to 0), or NaN where a value is none or larger than an f16 holds.
// Four lanes a block, eight values each.
struct Q4AppendArgs {
    const float* src[2];  // keys, values
    void* cache[2];
    const uint32_t* d_row;
    uint32_t row, n, max_seq, n_kv_heads, head_dim, stride;
};

template <int CTRL>
__device__ __forceinline__ float quad_moved(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ float quad_max(float v) {
    v = fmaxf(v, quad_moved<0xB1>(v));
    return fmaxf(v, quad_moved<0x4E>(v));
}

__global__ __launch_bounds__(256) void kv_q4_append_kernel(Q4AppendArgs a) {
    const uint32_t words = a.head_dim / 8u;
    const uint64_t per_cache = (uint64_t)a.n_kv_heads * a.n * words, at = (uint64_t)blockIdx.x * 256u + threadIdx.x;
    if (at >= 2u * per_cache) return;  // (whole blocks: words is a multiple of four)
    const uint32_t which = at >= per_cache;
    const uint64_t i = which ? at - per_cache : at;
    const uint32_t w = (uint32_t)(i % words), j = (uint32_t)(i / words % a.n), c = (uint32_t)(i / words / a.n);
    const float* const src = (which ? a.src[1] : a.src[0]) + (size_t)j * a.stride + (size_t)c * a.head_dim + 8u * w;
    const float4 x0 = *reinterpret_cast<const float4*>(src), x1 = *reinterpret_cast<const float4*>(src + 4);
    const float x[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
    float high = x[0], low = -x[0];  // (low: of the negated values)
    bool fits = true;
#pragma unroll
    for (int e = 0; e < 8; e++) high = fmaxf(high, x[e]), low = fmaxf(low, -x[e]), fits = fits && fabsf(x[e]) <= kQ4Largest;
    high = quad_max(high), low = quad_max(low);
    fits = quad_max(fits ? 0.0f : 1.0f) == 0.0f;
    const float d = (high >= low ? high : -low) * -0.125f;
    const bool full = fits && (_Float16)d != (_Float16)0.0f;
    const _Float16 held = full ? (_Float16)d : fits ? (_Float16)0.0f : (_Float16)__builtin_nanf("");
    const float inverse = full ? __fdiv_rn(1.0f, d) : 0.0f;
    uint32_t q = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const int n = (int)__fadd_rn(full ? __fmul_rn(x[e], inverse) : 0.0f, 8.5f);
        q |= (uint32_t)(n < 15 ? n : 15) << (4 * (e >> 1) + 16 * (e & 1));
    }
    const uint64_t row = (uint64_t)(a.d_row ? *a.d_row : a.row) + j;
    if (row >= a.max_seq) return;  // the host checks a by-value row; rows past the cache behind a device-side one are dropped
    const Q4Cache cache = q4_planes(which ? a.cache[1] : a.cache[0], a.max_seq, a.n_kv_heads, a.head_dim);
    const size_t to = (size_t)c * a.max_seq + row;
    cache.quants[to * words + w] = q;
    if ((w & 3u) == 0) cache.scales[to * (words / 4u) + w / 4u] = __builtin_bit_cast(uint16_t, held);
}

// Rows [row, row + n) as floats, token-major: out[j * stride + c * head_dim + i].
__global__ __launch_bounds__(256) void kv_q4_read_kernel(const void* p, float* __restrict__ out, uint32_t stride, uint32_t row, uint32_t n, uint32_t max_seq,
                                                         uint32_t n_kv_heads, uint32_t head_dim) {
    const uint32_t words = head_dim / 8u;
    const uint64_t i = (uint64_t)blockIdx.x * 256u + threadIdx.x;
    if (i >= (uint64_t)n_kv_heads * n * words) return;
    const uint32_t w = (uint32_t)(i % words), j = (uint32_t)(i / words % n), c = (uint32_t)(i / words / n);
    const Q4Cache cache = q4_planes(const_cast<void*>(p), max_seq, n_kv_heads, head_dim);
    const size_t from = (size_t)c * max_seq + row + j;
    const uint32_t q = cache.quants[from * words + w];
    const float d = f16_bits_to_f32(cache.scales[from * (words / 4u) + w / 4u]);
    float* const to = out + (size_t)j * stride + (size_t)c * head_dim + 8u * w;
#pragma unroll
    for (int e = 0; e < 8; e += 4)
        *reinterpret_cast<float4*>(to + e) = make_float4(q4_value(q, e, d), q4_value(q, e + 1, d), q4_value(q, e + 2, d), q4_value(q, e + 3, d));
}

// ---- eviction -------------------------------------------------------------------------------
struct Q4EvictArgs {
    void* cache[2];
    float* weights;
    uint32_t* kept;  // [n_kv_heads][seq_len - n_drop]
    uint32_t seq_len, n_keep, n_recent, n_drop, max_seq, n_kv_heads, head_dim;
};

// A weight as an unsigned number of the same order: NaN least, the zeros alike.
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) return 0u;
    const uint32_t b = __float_as_uint(w + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// The rows of one KV head that stay, in order.  Of the candidates' keys the n_drop-th smallest is found a byte at a time, from
// the highest: a histogram of that byte among the keys that share the bytes found so far.  Every thread owns a run of rows; of those that
// have just this key the lower ones leave, as many as are still to go.
constexpr uint32_t kEvictThreads = 1024;
__global__ __launch_bounds__(kEvictThreads) void kv_q4_select_kernel(Q4EvictArgs a) {
    __shared__ uint32_t hist[256], scan[2][kEvictThreads / 64], found[2];
    const uint32_t c = blockIdx.x, tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
    const float* const w = a.weights + (size_t)c * a.max_seq;
    const uint32_t from = a.n_keep, to = a.seq_len - a.n_recent;
    uint32_t prefix = 0, left = a.n_drop;  // bytes found so far; how many of the keys that share them leave
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (tid < 256u) hist[tid] = 0;
        __syncthreads();
        for (uint32_t t = from + tid; t < to; t += kEvictThreads) {
            const uint32_t key = weight_key(w[t]);
            if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[key >> shift & 255u], 1u);
        }
        __syncthreads();
        if (tid == 0) {
            uint32_t b = 0, below = 0;
            while (below + hist[b] < left) below += hist[b++];  // (left is at most how many there are)
            found[0] = b, found[1] = below;
        }
        __syncthreads();
        prefix |= found[0] << shift, left -= found[1];
    }
    // exclusive sum over the workgroup's threads
    const auto before = [&](uint32_t v, int slot) {
        uint32_t sum = v;
        for (uint32_t off = 1; off < 64u; off <<= 1) {
            const uint32_t up = __shfl_up(sum, off, 64);
            if (lane >= off) sum += up;
        }
        if (lane == 63u) scan[slot][wave] = sum;
        __syncthreads();
        for (uint32_t i = 0; i < wave; i++) sum += scan[slot][i];
        return sum - v;
    };
    const uint32_t run = (a.seq_len + kEvictThreads - 1u) / kEvictThreads, r0 = min(tid * run, a.seq_len), r1 = min(r0 + run, a.seq_len);  // (at most 2^30)
    uint32_t equal = 0, less = 0;
    for (uint32_t t = max(r0, from); t < min(r1, to); t++) {
        const uint32_t key = weight_key(w[t]);
        equal += key == prefix, less += key < prefix;
    }
    uint32_t go = before(equal, 0);
    go = go < left ? left - go : 0u;  // of this thread's rows with just this key: the first `go`
    const uint32_t dropped = less + min(go, equal);
    uint32_t* kept = a.kept + (size_t)c * (a.seq_len - a.n_drop) + before(r1 - r0 - dropped, 1);
    for (uint32_t t = r0; t < r1; t++) {
        bool stays = t < from || t >= to;
        if (!stays) {
            const uint32_t key = weight_key(w[t]);
            if (key == prefix) stays = go == 0, go -= !stays;
            else stays = key > prefix;
        }
        if (stays) *kept++ = t;
    }
}

// Moves the kept rows of one plane of one head (T: a piece of a row) together in place.  A row moves down or stays, so that chunks of
// rows are moved in ascending order: nothing that a chunk overwrites is read behind it, and all of it has arrived in
// registers (the barrier) before the first piece is written.
template <typename T>
__device__ __forceinline__ void move_rows(T* base, uint32_t pieces, const uint32_t* kept, uint32_t n) {
    const uint64_t total = (uint64_t)n * pieces;
    for (uint64_t i0 = 0; i0 < total; i0 += kEvictThreads) {
        const uint64_t i = i0 + threadIdx.x;
        T v{};
        if (i < total) v = base[(size_t)kept[i / pieces] * pieces + i % pieces];
        asm volatile("s_waitcnt vmcnt(0)" : "+v"(v) : : "memory");
        __syncthreads();
        if (i < total) base[i] = v;
    }
}

__global__ __launch_bounds__(kEvictThreads) void kv_q4_move_kernel(Q4EvictArgs a) {
    const uint32_t c = blockIdx.x, n = a.seq_len - a.n_drop;
    const uint32_t* const kept = a.kept + (size_t)c * n;
    const size_t first = (size_t)c * a.max_seq;
    if (blockIdx.y == 4u) {
        move_rows(a.weights + first, 1u, kept, n);
        for (uint32_t t = n + threadIdx.x; t < a.seq_len; t += kEvictThreads) a.weights[first + t] = 0.0f;
        return;
    }
    const Q4Cache cache = q4_planes(blockIdx.y & 1u ? a.cache[1] : a.cache[0], a.max_seq, a.n_kv_heads, a.head_dim);
    if (blockIdx.y < 2u) move_rows(cache.quants + first * (a.head_dim / 8u), a.head_dim / 8u, kept, n);
    else move_rows(cache.scales + first * (a.head_dim / 32u), a.head_dim / 32u, kept, n);
}

}  // namespace

size_t kv_q4_bytes(uint32_t max_seq, uint32_t n_kv_heads, uint32_t head_dim) { return (size_t)n_kv_heads * max_seq * (head_dim / 2u + head_dim / 16u); }

hipError_t launch_kv_q4_append(const float* d_k, const float* d_v, uint32_t kv_stride, void* d_k_cache, void* d_v_cache, uint32_t row, const uint32_t* d_row,
                               uint32_t n, uint32_t max_seq, uint32_t n_kv_heads, uint32_t head_dim, const Launch& L) {
    if (n == 0) return hipSuccess;
    const Q4AppendArgs a{{d_k, d_v}, {d_k_cache, d_v_cache}, d_row, row, n, max_seq, n_kv_heads, head_dim, kv_stride};
    const uint64_t threads = 2 * (uint64_t)n_kv_heads * n * (head_dim / 8u);
    return launch_kernel(L, kFamOther, kv_q4_append_kernel, dim3((uint32_t)((threads + 255) / 256)), dim3(256), a);
}

hipError_t launch_kv_q4_read(const void* d_cache, float* d_out, uint32_t out_stride, uint32_t row, uint32_t n, uint32_t max_seq, uint32_t n_kv_heads,
                             uint32_t head_dim, const Launch& L) {
    if (n == 0) return hipSuccess;
    const uint64_t threads = (uint64_t)n_kv_heads * n * (head_dim / 8u);
    return launch_kernel(L, kFamOther, kv_q4_read_kernel, dim3((uint32_t)((threads + 255) / 256)), dim3(256), d_cache, d_out, out_stride, row, n, max_seq,
                         n_kv_heads, head_dim);
}

size_t kv_q4_evict_scratch_floats(uint32_t seq_len, uint32_t n_kv_heads) {
    (void)seq_len, (void)n_kv_heads;
    return 0;
}

hipError_t launch_kv_q4_evict(void* d_k_cache, void* d_v_cache, float* d_weights, uint32_t* d_kept, float* d_scratch, uint32_t seq_len, uint32_t n_keep,
                              uint32_t n_recent, uint32_t n_drop, uint32_t max_seq, uint32_t n_kv_heads, uint32_t head_dim, const Launch& L) {
    (void)d_scratch;
    const Q4EvictArgs a{{d_k_cache, d_v_cache}, d_weights, d_kept, seq_len, n_keep, n_recent, n_drop, max_seq, n_kv_heads, head_dim};
    hipError_t e = launch_kernel(L, kFamOther, kv_q4_select_kernel, dim3(n_kv_heads), dim3(kEvictThreads), a);
    if (e == hipSuccess) e = launch_kernel(L, kFamOther, kv_q4_move_kernel, dim3(n_kv_heads, 5), dim3(kEvictThreads), a);
    return e;
}

}  // namespace wick_rocm
