// The KV cache held in 4 bits (its layout: kv_q4_device.h): rows appended and read back, eviction of the rows that have gathered
// the least attention weight.
#include <type_traits>

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

// Sum over the workgroup's threads in front of this one, and over all of them.  `slots`: one per wave, of this call alone.
constexpr uint32_t kEvictThreads = 1024, kEvictWaves = kEvictThreads / 64;
__device__ __forceinline__ uint32_t sum_before(uint32_t v, uint32_t* slots, uint32_t& total) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    uint32_t sum = v;
#pragma unroll
    for (uint32_t off = 1; off < 64u; off <<= 1) {
        const uint32_t up = __shfl_up(sum, off, 64);
        if (lane >= off) sum += up;
    }
    if (lane == 63u) slots[wave] = sum;
    __syncthreads();
    uint32_t front = 0, all = 0;
#pragma unroll
    for (uint32_t i = 0; i < kEvictWaves; i++) {
        const uint32_t s = slots[i];
        front += i < wave ? s : 0u, all += s;
    }
    total = all;
    return front + sum - v;
}

// The rows of one KV head that stay, in order.  Of the candidates' keys the n_drop-th smallest is found 11, 11 and 10 bits at a time from the highest, by a
// histogram of those bits among the keys that share the bits found so far (11 bits are the exponent and two bits behind it: weights spread over
// many bins, so that a wave's additions seldom meet).  Of those that have just this key the lower rows leave, as many as are still to go.  A wave's 64
// consecutive rows are one vote: a row's place is the rows that stay in the votes before, which are added up over the workgroup, and those in front of it in its own.
// Up to 32768 rows are read once and stay in registers (28 us for 8 heads of 32768 rows; read anew for each step 38), longer caches are read anew for each step.
// Bound by one CU's instructions per head and, for few rows, by the latency of some 20 barriers and as many trips to LDS (3000 rows 7.3 us); 32768 rows
// took 76 us with bytes for digits, one lane walking the bins and a run of rows to each thread, which writes no whole lines.
// ROWS: of a thread at a time (3000 rows as 32 a thread: 24 us); LONG: there are more, in chunks.
template <uint32_t ROWS, bool LONG>
__global__ __launch_bounds__(kEvictThreads) void kv_q4_select_kernel(Q4EvictArgs a) {
    constexpr uint32_t kBins = 2048, kChunk = ROWS * kEvictThreads, kVotes = ROWS * kEvictWaves;
    static_assert(ROWS <= 32 && kVotes <= kEvictThreads, "a bit a row, a thread a vote");
    __shared__ uint32_t hist[kBins + 64], slots[8][kEvictWaves], votes[kVotes], found[2];
    const uint32_t c = blockIdx.x, tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
    const uint64_t in_front = (1ull << lane) - 1ull;
    // (a read behind the last row gives 0, for nobody)
    const auto w = __builtin_amdgcn_make_buffer_rsrc(a.weights + (size_t)c * a.max_seq, 0, (int)(4u * a.seq_len), 0x27000);
    const uint32_t from = a.n_keep, to = a.seq_len - a.n_recent;
    const uint32_t rows = LONG ? a.seq_len : 1u;  // (one chunk)
    uint32_t keys[ROWS], candidates;  // bit i: row i of this thread may leave
    const auto load = [&](uint32_t base) {
        candidates = 0;
#pragma unroll
        for (uint32_t i = 0; i < ROWS; i++) keys[i] = __builtin_amdgcn_raw_buffer_load_b32(w, 4u * (base + i * kEvictThreads + tid), 0, 0);
#pragma unroll
        for (uint32_t i = 0; i < ROWS; i++) {
            candidates |= (uint32_t)(base + i * kEvictThreads + tid - from < to - from) << i;
            keys[i] = weight_key(__uint_as_float(keys[i]));
        }
    };
    load(0);
    uint32_t prefix = 0, left = a.n_drop;  // bits found so far; how many of the keys that share them leave
#pragma unroll
    for (int digit = 0; digit < 3; digit++) {
        const uint32_t shift = digit == 0 ? 21u : digit == 1 ? 10u : 0u, mask = digit == 2 ? 1023u : 2047u, above = digit == 1 ? 21u : 10u;
        hist[tid] = hist[tid + kEvictThreads] = 0;
        __syncthreads();
        for (uint32_t base = 0; base < rows; base += kChunk) {
            if (LONG && (digit > 0 || base > 0)) load(base);
#pragma unroll
            for (uint32_t i = 0; i < ROWS; i++) {
                // What does not count goes to a bin of its lane's own (no branch, no two at one address), and so do the lanes that meet the first one: it
                // adds for all of them (rows that are new have no weight at all).
                const bool counts = (candidates >> i & 1u) && (digit == 0 || keys[i] >> above == prefix >> above);
                const uint32_t bin = counts ? keys[i] >> shift & mask : kBins + lane, first = (uint32_t)__builtin_amdgcn_readfirstlane((int)bin);
                const uint64_t same = __ballot(bin == first);
                atomicAdd(&hist[bin == first && lane != 0 ? kBins + lane : bin], lane == 0 ? (uint32_t)__popcll(same) : 1u);
            }
        }
        __syncthreads();
        const uint32_t h0 = hist[2u * tid], h1 = hist[2u * tid + 1u];
        uint32_t all;
        const uint32_t before = sum_before(h0 + h1, slots[digit], all);
        if (before < left && left <= before + h0 + h1) {  // one thread's (left is at least one and at most how many there are)
            const bool second = left > before + h0;
            found[0] = 2u * tid + second, found[1] = before + (second ? h0 : 0u);
        }
        __syncthreads();
        prefix |= found[0] << shift, left -= found[1];
        __syncthreads();  // (found and hist are written again)
    }
    // Bit i of every thread is row i's vote: how many have been given before each wave's, in lane i (and `before` in all: those of earlier chunks).
    const auto count_votes = [&](uint32_t bits, uint32_t* table, uint32_t* sums, uint32_t& before) {
        uint32_t counts = 0;
#pragma unroll
        for (uint32_t i = 0; i < ROWS; i++) {
            const uint32_t n = (uint32_t)__popcll(__ballot(bits >> i & 1u));
            counts = lane == i ? n : counts;
        }
        if (lane < ROWS) table[lane * kEvictWaves + wave] = counts;
        __syncthreads();
        uint32_t all;
        const uint32_t sum = sum_before(tid < kVotes ? table[tid] : 0u, sums, all) + before;
        if (tid < kVotes) table[tid] = sum;
        before += all;
        __syncthreads();
        const uint32_t at = lane < ROWS ? table[lane * kEvictWaves + wave] : 0u;
        __syncthreads();  // (the table is written again)
        return at;
    };
    uint32_t equal_before = 0, stay_before = 0;
    uint32_t* const kept = a.kept + (size_t)c * (a.seq_len - a.n_drop);
    for (uint32_t base = 0; base < rows; base += kChunk) {
        if (LONG) load(base);
        uint32_t equal = 0, stays = 0;
#pragma unroll
        for (uint32_t i = 0; i < ROWS; i++) {
            equal |= (candidates >> i & (uint32_t)(keys[i] == prefix)) << i;
            stays |= (uint32_t)(base + i * kEvictThreads + tid < a.seq_len && (!(candidates >> i & 1u) || keys[i] > prefix)) << i;
        }
        uint32_t at = count_votes(equal, votes, slots[3], equal_before);
        if (__ballot(equal != 0) != 0) {  // (few waves)
#pragma unroll
            for (uint32_t i = 0; i < ROWS; i++) {
                const uint32_t rank = (uint32_t)__builtin_amdgcn_readlane((int)at, (int)i) + (uint32_t)__popcll(__ballot(equal >> i & 1u) & in_front);
                stays |= (equal >> i & (uint32_t)(rank >= left)) << i;
            }
        }
        at = count_votes(stays, votes, slots[4], stay_before);
#pragma unroll
        for (uint32_t i = 0; i < ROWS; i++) {
            const uint64_t vote = __ballot(stays >> i & 1u);
            const uint32_t to = (uint32_t)__builtin_amdgcn_readlane((int)at, (int)i) + (uint32_t)__popcll(vote & in_front);
            if (stays >> i & 1u) kept[to] = base + i * kEvictThreads + tid;
        }
    }
}

// Moves the kept rows of one stream of a head together in place: C neighbouring pieces (of type T) of every row, rows being `stride`
// pieces.  A row moves down or stays, so chunks of rows are moved in ascending order: nothing that a chunk overwrites is read behind it,
// and all of the chunk itself has arrived in registers (the barrier) before its first piece is written.  The next chunk's pieces, which
// lie behind what this one overwrites, are on their way meanwhile, and its rows' numbers before that.  Bound by the latency of a
// workgroup's chunks, one behind the other, so a row's quants are several streams with a workgroup each: 24576 rows of 8 heads of 64
// values took 18.2 us, with whole rows 21.4.
template <typename T, uint32_t C, int PER>
__device__ __forceinline__ void move_rows(T* base, uint32_t stride, const uint32_t* kept, uint32_t first, uint32_t n) {
    constexpr uint32_t kChunk = kEvictThreads * PER / C;  // rows
    const uint32_t row = threadIdx.x / C, piece = threadIdx.x % C;
    uint32_t at[2][PER];
    T v[2][PER];
    const auto rows = [&](uint32_t i0, uint32_t (&r)[PER]) {
#pragma unroll
        for (int i = 0; i < PER; i++) r[i] = kept[min(i0 + i * (kEvictThreads / C) + row, n - 1u)];
    };
    const auto read = [&](const uint32_t (&r)[PER], T (&x)[PER]) {
#pragma unroll
        for (int i = 0; i < PER; i++) x[i] = base[(size_t)r[i] * stride + piece];
    };
    const auto write = [&](uint32_t i0, T (&x)[PER]) {
#pragma unroll
        for (int i = 0; i < PER; i++) asm volatile("" : "+v"(x[i]));  // (has arrived)
        __syncthreads();
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const uint32_t to = i0 + i * (kEvictThreads / C) + row;
            if (to < n) base[(size_t)to * stride + piece] = x[i];
        }
    };
    if (first >= n) return;
    rows(first, at[0]);
    read(at[0], v[0]);
    rows(first + kChunk, at[1]);
    for (uint32_t i0 = first; i0 < n; i0 += 2u * kChunk) {
        read(at[1], v[1]);  // (past the end: the last row, for nobody)
        rows(i0 + 2u * kChunk, at[0]);
        write(i0, v[0]);
        if (i0 + kChunk >= n) break;
        read(at[0], v[0]);
        rows(i0 + 3u * kChunk, at[1]);
        write(i0 + kChunk, v[1]);
    }
}

template <int HD>
constexpr uint32_t kMovePieces = HD <= 64 ? 1 : 2;  // of 16 bytes, of a row's quants, in a stream
template <int HD>
__global__ __launch_bounds__(kEvictThreads) void kv_q4_move_kernel(Q4EvictArgs a) {
    typedef uint32_t Two __attribute__((ext_vector_type(2)));
    typedef uint32_t Four __attribute__((ext_vector_type(4)));
    using Scales = typename std::conditional<HD == 32, uint16_t, typename std::conditional<HD == 64, uint32_t, typename std::conditional<HD == 128, Two, Four>::type>::type>::type;
    constexpr uint32_t C = kMovePieces<HD>, kPieces = HD / 32, kStreams = kPieces / C;
    const uint32_t c = blockIdx.x, n = a.seq_len - a.n_drop, first = a.n_keep;  // (rows in front of n_keep stay where they are)
    const uint32_t* const kept = a.kept + (size_t)c * n;
    const size_t head = (size_t)c * a.max_seq;
    const Q4Cache cache = q4_planes(blockIdx.y & 1u ? a.cache[1] : a.cache[0], a.max_seq, a.n_kv_heads, HD);
    if (blockIdx.y < 2u * kStreams) {
        move_rows<Four, C, 4>(reinterpret_cast<Four*>(cache.quants) + head * kPieces + blockIdx.y / 2u * C, kPieces, kept, first, n);
    } else if (blockIdx.y < 2u * kStreams + 2u) {
        move_rows<Scales, 1, 4>(reinterpret_cast<Scales*>(cache.scales) + head, 1u, kept, first, n);
    } else {
        move_rows<float, 1, 4>(a.weights + head, 1u, kept, first, n);
        __syncthreads();  // (the last chunk's reads)
        for (uint32_t t = n + threadIdx.x; t < a.seq_len; t += kEvictThreads) a.weights[head + t] = 0.0f;
    }
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
    const auto select = seq_len <= 4u * kEvictThreads ? kv_q4_select_kernel<4, false> : seq_len <= 32u * kEvictThreads ? kv_q4_select_kernel<32, false> : kv_q4_select_kernel<32, true>;
    const hipError_t e = launch_kernel(L, kFamOther, select, dim3(n_kv_heads), dim3(kEvictThreads), a);
    if (e != hipSuccess) return e;
    const auto move = [&](auto kernel, uint32_t streams) { return launch_kernel(L, kFamOther, kernel, dim3(n_kv_heads, 2u * streams + 3u), dim3(kEvictThreads), a); };
    switch (head_dim) {
        case 32: return move(kv_q4_move_kernel<32>, 1 / kMovePieces<32>);
        case 64: return move(kv_q4_move_kernel<64>, 2 / kMovePieces<64>);
        case 128: return move(kv_q4_move_kernel<128>, 4 / kMovePieces<128>);
        default: return move(kv_q4_move_kernel<256>, 8 / kMovePieces<256>);
    }
}

}  // namespace wick_rocm
