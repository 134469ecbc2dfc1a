// The KV cache held in 4 bits (its layout: kv_q4_device.h): rows appended and read back, eviction of the rows that have gathered
// the least attention weight.
#include <type_traits>

#include "kv_q4_device.h"
#include "wick_rocm_internal.h"

namespace wick_rocm {

namespace {

constexpr float kQ4Largest = 65504.0f;  // of a value that a block can hold: eight times its scale is an f16, whatever product takes it

// ---- append, read back ---------------------------------------------------------------------
// GGUF's Q4_0 rule: a block's scale is its value of largest magnitude over -8 (the positive one of two), so that this value is held as it is up to
// the scale's rounding to f16; the quants come from the unrounded scale: n = min(15, trunc(x * (1 / d) + 8.5)), each step one f32
// operation.  A block without a scale holds zeros (d rounds to 0), or NaN where a value is none or larger than an f16 holds.
// Four lanes a block, eight values each.  Bound by memory: 2002 tokens of 8 heads of 64 (10.5 MB) 4.0 us, 3.5 us to read one cache's rows back (5.2 MB).
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
struct Q4ReadArgs {
    void* cache;
    float* out;
    uint32_t stride, row, n, max_seq, n_kv_heads, head_dim;
};
__global__ __launch_bounds__(256) void kv_q4_read_kernel(Q4ReadArgs a) {
    const uint32_t words = a.head_dim / 8u;
    const uint64_t i = (uint64_t)blockIdx.x * 256u + threadIdx.x;
    if (i >= (uint64_t)a.n_kv_heads * a.n * words) return;
    const uint32_t w = (uint32_t)(i % words), j = (uint32_t)(i / words % a.n), c = (uint32_t)(i / words / a.n);
    const Q4Cache cache = q4_planes(a.cache, a.max_seq, a.n_kv_heads, a.head_dim);
    const size_t from = (size_t)c * a.max_seq + a.row + j;
    const uint32_t q = cache.quants[from * words + w];
    const float d = f16_bits_to_f32(cache.scales[from * (words / 4u) + w / 4u]);
    float* const to = a.out + (size_t)j * a.stride + (size_t)c * a.head_dim + 8u * w;
#pragma unroll
    for (int e = 0; e < 8; e += 4)
        *reinterpret_cast<float4*>(to + e) = make_float4(q4_value(q, e, d), q4_value(q, e + 1, d), q4_value(q, e + 2, d), q4_value(q, e + 3, d));
}

// ---- eviction -------------------------------------------------------------------------------
constexpr uint32_t kStateLine = 32;
struct SelectRecord {  // what a part of a head knows
    uint32_t prefix, left, smaller_before;  // bits found, keys that share them and leave, keys of the parts in front that are smaller than those
};
struct Q4EvictArgs {
    void* cache[2];
    float* weights;
    uint32_t* kept;   // [n_kv_heads][seq_len - n_drop]
    uint32_t* hists;    // of more than kSelectLargest rows: [2][n_kv_heads][parts][kBins]
    SelectRecord* records;  // [n_kv_heads][parts]
    uint32_t* state;    // [2 n_kv_heads]: segments taken, and a line behind it which of `segments` are in registers
    uint32_t segments;  // of rows that stay
    uint32_t seq_len, n_keep, n_recent, n_drop, max_seq, n_kv_heads, head_dim;
};

// A weight as an unsigned number of the same order: NaN least, the zeros alike.
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) return 0u;
    const uint32_t b = __float_as_uint(w + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// Sum over a wave's lanes up to this one.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t moved_or_zero(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
    v += moved_or_zero<0x111, 0xf>(v), v += moved_or_zero<0x112, 0xf>(v), v += moved_or_zero<0x114, 0xf>(v), v += moved_or_zero<0x118, 0xf>(v);  // in rows of 16 lanes
    v += moved_or_zero<0x142, 0xa>(v);  // the last of a row to the next: rows 1 and 3,
    v += moved_or_zero<0x143, 0xc>(v);  // and that of the first half to the second
    return v;
}

// Sum over the workgroup's threads in front of this one, and over all of them.  `slots`: one per wave, of this call alone.
constexpr uint32_t kEvictThreads = 1024, kEvictWaves = kEvictThreads / 64;
__device__ __forceinline__ uint32_t sum_before(uint32_t v, uint32_t* slots, uint32_t& total) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, sum = wave_scan(v);
    if (lane == 63u) slots[wave] = sum;
    __syncthreads();
    const uint32_t sums = wave_scan(lane < kEvictWaves ? slots[lane] : 0u);
    total = (uint32_t)__builtin_amdgcn_readlane((int)sums, 63);
    const uint32_t w = (uint32_t)__builtin_amdgcn_readfirstlane((int)wave);
    return sum - v + (w > 0 ? (uint32_t)__builtin_amdgcn_readlane((int)sums, (int)w - 1) : 0u);
}

// The rows of one KV head that stay, in order.  Of the candidates' keys the n_drop-th smallest is found 11, 11 and 10 bits at a time from the highest, by a
// histogram of those bits among the keys that share the bits found so far (11 bits are the exponent and two bits behind it: weights spread over
// many bins, so that a wave's additions seldom meet).  Of those that have just this key the lower rows leave, as many as are still to go.  A wave's 64
// consecutive rows are one vote: a row's place is the rows that stay in the votes before, which are added up over the workgroup, and those in front of it in its own.
// Up to 16384 rows: one workgroup a head, which reads them once; bound by the latency of some 15 barriers and as many trips to LDS, and with more rows by
// its CU's instructions (8 heads of 3000 rows 6.5 us, 8000 10.4, 16000 14.4; of 32768, 28).
// More: the head in parts of a workgroup each, a launch to each digit and one to place the rows, every one of which begins with adding up the parts'
// histograms of the launch before (32768 rows of 8 heads 3.7 + 5.3 + 5.5 + 6.3 us, 8000 rows 3.4 + 4.9 + 5.1 + 5.9: each bound by the same latencies).
constexpr uint32_t kPartRows = 4, kPartChunk = kPartRows * kEvictThreads;  // rows of a thread and of a part's workgroup at a time
constexpr uint32_t kBins = 2048, kMaxParts = 32, kSelectLargest = 16 * kEvictThreads;

__host__ __device__ inline uint32_t select_parts(uint32_t seq_len) {
    const uint32_t chunks = (seq_len + kPartChunk - 1u) / kPartChunk;
    return chunks < kMaxParts ? chunks : kMaxParts;
}

constexpr uint32_t digit_shift(int digit) { return digit == 0 ? 21u : digit == 1 ? 10u : 0u; }

template <uint32_t ROWS>
struct SelectShared {
    uint32_t hist[kBins + 64], slots[3][kEvictWaves], votes[2][ROWS * kEvictWaves], found[2];
};

template <uint32_t ROWS>
struct SelectKeys {
    uint32_t k[ROWS], candidates;  // bit i: row i of this thread may leave
    // (a read behind the last row gives 0, for nobody)
    __device__ __forceinline__ void load(const Q4EvictArgs& a, uint32_t c, uint32_t base) {
        const auto w = __builtin_amdgcn_make_buffer_rsrc(a.weights + (size_t)c * a.max_seq, 0, (int)(4u * a.seq_len), 0x27000);
        const uint32_t first = base + threadIdx.x - a.n_keep, n = a.seq_len - a.n_recent - a.n_keep;
#pragma unroll
        for (uint32_t i = 0; i < ROWS; i++) k[i] = __builtin_amdgcn_raw_buffer_load_b32(w, 4u * (base + i * kEvictThreads + threadIdx.x), 0, 0);
        candidates = 0;
#pragma unroll
        for (uint32_t i = 0; i < ROWS; i++) candidates |= (uint32_t)(first + i * kEvictThreads < n) << i, k[i] = weight_key(__uint_as_float(k[i]));
    }
    __device__ __forceinline__ void count(uint32_t* hist, int digit, uint32_t prefix) const {
        const uint32_t shift = digit_shift(digit), mask = digit == 2 ? 1023u : 2047u, above = digit == 1 ? 21u : 10u, lane = threadIdx.x & 63u;
#pragma unroll
        for (uint32_t i = 0; i < ROWS; i++) {
            // What does not count goes to a bin of its lane's own (no branch, no two at one address), and so do the lanes that meet the first one: it
            // adds for all of them (rows that are new have no weight at all).
            const bool counts = (candidates >> i & 1u) && (digit == 0 || k[i] >> above == prefix >> above);
            const uint32_t bin = counts ? k[i] >> shift & mask : kBins + lane, first = (uint32_t)__builtin_amdgcn_readfirstlane((int)bin);
            const uint64_t same = __ballot(bin == first);
            atomicAdd(&hist[bin == first && lane != 0 ? kBins + lane : bin], lane == 0 ? (uint32_t)__popcll(same) : 1u);
        }
    }
};

// The bin that the left-th key is in, this thread having the counts of bins 2 tid and 2 tid + 1; `left` becomes how many of that bin's leave.
__device__ __forceinline__ uint32_t find_bin(uint32_t* found, uint32_t h0, uint32_t h1, uint32_t* slots, uint32_t& left) {
    uint32_t all;
    const uint32_t before = sum_before(h0 + h1, slots, all);
    if (before < left && left <= before + h0 + h1) {  // one thread's (left is at least one and at most how many there are)
        const bool second = left > before + h0;
        found[0] = 2u * threadIdx.x + second, found[1] = before + (second ? h0 : 0u);
    }
    __syncthreads();
    const uint32_t bin = found[0];
    left -= found[1];
    __syncthreads();  // (found is written again)
    return bin;
}

// Bit i of every thread is row i's vote: how many have been given before this wave's, in lane (16 i + its number) / kEach (and `before` in all: those of earlier chunks).
template <uint32_t ROWS>
__device__ __forceinline__ uint32_t count_votes(uint32_t* votes, uint32_t bits, uint32_t& before) {
    constexpr uint32_t kEach = ROWS * kEvictWaves / 64u;  // votes of a lane
    static_assert(kEvictWaves == 16 && kEach >= 1 && kEach <= 16, "a row's votes are those of whole lanes");
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    uint32_t counts = 0;
#pragma unroll
    for (uint32_t i = 0; i < ROWS; i++) {
        const uint32_t n = (uint32_t)__popcll(__ballot(bits >> i & 1u));
        counts = lane == i ? n : counts;
    }
    if (lane < ROWS) votes[lane * kEvictWaves + wave] = counts;
    __syncthreads();
    uint32_t n[kEach], sum = 0, at = 0;
#pragma unroll
    for (uint32_t j = 0; j < kEach; j++) n[j] = votes[lane * kEach + j], sum += n[j];
    const uint32_t scan = wave_scan(sum);
    uint32_t front = scan - sum + before;
#pragma unroll
    for (uint32_t j = 0; j < kEach; j++) at = wave % kEach == j ? front : at, front += n[j];  // (of this wave's among a lane's)
    before += (uint32_t)__builtin_amdgcn_readlane((int)scan, 63);
    return at;
}

// Of a chunk, the rows whose keys are larger than `key` stay, and of those equal to it all but the first `left` of the head (equal_before: how many there are
// in front of the chunk; stay_before: rows that stay in front of it).
template <uint32_t ROWS>
__device__ __forceinline__ void place(SelectShared<ROWS>& s, const Q4EvictArgs& a, uint32_t c, const SelectKeys<ROWS>& keys, uint32_t base, uint32_t key, uint32_t left,
                                      uint32_t& equal_before, uint32_t& stay_before) {
    const uint32_t tid = threadIdx.x;
    const uint64_t in_front = (1ull << (tid & 63u)) - 1ull;
    uint32_t* const kept = a.kept + (size_t)c * (a.seq_len - a.n_drop);
    uint32_t equal = 0, stays = 0;
#pragma unroll
    for (uint32_t i = 0; i < ROWS; i++) {
        equal |= (keys.candidates >> i & (uint32_t)(keys.k[i] == key)) << i;
        stays |= (uint32_t)(base + i * kEvictThreads + tid < a.seq_len && (!(keys.candidates >> i & 1u) || keys.k[i] > key)) << i;
    }
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tid >> 6));
    uint32_t at = count_votes<ROWS>(s.votes[0], equal, equal_before);
    if (__ballot(equal != 0) != 0) {  // (few waves)
#pragma unroll
        for (uint32_t i = 0; i < ROWS; i++) {
            const uint32_t rank = (uint32_t)__builtin_amdgcn_readlane((int)at, (int)(4u * kEvictWaves / ROWS * i + wave * 4u / ROWS)) + (uint32_t)__popcll(__ballot(equal >> i & 1u) & in_front);
            stays |= (equal >> i & (uint32_t)(rank >= left)) << i;
        }
    }
    at = count_votes<ROWS>(s.votes[1], stays, stay_before);
#pragma unroll
    for (uint32_t i = 0; i < ROWS; i++) {
        const uint64_t vote = __ballot(stays >> i & 1u);
        const uint32_t to = (uint32_t)__builtin_amdgcn_readlane((int)at, (int)(4u * kEvictWaves / ROWS * i + wave * 4u / ROWS)) + (uint32_t)__popcll(vote & in_front);
        if (stays >> i & 1u) kept[to] = base + i * kEvictThreads + tid;
    }
}

__device__ __forceinline__ void clear_move_state(const Q4EvictArgs& a, uint32_t c) {  // (for the launch behind)
    const uint32_t n = 2u * (kStateLine + a.segments);
    for (uint32_t i = threadIdx.x; i < n; i += kEvictThreads) a.state[(size_t)c * n + i] = 0u;
}

template <uint32_t ROWS>
__global__ __launch_bounds__(kEvictThreads) void kv_q4_select_kernel(Q4EvictArgs a) {
    __shared__ SelectShared<ROWS> s;
    const uint32_t c = blockIdx.x, tid = threadIdx.x;
    clear_move_state(a, c);
    SelectKeys<ROWS> keys;
    keys.load(a, c, 0);
    uint32_t prefix = 0, left = a.n_drop;  // bits found so far; how many of the keys that share them leave
#pragma unroll
    for (int digit = 0; digit < 3; digit++) {
        s.hist[tid] = s.hist[tid + kEvictThreads] = 0;
        __syncthreads();
        keys.count(s.hist, digit, prefix);
        __syncthreads();
        prefix |= find_bin(s.found, s.hist[2u * tid], s.hist[2u * tid + 1u], s.slots[digit], left) << digit_shift(digit);
    }
    uint32_t equal_before = 0, stay_before = 0;
    place(s, a, c, keys, 0, prefix, left, equal_before, stay_before);
}

// STEP 0 .. 2: a part's histogram of that digit; 3: its rows placed.  What a part knows goes from launch to launch in a record of its own.
template <int STEP>
__global__ __launch_bounds__(kEvictThreads) void kv_q4_select_part_kernel(Q4EvictArgs a) {
    __shared__ SelectShared<kPartRows> s;
    const uint32_t parts = gridDim.x, part = blockIdx.x, c = blockIdx.y, tid = threadIdx.x;
    const uint32_t chunks = (a.seq_len + kPartChunk - 1u) / kPartChunk, chunk0 = (uint32_t)((uint64_t)chunks * part / parts), chunk_end = (uint32_t)((uint64_t)chunks * (part + 1u) / parts);
    const auto hist_of = [&](int step, uint32_t p) { return reinterpret_cast<uint2*>(a.hists + ((size_t)(step & 1) * a.n_kv_heads * parts + (size_t)c * parts + p) * kBins); };
    SelectRecord& record = a.records[(size_t)c * parts + part];
    SelectKeys<kPartRows> keys;
    keys.load(a, c, chunk0 * kPartChunk);
    uint32_t prefix = 0, left = a.n_drop, smaller_before = 0, equal_before = 0;
    if constexpr (STEP == 0) {
        if (part == 0) clear_move_state(a, c);
    } else {
        if constexpr (STEP > 1) prefix = record.prefix, left = record.left, smaller_before = record.smaller_before;
        uint2 sum = {0, 0}, before = {0, 0};  // over all parts, over those in front
        for (uint32_t p0 = 0; p0 < parts; p0 += 8u) {
            uint2 h[8];
#pragma unroll
            for (uint32_t i = 0; i < 8u; i++) h[i] = hist_of(STEP - 1, min(p0 + i, parts - 1u))[tid];
#pragma unroll
            for (uint32_t i = 0; i < 8u; i++) {
                const uint32_t p = p0 + i;
                if (p < parts) sum.x += h[i].x, sum.y += h[i].y;
                if (p < part) before.x += h[i].x, before.y += h[i].y;
            }
        }
        const uint32_t bin = find_bin(s.found, sum.x, sum.y, s.slots[0], left);
        prefix |= bin << digit_shift(STEP - 1);
        uint32_t smaller;
        (void)sum_before((2u * tid < bin ? before.x : 0u) + (2u * tid + 1u < bin ? before.y : 0u), s.slots[1], smaller);
        smaller_before += smaller;
        if constexpr (STEP == 3) (void)sum_before(2u * tid == bin ? before.x : 2u * tid + 1u == bin ? before.y : 0u, s.slots[2], equal_before);
    }
    if constexpr (STEP < 3) {
        if (STEP > 0 && tid == 0) record = {prefix, left, smaller_before};
        s.hist[tid] = s.hist[tid + kEvictThreads] = 0;
        __syncthreads();
        for (uint32_t i = chunk0;;) {
            keys.count(s.hist, STEP, prefix);
            if (++i >= chunk_end) break;
            keys.load(a, c, i * kPartChunk);
        }
        __syncthreads();
        hist_of(STEP, part)[tid] = make_uint2(s.hist[2u * tid], s.hist[2u * tid + 1u]);
    } else {
        uint32_t stay_before = chunk0 * kPartChunk - smaller_before - min(equal_before, left);
        for (uint32_t i = chunk0;;) {
            place(s, a, c, keys, i * kPartChunk, prefix, left, equal_before, stay_before);
            if (++i >= chunk_end) break;
            keys.load(a, c, i * kPartChunk);
        }
    }
}

// Moves the kept rows together in place, a segment of rows of one head's keys (with the weights) or values per workgroup.  A row moves down or stays: what a
// segment overwrites is read by itself and by segments in front of it.  So a workgroup reads its rows into registers, tells that it has, waits until the segments
// in front of it that can have rows in its place (n_drop rows at most) have told so too, and writes.  Every wait ends: segments are taken by a counter, so
// those in front of one that waits have been taken by workgroups that run already, and these tell before they wait for anybody.  (No order but that of these reads
// before those writes is asked of the memory: nothing that this launch writes is read in it.)
// Weights behind the last row that stays are cleared by segments that have nothing to read.
// Bound by memory latency: taking a segment, its rows' numbers, the rows, the word of the segments in front, one behind the other; 24576 rows of 8 heads of
// 64 values 13.4 us (12.2 when it was built, 18.1 with one workgroup for all rows of a fifth of a head's planes, one chunk of rows behind the other; of one head of 256 values 8.8
// and 50.6).
constexpr uint32_t kMoveThreads = 256, kMoveLeast = 256;  // threads; rows of a segment at least
template <int HD>
constexpr uint32_t kMoveRows = HD <= 64 ? 512 : 256;  // 16 KiB of quants and more: enough workgroups, and four and more loads of a thread on their way

template <int HD>
__global__ __launch_bounds__(kMoveThreads) void kv_q4_move_kernel(Q4EvictArgs a) {
    typedef uint32_t Two __attribute__((ext_vector_type(2)));
    typedef uint32_t Four __attribute__((ext_vector_type(4)));
    using Scales = typename std::conditional<HD == 32, uint16_t, typename std::conditional<HD == 64, uint32_t, typename std::conditional<HD == 128, Two, Four>::type>::type>::type;
    constexpr uint32_t R = kMoveRows<HD>, kPieces = HD / 32, kPer = R * kPieces / kMoveThreads, kRows = R / kMoveThreads;
    __shared__ uint32_t taken;
    const uint32_t tid = threadIdx.x;
    const uint32_t stream = blockIdx.x % (2u * a.n_kv_heads), c = stream >> 1;
    uint32_t* const state = a.state + (size_t)stream * (kStateLine + a.segments);
    if (tid == 0) taken = __hip_atomic_fetch_add(state, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    const uint32_t segment = taken;
    const bool keys = (stream & 1u) == 0;
    const uint32_t n = a.seq_len - a.n_drop, first = a.n_keep, row0 = first + segment * R;  // (rows in front of n_keep stay where they are)
    const bool reads = row0 < n;
    if (!reads && !keys) return;
    const size_t head = (size_t)c * a.max_seq;
    const Q4Cache cache = q4_planes(keys ? a.cache[0] : a.cache[1], a.max_seq, a.n_kv_heads, HD);
    const auto plane = [&](void* p, uint32_t row_bytes, uint32_t rows) { return __builtin_amdgcn_make_buffer_rsrc(p, 0, (int)(rows * row_bytes), 0x27000); };
    uint32_t* const quants = cache.quants + head * (HD / 8);
    uint16_t* const scales = cache.scales + head * (HD / 32);
    Four q[kPer];
    Scales d[kRows];
    uint32_t w[kRows];
    uint32_t* const told = state + kStateLine;
    if (reads) {
        // (numbers behind the last row read as 0: a row for nobody)
        const auto numbers = plane(a.kept + (size_t)c * n, 4, n), from = plane(quants, HD / 2, a.seq_len), scales_from = plane(scales, HD / 16, a.seq_len),
                   weights_from = plane(a.weights + head, 4, a.seq_len);
        uint32_t q_row[kPer], row[kRows];
#pragma unroll
        for (uint32_t i = 0; i < kPer; i++) q_row[i] = __builtin_amdgcn_raw_buffer_load_b32(numbers, 4u * (row0 + (i * kMoveThreads + tid) / kPieces), 0, 0);
#pragma unroll
        for (uint32_t i = 0; i < kRows; i++) row[i] = __builtin_amdgcn_raw_buffer_load_b32(numbers, 4u * (row0 + i * kMoveThreads + tid), 0, 0);
#pragma unroll
        for (uint32_t i = 0; i < kPer; i++) q[i] = __builtin_amdgcn_raw_buffer_load_b128(from, q_row[i] * (HD / 2) + (i * kMoveThreads + tid) % kPieces * 16u, 0, 0);
#pragma unroll
        for (uint32_t i = 0; i < kRows; i++) {
            if constexpr (HD == 32) d[i] = __builtin_amdgcn_raw_buffer_load_b16(scales_from, row[i] * 2u, 0, 0);
            else if constexpr (HD == 64) d[i] = __builtin_amdgcn_raw_buffer_load_b32(scales_from, row[i] * 4u, 0, 0);
            else if constexpr (HD == 128) d[i] = __builtin_amdgcn_raw_buffer_load_b64(scales_from, row[i] * 8u, 0, 0);
            else d[i] = __builtin_amdgcn_raw_buffer_load_b128(scales_from, row[i] * 16u, 0, 0);
            w[i] = keys ? __builtin_amdgcn_raw_buffer_load_b32(weights_from, row[i] * 4u, 0, 0) : 0u;
        }
#pragma unroll
        for (uint32_t i = 0; i < kPer; i++) asm volatile("" : "+v"(q[i]));  // (has arrived)
#pragma unroll
        for (uint32_t i = 0; i < kRows; i++) asm volatile("" : "+v"(d[i]), "+v"(w[i]));
        __syncthreads();
        if (tid == 0) __hip_atomic_store(told + segment, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    const uint32_t nearest = min(segment, a.segments), farthest = segment * R > a.n_drop ? (segment * R - a.n_drop) / R : 0u;
    for (uint32_t i = farthest + tid; i < nearest; i += kMoveThreads)
        while (__hip_atomic_load(told + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == 0u) __builtin_amdgcn_s_sleep(1);
    __syncthreads();
    if (reads) {
        const auto to = plane(quants, HD / 2, n), scales_to = plane(scales, HD / 16, n);  // (writes behind the last row are dropped)
#pragma unroll
        for (uint32_t i = 0; i < kPer; i++) __builtin_amdgcn_raw_buffer_store_b128(q[i], to, row0 * (HD / 2) + (i * kMoveThreads + tid) * 16u, 0, 0);
#pragma unroll
        for (uint32_t i = 0; i < kRows; i++) {
            const uint32_t row = row0 + i * kMoveThreads + tid;
            if constexpr (HD == 32) __builtin_amdgcn_raw_buffer_store_b16(d[i], scales_to, row * 2u, 0, 0);
            else if constexpr (HD == 64) __builtin_amdgcn_raw_buffer_store_b32(d[i], scales_to, row * 4u, 0, 0);
            else if constexpr (HD == 128) __builtin_amdgcn_raw_buffer_store_b64(d[i], scales_to, row * 8u, 0, 0);
            else __builtin_amdgcn_raw_buffer_store_b128(d[i], scales_to, row * 16u, 0, 0);
        }
    }
    if (keys) {
        const auto weights_to = plane(a.weights + head, 4, a.seq_len);
#pragma unroll
        for (uint32_t i = 0; i < kRows; i++) {
            const uint32_t row = row0 + i * kMoveThreads + tid;
            __builtin_amdgcn_raw_buffer_store_b32(row < n ? w[i] : 0u, weights_to, row * 4u, 0, 0);
        }
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
    const Q4ReadArgs a{const_cast<void*>(d_cache), d_out, out_stride, row, n, max_seq, n_kv_heads, head_dim};
    return launch_kernel(L, kFamOther, kv_q4_read_kernel, dim3((uint32_t)((threads + 255) / 256)), dim3(256), a);
}

// Histograms, records, state of the move.
static size_t evict_hist_words(uint32_t seq_len, uint32_t n_kv_heads) { return seq_len <= kSelectLargest ? 0 : 2 * (size_t)n_kv_heads * select_parts(seq_len) * kBins; }
static size_t evict_record_words(uint32_t seq_len, uint32_t n_kv_heads) {
    return seq_len <= kSelectLargest ? 0 : (size_t)n_kv_heads * select_parts(seq_len) * (sizeof(SelectRecord) / 4);
}
size_t kv_q4_evict_scratch_floats(uint32_t seq_len, uint32_t n_kv_heads) {
    return evict_hist_words(seq_len, n_kv_heads) + evict_record_words(seq_len, n_kv_heads) +
           2 * (size_t)n_kv_heads * (kStateLine + (seq_len + kMoveLeast - 1u) / kMoveLeast);
}

namespace {

template <int HD>
hipError_t launch_evict(Q4EvictArgs a, const Launch& L) {
    constexpr uint32_t R = kMoveRows<HD>;
    static_assert(R >= kMoveLeast, "the scratch is sized for it");
    a.segments = (a.seq_len - a.n_drop - a.n_keep + R - 1u) / R;
    hipError_t e = hipSuccess;
    if (a.seq_len <= kSelectLargest) {
        const auto select = a.seq_len <= 4u * kEvictThreads ? kv_q4_select_kernel<4> : a.seq_len <= 8u * kEvictThreads ? kv_q4_select_kernel<8> : kv_q4_select_kernel<16>;
        e = launch_kernel(L, kFamOther, select, dim3(a.n_kv_heads), dim3(kEvictThreads), a);
    } else {
        for (const auto step : {kv_q4_select_part_kernel<0>, kv_q4_select_part_kernel<1>, kv_q4_select_part_kernel<2>, kv_q4_select_part_kernel<3>})
            if (e == hipSuccess) e = launch_kernel(L, kFamOther, step, dim3(select_parts(a.seq_len), a.n_kv_heads), dim3(kEvictThreads), a);
    }
    if (e != hipSuccess) return e;
    return launch_kernel(L, kFamOther, kv_q4_move_kernel<HD>, dim3(2u * a.n_kv_heads * ((a.seq_len - a.n_keep + R - 1u) / R)), dim3(kMoveThreads), a);
}

}  // namespace

hipError_t launch_kv_q4_evict(void* d_k_cache, void* d_v_cache, float* d_weights, uint32_t* d_kept, float* d_scratch, uint32_t seq_len, uint32_t n_keep,
                              uint32_t n_recent, uint32_t n_drop, uint32_t max_seq, uint32_t n_kv_heads, uint32_t head_dim, const Launch& L) {
    uint32_t *const hists = reinterpret_cast<uint32_t*>(d_scratch), *const records = hists + evict_hist_words(seq_len, n_kv_heads),
             *const state = records + evict_record_words(seq_len, n_kv_heads);
    const Q4EvictArgs a{{d_k_cache, d_v_cache}, d_weights, d_kept, hists, reinterpret_cast<SelectRecord*>(records), state, 0, seq_len, n_keep, n_recent, n_drop, max_seq, n_kv_heads, head_dim};
    switch (head_dim) {
        case 32: return launch_evict<32>(a, L);
        case 64: return launch_evict<64>(a, L);
        case 128: return launch_evict<128>(a, L);
        default: return launch_evict<256>(a, L);
    }
}

}  // namespace wick_rocm
