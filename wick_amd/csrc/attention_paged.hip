// Attention of one new token of every sequence over KV caches in pages (wick_rocm_kv_pages), on the matrix cores.
//
// With G = n_heads / n_kv_heads, the G query heads of a KV head read the same keys and values: up to 16 of them are one operand of
// 16x16 matrix instructions, both products transposed (a wave walks 32 rows of the cache at a time, as two halves of 16):
//   S^T[row][head] = sum_d K[row][d] Q[head][d]        lane l is left with rows 4 (l / 16) + i of each half for head l % 16;
//   O^T[d][head]  += sum_row V[row][d] P[row][head]    whose operand P is, per lane, the weights as they are in its registers: a matrix
//                                                      instruction's K steps are in any order, so a lane just reads the values of those rows.
// Nothing goes through LDS on the way: keys are read 16 bytes a lane in the operand's own order, values as 16 (or fewer) bytes of each of the
// lane's rows, from which the operand of dimension e is picked lane by lane.
//   f16 pages: v_mfma_f32_16x16x32_f16; the cached values are exact operands, a query row (scaled by a power of two to below 2^15) and the softmax weights (times
//   2^15) are split into two halves: a product with one is off by at most 2^-22 of it.  Two products.  What is so far below the row's largest that halves would lose its bits
//   goes through f32 products instead: elements of the query (Query) and the weights of a tile (State).  (All of it in f32 products: 73 us for the 59.3 of 32 sequences
//   below, 108 for the 99.5 of one, 11.4 for 7.3 with 701 rows.)
//   f32 pages: v_mfma_f32_16x16x4_f32, f32 products as they are.
// The softmax is a running one: maximum and sum of every head, rescaled when a tile has a larger score.
//
// The work of all sequences is one list of units of kUnitRows rows of one KV head (and 16 of its query heads), sequence by sequence, head by head; every
// workgroup takes an equal, contiguous share, whatever the lengths.  What covers a head's rows completely is written out; a share's
// first and last piece otherwise leave {maximum, sum, values} in the scratch, which a second launch joins.  (Joined by the last workgroup of a head to arrive
// instead, over device-scope atomics, 128,000 rows took 104 us, not 98.7: what the others wrote has to be read past the caches.)
//
// Reading the pages bounds it: every cached element is read once.  32 sequences of up to 8192 rows (8 KV heads of 64, f16: 278 MB) take 55 us, 5.0 TB/s,
// and 4.9 us to join; 64 of up to 2002 rows in f32 (271 MB) 53 us, 5.1 TB/s; one of 128,000 rows (8 KV heads of 128, f16: 524 MB) 92 us, 5.7 TB/s, and 7.6 us
// to join.  Loads of the next tile ahead of a tile's products (f32: 53 to 56 us) and waves that yield to those with more left (no difference) do not pay:
// with 8 waves a CU the loads of one fill the products of another.
#include <algorithm>
#include <type_traits>

#include "kv_paged_device.h"
#include "wick_rocm_internal.h"

namespace wick_rocm {

namespace {

constexpr uint32_t kUnitRows = 128, kTileRows = 32, kWaves = 4;  // a unit is a tile of each wave
constexpr uint32_t kShares = 512;                                 // workgroups, two on each of 256 CUs (one where the registers of a row of 256 leave room for one)
constexpr uint32_t kRecordHead = 4;                              // floats of a record in front of its values: maximum, sum, -, -
constexpr float kHalfScale = 32768.0f;                           // softmax weights are split below or at a half's largest power of two
// Two halves of a value of 2^-3 to 2^15 are off by at most 2^-22 of it, of a smaller one by 2^-25.
constexpr int kQueryBits = 18;   // queries down to 2^-18 of a head's largest are halves
constexpr int kWeightBits = 21;  // weights down to 2^-21 of the largest are: off by 2^-19 then, as f32's rounding of such an exponent makes them (with 18, ordinary scores have tiles of f32)
constexpr float kLog2e = 1.44269504088896340736f;

struct PagedAttentionArgs {
    const float* q;
    const void* pages[2];  // keys, values
    const uint32_t *table, *lens;
    float* out;
    float* parts;  // [shares][2][records of a piece][kRecordHead + head_dim]
    uint32_t n_seqs, max_pages, n_pages, page_shift, q_stride, out_stride, n_heads, n_kv_heads, group, tiles, shares;  // tiles: of 16 query heads, of a KV head
    float scale;
};

__device__ __forceinline__ uint32_t length(const PagedAttentionArgs& a, uint32_t s) { return min(a.lens[s], a.max_pages << a.page_shift); }
__device__ __forceinline__ uint32_t units_of(uint32_t len) { return (len + kUnitRows - 1u) / kUnitRows; }

// Units of all sequences, and of those in front of sequence `upto`.
__device__ __forceinline__ uint32_t all_units(const PagedAttentionArgs& a, uint32_t heads, uint32_t upto, uint32_t& before) {
    uint32_t sum = 0, front = 0;
    for (uint32_t s = threadIdx.x & 63u; s < a.n_seqs; s += 64u) {
        const uint32_t n = units_of(length(a, s)) * heads;
        sum += n, front += s < upto ? n : 0u;
    }
    before = (uint32_t)__builtin_amdgcn_readlane((int)lanes_upto(front), 63);
    return (uint32_t)__builtin_amdgcn_readlane((int)lanes_upto(sum), 63);
}

// Share `w` of the units, [begin, end), the sequence of its first unit (or its last one) and the units in front of that sequence.  64 sequences at a time, a lane
// each, the lengths of several 64s on their way together; the 64 that have the unit are then looked at once more.
struct Share {
    uint32_t units, begin, end, s, before;
};
__device__ __forceinline__ uint32_t share_begin(uint32_t units, uint32_t w, uint32_t shares) { return (uint32_t)((uint64_t)units * w / shares); }
__device__ __forceinline__ uint32_t share_of(uint32_t units, uint32_t u, uint32_t shares) { return (uint32_t)((((uint64_t)u + 1) * shares - 1) / units); }
__device__ __forceinline__ Share share(const PagedAttentionArgs& a, uint32_t heads, uint32_t w, bool its_last) {
    const uint32_t lane = threadIdx.x & 63u, runs = (a.n_seqs + 63u) / 64u;
    const auto units_at = [&](uint32_t s) { return s < a.n_seqs ? units_of(length(a, s)) * heads : 0u; };
    uint32_t n = units_at(lane), upto = lanes_upto(n);
    uint32_t sum = lane == 0 ? (uint32_t)__builtin_amdgcn_readlane((int)upto, 63) : 0u;  // of the lane's 64
#pragma unroll 8
    for (uint32_t i = 1; i < runs; i++) {
        const uint32_t all = (uint32_t)__builtin_amdgcn_readlane((int)lanes_upto(units_at(64u * i + lane)), 63);
        sum = lane == i ? all : sum;
    }
    const uint32_t runs_upto = lanes_upto(sum);
    Share x{};
    x.units = (uint32_t)__builtin_amdgcn_readlane((int)runs_upto, 63);
    const uint32_t shares = min(x.units, a.shares);  // (no share is empty)
    if (w >= shares) return x;
    x.begin = share_begin(x.units, w, shares), x.end = share_begin(x.units, w + 1u, shares);
    const uint32_t unit = its_last ? x.end - 1u : x.begin;
    const int run = __ffsll((unsigned long long)__ballot(runs_upto > unit)) - 1;
    x.before = (uint32_t)__builtin_amdgcn_readlane((int)(runs_upto - sum), run);
    if (run != 0) n = units_at(64u * (uint32_t)run + lane), upto = lanes_upto(n);
    const int at = __ffsll((unsigned long long)__ballot(x.before + upto > unit)) - 1;
    x.before += (uint32_t)__builtin_amdgcn_readlane((int)(upto - n), at), x.s = 64u * (uint32_t)run + (uint32_t)at;
    return x;
}

// The first sequence from `s` on that has rows, or n_seqs; 64 at a time.  (20 sequences of 2000 rows among 1024: 20.4 us, 28.5 one by one; among 4000, with the search
// above, 33 and 69.  32 with rows each take 0.7 of 59 us longer for it.)
__device__ __forceinline__ uint32_t next_with_rows(const PagedAttentionArgs& a, uint32_t s) {
    const uint32_t lane = threadIdx.x & 63u;
    for (; s < a.n_seqs; s += 64u) {
        const uint64_t some = __ballot(s + lane < a.n_seqs && a.lens[min(s + lane, a.n_seqs - 1u)] != 0);
        if (some != 0) return s + (uint32_t)__ffsll((unsigned long long)some) - 1u;
    }
    return a.n_seqs;
}

template <typename KV, int HD>
struct Tile {
    static constexpr bool kF16 = sizeof(KV) == 2;
    static constexpr int kPer = HD / 16;                         // values of a row that a lane holds
    static constexpr int kVec = kPer < (kF16 ? 8 : 4) ? kPer : (kF16 ? 8 : 4);  // ... in one load
    static constexpr int kLoads = kPer / kVec;
    static constexpr int kSteps = kF16 ? HD / 32 : HD / 16;      // 16-byte loads of a key
    typedef KV kvec __attribute__((ext_vector_type(kF16 ? 8 : 4)));
    typedef KV vvec __attribute__((ext_vector_type(kVec)));
    kvec k[2][kSteps];
    vvec v[2][4][kLoads];
};

template <typename KV, int HD>
struct Query;
// Elements below 2^-18 of their head's largest are left out of the halves; f32 products add them to the scores, four dimensions at a time and only where there are
// any: `rest_of` (LDS, HD / 4 floats of each lane) has them.  32 sequences of up to 8192 rows of 64: 50.4 us without, 53.6 with one such element in every head, 69.8 with 63.
template <int HD>
struct Query<_Float16, HD> {
    v4f x[HD / 32][2];
    h8 hi[HD / 32], lo[HD / 32];
    float factor, rest_factor;
    uint64_t rest;  // bit 8 j + i: some of dims 32 j + 8 g + i
    __device__ __forceinline__ void load(const float* q, bool there) {
        const uint32_t g = (threadIdx.x & 63u) >> 4;
#pragma unroll
        for (int j = 0; j < HD / 32; j++)
#pragma unroll
            for (int i = 0; i < 2; i++) x[j][i] = there ? *reinterpret_cast<const v4f*>(q + 32 * j + 8u * g + 4 * i) : v4f{0, 0, 0, 0};
    }
    __device__ __forceinline__ void split(float scale, float* rest_of) {
        float top = 0.0f;
        uint32_t least = 0xffffffffu;  // of the magnitudes that are not zero
#pragma unroll
        for (int j = 0; j < HD / 32; j++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float y = x[j][i / 4][i % 4];
                top = fmaxf(top, fabsf(y)), least = min(least, 2u * __float_as_uint(y) - 1u);
            }
        top = groups_max(top);
        const int e = max(__builtin_amdgcn_frexp_expf(top), -100) - 15;  // (from 2^-100 down no score matters)
        const float enough = ldexpf(1.0f, e + 15 - kQueryBits);
        rest_factor = scale * kLog2e, factor = ldexpf(rest_factor, e), rest = 0;
        if (__any(least < 2u * __float_as_uint(enough) - 1u))
#pragma unroll
            for (int j = 0; j < HD / 32; j++)
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float y = x[j][i / 4][i % 4];
                    const bool small = fabsf(y) < enough && y != 0.0f;
                    rest |= (uint64_t)(__any(small) != 0) << (8 * j + i);
                    rest_of[(8 * j + i) * 64 + (threadIdx.x & 63u)] = small ? y : 0.0f;
                    x[j][i / 4][i % 4] = small ? 0.0f : y;
                }
#pragma unroll
        for (int j = 0; j < HD / 32; j++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float y = ldexpf(x[j][i / 4][i % 4], -e);
                hi[j][i] = (_Float16)y, lo[j][i] = (_Float16)(y - (float)hi[j][i]);
            }
    }
    __device__ __forceinline__ v4f scores(const typename Tile<_Float16, HD>::kvec (&k)[HD / 32]) const {
        v4f s = {0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < HD / 32; j++) {
            s = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[j], lo[j], s, 0, 0, 0);
            s = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[j], hi[j], s, 0, 0, 0);
        }
        return s;
    }
    __device__ __forceinline__ void add_rest(const typename Tile<_Float16, HD>::kvec (&k)[2][HD / 32], const float* rest_of, float (&sc)[8]) const {
        v4f s[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
        for (int j = 0; j < HD / 32; j++)
#pragma unroll
            for (int i = 0; i < 8; i++)
                if ((rest >> (8 * j + i) & 1u) != 0) {
                    const float y = rest_of[(8 * j + i) * 64 + (threadIdx.x & 63u)];
#pragma unroll
                    for (int half = 0; half < 2; half++) s[half] = __builtin_amdgcn_mfma_f32_16x16x4f32((float)k[half][j][i], y, s[half], 0, 0, 0);
                }
#pragma unroll
        for (int i = 0; i < 8; i++) sc[i] += s[i / 4][i % 4] * rest_factor;
    }
};
template <int HD>
struct Query<float, HD> {
    v4f x[HD / 16];
    float factor;
    static constexpr uint64_t rest = 0;
    __device__ __forceinline__ void load(const float* q, bool there) {
        const uint32_t g = (threadIdx.x & 63u) >> 4;
#pragma unroll
        for (int j = 0; j < HD / 16; j++) x[j] = there ? *reinterpret_cast<const v4f*>(q + 16 * j + 4u * g) : v4f{0, 0, 0, 0};
    }
    __device__ __forceinline__ void split(float scale, float*) { factor = scale * kLog2e; }
    __device__ __forceinline__ v4f scores(const typename Tile<float, HD>::kvec (&k)[HD / 16]) const {
        v4f s = {0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < HD / 16; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) s = __builtin_amdgcn_mfma_f32_16x16x4f32(k[j][e], x[j][e], s, 0, 0, 0);
        return s;
    }
    __device__ __forceinline__ void add_rest(const typename Tile<float, HD>::kvec (&)[2][HD / 16], const float*, float (&)[8]) const {}
};

// What a wave has gathered of a piece: per lane its head's maximum (of a power of two), the sum over its own rows, and 4 dimensions of every tile of the values.
template <typename KV, int HD>
struct State {
    typedef Tile<KV, HD> T;
    float m = -__builtin_inff(), l = 0.0f;
    v4f o[T::kPer];

    // The value of dimension (x, e) of m index i is x * 16 kVec + kVec i + e.
    // `least`: no score of a row that is there is below it.
    __device__ __forceinline__ void add(const T& t, const float (&s)[8], float least) {
        float top = s[0];
#pragma unroll
        for (int i = 1; i < 8; i++) top = fmaxf(top, s[i]);
        if (__any(top > m)) {
            const float now = fmaxf(m, groups_max(top)), less = m == now ? 1.0f : __builtin_amdgcn_exp2f(m - now);
#pragma unroll
            for (int d = 0; d < T::kPer; d++) o[d] *= less;
            l *= less, m = now;
        }
        const float from = m == -__builtin_inff() ? 0.0f : m;
        float p[8];
#pragma unroll
        for (int i = 0; i < 8; i++) p[i] = __builtin_amdgcn_exp2f(s[i] - from);
        l += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
        if constexpr (T::kF16) {
#pragma unroll
            for (int i = 0; i < 8; i++) p[i] *= kHalfScale;
            if (!__any(least < m - kWeightBits)) {  // (32 sequences of scores that spread by 2^20 and more take 57.0 us, not 50.4)
                h8 hi, lo;
#pragma unroll
                for (int i = 0; i < 8; i++) hi[i] = (_Float16)p[i], lo[i] = (_Float16)(p[i] - (float)hi[i]);
#pragma unroll
                for (int x = 0; x < T::kLoads; x++) {
                    // (whole vectors first: elements picked from the array itself keep it out of registers)
                    const typename T::vvec r0 = t.v[0][0][x], r1 = t.v[0][1][x], r2 = t.v[0][2][x], r3 = t.v[0][3][x], r4 = t.v[1][0][x], r5 = t.v[1][1][x], r6 = t.v[1][2][x], r7 = t.v[1][3][x];
#pragma unroll
                    for (int e = 0; e < T::kVec; e++) {
                        const h8 v = {r0[e], r1[e], r2[e], r3[e], r4[e], r5[e], r6[e], r7[e]};
                        v4f& d = o[x * T::kVec + e];
                        d = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, lo, d, 0, 0, 0);
                        d = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, hi, d, 0, 0, 0);
                    }
                }
                return;
            }
        }
#pragma unroll
        for (int half = 0; half < 2; half++)
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int x = 0; x < T::kLoads; x++) {
                    const typename T::vvec r = t.v[half][i][x];
#pragma unroll
                    for (int e = 0; e < T::kVec; e++) {
                        v4f& d = o[x * T::kVec + e];
                        d = __builtin_amdgcn_mfma_f32_16x16x4f32((float)r[e], p[4 * half + i], d, 0, 0, 0);
                    }
                }
    }
};

// Where a tile's rows are: those at or behind `len` are the last one's (their weights are zero), those without a page the first page's.
struct Place {
    size_t base[2];  // rows in front of each half's page of this KV head
    uint32_t first, there;  // bit h of `there`: half h has a page
};
__device__ __forceinline__ Place place(const PagedAttentionArgs& a, const uint32_t* table, uint32_t c, uint32_t first, uint32_t len) {
    Place p{{0, 0}, first, 0};
#pragma unroll
    for (int half = 0; half < 2; half++) {
        const uint32_t page = table[min(first + 16u * half, len - 1u) >> a.page_shift];
        p.there |= (uint32_t)(page < a.n_pages) << half;
        p.base[half] = ((size_t)(page < a.n_pages ? page : 0u) * a.n_kv_heads + c) << a.page_shift;
    }
    return p;
}
template <typename KV, int HD>
__device__ __forceinline__ void load_tile(const PagedAttentionArgs& a, const Place& p, uint32_t len, Tile<KV, HD>& t) {
    typedef Tile<KV, HD> T;
    const uint32_t l16 = threadIdx.x & 15u, g = (threadIdx.x & 63u) >> 4, inside = (1u << a.page_shift) - 1u;
#pragma unroll
    for (int half = 0; half < 2; half++) {
        const KV* const k = static_cast<const KV*>(a.pages[0]) + (p.base[half] + (min(p.first + 16u * half + l16, len - 1u) & inside)) * HD + (T::kF16 ? 8u : 4u) * g;
#pragma unroll
        for (int j = 0; j < T::kSteps; j++) t.k[half][j] = *reinterpret_cast<const typename T::kvec*>(k + j * (T::kF16 ? 32 : 16));
    }
#pragma unroll
    for (int half = 0; half < 2; half++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const KV* const v = static_cast<const KV*>(a.pages[1]) + (p.base[half] + (min(p.first + 16u * half + 4u * g + i, len - 1u) & inside)) * HD + T::kVec * l16;
#pragma unroll
            for (int x = 0; x < T::kLoads; x++) t.v[half][i][x] = *reinterpret_cast<const typename T::vvec*>(v + x * 16 * T::kVec);
        }
}

// A half without a page: its values are zeros, whatever was read.
template <typename KV, int HD>
__device__ __forceinline__ void clear_values(Tile<KV, HD>& t, uint32_t there) {
#pragma unroll
    for (int half = 0; half < 2; half++)
        if ((there >> half & 1u) == 0)
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int x = 0; x < Tile<KV, HD>::kLoads; x++) t.v[half][i][x] = typename Tile<KV, HD>::vvec(0);
}

// Waves of a SIMD: exactly as many as there are.  (With registers for a third one in mind the compiler loads values behind the first products: 61.0 us, not 59.3.)
constexpr int waves_of_simd(int hd, int waves) { return waves == 16 ? 4 : hd == 256 ? 1 : 2; }

// A workgroup's share of all units, or, where the table has room for few rows (SHORT), all rows of one sequence's KV head (and 16 of its query heads): no piece is left.
template <typename KV, int HD, uint32_t WAVES, bool SHORT>
__global__ __launch_bounds__(64 * WAVES) __attribute__((amdgpu_waves_per_eu(waves_of_simd(HD, WAVES), waves_of_simd(HD, WAVES)))) void attention_paged_kernel(PagedAttentionArgs a) {
    typedef Tile<KV, HD> T;
    constexpr uint32_t kRow = HD + 4, kStep = WAVES * kTileRows;  // floats of a head's values in LDS; rows of all waves
    static_assert(SHORT || kStep == kUnitRows);
    __shared__ __align__(16) float values[WAVES][16][kRow];
    __shared__ float tops[WAVES][16], sums[WAVES][16];
    const uint32_t lane = threadIdx.x & 63u, l16 = lane & 15u, g = lane >> 4;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t heads = a.n_kv_heads * a.tiles, records = min(a.group, 16u);
    const Share sh = SHORT ? Share{0, 0, 1, blockIdx.x / heads, 0} : share(a, heads, blockIdx.x, false);
    uint32_t s = sh.s, before = sh.before;
    for (uint32_t u = sh.begin; u < sh.end && s < a.n_seqs;) {
        const uint32_t len = length(a, s), chunks = units_of(len);
        if (!SHORT && u - before >= chunks * heads) {
            before += chunks * heads, s = chunks != 0 ? s + 1u : next_with_rows(a, s + 1u);
            continue;
        }
        const uint32_t head = SHORT ? blockIdx.x % heads : (u - before) / chunks, chunk = SHORT ? 0u : (u - before) % chunks, take = SHORT ? 1u : min(chunks - chunk, sh.end - u);
        const uint32_t c = head / a.tiles, h0 = c * a.group + head % a.tiles * 16u, h_count = min(a.group - head % a.tiles * 16u, 16u);
        const uint32_t* const table = a.table + (size_t)s * a.max_pages;
        Query<KV, HD> q;
        q.load(a.q + (size_t)s * a.q_stride + (size_t)(h0 + min(l16, h_count - 1u)) * HD, l16 < h_count);
        float* const rest_of = &values[wave][0][0];  // (its own wave's, until the state goes there)
        q.split(a.scale, rest_of);
        State<KV, HD> st;
#pragma unroll
        for (int d = 0; d < T::kPer; d++) st.o[d] = v4f{0, 0, 0, 0};
        const uint32_t last = SHORT ? len : min(len, (chunk + take) * kUnitRows);
        const auto walk = [&](auto rest) __attribute__((always_inline)) {  // (a loop for either: a branch inside cost all queries 2 to 9 %, for values were loaded behind products)
            for (uint32_t first = chunk * kUnitRows + wave * kTileRows; first < last; first += kStep) {
                T t;
                const Place p = place(a, table, c, first, len);
                load_tile(a, p, len, t);
                float sc[8];
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    const v4f x = q.scores(t.k[half]);
#pragma unroll
                    for (int i = 0; i < 4; i++) sc[4 * half + i] = x[i] * q.factor;
                }
                if constexpr (decltype(rest)::value) q.add_rest(t.k, rest_of, sc);
                float least = sc[0];
#pragma unroll
                for (int i = 1; i < 8; i++) least = fminf(least, sc[i]);
                if (first + kTileRows > len || p.there != 3u) {
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        if (first + 16u * (i / 4) + 4u * g + i % 4 >= len || (p.there >> (i / 4) & 1u) == 0) sc[i] = -__builtin_inff();
                    clear_values(t, p.there);
                }
                st.add(t, sc, least);
            }
        };
        if (q.rest == 0) walk(std::false_type());
        else walk(std::bool_constant<T::kF16>());
        // The waves' states, one head after another
        st.l = groups_sum(st.l);
        if (g == 0) tops[wave][l16] = st.m, sums[wave][l16] = st.l;
        constexpr int kWide = T::kVec < 4 ? T::kVec : 4;
        typedef float wide __attribute__((ext_vector_type(kWide)));
#pragma unroll
        for (int x = 0; x < T::kLoads; x++)
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int e = 0; e < T::kVec; e += kWide) {
                    wide w;
#pragma unroll
                    for (int k = 0; k < kWide; k++) w[k] = st.o[x * T::kVec + e + k][r];
                    *reinterpret_cast<wide*>(&values[wave][l16][x * 16 * T::kVec + T::kVec * (4u * g + r) + e]) = w;
                }
        __syncthreads();
        const bool whole = SHORT || take == chunks;
        for (uint32_t i = threadIdx.x; i < h_count * (HD / 4); i += 64u * WAVES) {
            const uint32_t h = i / (HD / 4), d = i % (HD / 4) * 4u;
            float top = tops[0][h];
#pragma unroll
            for (uint32_t w = 1; w < WAVES; w++) top = fmaxf(top, tops[w][h]);
            const float from = top == -__builtin_inff() ? 0.0f : top;
            float sum = 0.0f;
            v4f v = {0, 0, 0, 0};
#pragma unroll
            for (uint32_t w = 0; w < WAVES; w++) {
                const float less = __builtin_amdgcn_exp2f(tops[w][h] - from);
                sum += sums[w][h] * less;
                v += *reinterpret_cast<const v4f*>(&values[w][h][d]) * less;
            }
            if (whole) {
                const float inverse = sum == 0.0f ? 0.0f : 1.0f / (T::kF16 ? sum * kHalfScale : sum);
                *reinterpret_cast<v4f*>(a.out + (size_t)s * a.out_stride + (size_t)(h0 + h) * HD + d) = v * inverse;
            } else {
                float* const to = a.parts + ((size_t)(blockIdx.x * 2u + (u == sh.begin ? 0u : 1u)) * records + h) * (kRecordHead + HD);
                if (d == 0) to[0] = top, to[1] = T::kF16 ? sum * kHalfScale : sum;
                *reinterpret_cast<v4f*>(to + kRecordHead + d) = v;
            }
        }
        if (SHORT) return;
        __syncthreads();
        u += take;
    }
    for (uint32_t e = blockIdx.x; e < a.n_seqs; e += gridDim.x)  // sequences without rows
        if (a.lens[e] == 0)
            for (uint32_t i = threadIdx.x; i < a.n_heads * (HD / 4); i += 64u * WAVES) reinterpret_cast<v4f*>(a.out + (size_t)e * a.out_stride)[i] = v4f{0, 0, 0, 0};
}

// Joins the pieces of a KV head (and 16 of its query heads) for one of the query heads, blockIdx.y.  Where there are more such heads than shares, the first
// of which a share leaves for the next one is the head that its last unit is in: one workgroup a share (BY_SHARE), otherwise one a head.  With 400
// sequences of 32 heads and up to 1024 rows, one workgroup a head took 20.9 us, one a share 11.3 us.
template <int HD, bool BY_SHARE>
__global__ __launch_bounds__(256) void attention_paged_join_kernel(PagedAttentionArgs a) {
    __shared__ float weights[kShares];
    __shared__ __align__(16) float values[256 / (HD / 4)][HD];
    __shared__ float tops[4], totals[4];
    const uint32_t heads = a.n_kv_heads * a.tiles, lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    uint32_t s, head, units, u0, chunks, w0;
    if constexpr (BY_SHARE) {
        const Share sh = share(a, heads, blockIdx.x, true);
        if (sh.begin == sh.end) return;
        s = sh.s, units = sh.units, w0 = blockIdx.x, chunks = units_of(length(a, s));
        head = (sh.end - 1u - sh.before) / chunks, u0 = sh.before + head * chunks;
        if (u0 < sh.begin || u0 + chunks == sh.end) return;  // begun by an earlier share, or whole
    } else {
        uint32_t before;
        s = blockIdx.x / heads, head = blockIdx.x % heads, units = all_units(a, heads, s, before), chunks = units_of(length(a, s)), u0 = before + head * chunks;
        if (chunks == 0) return;
        w0 = share_of(units, u0, min(units, a.shares));
    }
    const uint32_t shares = min(units, a.shares), n = share_of(units, u0 + chunks - 1u, shares) - w0 + 1u;
    const uint32_t in_tile = blockIdx.y, h = head / a.tiles * a.group + head % a.tiles * 16u + in_tile;
    if (n == 1 || head % a.tiles * 16u + in_tile >= a.group) return;
    float* const out = a.out + (size_t)s * a.out_stride + (size_t)h * HD;
    const uint32_t stride = 2u * min(a.group, 16u) * (kRecordHead + HD);  // of the first pieces of two shares; a share's second is half of it behind
    const float* const parts = a.parts + (size_t)w0 * stride + in_tile * (kRecordHead + HD);
    const uint32_t front = share_begin(units, w0, shares) != u0 ? stride / 2u : 0u;
    const auto record = [&](uint32_t i) { return parts + (i == 0 ? front : i * stride); };
    // A thread's records' heads, and its part of the first records' values, are read in one go.
    constexpr uint32_t kQuads = HD / 4, kGroups = 256 / kQuads, kAhead = 4;
    static_assert(kShares <= 512);
    const uint32_t d = threadIdx.x % kQuads, part = threadIdx.x / kQuads;
    float tops_of[2] = {-__builtin_inff(), -__builtin_inff()}, sums_of[2] = {0.0f, 0.0f};
    v4f ahead[kAhead];
#pragma unroll
    for (uint32_t x = 0; x < 2; x++)
        if (threadIdx.x + 256u * x < n) {
            const float* const r = record(threadIdx.x + 256u * x);
            tops_of[x] = r[0], sums_of[x] = r[1];
        }
#pragma unroll
    for (uint32_t x = 0; x < kAhead; x++)
        if (part + x * kGroups < n) ahead[x] = *reinterpret_cast<const v4f*>(record(part + x * kGroups) + kRecordHead + 4u * d);
    float top = wave_max_f32(fmaxf(tops_of[0], tops_of[1]));
    if (lane == 0) tops[wave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    const float from = top == -__builtin_inff() ? 0.0f : top;
    float sum = 0.0f;
#pragma unroll
    for (uint32_t x = 0; x < 2; x++)
        if (threadIdx.x + 256u * x < n) {
            const float w = __builtin_amdgcn_exp2f(tops_of[x] - from);
            weights[threadIdx.x + 256u * x] = w, sum += w * sums_of[x];
        }
    sum = wave_sum_f32(sum);
    if (lane == 0) totals[wave] = sum;
    __syncthreads();
    sum = (totals[0] + totals[1]) + (totals[2] + totals[3]);
    v4f v = {0, 0, 0, 0};
#pragma unroll
    for (uint32_t x = 0; x < kAhead; x++)
        if (part + x * kGroups < n) v += ahead[x] * weights[part + x * kGroups];
    for (uint32_t i = part + kAhead * kGroups; i < n; i += kGroups) v += *reinterpret_cast<const v4f*>(record(i) + kRecordHead + 4u * d) * weights[i];
    reinterpret_cast<v4f*>(values[part])[d] = v;
    __syncthreads();
    if (threadIdx.x < kQuads) {
        for (uint32_t p = 1; p < kGroups; p++) v += reinterpret_cast<const v4f*>(values[p])[d];
        reinterpret_cast<v4f*>(out)[d] = v * (sum == 0.0f ? 0.0f : 1.0f / sum);
    }
}

// Waves of a workgroup for short tables, as many as the registers allow.  A table is short where its rows are at most two tiles a wave: one launch without a join.
// For 32 heads of 64 in f16, 1 sequence of 512 rows takes 6.2 us, in shares 4.7 and 4.2 for the join; 32 of 1024 rows 12.8, in shares 13.6 and 4.2; 400 of up to
// 1024 rows 98, in shares 107 and 11.
template <typename KV, int HD>
constexpr uint32_t kShortWaves = HD * sizeof(KV) <= 128 ? 16 : HD * sizeof(KV) <= 256 ? 8 : 4;

template <typename KV, int HD>
hipError_t launch_paged(const PagedAttentionArgs& a, const Launch& L) {
    constexpr uint32_t W = kShortWaves<KV, HD>;
    if (((uint64_t)a.max_pages << a.page_shift) <= 2u * W * kTileRows)
        return launch_kernel(L, kFamOther, attention_paged_kernel<KV, HD, W, true>, dim3(a.n_seqs * a.n_kv_heads * a.tiles), dim3(64 * W), a);
    hipError_t e = launch_kernel(L, kFamOther, attention_paged_kernel<KV, HD, kWaves, false>, dim3(a.shares), dim3(64 * kWaves), a);
    if (e != hipSuccess) return e;
    const uint32_t heads = a.n_seqs * a.n_kv_heads * a.tiles, records = std::min(a.group, 16u);
    return heads > a.shares ? launch_kernel(L, kFamOther, attention_paged_join_kernel<HD, true>, dim3(a.shares, records), dim3(256), a)
                           : launch_kernel(L, kFamOther, attention_paged_join_kernel<HD, false>, dim3(heads, records), dim3(256), a);
}

template <typename KV>
hipError_t launch_paged(const PagedAttentionArgs& a, uint32_t head_dim, const Launch& L) {
    return head_dim == 32 ? launch_paged<KV, 32>(a, L) : head_dim == 64 ? launch_paged<KV, 64>(a, L) : head_dim == 128 ? launch_paged<KV, 128>(a, L) : launch_paged<KV, 256>(a, L);
}

}  // namespace

bool attention_paged_fits(const wick_rocm_kv_pages& p, uint32_t n_heads, uint32_t n_kv_heads) {
    const uint64_t tiles = (n_heads / n_kv_heads + 15u) / 16u, chunks = ((uint64_t)p.max_pages * p.page_rows + kUnitRows - 1u) / kUnitRows;
    // (each factor is at most 2^30; a launch has less than 2^32 threads, of which 1024 may go to a sequence's KV head)
    return p.n_seqs * chunks <= UINT32_MAX / 2u / (n_kv_heads * tiles) && (uint64_t)p.n_seqs * n_kv_heads * tiles <= 1u << 21;
}

size_t attention_paged_scratch_floats(uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim) {
    return (size_t)kShares * 2 * std::min(n_heads / n_kv_heads, 16u) * (kRecordHead + head_dim);
}

hipError_t launch_attention_paged(const wick_rocm_kv_pages& p, const float* d_q, uint32_t q_stride, const void* d_k_pages, const void* d_v_pages, bool kv_f16,
                                  float* d_out, uint32_t out_stride, float* d_scratch, uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim, float scale,
                                  const Launch& L) {
    const uint32_t group = n_heads / n_kv_heads;
    // Two workgroups of rows of 256 do not fit on a CU, and twice the shares only leave more to join: f16, 128,000 rows 185 and 7.8 us (512 shares: 190 and
    // 12.8), 128 sequences of up to 1024 rows 127 and 5.7 (144 and 8).  With rows of 128 it would be 53 us against 62.
    const uint32_t shares = head_dim == 256 ? kShares / 2 : kShares;
    const PagedAttentionArgs a{d_q, {d_k_pages, d_v_pages}, p.d_table, p.d_lens, d_out, d_scratch, p.n_seqs, p.max_pages, p.n_pages, (uint32_t)__builtin_ctz(p.page_rows),
                               q_stride, out_stride, n_heads, n_kv_heads, group, (group + 15u) / 16u, shares, scale};
    return kv_f16 ? launch_paged<_Float16>(a, head_dim, L) : launch_paged<float>(a, head_dim, L);
}

}  // namespace wick_rocm
