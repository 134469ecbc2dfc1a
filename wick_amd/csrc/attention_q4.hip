// Attention over KV caches held in 4 bits (kv_q4_device.h), on the f16 matrix cores at f32 accuracy.
//
// With G = n_heads / n_kv_heads, the query heads of KV head c over n tokens are n G rows, row r = token r / G, head c G + r % G:
// all of them read the same keys and values, and row r sees rows [0, pos0 + r / G] of the cache.  A workgroup takes 32 WQ of them and
// walks the cache in tiles of 32 WK rows: wave (wq, wk) multiplies 32 query rows with 32 rows of each tile, on
// v_mfma_f32_32x32x16_f16, both products transposed:
//   S^T[key][row] = sum_d K[key][d] Q[row][d]    lane l is left with keys 8 (i / 4) + 4 (l / 32) + i % 4 of row l % 32;
//   O^T[d][row]  += sum_key V[key][d] P[key][row]   whose B operand is, per lane, consecutive K steps of one row: the weights as they
//                                                   are in the lane's registers (an MFMA's K steps are in any order, so both
//                                                   operands agree on which key a lane's slot is).
// Accuracy: a cached value, four bits times an f16 scale, is the sum of two halves exactly (hi = f16(n d), lo = f16(n d - hi), 15 bits
// in all); a query row, scaled by a power of two to below 2^15, and a softmax weight, times 2^15, are split into two halves, which keep 22 bits of a
// value x, or what is above 2^-25: it is off by at most max(2^-22 |x|, 2^-40 of the row's largest query or weight).  (With the largest below 1 small values beside
// it would be off by 2^-25 of it: outputs by 9e-5 where channels of the keys are 1000 times as large as the others and the queries' as small.)
// a b = a_hi b_hi + a_hi b_lo + a_lo b_hi: each product of halves is exact, sums are f32's, what is dropped is below 2^-22.
// (One half for the weights or the queries would be off by 2^-12 of each: 100 times what f32 sums are.)
// Bound by the matrix and vector instructions of a unit of 32 rows and 32 keys (heads of 64: 24 matrix instructions of 32 cycles and 920 cycles of vector ones, of
// the softmax above all, in 2060 cycles): 2002 tokens of 32 heads over 8 of 64 59 us, 2048 behind 6144 of 16 heads over 4 of 128 300 us (three
// products are 307 at the 1175 TFLOP/s of a large library product; power).
#include <algorithm>

#include "attention_device.h"
#include "kv_q4_device.h"
#include "wick_rocm_internal.h"

namespace wick_rocm {

namespace {

constexpr int kHalfBits = 15;              // queries and weights are split below or at 2^15, a half's largest power of two, so that small ones keep their bits
constexpr float kWeightBits = kHalfBits;   // softmax weights are taken times 2^15
// Workgroups that share the rows of the cache among them at the most, so that a row's records stay few for the merge and the scratch small.  Nothing measured says that 96 is
// the best: with fewer than six KV heads of up to 128 values (three of 256) it leaves workgroups' places empty (a token over 100000 rows of one KV head 10.5 + 3.8 us, over
// 12500 of eight 7.2 + 3.5; of 128 values 15.9 + 4.0 and 10.2 + 3.9; of 256, 60000 rows and 7500, 20.1 + 6.2 and 13.1 + 3.9; two KV heads lie between).
constexpr uint32_t kMaxSplits = 96;
constexpr uint32_t kCus = 256;
constexpr uint32_t kSplitSlots = 2 * kCus; // workgroups that a split launch has at the most by its launcher's rule
constexpr uint32_t kMostRows = 128;        // query rows of a workgroup at the most
constexpr uint32_t kMostRecords = kSplitSlots * kMostRows;  // of all splits of a launch
constexpr float kLog2e = 1.44269504088896340736f;

struct Q4AttentionArgs {
    const float* q;  // [n][q_stride]
    const void* k_cache;
    const void* v_cache;
    float* out;      // [n][out_stride]
    float* parts;    // records of the splits, [n * n_heads][splits][4 + head_dim]: {maximum, sum, -, -, values}
    float* stats;    // {maximum (as a power of two), 1 / (sum 2^15)} of every (token, head)'s softmax, for the weights; may be null
    float* weights;  // [n_kv_heads][max_seq]
    const uint32_t* d_pos;
    uint32_t pos0, n, q_stride, out_stride, max_seq, n_heads, n_kv_heads, splits;
    uint32_t first_blocks;  // blocks of query rows that are taken in descending order
    float scale;
};

__device__ __forceinline__ uint32_t first_row(const Q4AttentionArgs& a) { return min(a.d_pos ? *a.d_pos : a.pos0, a.max_seq - 1u); }
// The row of the cache up to which query row r sees (rows past the last one: that one's).
__device__ __forceinline__ uint32_t sees(const Q4AttentionArgs& a, uint32_t base, uint32_t r, uint32_t rows, uint32_t group) {
    return min(base + min(r, rows - 1u) / group, a.max_seq - 1u);
}
// Splits that a workgroup of `tiles` tiles has in earnest: with the position on the device the host does not know.
__device__ __forceinline__ uint32_t used_splits(uint32_t splits, uint32_t tiles) { return min(splits, tiles); }

// Eight values of a word as two planes of halves, a pair at a time: nibbles in bits 0 .. 3 of a half are the last bits of 1024 + nibble, in bits 4 .. 7 those of
// 64 + nibble, so only the upper half of the pairs is shifted.  (The mask in a scalar and the offset's bits in a vector register: one instruction takes both.)
__device__ __forceinline__ void dequantize_pair(uint32_t w, h2 d, int i, int at, h8& hi, h8& lo) {
    const h2 offset = i & 1 ? h2{(_Float16)72.0f, (_Float16)72.0f} : h2{(_Float16)1032.0f, (_Float16)1032.0f};
    uint32_t mask = i & 1 ? 0x00f000f0u : 0x000f000fu, bits = i & 1 ? 0x54005400u : 0x64006400u;
    asm("" : "+s"(mask), "+v"(bits));
    const h2 n = __builtin_bit_cast(h2, ((i < 2 ? w : w >> 8) & mask) | bits) - offset;  // nibble - 8, exact
    const h2 h = n * d, l = __builtin_elementwise_fma(n, d, -h);
    hi[2 * at] = h[0], hi[2 * at + 1] = h[1], lo[2 * at] = l[0], lo[2 * at + 1] = l[1];
}
__device__ __forceinline__ void dequantize(uint32_t w, _Float16 scale, h8& hi, h8& lo) {
#pragma unroll
    for (int i = 0; i < 4; i++) dequantize_pair(w, h2{scale, scale}, i, i, hi, lo);
}

// Four f32 values as two planes: a pair at a time, then one instruction a value (y * 1 - hi, rounded to a half; the compiler does not see the 1 and cannot
// make two instructions of it).
__device__ __forceinline__ void split_halves(const v4f& y, h4& hi, h4& lo) {
    float one = 1.0f;
    asm("" : "+s"(one));
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
        const h2 h = __builtin_convertvector((v2f{y[i], y[i + 1]}), h2);
        hi[i] = h[0], hi[i + 1] = h[1];
        lo[i] = (_Float16)__builtin_fmaf(y[i], one, -(float)h[0]), lo[i + 1] = (_Float16)__builtin_fmaf(y[i + 1], one, -(float)h[1]);
    }
}

__device__ __forceinline__ float halves_max(float v) {  // over lanes l, l ^ 32
    const uint32_t b = __float_as_uint(v);
    const auto r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float halves_sum(float v) {
    const uint32_t b = __float_as_uint(v);
    const auto r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// The power of two that a query row whose largest magnitude is `top` is taken without, for its halves; its scores' factor has it again: the largest is below 2^15 then,
// and small ones beside it have as many bits of a half below them as there are.  From below 2^-100 on (where no score is above 2^-70) it stays where it is: a factor
// that rounds to zero would make NaN of a masked key's score, which is -infinity.
__device__ __forceinline__ int query_exponent(float top) { return max(__builtin_amdgcn_frexp_expf(top), -100) - kHalfBits; }

// 32 query rows as the B operand of the first product: dims 16 s + 8 h .. + 7 of row l32, times 2^-e (the row's largest below 2^15), and
// the factor that turns a product into a power of two.
template <int HD>
struct Queries {
    struct Raw {
        v4f x[HD / 8];
        __device__ __forceinline__ void request(const Q4AttentionArgs& a, uint32_t r, uint32_t c, uint32_t group, uint32_t h) {
            const float* const p = a.q + (size_t)(r / group) * a.q_stride + (size_t)(c * group + r % group) * HD + 8u * h;
#pragma unroll
            for (int i = 0; i < HD / 8; i++) x[i] = *reinterpret_cast<const v4f*>(p + 16 * (i / 2) + 4 * (i % 2));
        }
    };
    h8 hi[HD / 16], lo[HD / 16];
    float factor;
    __device__ __forceinline__ void take(const Raw& raw, float scale) {
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < HD / 8; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) top = fmaxf(top, fabsf(raw.x[i][e]));
        const int e = query_exponent(halves_max(top));
        factor = __builtin_amdgcn_ldexpf(scale * kLog2e, e);
#pragma unroll
        for (int s = 0; s < HD / 16; s++) {
            h4 u[2], l[2];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                v4f y;
#pragma unroll
                for (int k = 0; k < 4; k++) y[k] = __builtin_amdgcn_ldexpf(raw.x[2 * s + i][k], -e);
                split_halves(y, u[i], l[i]);
            }
            hi[s] = __builtin_shufflevector(u[0], u[1], 0, 1, 2, 3, 4, 5, 6, 7), lo[s] = __builtin_shufflevector(l[0], l[1], 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
};

// A tile of the cache in LDS, two planes of halves: keys as rows with 16 bytes between them (conflict-free reads of 16 bytes), values with piece p of
// 16 bytes of a row at p ^ swizzle(row), so that the 4 rows of 32 bytes that 16 lanes of a transposing read touch are on different banks.
template <int HD, int KT>
struct KeyTile {
    _Float16 h[2][KT][HD + 8];
};
template <int HD, int KT>
struct ValueTile {
    _Float16 h[2][KT][HD];
    static __device__ __forceinline__ uint32_t swizzle(uint32_t row) { return HD >= 64 ? (row & 3u) << 1 | (row >> 2 & 1u) : row & 2u; }
};

// A thread's share of a tile of keys or of values as loaded: P pieces of W words of one block of one row, and the block's scales.
template <int W, int P>
struct Raw {
    struct __attribute__((aligned(4 * W))) Words {
        uint32_t w[W];
    };
    Words w[P];
    uint16_t kd[P], vd[P];
};

template <int HD, int WQ, int WK, int PER_CU>
__global__ __launch_bounds__(64 * WQ * WK, PER_CU * WQ * WK / 4) void attention_q4_kernel(Q4AttentionArgs a) {
    constexpr int KT = 32 * WK, NT = 64 * WQ * WK, SLABS = HD / 16, DT = HD / 32, kWords = KT * HD / 8 / NT, W = kWords < 4 ? kWords : 4, P = kWords / W;
    constexpr int kStates = 2 + HD / 2;
    constexpr uint32_t RB = 32 * WQ;  // query rows of a workgroup
    static_assert(kWords >= 1 && W * P * NT == KT * HD / 8, "every thread moves the same number of words");
    using Share = Raw<W, P>;
    using VT = ValueTile<HD, KT>;
    constexpr size_t kTiles = 2 * (sizeof(KeyTile<HD, KT>) + sizeof(VT)), kStateBytes = sizeof(float) * kStates * 64 * WQ * (WK - 1);
    __shared__ __align__(16) uint8_t smem[kTiles > kStateBytes ? kTiles : kStateBytes];
    KeyTile<HD, KT>* const k_tile = reinterpret_cast<KeyTile<HD, KT>*>(smem);
    VT* const v_tile = reinterpret_cast<VT*>(smem + 2 * sizeof(KeyTile<HD, KT>));
    const uint32_t group = a.n_heads / a.n_kv_heads, rows = a.n * group, blocks = (rows + RB - 1u) / RB;
    // Workgroups go to the eight XCDs in turn: a KV head's share an L2 where there are eight of them.  Those with the most to see first; where all of them are on
    // the GPU at once, two a CU, the second half the other way round, so that a CU's two have as much together as any other's.
    const uint32_t c = blockIdx.x % a.n_kv_heads, split = blockIdx.x / a.n_kv_heads % a.splits, nth = blockIdx.x / a.n_kv_heads / a.splits;
    const uint32_t block = PER_CU == 2 && nth >= a.first_blocks ? nth - a.first_blocks : blocks - 1u - nth;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, l32 = lane & 31u, h = lane >> 5, l16 = lane & 15u;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tid >> 6)), wq = wave / WK, wk = wave % WK;
    const uint32_t base = first_row(a), r0 = block * RB + 32u * wq;
    const uint32_t wg_last = sees(a, base, block * RB + RB - 1u, rows, group), n_tiles = wg_last / KT + 1u, used = used_splits(a.splits, n_tiles);
    if (split >= used) return;
    const uint32_t t_first = (uint32_t)((uint64_t)n_tiles * split / used), t_end = (uint32_t)((uint64_t)n_tiles * (split + 1u) / used);
    const uint32_t r = min(r0 + l32, rows - 1u), mine = sees(a, base, r, rows, group), wave_first = sees(a, base, r0, rows, group);

    const Q4Cache kc = q4_planes(const_cast<void*>(a.k_cache), a.max_seq, a.n_kv_heads, HD), vc = q4_planes(const_cast<void*>(a.v_cache), a.max_seq, a.n_kv_heads, HD);
    const size_t first = (size_t)c * a.max_seq;
    // The tiles from t_first on, one behind the other, by offsets into what the workgroup's rows see of each plane: a read behind it gives zeros (whose weights
    // the mask makes zeros).
    const uint32_t from = t_first * KT, seen = wg_last + 1u - from;
    const auto plane = [&](const void* p, uint32_t row_bytes) {
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(static_cast<const uint8_t*>(p)) + (first + from) * row_bytes, 0, (int)(seen * row_bytes), 0x27000);
    };
    const auto kq = plane(kc.quants, HD / 2), vq = plane(vc.quants, HD / 2), ks = plane(kc.scales, HD / 16), vs = plane(vc.scales, HD / 16);
    uint32_t q_at[P], s_at[P];  // of this thread's pieces in the tile that is requested next
#pragma unroll
    for (int p = 0; p < P; p++) q_at[p] = (p * NT + tid) * W * 4u, s_at[p] = (p * NT + tid) * W / 4u * 2u;
    const auto fetch = [&](Share& x, bool keys) {
#pragma unroll
        for (int p = 0; p < P; p++) {
            if constexpr (W == 1) x.w[p].w[0] = __builtin_amdgcn_raw_buffer_load_b32(keys ? kq : vq, q_at[p], 0, 0);
            if constexpr (W == 2) x.w[p] = __builtin_bit_cast(typename Share::Words, __builtin_amdgcn_raw_buffer_load_b64(keys ? kq : vq, q_at[p], 0, 0));
            if constexpr (W == 4) x.w[p] = __builtin_bit_cast(typename Share::Words, __builtin_amdgcn_raw_buffer_load_b128(keys ? kq : vq, q_at[p], 0, 0));
            x.vd[p] = __builtin_amdgcn_raw_buffer_load_b16(vs, s_at[p], 0, 0);
            if (keys) x.kd[p] = __builtin_amdgcn_raw_buffer_load_b16(ks, s_at[p], 0, 0);
        }
    };
    const auto next_tile = [&] {
#pragma unroll
        for (int p = 0; p < P; p++) q_at[p] += KT * HD / 2, s_at[p] += KT * HD / 16;
    };
    // Values that are not finite would reach the rows that do not see them (0 times NaN): they are taken as zeros and their keys as NaN, whose scores the
    // mask replaces.  A thread's share is unpacked and stored in kSteps steps, a pair of values each.
    constexpr int kSteps = 4 * kWords;
    h8 step_hi, step_lo;
    _Float16 step_scale;
    const auto store_step = [&](int buffer, const Share& x, bool keys, int step) {
        const int p = step / 4 / W, e = step / 4 % W;
        const uint32_t i = (p * NT + tid) * W, row = i / (HD / 8), word = i % (HD / 8) + e;
        if (step % (4 * W) == 0) {
            const _Float16 vd = __builtin_bit_cast(_Float16, x.vd[p]), poison = vd * (_Float16)0.0f;
            step_scale = keys ? __builtin_bit_cast(_Float16, x.kd[p]) + poison : poison == poison ? vd : (_Float16)0.0f;
        }
        dequantize_pair(x.w[p].w[e], h2{step_scale, step_scale}, step % 4, step % 4, step_hi, step_lo);
        if (step % 4 != 3) return;
        _Float16* const hi = keys ? &k_tile[buffer].h[0][row][8u * word] : &v_tile[buffer].h[0][row][8u * (word ^ VT::swizzle(row))];
        *reinterpret_cast<h8*>(hi) = step_hi, *reinterpret_cast<h8*>(hi + (keys ? KT * (HD + 8) : KT * HD)) = step_lo;
    };
    const auto store = [&](int buffer, const Share& x, bool keys) {
#pragma unroll
        for (int step = 0; step < kSteps; step++) store_step(buffer, x, keys, step);
    };
    // V^T rows (dims) 32 i + l32, keys 16 s + 8 u + 4 h ..: the 16 lanes of a group point at 4 keys x 16 dims, lane j at key j / 4 and dims
    // 4 (j % 4) .. of them, and the read hands every lane four keys of one dim.
    const uint32_t vkey = 32u * wk + 4u * h + (l16 >> 2), vpiece = 2u * (lane >> 4 & 1u) + (l16 >> 1 & 1u);
    const auto read_v = [&](int buffer, int plane, int i, int s) {
        typedef short s4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) s4* lds_s4;
        const _Float16* const p = &v_tile[buffer].h[plane][vkey][8u * ((4u * i + vpiece) ^ VT::swizzle(vkey)) + 4u * (l16 & 1u)] + 16 * s * HD;  // (keys 8 apart swizzle alike)
        const h4 a0 = __builtin_bit_cast(h4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)p));
        const h4 a1 = __builtin_bit_cast(h4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(p + 8 * HD)));
        return h8{a0[0], a0[1], a0[2], a0[3], a1[0], a1[1], a1[2], a1[3]};
    };

    Queries<HD> q;
    v16f o[DT];
#pragma unroll
    for (int i = 0; i < DT; i++)
#pragma unroll
        for (int e = 0; e < 16; e++) o[i][e] = 0.0f;
    float m_run = -__builtin_inff(), l_run = 0.0f, top;  // (top: of a row's scores of the tile at hand)
    // One tile's arithmetic, with the scores of the next tile (in the other buffer) and the unpacking of what is stored next in between: a wave's matrix
    // instructions run beside its vector instructions where they take turns in its program, so they do, in this very order.  (A wave that sees none of the tile's
    // keys goes along: the workgroup's barriers wait for the others anyway.)
    const auto attend = [&](int buffer, uint32_t t, v16f& sc, v16f& next, const Share& kraw, const Share& vraw) {
        const uint32_t key0 = t * KT + 32u * wk;
        if (key0 + 31u > wave_first) {  // some query row does not see all of the keys
#pragma unroll
            for (int e = 0; e < 16; e++)
                if (key0 + 8u * (e >> 2) + 4u * h + (e & 3) > mine) sc[e] = -__builtin_inff();
            top = sc[0];
#pragma unroll
            for (int e = 1; e < 16; e++) top = fmaxf(top, sc[e]);
            top = halves_max(top);
        }
        const _Float16* const keys = &k_tile[buffer ^ 1].h[0][32u * wk + l32][8 * h];  // (behind the last tile: whatever is there, for nobody)
        const auto key = [&](int plane, int s) { return *reinterpret_cast<const h8*>(keys + plane * (KT * (HD + 8)) + 16 * s); };
        // operands are read kAhead slabs (three matrix instructions each) before their use: as long as LDS takes to answer
        constexpr int kAhead = HD == 64 ? 3 : 2;
        h8 kl[SLABS], kh[SLABS], vl[2 * DT], vh[2 * DT];
#pragma unroll
        for (int s = 0; s < kAhead && s < SLABS; s++) kl[s] = key(1, s), kh[s] = key(0, s);
        const float m_new = fmaxf(m_run, top * q.factor), m_sub = m_new == -__builtin_inff() ? 0.0f : m_new;
        if (__builtin_amdgcn_ballot_w64(m_new > m_run) != 0) {  // else every factor is one (or acts on zeros)
            const float alpha = __builtin_amdgcn_exp2f(m_run - m_sub);
            m_run = m_new, l_run *= alpha;
#pragma unroll
            for (int i = 0; i < DT; i++) o[i] *= alpha;
        }
        const float shift = m_sub - kWeightBits;
        h4 hi[4], lo[4];
        v4f w[4];
        const auto softmax_step = [&](int step) {  // 12 of them: the exponentials of four weights two steps ahead of their split
            if (step % 3 == 0) {
#pragma unroll
                for (int i = 0; i < 4; i++) w[step / 3][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[4 * (step / 3) + i], q.factor, -shift));
            } else if (step % 3 == 1) {
                l_run += (w[step / 3][0] + w[step / 3][1]) + (w[step / 3][2] + w[step / 3][3]);
            } else {
                split_halves(w[step / 3], hi[step / 3], lo[step / 3]);
            }
        };
#pragma unroll
        for (int e = 0; e < 16; e++) next[e] = 0.0f;
#pragma unroll
        for (int i = 0; i < 3 * SLABS; i++) {
            const int s = i / 3, then = s + kAhead;
            if (i % 3 == 0) next = __builtin_amdgcn_mfma_f32_32x32x16_f16(kl[s], q.hi[s], next, 0, 0, 0);
            if (i % 3 == 1) next = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh[s], q.lo[s], next, 0, 0, 0);
            if (i % 3 == 2) next = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh[s], q.hi[s], next, 0, 0, 0);
            if (i % 3 == 0 && then < SLABS) kl[then] = key(1, then), kh[then] = key(0, then);
            if (i % 3 == 0 && then >= SLABS && then - SLABS < 2 * DT) vl[then - SLABS] = read_v(buffer, 1, (then - SLABS) % DT, (then - SLABS) / DT), vh[then - SLABS] = read_v(buffer, 0, (then - SLABS) % DT, (then - SLABS) / DT);
#pragma unroll
            for (int step = 12 * i / (3 * SLABS); step < 12 * (i + 1) / (3 * SLABS); step++) softmax_step(step);
            __builtin_amdgcn_sched_barrier(0);
        }
        const h8 ph[2] = {__builtin_shufflevector(hi[0], hi[1], 0, 1, 2, 3, 4, 5, 6, 7), __builtin_shufflevector(hi[2], hi[3], 0, 1, 2, 3, 4, 5, 6, 7)};
        const h8 pl[2] = {__builtin_shufflevector(lo[0], lo[1], 0, 1, 2, 3, 4, 5, 6, 7), __builtin_shufflevector(lo[2], lo[3], 0, 1, 2, 3, 4, 5, 6, 7)};
#pragma unroll
        for (int i = 0; i < 6 * DT; i++) {
            const int n = i / 3, d = n % DT, s = n / DT, then = n + kAhead;
            if (i % 3 == 0) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vl[n], ph[s], o[d], 0, 0, 0);
            if (i % 3 == 1) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vh[n], pl[s], o[d], 0, 0, 0);
            if (i % 3 == 2) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vh[n], ph[s], o[d], 0, 0, 0);
            if (i % 3 == 0 && then < 2 * DT) vl[then] = read_v(buffer, 1, then % DT, then / DT), vh[then] = read_v(buffer, 0, then % DT, then / DT);
#pragma unroll
            for (int step = 2 * kSteps * i / (6 * DT); step < 2 * kSteps * (i + 1) / (6 * DT); step++) {
                if (step < kSteps) store_step(buffer ^ 1, vraw, false, step);
                else store_step(buffer, kraw, true, step - kSteps);
            }
            if (i == 6 * DT - 2) {  // the next tile's maximum, if it needs no mask
                top = next[0];
#pragma unroll
                for (int e = 1; e < 16; e++) top = fmaxf(top, next[e]);
            }
            if (i == 6 * DT - 1) top = halves_max(top);
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    // While the arithmetic of tile t runs, the values of t and the keys of t + 1 sit in LDS; the values of t + 1 and the keys of t + 2 are in registers and
    // go where those of t - 1 and t were; behind them the next are requested.  (Requests past the end give zeros.)
    Share kraw, vraw;
    v16f sc[2];
    fetch(kraw, true);
    fetch(vraw, false);
    next_tile();
    {
        typename Queries<HD>::Raw raw;
        raw.request(a, r, c, group, h);
        q.take(raw, a.scale);
    }
    store(0, kraw, true);
    fetch(kraw, true);
    store(0, vraw, false);
    fetch(vraw, false);
    next_tile();
    store(1, kraw, true);
    fetch(kraw, true);
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 16; e++) sc[0][e] = 0.0f;
#pragma unroll
    for (int s = 0; s < SLABS; s++) {
        const h8 kh = *reinterpret_cast<const h8*>(&k_tile[0].h[0][32u * wk + l32][16 * s + 8 * h]), kl = *reinterpret_cast<const h8*>(&k_tile[0].h[1][32u * wk + l32][16 * s + 8 * h]);
        sc[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kl, q.hi[s], sc[0], 0, 0, 0);
        sc[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh, q.lo[s], sc[0], 0, 0, 0);
        sc[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh, q.hi[s], sc[0], 0, 0, 0);
    }
    top = sc[0][0];
#pragma unroll
    for (int e = 1; e < 16; e++) top = fmaxf(top, sc[0][e]);
    top = halves_max(top);
    __syncthreads();
    const auto tile = [&](int buffer, uint32_t t) {
        attend(buffer, t, sc[buffer], sc[buffer ^ 1], kraw, vraw);
        fetch(vraw, false);  // (of tile t + 2, and keys of t + 3)
        next_tile();
        fetch(kraw, true);
        __syncthreads();
    };
    for (uint32_t t = t_first;; t += 2u) {
        tile(0, t);
        if (t + 1u >= t_end) break;
        tile(1, t + 1u);
        if (t + 2u >= t_end) break;
    }

    l_run = halves_sum(l_run);
    if constexpr (WK > 1) {  // the waves of other keys hand their states to the first
        float* const state = reinterpret_cast<float*>(smem) + (size_t)wq * (WK - 1) * kStates * 64u + lane;
        if (wk != 0) {
            float* const to = state + (size_t)(wk - 1u) * kStates * 64u;
            to[0] = m_run, to[64] = l_run;
#pragma unroll
            for (int i = 0; i < DT; i++)
#pragma unroll
                for (int e = 0; e < 16; e++) to[(2 + 16 * i + e) * 64] = o[i][e];
        }
        __syncthreads();
        if (wk != 0) return;
        float m_all = m_run;
        for (int k = 0; k < WK - 1; k++) m_all = fmaxf(m_all, state[k * kStates * 64]);
        const float m_sub = m_all == -__builtin_inff() ? 0.0f : m_all;
        float f = __builtin_amdgcn_exp2f(m_run - m_sub);
        l_run *= f;
#pragma unroll
        for (int i = 0; i < DT; i++) o[i] *= f;
        for (int k = 0; k < WK - 1; k++) {
            const float* const from = state + k * kStates * 64;
            f = __builtin_amdgcn_exp2f(from[0] - m_sub);
            l_run = __builtin_fmaf(from[64], f, l_run);
#pragma unroll
            for (int i = 0; i < DT; i++)
#pragma unroll
                for (int e = 0; e < 16; e++) o[i][e] = __builtin_fmaf(from[(2 + 16 * i + e) * 64], f, o[i][e]);
        }
        m_run = m_all;
    }
    if (r0 + l32 >= rows) return;
    // register e of o[i] holds dim 32 i + 8 (e / 4) + 4 h + e % 4 of row l32
    const uint32_t token = r / group, head = c * group + r % group;
    float* to;
    float inverse = 1.0f;
    if (a.splits == 1u) {
        to = a.out + (size_t)token * a.out_stride + (size_t)head * HD;
        inverse = __fdiv_rn(1.0f, l_run);
        if (a.stats && h == 0) {
            float* const st = a.stats + 2u * ((size_t)token * a.n_heads + head);
            st[0] = m_run, st[1] = inverse;
        }
    } else {
        to = a.parts + (((size_t)token * a.n_heads + head) * a.splits + split) * (HD + 4);
        if (h == 0) to[0] = m_run, to[1] = l_run;
        to += 4;
    }
#pragma unroll
    for (int i = 0; i < DT; i++)
#pragma unroll
        for (int k = 0; k < 4; k++)
            *reinterpret_cast<v4f*>(to + 32 * i + 8 * k + 4 * h) = v4f{o[i][4 * k], o[i][4 * k + 1], o[i][4 * k + 2], o[i][4 * k + 3]} * inverse;
}

// The splits of a (token, head) merged, by G groups of HD / 4 lanes that share the splits among them (G = 1: no exchange, for launches of many rows).
// Everything is requested at once: a record's values do not wait for its maximum.
template <int HD, int G>
__device__ __forceinline__ void merge_splits(const Q4AttentionArgs& a, uint32_t wg_rows, uint32_t tile) {
    constexpr uint32_t Q = HD / 4, RPB = 256 / (Q * G), kBatch = 4;  // rows of a workgroup
    __shared__ __align__(16) v4f sums[G > 1 ? 256 : 1];
    __shared__ float2 states[G > 1 ? 256 / Q : 1];
    const uint32_t tid = threadIdx.x, d = tid % Q, grp = tid / Q % G, at = blockIdx.x * RPB + tid / (Q * G);
    if (G == 1 && at >= a.n * a.n_heads) return;  // (else a workgroup is whole: RPB divides, see the launch)
    const uint32_t token = at / a.n_heads, head = at % a.n_heads, group = a.n_heads / a.n_kv_heads, rows = a.n * group, r = token * group + head % group;
    const uint32_t used = used_splits(a.splits, sees(a, first_row(a), r / wg_rows * wg_rows + wg_rows - 1u, rows, group) / tile + 1u);
    const float* const parts = a.parts + (size_t)at * a.splits * (HD + 4);
    float m = -__builtin_inff(), l = 0.0f;
    v4f o = {0.f, 0.f, 0.f, 0.f};
    for (uint32_t i0 = grp; i0 < used; i0 += G * kBatch) {
        float2 ml[kBatch];
        v4f v[kBatch];
#pragma unroll
        for (uint32_t b = 0; b < kBatch; b++) {
            const float* const rec = parts + (size_t)min(i0 + b * G, used - 1u) * (HD + 4);
            ml[b] = *reinterpret_cast<const float2*>(rec), v[b] = *reinterpret_cast<const v4f*>(rec + 4 + 4 * d);
        }
        float top = m;
#pragma unroll
        for (uint32_t b = 0; b < kBatch; b++) top = fmaxf(top, ml[b].x);
        const float sub = top == -__builtin_inff() ? 0.0f : top, f = __builtin_amdgcn_exp2f(m - sub);
        l *= f, o *= f, m = top;
#pragma unroll
        for (uint32_t b = 0; b < kBatch; b++) {
            const float w = i0 + b * G < used ? __builtin_amdgcn_exp2f(ml[b].x - sub) : 0.0f;
            if (i0 + b * G < used) l = __builtin_fmaf(ml[b].y, w, l), o += v[b] * w;
        }
    }
    if constexpr (G > 1) {
        sums[tid] = o;
        if (d == 0) states[tid / Q] = make_float2(m, l);
        __syncthreads();
        if (grp != 0) return;
        float top = m;
#pragma unroll
        for (uint32_t i = 1; i < G; i++) top = fmaxf(top, states[tid / Q + i].x);
        const float sub = top == -__builtin_inff() ? 0.0f : top, f = __builtin_amdgcn_exp2f(m - sub);
        l *= f, o *= f, m = top;
#pragma unroll
        for (uint32_t i = 1; i < G; i++) {
            const float2 st = states[tid / Q + i];
            const float w = __builtin_amdgcn_exp2f(st.x - sub);
            l = __builtin_fmaf(st.y, w, l), o += sums[tid + i * Q] * w;
        }
    }
    const float inverse = __fdiv_rn(1.0f, l);
    if (a.stats && d == 0) a.stats[2u * at] = m, a.stats[2u * at + 1u] = inverse;
    *reinterpret_cast<v4f*>(a.out + (size_t)token * a.out_stride + (size_t)head * HD + 4u * d) = o * inverse;
}
template <int HD, int G>
__global__ __launch_bounds__(256) void attention_q4_merge_kernel(Q4AttentionArgs a, uint32_t wg_rows, uint32_t tile) {
    merge_splits<HD, G>(a, wg_rows, tile);
}

// ---- few query rows ----
// Up to 16 query rows of a KV head (the heads of one token, of a few tokens) per workgroup, and a part of the cache to each of its waves, 32 rows
// at a time, on v_mfma_f32_16x16x32_f16.  Nothing goes through LDS but the states at the end: a lane loads the words of a key row that it multiplies (lane
// group g HD / 32 of them from word g HD / 32 on, the order of an MFMA's K steps being free), and of the values one word of eight rows, the rows whose weights it
// holds: two rows' words are transposed to pairs of one dim's values with one byte permutation each.  Keys are multiplied as nibbles less 8, one exact half, a
// block's 32 dims at a time, and the block's scale is taken into the sum: two products of halves instead of three.
// Bound at long context by the loads and the unpacking, which overlap in part: one token of 32 heads over 8 of 128 behind 128000 rows (147 MB) 39 us, its
// loads alone 26; with values through LDS and both planes of the keys 45, and 42 before waves yielded (see below).  At short context by two or three round trips to memory: 16 heads over 9000 rows 7.2 us.
struct FewArgs {
    Q4AttentionArgs at;
    float* scores;  // [n_heads][max_seq], of one token's heads in powers of two, for the weights; may be null
};
constexpr uint32_t kFewRows = 16, kFewKeys = 32, kFewWaves = 4;
template <int HD>
constexpr uint32_t kFewSlots = kCus * (HD <= 128 ? 2 : 1);  // workgroups that the GPU has at once

// A wave with `left` of its steps to go yields to those of its SIMD that have more (of `longest` at the most): left to themselves, the oldest wave
// goes first, and when it has gone the last one's latencies are nobody's to hide (128000 rows: first waves done at 26 us, last at 41; so 33 and 40).
__device__ __forceinline__ void yield_to_longer(uint32_t left, uint32_t longest) {
    if (left > longest / 2u) __builtin_amdgcn_s_setprio(3);
    else if (left > longest / 4u) __builtin_amdgcn_s_setprio(2);
    else if (left > longest / 8u) __builtin_amdgcn_s_setprio(1);
    else __builtin_amdgcn_s_setprio(0);
}

template <int HD>
__global__ __launch_bounds__(64 * kFewWaves, HD == 32 ? 4 : HD <= 128 ? 2 : 1) void attention_q4_few_kernel(FewArgs args) {
    const Q4AttentionArgs& a = args.at;
    constexpr uint32_t kWaves = kFewWaves;
    constexpr int SLABS = HD / 32, CS = HD / 16, kStates = 2 + HD / 4, kLoad = SLABS < 4 ? SLABS : 4, kLoads = SLABS / kLoad;  // words a load, loads a row
    // a value row's words: lane l16 has word l16 % kOctets (and the one kOctets behind it), or as many dims of it as lanes do not share it
    constexpr int kOctets = HD < 128 ? HD / 8 : 16, kSharers = 16 / kOctets, kMine = HD / 8 / kOctets, kVd = 8 * kMine, kKd = HD == 32 ? 4 : HD / 16;
    __shared__ float smem[kStates * 64 * kWaves];
    const uint32_t group = a.n_heads / a.n_kv_heads, rows = a.n * group;
    const uint32_t c = blockIdx.x % a.n_kv_heads, split = blockIdx.x / a.n_kv_heads % a.splits, r0 = ((rows + kFewRows - 1u) / kFewRows - 1u - blockIdx.x / a.n_kv_heads / a.splits) * kFewRows;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, l16 = lane & 15u, g = lane >> 4, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tid >> 6));
    const uint32_t base = first_row(a), last = sees(a, base, r0 + kFewRows - 1u, rows, group), used = used_splits(a.splits, last / (kFewKeys * kWaves) + 1u);
    if (split >= used) return;
    const uint32_t units = last / kFewKeys + 1u, nth = split * kWaves + wave;
    const uint32_t u_first = (uint32_t)((uint64_t)units * nth / (used * kWaves)), u_end = (uint32_t)((uint64_t)units * (nth + 1u) / (used * kWaves));
    const uint32_t r = min(r0 + l16, rows - 1u), mine = sees(a, base, r, rows, group), first_sees = sees(a, base, r0, rows, group);
    const uint32_t token = r / group, head = c * group + r % group;
    const uint32_t octet = l16 % kOctets, sharer = l16 / kOctets;

    const Q4Cache kc = q4_planes(const_cast<void*>(a.k_cache), a.max_seq, a.n_kv_heads, HD), vc = q4_planes(const_cast<void*>(a.v_cache), a.max_seq, a.n_kv_heads, HD);
    const size_t first = (size_t)c * a.max_seq;
    const auto plane = [&](const void* p, uint32_t row_bytes) {  // (a read behind the last row gives zeros, whose weights the mask makes zeros)
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(static_cast<const uint8_t*>(p)) + first * row_bytes, 0, (int)((last + 1u) * row_bytes), 0x27000);
    };
    const auto kq = plane(kc.quants, HD / 2), vq = plane(vc.quants, HD / 2), ks = plane(kc.scales, HD / 16), vs = plane(vc.scales, HD / 16);
    struct Unit {
        struct __attribute__((aligned(4 * kLoad))) Words {
            uint32_t w[kLoad];
        };
        Words k[2][kLoads];  // of keys l16 and 16 + l16
        uint32_t kd[2][kKd];   // scales of all blocks of keys 4 g .. and 16 + 4 g .., one row behind the other
        uint32_t v[8][kMine];  // of values 4 g .. and 16 + 4 g ..
        uint32_t vd[kVd];      // and their scales: of the word's block (heads of 64 values: of both blocks)
    };
    const auto load = [&](decltype(kq) from, uint32_t at) {
        if constexpr (kLoad == 1) return __builtin_bit_cast(typename Unit::Words, __builtin_amdgcn_raw_buffer_load_b32(from, at, 0, 0));
        else if constexpr (kLoad == 2) return __builtin_bit_cast(typename Unit::Words, __builtin_amdgcn_raw_buffer_load_b64(from, at, 0, 0));
        else return __builtin_bit_cast(typename Unit::Words, __builtin_amdgcn_raw_buffer_load_b128(from, at, 0, 0));
    };
    const auto fetch = [&](uint32_t unit, Unit& x) {
#pragma unroll
        for (uint32_t u = 0; u < 2; u++)
#pragma unroll
            for (uint32_t i = 0; i < kLoads; i++) {
                const uint32_t row = unit * kFewKeys + 16u * u + l16, word = g * SLABS + i * kLoad;
                x.k[u][i] = load(kq, row * (HD / 2) + 4u * word);
            }
#pragma unroll
        for (uint32_t u = 0; u < 2; u++)
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) {
                const uint32_t at = (unit * kFewKeys + 16u * u + 4u * g) * (HD / 16);
                if constexpr (HD == 32) x.kd[u][i] = __builtin_amdgcn_raw_buffer_load_b16(ks, at + 2u * i, 0, 0);
                else if (i < kKd / 4) {
                    const auto d = __builtin_amdgcn_raw_buffer_load_b128(ks, at + 16u * i, 0, 0);
#pragma unroll
                    for (uint32_t j = 0; j < 4; j++) x.kd[u][4 * i + j] = d[j];
                }
            }
#pragma unroll
        for (uint32_t j = 0; j < 8; j++)
#pragma unroll
            for (uint32_t i = 0; i < kMine; i++) {
                const uint32_t row = unit * kFewKeys + 16u * (j / 4u) + 4u * g + j % 4u, word = octet + i * kOctets;
                x.v[j][i] = __builtin_amdgcn_raw_buffer_load_b32(vq, row * (HD / 2) + 4u * word, 0, 0);
                if constexpr (HD != 64) x.vd[j * kMine + i] = __builtin_amdgcn_raw_buffer_load_b16(vs, row * (HD / 16) + word / 4u * 2u, 0, 0);
            }
        if constexpr (HD == 64) {
#pragma unroll
            for (uint32_t u = 0; u < 2; u++) {
                const auto d = __builtin_amdgcn_raw_buffer_load_b128(vs, (unit * kFewKeys + 16u * u + 4u * g) * (HD / 16), 0, 0);
#pragma unroll
                for (uint32_t j = 0; j < 4; j++) x.vd[4 * u + j] = d[j];
            }
        }
    };
    // A lane's words of a key row to one of each block: blocks(w)[s] is word word_of(s) of the row, whatever lane had it.
    const auto word_of = [&](uint32_t s) { return HD == 32 ? g : HD == 64 ? 4u * s + 2u * (g & 1u) + (g >> 1) : HD == 128 ? 4u * s + g : 4u * (2u * (s & 3u) + (s >> 2)) + g; };
    const auto blocks = [&](const typename Unit::Words (&x)[kLoads], uint32_t (&w)[SLABS]) {
#pragma unroll
        for (int i = 0; i < kLoads; i++) {
#pragma unroll
            for (int j = 0; j < kLoad; j++) w[i * kLoad + j] = x[i].w[j];
            const auto exchange = [&](int j, int k, bool halves) {
                uint32_t &p = w[i * kLoad + j], &q = w[i * kLoad + k];
                const auto r = halves ? __builtin_amdgcn_permlane32_swap(p, q, false, false) : __builtin_amdgcn_permlane16_swap(p, q, false, false);
                p = r[0], q = r[1];
            };
            if constexpr (kLoad == 2) exchange(0, 1, true);
            if constexpr (kLoad == 4) exchange(0, 2, true), exchange(1, 3, true), exchange(0, 1, false), exchange(2, 3, false);
        }
    };
    Unit units_ahead[2];
    fetch(u_first, units_ahead[0]);

    // the query rows: dims 8 word_of(s) .. of row l16 in slab s, times 2^-e
    h8 qh[SLABS], ql[SLABS];
    float factor;
    {
        const float* const p = a.q + (size_t)token * a.q_stride + (size_t)head * HD;
        v4f x[2 * SLABS];
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < 2 * SLABS; i++) {
            x[i] = *reinterpret_cast<const v4f*>(p + 8u * word_of(i / 2) + 4 * (i % 2));
#pragma unroll
            for (int e = 0; e < 4; e++) top = fmaxf(top, fabsf(x[i][e]));
        }
        const int e = query_exponent(groups_max(top));
        factor = __builtin_amdgcn_ldexpf(a.scale * kLog2e, e);
#pragma unroll
        for (int s = 0; s < SLABS; s++) {
            h4 u[2], l[2];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                v4f y;
#pragma unroll
                for (int k = 0; k < 4; k++) y[k] = __builtin_amdgcn_ldexpf(x[2 * s + i][k], -e);
                split_halves(y, u[i], l[i]);
            }
            qh[s] = __builtin_shufflevector(u[0], u[1], 0, 1, 2, 3, 4, 5, 6, 7), ql[s] = __builtin_shufflevector(l[0], l[1], 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
    // bytes of two rows' words that make one: their lower halves or their upper ones, or one byte of each
    const uint32_t pick = kSharers == 1 ? 0x05040100u : kSharers == 2 ? (sharer ? 0x07060302u : 0x05040100u) : 0x0c040c00u + 0x00010001u * (2u * (sharer & 1u) + (sharer >> 1));
    const uint32_t pick_scale = octet < 4u ? 0x05040100u : 0x07060302u;
    v4f o[CS];
#pragma unroll
    for (int i = 0; i < CS; i++) o[i] = v4f{0.f, 0.f, 0.f, 0.f};
    float m_run = -__builtin_inff(), l_run = 0.0f;
    const auto attend = [&](uint32_t unit, Unit& now, Unit& then) {
        fetch(unit + 1u, then);  // (of the last one: for nobody)
        const uint32_t key0 = unit * kFewKeys;
        // Values that are not finite are taken as zeros and their keys as NaN (see attention_q4_kernel): seldom, and then by looking at their scales again.
        h2 vd[4][kMine], nan = {(_Float16)0.0f, (_Float16)0.0f};
        uint32_t first_bits[2] = {0x64006400u, 0x64006400u}, second_bits[2] = {0x54005400u, 0x54005400u};  // of the keys' nibbles; a NaN's
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int i = 0; i < kMine; i++) {
                uint32_t d;
                if constexpr (HD == 64) d = __builtin_amdgcn_perm(now.vd[2 * j + 1], now.vd[2 * j], pick_scale);
                else d = now.vd[(2 * j + 1) * kMine + i] << 16 | now.vd[2 * j * kMine + i];
                vd[j][i] = __builtin_bit_cast(h2, d);
                nan = __builtin_elementwise_fma(vd[j][i], h2{(_Float16)0.0f, (_Float16)0.0f}, nan);
            }
        if (__builtin_amdgcn_ballot_w64(nan[0] != nan[0] || nan[1] != nan[1]) != 0) {
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int i = 0; i < kMine; i++) {
                    const _Float16 d0 = vd[j][i][0], d1 = vd[j][i][1], zero = (_Float16)0.0f;
                    vd[j][i] = h2{d0 * zero == zero ? d0 : zero, d1 * zero == zero ? d1 : zero};
                }
#pragma unroll
            for (uint32_t u = 0; u < 2; u++)
#pragma unroll
                for (uint32_t i = 0; i < HD / 32; i++) {
                    const uint16_t d = __builtin_amdgcn_raw_buffer_load_b16(vs, (key0 + 16u * u + l16) * (HD / 16) + 2u * i, 0, 0);
                    if (__builtin_bit_cast(_Float16, d) * (_Float16)0.0f != (_Float16)0.0f) first_bits[u] = second_bits[u] = 0x7e007e00u;
                }
        }
        // A block's products of 16 keys: the nibbles unpacked one step ahead, between the matrix instructions (in this very order, in which no instruction waits for
        // the one before it), and scaled two steps behind.
        v4f sc[2], acc[3];
        uint32_t w[2][SLABS], n_bits[4];
        h8 k[2];
        blocks(now.k[0], w[0]), blocks(now.k[1], w[1]);
        const auto unpack = [&](int n) {
            uint32_t first = 0x000f000fu, second = 0x00f000f0u;
            asm("" : "+s"(first), "+s"(second));
            const uint32_t x = w[n % 2][n / 2], high = x >> 8, f = first_bits[n % 2], s = second_bits[n % 2];
            n_bits[0] = (x & first) | f, n_bits[1] = (x & second) | s, n_bits[2] = (high & first) | f, n_bits[3] = (high & second) | s;
        };
        const auto center = [&](int n) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const h2 x = __builtin_bit_cast(h2, n_bits[i]) - (i & 1 ? h2{(_Float16)72.0f, (_Float16)72.0f} : h2{(_Float16)1032.0f, (_Float16)1032.0f});
                k[n % 2][2 * i] = x[0], k[n % 2][2 * i + 1] = x[1];
            }
        };
        const auto scale = [&](int n) {
            const int u = n % 2, s = n / 2, block = HD == 256 ? 2 * (s & 3) + (s >> 2) : s;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float d = (float)__builtin_bit_cast(h2, now.kd[u][HD == 32 ? e : e * (HD / 64) + block / 2])[block & 1];
                sc[u][e] = s == 0 ? acc[n % 3][e] * d : __builtin_fmaf(acc[n % 3][e], d, sc[u][e]);
            }
        };
        unpack(0), center(0);
#pragma unroll
        for (int n = 0; n < 2 * SLABS + 2; n++) {
            if (n < 2 * SLABS) acc[n % 3] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[n % 2], ql[n / 2], v4f{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
            if (n + 1 < 2 * SLABS) unpack(n + 1);
            __builtin_amdgcn_sched_barrier(0);
            if (n >= 1 && n <= 2 * SLABS) acc[(n - 1) % 3] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[(n - 1) % 2], qh[(n - 1) / 2], acc[(n - 1) % 3], 0, 0, 0);
            if (n + 1 < 2 * SLABS) center(n + 1);
            if (n >= 2) scale(n - 2);
            __builtin_amdgcn_sched_barrier(0);
        }
        if (args.scores && r0 + l16 < rows) {
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const uint32_t key = key0 + 16u * u + 4u * g + e;
                    if (key <= mine) args.scores[(size_t)head * a.max_seq + key] = sc[u][e] * factor;
                }
        }
        if (key0 + kFewKeys - 1u > first_sees) {
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (key0 + 16u * u + 4u * g + e > mine) sc[u][e] = -__builtin_inff();
        }
        float top = -__builtin_inff();
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int e = 0; e < 4; e++) top = fmaxf(top, sc[u][e]);
        const float m_new = fmaxf(m_run, groups_max(top) * factor), m_sub = m_new == -__builtin_inff() ? 0.0f : m_new;
        if (__builtin_amdgcn_ballot_w64(m_new > m_run) != 0) {
            const float alpha = __builtin_amdgcn_exp2f(m_run - m_sub);
            m_run = m_new, l_run *= alpha;
#pragma unroll
            for (int i = 0; i < CS; i++) o[i] *= alpha;
        }
        const float shift = m_sub - kWeightBits;
        h4 hi[2], lo[2];
#pragma unroll
        for (int u = 0; u < 2; u++) {
            v4f w;
#pragma unroll
            for (int e = 0; e < 4; e++) w[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[u][e], factor, -shift));
            l_run += (w[0] + w[1]) + (w[2] + w[3]);
            split_halves(w, hi[u], lo[u]);
        }
        const h8 ph = __builtin_shufflevector(hi[0], hi[1], 0, 1, 2, 3, 4, 5, 6, 7), pl = __builtin_shufflevector(lo[0], lo[1], 0, 1, 2, 3, 4, 5, 6, 7);
        uint32_t pairs[4][kMine][kSharers == 1 ? 2 : 1];
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int i = 0; i < kMine; i++) {
                pairs[j][i][0] = __builtin_amdgcn_perm(now.v[2 * j + 1][i], now.v[2 * j][i], pick);
                if constexpr (kSharers == 1) pairs[j][i][1] = __builtin_amdgcn_perm(now.v[2 * j + 1][i], now.v[2 * j][i], 0x07060302u);
            }
        // (and the values, likewise)
        h2 x[4];
        h8 vh[2], vl[2];
        const auto unpack_values = [&](int d, int step) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int i = kSharers == 1 ? d / 2 % 4 : d, oct = kSharers == 1 ? d / 8 : 0;
                uint32_t mask = i & 1 ? 0x00f000f0u : 0x000f000fu, bits = i & 1 ? 0x54005400u : 0x64006400u;
                asm("" : "+s"(mask), "+v"(bits));
                const uint32_t p = pairs[j][oct][kSharers == 1 ? d & 1 : 0];
                if (step == 0) x[j] = __builtin_bit_cast(h2, ((i < 2 ? p : p >> 8) & mask) | bits);
                if (step == 1) x[j] -= i & 1 ? h2{(_Float16)72.0f, (_Float16)72.0f} : h2{(_Float16)1032.0f, (_Float16)1032.0f};
                if (step == 2) {
                    const h2 h = x[j] * vd[j][oct];
                    vh[d % 2][2 * j] = h[0], vh[d % 2][2 * j + 1] = h[1];
                }
                if (step == 3) {
                    const h2 l = __builtin_elementwise_fma(x[j], vd[j][oct], h2{-vh[d % 2][2 * j], -vh[d % 2][2 * j + 1]});
                    vl[d % 2][2 * j] = l[0], vl[d % 2][2 * j + 1] = l[1];
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        };
#pragma unroll
        for (int step = 0; step < 4; step++) unpack_values(0, step);
#pragma unroll
        for (int d = 0; d < CS; d++) {
            o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vl[d % 2], ph, o[d], 0, 0, 0);
            if (d + 1 < CS) unpack_values(d + 1, 0);
            o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh[d % 2], pl, o[d], 0, 0, 0);
            if (d + 1 < CS) unpack_values(d + 1, 1), unpack_values(d + 1, 2);
            o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh[d % 2], ph, o[d], 0, 0, 0);
            if (d + 1 < CS) unpack_values(d + 1, 3);
        }
    };
    const uint32_t mine_in_all = u_end - u_first;
    for (uint32_t unit = u_first; unit < u_end; unit += 2u) {
        yield_to_longer(u_end - unit, mine_in_all);
        attend(unit, units_ahead[0], units_ahead[1]);
        if (unit + 1u >= u_end) break;
        attend(unit + 1u, units_ahead[1], units_ahead[0]);
    }
    l_run = groups_sum(l_run);
    // The waves' states side by side, then every wave merges its share of the values: those of MFMA row 4 g + wave.
    static_assert(kWaves == 4, "an element of a lane's vectors each");
    float* const states = smem + lane;
    {
        float* const to = states + wave * (kStates * 64u);
        to[0] = m_run, to[64] = l_run;
#pragma unroll
        for (int i = 0; i < CS; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) to[(2 + 4 * i + e) * 64] = o[i][e];
    }
    __syncthreads();
    if (r0 + l16 >= rows) return;
    float m = -__builtin_inff(), l = 0.0f, sums[CS];
#pragma unroll
    for (uint32_t k = 0; k < kWaves; k++) m = fmaxf(m, states[k * (kStates * 64u)]);
    const float m_sub = m == -__builtin_inff() ? 0.0f : m;
#pragma unroll
    for (int i = 0; i < CS; i++) sums[i] = 0.0f;
#pragma unroll
    for (uint32_t k = 0; k < kWaves; k++) {
        const float* const from = states + k * (kStates * 64u);
        const float f = __builtin_amdgcn_exp2f(from[0] - m_sub);
        l = __builtin_fmaf(from[64], f, l);
#pragma unroll
        for (int i = 0; i < CS; i++) sums[i] = __builtin_fmaf(from[(2 + 4 * i + wave) * 64u], f, sums[i]);
    }
    float* to;
    float inverse = 1.0f;
    if (a.splits == 1u && !args.scores) {
        to = a.out + (size_t)token * a.out_stride + (size_t)head * HD;
        inverse = __fdiv_rn(1.0f, l);
        if (a.stats && g == 0 && wave == 0) {
            float* const st = a.stats + 2u * ((size_t)token * a.n_heads + head);
            st[0] = m, st[1] = inverse;
        }
    } else {
        to = a.parts + (((size_t)token * a.n_heads + head) * a.splits + split) * (HD + 4);
        if (g == 0 && wave == 0) to[0] = m, to[1] = l;
        to += 4;
    }
    const uint32_t m_row = 4u * g + wave, first_dim = 8u * (m_row % kOctets) + (kSharers == 1 ? 0u : m_row / kOctets % 2u + 4u * (m_row / kOctets / 2u));
#pragma unroll
    for (int i = 0; i < CS; i++) to[first_dim + (kSharers == 1 ? 8 * kOctets * (i / 8) + i % 8 : 2 * i)] = sums[i] * inverse;
}

// One token's splits merged and, in workgroups of their own, its weights added to what the rows have gathered: from the scores that the launch before left, with
// each head's maximum and sum worked out from its splits once more.  (9001 rows of 16 heads 3.4 us: a launch and two round trips.)
template <int HD>
__global__ __launch_bounds__(256) void attention_q4_finish_kernel(FewArgs args) {
    const Q4AttentionArgs& a = args.at;
    if (blockIdx.x < a.n_heads) return merge_splits<HD, 1024 / HD>(a, kFewRows, kFewKeys * kFewWaves);
    const uint32_t group = a.n_heads / a.n_kv_heads, nth = blockIdx.x - a.n_heads, c = nth % a.n_kv_heads, t = nth / a.n_kv_heads * 256u + threadIdx.x, lane = threadIdx.x & 63u;
    const uint32_t last = first_row(a), used = used_splits(a.splits, last / (kFewKeys * kFewWaves) + 1u);
    if (t - threadIdx.x > last) return;
    constexpr uint32_t kPerLane = (kMaxSplits + 63u) / 64u;
    const uint32_t at = min(t, last);
    float sum = 0.0f;
    for (uint32_t h = c * group; h < (c + 1u) * group; h++) {
        const float* const parts = a.parts + (size_t)h * a.splits * (HD + 4);
        const float score = args.scores[(size_t)h * a.max_seq + at];
        float m_i[kPerLane], l_i[kPerLane], top = -__builtin_inff(), l = 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < kPerLane; i++) {
            const uint32_t nth_split = lane + 64u * i;
            m_i[i] = nth_split < used ? parts[(size_t)nth_split * (HD + 4)] : -__builtin_inff(), l_i[i] = nth_split < used ? parts[(size_t)nth_split * (HD + 4) + 1] : 0.0f;
            top = fmaxf(top, m_i[i]);
        }
        const float m = wave_max_f32(top), m_sub = m == -__builtin_inff() ? 0.0f : m;
#pragma unroll
        for (uint32_t i = 0; i < kPerLane; i++) l = __builtin_fmaf(l_i[i], __builtin_amdgcn_exp2f(m_i[i] - m_sub), l);
        l = wave_sum_f32(l);
        sum += __fdiv_rn(__builtin_amdgcn_exp2f(score - m_sub + kWeightBits), l);
    }
    if (t <= last) a.weights[(size_t)c * a.max_seq + t] += sum;
}

// What rows of a KV head have gathered over a prompt: the scores once more, now that every softmax's maximum and sum is known, and their weights added
// up over the query rows.  Every wave keeps 32 keys as matrix operands in registers; the workgroup walks query rows in blocks of 32 that it splits into
// halves once for its four waves, through LDS, the next block's on their way meanwhile.  The rows are shared out among `shares` workgroups, whose sums the next launch adds.
// All sums in one order.  Bound by vector instructions (exponentials, and the queries' split: a block is split in every workgroup that sees it) and, for few
// rows, by latency: 555 tokens of 16 heads over 8 of 64 8.0 and 3.0 us for the addition, 1500 of 32 heads 26, 4000 of them 138, 500 of 16 over 4 of 128 9.5 (keys
// in LDS, the queries split by every wave for itself: 12.7, 54, 257 and 37).  128 keys a workgroup: with 256 and eight waves behind one barrier 9.9, 38, 190 and 17.  Workgroups with fewer
// blocks to go yield (834 tokens behind 3353, 24 heads over 3 of 64: 44.8 -> 41.2).
struct WeightArgs {
    Q4AttentionArgs at;
    float* sums;  // [shares][n_kv_heads][stride], unless there is one share
    uint32_t shares, stride;
};
constexpr uint32_t kWeightKeys = 128, kMaxShares = 16;  // (one KV head of 64 values: 256 of 1024 places over 2048 rows; other limits were not measured)
template <int HD>
constexpr uint32_t kWeightSlots = kCus * (HD <= 64 ? 4 : HD == 128 ? 3 : 2);  // workgroups that the GPU has at once
constexpr uint32_t kWeightSums = 4 * kCus * kWeightKeys;  // that the shares of a launch have room for

template <int HD>
__global__ __launch_bounds__(256, kWeightSlots<HD> / kCus) void attention_q4_weights_kernel(WeightArgs args) {
    const Q4AttentionArgs& a = args.at;
    const uint32_t shares = args.shares;
    constexpr int SLABS = HD / 16, V = HD / 32;  // four values, of a thread's share of a query row
    struct Block {
        _Float16 q[2][32][HD + 8];
        v4f row[32];  // {factor, shift, 1 / sum, -}
    };
    __shared__ __align__(16) Block blocks[2];
    const uint32_t c = blockIdx.x % a.n_kv_heads, share = blockIdx.x / a.n_kv_heads % shares, key0 = blockIdx.x / a.n_kv_heads / shares * kWeightKeys;
    const uint32_t group = a.n_heads / a.n_kv_heads, rows = a.n * group;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, l32 = lane & 31u, h = lane >> 5, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tid >> 6));
    const uint32_t base = first_row(a), last = sees(a, base, rows - 1u, rows, group);
    if (key0 > last) return;
    const uint32_t r_first = key0 > base ? (key0 - base) * group / 32u : 0u, r_end = (rows + 31u) / 32u;  // blocks; rows in front see none of the keys
    const uint32_t b_first = r_first + (uint32_t)((uint64_t)(r_end - r_first) * share / shares), b_end = r_first + (uint32_t)((uint64_t)(r_end - r_first) * (share + 1u) / shares);

    // this thread's share of a block of query rows: V times four values, 32 apart, of row tid / 8
    const uint32_t q_row = tid >> 3, q_at = 4u * (tid & 7u);
    struct {
        v4f x[V];
        float2 stat;
    } raw;
    // (its token and head one block after the other, without a division)
    uint32_t token = (32u * b_first + q_row) / group, of_group = (32u * b_first + q_row) % group;
    const uint32_t tokens_on = 32u / group, rows_on = 32u % group;
    const auto request = [&] {  // (of rows past the last: the last one's, for nobody)
        const uint32_t at = min(token, a.n - 1u), head = c * group + (token < a.n ? of_group : group - 1u);
        token += tokens_on, of_group += rows_on;
        if (of_group >= group) of_group -= group, token++;
        const float* const p = a.q + (size_t)at * a.q_stride + (size_t)head * HD + q_at;
#pragma unroll
        for (int i = 0; i < V; i++) raw.x[i] = *reinterpret_cast<const v4f*>(p + 32 * i);
        raw.stat = *reinterpret_cast<const float2*>(a.stats + 2u * ((size_t)at * a.n_heads + head));
    };
    const auto store = [&](Block& to, uint32_t b) {
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < V; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) top = fmaxf(top, fabsf(raw.x[i][e]));
        const int e = query_exponent(group_max8(top));
#pragma unroll
        for (int i = 0; i < V; i++) {
            v4f y;
            h4 hi, lo;
#pragma unroll
            for (int k = 0; k < 4; k++) y[k] = __builtin_amdgcn_ldexpf(raw.x[i][k], -e);
            split_halves(y, hi, lo);
            *reinterpret_cast<h4*>(&to.q[0][q_row][q_at + 32 * i]) = hi, *reinterpret_cast<h4*>(&to.q[1][q_row][q_at + 32 * i]) = lo;
        }
        if ((tid & 7u) == 0)
            to.row[q_row] = v4f{__builtin_amdgcn_ldexpf(a.scale * kLog2e, e), (raw.stat.x == -__builtin_inff() ? 0.0f : raw.stat.x) - kWeightBits,
                                32u * b + q_row < rows ? raw.stat.y : 0.0f, 0.0f};
    };
    if (b_first < b_end) request();
    // this lane's key, dims 16 s + 8 h ..
    h8 kh[SLABS], kl[SLABS];
    const uint32_t first_key = key0 + 32u * wave;
    {
        const Q4Cache kc = q4_planes(const_cast<void*>(a.k_cache), a.max_seq, a.n_kv_heads, HD), vc = q4_planes(const_cast<void*>(a.v_cache), a.max_seq, a.n_kv_heads, HD);
        const size_t at = (size_t)c * a.max_seq + min(first_key + l32, last);
        _Float16 poison = (_Float16)0.0f;  // (as its token's sum has it)
#pragma unroll
        for (int i = 0; i < HD / 32; i++) poison += __builtin_bit_cast(_Float16, vc.scales[at * (HD / 32) + i]) * (_Float16)0.0f;
#pragma unroll
        for (int s = 0; s < SLABS; s++)
            dequantize(kc.quants[at * (HD / 8) + 2u * s + h], __builtin_bit_cast(_Float16, kc.scales[at * (HD / 32) + s / 2]) + poison, kh[s], kl[s]);
    }
    const uint32_t b_all = first_key + 31u > base ? (uint32_t)(((uint64_t)(first_key + 31u - base) * group + 31u) / 32u) : 0u;  // from there on rows see all of the wave's keys
    float acc[16];
#pragma unroll
    for (int e = 0; e < 16; e++) acc[e] = 0.0f;
    if (b_first < b_end) {
        store(blocks[0], b_first);
        if (b_first + 1u < b_end) request();
        __syncthreads();
        const auto add = [&](uint32_t b, const Block& now, Block& then) {
            const v4f row = now.row[l32];
            v16f sc;
#pragma unroll
            for (int e = 0; e < 16; e++) sc[e] = 0.0f;
#pragma unroll
            for (int s = 0; s < SLABS; s++) {
                const h8 qh = *reinterpret_cast<const h8*>(&now.q[0][l32][16 * s + 8 * h]), ql = *reinterpret_cast<const h8*>(&now.q[1][l32][16 * s + 8 * h]);
                sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(kl[s], qh, sc, 0, 0, 0);
                sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh[s], ql, sc, 0, 0, 0);
                sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh[s], qh, sc, 0, 0, 0);
            }
            if (b + 1u < b_end) store(then, b + 1u);
            if (b + 2u < b_end) request();
            if (b < b_all) {  // some query row does not see all of the keys
                const uint32_t mine = sees(a, base, 32u * b + l32, rows, group);
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[e], row[0], -row[1])) * row[2];
                    acc[e] += first_key + 8u * (e >> 2) + 4u * h + (e & 3) > mine ? 0.0f : w;
                }
            } else {
#pragma unroll
                for (int e = 0; e < 16; e++) acc[e] = __builtin_fmaf(__builtin_amdgcn_exp2f(__builtin_fmaf(sc[e], row[0], -row[1])), row[2], acc[e]);
            }
            __syncthreads();
        };
        for (uint32_t b = b_first; b < b_end; b += 2u) {
            yield_to_longer(b_end - b, r_end / shares);
            add(b, blocks[0], blocks[1]);
            if (b + 1u >= b_end) break;
            add(b + 1u, blocks[1], blocks[0]);
        }
    }
    float* const to = shares == 1u ? a.weights + (size_t)c * a.max_seq : args.sums + (size_t)(share * a.n_kv_heads + c) * args.stride;
#pragma unroll
    for (int e = 0; e < 16; e++) {
        const float w = group_sum<32>(acc[e]);
        const uint32_t key = first_key + 8u * (e >> 2) + 4u * h + (e & 3);
        if (l32 == 0 && key <= last) {
            if (shares == 1u) to[key] += w;
            else to[key] = w;
        }
    }
}
__global__ __launch_bounds__(256) void attention_q4_add_weights_kernel(WeightArgs args) {
    const Q4AttentionArgs& a = args.at;
    const uint32_t shares = args.shares;
    const uint32_t c = blockIdx.y, t = blockIdx.x * 256u + threadIdx.x, group = a.n_heads / a.n_kv_heads, rows = a.n * group;
    if (t > sees(a, first_row(a), rows - 1u, rows, group)) return;
    float w = 0.0f;
    for (uint32_t i0 = 0; i0 < shares; i0 += 8u) {
        float x[8];
#pragma unroll
        for (uint32_t i = 0; i < 8u; i++) x[i] = args.sums[(size_t)(min(i0 + i, shares - 1u) * a.n_kv_heads + c) * args.stride + t];
#pragma unroll
        for (uint32_t i = 0; i < 8u; i++) w += i0 + i < shares ? x[i] : 0.0f;
    }
    a.weights[(size_t)c * a.max_seq + t] += w;
}

// As many splits as there are records for, each split leaving one to every row (`rows` in all) in the scratch, or one: whatever a launcher asks for, what it gets fits
// what part_floats() sizes.
uint32_t splits_with_records(uint32_t splits, uint64_t rows) { return (uint32_t)std::max<uint64_t>(std::min<uint64_t>({splits, kMaxSplits, kMostRecords / rows}), 1u); }

// Up to `few` splits are merged by HD / 4 lanes a row, more by a workgroup a row (us with what is before it, the second and the first: 60 tokens of 32 heads
// of 64 values behind 2500 in four splits 15.8 and 14.7, 120 behind 5000 in two 35.2 and 32.3, 30 behind 2500 in eight 12.0 and 12.7).
template <int HD>
hipError_t launch_merge(const Q4AttentionArgs& a, uint32_t wg_rows, uint32_t tile, uint32_t few, const Launch& L) {
    constexpr uint32_t kRows = 1024 / HD;  // of a workgroup, HD / 4 lanes each
    const uint32_t rows = a.n * a.n_heads;
    return a.splits > few ? launch_kernel(L, kFamOther, attention_q4_merge_kernel<HD, 1024 / HD>, dim3(rows), dim3(256), a, wg_rows, tile)
                          : launch_kernel(L, kFamOther, attention_q4_merge_kernel<HD, 1>, dim3((rows + kRows - 1u) / kRows), dim3(256), a, wg_rows, tile);
}

// Large launches: as many splits as workgroups fit on the GPU (kMaxSplits at the most), three tiles or more each (a split's state is written and read again).
template <int HD, int WQ, int WK, int PER_CU>
hipError_t launch_tiles(Q4AttentionArgs a, uint64_t seen, const Launch& L) {
    constexpr uint32_t RB = 32 * WQ, KT = 32 * WK;
    static_assert(PER_CU * kCus <= kSplitSlots && RB <= kMostRows, "there are records for all splits that fit on the GPU");
    const uint32_t rows = a.n * (a.n_heads / a.n_kv_heads), blocks = (rows + RB - 1u) / RB, base = a.n_kv_heads * blocks;
    const uint32_t room = kCus * PER_CU / base, most = (uint32_t)((seen + 3u * KT - 1u) / (3u * KT));
    a.splits = splits_with_records(std::min(room, most), (uint64_t)a.n * a.n_heads);
    const uint32_t per_block = a.n_kv_heads * a.splits;
    a.first_blocks = base * a.splits > kCus && base * a.splits <= 2u * kCus ? (kCus + per_block - 1u) / per_block : blocks;
    const hipError_t e = launch_kernel(L, kFamOther, attention_q4_kernel<HD, WQ, WK, PER_CU>, dim3(base * a.splits), dim3(64 * WQ * WK), a);
    if (e != hipSuccess || a.splits == 1u) return e;
    return launch_merge<HD>(a, RB, KT, 8, L);
}

// Small ones: workgroups of 16 query rows and as many splits as fill the GPU, but no more than kMaxSplits, down to a unit of keys for each wave; but none where walking some more units one
// behind the other takes less than the merge, which takes the longer the more rows there are (us, split and alone, 32 heads over 8; of 64 values: a token over
// 512 rows 6.9 and 6.0, 768 7.1 and 7.4; 30 tokens behind 900 10.0 and 9.4, 1300 11.3 and 11.6; 60 behind 1300 13.3 and 11.8, 2500 15.8 and 18.4; 120 behind
// 600 15.3 and 8.2, 2500 24.1 and 19.9; of 128: a token over 256 7.7 and 6.0, 512 7.7 and 8.3; 60 behind 800 15.6 and 13.3, 1800 19.9 and 23.6; of 256: 25 behind
// 300 13.7 and 14.5).
template <int HD>
hipError_t launch_few(FewArgs f, uint64_t seen, const Launch& L) {
    const Q4AttentionArgs& a = f.at;
    constexpr uint32_t kSpan = kFewKeys * kFewWaves;
    static_assert(kFewSlots<HD> * kFewRows <= kMostRecords, "there are records for all splits that fit on the GPU");
    const uint32_t rows = a.n * (a.n_heads / a.n_kv_heads), base = a.n_kv_heads * ((rows + kFewRows - 1u) / kFewRows);
    const uint32_t spans = (uint32_t)((seen + kSpan - 1u) / kSpan);
    const uint32_t alone = HD <= 64 ? std::max(5u, 3u + base / 12u) : HD == 128 ? std::max(3u, 1u + base / 12u) : std::max(1u, base / 24u);
    f.at.splits = spans <= alone && !f.scores ? 1u : splits_with_records(std::min(kFewSlots<HD> / base, spans), (uint64_t)a.n * a.n_heads);
    const hipError_t e = launch_kernel(L, kFamOther, attention_q4_few_kernel<HD>, dim3(base * a.splits), dim3(64 * kFewWaves), f);
    if (e != hipSuccess) return e;
    if (f.scores) return launch_kernel(L, kFamOther, attention_q4_finish_kernel<HD>, dim3(a.n_heads + a.n_kv_heads * (uint32_t)((seen + 255u) / 256u)), dim3(256), f);
    return a.splits == 1u ? e : launch_merge<HD>(a, kFewRows, kSpan, HD == 256 ? 8u : 4u, L);
}

// Which kernel: the one for few rows wastes nothing on them and fills the GPU with little work, the tiled one reads and unpacks the cache for up to eight
// times as many rows at once.  Up to 64 rows of a KV head the first is as fast or faster at any length (us: 32 query heads of 64 values over 8 KV heads,
// 32 rows behind 100000 41 against 78, 64 behind 60000 47 and 54, 96 behind 60000 69 and 56; of 32 values over 4, 64 behind 60000 24 and 21), with more
// rows up to some 12 million pairs of a query and a key: of 64 values, 555 tokens of 16 heads 9.7 and 17.0, 1500 of 6 16.8 and 24.0, 1000 of 32 30.1 and
// 28.8, 2002 of 32 89 and 63; of 32 values, 1400 of 16 20.0 and 19.6; of 128, 1000 of 8 18.4 and 30.0, 1000 of 32 50.1 and 47.8; of 256, 500 of
// 8 behind 500 30 and 42, 1000 of 8 behind 1000 84 and 81.
template <int HD>
hipError_t launch_head_dim(const Q4AttentionArgs& a, float* d_scores, const Launch& L) {
    const uint32_t rows = a.n * (a.n_heads / a.n_kv_heads);
    const uint64_t seen = a.d_pos ? a.max_seq : (uint64_t)a.pos0 + a.n, pairs = (uint64_t)a.n * a.n_heads * (seen - a.n / 2u);
    hipError_t e;
    if (rows <= 64u || pairs <= 12u << 20) {
        float* const scores = a.n == 1u && a.weights ? d_scores : nullptr;
        e = launch_few<HD>(FewArgs{a, scores}, seen, L);
        if (scores) return e;
    } else if constexpr (HD == 32) {
        e = launch_tiles<HD, 2, 2, 2>(a, seen, L);
    } else if constexpr (HD <= 128) {
        // Where every CU has a block of rows of its own, two workgroups of half the keys a CU (2048 tokens behind 6144 of 16 heads of 128 values 332 us
        // against 345, 4000 tokens of 32 heads of 64 values 210 against 230), else one (500 behind 2000 of those 43 against 44).
        const bool many = a.n_kv_heads * ((rows + 127u) / 128u) >= kCus;
        e = many ? launch_tiles<HD, 4, 1, 2>(a, seen, L) : launch_tiles<HD, 4, 2, 1>(a, seen, L);
    } else {
        e = launch_tiles<HD, 4, 1, 1>(a, seen, L);
    }
    if (e != hipSuccess || !a.weights) return e;
    const uint32_t tiles = (uint32_t)((seen + kWeightKeys - 1u) / kWeightKeys), base = a.n_kv_heads * tiles, blocks = (rows + 31u) / 32u;
    const uint32_t room = std::min(kWeightSlots<HD>, kWeightSums / kWeightKeys) / base;  // (with one share nothing is left in the scratch)
    const WeightArgs w{a, d_scores, std::max(std::min({room, kMaxShares, (blocks + 1u) / 2u}), 1u), tiles * kWeightKeys};
    e = launch_kernel(L, kFamOther, attention_q4_weights_kernel<HD>, dim3(base * w.shares), dim3(256), w);
    if (e != hipSuccess || w.shares == 1u) return e;
    return launch_kernel(L, kFamOther, attention_q4_add_weights_kernel, dim3((uint32_t)((seen + 255u) / 256u), a.n_kv_heads), dim3(256), w);
}

// Floats of the splits' records: what a split launch has at most, for any number of tokens up to n, and a token's that gathers weights (which leaves its
// only split as one, however many its heads).
size_t part_floats(uint32_t n, uint32_t n_heads, uint32_t head_dim) {
    const size_t rows = (size_t)n * n_heads;
    return std::max(std::min(rows * kMaxSplits, (size_t)kMostRecords), (size_t)n_heads) * (head_dim + 4u);
}

}  // namespace

size_t attention_q4_scratch_floats(uint32_t n, uint32_t max_seq, uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim, bool weights) {
    // records, statistics, a token's scores or the shares of a prompt's weights
    return part_floats(n, n_heads, head_dim) + (weights ? 2 * (size_t)n * n_heads + std::max((size_t)n_heads * max_seq, (size_t)kWeightSums) : 0);
}

hipError_t launch_attention_q4(const float* d_q, uint32_t q_stride, const void* d_k_cache, const void* d_v_cache, float* d_out, uint32_t out_stride,
                               float* d_weights, float* d_scratch, uint32_t pos0, const uint32_t* d_pos, uint32_t n, uint32_t max_seq, uint32_t n_heads,
                               uint32_t n_kv_heads, uint32_t head_dim, float scale, const Launch& L) {
    if (n == 0) return hipSuccess;
    float *const d_stats = d_scratch + part_floats(n, n_heads, head_dim), *const d_scores = d_stats + 2 * (size_t)n * n_heads;
    const Q4AttentionArgs a{d_q, d_k_cache, d_v_cache, d_out, d_scratch, d_weights ? d_stats : nullptr, d_weights, d_pos,
                            pos0, n, q_stride, out_stride, max_seq, n_heads, n_kv_heads, 1, 0, scale};
    switch (head_dim) {
        case 32: return launch_head_dim<32>(a, d_scores, L);
        case 64: return launch_head_dim<64>(a, d_scores, L);
        case 128: return launch_head_dim<128>(a, d_scores, L);
        default: return launch_head_dim<256>(a, d_scores, L);
    }
}

}  // namespace wick_rocm
