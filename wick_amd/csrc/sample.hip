// Sampling: a row's next token by temperature, top-k, top-p and min-p from a given uniform number.
//
// With y_i = l_i log2(e) / T, rounded to f64, and E the whole number below the largest, token i weighs W_i = 2^(y_i - E) in whole numbers of 2^-43: masses are
// whole numbers, whose sums are the same in every order.  Both cuts are cuts in the order of (logit, lower index first), a 64-bit key of which no two are
// alike, so what is wanted is one threshold key; and a token's weight follows from its key.  Bins are a quarter of a power of two wide, counted from E down.
//   1. parts of a row on workgroups of their own: histogram of the part's tokens and masses over the bins, relative to the part's own E;
//   2. the same parts: the row's histogram (the parts', shifted) says in which bins the cuts can be; the part lists its tokens there, and adds up what is
//      certainly kept;
//   3. one workgroup a row: the cuts exactly, from the listed tokens; the mass of every part; the part in which the pick is, token by token.
// Where top-k leaves few, tokens are only counted in 1., and all that may be taken are listed: no weights but theirs.  What is listed is at most some hundred
// tokens as a rule, which 3. sorts, and a row's all in the worst case (all logits alike), for which there is room.
//
// Three dependent launches bound a single row (65536 tokens, top-k 40: 4.3, 7.8 and 4.7 us, each a chain of round trips); f64 arithmetic, of which every weight takes some
// twenty instructions, many (64 rows of 65536 under top-p: 9.4, 12.6 and 11.6 us; reading them alone would take 3.5).  65536 tokens that are all alike take 0.38 ms,
// 0.41 in 64 rows: passes over a long list.
#include <algorithm>
#include <type_traits>

#include "wick_rocm_device.h"
#include "wick_rocm_internal.h"

namespace wick_rocm {

namespace {

constexpr uint32_t kPart = 4096, kMaxParts = kSampleMaxTokens / kPart;  // tokens of a part
constexpr int kOctaves = 46, kSteps = 4;                                // bins: kSteps to a power of two
constexpr uint32_t kBins = kOctaves * kSteps, kLaneBins = 3;            // every wave has them all, three a lane
static_assert(kBins <= 64 * kLaneBins && kMaxParts <= 128);
constexpr uint32_t kFew = 512; // top-k up to which all that it leaves is listed: 3. sorts up to 1024 tokens, and the last bin may be half of them
constexpr double kLog2e = 1.4426950408889634;
constexpr double kInfinite4 = 0x1p1000;                                 // 4 y of an infinite logit

struct SamplePart {
    uint64_t sure;  // mass that is certainly kept
    float largest;  // logit
    uint32_t listed;
    uint64_t mass[kBins];
    uint32_t count[kBins];
};

// What 2. knows of a row and hands on to 3.: every bin's tokens and mass with those in front of it, and where the cuts can be.
struct SampleRow {
    double top4, floor;  // 4 E; the mass that min-p asks for
    uint32_t k_bin, p_first, p_last, pad;
    uint64_t mass[64 * kLaneBins];
    uint32_t count[64 * kLaneBins];
};

struct SampleArgs {
    const float* logits;
    const wick_rocm_sample_params* params;
    const float* uniform;
    uint32_t* out;
    float* prob;
    SampleRow* rows;
    SamplePart* parts;  // [rows][n_parts]
    uint64_t* lists;    // [rows][n] keys: part p's tokens from p kPart on
    uint32_t n, stride, n_parts;
};

struct Rule {
    double inverse4;  // 4 log2(e) / T
    uint32_t top_k;
    double top_p, min_p;
    uint32_t n;
    __device__ __forceinline__ bool few() const { return top_k <= kFew; }
    __device__ __forceinline__ bool masses() const { return top_p < 1.0 && !few(); }  // 1. adds up masses,
    __device__ __forceinline__ bool counts() const { return top_k < n || few(); }     // counts tokens
};
__device__ __forceinline__ Rule rule_of(const SampleArgs& a, uint32_t row) {
    const wick_rocm_sample_params p = a.params[row];
    Rule r{kSteps * kLog2e, p.top_k == 0 ? a.n : min(p.top_k, a.n), p.top_p >= 0.0f ? fmin((double)p.top_p, 1.0) : p.top_p < 0.0f ? 0.0 : 1.0,
           p.min_p >= 0.0f ? fmin((double)p.min_p, 1.0) : 0.0, a.n};
    if (p.temperature > 0.0f) r.inverse4 = kSteps * kLog2e / (double)p.temperature;
    else r.top_k = 1;
    return r;
}

// What a row's tokens are measured from: 4 E.  Wild: E is of no use to the short forms below, for an infinite logit is the largest, or E is beyond 2^48.
struct Origin {
    double top4;  // -infinity: nothing may be taken
    bool wild;
    __device__ __forceinline__ bool none() const { return !(top4 > -__builtin_inf()); }
};
__device__ __forceinline__ Origin origin(double top4) { return {top4, !(__builtin_fabs(top4) < 0x1p50)}; }
__device__ __forceinline__ Origin origin_of(float largest, const Rule& r) {
    if (!(largest > -__builtin_inff())) return origin(-__builtin_inf());
    if (largest == __builtin_inff()) return origin(kInfinite4);
    return origin(kSteps * __builtin_floor((double)largest * r.inverse4 / kSteps));
}
// A token's 4 y; of one that is never taken, -infinity or NaN.  (T may be infinite too.)
template <bool WILD>
__device__ __forceinline__ double quarters(float l, const Rule& r, const Origin& o) {
    const double y4 = (double)l * r.inverse4;
    return WILD && o.top4 == kInfinite4 ? (l == __builtin_inff() ? kInfinite4 : -__builtin_inf()) : y4;
}
// The bin of a token: 4 y rounded to a whole number, counted from 4 E + 4 down, or kBins: it weighs nothing.  The whole number is the token's own, so that the bins of
// another E are the same ones, counted from elsewhere.  (The short form has it in the lower bits of 4 y + 1.5 2^52, without the vector unit's
// conversions, which take four times as long as an addition.)
constexpr double kRound = 0x1.8p52;
template <bool WILD>
__device__ __forceinline__ uint32_t bin_of(double y4, const Origin& o) {
    if constexpr (WILD) {
        const double below = (o.top4 - __builtin_rint(y4)) + kSteps;
        return below < (double)kBins ? (uint32_t)fmax(below, 0.0) : kBins;
    } else {
        const double from = o.top4 + (kRound + kSteps), at = y4 + kRound;  // (both whole, and their difference)
        return from - at < (double)kBins ? __double2loint(from) - __double2loint(at) : kBins;
    }
}
// 2^(y - E) times 2^43 (up to 2^19 tokens of less than 2 each), for y of a bin: 2^(g / 4) for |g| <= 2 by the polynomial that interpolates it at the Chebyshev nodes (off by 5e-16), put in place by adding
// to its exponent; 1.5 2^54 rounds to whole fours.
struct Power {  // (its coefficients are kept in scalar registers)
    double c[11] = {0x1p43, 0x1.62e42fefa3a19p40, 0x1.ebfbdff82c598p36, 0x1.c6b08d703ce45p32, 0x1.3b2ab6fba1dcfp28, 0x1.5d87fe9d7ab38p23, 0x1.4309130972582p18,
                    0x1.ffcb54054027cp12, 0x1.62bfd472738fap7, 0x1.b675bd7308f14p1, 0x1.e606452d2a4bep-5};
    __device__ __forceinline__ void keep() {
#pragma unroll
        for (int i = 0; i < 11; i++) asm("" : "+s"(c[i]));
    }
    __device__ __forceinline__ double exact(double y4, const Origin& o) const {
        const double d = y4 - o.top4, n = d + 0x1.8p54, g = d - (n - 0x1.8p54);
        double p = c[10];
#pragma unroll
        for (int i = 9; i >= 0; i--) p = __builtin_fma(p, g, c[i]);
        return __hiloint2double(__double2hiint(p) + (int)((uint32_t)__double2loint(n) << 20), __double2loint(p));
    }
    // ... in whole numbers: rounded by adding 2^52.
    __device__ __forceinline__ uint64_t whole(double y4, const Origin& o) const {
        return __builtin_bit_cast(uint64_t, exact(y4, o) + 0x1p52) & ((1ull << 52) - 1u);
    }
};
__device__ __forceinline__ double exact_weight(double y4, const Origin& o) { return Power().exact(y4, o); }
__device__ __forceinline__ uint64_t weight_of(double y4, const Origin& o) { return Power().whole(y4, o); }

// (logit, lower index first) as one number, of a logit that may be taken; no key is 0.
__device__ __forceinline__ uint64_t key_of(float l, uint32_t i) {
    const uint32_t b = __float_as_uint(l + 0.0f);  // (the zeros alike)
    return (uint64_t)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | (uint32_t)~i;
}
__device__ __forceinline__ uint32_t index_of(uint64_t key) { return ~(uint32_t)key; }
__device__ __forceinline__ float logit_of(uint64_t key) {
    const uint32_t b = (uint32_t)(key >> 32);
    return __uint_as_float(b & 0x80000000u ? b ^ 0x80000000u : ~b);
}

__device__ __forceinline__ uint64_t read_lane(uint64_t v, uint32_t lane) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), (int)lane) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)v, (int)lane);
}
// Sum over a wave's lanes up to this one, without LDS: inside rows of 16 lanes, then the last of a row to the next one, and of a half to the other.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t moved_or_zero(uint64_t v) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xf, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xf, false);
    return (uint64_t)hi << 32 | lo;
}
__device__ __forceinline__ uint64_t lanes_upto(uint64_t v) {
    v += moved_or_zero<0x111, 0xf>(v), v += moved_or_zero<0x112, 0xf>(v), v += moved_or_zero<0x114, 0xf>(v), v += moved_or_zero<0x118, 0xf>(v);
    v += moved_or_zero<0x142, 0xa>(v), v += moved_or_zero<0x143, 0xc>(v);
    return v;
}
__device__ __forceinline__ uint32_t lanes_upto(uint32_t v) { return (uint32_t)lanes_upto((uint64_t)v); }
// Sum over the workgroup's threads in front of this one, and over all of them.  `slots`: one per wave, of this call alone until the next barrier.
template <uint32_t WAVES>
__device__ __forceinline__ uint64_t sum_before(uint64_t v, uint64_t* slots, uint64_t& total) {
    const uint32_t lane = threadIdx.x & 63u, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint64_t upto = lanes_upto(v);
    if (lane == 63u) slots[wave] = upto;
    __syncthreads();
    const uint64_t sums = lanes_upto(lane < WAVES ? slots[lane] : 0);
    total = read_lane(sums, 63);
    return upto - v + (wave > 0 ? read_lane(sums, wave - 1u) : 0);
}

constexpr uint32_t kPartThreads = 256, kPartLoads = kPart / kPartThreads;

// 1.
__global__ __launch_bounds__(kPartThreads) void sample_bins_kernel(SampleArgs a) {
    __shared__ uint32_t count[kBins];
    __shared__ unsigned long long mass[kBins];
    __shared__ float tops[kPartThreads / 64];
    const uint32_t row = blockIdx.y, first = blockIdx.x * kPart;
    const float* const logits = a.logits + (size_t)row * a.stride;
    float l[kPartLoads], top = -__builtin_inff();
#pragma unroll
    for (uint32_t k = 0; k < kPartLoads; k++) {
        const uint32_t i = first + k * kPartThreads + threadIdx.x;
        l[k] = i < a.n ? logits[i] : -__builtin_inff();
    }
    const Rule r = rule_of(a, row);
    const bool counts = r.counts(), masses = r.masses();
#pragma unroll
    for (uint32_t k = 0; k < kPartLoads; k++) top = fmaxf(top, l[k]);  // (NaN is passed over)
    for (uint32_t b = threadIdx.x; b < kBins; b += kPartThreads) count[b] = 0, mass[b] = 0;
    top = wave_max_f32(top);
    if ((threadIdx.x & 63u) == 0) tops[threadIdx.x >> 6] = top;
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < kPartThreads / 64; w++) top = fmaxf(top, tops[w]);
    const Origin o = origin_of(top, r);
    const auto add = [&](auto wild) {
        Power power;
        power.keep();
#pragma unroll
        for (uint32_t k = 0; k < kPartLoads; k++) {
            const double y4 = quarters<decltype(wild)::value>(l[k], r, o);
            const uint32_t b = bin_of<decltype(wild)::value>(y4, o);
            if (b >= kBins) continue;
            if (counts) atomicAdd(&count[b], 1u);
            if (masses) atomicAdd(&mass[b], (unsigned long long)power.whole(y4, o));
        }
    };
    if (!o.none() && (counts || masses)) {
        if (o.wild) add(std::true_type());
        else add(std::false_type());
    }
    __syncthreads();
    SamplePart& part = a.parts[(size_t)row * a.n_parts + blockIdx.x];
    if (threadIdx.x == 0) part.largest = top;
    for (uint32_t b = threadIdx.x; b < kBins; b += kPartThreads) {
        if (counts) part.count[b] = count[b];
        if (masses) part.mass[b] = mass[b];
    }
}

// A row's histogram from its parts', every wave with all of it: lane i has bins 3 i .. 3 i + 2, each with those in front of it; and where the cuts can be.
struct RowBins {
    uint64_t mass[kLaneBins], count[kLaneBins];
    Origin o;
    double floor;              // the mass that min-p asks for
    uint32_t k_bin;            // the bin with the top_k-th token; kBins: all are taken
    uint32_t p_first, p_last;  // bins that the nucleus can end in; p_first = kBins: there is none
    bool whole;                // all up to k_bin is listed

    __device__ __forceinline__ uint32_t sure() const { return whole ? 0u : min(k_bin, p_first); }  // the first bin that is not kept for certain
    __device__ __forceinline__ bool lists(uint32_t b) const { return whole ? b <= k_bin : b == k_bin || (b >= p_first && b <= p_last); }
    // What is in front of bin b, the same one for all lanes; where all of them are at it (another lane's values are read).
    static __device__ __forceinline__ uint64_t before(const uint64_t (&v)[kLaneBins], uint32_t b) {
        if (b == 0) return 0;
        const uint32_t lane = (b - 1u) / kLaneBins, i = (b - 1u) % kLaneBins;
        return read_lane(i == 0 ? v[0] : i == 1 ? v[1] : v[2], lane);
    }
    // The first bin up to which there is at least `target`, or kBins.
    static __device__ __forceinline__ uint32_t reaching(const uint64_t (&v)[kLaneBins], uint64_t target) {
        const uint64_t past = __ballot(v[2] >= target);  // (all lanes are here)
        if (past == 0) return kBins;
        const uint32_t lane = (uint32_t)__ffsll((unsigned long long)past) - 1u;
        return lane * kLaneBins + (read_lane(v[0], lane) >= target ? 0u : read_lane(v[1], lane) >= target ? 1u : 2u);
    }
};
__device__ __forceinline__ uint64_t share_of_mass(double share, uint64_t mass) {  // at least 1, so that a token is taken
    const uint64_t t = (uint64_t)__builtin_ceil(share * (double)mass);
    return t == 0 ? 1u : t < mass ? t : mass;
}

constexpr uint32_t kAtOnce = 8;
struct BinShared {
    uint64_t mass[64 * kLaneBins];
    uint32_t count[64 * kLaneBins];
};

// `meanwhile`: what else is to be asked of memory, behind the parts' histograms, whose registers it may have.
template <typename F>
__device__ __forceinline__ RowBins row_bins(const SampleArgs& a, uint32_t row, const Rule& r, BinShared& sh, F meanwhile) {
    const SamplePart* const parts = a.parts + (size_t)row * a.n_parts;
    const uint32_t lane = threadIdx.x & 63u;
    const float largest[2] = {lane < a.n_parts ? parts[lane].largest : -__builtin_inff(), lane + 64u < a.n_parts ? parts[lane + 64u].largest : -__builtin_inff()};
    const float most = wave_max_f32(fmaxf(largest[0], largest[1]));
    RowBins bins;
    bins.o = origin_of(most, r);
    bins.floor = 0.0, bins.k_bin = bins.p_first = kBins, bins.p_last = 0, bins.whole = r.few();
#pragma unroll
    for (uint32_t i = 0; i < kLaneBins; i++) bins.mass[i] = bins.count[i] = 0;
    int off[2];  // whole powers of two that a part's E is below the row's
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const double d = (bins.o.top4 - origin_of(largest[i], r).top4) * (1.0 / kSteps);  // (infinite or NaN where there is nothing)
        off[i] = d < (double)kOctaves ? (int)d : kOctaves;
    }
    if (bins.o.none()) return bins;
    bins.floor = r.min_p * (double)weight_of(quarters<true>(most, r, bins.o), bins.o);
    const bool counts = r.counts(), masses = r.masses();
    if (!counts && !masses) {
        meanwhile();
        return bins;
    }
    for (uint32_t b = threadIdx.x; b < 64u * kLaneBins; b += blockDim.x) {
        uint64_t mass = 0;
        uint32_t count = 0;
        for (uint32_t p0 = 0; p0 < a.n_parts; p0 += kAtOnce) {  // (loads of several parts on their way together)
            uint32_t shift[kAtOnce], counted[kAtOnce];
            uint64_t weighed[kAtOnce];
#pragma unroll
            for (uint32_t i = 0; i < kAtOnce; i++) {
                const uint32_t p = min(p0 + i, a.n_parts - 1u);
                shift[i] = (uint32_t)__builtin_amdgcn_readlane(p < 64u ? off[0] : off[1], (int)(p & 63u));
                const uint32_t from = b - shift[i] * kSteps;  // (wraps where the part has nothing so far up)
                const bool in = from < kBins && b < kBins && p0 + i < a.n_parts;
                counted[i] = counts && in ? parts[p].count[from] : 0u, weighed[i] = masses && in ? parts[p].mass[from] : 0u;
            }
#pragma unroll
            for (uint32_t i = 0; i < kAtOnce; i++) count += counted[i], mass += weighed[i] >> shift[i];
        }
        sh.count[b] = count, sh.mass[b] = mass;
    }
    meanwhile();
    __syncthreads();
    uint64_t sum = 0, tokens = 0;
#pragma unroll
    for (uint32_t i = 0; i < kLaneBins; i++) bins.mass[i] = sum += sh.mass[kLaneBins * lane + i], bins.count[i] = tokens += sh.count[kLaneBins * lane + i];
    const uint64_t mass_front = lanes_upto(sum) - sum, count_front = lanes_upto(tokens) - tokens;
#pragma unroll
    for (uint32_t i = 0; i < kLaneBins; i++) bins.mass[i] += mass_front, bins.count[i] += count_front;
    if (counts) bins.k_bin = RowBins::reaching(bins.count, r.top_k);
    if (masses) {
        // the mass of what top-k leaves lies between that in front of its bin and that with it
        const uint64_t least = RowBins::before(bins.mass, bins.k_bin), most_mass = RowBins::before(bins.mass, min(bins.k_bin + 1u, kBins));
        bins.p_first = min(RowBins::reaching(bins.mass, share_of_mass(r.top_p, least)), bins.k_bin);
        bins.p_last = min(RowBins::reaching(bins.mass, share_of_mass(r.top_p, most_mass)), bins.k_bin);
    }
    return bins;
}

__device__ __forceinline__ void hand_on(const RowBins& bins, SampleRow& row) {  // one wave
    const uint32_t lane = threadIdx.x & 63u;
    if (lane == 0) row.top4 = bins.o.top4, row.floor = bins.floor, row.k_bin = bins.k_bin, row.p_first = bins.p_first, row.p_last = bins.p_last;
#pragma unroll
    for (uint32_t i = 0; i < kLaneBins; i++) row.mass[kLaneBins * lane + i] = bins.mass[i], row.count[kLaneBins * lane + i] = (uint32_t)bins.count[i];
}
__device__ __forceinline__ RowBins handed_on(const SampleRow& row, const Rule& r) {
    RowBins bins;
    const uint32_t lane = threadIdx.x & 63u;
    bins.o = origin(row.top4), bins.floor = row.floor, bins.k_bin = row.k_bin, bins.p_first = row.p_first, bins.p_last = row.p_last, bins.whole = r.few();
#pragma unroll
    for (uint32_t i = 0; i < kLaneBins; i++) bins.mass[i] = row.mass[kLaneBins * lane + i], bins.count[i] = row.count[kLaneBins * lane + i];
    return bins;
}

// 2.
__global__ __launch_bounds__(kPartThreads, 8) void sample_list_kernel(SampleArgs a) {
    __shared__ BinShared shared_bins;
    __shared__ uint64_t slots[kPartThreads / 64];
    __shared__ float candidates[kPart / 2];
    __shared__ uint16_t places[kPart / 2];
    __shared__ uint32_t listed, together;
    const uint32_t row = blockIdx.y, first = blockIdx.x * kPart;
    const float* const logits = a.logits + (size_t)row * a.stride;
    const Rule r = rule_of(a, row);
    if (threadIdx.x == 0) listed = 0, together = 0;
    float l[kPartLoads];
    const RowBins bins = row_bins(a, row, r, shared_bins, [&] {
#pragma unroll
        for (uint32_t k = 0; k < kPartLoads; k++) {
            const uint32_t i = first + k * kPartThreads + threadIdx.x;
            l[k] = i < a.n ? logits[i] : -__builtin_inff();
        }
    });
    if (blockIdx.x == 0 && threadIdx.x < 64u) hand_on(bins, a.rows[row]);
    if (bins.o.none()) return;
    __syncthreads();
    uint64_t sure = 0;
    uint64_t* const list = a.lists + (size_t)row * a.n + first;
    const uint32_t sure_bins = bins.sure();
    Power power;
    power.keep();
    const auto take = [&](auto wild, float x, uint32_t i) {
        const double y4 = quarters<decltype(wild)::value>(x, r, bins.o);
        const uint32_t b = bin_of<decltype(wild)::value>(y4, bins.o);
        if (b < sure_bins) {
            const uint64_t w = power.whole(y4, bins.o);
            sure += (double)w >= bins.floor ? w : 0;
        } else if (b < kBins && bins.lists(b)) {
            list[atomicAdd(&listed, 1u)] = key_of(x, i);
        }
    };
    // The last bin that matters; as a rule it is far above most tokens.  Those that may be in it or above (by their logit, with room for rounding) are put together
    // first, so that few waves do the rest.
    const uint32_t last = bins.k_bin < kBins || bins.p_first == kBins ? bins.k_bin : bins.p_last;
    // Where min-p alone cuts, only the weights that it leaves matter: from an octave below its floor up (200 rows of 50257 under min-p alone: 34.5 us with all of them, 27.6).  Top-p's
    // share is of what is below the floor too, and where tokens are only counted no bin says that it cuts.
    const bool uncut = bins.k_bin == kBins && bins.p_first == kBins && r.top_p >= 1.0;
    if (last == kBins && !bins.o.wild && !(uncut && bins.floor > 0.0)) {
#pragma unroll
        for (uint32_t k = 0; k < kPartLoads; k++) take(std::false_type(), l[k], first + k * kPartThreads + threadIdx.x);
    } else {
        // (a bin goes half a step further down than its whole number, which is at 4 E + 4 - bin; the floor is 2^43 times one of 2^(y - E))
        const double below = uncut && bins.floor > 0.0 ? (double)(kSteps * (45 - __builtin_amdgcn_frexp_exp(bins.floor))) : (double)last;
        const double lowest = fmin((bins.o.top4 - below) / r.inverse4, kInfinite4);
        const float low = (float)(lowest - __builtin_fabs(lowest) * 0x1p-20 - 0x1p-140);
#pragma unroll
        for (uint32_t half = 0; half < 2; half++) {
            if (half != 0) {
                __syncthreads();
                if (threadIdx.x == 0) together = 0;
                __syncthreads();
            }
            uint32_t count = 0;
#pragma unroll
            for (uint32_t k = half * kPartLoads / 2; k < (half + 1) * kPartLoads / 2; k++) count += l[k] >= low;
            const uint32_t upto = lanes_upto(count);
            uint32_t at = 0;
            if ((threadIdx.x & 63u) == 63u) at = atomicAdd(&together, upto);
            at = (uint32_t)__builtin_amdgcn_readlane((int)at, 63) + upto - count;
#pragma unroll
            for (uint32_t k = half * kPartLoads / 2; k < (half + 1) * kPartLoads / 2; k++)
                if (l[k] >= low) candidates[at] = l[k], places[at] = (uint16_t)(k * kPartThreads + threadIdx.x), at++;
            __syncthreads();
            for (uint32_t i = threadIdx.x; i < together; i += kPartThreads) {
                if (bins.o.wild) take(std::true_type(), candidates[i], first + places[i]);
                else take(std::false_type(), candidates[i], first + places[i]);
            }
        }
        __syncthreads();  // (listed)
    }
    uint64_t all;
    sum_before<kPartThreads / 64>(sure, slots, all);
    SamplePart& part = a.parts[(size_t)row * a.n_parts + blockIdx.x];
    if (threadIdx.x == 0) part.sure = all, part.listed = listed;
}

// 3.
// (Sixteen waves: 64 rows' nuclei and 200 rows' mixed rules take 13.1 and 16.2 us; with four 15.9 and 25.1, with eight 12.9 and 17.7.)
constexpr uint32_t kPickThreads = 1024, kPickWaves = kPickThreads / 64, kDigit = 10, kDigits = 1u << kDigit, kOwn = 1, kLoadsAtOnce = 2;
constexpr uint32_t kEach = kPart / kPickThreads, kDigitsEach = kDigits / kPickThreads;

struct PickShared {
    uint64_t slots[4][kPickWaves], part_mass[kMaxParts], found[4], key[64];
    uint32_t listed[kMaxParts], together;
    uint32_t count[kDigits];
    unsigned long long mass[kDigits];
};

// Lane i's value from lane i ^ DISTANCE, without LDS.
template <uint32_t DISTANCE>
__device__ __forceinline__ uint32_t exchanged(uint32_t v) {
    if constexpr (DISTANCE == 1) return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, false);  // quad_perm [1,0,3,2]
    if constexpr (DISTANCE == 2) return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, false);  // quad_perm [2,3,0,1]
    if constexpr (DISTANCE == 4) {  // quads 0 and 2 from the right, 1 and 3 from the left
        const int right = __builtin_amdgcn_update_dpp(0, (int)v, 0x104, 0xf, 0x5, false);
        return (uint32_t)__builtin_amdgcn_update_dpp(right, (int)v, 0x114, 0xf, 0xa, false);
    }
    if constexpr (DISTANCE == 8) return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, false);  // row_ror:8
    if constexpr (DISTANCE == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        return (threadIdx.x & 16u) != 0 ? r[0] : r[1];
    }
    if constexpr (DISTANCE == 32) {
        const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return (threadIdx.x & 32u) != 0 ? r[0] : r[1];
    }
}
template <uint32_t RUN, uint32_t DISTANCE>
__device__ __forceinline__ void sort_step(uint64_t& key) {
    const uint64_t other = (uint64_t)exchanged<DISTANCE>((uint32_t)(key >> 32)) << 32 | exchanged<DISTANCE>((uint32_t)key);
    const bool larger = ((threadIdx.x & DISTANCE) == 0) == ((threadIdx.x & RUN) == 0 || RUN == 64);
    if (larger == (other > key)) key = other;  // (equal ones: either)
    if constexpr (DISTANCE > 1) sort_step<RUN, DISTANCE / 2>(key);
    else if constexpr (RUN < 64) sort_step<RUN * 2, RUN>(key);
}
// Lane i of the wave gets the i-th largest of its keys (a bitonic network).
__device__ __forceinline__ uint64_t sorted(uint64_t key) {
    sort_step<2, 1>(key);
    return key;
}

// MANY: more tokens are listed than threads.  The usual row, which has fewer, keeps code of its own: with the loops over long lists in it 64 rows took 12.2 us, not 11.6, and
// 200 16.3, not 15.7.
template <bool MANY>
struct Picker {
    const SampleArgs& a;
    const Rule& r;
    const RowBins& bins;
    PickShared& sh;
    uint32_t row, tokens;  // tokens: listed ones
    uint64_t own[kOwn];    // this thread's first ones

    __device__ __forceinline__ uint64_t load(uint32_t f) const {
        uint32_t low = 0, high = a.n_parts;
        while (high - low > 1) {
            const uint32_t mid = (low + high) / 2u;
            (sh.listed[mid] <= f ? low : high) = mid;
        }
        return a.lists[(size_t)row * a.n + (size_t)low * kPart + (f - sh.listed[low])];
    }
    // All listed tokens, each by a thread of its own.
    template <typename F>
    __device__ __forceinline__ void for_all(F f) const {
#pragma unroll
        for (uint32_t i = 0; i < kOwn; i++)
            if (threadIdx.x + i * kPickThreads < tokens) f(own[i]);
        if constexpr (!MANY) return;
        for (uint32_t t = threadIdx.x + kOwn * kPickThreads; t < tokens; t += kLoadsAtOnce * kPickThreads) {
            uint64_t key[kLoadsAtOnce];
#pragma unroll
            for (uint32_t i = 0; i < kLoadsAtOnce; i++) key[i] = t + i * kPickThreads < tokens ? load(t + i * kPickThreads) : 0;
#pragma unroll
            for (uint32_t i = 0; i < kLoadsAtOnce; i++)
                if (key[i] != 0) f(key[i]);
        }
    }
    // *sum += v of every lane that is here.  Where there are many tokens, lanes with the same v at the same place (tokens that are alike) are one addition.
    static __device__ __forceinline__ void add_to(unsigned long long* sum, uint64_t v) {
        if constexpr (!MANY) {
            atomicAdd(sum, (unsigned long long)v);
            return;
        }
        const uint64_t here = __ballot(true), first = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)v);
        const uint32_t place = (uint32_t)(uintptr_t)sum;
        if (__ballot(v == first && place == (uint32_t)__builtin_amdgcn_readfirstlane((int)place)) == here) {
            if ((threadIdx.x & 63u) == (uint32_t)__ffsll((unsigned long long)here) - 1u) atomicAdd(sum, (unsigned long long)(first * (uint32_t)__popcll(here)));
        } else {
            atomicAdd(sum, (unsigned long long)v);
        }
    }
    __device__ __forceinline__ double quarters_of(uint64_t key) const { return quarters<true>(logit_of(key), r, bins.o); }
    __device__ __forceinline__ uint64_t weight(uint64_t key) const { return weight_of(quarters_of(key), bins.o); }

    // Of the listed tokens of one bin whose keys are from `least` on, from the largest key down, as many as are `goal` tokens, or as their masses take to reach `goal`: the
    // smallest key of those, and their mass.
    __device__ __forceinline__ uint64_t select(uint32_t bin, uint64_t least, uint64_t goal, bool by_mass, uint64_t& mass) {
        // A bin is 1024 steps of y wide first, of which the one where the goal is reached holds few tokens, as a rule; else their keys' digits, from the highest.
        uint64_t prefix = 0;  // of the keys that are left, from bit `known` up
        uint32_t step = 0;
        mass = 0;
        const auto next = [](int known) { return known > (int)kDigit ? known - (int)kDigit : 0; };
        for (int known = 64, shift = 64;;) {
            const auto is_left = [&](uint64_t key, double& y4, double& place) {
                y4 = quarters_of(key), place = y4 - __builtin_rint(y4);  // within half a step, more of a larger one
                return key >= least && bin_of<true>(y4, bins.o) == bin && (shift == 64 || (step_of(place) == step && (known == 64 || key >> known == prefix >> known)));
            };
            __syncthreads();
            if (threadIdx.x < 4) sh.found[threadIdx.x] = 0;
            if (threadIdx.x == 0) sh.together = 0;
            for (uint32_t d = threadIdx.x; d < kDigits; d += kPickThreads) sh.count[d] = 0, sh.mass[d] = 0;
            __syncthreads();
            for_all([&](uint64_t key) {
                double y4, place;
                if (!is_left(key, y4, place)) return;
                const uint32_t d = shift == 64 ? step_of(place) : (uint32_t)(key >> shift) & (kDigits - 1u);
                atomicAdd(&sh.count[d], 1u), add_to(&sh.mass[d], weight_of(y4, bins.o));
            });
            __syncthreads();
            // the digits from the highest
            uint64_t sum = 0, masses = 0;
#pragma unroll
            for (uint32_t i = 0; i < kDigitsEach; i++) {
                const uint32_t d = kDigits - 1u - kDigitsEach * threadIdx.x - i;
                masses += sh.mass[d], sum += by_mass ? sh.mass[d] : sh.count[d];
            }
            uint64_t all, all_mass;
            uint64_t before = sum_before<kPickWaves>(sum, sh.slots[0], all), mass_before = by_mass ? before : sum_before<kPickWaves>(masses, sh.slots[1], all_mass);
            goal = goal < all ? goal : all;  // (what there is may be a little less than the bins' masses said)
            if (before < goal && goal <= before + sum) {
                uint32_t d = kDigits - 1u - kDigitsEach * threadIdx.x;
                for (uint64_t n; before + (n = by_mass ? sh.mass[d] : sh.count[d]) < goal; d--) before += n, mass_before += sh.mass[d];
                sh.found[0] = d, sh.found[1] = goal - before, sh.found[2] = mass_before;
            }
            __syncthreads();
            const uint32_t digit = (uint32_t)sh.found[0];
            goal = sh.found[1], mass += sh.found[2];
            if (shift == 64) step = digit;
            else prefix = (prefix & ~((uint64_t)(kDigits - 1u) << shift)) | (uint64_t)digit << shift;
            if (sh.count[digit] > 64u) {  // (a key's last digit leaves one)
                if (shift != 64) {
                    known = shift, shift = next(known);
                    continue;
                }
                // the digits begin where those that are left differ: only in their indexes, if many are alike
                __syncthreads();
                if (threadIdx.x == 0) sh.found[0] = 0, sh.found[1] = ~0ull;
                __syncthreads();
                uint64_t any = 0, every = ~0ull;
                for_all([&](uint64_t key) {
                    const double y4 = quarters_of(key);
                    if (key >= least && bin_of<true>(y4, bins.o) == bin && step_of(y4 - __builtin_rint(y4)) == step) any |= key, every &= key;
                });
                atomicOr(reinterpret_cast<unsigned long long*>(&sh.found[0]), (unsigned long long)any);
                atomicAnd(reinterpret_cast<unsigned long long*>(&sh.found[1]), (unsigned long long)every);
                __syncthreads();
                prefix = sh.found[0], known = 64 - __builtin_clzll(sh.found[0] ^ sh.found[1]), shift = next(known);  // (more than 64 differ)
                continue;
            }
            // what is left has a lane each
            for_all([&](uint64_t key) {
                const double y4 = quarters_of(key);
                if (key >= least && bin_of<true>(y4, bins.o) == bin && step_of(y4 - __builtin_rint(y4)) == step && (shift == 64 || key >> shift == prefix >> shift))
                    sh.key[atomicAdd(&sh.together, 1u)] = key;
            });
            __syncthreads();
            if (threadIdx.x < 64u) {
                const uint64_t key = sorted(threadIdx.x < sh.together ? sh.key[threadIdx.x] : 0), w = key != 0 ? weight(key) : 0, upto = lanes_upto(w);
                const bool taken = key != 0 && (by_mass ? upto - w < goal : threadIdx.x < goal);
                const uint64_t takers = __ballot(taken);  // (from lane 0 on)
                if (threadIdx.x + 1u == (uint32_t)__popcll(takers)) sh.found[3] = key, sh.found[2] = upto;
            }
            __syncthreads();
            mass += sh.found[2];
            return sh.found[3];
        }
    }
    static __device__ __forceinline__ uint32_t step_of(double place) { return min((uint32_t)(place * (double)kDigits + (double)(kDigits / 2u)), kDigits - 1u); }

    // The smallest key that is kept.
    __device__ __forceinline__ uint64_t threshold() {
        uint64_t least = 0, mass = r.masses() ? RowBins::before(bins.mass, bins.k_bin) : 0, in_bin;
        if (bins.k_bin < kBins) {
            least = select(bins.k_bin, 0, r.top_k - RowBins::before(bins.count, bins.k_bin), false, in_bin);
            mass += in_bin;
        }
        if (r.top_p >= 1.0) return least;
        if (!bins.whole) {
            const uint64_t target = share_of_mass(r.top_p, mass);
            const uint32_t end = max(min(min(RowBins::reaching(bins.mass, target), bins.k_bin), bins.p_last), bins.p_first);
            const uint64_t in_front = RowBins::before(bins.mass, end);
            return max(select(end, least, target > in_front ? target - in_front : 1, true, in_bin), least);
        }
        // nobody has weighed the bins of what top-k leaves
        __syncthreads();
        if (threadIdx.x < 64u * kLaneBins) sh.mass[threadIdx.x] = 0;
        __syncthreads();
        for_all([&](uint64_t key) {
            if (key < least) return;
            const double y4 = quarters_of(key);
            add_to(&sh.mass[bin_of<true>(y4, bins.o)], weight_of(y4, bins.o));
        });
        __syncthreads();
        uint64_t of[kLaneBins], sum = 0;
        const uint32_t lane = threadIdx.x & 63u;
#pragma unroll
        for (uint32_t i = 0; i < kLaneBins; i++) of[i] = sum += sh.mass[kLaneBins * lane + i];
        const uint64_t front = lanes_upto(sum) - sum;
#pragma unroll
        for (uint32_t i = 0; i < kLaneBins; i++) of[i] += front;
        const uint64_t target = share_of_mass(r.top_p, RowBins::before(of, kBins));
        const uint32_t end = min(RowBins::reaching(of, target), kBins - 1u);
        return max(select(end, least, target - RowBins::before(of, end), true, in_bin), least);
    }
};

// All of it where one wave has every token that may be taken: sorted by key for the cuts, then by index.
__device__ __forceinline__ void pick_in_a_wave(const SampleArgs& a, uint32_t row, const Rule& r, const RowBins& bins, const Picker<false>& pick, float u) {
    const uint64_t key = sorted(pick.own[0]), w = key != 0 ? pick.weight(key) : 0;
    bool taken = key != 0 && threadIdx.x < r.top_k;
    if (r.top_p < 1.0) {
        const uint64_t upto = lanes_upto(taken ? w : 0), target = share_of_mass(r.top_p, read_lane(upto, 63));
        taken = taken && upto - w < target;
    }
    taken = taken && (double)w >= bins.floor;
    // (the lower half of a key falls with the index; what is not taken goes behind)
    const uint64_t by_index = sorted(taken ? key << 32 | key >> 32 : 0);
    const uint64_t back = by_index << 32 | by_index >> 32, weight = by_index != 0 ? pick.weight(back) : 0, upto = lanes_upto(weight), mass = read_lane(upto, 63);
    const double at = (u > 0.0f ? (double)u : 0.0) * (double)mass;
    const uint64_t target = at < (double)mass ? min((uint64_t)at, mass - 1u) : mass - 1u;  // the pick is the first to exceed it
    if (upto - weight <= target && target < upto) {
        a.out[row] = index_of(back);
        if (a.prob) a.prob[row] = (float)(exact_weight(pick.quarters_of(back), bins.o) / (double)mass);
    }
}

// The cuts and the pick, from the tokens that are listed and the masses that parts keep for certain (in sh).
template <bool MANY>
__device__ __forceinline__ void pick_of(const SampleArgs& a, uint32_t row, const Rule& r, const RowBins& bins, PickShared& sh, uint32_t tokens, float u) {
    const float* const logits = a.logits + (size_t)row * a.stride;
    const double floor = bins.floor;
    Picker<MANY> pick{a, r, bins, sh, row, tokens, {}};
#pragma unroll
    for (uint32_t i = 0; i < kOwn; i++)
        if (threadIdx.x + i * kPickThreads < tokens) pick.own[i] = pick.load(threadIdx.x + i * kPickThreads);
    if constexpr (!MANY)
        if (bins.whole && tokens <= 64) {
            if (threadIdx.x < 64u) pick_in_a_wave(a, row, r, bins, pick, u);
            return;
        }
    const uint64_t threshold = tokens == 0 ? 0 : pick.threshold();
    // what every part keeps
    pick.for_all([&](uint64_t key) {
        const uint64_t w = key >= threshold ? pick.weight(key) : 0;
        if ((double)w >= floor && w != 0) Picker<MANY>::add_to(reinterpret_cast<unsigned long long*>(&sh.part_mass[index_of(key) / kPart]), w);
    });
    __syncthreads();
    uint64_t mass;
    const uint64_t in_part = threadIdx.x < a.n_parts ? sh.part_mass[threadIdx.x] : 0, in_front = sum_before<kPickWaves>(in_part, sh.slots[2], mass);
    const double at = (u > 0.0f ? (double)u : 0.0) * (double)mass;
    const uint64_t target = at < (double)mass ? min((uint64_t)at, mass - 1u) : mass - 1u;  // the pick is the first to exceed it
    if (in_front <= target && target < in_front + in_part) sh.found[0] = threadIdx.x, sh.found[1] = target - in_front;  // (one thread: the mass is not 0)
    __syncthreads();
    const uint32_t part = min((uint32_t)sh.found[0], a.n_parts - 1u);
    const uint64_t goal = sh.found[1];
    float l[kEach];
    const uint32_t first = part * kPart + threadIdx.x * kEach;
    if (first + kEach <= a.n) {
#pragma unroll
        for (uint32_t k = 0; k < kEach; k += 4) {
            const u32x4_a4 x = *reinterpret_cast<const u32x4_a4*>(logits + first + k);
#pragma unroll
            for (uint32_t e = 0; e < 4; e++) l[k + e] = __uint_as_float(x.v[e]);
        }
    } else {
#pragma unroll
        for (uint32_t k = 0; k < kEach; k++) l[k] = first + k < a.n ? logits[first + k] : -__builtin_inff();
    }
    uint64_t weight[kEach], sum = 0;
#pragma unroll
    for (uint32_t k = 0; k < kEach; k++) {
        weight[k] = 0;
        const double y4 = quarters<true>(l[k], r, bins.o);
        if (bin_of<true>(y4, bins.o) >= kBins || key_of(l[k], first + k) < threshold) continue;
        const uint64_t w = weight_of(y4, bins.o);
        weight[k] = (double)w >= floor ? w : 0;
        sum += weight[k];
    }
    uint64_t all, before = sum_before<kPickWaves>(sum, sh.slots[3], all);
    if (before <= goal && goal < before + sum) {
        uint32_t i = first;
#pragma unroll
        for (uint32_t k = 0; k < kEach; k++) before += weight[k], i += before <= goal;
        a.out[row] = i;
        if (a.prob) a.prob[row] = (float)(exact_weight(quarters<true>(logits[i], r, bins.o), bins.o) / (double)mass);
    }
}

__global__ __launch_bounds__(kPickThreads) void sample_pick_kernel(SampleArgs a) {
    __shared__ PickShared sh;
    const uint32_t row = blockIdx.x;
    const SamplePart* const parts = a.parts + (size_t)row * a.n_parts;
    const uint64_t sure = threadIdx.x < a.n_parts ? parts[threadIdx.x].sure : 0;
    const uint32_t listed = threadIdx.x < a.n_parts ? parts[threadIdx.x].listed : 0;
    const float u = a.uniform[row];
    const Rule r = rule_of(a, row);
    const RowBins bins = handed_on(a.rows[row], r);
    if (bins.o.none()) {
        if (threadIdx.x == 0) {
            a.out[row] = WICK_ROCM_NO_TOKEN;
            if (a.prob) a.prob[row] = 0.0f;
        }
        return;
    }
    uint64_t tokens;
    const uint64_t upto = sum_before<kPickWaves>(listed, sh.slots[0], tokens);
    if (threadIdx.x < a.n_parts) sh.listed[threadIdx.x] = (uint32_t)upto, sh.part_mass[threadIdx.x] = sure;
    __syncthreads();
    if (tokens > kOwn * kPickThreads) return pick_of<true>(a, row, r, bins, sh, (uint32_t)tokens, u);
    pick_of<false>(a, row, r, bins, sh, (uint32_t)tokens, u);
}

size_t parts_of(uint32_t n) { return (n + kPart - 1u) / kPart; }

}  // namespace

size_t sample_scratch_bytes(uint32_t rows, uint32_t n) {
    return (size_t)rows * (sizeof(SampleRow) + parts_of(n) * sizeof(SamplePart) + (size_t)n * sizeof(uint64_t));
}

hipError_t launch_sample(const float* d_logits, uint32_t stride, uint32_t rows, uint32_t n, const wick_rocm_sample_params* d_params, const float* d_uniform,
                         uint32_t* d_out, float* d_prob, void* d_scratch, const Launch& L) {
    if (rows == 0) return hipSuccess;
    SampleArgs a{d_logits, d_params, d_uniform, d_out, d_prob, static_cast<SampleRow*>(d_scratch), nullptr, nullptr, n, stride, (uint32_t)parts_of(n)};
    a.parts = reinterpret_cast<SamplePart*>(a.rows + rows);
    a.lists = reinterpret_cast<uint64_t*>(a.parts + (size_t)rows * a.n_parts);
    hipError_t e = launch_kernel(L, kFamOther, sample_bins_kernel, dim3(a.n_parts, rows), dim3(kPartThreads), a);
    if (e == hipSuccess) e = launch_kernel(L, kFamOther, sample_list_kernel, dim3(a.n_parts, rows), dim3(kPartThreads), a);
    if (e == hipSuccess) e = launch_kernel(L, kFamOther, sample_pick_kernel, dim3(rows), dim3(kPickThreads), a);
    return e;
}

}  // namespace wick_rocm
