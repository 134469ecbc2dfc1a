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
#include <algorithm>

#include "wick_rocm_device.h"
#include "wick_rocm_internal.h"

namespace wick_rocm {

namespace {

constexpr uint32_t kPart = 4096, kMaxParts = kSampleMaxTokens / kPart;  // tokens of a part
constexpr int kOctaves = 46, kSteps = 4;                                // bins: kSteps to a power of two
constexpr uint32_t kBins = kOctaves * kSteps, kLaneBins = 3;            // every wave has them all, three a lane
static_assert(kBins <= 64 * kLaneBins && kMaxParts <= 128);
constexpr int kFraction = 43;  // masses are whole numbers of 2^-43: up to 2^19 tokens of less than 2 each
constexpr uint32_t kFew = 512; // top-k up to which all that it leaves is listed: 3. sorts up to 1024 tokens, and the last bin may be half of them
constexpr double kLog2e = 1.4426950408889634;
constexpr double kNever = -__builtin_inf(), kInfinite = 0x1p1000;       // y of what is never taken, and of an infinite logit

struct SamplePart {
    uint64_t sure;  // mass that is certainly kept
    float largest;  // logit
    uint32_t listed;
    uint64_t mass[kBins];
    uint32_t count[kBins];
};

struct SampleArgs {
    const float* logits;
    const wick_rocm_sample_params* params;
    const float* uniform;
    uint32_t* out;
    float* prob;
    SamplePart* parts;  // [rows][n_parts]
    uint32_t* lists;    // [rows][n]: part p's tokens from p kPart on
    uint32_t n, stride, n_parts;
};

struct Rule {
    double inverse;  // log2(e) / T
    uint32_t top_k;
    double top_p, min_p;
    __device__ __forceinline__ bool few() const { return top_k <= kFew; }
    __device__ __forceinline__ bool masses() const { return top_p < 1.0 && !few(); }  // 1. adds up masses,
    uint32_t n;
    __device__ __forceinline__ bool counts() const { return top_k < n || few(); }     // counts tokens
};
__device__ __forceinline__ Rule rule_of(const SampleArgs& a, uint32_t row) {
    const wick_rocm_sample_params p = a.params[row];
    Rule r{kLog2e, p.top_k == 0 ? a.n : min(p.top_k, a.n), p.top_p >= 0.0f ? fmin((double)p.top_p, 1.0) : p.top_p < 0.0f ? 0.0 : 1.0,
           p.min_p >= 0.0f ? fmin((double)p.min_p, 1.0) : 0.0, a.n};
    if (p.temperature > 0.0f) r.inverse = kLog2e / (double)p.temperature;
    else r.top_k = 1;
    return r;
}

__device__ __forceinline__ double power_of(float l, const Rule& r) {
    if (!(l > -__builtin_inff())) return kNever;
    return l == __builtin_inff() ? kInfinite : (double)l * r.inverse;
}
// The bin of a token (kBins: it weighs nothing).  Falls with rising y; every step is exact, so that the bins of another E are the same ones, counted from elsewhere.
__device__ __forceinline__ uint32_t bin_of(double y, double top) {
    const double below = (kSteps * top - __builtin_floor(kSteps * y)) + (kSteps - 1);
    return below < (double)kBins ? (uint32_t)below : kBins;
}
// 2^(y - top) times 2^kFraction, for y of a bin: 2^f for |f| <= 1/2 by the polynomial that interpolates it at the Chebyshev nodes (off by 5e-16), put in place by its
// exponent.
__device__ __forceinline__ double exact_weight(double y, double top) {
    const double v = y - top, n = __builtin_rint(v), f = v - n;
    double p = 0x1.e606452d2a4bep-28;
    p = __builtin_fma(p, f, 0x1.b675bd7308f14p-24), p = __builtin_fma(p, f, 0x1.62bfd472738fap-20), p = __builtin_fma(p, f, 0x1.ffcb54054027cp-17);
    p = __builtin_fma(p, f, 0x1.4309130972582p-13), p = __builtin_fma(p, f, 0x1.5d87fe9d7ab38p-10), p = __builtin_fma(p, f, 0x1.3b2ab6fba1dcfp-7);
    p = __builtin_fma(p, f, 0x1.c6b08d703ce45p-5), p = __builtin_fma(p, f, 0x1.ebfbdff82c598p-3), p = __builtin_fma(p, f, 0x1.62e42fefa3a19p-1);
    p = __builtin_fma(p, f, 1.0);
    return __builtin_ldexp(p, (int)n + kFraction);
}
// ... in whole numbers: rounded by adding 2^52.
__device__ __forceinline__ uint64_t weight_of(double y, double top) {
    return __builtin_bit_cast(uint64_t, exact_weight(y, top) + 0x1p52) & ((1ull << 52) - 1u);
}

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
    const double e = __builtin_floor(power_of(top, r));
    if (e > kNever && (counts || masses)) {
#pragma unroll
        for (uint32_t k = 0; k < kPartLoads; k++) {
            const double y = power_of(l[k], r);
            const uint32_t b = y > kNever ? bin_of(y, e) : kBins;
            if (b >= kBins) continue;
            if (counts) atomicAdd(&count[b], 1u);
            if (masses) atomicAdd(&mass[b], (unsigned long long)weight_of(y, e));
        }
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
    double top, floor;         // E, and the mass that min-p asks for
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
        const uint64_t past = __ballot(v[2] >= target);
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

__device__ __forceinline__ RowBins row_bins(const SampleArgs& a, uint32_t row, const Rule& r, BinShared& sh) {
    const SamplePart* const parts = a.parts + (size_t)row * a.n_parts;
    const uint32_t lane = threadIdx.x & 63u;
    const float largest[2] = {lane < a.n_parts ? parts[lane].largest : -__builtin_inff(), lane + 64u < a.n_parts ? parts[lane + 64u].largest : -__builtin_inff()};
    const float most = wave_max_f32(fmaxf(largest[0], largest[1]));
    RowBins bins;
    bins.top = __builtin_floor(power_of(most, r));
    bins.floor = 0.0, bins.k_bin = bins.p_first = kBins, bins.p_last = 0, bins.whole = r.few();
    int off[2];  // whole powers of two that a part's E is below the row's
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const double d = bins.top - __builtin_floor(power_of(largest[i], r));  // (infinite or NaN where there is nothing)
        off[i] = d < (double)kOctaves ? (int)d : kOctaves;
    }
    if (!(bins.top > kNever)) return bins;
    bins.floor = r.min_p * (double)weight_of(power_of(most, r), bins.top);
    const bool counts = r.counts(), masses = r.masses();
    if (!counts && !masses) return bins;
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

// 2.
__global__ __launch_bounds__(kPartThreads) void sample_list_kernel(SampleArgs a) {
    __shared__ BinShared shared_bins;
    __shared__ uint64_t slots[kPartThreads / 64];
    __shared__ uint32_t listed;
    const uint32_t row = blockIdx.y, first = blockIdx.x * kPart;
    const float* const logits = a.logits + (size_t)row * a.stride;
    float l[kPartLoads];
#pragma unroll
    for (uint32_t k = 0; k < kPartLoads; k++) {
        const uint32_t i = first + k * kPartThreads + threadIdx.x;
        l[k] = i < a.n ? logits[i] : -__builtin_inff();
    }
    const Rule r = rule_of(a, row);
    if (threadIdx.x == 0) listed = 0;
    const RowBins bins = row_bins(a, row, r, shared_bins);
    const double top = bins.top;
    if (!(top > kNever)) return;
    __syncthreads();
    uint64_t sure = 0;
    uint32_t* const list = a.lists + (size_t)row * a.n + first;
#pragma unroll
    for (uint32_t k = 0; k < kPartLoads; k++) {
        const uint32_t i = first + k * kPartThreads + threadIdx.x;
        const double y = power_of(l[k], r);
        const uint32_t b = y > kNever ? bin_of(y, top) : kBins;
        if (b >= kBins) continue;
        if (b < bins.sure()) {
            const uint64_t w = weight_of(y, top);
            sure += (double)w >= bins.floor ? w : 0;
        } else if (bins.lists(b)) {
            list[atomicAdd(&listed, 1u)] = i;
        }
    }
    uint64_t all;
    sum_before<kPartThreads / 64>(sure, slots, all);
    SamplePart& part = a.parts[(size_t)row * a.n_parts + blockIdx.x];
    if (threadIdx.x == 0) part.sure = all, part.listed = listed;
}

// 3.
constexpr uint32_t kPickThreads = 1024, kPickWaves = kPickThreads / 64, kDigit = 11, kDigits = 1u << kDigit;

struct PickShared {
    BinShared bins;
    uint64_t slots[4][kPickWaves], part_mass[kMaxParts], found[4];
    uint32_t listed[kMaxParts];
    union {
        uint64_t key[kPickThreads];
        struct {
            uint32_t count[kDigits];
            unsigned long long mass[kDigits];
        } digit;
    };
};

__device__ __forceinline__ uint64_t exchanged(uint64_t v, uint32_t distance) {
    return (uint64_t)__shfl_xor((unsigned long long)v, (int)distance, 64);
}

struct Picker {
    const SampleArgs& a;
    const Rule& r;
    const RowBins& bins;
    PickShared& sh;
    uint32_t row, tokens;  // tokens: listed ones

    // The key of listed token f.
    __device__ __forceinline__ uint64_t token(uint32_t f) const {
        uint32_t low = 0, high = a.n_parts;
        while (high - low > 1) {
            const uint32_t mid = (low + high) / 2u;
            (sh.listed[mid] <= f ? low : high) = mid;
        }
        const uint32_t i = a.lists[(size_t)row * a.n + (size_t)low * kPart + (f - sh.listed[low])];
        return key_of(a.logits[(size_t)row * a.stride + i], i);
    }
    __device__ __forceinline__ uint64_t weight(uint64_t key) const { return weight_of(power_of(logit_of(key), r), bins.top); }
    __device__ __forceinline__ uint32_t bin(uint64_t key) const { return bin_of(power_of(logit_of(key), r), bins.top); }

    // Thread i gets the i-th largest of the workgroup's keys: a bitonic network, whose steps over less than a wave need no barrier.
    __device__ __forceinline__ uint64_t sorted(uint64_t key) {
        uint32_t size = 64;
        while (size < tokens) size *= 2u;
        const uint32_t i = threadIdx.x;
        for (uint32_t run = 2; run <= size; run *= 2u)
            for (uint32_t distance = run / 2u; distance != 0; distance /= 2u) {
                uint64_t other;
                if (distance >= 64u) {
                    __syncthreads();
                    sh.key[i] = key;
                    __syncthreads();
                    other = sh.key[i ^ distance];
                } else {
                    other = exchanged(key, distance);
                }
                const bool larger = ((i & distance) == 0) == ((i & run) == 0 || run == size);
                if (larger ? other > key : other < key) key = other;
            }
        return key;
    }

    // The threshold where every listed token has a thread.
    __device__ __forceinline__ uint64_t few_threshold() {
        const uint64_t key = sorted(threadIdx.x < tokens ? token(threadIdx.x) : 0);
        const bool in = threadIdx.x < tokens;
        const uint32_t b = in ? bin(key) : kBins;
        const uint64_t w = in ? weight(key) : 0;
        bool taken = in && b <= bins.k_bin;
        uint64_t mass = bins.whole || !r.masses() ? 0 : RowBins::before(bins.mass, bins.k_bin);
        if (bins.k_bin < kBins) {  // of the last bin as many as are missing
            uint64_t in_front;
            sum_before<kPickWaves>(in && b < bins.k_bin, sh.slots[0], in_front);
            const uint64_t missing = r.top_k - RowBins::before(bins.count, bins.k_bin);
            taken = in && (b < bins.k_bin || (b == bins.k_bin && threadIdx.x - in_front < missing));
        }
        if (r.top_p < 1.0) {
            // masses in front of each: of a whole list as they are, else of a bin in which the nucleus may end, behind what the histogram has in front of it
            uint64_t kept;
            const uint64_t of_last = sum_before<kPickWaves>(taken && (bins.whole || b == bins.k_bin) ? w : 0, sh.slots[1], kept);
            mass += kept;
            const uint64_t target = share_of_mass(r.top_p, mass);
            if (bins.whole) {
                taken = taken && of_last < target;
            } else {
                const uint32_t end = max(min(min(RowBins::reaching(bins.mass, target), bins.k_bin), bins.p_last), bins.p_first);
                uint64_t all;
                const uint64_t in_front = RowBins::before(bins.mass, end), in_bin = sum_before<kPickWaves>(b == end ? w : 0, sh.slots[2], all);
                taken = taken && (b < end || (b == end && (in_bin == 0 || in_front + in_bin < target)));
            }
        }
        uint64_t n;
        sum_before<kPickWaves>(taken, sh.slots[3], n);  // what is taken is in front
        if (taken && threadIdx.x + 1u == n) sh.found[0] = key;
        __syncthreads();
        return sh.found[0];
    }

    // Of the listed tokens whose keys are from `least` on and whose bin is `bin_` (kBins: any), from the largest key down, as many as are `target` tokens, or as their
    // masses take to reach `target`: the smallest key of those, and their mass.
    __device__ __forceinline__ uint64_t select(uint32_t bin_, uint64_t least, uint64_t target, bool by_mass, uint64_t& mass) {
        uint64_t threshold = 0, left = target;
        mass = 0;
        for (int known = 64, shift = 64 - (int)kDigit;; known = shift, shift = shift > (int)kDigit ? shift - (int)kDigit : 0) {
            // digits from the highest; the last one overlaps the one before it, whose bits are the same for all that are left
            __syncthreads();
            if (threadIdx.x < 4) sh.found[threadIdx.x] = 0;
            for (uint32_t d = threadIdx.x; d < kDigits; d += kPickThreads) sh.digit.count[d] = 0, sh.digit.mass[d] = 0;
            __syncthreads();
            for (uint32_t f = threadIdx.x; f < tokens; f += kPickThreads) {
                const uint64_t key = token(f);
                if (key < least || (known < 64 && key >> known != threshold >> known) || (bin_ < kBins && bin(key) != bin_)) continue;
                const uint32_t d = (uint32_t)(key >> shift) & (kDigits - 1u);
                atomicAdd(&sh.digit.count[d], 1u), atomicAdd(&sh.digit.mass[d], (unsigned long long)weight(key));
            }
            __syncthreads();
            // thread t has digits 2047 - 2 t and the one below
            const uint32_t d0 = kDigits - 1u - 2u * threadIdx.x, d1 = d0 - 1u;
            const uint64_t m0 = sh.digit.mass[d0], m1 = sh.digit.mass[d1], n0 = by_mass ? m0 : sh.digit.count[d0], n1 = by_mass ? m1 : sh.digit.count[d1];
            uint64_t all, all_mass;
            const uint64_t before = sum_before<kPickWaves>(n0 + n1, sh.slots[0], all), mass_before = sum_before<kPickWaves>(m0 + m1, sh.slots[1], all_mass);
            const uint64_t goal = left < all ? left : all;  // (what there is may be a little less than the bins' masses said)
            if (before < goal && goal <= before + n0 + n1) {
                const bool second = goal > before + n0;
                sh.found[0] = second ? d1 : d0, sh.found[1] = goal - before - (second ? n0 : 0), sh.found[2] = mass_before + (second ? m0 : 0);
            }
            __syncthreads();
            const uint64_t digit = sh.found[0];
            left = sh.found[1], mass += sh.found[2];
            threshold = (threshold & ~((uint64_t)(kDigits - 1u) << shift)) | digit << shift;
            if (shift != 0 && sh.digit.count[digit] != 1u) continue;
            mass += sh.digit.mass[digit];  // the one token that is left
            if (shift == 0) return threshold;
            for (uint32_t f = threadIdx.x; f < tokens; f += kPickThreads) {
                const uint64_t key = token(f);
                if (key >= least && key >> shift == threshold >> shift && (bin_ == kBins || bin(key) == bin_)) sh.found[3] = key;
            }
            __syncthreads();
            return sh.found[3];
        }
    }

    // The threshold where there are more listed tokens than threads.
    __device__ __forceinline__ uint64_t many_threshold() {
        uint64_t threshold = 0, mass = r.masses() ? RowBins::before(bins.mass, bins.k_bin) : 0;
        if (bins.k_bin < kBins) {
            uint64_t in_bin;
            threshold = select(bins.k_bin, 0, r.top_k - RowBins::before(bins.count, bins.k_bin), false, in_bin);
            mass += in_bin;
        }
        if (r.top_p >= 1.0) return threshold;
        if (bins.whole) {
            uint64_t sum = 0;
            for (uint32_t f = threadIdx.x; f < tokens; f += kPickThreads) {
                const uint64_t key = token(f);
                sum += key >= threshold ? weight(key) : 0;
            }
            __syncthreads();
            sum_before<kPickWaves>(sum, sh.slots[2], mass);
            return select(kBins, threshold, share_of_mass(r.top_p, mass), true, sum);
        }
        const uint64_t target = share_of_mass(r.top_p, mass);
        const uint32_t end = max(min(min(RowBins::reaching(bins.mass, target), bins.k_bin), bins.p_last), bins.p_first);
        const uint64_t in_front = RowBins::before(bins.mass, end);
        return select(end, threshold, target > in_front ? target - in_front : 1, true, mass);
    }
};

__global__ __launch_bounds__(kPickThreads) void sample_pick_kernel(SampleArgs a) {
    __shared__ PickShared sh;
    const uint32_t row = blockIdx.x;
    const float* const logits = a.logits + (size_t)row * a.stride;
    const SamplePart* const parts = a.parts + (size_t)row * a.n_parts;
    const uint64_t sure = threadIdx.x < a.n_parts ? parts[threadIdx.x].sure : 0;
    const uint32_t listed = threadIdx.x < a.n_parts ? parts[threadIdx.x].listed : 0;
    const float u = a.uniform[row];
    const Rule r = rule_of(a, row);
    const RowBins bins = row_bins(a, row, r, sh.bins);
    const double top = bins.top, floor = bins.floor;
    if (!(top > kNever)) {
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
    Picker pick{a, r, bins, sh, row, (uint32_t)tokens};
    const uint64_t threshold = tokens == 0 ? 0 : tokens <= kPickThreads ? pick.few_threshold() : pick.many_threshold();
    // what every part keeps
    for (uint32_t f = threadIdx.x; f < tokens; f += kPickThreads) {
        const uint64_t key = pick.token(f), w = key >= threshold ? pick.weight(key) : 0;
        if ((double)w >= floor && w != 0) atomicAdd(reinterpret_cast<unsigned long long*>(&sh.part_mass[index_of(key) / kPart]), (unsigned long long)w);
    }
    __syncthreads();
    uint64_t mass;
    const uint64_t in_part = threadIdx.x < a.n_parts ? sh.part_mass[threadIdx.x] : 0, in_front = sum_before<kPickWaves>(in_part, sh.slots[0], mass);
    const double at = (u > 0.0f ? (double)u : 0.0) * (double)mass;
    const uint64_t target = at < (double)mass ? min((uint64_t)at, mass - 1u) : mass - 1u;  // the pick is the first to exceed it
    if (in_front <= target && target < in_front + in_part) sh.found[0] = threadIdx.x, sh.found[1] = target - in_front;  // (one thread: the mass is not 0)
    __syncthreads();
    const uint32_t part = min((uint32_t)sh.found[0], a.n_parts - 1u);
    const uint64_t goal = sh.found[1];
    uint64_t weight[kPart / kPickThreads], sum = 0;
#pragma unroll
    for (uint32_t k = 0; k < kPart / kPickThreads; k++) {
        const uint32_t i = part * kPart + threadIdx.x * (kPart / kPickThreads) + k;
        weight[k] = 0;
        if (i >= a.n) continue;
        const float l = logits[i];
        const double y = power_of(l, r);
        if (!(y > kNever) || bin_of(y, top) >= kBins || key_of(l, i) < threshold) continue;
        const uint64_t w = weight_of(y, top);
        weight[k] = (double)w >= floor ? w : 0;
        sum += weight[k];
    }
    uint64_t all, before = sum_before<kPickWaves>(sum, sh.slots[1], all);
    if (before <= goal && goal < before + sum) {
        uint32_t i = part * kPart + threadIdx.x * (kPart / kPickThreads);
#pragma unroll
        for (uint32_t k = 0; k < kPart / kPickThreads; k++) before += weight[k], i += before <= goal;
        a.out[row] = i;
        if (a.prob) a.prob[row] = (float)(exact_weight(power_of(logits[i], r), top) / (double)mass);
    }
}

size_t parts_of(uint32_t n) { return (n + kPart - 1u) / kPart; }

}  // namespace

size_t sample_scratch_bytes(uint32_t rows, uint32_t n) { return (size_t)rows * (parts_of(n) * sizeof(SamplePart) + (size_t)n * sizeof(uint32_t)); }

hipError_t launch_sample(const float* d_logits, uint32_t stride, uint32_t rows, uint32_t n, const wick_rocm_sample_params* d_params, const float* d_uniform,
                         uint32_t* d_out, float* d_prob, void* d_scratch, const Launch& L) {
    if (rows == 0) return hipSuccess;
    SampleArgs a{d_logits, d_params, d_uniform, d_out, d_prob, static_cast<SamplePart*>(d_scratch), nullptr, n, stride, (uint32_t)parts_of(n)};
    a.lists = reinterpret_cast<uint32_t*>(a.parts + (size_t)rows * a.n_parts);
    hipError_t e = launch_kernel(L, kFamOther, sample_bins_kernel, dim3(a.n_parts, rows), dim3(kPartThreads), a);
    if (e == hipSuccess) e = launch_kernel(L, kFamOther, sample_list_kernel, dim3(a.n_parts, rows), dim3(kPartThreads), a);
    if (e == hipSuccess) e = launch_kernel(L, kFamOther, sample_pick_kernel, dim3(rows), dim3(kPickThreads), a);
    return e;
}

}  // namespace wick_rocm
