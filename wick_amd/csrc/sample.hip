// Sampling: a row's next token by temperature, top-k, top-p and min-p from a given uniform number.
//
// With y_i = l_i log2(e) / T, rounded to f64, and E the whole number below the largest, token i weighs W_i = 2^(y_i - E) in whole numbers of 2^-43: masses are
// whole numbers, whose sums are the same in every order.  Both cuts are cuts in the order of (logit, lower index first), a 64-bit key of which no two are
// alike, so what is wanted is one threshold key; and a token's weight follows from its bin (a quarter of a power of two wide, counted from E down) and its key:
//   1. parts of a row on workgroups of their own: histogram of the part's tokens and masses over the bins, relative to the part's own E;
//   2. the same parts: the row's histogram (the parts', shifted) says in which bins the cuts can be; the part lists its tokens there, and adds up what is
//      certainly kept;
//   3. one workgroup a row: the cuts exactly, from the listed tokens; the mass of every part; the part in which the pick is, token by token.
// What is listed is a few hundred tokens as a rule, and a row's all in the worst case (all logits alike), for which there is room.
#include <algorithm>

#include "wick_rocm_device.h"
#include "wick_rocm_internal.h"

namespace wick_rocm {

namespace {

constexpr uint32_t kPart = 4096, kMaxParts = kSampleMaxTokens / kPart;  // tokens of a part
constexpr int kOctaves = 46, kSteps = 4;                                // bins: kSteps to a power of two
constexpr uint32_t kBins = kOctaves * kSteps;
constexpr int kFraction = 43;  // masses are whole numbers of 2^-43: up to 2^19 tokens of less than 2 each
constexpr double kLog2e = 1.4426950408889634;
constexpr double kNever = -__builtin_inf(), kInfinite = 0x1p1000;       // y of what is never taken, and of an infinite logit

struct SamplePart {
    double top;       // E of the part; kNever: nothing to take
    uint64_t sure;    // mass that is certainly kept
    float largest;    // logit
    uint32_t listed, pad[2];
    uint32_t count[kBins];
    uint64_t mass[kBins];
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
};
__device__ __forceinline__ Rule rule_of(const SampleArgs& a, uint32_t row) {
    const wick_rocm_sample_params p = a.params[row];
    Rule r{kLog2e, p.top_k == 0 ? a.n : min(p.top_k, a.n), p.top_p >= 0.0f ? fmin((double)p.top_p, 1.0) : p.top_p < 0.0f ? 0.0 : 1.0,
           p.min_p >= 0.0f ? fmin((double)p.min_p, 1.0) : 0.0};
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

// (logit, lower index first) as one number; the logit is none that is never taken.
__device__ __forceinline__ uint64_t key_of(float l, uint32_t i) {
    const uint32_t b = __float_as_uint(l + 0.0f);  // (the zeros alike)
    return (uint64_t)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | (uint32_t)~i;
}

__device__ __forceinline__ uint64_t shuffle_up(uint64_t v, int d) { return (uint64_t)__shfl_up((unsigned long long)v, d, 64); }
__device__ __forceinline__ uint64_t lanes_upto(uint64_t v) {
    const uint32_t lane = threadIdx.x & 63u;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t other = shuffle_up(v, d);
        if (lane >= (uint32_t)d) v += other;
    }
    return v;
}
// Sum over the workgroup's threads in front of this one, and over all of them.
template <uint32_t WAVES>
__device__ __forceinline__ uint64_t sum_before(uint64_t v, uint64_t* slots, uint64_t& total) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint64_t upto = lanes_upto(v);
    __syncthreads();
    if (lane == 63u) slots[wave] = upto;
    __syncthreads();
    uint64_t before = upto - v;
    total = 0;
    for (uint32_t w = 0; w < WAVES; w++) {
        if (w < wave) before += slots[w];
        total += slots[w];
    }
    return before;
}

constexpr uint32_t kPartThreads = 256, kPartLoads = kPart / kPartThreads;

// 1.
__global__ __launch_bounds__(kPartThreads) void sample_bins_kernel(SampleArgs a) {
    __shared__ uint32_t count[kBins];
    __shared__ unsigned long long mass[kBins];
    __shared__ float tops[kPartThreads / 64];
    const uint32_t row = blockIdx.y, first = blockIdx.x * kPart;
    const float* const logits = a.logits + (size_t)row * a.stride;
    const Rule r = rule_of(a, row);
    float l[kPartLoads], top = -__builtin_inff();
#pragma unroll
    for (uint32_t k = 0; k < kPartLoads; k++) {
        const uint32_t i = first + k * kPartThreads + threadIdx.x;
        l[k] = i < a.n ? logits[i] : -__builtin_inff();
        top = fmaxf(top, l[k]);  // (NaN is passed over)
    }
    for (uint32_t b = threadIdx.x; b < kBins; b += kPartThreads) count[b] = 0, mass[b] = 0;
    top = wave_max_f32(top);
    if ((threadIdx.x & 63u) == 0) tops[threadIdx.x >> 6] = top;
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < kPartThreads / 64; w++) top = fmaxf(top, tops[w]);
    const double most = power_of(top, r), e = __builtin_floor(most);
    if (most > kNever) {
#pragma unroll
        for (uint32_t k = 0; k < kPartLoads; k++) {
            const double y = power_of(l[k], r);
            const uint32_t b = y > kNever ? bin_of(y, e) : kBins;
            if (b < kBins) atomicAdd(&count[b], 1u), atomicAdd(&mass[b], (unsigned long long)weight_of(y, e));
        }
    }
    __syncthreads();
    SamplePart& part = a.parts[(size_t)row * a.n_parts + blockIdx.x];
    if (threadIdx.x == 0) part.top = most > kNever ? e : kNever, part.largest = top;
    for (uint32_t b = threadIdx.x; b < kBins; b += kPartThreads) part.count[b] = count[b], part.mass[b] = mass[b];
}

// A row's histogram from its parts', each bin with those in front of it, and where the cuts can be.
struct RowBins {
    double top, floor;  // floor: the mass that min-p asks for
    uint64_t mass[kBins];
    uint32_t count[kBins];
};
struct Cuts {
    uint32_t k_bin;            // the bin with the top_k-th token; kBins: all are taken
    uint32_t p_first, p_last;  // bins that the nucleus can end in (top_p < 1)
    __device__ __forceinline__ uint32_t sure() const { return min(k_bin, p_first); }  // the first bin that is not kept for certain
    __device__ __forceinline__ bool lists(uint32_t b) const { return b == k_bin || (b >= p_first && b <= p_last); }
};

// The first bin up to which there is at least `target`, or kBins.
template <typename T>
__device__ __forceinline__ uint32_t first_reaching(const T* upto, T target) {
    uint32_t low = 0, high = kBins;
    while (low < high) {
        const uint32_t mid = (low + high) / 2u;
        if (upto[mid] >= target) high = mid;
        else low = mid + 1u;
    }
    return low;
}
__device__ __forceinline__ uint64_t share_of_mass(double share, uint64_t mass) {  // at least 1, so that a token is taken
    const uint64_t t = (uint64_t)__builtin_ceil(share * (double)mass);
    return t == 0 ? 1u : t < mass ? t : mass;
}

template <uint32_t THREADS>
__device__ __forceinline__ Cuts row_bins(const SampleArgs& a, uint32_t row, const Rule& r, RowBins& bins) {
    static_assert(THREADS >= kBins);
    const SamplePart* const parts = a.parts + (size_t)row * a.n_parts;
    double top = kNever;
    float largest = -__builtin_inff();
    for (uint32_t p = 0; p < a.n_parts; p++) top = fmax(top, parts[p].top), largest = fmaxf(largest, parts[p].largest);
    if (threadIdx.x < kBins) {
        uint32_t count = 0;
        uint64_t mass = 0;
        for (uint32_t p = 0; p < a.n_parts; p++) {
            const double off = top - parts[p].top;  // whole; infinite or NaN where a part has nothing
            if (!(off < (double)kOctaves) || threadIdx.x < (uint32_t)off * kSteps) continue;
            const uint32_t b = threadIdx.x - (uint32_t)off * kSteps;
            count += parts[p].count[b], mass += parts[p].mass[b] >> (uint32_t)off;
        }
        bins.count[threadIdx.x] = count, bins.mass[threadIdx.x] = mass;
    }
    if (threadIdx.x == 0) bins.top = top, bins.floor = top > kNever ? r.min_p * (double)weight_of(power_of(largest, r), top) : 0.0;
    __syncthreads();
    if (threadIdx.x < 64u) {  // every bin with those in front of it
        constexpr uint32_t kEach = (kBins + 63u) / 64u;
        uint64_t sum = 0, tokens = 0;
        for (uint32_t i = 0; i < kEach; i++)
            if (const uint32_t b = threadIdx.x * kEach + i; b < kBins) sum += bins.mass[b], tokens += bins.count[b];
        sum = lanes_upto(sum) - sum, tokens = lanes_upto(tokens) - tokens;
        for (uint32_t i = 0; i < kEach; i++)
            if (const uint32_t b = threadIdx.x * kEach + i; b < kBins) bins.mass[b] = sum += bins.mass[b], bins.count[b] = (uint32_t)(tokens += bins.count[b]);
    }
    __syncthreads();
    Cuts c{first_reaching(bins.count, r.top_k), kBins, 0};
    if (r.top_p < 1.0) {
        // the mass of what top-k leaves lies between that in front of its bin and that with it
        const uint64_t all = bins.mass[kBins - 1], least = c.k_bin == kBins ? all : c.k_bin == 0 ? 0 : bins.mass[c.k_bin - 1], most = c.k_bin == kBins ? all : bins.mass[c.k_bin];
        c.p_first = min(first_reaching(bins.mass, share_of_mass(r.top_p, least)), c.k_bin);
        c.p_last = min(first_reaching(bins.mass, share_of_mass(r.top_p, most)), c.k_bin);
    }
    return c;
}

// 2.
__global__ __launch_bounds__(kPartThreads) void sample_list_kernel(SampleArgs a) {
    __shared__ RowBins bins;
    __shared__ uint64_t slots[kPartThreads / 64];
    __shared__ uint32_t listed;
    const uint32_t row = blockIdx.y, first = blockIdx.x * kPart;
    const float* const logits = a.logits + (size_t)row * a.stride;
    const Rule r = rule_of(a, row);
    float l[kPartLoads];
#pragma unroll
    for (uint32_t k = 0; k < kPartLoads; k++) {
        const uint32_t i = first + k * kPartThreads + threadIdx.x;
        l[k] = i < a.n ? logits[i] : -__builtin_inff();
    }
    if (threadIdx.x == 0) listed = 0;
    const Cuts cuts = row_bins<kPartThreads>(a, row, r, bins);
    const double top = bins.top;
    if (!(top > kNever)) return;
    uint64_t sure = 0;
    uint32_t* const list = a.lists + (size_t)row * a.n + first;
#pragma unroll
    for (uint32_t k = 0; k < kPartLoads; k++) {
        const uint32_t i = first + k * kPartThreads + threadIdx.x;
        const double y = power_of(l[k], r);
        const uint32_t b = y > kNever ? bin_of(y, top) : kBins;
        if (b >= kBins) continue;
        if (b < cuts.sure()) {
            const uint64_t w = weight_of(y, top);
            sure += (double)w >= bins.floor ? w : 0;
        } else if (cuts.lists(b)) list[atomicAdd(&listed, 1u)] = i;
    }
    uint64_t all;
    sum_before<kPartThreads / 64>(sure, slots, all);
    SamplePart& part = a.parts[(size_t)row * a.n_parts + blockIdx.x];
    if (threadIdx.x == 0) part.sure = all, part.listed = listed;
}

// 3.
constexpr uint32_t kPickThreads = 1024, kPickWaves = kPickThreads / 64, kDigit = 11, kDigits = 1u << kDigit;

struct Token {
    uint64_t key, weight;
    uint32_t part, bin;
};
struct PickShared {
    RowBins bins;
    uint64_t slots[kPickWaves], part_mass[kMaxParts], found[3];
    uint32_t listed[kMaxParts + 1];
    union {
        struct {
            uint64_t key[kPickThreads], weight[kPickThreads];
        } few;
        struct {
            uint32_t count[kDigits];
            unsigned long long mass[kDigits];
        } many;
    };
};

__device__ __forceinline__ uint64_t lanes_min(uint64_t v) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t other = (uint64_t)__shfl_xor((unsigned long long)v, d, 64);
        v = other < v ? other : v;
    }
    return v;
}

struct Picker {
    const SampleArgs& a;
    const Rule& r;
    PickShared& sh;
    uint32_t row, tokens;  // tokens: listed ones

    // Listed token f.
    __device__ __forceinline__ Token token(uint32_t f) const {
        uint32_t low = 0, high = a.n_parts;
        while (high - low > 1) {
            const uint32_t mid = (low + high) / 2u;
            (sh.listed[mid] <= f ? low : high) = mid;
        }
        const uint32_t i = a.lists[(size_t)row * a.n + (size_t)low * kPart + (f - sh.listed[low])];
        const float l = a.logits[(size_t)row * a.stride + i];
        const double y = power_of(l, r);
        return {key_of(l, i), weight_of(y, sh.bins.top), low, bin_of(y, sh.bins.top)};
    }

    // Of the listed tokens of one bin, from the largest key (all at or above `least`) down, as many as are `target` tokens, or as their masses take
    // to reach `target`: the smallest key of those, and their mass.
    __device__ __forceinline__ void select(uint32_t bin, uint64_t least, uint64_t target, bool by_mass, const Token& mine, uint64_t& threshold, uint64_t& mass) {
        if (tokens <= kPickThreads) {  // every thread one token: what is above it
            const bool in = threadIdx.x < tokens && mine.bin == bin && mine.key >= least;
            __syncthreads();
            sh.few.key[threadIdx.x] = in ? mine.key : 0, sh.few.weight[threadIdx.x] = mine.weight;
            __syncthreads();
            uint64_t before = 0;
            if (in)
                for (uint32_t j = 0; j < tokens; j++) before += sh.few.key[j] > mine.key ? (by_mass ? sh.few.weight[j] : 1u) : 0u;
            const bool taken = in && before < target;
            const uint64_t low = lanes_min(taken ? mine.key : ~0ull);
            sum_before<kPickWaves>(taken ? mine.weight : 0, sh.slots, mass);
            __syncthreads();
            if ((threadIdx.x & 63u) == 0) sh.slots[threadIdx.x >> 6] = low;
            __syncthreads();
            threshold = ~0ull;
            for (uint32_t w = 0; w < kPickWaves; w++) threshold = min(threshold, sh.slots[w]);
            return;
        }
        threshold = 0, mass = 0;
        uint64_t left = target;
        for (int known = 64, shift = 64 - (int)kDigit;; known = shift, shift = shift > (int)kDigit ? shift - (int)kDigit : 0) {
            // digits from the highest; the last one overlaps the one before it, whose bits are the same for all that are left
            __syncthreads();
            if (threadIdx.x == 0) sh.found[0] = sh.found[1] = sh.found[2] = 0;
            for (uint32_t d = threadIdx.x; d < kDigits; d += kPickThreads) sh.many.count[d] = 0, sh.many.mass[d] = 0;
            __syncthreads();
            for (uint32_t f = threadIdx.x; f < tokens; f += kPickThreads) {
                const Token t = token(f);
                if (t.bin != bin || t.key < least || (known < 64 && t.key >> known != threshold >> known)) continue;
                const uint32_t d = (uint32_t)(t.key >> shift) & (kDigits - 1u);
                atomicAdd(&sh.many.count[d], 1u), atomicAdd(&sh.many.mass[d], (unsigned long long)t.weight);
            }
            __syncthreads();
            // thread t has digits 2047 - 2 t and the one below
            const uint32_t d0 = kDigits - 1u - 2u * threadIdx.x, d1 = d0 - 1u;
            const uint64_t n0 = by_mass ? sh.many.mass[d0] : sh.many.count[d0], n1 = by_mass ? sh.many.mass[d1] : sh.many.count[d1];
            const uint64_t m0 = sh.many.mass[d0], m1 = sh.many.mass[d1];
            uint64_t all, all_mass;
            const uint64_t before = sum_before<kPickWaves>(n0 + n1, sh.slots, all), mass_before = sum_before<kPickWaves>(m0 + m1, sh.slots, all_mass);
            const uint64_t goal = left < all ? left : all;  // (what there is may be a little less than the bins' masses said)
            __syncthreads();
            if (before < goal && goal <= before + n0 + n1) {
                const bool second = goal > before + n0;
                sh.found[0] = second ? d1 : d0, sh.found[1] = goal - before - (second ? n0 : 0), sh.found[2] = mass_before + (second ? m0 : 0);
            }
            __syncthreads();
            const uint64_t digit = sh.found[0];
            left = sh.found[1], mass += sh.found[2];
            threshold = (threshold & ~((uint64_t)(kDigits - 1u) << shift)) | digit << shift;
            if (shift == 0) {
                mass += sh.many.mass[digit];  // the one token of this key
                return;
            }
        }
    }
};

__global__ __launch_bounds__(kPickThreads) void sample_pick_kernel(SampleArgs a) {
    __shared__ PickShared sh;
    const uint32_t row = blockIdx.x;
    const float* const logits = a.logits + (size_t)row * a.stride;
    const SamplePart* const parts = a.parts + (size_t)row * a.n_parts;
    const Rule r = rule_of(a, row);
    const Cuts cuts = row_bins<kPickThreads>(a, row, r, sh.bins);
    const double top = sh.bins.top, floor = sh.bins.floor;
    if (!(top > kNever)) {
        if (threadIdx.x == 0) {
            a.out[row] = WICK_ROCM_NO_TOKEN;
            if (a.prob) a.prob[row] = 0.0f;
        }
        return;
    }
    if (threadIdx.x < kMaxParts) sh.part_mass[threadIdx.x] = threadIdx.x < a.n_parts ? parts[threadIdx.x].sure : 0;
    uint64_t tokens;
    const uint64_t upto = sum_before<kPickWaves>(threadIdx.x < a.n_parts ? parts[threadIdx.x].listed : 0, sh.slots, tokens);
    if (threadIdx.x < a.n_parts) sh.listed[threadIdx.x] = (uint32_t)upto;
    __syncthreads();
    Picker pick{a, r, sh, row, (uint32_t)tokens};
    Token mine{0, 0, 0, kBins};
    if (tokens <= kPickThreads && threadIdx.x < tokens) mine = pick.token(threadIdx.x);
    uint64_t threshold = 0;
    if (tokens != 0) {
        uint64_t mass = sh.bins.mass[kBins - 1];
        if (cuts.k_bin < kBins) {
            const uint32_t in_front = cuts.k_bin == 0 ? 0 : sh.bins.count[cuts.k_bin - 1];
            uint64_t in_bin;
            pick.select(cuts.k_bin, 0, r.top_k - in_front, false, mine, threshold, in_bin);
            mass = (cuts.k_bin == 0 ? 0 : sh.bins.mass[cuts.k_bin - 1]) + in_bin;
        }
        if (r.top_p < 1.0) {
            const uint64_t target = share_of_mass(r.top_p, mass);
            const uint32_t bin = max(min(min(first_reaching(sh.bins.mass, target), cuts.k_bin), cuts.p_last), cuts.p_first);
            const uint64_t in_front = bin == 0 ? 0 : sh.bins.mass[bin - 1];
            uint64_t in_bin;
            pick.select(bin, threshold, target > in_front ? target - in_front : 1, true, mine, threshold, in_bin);
        }
    }
    // what every part keeps
    for (uint32_t f = threadIdx.x; f < tokens; f += kPickThreads) {
        const Token t = tokens <= kPickThreads ? mine : pick.token(f);
        if (t.key >= threshold && (double)t.weight >= floor) atomicAdd(reinterpret_cast<unsigned long long*>(&sh.part_mass[t.part]), (unsigned long long)t.weight);
    }
    __syncthreads();
    uint64_t mass;
    const uint64_t in_part = threadIdx.x < a.n_parts ? sh.part_mass[threadIdx.x] : 0, in_front = sum_before<kPickWaves>(in_part, sh.slots, mass);
    if (threadIdx.x == 0) sh.found[0] = sh.found[1] = 0;
    const float u = a.uniform[row];
    const double at = (u > 0.0f ? (double)u : 0.0) * (double)mass;
    const uint64_t target = at < (double)mass ? min((uint64_t)at, mass - 1u) : mass - 1u;  // the pick is the first to exceed it
    __syncthreads();
    if (in_front <= target && target < in_front + in_part) sh.found[0] = threadIdx.x, sh.found[1] = target - in_front;
    __syncthreads();
    const uint32_t part = (uint32_t)sh.found[0];
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
    uint64_t all, before = sum_before<kPickWaves>(sum, sh.slots, all);
    if (before <= goal && goal < before + sum) {
        for (uint32_t k = 0; k < kPart / kPickThreads; before += weight[k++])
            if (goal < before + weight[k]) {
                const uint32_t i = part * kPart + threadIdx.x * (kPart / kPickThreads) + k;
                a.out[row] = i;
                if (a.prob) a.prob[row] = (float)(exact_weight(power_of(logits[i], r), top) / (double)mass);
                break;
            }
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
