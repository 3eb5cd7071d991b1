// Sampling a token of each row of logits, by temperature, top-k, top-p and min-p, from a given uniform number.
//
// Formulas. w_i = e^((l_i - max l) / T). Sorted by logit, equal ones by index: S1, the first k; S2, the shortest prefix of
// S1 with sum w >= p * (sum of S1's w); S3, those with w >= min_p. The token is the first of S2 and S3, by index, whose
// running sum of w passes u * (their sum).
//
// Numbers. A vocabulary has some 10^5 borders between tokens, and f32 weights, off by 2^-24, would put about one sample in
// 10^4 on the wrong side of one. Weights are e^x in double, and exactly 1 for the largest logit, so that rows of equal
// logits are cut at whole numbers of tokens; running sums are in double, in an order that the vocabulary alone sets. Sums
// over a histogram's bin are in fixed point (each weight to 2^-30 of itself or better), whose order does not matter, so
// atomics in LDS may take any.
//
// Launches, several workgroups ("parts") to a row in 1 and 3:
//   1 each part's largest logit and, of rows with a top-k or top-p, a histogram of its tokens' number and weight over the
//     logit, 1024 bins of T / 32 down from its largest's. Bins stand at fixed places of z = 32 l / T, not of the largest,
//     which no part knows: parts' histograms are shifted and added by whoever reads them. A weight is held relative to its
//     bin's middle, e^(f / 32) with f = z - rint z: a short polynomial and no table, and one atomic for number and sum.
//   2 one workgroup to a row (with a top-k or top-p): the row's histogram, and the bins in which the cuts fall
//   3 tokens above those bins are kept, and their weights' sums of blocks of 2048 tokens are written; tokens in them, some
//     hundreds, are listed
//   4 one workgroup to a row: the cuts within the list, its kept tokens' weights added to their blocks' sums, and the block
//     and in it the token that u falls on
//
// What bounds it: one row of 151936 f16 logits, 27 us, four launches that need each other (6.6, 9.1, 4.7 and 8.4 by
// themselves, most of each loads and barriers in turn). 128 such rows in f32, their settings mixed, 73 us: 26.5 of launch 1, of
// which 13 are the reading (6 TB/s, from the last-level cache in part) and the rest some 33 instructions a token, half of them
// in double (the same without the atomics); 9.3 of 2; 24 of 3, where rows that keep most of the vocabulary take the weights'
// exponentials again; 13.9 of 4. In f16 73 too (26.2, 9.4, 25.5 and 14.2): half the reading, the same arithmetic. Where a cut's
// bin holds more than 4096 tokens one workgroup reads the row again, some five times for a cut: 8 rows of 262144 logits of a
// spread of 0.2 at a temperature of 1.5, top-p 0.5, 413 us (44 with a spread of 1.2), one of 2^24 49 ms.
// Not kept: launch 3 by the polynomial for rows of many kept tokens too (rows with a top-p of 0.9 32 -> 37 us, of 0.99 46 -> 42);
// the largest logits of 64 tokens each, so that launch 3 reads no others (no faster, launch 1 1.7 us slower); the bins' polynomial
// with its scale in its coefficients (f32 28.0 -> 26.3, but f16 parts, of three steps then, spilled more: without a histogram 11.5 -> 14.7).
#include <algorithm>

#include "internal.h"
#include "paged_device.h"

namespace neko_hip {
namespace {

constexpr int kThreads = 1024;
constexpr int kBins = 1024;  // one to a thread; the last holds whatever is further down
constexpr double kBinsPerT = 32.0;
constexpr int kBlockTokens = 2048;               // of a sum: 256 threads of 8
constexpr int kStepTokens = kThreads * 8;        // four blocks
// Of a part: a thread holds its tokens in registers. Three of f16 spill beside their conversions (128 rows of 151936 with a
// top-k of 50 70.6 us, of two steps 56.3; with none of the cuts 45.8 and 41.9).
template <typename T>
constexpr int kMostSteps = sizeof(T) == 2 ? 2 : 3;
constexpr int kMostBlocks = 16;                  // of a workgroup in launch 3
// Rows' counters a cache line apart: workgroups of all XCDs add to them (launch 3 of 128 rows with a top-k of 50 17 us, on four
// lines 21).
constexpr int kLine = 32;
constexpr int kGroupListed = 512;                // tokens of its own that one lists in LDS first
constexpr int kListed = 4096;                    // tokens in the cuts' bins that are held in LDS
// Parts' bins that are on their way at once in launch 2: a round holds those of one row of 160 thousand tokens, of which each part
// is one step; more take rounds.
constexpr int kAtOnce = 20;
constexpr int kRanked = 256;                     // of those, what is sorted by ranks
constexpr int64_t kSlabRows = 1024;              // of a launch: the workspace holds so many,
constexpr size_t kSlabBytes = size_t(256) << 20; // or as many as take this
constexpr uint32_t kMinusInf = 0x007fffffu;      // its key; tokens at or below are left out

// What launch 1 leaves of a part.
struct Part {
    uint64_t best;    // key << 32 | ~index of its largest (greedy rows; the others' has no index)
    double weight;    // its tokens' weights, relative to the middle of its largest's bin
    uint32_t count;   // its tokens
    uint32_t unused;
};

// What launch 2 finds of a row (of one without cuts, `best` alone): cuts that fall into bins lo .. hi (top-p) and by_k (top-k: after `need` of its tokens).
struct Found {
    int32_t lo, hi, bin_k;
    uint32_t need;
    uint32_t listed;            // tokens of those bins
    // Logits: at least above_lo, in a bin before lo; at least above_hi, up to hi; at least above_k and not before_k, bin_k's
    // (where that is past hi). NaN: none.
    float above_lo, above_hi, above_k, before_k;
    uint32_t few;               // all tokens that may stay are listed, up to kRanked
    uint64_t best;              // as of launch 1, over the row's parts
    double below_lo, below_k;   // weights' sums of the bins before lo and bin_k
    double total;               // of the row
};  // (weights relative to the row's largest)

struct SampleArgs {
    const void* logits;
    int64_t stride;
    const float* temperature;  // each per row or null
    const int32_t* top_k;
    const float* top_p;
    const float* min_p;
    const float* u;
    int32_t* out;
    int32_t vocab;
    int32_t parts, part_tokens;  // of a row; whole steps
    int32_t n_blocks;            // blocks of a row
    int32_t groups, group_blocks;  // workgroups of a row in launch 3, and their blocks
    int32_t count_bits;          // the low bits of a bin: its tokens; the others: their weights in units of 2^-fixed
    int32_t fixed;
    int32_t narrow;              // fixed-point weights of a cut's parts, relative to the row's largest: units of 2^-narrow, and of 2^-32 of those
    Part* part;                  // [rows][parts]
    uint64_t* bins;              // [rows][parts][kBins]
    Found* found;                // [rows]
    uint32_t* listed;            // [rows][kLine] tokens listed so far
    uint64_t* list;              // [rows][kListed] ~key << 32 | index: ascending is the order of the cuts
    double* sums;                // [rows][n_blocks]
};

// What a row asks for, as its numbers are read: a temperature that is not positive is the largest logit's token, a k not
// positive, a p of 1 or more and a min_p not positive cut off nothing, nor does a NaN.
struct Row {
    bool greedy, by_k, by_p;
    double inv_t, p, min_p;
    int32_t k;
    __device__ bool cuts() const { return !greedy && (by_k || by_p); }
};
__device__ __forceinline__ Row row_of(const SampleArgs& a, int64_t r) {
    Row w;
    const float t = a.temperature ? a.temperature[r] : 1.0f;
    w.greedy = !(t > 0.0f);
    w.inv_t = 1.0 / static_cast<double>(t);
    w.k = a.top_k ? a.top_k[r] : 0;
    w.by_k = w.k > 0 && w.k < a.vocab;
    const float p = a.top_p ? a.top_p[r] : 1.0f;
    w.by_p = p < 1.0f;
    w.p = static_cast<double>(p);
    const float m = a.min_p ? a.min_p[r] : 0.0f;
    w.min_p = m > 0.0f ? fminf(m, 1.0f) : 0.0;
    return w;
}

// Keys in the order of the values, both zeros alike; NaN as -inf.
__device__ __forceinline__ uint32_t key_of(float l) {
    const uint32_t b = __builtin_bit_cast(uint32_t, l + 0.0f);
    const uint32_t k = b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
    return l != l ? kMinusInf : k;
}
__device__ __forceinline__ float value_of(uint32_t k) {
    return __builtin_bit_cast(float, k ^ (k & 0x80000000u ? 0x80000000u : 0xffffffffu));
}

// A logit's place among the bins, monotone in it as every rounding here is, and the number of its bin down from that of
// place `top`. (An infinite logit stands at 1e300; an infinite temperature leaves all finite ones in one bin.)
__device__ __forceinline__ double bins_per(double inv_t) { return fmax(kBinsPerT * inv_t, 1e-300); }
__device__ __forceinline__ double place_of(float l, double inv_t) { return fmin(static_cast<double>(l) * bins_per(inv_t), 1e300); }
__device__ __forceinline__ int bin_at(double place, double top) { return static_cast<int>(fmax(fmin(rint(top) - rint(place), kBins - 1.0), 0.0)); }
// From this place on other logits than the largest are at least 2^21 bins away, and only those equal to it weigh anything.
constexpr double kFarPlace = 0x1p45;
// What a logit lies past the middle of its bin, that of place g: the product's exact value counts (a rounded one is off by 2^-53
// of the place, 2^-26 of the weight for a logit of 2^27 temperatures).
__device__ __forceinline__ double past_middle(float l, double per, double g) { return __builtin_fma(static_cast<double>(l), per, -g); }
// e^(f / 32) for -1/2 <= f <= 1/2, and a little more: the series, cut off by (1/64)^5 / 5! = 8e-12 or (LONG) (1/64)^7 / 7! = 5e-17.
template <bool LONG>
__device__ __forceinline__ double edge_weight(double f) {
    const double x = f * (1.0 / 32.0);
    double y = LONG ? __builtin_fma(x, 1.0 / 720.0, 1.0 / 120.0) : 1.0 / 24.0;
    if (LONG) y = __builtin_fma(x, y, 1.0 / 24.0);
    y = __builtin_fma(x, y, 1.0 / 6.0);
    y = __builtin_fma(x, y, 0.5);
    y = __builtin_fma(x, y, 1.0);
    return __builtin_fma(x, y, 1.0);
}
// The same in fixed point, cut down to units of 2^-fixed and shifted by count_bits, as a bin sums it up: the low bits of
// its sum with 2^52, whose own high bits come with it.
constexpr uint64_t kHigh = 0x4330000000000000ull;
__device__ __forceinline__ uint64_t bin_weight(double f, double units, uint32_t count_mask) {
    const uint64_t y = __builtin_bit_cast(uint64_t, __builtin_fma(edge_weight<false>(f), units, 0x1p52));
    return (y & 0xffffffff00000000ull) | (static_cast<uint32_t>(y) & ~count_mask);
}
// A weight of launch 3 without cuts -- two tables' values, the polynomial and their products, from the same exponent -- and
// weight_of differ by less than five units of 2^-52, so where they may fall on either side of a number this tells.
constexpr double kNear = 0x1p-48;
__device__ __forceinline__ double weight_of(float l, float top, double inv_t) {
    const double w = exp((static_cast<double>(l) - static_cast<double>(top)) * inv_t);
    return l == top ? 1.0 : w == w ? w : 0.0;  // (no number: an infinite distance at an infinite temperature)
}
// w * units, rounded, below 2^52: the low bits of its sum with 2^52.
__device__ __forceinline__ uint64_t fixed_of(double w, double units) {
    return __builtin_bit_cast(uint64_t, __builtin_fma(w, units, 0x1p52)) - __builtin_bit_cast(uint64_t, 0x1p52);
}

// What that leaves of w * units, half a unit at most either way, in 2^-32 of one (a sum of 2^24 of them below 2^56). units: a
// power of two, so that both differences are exact.
__device__ __forceinline__ uint64_t fixed_left(double w, double units) {
    const double left = __builtin_fma(w, units, -(__builtin_fma(w, units, 0x1p52) - 0x1p52));
    return __builtin_bit_cast(uint64_t, __builtin_fma(left, 0x1p32, 0x1.8p52)) - __builtin_bit_cast(uint64_t, 0x1.8p52);
}

// Logits i .. i + 7 of a row, -inf from n on. Rows may stand at any element.
template <typename T>
struct Eight {
    T v[8];
};
template <typename T>
__device__ __forceinline__ Eight<T> load8(const T* row, int32_t i, int32_t n) {
    Eight<T> x;
    if (i + 8 <= n) {
        __builtin_memcpy(x.v, row + i, sizeof(x.v));
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) x.v[e] = i + e < n ? row[i + e] : static_cast<T>(-__builtin_inff());
    }
    return x;
}

__device__ __forceinline__ uint64_t wave_max_u64(uint64_t v) {
    const uint32_t hi = static_cast<uint32_t>(v >> 32), most = wave_max_u32(hi);
    return static_cast<uint64_t>(most) << 32 | wave_max_u32(hi == most ? static_cast<uint32_t>(v) : 0u);
}

// The largest logit of a row, from launch 1's parts, by every wave for itself: key << 32 | ~index.
__device__ __forceinline__ uint64_t best_of_parts(const SampleArgs& a, int64_t r) {
    uint64_t b = 0;
    for (int32_t i = static_cast<int32_t>(threadIdx.x) & 63; i < a.parts; i += 64) {
        const uint64_t o = a.part[r * a.parts + i].best;
        b = b > o ? b : o;
    }
    return wave_max_u64(b);
}
__device__ __forceinline__ uint64_t row_best(const SampleArgs& a, int64_t r) {
    return a.top_k || a.top_p ? a.found[r].best : best_of_parts(a, r);
}

typedef unsigned long long u64;

// Inclusive sum over the lanes below and at each, within 16 lanes and on (DPP, as wave_scan_u32).
template <typename V>
__device__ __forceinline__ V wave_scan(V v) {
    auto add = [&](auto ctrl, auto rows) {
        if constexpr (sizeof(V) == 4) {
            v += __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), decltype(ctrl)::value, decltype(rows)::value, 0xF, false));
        } else {
            const uint64_t b = __builtin_bit_cast(uint64_t, v);
            const uint32_t lo = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(static_cast<uint32_t>(b)), decltype(ctrl)::value, decltype(rows)::value, 0xF, false));
            const uint32_t hi = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(static_cast<uint32_t>(b >> 32)), decltype(ctrl)::value, decltype(rows)::value, 0xF, false));
            v += __builtin_bit_cast(V, static_cast<uint64_t>(hi) << 32 | lo);
        }
    };
    add(std::integral_constant<int, 0x111>{}, std::integral_constant<int, 0xF>{});  // row_shr 1, 2, 4, 8
    add(std::integral_constant<int, 0x112>{}, std::integral_constant<int, 0xF>{});
    add(std::integral_constant<int, 0x114>{}, std::integral_constant<int, 0xF>{});
    add(std::integral_constant<int, 0x118>{}, std::integral_constant<int, 0xF>{});
    add(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xA>{});  // row_bcast 15 into rows 1 and 3
    add(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xC>{});  // row_bcast 31 into rows 2 and 3
    return v;
}
// The sum of the threads' values up to each thread's own. sh: one for each wave.
template <typename V>
__device__ __forceinline__ V block_scan(V* sh, V v) {
    const int lane = static_cast<int>(threadIdx.x) & 63, wave = static_cast<int>(threadIdx.x) >> 6;
    v = wave_scan(v);
    __syncthreads();
    if (lane == 63) sh[wave] = v;
    __syncthreads();
    const V before = wave_scan(lane < wave ? sh[lane] : V(0));
    if constexpr (sizeof(V) == 8) return readlane_f64(before, 63) + v;
    else return static_cast<V>(__builtin_amdgcn_readlane(static_cast<int>(before), 63)) + v;
}


// The first (or LAST) thread of which something holds, kThreads (-1) if it holds of none. (Atomics on one address by all
// threads took 12 us.)
template <bool LAST>
__device__ __forceinline__ int block_first(int32_t* sh, bool is) {
    const int wave = static_cast<int>(threadIdx.x) >> 6;
    const uint64_t in = __ballot(is);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[wave] = in ? 64 * wave + (LAST ? 63 - __builtin_clzll(in) : __builtin_ctzll(in)) : LAST ? -1 : kThreads;
    __syncthreads();
    int v = sh[0];
#pragma unroll
    for (int i = 1; i < kThreads / 64; i++) v = LAST ? std::max(v, sh[i]) : std::min(v, sh[i]);
    return v;
}

// ------------------------------------------------------------------ 1: parts' largest and histograms

// STEPS: of the call's parts.
template <typename T, int STEPS>
__global__ __launch_bounds__(kThreads, 8) void sample_parts(SampleArgs a) {
    __shared__ u64 bins[kBins];
    __shared__ uint32_t sh_top[kThreads / 64];
    __shared__ uint32_t sh_at;
    __shared__ double sh_sum[kThreads / 64];
    __shared__ uint32_t sh_count[kThreads / 64];
    const int tid = static_cast<int>(threadIdx.x), lane = tid & 63;
    const int64_t r = blockIdx.x / static_cast<uint32_t>(a.parts);
    const int32_t part = static_cast<int32_t>(blockIdx.x - static_cast<uint32_t>(r) * static_cast<uint32_t>(a.parts));
    const int32_t begin = part * a.part_tokens + tid * 8;
    Eight<T> x[STEPS];
#pragma unroll
    for (int s = 0; s < STEPS; s++) x[s] = load8(static_cast<const T*>(a.logits) + r * a.stride, begin + s * kStepTokens, a.vocab);
    const Row w = row_of(a, r);
    float top = -__builtin_inff();
#pragma unroll
    for (int s = 0; s < STEPS; s++)
#pragma unroll
        for (int e = 0; e < 8; e++) top = fmaxf(top, to_f32(x[s].v[e]));  // (the other one of a NaN)
    bins[tid] = 0;
    if (tid == 0) sh_at = 0xffffffffu;
    uint32_t key = wave_max_u32(key_of(top));
    if (lane == 0) sh_top[tid >> 6] = key;
    __syncthreads();
    key = wave_max_u32(sh_top[lane & (kThreads / 64 - 1)]);
    top = value_of(key);
    Part* out = a.part + blockIdx.x;
    if (w.greedy) {
        // The first that has it.
        uint32_t at = 0xffffffffu;
#pragma unroll
        for (int s = STEPS - 1; s >= 0; s--)
#pragma unroll
            for (int e = 7; e >= 0; e--)
                if (to_f32(x[s].v[e]) == top) at = static_cast<uint32_t>(begin + s * kStepTokens + e);
        if (at != 0xffffffffu) atomicMin(&sh_at, at);
        __syncthreads();
        if (tid == 0) out->best = static_cast<uint64_t>(key) << 32 | (0xffffffffu - sh_at);
        return;
    }
    if (tid == 0) {
        out->best = static_cast<uint64_t>(key) << 32;
        if (part == 0) a.listed[r * kLine] = 0;
    }
    if (!w.cuts() || key <= kMinusInf) return;
    const double per = bins_per(w.inv_t), first = rint(place_of(top, w.inv_t)), units = ldexp(1.0, a.fixed + a.count_bits);
    const uint32_t mask = (1u << a.count_bits) - 1;
    double further = 0.0;  // what the last bin's tokens weigh
    uint32_t n = 0;        // and how many there are
    if (fabs(first) >= kFarPlace) {  // (infinities too)
#pragma unroll
        for (int s = 0; s < STEPS; s++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float l = to_f32(x[s].v[e]);
                if (l == top) atomicAdd(&bins[0], static_cast<u64>(bin_weight(0.0, units, mask) | 1u));
                else if (l > -__builtin_inff()) n++;
            }
    } else {
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            u64 y[8];
            int b[8];
            bool far = false;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float l = fmaxf(to_f32(x[s].v[e]), -__builtin_inff());  // (NaN: -inf)
                const double g = rint(static_cast<double>(l) * per);
                b[e] = static_cast<int>(fmin(first - g, kBins - 1.0));
                y[e] = bin_weight(past_middle(l, per, g), units, mask) | 1u;
                far |= b[e] == kBins - 1 && l > -__builtin_inff();
            }
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (b[e] < kBins - 1) atomicAdd(&bins[b[e]], y[e]);
            if (__any(far)) {
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float l = to_f32(x[s].v[e]);
                    if (b[e] == kBins - 1 && l > -__builtin_inff()) {
                        n++;
                        further += exp((static_cast<double>(l) * per - first) * (1.0 / kBinsPerT));
                    }
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    __syncthreads();
    // (without the high bits of each 2^52)
    u64 mine = bins[tid];
    mine -= (mine & mask) * kHigh;
    a.bins[static_cast<int64_t>(blockIdx.x) * kBins + tid] = mine;
    n += static_cast<uint32_t>(mine) & mask;
    const double sum = static_cast<double>(mine >> a.count_bits) * ldexp(exp(tid * (-1.0 / kBinsPerT)), -a.fixed) + further;
    const double sums = wave_sum_f64(sum);
    const uint32_t counts = wave_scan(n);
    if (lane == 63) {
        sh_sum[tid >> 6] = sums;
        sh_count[tid >> 6] = counts;
    }
    __syncthreads();
    if (tid == 0) {
        double all = 0.0;
        uint32_t many = 0;
        for (int i = 0; i < kThreads / 64; i++) {
            all += sh_sum[i];
            many += sh_count[i];
        }
        out->count = many;
        out->weight = all;
    }
}

// ------------------------------------------------------------------ 2: the cuts' bins

// Thread t's bin of the row, counted down from the largest's: its tokens and their weights, relative to the row's largest.
// sh_off, sh_n, sh_by: by part, a round of kThreads parts at a time. held: where there are at most 64, each lane's.
__device__ __forceinline__ void row_bin(const SampleArgs& a, int64_t r, const Row& w, float top, const Part& held, int* sh_off, uint32_t* sh_n, double* sh_by, uint32_t* count,
                                        double* weight, uint32_t* all, double* total) {
    const int t = static_cast<int>(threadIdx.x);
    const double place = place_of(top, w.inv_t), first = rint(place);
    // (in units of the largest's own fixed-point weight)
    const double rest = fabs(first) < kFarPlace ? past_middle(top, bins_per(w.inv_t), first) : 0.0;
    const double unit = static_cast<double>((bin_weight(rest, ldexp(1.0, a.fixed + a.count_bits), (1u << a.count_bits) - 1) - kHigh) >> a.count_bits);
    uint32_t n = 0, n_all = 0;
    double s = 0.0, s_all = 0.0, edge = 0.0;
    const uint64_t* bins = a.bins + r * a.parts * kBins;
    for (int32_t i0 = 0; i0 < a.parts; i0 += kThreads) {
        const int32_t here = std::min(a.parts - i0, kThreads);
        __syncthreads();
        for (int32_t i = t; i < here + kAtOnce; i += kThreads) {  // (past the last: parts that hold nothing)
            int off = -1;
            double by = 0.0;
            uint32_t many = 0;
            if (i < here) {
                const Part p = a.parts <= 64 ? held : a.part[r * a.parts + i0 + i];
                const uint32_t key = static_cast<uint32_t>(p.best >> 32);
                if (key > kMinusInf) {
                    const double its = place_of(value_of(key), w.inv_t);
                    off = bin_at(its, place);
                    by = p.weight * exp((rint(its) - rint(place)) * (1.0 / kBinsPerT));
                    many = p.count;
                }
            }
            sh_off[i] = off;
            sh_by[i] = by;
            sh_n[i] = many;
        }
        __syncthreads();
        for (int32_t i = 0; i < here; i += kAtOnce) {
            u64 x[kAtOnce];
#pragma unroll
            for (int j = 0; j < kAtOnce; j++) {
                const int off = sh_off[i + j];
                x[j] = 0;
                if (off >= 0 && t >= off && t < kBins - 1) {
                    const uint32_t at = (static_cast<uint32_t>(i0 + i + j) * kBins + static_cast<uint32_t>(t - off)) * 8u;
                    x[j] = *reinterpret_cast<const u64*>(reinterpret_cast<const char*>(bins) + at);
                }
            }
            if (i0 == 0 && i == 0) edge = exp(t * (-1.0 / kBinsPerT)) / unit;  // (while they are on their way)
#pragma unroll
            for (int j = 0; j < kAtOnce; j++) {
                n += static_cast<uint32_t>(x[j]) & ((1u << a.count_bits) - 1);
                s += static_cast<double>(x[j] >> a.count_bits);
                s_all += sh_by[i + j];
                n_all += sh_n[i + j];
            }
        }
    }
    // (the first bin's by a quotient: equal logits sum up to whole numbers)
    *count = n;
    *weight = t == 0 ? s / unit : s * edge;
    *all = n_all;
    *total = ldexp(s_all, a.fixed) / unit;
}

// The smallest logit of the bins up to b, down from place `top`'s: a logit is of those if it is at least that (b = -1: none
// is). By a wave, 64 keys a step.
__device__ __forceinline__ float bin_value(int b, double top, double inv_t) {
    if (b < 0) return __builtin_nanf("");
    const uint32_t lane = threadIdx.x & 63;
    uint32_t lo = b < kBins - 1 ? kMinusInf + 1 : 0xff800000u, hi = 0xff800000u;  // (of infinity)
    while (lo < hi) {
        const uint32_t step = (hi - lo + 63) / 64, k = hi - lo < lane * step ? hi : lo + lane * step;
        const uint64_t in = __ballot(bin_at(place_of(value_of(k), inv_t), top) <= b);
        const int l = in ? __builtin_ctzll(in) : 64;
        const uint32_t next = static_cast<uint32_t>(l) * step;
        if (l < 64) hi = hi - lo < next ? hi : lo + next;
        if (l > 0) lo = hi - lo < next - step + 1 ? hi : lo + next - step + 1;
    }
    return b < kBins - 1 ? value_of(hi) : -__FLT_MAX__;
}

__global__ __launch_bounds__(kThreads) void sample_find(SampleArgs a) {
    __shared__ uint32_t sh_count[kThreads / 64];
    __shared__ double sh_weight[kThreads / 64];
    __shared__ Found f_sh;
    __shared__ int32_t first_sh[kThreads / 64], off_sh[kThreads + kAtOnce];
    __shared__ uint32_t n_sh[kThreads + kAtOnce];
    __shared__ double by_sh[kThreads + kAtOnce];
    const int tid = static_cast<int>(threadIdx.x), lane = tid & 63, wave = tid >> 6;
    const int64_t r = blockIdx.x;
    const Row w = row_of(a, r);
    Part held = {};
    if (a.parts <= 64 && lane < a.parts) held = a.part[r * a.parts + lane];
    const uint64_t best = a.parts <= 64 ? wave_max_u64(held.best) : best_of_parts(a, r);
    const uint32_t best_key = static_cast<uint32_t>(best >> 32);
    if (!w.cuts() || best_key <= kMinusInf) {
        if (tid == 0) a.found[r].best = best;
        return;
    }
    const float top = value_of(best_key);
    const double place = place_of(top, w.inv_t);
    int32_t lo = kBins, hi = -1, bin_k = -1;
    uint32_t n, all;
    double s, total;
    row_bin(a, r, w, top, held, off_sh, n_sh, by_sh, &n, &s, &all, &total);
    // (the last bin: what the others leave)
    uint32_t counts = block_scan(sh_count, n);
    double weights = block_scan(sh_weight, s);
    if (tid == kBins - 1) {
        n = all - counts;
        s = total > weights ? total - weights : 0.0;
        counts = all;
        weights += s;
    }
    const bool by_k = w.by_k && static_cast<uint32_t>(w.k) < all;
    auto first_bin = [&](bool is) { return std::min(block_first<false>(first_sh, is), kBins - 1); };
    if (tid == 0) {
        f_sh.listed = 0;
        f_sh.few = 0;
        f_sh.need = 0;
        f_sh.below_k = 0.0;
    }
    if (by_k) bin_k = first_bin(counts >= static_cast<uint32_t>(w.k));
    __syncthreads();
    // The sum of what top-k leaves lies between that without its bin and that with it.
    if (tid == bin_k) {
        f_sh.below_k = weights - s;
        f_sh.total = weights;
        f_sh.need = static_cast<uint32_t>(w.k) - (counts - n);
    }
    __syncthreads();
    if (w.by_p) {
        // (a little more either way: the list's weights are not rounded as the histogram's)
        lo = first_bin(n && weights >= w.p * (by_k ? f_sh.below_k : total) * (1.0 - 0x1p-28));
        hi = first_bin(n && weights >= w.p * (by_k ? f_sh.total : total) * (1.0 + 0x1p-28));
        if (by_k && hi > bin_k) hi = bin_k;
        if (lo > hi) lo = hi;
    } else if (by_k) {
        lo = hi = bin_k;
    }
    if (lo < kBins) {
        // Where all that may stay is little it is listed whole, and launch 4 needs no sums.
        const int32_t end = by_k ? bin_k : hi;
        if (tid == end && counts <= kRanked) f_sh.few = counts;
        __syncthreads();
        const bool few = f_sh.few != 0;
        const uint32_t here = few ? 0u : wave_scan((tid >= lo && tid <= hi) || tid == bin_k ? n : 0u);
        if (lane == 63 && here) atomicAdd(&f_sh.listed, here);
        if (tid == lo) f_sh.below_lo = weights - s;
        if (wave < 4) {
            const int b = wave == 0 ? lo - 1 : wave == 1 ? hi : bin_k > hi ? bin_k - (wave == 3) : -1;
            const float v = bin_value(few ? (wave == 1 ? end : -1) : b, place, w.inv_t);
            if (lane == 0) (wave == 0 ? f_sh.above_lo : wave == 1 ? f_sh.above_hi : wave == 2 ? f_sh.above_k : f_sh.before_k) = v;
        }
        __syncthreads();
    }
    if (tid == 0) {
        Found f = f_sh;
        f.lo = lo;
        f.hi = hi;
        f.bin_k = bin_k;
        f.total = total;
        f.best = best;
        if (f.few) f.listed = f.few;
        a.found[r] = f;
    }
}

// ------------------------------------------------------------------ 3: kept blocks' sums, and the list

// Some blocks to a workgroup of 256 threads, the next one's tokens on their way while one's are weighed.
template <typename T>
__global__ __launch_bounds__(256) void sample_sums(SampleArgs a) {
    __shared__ double by_sh[64];  // e^(-b / 32) of b = 32 i + j: i's, and j's
    __shared__ double sh_weight[kMostBlocks][4];
    __shared__ u64 list_sh[kGroupListed];
    __shared__ uint32_t n_sh, from_sh;
    const int tid = static_cast<int>(threadIdx.x), lane = tid & 63, wave = tid >> 6;
    const int64_t r = blockIdx.x / static_cast<uint32_t>(a.groups);
    const int32_t group = static_cast<int32_t>(blockIdx.x - static_cast<uint32_t>(r) * static_cast<uint32_t>(a.groups));
    const int32_t first_block = group * a.group_blocks, blocks = std::min(a.group_blocks, a.n_blocks - first_block);
    int32_t i0 = first_block * kBlockTokens + tid * 8;
    const T* row = static_cast<const T*>(a.logits) + r * a.stride;
    Eight<T> next = load8(row, i0, a.vocab);
    const Row w = row_of(a, r);
    if (w.greedy) return;
    const uint32_t best = static_cast<uint32_t>(row_best(a, r) >> 32);
    if (best <= kMinusInf) return;
    const float top = value_of(best);
    // Of rows without cuts every token weighs in, of the others few do: a comparison of the logits tells which.
    Found f;
    f.lo = kBins;
    if (w.cuts()) f = a.found[r];
    const bool whole = f.lo == kBins, lists = !whole && f.listed <= kListed;
    const double per = bins_per(w.inv_t);
    if (tid == 0) n_sh = 0;
    if (!whole) __syncthreads();
    if (whole) {
        if (tid < 64) by_sh[tid] = tid < 32 ? exp(-1.0 * tid) : exp((tid - 32) * (-1.0 / kBinsPerT));
        __syncthreads();
    }
#pragma unroll 1
    for (int s = 0; s < blocks; s++, i0 += kBlockTokens) {
        const Eight<T> x = next;
        if (s + 1 < blocks) next = load8(row, i0 + kBlockTokens, a.vocab);
        double sum = 0.0;
        if (whole) {
            bool near = false;
            // e^(z / 32), by e^(-b / 32) of whole steps b down from the largest and the polynomial. (z from the difference,
            // which is exact: a difference of places is off by their own rounding, 2^-33 of the weight for logits of 10^6.)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float l = fmaxf(to_f32(x.v[e]), -__builtin_inff());  // (NaN: -inf)
                const double z = (static_cast<double>(l) - static_cast<double>(top)) * per, g = rint(z);
                const int b = static_cast<int>(fmin(-g, kBins - 1.0));
                double y = by_sh[b >> 5] * by_sh[32 + (b & 31)] * edge_weight<true>(z - g);
                if (b == kBins - 1) y = l > -__builtin_inff() ? weight_of(l, top, w.inv_t) : 0.0;
                if (l == top) y = 1.0;
                near |= fabs(y - w.min_p) < w.min_p * kNear;
                sum += y >= w.min_p ? y : 0.0;
            }
            // Launch 4 takes exponentials: next to min_p they decide here too, or it finds a block whose only token it drops.
            if (__any(near)) {
                sum = 0.0;
#pragma unroll 1
                for (int e = 0; e < 8; e++) {
                    float l = -__builtin_inff();
#pragma unroll
                    for (int i = 0; i < 8; i++) l = i == e ? fmaxf(to_f32(x.v[i]), l) : l;
                    const double y = weight_of(l, top, w.inv_t);
                    sum += y >= w.min_p ? y : 0.0;
                }
            }
        } else {
            uint32_t kept = 0, picked = 0;  // tokens that are surely kept; tokens of the list
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float l = to_f32(x.v[e]);
                kept |= l >= f.above_lo ? 1u << e : 0u;
                picked |= l >= f.above_hi || (l >= f.above_k && !(l >= f.before_k)) ? 1u << e : 0u;
            }
            picked &= ~kept;
            auto at = [&](int i) {
                float l = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; e++) l = i == e ? to_f32(x.v[e]) : l;
                return l;
            };
            // One of each lane's at a time: a wave has few of them, and most lanes none.
            for (uint32_t left = kept; left; left &= left - 1) {
                const double y = weight_of(at(__builtin_ctz(left)), top, w.inv_t);
                sum += y >= w.min_p ? y : 0.0;
            }
            if (lists && __any(picked != 0)) {
                const uint32_t mine = static_cast<uint32_t>(__popc(picked)), upto = wave_scan(mine);
                uint32_t from = 0;
                if (lane == 63) from = atomicAdd(&n_sh, upto);
                uint32_t to = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(from), 63)) + upto - mine;
                for (uint32_t left = picked; left; left &= left - 1, to++) {
                    const int i = __builtin_ctz(left);
                    const u64 x = static_cast<u64>(~key_of(at(i))) << 32 | static_cast<uint32_t>(i0 + i);
                    if (to < kGroupListed) {
                        list_sh[to] = x;
                    } else {
                        const uint32_t k = atomicAdd(a.listed + r * kLine, 1u);
                        if (k < kListed) a.list[r * kListed + k] = x;
                    }
                }
            }
        }
        sum = wave_sum_f64(sum);
        if (lane == 0) sh_weight[s][wave] = sum;
    }
    __syncthreads();
    if (lists) {
        // (one place in the list for all: a wave that asks for its own waits 2 us for it)
        const uint32_t n = std::min<uint32_t>(n_sh, kGroupListed);
        if (tid == 0 && n) from_sh = atomicAdd(a.listed + r * kLine, n);
        __syncthreads();
        for (uint32_t i = tid; i < n; i += 256)
            if (from_sh + i < kListed) a.list[r * kListed + from_sh + i] = list_sh[i];
    }
    if (tid < blocks) a.sums[r * a.n_blocks + first_block + tid] = (sh_weight[tid][0] + sh_weight[tid][1]) + (sh_weight[tid][2] + sh_weight[tid][3]);
}

// ------------------------------------------------------------------ 4: the cuts, and the token

// The order of the cuts: ascending.
__device__ __forceinline__ u64 order_of(uint32_t key, int32_t i) { return static_cast<u64>(~key) << 32 | static_cast<uint32_t>(i); }
__device__ __forceinline__ float ordered_value(u64 x) { return value_of(~static_cast<uint32_t>(x >> 32)); }

struct PickShared {
    u64 list[kListed];
    u64 weight[kBins], low[kBins];
    uint32_t count[kBins];
    u64 few[kRanked], sorted[kRanked];
    double few_weight[kRanked];
    uint32_t scan[kThreads / 64];
    double scan_f[kThreads / 64];
    u64 least, most, cut;
    double before, taken, left;
    uint32_t before_n, n;
    int32_t block, first[kThreads / 64];
};

// A cut: after `need` tokens (by_count), or where the weights' sum first reaches `target`.
struct Goal {
    bool by_count;
    uint32_t need;
    double target;
};

// The rank of thread e's number of sh.few (e < n <= kRanked) among the n, all different: four threads to each. sh.count
// holds it afterwards.
__device__ __forceinline__ void rank_few(PickShared& sh, int n) {
    const int tid = static_cast<int>(threadIdx.x), e = tid & (kRanked - 1);
    if (tid < kRanked) sh.count[tid] = 0;
    __syncthreads();
    const u64 x = sh.few[e];
    uint32_t rank = 0;
    for (int j = tid / kRanked; j < n; j += kThreads / kRanked) rank += sh.few[j] < x;
    if (e < n && rank) atomicAdd(&sh.count[e], rank);
    __syncthreads();
}

// Of tokens (each(f) calls f(its place in the order) for every one, at most n of them) the last that the goal takes,
// before_n tokens of the sum `before` coming before them: its place; the sum with it in sh.taken. More than a few are
// narrowed first, to one of 1024 equal parts of the order's range and again, by histograms in fixed point. There a weight is
// two whole numbers, the units and what their rounding left in 2^-32 of them: 2^24 equal weights far below the row's largest,
// which the units alone hold to 2^-38 each, are all off the same way (the sum by 2^-14; of both numbers, 2^-46).
template <typename Each>
__device__ u64 find_cut(PickShared& sh, const Row& w, float top, int fixed, const Goal& g, uint32_t n, uint32_t before_n, double before, Each&& each) {
    const int tid = static_cast<int>(threadIdx.x);
    const double units = ldexp(1.0, fixed);
    u64 lo = 0, hi = ~u64(0);
    if (n > kRanked) {
        __syncthreads();
        if (tid == 0) {
            sh.least = ~u64(0);
            sh.most = 0;
        }
        __syncthreads();
        u64 least = ~u64(0), most = 0;
        each([&](u64 x) {
            least = least < x ? least : x;
            most = most > x ? most : x;
        });
        least = ~wave_max_u64(~least);
        most = wave_max_u64(most);
        if ((tid & 63) == 0 && least <= most) {
            atomicMin(&sh.least, least);
            atomicMax(&sh.most, most);
        }
        __syncthreads();
        lo = sh.least;
        hi = sh.most;
        while (n > kRanked && lo < hi) {
            const int bits = 64 - __clzll(static_cast<long long>(hi - lo)), shift = bits > 10 ? bits - 10 : 0;
            __syncthreads();
            sh.count[tid] = 0;
            sh.weight[tid] = 0;
            sh.low[tid] = 0;
            __syncthreads();
            each([&](u64 x) {
                if (x < lo || x > hi) return;
                const int to = static_cast<int>((x - lo) >> shift);
                const double y = weight_of(ordered_value(x), top, w.inv_t);
                atomicAdd(&sh.count[to], 1u);
                atomicAdd(&sh.weight[to], static_cast<u64>(fixed_of(y, units)));
                atomicAdd(&sh.low[to], static_cast<u64>(fixed_left(y, units)));
            });
            __syncthreads();
            const uint32_t c = sh.count[tid];
            const double s = (static_cast<double>(sh.weight[tid]) + static_cast<double>(static_cast<int64_t>(sh.low[tid])) * 0x1p-32) / units;
            const uint32_t cs = before_n + block_scan(sh.scan, c);
            const double ss = before + block_scan(sh.scan_f, s);
            int at = block_first<false>(sh.first, c && (g.by_count ? cs >= g.need : ss >= g.target));
            if (at == kThreads) at = block_first<true>(sh.first, c != 0);  // (none reaches it: the last)
            if (tid == at) {
                sh.before_n = cs - c;
                sh.before = ss - s;
            }
            __syncthreads();
            before_n = sh.before_n;
            before = sh.before;
            n = sh.count[at];
            lo += static_cast<u64>(at) << shift;
            const u64 last = lo + ((u64(1) << shift) - 1);
            hi = hi < last ? hi : last;
        }
    }
    // Those, sorted by how many are smaller.
    __syncthreads();
    if (tid == 0) sh.n = 0;
    __syncthreads();
    each([&](u64 x) {
        if (x < lo || x > hi) return;
        const uint32_t at = atomicAdd(&sh.n, 1u);
        if (at < kRanked) sh.few[at] = x;
    });
    __syncthreads();
    const int many = static_cast<int>(std::min<uint32_t>(sh.n, kRanked));
    rank_few(sh, many);
    if (tid < many) sh.sorted[sh.count[tid]] = sh.few[tid];
    __syncthreads();
    const double mine = tid < many ? weight_of(ordered_value(sh.sorted[tid]), top, w.inv_t) : 0.0;
    const double upto = before + block_scan(sh.scan_f, mine);
    const int at = block_first<false>(sh.first, tid < many && (tid == many - 1 || (g.by_count ? before_n + static_cast<uint32_t>(tid) + 1 >= g.need : upto >= g.target)));
    if (tid == at) {
        sh.taken = upto;
        sh.cut = sh.sorted[tid];
    }
    __syncthreads();
    return sh.cut;
}

// The token of a row of which everything that may stay is listed.
__device__ __forceinline__ void pick_few(const SampleArgs& a, PickShared& sh, int64_t r, const Row& w, float top, const Found& f) {
    const int tid = static_cast<int>(threadIdx.x);
    const int n = static_cast<int>(std::min<uint32_t>(f.few, kRanked));
    if (tid < n) sh.few[tid] = a.list[r * kListed + tid];
    __syncthreads();
    rank_few(sh, n);
    if (tid < n) sh.sorted[sh.count[tid]] = sh.few[tid];
    __syncthreads();
    const u64 x = tid < n ? sh.sorted[tid] : 0;
    const double y = tid < n ? weight_of(ordered_value(x), top, w.inv_t) : 0.0;
    const double upto = block_scan(sh.scan_f, y);
    int stay = f.bin_k >= 0 ? std::min(n, w.k) : n;
    if (tid == stay - 1) sh.taken = upto;
    __syncthreads();
    if (w.by_p) stay = std::min(stay, block_first<false>(sh.first, tid < stay && upto >= w.p * (f.bin_k >= 0 ? sh.taken : f.total)) + 1);
    const bool stays = tid < stay && y >= w.min_p;
    // The same by index.
    if (tid < n) sh.few[tid] = stays ? static_cast<uint32_t>(x) : ~u64(0) - static_cast<u64>(tid);
    __syncthreads();
    rank_few(sh, n);
    if (tid < n) {
        sh.sorted[sh.count[tid]] = static_cast<uint32_t>(x);
        sh.few_weight[sh.count[tid]] = stays ? y : 0.0;
    }
    __syncthreads();
    const double mine = tid < n ? sh.few_weight[tid] : 0.0, at = block_scan(sh.scan_f, mine);
    if (tid == n - 1) sh.left = at;
    __syncthreads();
    const float u = a.u[r];
    const double target = (u > 0.0f ? static_cast<double>(fminf(u, 0x1.fffffep-1f)) : 0.0) * sh.left;
    int of = block_first<false>(sh.first, mine > 0.0 && at > target);
    if (of == kThreads) of = block_first<true>(sh.first, mine > 0.0);
    if (tid == of) a.out[r] = static_cast<int32_t>(sh.sorted[tid]);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_pick(SampleArgs a) {
    __shared__ PickShared sh;
    const int64_t r = blockIdx.x;
    const int tid = static_cast<int>(threadIdx.x), lane = tid & 63, wave = tid >> 6;
    const Row w = row_of(a, r);
    const uint64_t best = row_best(a, r);
    const uint32_t best_key = static_cast<uint32_t>(best >> 32);
    if (best_key <= kMinusInf || w.greedy) {
        if (tid == 0) a.out[r] = best_key <= kMinusInf ? -1 : static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(best));
        return;
    }
    const float top = value_of(best_key);
    const T* row = static_cast<const T*>(a.logits) + r * a.stride;
    double* sums = a.sums + r * a.n_blocks;
    u64 cut = order_of(kMinusInf + 1, 0x7fffffff);  // what stays: tokens up to it
    if (w.cuts()) {
        const Found f = a.found[r];
        if (f.lo < kBins && f.few > 0) {
            pick_few(a, sh, r, w, top, f);
            return;
        }
        if (f.lo < kBins && f.listed > 0) {
            const double place = place_of(top, w.inv_t);
            // The tokens of the cuts' bins: from the list, or, where there are more than it holds (logits much alike, high
            // temperatures), from the row again, by this workgroup alone.
            const bool crowded = f.listed > kListed;
            const int n = crowded ? 0 : static_cast<int>(f.listed);
            for (int i = tid; i < n; i += kThreads) sh.list[i] = a.list[r * kListed + i];
            __syncthreads();
            int b0 = f.lo, b1 = f.hi;
            auto each = [&](auto&& g) __attribute__((always_inline)) {
                auto one = [&](float l, u64 x) __attribute__((always_inline)) {
                    const int b = bin_at(place_of(l, w.inv_t), place);
                    if (b >= b0 && b <= b1 && x <= cut) g(x);
                };
                for (int i = tid; i < n; i += kThreads) one(ordered_value(sh.list[i]), sh.list[i]);
                if (!crowded) return;
                for (int32_t i = tid * 8; i < a.vocab; i += kStepTokens) {
                    const Eight<T> x = load8(row, i, a.vocab);
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const float l = to_f32(x.v[e]);
                        if (l > -__builtin_inff()) one(l, order_of(key_of(l), i + e));
                    }
                }
            };
            double total = f.total;
            if (f.bin_k >= 0) {
                b0 = b1 = f.bin_k;
                cut = find_cut(sh, w, top, a.narrow, Goal{true, static_cast<uint32_t>(w.k), 0.0}, f.listed, static_cast<uint32_t>(w.k) - f.need, f.below_k, each);
                total = sh.taken;
            }
            if (w.by_p) {
                b0 = f.lo;
                b1 = f.hi;
                cut = find_cut(sh, w, top, a.narrow, Goal{false, 0, w.p * total}, f.listed, 0, f.below_lo, each);
            }
            // The kept ones' weights to their blocks' sums: in fixed point, as they come in any order.
            b0 = f.lo;
            b1 = kBins - 1;
            for (int32_t from = 0; from < a.n_blocks; from += kBins) {
                __syncthreads();
                sh.weight[tid] = 0;
                __syncthreads();
                each([&](u64 x) {
                    const int b = static_cast<int>(static_cast<uint32_t>(x) / kBlockTokens) - from;
                    const double y = weight_of(ordered_value(x), top, w.inv_t);
                    if (b >= 0 && b < kBins && y >= w.min_p) atomicAdd(&sh.weight[b], static_cast<u64>(fixed_of(y, 0x1p44)));
                });
                __syncthreads();
                if (from + tid < a.n_blocks && sh.weight[tid]) sums[from + tid] += static_cast<double>(sh.weight[tid]) * 0x1p-44;
            }
            __syncthreads();
        }
    }
    if (wave == 0) {
        double total = 0.0;
        for (int32_t b0 = 0; b0 < a.n_blocks; b0 += 64) total += wave_sum_f64(b0 + lane < a.n_blocks ? sums[b0 + lane] : 0.0);
        const float u = a.u[r];
        const double target = (u > 0.0f ? static_cast<double>(fminf(u, 0x1.fffffep-1f)) : 0.0) * total;
        // The first block whose running sum passes the target; by rounding none may: the last with a weight.
        double past = 0.0, left = 0.0;
        int32_t block = -1, last = 0;
        for (int32_t b0 = 0; b0 < a.n_blocks && block < 0; b0 += 64) {
            const double x = b0 + lane < a.n_blocks ? sums[b0 + lane] : 0.0;
            const double upto = past + wave_scan(x);
            const uint64_t over = __ballot(x > 0.0 && upto > target), some = __ballot(x > 0.0);
            if (some) last = b0 + 63 - __builtin_clzll(some);
            if (over) {
                const int l = __builtin_ctzll(over);
                block = b0 + l;
                left = target - readlane_f64(upto - x, l);
            }
            past = readlane_f64(upto, 63);
        }
        if (lane == 0) {
            sh.block = block < 0 ? last : block;
            sh.left = block < 0 ? __builtin_inf() : left;
        }
    }
    __syncthreads();
    // Two tokens to a thread. (Some thread has one: a block of a sum above 0 holds a token of that weight, by the same
    // exponential and comparisons in launch 3.)
    constexpr int PER = kBlockTokens / kThreads;
    const int32_t i0 = sh.block * kBlockTokens + tid * PER;
    double y[PER], sum = 0.0;
#pragma unroll
    for (int e = 0; e < PER; e++) {
        const float l = i0 + e < a.vocab ? to_f32(row[i0 + e]) : -__builtin_inff();
        y[e] = 0.0;
        if (l > -__builtin_inff() && order_of(key_of(l), i0 + e) <= cut) y[e] = weight_of(l, top, w.inv_t);
        if (y[e] < w.min_p) y[e] = 0.0;
        sum += y[e];
    }
    double at = block_scan(sh.scan_f, sum) - sum;
    int32_t mine = -1;  // this thread's first token past u, or its last of any weight
    bool past = false;
#pragma unroll
    for (int e = 0; e < PER; e++) {
        at += y[e];
        if (y[e] > 0.0 && !past) {
            mine = i0 + e;
            past = at > sh.left;
        }
    }
    int of = block_first<false>(sh.first, past);
    if (of == kThreads) of = block_first<true>(sh.first, mine >= 0);
    if (tid == of) a.out[r] = mine;
}

template <typename T>
int launch(neko_hip_ctx* ctx, const char* what, SampleArgs a, int64_t rows, int64_t slab) {
    const SampleArgs all = a;
    for (int64_t r = 0; r < rows; r += slab) {
        const int64_t n = std::min(slab, rows - r);
        const uint32_t parts = static_cast<uint32_t>(n * a.parts);
        auto from = [&](auto* p) { return p ? p + r : p; };
        a.logits = static_cast<const T*>(all.logits) + r * all.stride;
        a.temperature = from(all.temperature);
        a.top_k = from(all.top_k);
        a.top_p = from(all.top_p);
        a.min_p = from(all.min_p);
        a.u = from(all.u);
        a.out = from(all.out);
        const dim3 by_row(static_cast<uint32_t>(n));
        auto parts_of = [&](auto steps) { hipLaunchKernelGGL((sample_parts<T, decltype(steps)::value>), dim3(parts), dim3(kThreads), 0, ctx->stream, a); };
        switch (a.part_tokens / kStepTokens) {
            case 1: parts_of(std::integral_constant<int, 1>{}); break;
            case 2: parts_of(std::integral_constant<int, 2>{}); break;
            default:
                if constexpr (kMostSteps<T> > 2) parts_of(std::integral_constant<int, kMostSteps<T>>{});
        }
        if (int rc = after_launch(ctx, what)) return rc;
        if (a.top_k || a.top_p) {
            hipLaunchKernelGGL(sample_find, by_row, dim3(kThreads), 0, ctx->stream, a);
            if (int rc = after_launch(ctx, what)) return rc;
        }
        const uint32_t groups = static_cast<uint32_t>(n * a.groups);
        hipLaunchKernelGGL((sample_sums<T>), dim3(groups), dim3(256), 0, ctx->stream, a);
        if (int rc = after_launch(ctx, what)) return rc;
        hipLaunchKernelGGL((sample_pick<T>), by_row, dim3(kThreads), 0, ctx->stream, a);
        if (int rc = after_launch(ctx, what)) return rc;
    }
    return NEKO_OK;
}

}  // namespace
}  // namespace neko_hip

using namespace neko_hip;

extern "C" int neko_hip_sample(neko_hip_ctx* ctx, const void* logits, int64_t stride, int64_t rows, int64_t vocab,
                               const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                               const float* u, int32_t* tokens, int dtype) {
    const char* what = "neko_hip_sample";
    NEKO_ENTER(ctx);
    NEKO_REQUIRE(ctx, valid_dtype(dtype), "%s: bad dtype %d", what, dtype);
    NEKO_REQUIRE(ctx, rows >= 0 && rows <= (1 << 20) && vocab > 0 && vocab <= (1 << 24), "%s: bad shape rows=%lld vocab=%lld", what,
                 (long long)rows, (long long)vocab);
    if (rows == 0) return NEKO_OK;
    NEKO_REQUIRE(ctx, logits && u && tokens, "%s: null pointer", what);
    NEKO_REQUIRE(ctx, stride >= vocab, "%s: row stride %lld below the vocabulary's %lld", what, (long long)stride, (long long)vocab);
    const size_t esz = dtype_size(dtype), n = static_cast<size_t>(rows) * 4;
    NEKO_REQUIRE(ctx, aligned(logits, esz) && aligned(temperature, 4) && aligned(top_k, 4) && aligned(top_p, 4) && aligned(min_p, 4) &&
                 aligned(u, 4) && aligned(tokens, 4), "%s: misaligned pointer", what);
    const size_t span = rows_span(rows, vocab, stride, esz);
    NEKO_REQUIRE(ctx, span != 0, "%s: rows span more than 2^62 bytes", what);
    NEKO_REQUIRE(ctx, !overlaps(tokens, n, logits, span), "%s: tokens may not overlap the logits", what);
    for (const void* q : {static_cast<const void*>(temperature), static_cast<const void*>(top_k), static_cast<const void*>(top_p),
                          static_cast<const void*>(min_p), static_cast<const void*>(u)})
        NEKO_REQUIRE(ctx, !q || !overlaps(tokens, n, q, n), "%s: tokens may not overlap the settings", what);
    SampleArgs a{};
    a.logits = logits;
    a.stride = stride;
    a.temperature = temperature;
    a.top_k = top_k;
    a.top_p = top_p;
    a.min_p = min_p;
    a.u = u;
    a.out = tokens;
    a.vocab = static_cast<int32_t>(vocab);
    a.n_blocks = static_cast<int32_t>((vocab + kBlockTokens - 1) / kBlockTokens);
    // Two workgroups to a CU over all rows, as many as are resident.
    const int64_t steps = (vocab + kStepTokens - 1) / kStepTokens;
    const int64_t held = std::min(rows, kSlabRows);
    const int64_t wanted = std::max<int64_t>(1, std::min<int64_t>(steps, (2LL * ctx->cu_count + held - 1) / held));
    const int64_t even = (steps + wanted - 1) / wanted, each = std::min<int64_t>(even, dtype == NEKO_DT_F16 ? kMostSteps<half_t> : kMostSteps<float>);
    a.parts = static_cast<int32_t>((steps + each - 1) / each);
    a.part_tokens = static_cast<int32_t>(each * kStepTokens);
    // Ten workgroups to a CU, of as many blocks as that takes: twice what is resident, since rows without cuts take longer.
    a.group_blocks = static_cast<int32_t>(std::clamp<int64_t>((a.n_blocks * held + 10 * ctx->cu_count - 1) / (10 * ctx->cu_count), 1, kMostBlocks));
    a.groups = (a.n_blocks + a.group_blocks - 1) / a.group_blocks;
    // A bin's number of tokens, up to part_tokens, and above it their weights, each below 1.04 units.
    auto bits_of = [](int64_t n) {
        int bits = 0;
        while ((int64_t(1) << bits) <= n) bits++;
        return bits;
    };
    a.count_bits = bits_of(a.part_tokens);
    a.fixed = std::min(44, 63 - 2 * a.count_bits);
    a.narrow = std::min(44, 62 - bits_of(vocab));
    const bool hist = a.top_k || a.top_p;
    // (of either type: what a call of one has made room for holds the other)
    const size_t parts = static_cast<size_t>((steps + std::min<int64_t>(even, kMostSteps<half_t>) - 1) / std::min<int64_t>(even, kMostSteps<half_t>));
    size_t bytes[] = {parts * sizeof(Part), static_cast<size_t>(a.n_blocks) * 8, sizeof(Found), hist ? parts * kBins * 8 : 0, hist ? kListed * size_t(8) : 0,
                      kLine * sizeof(uint32_t)};  // of a row
    size_t of_row = 0;
    for (size_t b : bytes) of_row += b;
    const int64_t slab = std::clamp<int64_t>(static_cast<int64_t>(kSlabBytes / of_row), 1, held);
    for (size_t& b : bytes) b *= static_cast<size_t>(slab);
    size_t all = 0;
    for (size_t b : bytes) all += b;
    void* ws = nullptr;
    if (int rc = workspace(ctx, all, &ws)) return rc;
    void* at[6];
    char* p = static_cast<char*>(ws);
    for (int i = 0; i < 6; i++) {
        at[i] = p;
        p += bytes[i];
    }
    a.part = static_cast<Part*>(at[0]);
    a.sums = static_cast<double*>(at[1]);
    a.found = static_cast<Found*>(at[2]);
    a.bins = static_cast<uint64_t*>(at[3]);
    a.list = static_cast<uint64_t*>(at[4]);
    a.listed = static_cast<uint32_t*>(at[5]);
    return dtype == NEKO_DT_F16 ? launch<half_t>(ctx, what, a, rows, slab) : launch<float>(ctx, what, a, rows, slab);
}
