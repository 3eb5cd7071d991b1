// Sampling a token of each row of logits, by temperature, top-k, top-p and min-p, from a given uniform number.
//
// Formulas. w_i = e^((l_i - max l) / T). Sorted by logit, equal ones by index: S1, the first k; S2, the shortest prefix of
// S1 with sum w >= p * (sum of S1's w); S3, those with w >= min_p. The token is the first of S2 and S3, by index, whose
// running sum of w passes u * (their sum).
//
// Numbers. A vocabulary has some 10^5 borders between tokens, and f32 weights, off by 2^-24, would put about one sample in
// 10^4 on the wrong side of one. Weights are e^x in double; the sums that cut off S1 and S2 are of weights in fixed point
// (2^-44 of the largest for up to 2^18 tokens), whose order does not matter, so atomics in LDS may take any; the running
// sum is in double, in an order that the vocabulary alone sets.
//
// Launches, several workgroups to a row in 1, 2 and 4:
//   1 the largest logit
//   2 a histogram of weights and counts over the distance from it, 512 bins of T / 16 (rows with a top-k or top-p)
//   3 the bin of each cut from that, the few tokens in it sorted: the last logit kept, and of those equal to it the last
//     index (one workgroup to a row)
//   4 the kept weights' sums of blocks of 2048 tokens
//   5 the block, and in it the token
#include <algorithm>

#include "internal.h"
#include "paged_device.h"

namespace neko_hip {
namespace {

constexpr int kBins = 512;
constexpr float kBinsPerNat = 16.0f;
constexpr int kBlockTokens = 2048;  // of a sum in launch 4: 256 threads of 8
constexpr int kListed = 4096;       // tokens of a bin that launch 3 sorts in LDS
constexpr uint32_t kMinusInf = 0x007fffffu;  // its key; tokens at or below are left out

struct Cut {
    uint32_t key;  // kept: keys above, and of those equal the indices up to `last`
    int32_t last;
};

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
    int32_t n_max, max_tokens;    // workgroups of a row in launches 1 and 4, and their tokens (whole blocks)
    int32_t n_hist, hist_tokens;  // of launch 2
    int32_t n_blocks;             // blocks of a row
    int32_t fixed;                // fixed-point weights: units of 2^-fixed
    uint64_t* best;               // [rows][n_max] key << 32 | ~index
    uint32_t* counts;             // [rows][n_hist][kBins]
    uint64_t* weights;
    Cut* cuts;                    // [rows]
    double* sums;                 // [rows][n_blocks]
};

// What a row asks for, as its numbers are read: a temperature that is not positive is the largest logit's token, a k not
// positive, a p of 1 or more and a min_p not positive cut off nothing, nor does a NaN.
struct Row {
    bool greedy, by_k, by_p;
    float bins;     // per unit of distance
    double inv_t, p, min_p;
    int32_t k;
};
__device__ __forceinline__ Row row_of(const SampleArgs& a, int64_t r) {
    Row w;
    const float t = a.temperature ? a.temperature[r] : 1.0f;
    w.greedy = !(t > 0.0f);
    w.inv_t = 1.0 / static_cast<double>(t);
    w.bins = kBinsPerNat / t;
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

// The bin of a logit below or at the largest: monotone in it, as every rounding here is.
__device__ __forceinline__ int bin_of(float l, float top, float per) {
    return l == top ? 0 : static_cast<int>(fminf((top - l) * per, static_cast<float>(kBins - 1)));  // (NaN, an infinite distance at no slope: the last)
}
__device__ __forceinline__ double weight_of(float l, float top, double inv_t) {
    const double w = exp((static_cast<double>(l) - static_cast<double>(top)) * inv_t);
    return l == top ? 1.0 : w == w ? w : 0.0;
}
__device__ __forceinline__ uint64_t fixed_of(double w, int bits) { return static_cast<uint64_t>(ldexp(w, bits) + 0.5); }

// Logits i .. i + 7 of a row of n, -inf past it. Rows may stand at any element.
template <typename T>
__device__ __forceinline__ void load8(const T* row, int32_t i, int32_t n, float* x) {
    T v[8];
    if (i + 8 <= n) {
        __builtin_memcpy(v, row + i, sizeof(v));
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = to_f32(v[e]);
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = i + e < n ? to_f32(row[i + e]) : -__builtin_inff();
    }
}

__device__ __forceinline__ uint64_t wave_max_u64(uint64_t v) {
#pragma unroll
    for (int m = 1; m < 64; m *= 2) {
        const uint64_t o = static_cast<uint64_t>(__shfl_xor(static_cast<unsigned long long>(v), m));
        v = v > o ? v : o;
    }
    return v;
}

// The largest logit of a row, from launch 1's parts, by every wave for itself: key << 32 | ~index.
__device__ __forceinline__ uint64_t row_best(const SampleArgs& a, int64_t r) {
    uint64_t b = 0;
    for (int32_t i = static_cast<int32_t>(threadIdx.x) & 63; i < a.n_max; i += 64) {
        const uint64_t o = a.best[r * a.n_max + i];
        b = b > o ? b : o;
    }
    return wave_max_u64(b);
}

// ------------------------------------------------------------------ 1: the largest

template <typename T>
__global__ __launch_bounds__(256) void sample_max(SampleArgs a) {
    __shared__ uint64_t sh[4];
    const int64_t r = blockIdx.x / static_cast<uint32_t>(a.n_max);
    const int32_t part = static_cast<int32_t>(blockIdx.x - static_cast<uint32_t>(r) * static_cast<uint32_t>(a.n_max));
    const T* row = static_cast<const T*>(a.logits) + r * a.stride;
    const int32_t end = static_cast<int32_t>(std::min<int64_t>(a.vocab, static_cast<int64_t>(part + 1) * a.max_tokens));
    uint32_t top = 0, at = 0;
    for (int32_t i = part * a.max_tokens + static_cast<int32_t>(threadIdx.x) * 8; i < end; i += kBlockTokens) {
        float x[8];
        load8(row, i, a.vocab, x);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const uint32_t k = key_of(x[e]);
            if (k > top) {
                top = k;
                at = static_cast<uint32_t>(i + e);
            }
        }
    }
    const uint64_t b = wave_max_u64(static_cast<uint64_t>(top) << 32 | (0xffffffffu - at));
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = b;
    __syncthreads();
    if (threadIdx.x == 0) a.best[blockIdx.x] = std::max(std::max(sh[0], sh[1]), std::max(sh[2], sh[3]));
}

// ------------------------------------------------------------------ 2: the histogram

template <typename T>
__global__ __launch_bounds__(256) void sample_hist(SampleArgs a) {
    __shared__ uint32_t count[kBins];
    __shared__ unsigned long long weight[kBins];
    const int64_t r = blockIdx.x / static_cast<uint32_t>(a.n_hist);
    const int32_t part = static_cast<int32_t>(blockIdx.x - static_cast<uint32_t>(r) * static_cast<uint32_t>(a.n_hist));
    const Row w = row_of(a, r);
    if (w.greedy || !(w.by_k || w.by_p)) return;
    const float top = value_of(static_cast<uint32_t>(row_best(a, r) >> 32));
    for (int i = static_cast<int>(threadIdx.x); i < kBins; i += 256) {
        count[i] = 0;
        weight[i] = 0;
    }
    __syncthreads();
    const T* row = static_cast<const T*>(a.logits) + r * a.stride;
    const int32_t end = static_cast<int32_t>(std::min<int64_t>(a.vocab, static_cast<int64_t>(part + 1) * a.hist_tokens));
    for (int32_t i = part * a.hist_tokens + static_cast<int32_t>(threadIdx.x) * 8; i < end; i += kBlockTokens) {
        float x[8];
        load8(row, i, a.vocab, x);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            if (key_of(x[e]) <= kMinusInf) continue;
            const int b = bin_of(x[e], top, w.bins);
            atomicAdd(&count[b], 1u);
            atomicAdd(&weight[b], static_cast<unsigned long long>(fixed_of(weight_of(x[e], top, w.inv_t), a.fixed)));
        }
    }
    __syncthreads();
    for (int i = static_cast<int>(threadIdx.x); i < kBins; i += 256) {
        a.counts[static_cast<int64_t>(blockIdx.x) * kBins + i] = count[i];
        a.weights[static_cast<int64_t>(blockIdx.x) * kBins + i] = weight[i];
    }
}

// ------------------------------------------------------------------ 3: the cuts

constexpr int kCutThreads = 1024;

struct CutShared {
    uint64_t list[kListed];  // ~key << 32 | index: ascending is the order of the cuts
    unsigned long long weight[kBins];
    uint32_t count[kBins];
    uint64_t scan[kCutThreads / 64];
    uint64_t before_weight, taken_weight;
    uint32_t before_count, n, at;
    uint32_t key;
    int32_t last;
};

__device__ __forceinline__ uint64_t wave_scan_u64(uint64_t v) {
    const int lane = static_cast<int>(threadIdx.x) & 63;
#pragma unroll
    for (int m = 1; m < 64; m *= 2) {
        const uint64_t o = static_cast<uint64_t>(__shfl_up(static_cast<unsigned long long>(v), m));
        v += lane >= m ? o : 0;
    }
    return v;
}
// The sum of the threads' values up to each thread's own.
__device__ __forceinline__ uint64_t block_scan(CutShared& sh, uint64_t v) {
    const int wave = static_cast<int>(threadIdx.x) >> 6;
    v = wave_scan_u64(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) sh.scan[wave] = v;
    __syncthreads();
    for (int i = 0; i < wave; i++) v += sh.scan[i];
    return v;
}

// A cut: after `need` tokens (by_count), or where the weights' sum first reaches `target`.
struct Goal {
    bool by_count;
    uint32_t need;
    double target;
};
__device__ __forceinline__ bool reached(const Goal& g, uint64_t count, uint64_t weight) {
    return g.by_count ? count >= g.need : static_cast<double>(weight) >= g.target;
}

// Of n groups in sh.count / sh.weight, in order, the one that reaches the goal, from `count0` tokens and `weight0` before
// the first (none does: the last that has tokens). Leaves sh.at, and what stands before it.
__device__ __forceinline__ void find_group(CutShared& sh, const Goal& g, int n, uint32_t count0, uint64_t weight0) {
    const int i = static_cast<int>(threadIdx.x);
    const uint64_t c = i < n ? sh.count[i] : 0, w = i < n ? sh.weight[i] : 0;
    const uint64_t cs = block_scan(sh, c) + count0, ws = block_scan(sh, w) + weight0;
    if (i == 0) sh.at = 0xffffffffu;
    __syncthreads();
    if (i < n && c && reached(g, cs, ws)) atomicMin(&sh.at, static_cast<uint32_t>(i));
    __syncthreads();
    if (sh.at == 0xffffffffu) {
        __syncthreads();
        if (i < n && c) atomicMin(&sh.at, 0xffffffffu - static_cast<uint32_t>(i) - 1u);
        __syncthreads();
        if (i == 0) sh.at = sh.at == 0xffffffffu ? 0u : 0xfffffffeu - sh.at;
        __syncthreads();
    }
    if (static_cast<uint32_t>(i) == sh.at) {
        sh.before_count = static_cast<uint32_t>(cs - c);
        sh.before_weight = ws - w;
    }
    __syncthreads();
}

// The goal's last token within bin `bin` of the row, `count` tokens of it, before_* in sh: sh.key, sh.last and the
// weights' sum with it, sh.taken_weight.
template <typename T>
__device__ void cut_bin(const SampleArgs& a, CutShared& sh, const Row& w, const T* row, float top, const Goal& g, int bin, uint32_t count) {
    const int tid = static_cast<int>(threadIdx.x);
    uint32_t prefix = 0, mask = 0;
    auto each = [&](auto&& f) __attribute__((always_inline)) {
        for (int32_t i = tid * 8; i < a.vocab; i += kCutThreads * 8) {
            float x[8];
            load8(row, i, a.vocab, x);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const uint32_t k = key_of(x[e]);
                if (k > kMinusInf && bin_of(x[e], top, w.bins) == bin && (k & mask) == prefix) f(k, x[e], i + e);
            }
        }
    };
    // More of them than are sorted: the keys' bits, eight at a time.
    for (int shift = 24; count > kListed && shift >= 0; shift -= 8) {
        __syncthreads();
        const uint32_t count0 = sh.before_count;
        const uint64_t weight0 = sh.before_weight;
        if (tid < 256) {
            sh.count[tid] = 0;
            sh.weight[tid] = 0;
        }
        __syncthreads();
        each([&](uint32_t k, float l, int32_t) {
            const int at = 255 - static_cast<int>((k >> shift) & 255u);  // (the larger ones first)
            atomicAdd(&sh.count[at], 1u);
            atomicAdd(&sh.weight[at], static_cast<unsigned long long>(fixed_of(weight_of(l, top, w.inv_t), a.fixed)));
        });
        __syncthreads();
        find_group(sh, g, 256, count0, weight0);
        count = sh.count[sh.at];
        prefix |= (255u - sh.at) << shift;
        mask |= 255u << shift;
    }
    const uint32_t count0 = sh.before_count;
    const uint64_t weight0 = sh.before_weight;
    __syncthreads();
    if (count > kListed) {
        // All are one value, `prefix`: how many of them, then the index of the last.
        const uint64_t one = fixed_of(weight_of(value_of(prefix), top, w.inv_t), a.fixed);
        uint32_t take = count;
        if (g.by_count) {
            take = g.need - count0;
        } else if (one) {
            const double most = ceil((g.target - static_cast<double>(weight0)) / static_cast<double>(one));
            take = most < static_cast<double>(count) ? static_cast<uint32_t>(most > 1.0 ? most : 1.0) : count;
            if (take > 1 && reached(g, 0, weight0 + (take - 1) * one)) take--;  // (the quotient's rounding)
        }
        uint64_t past = 0;
        for (int32_t i0 = 0; i0 < a.vocab && past < take; i0 += kCutThreads) {
            const int32_t i = i0 + tid;
            const bool is = i < a.vocab && key_of(to_f32(row[i])) == prefix;
            const uint64_t sum = past + block_scan(sh, is ? 1 : 0);
            if (is && sum == take) sh.last = i;
            if (tid == kCutThreads - 1) sh.n = static_cast<uint32_t>(sum);
            __syncthreads();
            past = sh.n;
        }
        if (tid == 0) {
            sh.key = prefix;
            sh.taken_weight = weight0 + take * one;
        }
        __syncthreads();
        return;
    }
    // The list, sorted (bitonic, over a power of two), then the first place that reaches the goal.
    if (tid == 0) sh.n = 0;
    __syncthreads();
    each([&](uint32_t k, float, int32_t i) {
        const uint32_t at = atomicAdd(&sh.n, 1u);
        if (at < kListed) sh.list[at] = static_cast<uint64_t>(~k) << 32 | static_cast<uint32_t>(i);
    });
    __syncthreads();
    const int n = static_cast<int>(std::min<uint32_t>(std::max<uint32_t>(sh.n, 1u), kListed));
    int size = 2;
    while (size < n) size *= 2;
    for (int i = n + tid; i < size; i += kCutThreads) sh.list[i] = ~uint64_t(0);
    __syncthreads();
    for (int run = 2; run <= size; run *= 2)
        for (int step = run / 2; step > 0; step /= 2) {
            for (int i = tid; i < size / 2; i += kCutThreads) {
                const int lo = 2 * i - (i & (step - 1)), hi = lo + step;
                const uint64_t x = sh.list[lo], y = sh.list[hi];
                if ((x > y) == ((lo & run) == 0)) {
                    sh.list[lo] = y;
                    sh.list[hi] = x;
                }
            }
            __syncthreads();
        }
    constexpr int PER = kListed / kCutThreads;
    uint64_t mine[PER], sum = 0;
#pragma unroll
    for (int e = 0; e < PER; e++) {
        const int i = tid * PER + e;
        mine[e] = i < n ? fixed_of(weight_of(value_of(~static_cast<uint32_t>(sh.list[i] >> 32)), top, w.inv_t), a.fixed) : 0;
        sum += mine[e];
    }
    uint64_t at = block_scan(sh, sum) - sum + weight0;
    if (tid == 0) sh.at = static_cast<uint32_t>(n - 1);
    __syncthreads();
    uint32_t first = 0xffffffffu;
    uint64_t upto[PER];
#pragma unroll
    for (int e = 0; e < PER; e++) {
        const int i = tid * PER + e;
        at += mine[e];
        upto[e] = at;
        if (i < n && first == 0xffffffffu && reached(g, static_cast<uint64_t>(count0) + static_cast<uint64_t>(i) + 1, at)) first = static_cast<uint32_t>(i);
    }
    if (first != 0xffffffffu) atomicMin(&sh.at, first);
    __syncthreads();
    if (static_cast<int>(sh.at) / PER == tid) {
        const uint64_t x = sh.list[sh.at];
        sh.key = ~static_cast<uint32_t>(x >> 32);
        sh.last = static_cast<int32_t>(static_cast<uint32_t>(x));
#pragma unroll
        for (int e = 0; e < PER; e++)
            if (tid * PER + e == static_cast<int>(sh.at)) sh.taken_weight = upto[e];
    }
    __syncthreads();
}

template <typename T>
__global__ __launch_bounds__(kCutThreads) void sample_cut(SampleArgs a) {
    __shared__ CutShared sh;
    const int64_t r = blockIdx.x;
    const int tid = static_cast<int>(threadIdx.x);
    const Row w = row_of(a, r);
    if (w.greedy) return;
    if (!(w.by_k || w.by_p)) {
        if (tid == 0) a.cuts[r] = Cut{kMinusInf, -1};
        return;
    }
    const uint64_t best = row_best(a, r);
    const uint32_t best_key = static_cast<uint32_t>(best >> 32);
    if (best_key <= kMinusInf) return;  // nothing to choose from
    const float top = value_of(best_key);
    const T* row = static_cast<const T*>(a.logits) + r * a.stride;
    uint32_t count = 0;
    uint64_t weight = 0;
    if (tid < kBins) {
        for (int32_t i = 0; i < a.n_hist; i++) {
            count += a.counts[(r * a.n_hist + i) * kBins + tid];
            weight += a.weights[(r * a.n_hist + i) * kBins + tid];
        }
    }
    const uint64_t counts = block_scan(sh, count), weights = block_scan(sh, weight);
    if (tid == kCutThreads - 1) {
        sh.before_count = static_cast<uint32_t>(counts);
        sh.taken_weight = weights;
    }
    __syncthreads();
    const uint32_t all = sh.before_count;
    uint64_t total = sh.taken_weight;
    __syncthreads();
    auto groups = [&]() {
        if (tid < kBins) {
            sh.count[tid] = count;
            sh.weight[tid] = weight;
        }
        __syncthreads();
    };
    Cut cut = {kMinusInf, -1};
    if (w.by_k && static_cast<uint32_t>(w.k) < all) {
        const Goal g = {true, static_cast<uint32_t>(w.k), 0.0};
        groups();
        find_group(sh, g, kBins, 0, 0);
        const int bin = static_cast<int>(sh.at);
        const uint32_t n = sh.count[bin];
        cut_bin(a, sh, w, row, top, g, bin, n);
        cut = Cut{sh.key, sh.last};
        total = sh.taken_weight;
        __syncthreads();
    }
    if (w.by_p) {
        const Goal g = {false, 0, w.p * static_cast<double>(total)};
        if (!(g.target > 0.0)) {  // the first alone
            cut = Cut{best_key, static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(best))};
        } else {
            groups();
            find_group(sh, g, kBins, 0, 0);
            const int bin = static_cast<int>(sh.at);
            const uint32_t n = sh.count[bin];
            cut_bin(a, sh, w, row, top, g, bin, n);
            cut = Cut{sh.key, sh.last};
        }
    }
    if (tid == 0) a.cuts[r] = cut;
}

// ------------------------------------------------------------------ 4 and 5: the kept weights, and the token

// The weight that token i counts with, 0 if it is cut off.
__device__ __forceinline__ double kept_weight(float l, int32_t i, float top, const Row& w, const Cut& c) {
    const uint32_t k = key_of(l);
    if (k <= kMinusInf || k < c.key || (k == c.key && i > c.last)) return 0.0;
    const double x = weight_of(l, top, w.inv_t);
    return x >= w.min_p ? x : 0.0;
}

__device__ __forceinline__ Cut cut_of(const SampleArgs& a, int64_t r, const Row& w) {
    return w.by_k || w.by_p ? a.cuts[r] : Cut{kMinusInf, -1};
}

template <typename T>
__global__ __launch_bounds__(256) void sample_sum(SampleArgs a) {
    __shared__ double sh[4];
    const int64_t r = blockIdx.x / static_cast<uint32_t>(a.n_max);
    const int32_t part = static_cast<int32_t>(blockIdx.x - static_cast<uint32_t>(r) * static_cast<uint32_t>(a.n_max));
    const Row w = row_of(a, r);
    if (w.greedy) return;
    const uint32_t best = static_cast<uint32_t>(row_best(a, r) >> 32);
    if (best <= kMinusInf) return;
    const float top = value_of(best);
    const Cut c = cut_of(a, r, w);
    const T* row = static_cast<const T*>(a.logits) + r * a.stride;
    const int32_t end = static_cast<int32_t>(std::min<int64_t>(a.vocab, static_cast<int64_t>(part + 1) * a.max_tokens));
    for (int32_t i0 = part * a.max_tokens; i0 < end; i0 += kBlockTokens) {
        const int32_t i = i0 + static_cast<int32_t>(threadIdx.x) * 8;
        double sum = 0.0;
        if (i < a.vocab) {
            float x[8];
            load8(row, i, a.vocab, x);
#pragma unroll
            for (int e = 0; e < 8; e++) sum += kept_weight(x[e], i + e, top, w, c);
        }
        sum = wave_sum_f64(sum);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = sum;
        __syncthreads();
        if (threadIdx.x == 0) a.sums[r * a.n_blocks + i0 / kBlockTokens] = (sh[0] + sh[1]) + (sh[2] + sh[3]);
    }
}

__device__ __forceinline__ double wave_scan_f64(double v) {
    const int lane = static_cast<int>(threadIdx.x) & 63;
#pragma unroll
    for (int m = 1; m < 64; m *= 2) {
        const double o = __shfl_up(v, m);
        v += lane >= m ? o : 0.0;
    }
    return v;
}

template <typename T>
__global__ __launch_bounds__(256) void sample_pick(SampleArgs a) {
    __shared__ double sh[4], left_sh;
    __shared__ int32_t block_sh;
    __shared__ uint32_t found;
    const int64_t r = blockIdx.x;
    const int tid = static_cast<int>(threadIdx.x), lane = tid & 63, wave = tid >> 6;
    const Row w = row_of(a, r);
    const uint64_t best = row_best(a, r);
    const uint32_t best_key = static_cast<uint32_t>(best >> 32), best_at = 0xffffffffu - static_cast<uint32_t>(best);
    if (best_key <= kMinusInf || w.greedy) {
        if (tid == 0) a.out[r] = best_key <= kMinusInf ? -1 : static_cast<int32_t>(best_at);
        return;
    }
    const double* sums = a.sums + r * a.n_blocks;
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
            const double upto = past + wave_scan_f64(x);
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
            block_sh = block < 0 ? last : block;
            left_sh = block < 0 ? __builtin_inf() : left;
            found = 0xffffffffu;
        }
    }
    __syncthreads();
    const float top = value_of(best_key);
    const Cut c = cut_of(a, r, w);
    const T* row = static_cast<const T*>(a.logits) + r * a.stride;
    const int32_t i = block_sh * kBlockTokens + tid * 8;
    double y[8], sum = 0.0;
    float x[8];
    load8(row, std::min(i, a.vocab), a.vocab, x);
#pragma unroll
    for (int e = 0; e < 8; e++) {
        y[e] = i < a.vocab ? kept_weight(x[e], i + e, top, w, c) : 0.0;
        sum += y[e];
    }
    double at = wave_scan_f64(sum);
    if (lane == 63) sh[wave] = at;
    __syncthreads();
    at -= sum;
    for (int k = 0; k < wave; k++) at += sh[k];
    uint32_t last = 0, first = 0xffffffffu;  // (the last one's index and one)
#pragma unroll
    for (int e = 0; e < 8; e++) {
        at += y[e];
        if (y[e] > 0.0) {
            last = static_cast<uint32_t>(i + e) + 1;
            if (first == 0xffffffffu && at > left_sh) first = static_cast<uint32_t>(i + e);
        }
    }
    if (first != 0xffffffffu) atomicMin(&found, first);
    __syncthreads();
    if (found != 0xffffffffu) {
        if (tid == 0) a.out[r] = static_cast<int32_t>(found);
        return;
    }
    __syncthreads();
    if (last) atomicMin(&found, 0xffffffffu - last);
    __syncthreads();
    if (tid == 0) a.out[r] = found != 0xffffffffu ? static_cast<int32_t>(0xffffffffu - found - 1) : static_cast<int32_t>(best_at);
}

template <typename T>
int launch(neko_hip_ctx* ctx, const char* what, const SampleArgs& a, int64_t rows) {
    const uint32_t parts = static_cast<uint32_t>(rows * a.n_max);
    hipLaunchKernelGGL((sample_max<T>), dim3(parts), dim3(256), 0, ctx->stream, a);
    if (int rc = after_launch(ctx, what)) return rc;
    if (a.top_k || a.top_p) {
        hipLaunchKernelGGL((sample_hist<T>), dim3(static_cast<uint32_t>(rows * a.n_hist)), dim3(256), 0, ctx->stream, a);
        if (int rc = after_launch(ctx, what)) return rc;
        hipLaunchKernelGGL((sample_cut<T>), dim3(static_cast<uint32_t>(rows)), dim3(kCutThreads), 0, ctx->stream, a);
        if (int rc = after_launch(ctx, what)) return rc;
    }
    hipLaunchKernelGGL((sample_sum<T>), dim3(parts), dim3(256), 0, ctx->stream, a);
    if (int rc = after_launch(ctx, what)) return rc;
    hipLaunchKernelGGL((sample_pick<T>), dim3(static_cast<uint32_t>(rows)), dim3(256), 0, ctx->stream, a);
    return after_launch(ctx, what);
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
    for (const void* p : {static_cast<const void*>(temperature), static_cast<const void*>(top_k), static_cast<const void*>(top_p),
                          static_cast<const void*>(min_p), static_cast<const void*>(u)})
        NEKO_REQUIRE(ctx, !p || !overlaps(tokens, n, p, n), "%s: tokens may not overlap the settings", what);
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
    // About four workgroups to a CU over all rows; a histogram is read again whole, so fewer of those.
    auto split = [&](int64_t wanted, int32_t* parts, int32_t* tokens_of) {
        const int64_t most = std::max<int64_t>(1, std::min<int64_t>(a.n_blocks, (wanted + rows - 1) / rows));
        const int64_t blocks = (a.n_blocks + most - 1) / most;
        *parts = static_cast<int32_t>((a.n_blocks + blocks - 1) / blocks);
        *tokens_of = static_cast<int32_t>(blocks * kBlockTokens);
    };
    split(4LL * ctx->cu_count, &a.n_max, &a.max_tokens);
    split(std::min<int64_t>(4LL * ctx->cu_count, 24 * rows), &a.n_hist, &a.hist_tokens);
    int bits = 0;
    while ((int64_t(1) << bits) < vocab) bits++;
    a.fixed = std::min(44, 62 - bits);
    const size_t best = static_cast<size_t>(rows) * a.n_max * 8, sums = static_cast<size_t>(rows) * a.n_blocks * 8,
                 hist = static_cast<size_t>(rows) * a.n_hist * kBins, cuts = static_cast<size_t>(rows) * sizeof(Cut);
    void* ws = nullptr;
    if (int rc = workspace(ctx, best + sums + cuts + hist * 12, &ws)) return rc;
    char* at = static_cast<char*>(ws);
    auto take = [&](size_t bytes) {
        char* p = at;
        at += bytes;
        return p;
    };
    a.best = reinterpret_cast<uint64_t*>(take(best));
    a.sums = reinterpret_cast<double*>(take(sums));
    a.cuts = reinterpret_cast<Cut*>(take(cuts));
    a.weights = reinterpret_cast<uint64_t*>(take(hist * 8));
    a.counts = reinterpret_cast<uint32_t*>(take(hist * 4));
    return dtype == NEKO_DT_F16 ? launch<half_t>(ctx, what, a, rows) : launch<float>(ctx, what, a, rows);
}
