// Shared by the paged attention kernels: the launch arguments, a workgroup's item, masks and partial results.
#pragma once

#include "internal.h"
#include "paged_device.h"

namespace neko_hip {

struct PagedAttnArgs {
    Paged p;
    AttnTiling t;
    const void* q;
    int64_t qs;
    void* out;
    int64_t os;
    int32_t n_head;
    FastDiv by_group;  // flattened row -> token
    FastDiv by_kv;     // workgroup -> (item, kv head)
    float scale;     // of the scores; its sign goes into q
    float softcap;   // 0: none
    const float* slopes;
    // Drafted trees (words 0: none): a row's depth in its tree, and a bit for each row of the tree that it sees.
    const int32_t* depth;
    const uint32_t* mask;
    int64_t mask_stride;
    int32_t words;
    int32_t tree_rows;  // of a tree, at most
    float* part;  // [blocks][tile_rows][head size of the kernel] accumulators of split items
    float* ml;    // [blocks][tile_rows][4]: their maximum, sum, whether any key was seen
    uint32_t blocks;  // that part and ml hold
};

// The tiling's derived fields. A tile of a tree's rows may see all of its tokens besides its window.
inline void attn_form(PagedAttnArgs& a) {
    attn_set(a.t);
    const int64_t span = static_cast<int64_t>(a.t.span) + a.tree_rows;
    a.t.span = span < (1 << 30) ? static_cast<int32_t>(span) : 1 << 30;
}

constexpr float kAttnLog2e = 1.44269504088896341f;
constexpr int kPOffset = 15;  // weights go to f16 times 2^kPOffset, the largest power that it holds
constexpr float kPScale = 1 << kPOffset;

// A weight's exponent is s * f + ve - m, rounded once, where m is the largest s * f + ve of the row, rounded before that.
// Past 2^24 the first may pass the second by a whole power of two or more, and the weight what f16 holds. Rows whose m is
// past this (by less than an eighth below it) take the rounded s * f + ve for both: the largest weight is 1 again.
constexpr float kFarMax = 0x1p22f;
__device__ __forceinline__ float exponent_of(float s, float f, float ve, float m) {
    return fabsf(m) >= kFarMax ? __builtin_fmaf(s, f, ve) - m : __builtin_fmaf(s, f, ve - m);
}

struct AttnItem {
    int32_t s, tile, split, splits;
    int32_t chunk;  // units of a split
    uint32_t block;  // index of the (tile, split) among those of a kv head
};

// Inclusive sum over the lanes below and at each (DPP: shifts within 16 lanes, then the rows' last lanes carried on).
__device__ __forceinline__ uint32_t wave_scan_u32(uint32_t v) {
    auto add = [&](auto ctrl, auto rows) {
        v += static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), decltype(ctrl)::value, decltype(rows)::value, 0xF, false));
    };
    add(std::integral_constant<int, 0x111>{}, std::integral_constant<int, 0xF>{});  // row_shr 1, 2, 4, 8
    add(std::integral_constant<int, 0x112>{}, std::integral_constant<int, 0xF>{});
    add(std::integral_constant<int, 0x114>{}, std::integral_constant<int, 0xF>{});
    add(std::integral_constant<int, 0x118>{}, std::integral_constant<int, 0xF>{});
    add(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xA>{});  // row_bcast 15 into rows 1 and 3
    add(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xC>{});  // row_bcast 31 into rows 2 and 3
    return v;
}

// The item of workgroup j of a kv head (SPLIT: the j-th tile that has splits, its first one), by every wave for itself:
// sequences' tiles and splits are summed 64 * K at a time, K of them to a lane. False past the last.
// TREE: as many splits as are resident at once and no more. A tree's sequence is all tiles of one length, and with a few
// workgroups past those the launch takes as long as with as many again (16 trees of up to 64 rows over up to 8192 keys: 616
// of 512 84 us, no more than these 74).
template <bool SPLIT, bool TREE, int K>
__device__ __forceinline__ bool attn_find_by(const Paged& p, const AttnTiling& t, uint32_t j, AttnItem* it) {
    const int32_t lane = static_cast<int32_t>(threadIdx.x) & 63;
    const int32_t reach = paged_reach(p);
    int32_t tiles[K], units[K];
    auto load = [&](int32_t base) {
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int32_t s = base + lane * K + k;
            const SeqRows r = paged_seq(p, s < p.n_seq ? s : p.n_seq - 1);
            tiles[k] = s < p.n_seq ? attn_tiles(t, r) : 0;
            units[k] = attn_units(t, reach, r);
        }
    };
    if (K == 1) load(0);
    int32_t chunk = attn_plan(t, p, [&](double& work, int64_t& n) {
        work = 0.0;  // (whole numbers below 2^53: exact)
        uint32_t all = 0;
        for (int32_t base = 0; base < p.n_seq; base += 64 * K) {
            if (K > 1) load(base);
#pragma unroll
            for (int k = 0; k < K; k++) {
                work += static_cast<double>(tiles[k]) * static_cast<double>(units[k]);
                all += static_cast<uint32_t>(tiles[k]);
            }
        }
        all = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(wave_scan_u32(all)), 63));
        work = wave_sum_f64(work) * p.n_kv;
        n = static_cast<int64_t>(all) * p.n_kv;
    });
    if (TREE && K == 1 && chunk < kUnsplit) {
        // 64 chunks from this one to about twice it, one to a lane (a quotient's rounding may count a split too many or few).
        const int32_t step = chunk / 64 + 1;
        const float by = __builtin_amdgcn_rcpf(static_cast<float>(chunk + lane * step));
        const float n = static_cast<float>(tiles[0]), of = static_cast<float>(units[0]);
        float blocks = 0.0f, all = 0.0f;
        for (int32_t s = 0; s < p.n_seq; s++) {
            const float n1 = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, n), s));
            const float of1 = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, of), s));
            blocks = __builtin_fmaf(n1, ceilf(of1 * by), blocks);
            all += n1;
        }
        const float room = static_cast<float>(t.target) * __builtin_amdgcn_rcpf(static_cast<float>(p.n_kv)) * 1.0001f;
        const uint64_t fits = __ballot(blocks <= room);
        if (__builtin_amdgcn_readfirstlane(all < room)) chunk += (fits ? __builtin_ctzll(fits) : 63) * step;
    }
    uint32_t past_tiles = 0, past = 0;  // of the sequences before
    for (int32_t base = 0; base < p.n_seq; base += 64 * K) {
        if (K > 1) load(base);
        int32_t splits[K];
        uint32_t n = 0, split_tiles = 0;
#pragma unroll
        for (int k = 0; k < K; k++) {
            splits[k] = attn_splits(units[k], chunk);
            n += static_cast<uint32_t>(tiles[k]) * static_cast<uint32_t>(splits[k]);
            split_tiles += splits[k] > 1 ? static_cast<uint32_t>(tiles[k]) : 0;
        }
        const uint32_t sum = wave_scan_u32(n), sum_tiles = SPLIT ? wave_scan_u32(split_tiles) : 0;
        const uint64_t at = __ballot(SPLIT ? past_tiles + sum_tiles > j : past + sum > j);
        if (at) {
            const int l = __builtin_ctzll(at);
            past += static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(sum - n), l));
            if constexpr (SPLIT) past_tiles += static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(sum_tiles - split_tiles), l));
            bool found = false;
#pragma unroll
            for (int k = 0; k < K; k++) {  // the lane's sequence that has it
                const int32_t n_tiles = __builtin_amdgcn_readlane(tiles[k], l), n_splits = __builtin_amdgcn_readlane(splits[k], l);
                const uint32_t here = static_cast<uint32_t>(n_tiles) * static_cast<uint32_t>(n_splits);
                const uint32_t split_here = n_splits > 1 ? static_cast<uint32_t>(n_tiles) : 0;
                if (!found && (SPLIT ? past_tiles + split_here > j : past + here > j)) {
                    found = true;
                    it->s = base + l * K + k;
                    it->splits = n_splits;
                    it->chunk = attn_splits(__builtin_amdgcn_readlane(units[k], l), n_splits);  // even ones
                    if constexpr (SPLIT) {
                        const uint32_t local = j - past_tiles;
                        it->tile = n_tiles - 1 - static_cast<int32_t>(local);
                        it->split = 0;
                        it->block = past + local * static_cast<uint32_t>(n_splits);
                    } else {  // the last tiles, which see the most keys, first
                        const uint32_t local = j - past;
                        const uint32_t up = n_splits == 1 ? local : local / static_cast<uint32_t>(n_splits);
                        it->tile = n_tiles - 1 - static_cast<int32_t>(up);
                        it->split = static_cast<int32_t>(local - up * static_cast<uint32_t>(n_splits));
                        it->block = j;
                    }
                }
                past += found ? 0 : here;
                past_tiles += found ? 0 : split_here;
            }
            return found;
        }
        past += static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(sum), 63));
        if constexpr (SPLIT) past_tiles += static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(sum_tiles), 63));
    }
    return false;
}
// One sequence to a lane where that holds the batch, else eight, whose loads wait for each other no more.
template <bool SPLIT, bool TREE>
__device__ __forceinline__ bool attn_find(const Paged& p, const AttnTiling& t, uint32_t j, AttnItem* it) {
    return p.n_seq <= 64 ? attn_find_by<SPLIT, TREE, 1>(p, t, j, it) : attn_find_by<SPLIT, TREE, 8>(p, t, j, it);
}

// The keys that a tile's rows see, first and last row: row i sees [lo(i), hi(i)).
struct TileKeys {
    int32_t lo_min, lo_max, hi_min, hi_max;
    int32_t k0, k1;  // this split's, k0 a multiple of 32
};
__device__ __forceinline__ int32_t key_lo(int32_t pos, int32_t window) { return window > 0 && pos >= window ? pos - window + 1 : 0; }
// This split's part of the keys that a tile's rows see.
__device__ __forceinline__ void split_keys(const PagedAttnArgs& a, const AttnItem& it, TileKeys& k) {
    k.k0 = k.lo_min & ~31;
    k.k1 = k.hi_max;
    if (it.splits > 1) {
        const int64_t per = static_cast<int64_t>(it.chunk) << a.t.unit_log2, from = k.k0 + it.split * per;
        k.k0 = static_cast<int32_t>(from < (1 << 30) ? from : 1 << 30);
        if (from + per < k.k1) k.k1 = static_cast<int32_t>(from + per);
    }
}
__device__ __forceinline__ TileKeys tile_keys(const PagedAttnArgs& a, const SeqRows& r, const AttnItem& it) {
    const int32_t n_rows = r.n * a.t.group, row0 = it.tile << a.t.tile_log2;
    const int32_t row1 = min(row0 + (1 << a.t.tile_log2), n_rows) - 1;
    const int32_t first = r.len - r.n + static_cast<int32_t>(fast_div(static_cast<uint32_t>(row0), a.by_group));
    const int32_t last = r.len - r.n + static_cast<int32_t>(fast_div(static_cast<uint32_t>(row1), a.by_group));
    const int32_t reach = min(r.len, paged_reach(a.p));
    TileKeys k;
    k.lo_min = key_lo(first, a.t.window);
    k.lo_max = key_lo(last, a.t.window);
    k.hi_min = min(first + 1, reach);
    k.hi_max = min(last + 1, reach);
    split_keys(a, it, k);
    return k;
}

// ---- drafted trees. Row i of a sequence's n, at depth d_i, stands at place base + d_i of the text, base = len - n being
// the tokens before the tree; it sees of those what its window allows and, of the tree, the slots base + k whose bit k is
// set in its row of the mask (places base + d_k).

// The keys that the tree's rows see: all of them, up to what the mask has bits for.
__device__ __forceinline__ int32_t tree_reach(const PagedAttnArgs& a, const SeqRows& r) {
    const int32_t base = r.len - r.n;
    if (base < 0) return 0;
    return min(min(r.len, paged_reach(a.p)), base + min(r.n, 32 * a.words));
}
__device__ __forceinline__ TileKeys tree_tile_keys(const PagedAttnArgs& a, const SeqRows& r, const AttnItem& it) {
    const int32_t base = max(r.len - r.n, 0), reach = tree_reach(a, r);
    TileKeys k;
    k.lo_min = key_lo(base, a.t.window);
    k.lo_max = key_lo(base + r.n, a.t.window);
    k.hi_min = min(base, reach);
    k.hi_max = reach;
    split_keys(a, it, k);
    return k;
}
// The depth of a row, -1 where it sees nothing.
__device__ __forceinline__ int32_t tree_depth(const PagedAttnArgs& a, const SeqRows& r, int32_t tok) {
    const int32_t d = a.depth[r.begin + tok];
    return r.len < r.n || d < 0 || d >= r.n ? -1 : d;
}
// Which of the keys j0 .. j0 + 31 the row `tok` at depth d sees, a bit each, pages aside. lo, hi: of the keys before the tree.
__device__ __forceinline__ uint32_t tree_sees(const PagedAttnArgs& a, const SeqRows& r, int32_t tok, int32_t d, int32_t lo, int32_t hi, int32_t j0) {
    auto below = [](int32_t n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u; };  // the first n
    uint32_t sees = below(hi - j0) & ~below(lo - j0);
    const int32_t base = r.len - r.n, k0 = j0 - base;  // the first key's row of the tree
    if (k0 > -32 && k0 < 32 * a.words) {
        const uint32_t* m = a.mask + static_cast<int64_t>(r.begin + tok) * a.mask_stride;
        const int32_t w = k0 >> 5, by = k0 & 31;
        const uint32_t m0 = w >= 0 ? m[w] : 0u, m1 = w + 1 < a.words ? m[w + 1] : 0u;
        uint32_t bits = (m0 >> by | (by ? m1 << (32 - by) : 0u)) & below(tree_reach(a, r) - j0);
        if (a.t.window > 0 && d >= a.t.window - 1) {  // a window that ends inside the tree (or at its root)
            for (uint32_t left = bits; left; left &= left - 1) {
                const int32_t k = __builtin_ctz(left);
                if (a.depth[r.begin + k0 + k] <= d - a.t.window) bits &= ~(1u << k);
            }
        }
        sees |= bits;
    }
    return d < 0 ? 0u : sees;
}
// The place in the text of key j, which holds a token.
__device__ __forceinline__ int32_t tree_key_place(const PagedAttnArgs& a, const SeqRows& r, int32_t j) {
    const int32_t base = r.len - r.n, k = j - base;
    return k < 0 || k >= r.n ? j : base + a.depth[r.begin + k];
}

// cap * tanh(s / cap) to a few roundings of the value: Lambert's continued fraction for tanh, cut after its fifth
// term, up to 0.9 (off by 0.9^10 / (945^2 * 11) = 4e-8 there, relative), 1 - 2 / (e^2x + 1) past it. (The latter
// alone is off by 2^-24 * cap whatever the score: 1.5e-6 of the results of prompts of up to 2048 keys with a cap of 50, 4.1e-7 now.)
__device__ __forceinline__ float cap_score(float s, float cap, float inv_cap) {
    const float x = s * inv_cap, x2 = x * x;
    const float n = __builtin_fmaf(x2, 105.0f + x2, 945.0f), d = __builtin_fmaf(x2, __builtin_fmaf(x2, 15.0f, 420.0f), 945.0f);
    const float near = s * n * __builtin_amdgcn_rcpf(d);
    const float far = cap * (1.0f - 2.0f * __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(x * (2.0f * kAttnLog2e)) + 1.0f));
    return fabsf(x) < 0.9f ? near : far;
}

// The larger of a lane's and its partner's, neither NaN (fmaxf quiets both first, an instruction each).
__device__ __forceinline__ float swap16_max(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    return __builtin_elementwise_maximum(__builtin_bit_cast(float, static_cast<uint32_t>(r[0])), __builtin_bit_cast(float, static_cast<uint32_t>(r[1])));
}
__device__ __forceinline__ float swap32_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    return __builtin_elementwise_maximum(__builtin_bit_cast(float, static_cast<uint32_t>(r[0])), __builtin_bit_cast(float, static_cast<uint32_t>(r[1])));
}
__device__ __forceinline__ float swap16_sum(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    return __builtin_bit_cast(float, static_cast<uint32_t>(r[0])) + __builtin_bit_cast(float, static_cast<uint32_t>(r[1]));
}
__device__ __forceinline__ float swap32_sum(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    return __builtin_bit_cast(float, static_cast<uint32_t>(r[0])) + __builtin_bit_cast(float, static_cast<uint32_t>(r[1]));
}

// Workgroup -> item number and kv head: the kv head fastest, so that with eight of them each XCD reads one head's part
// of the pages.
__device__ __forceinline__ uint32_t item_of(const PagedAttnArgs& a, int* kvh) {
    const uint32_t j = fast_div(blockIdx.x, a.by_kv);
    *kvh = static_cast<int>(blockIdx.x - j * a.by_kv.d);
    return j;
}

// The bytes of x that are NaN codes, as 0x80 each.
__device__ __forceinline__ uint32_t nan_codes(uint32_t x) { return ((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// x, or NaN where bit `bit` is set: two vector operations and no condition, of which dozens held at once would push the
// scalar registers of the whole kernel out (108 of them were, in the tiles of 128 dimensions).
__device__ __forceinline__ float nan_if(float x, uint32_t bits, int bit) {
    const uint32_t all = static_cast<uint32_t>(static_cast<int32_t>(bits << (31 - bit)) >> 31);
    return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, x) | (all & 0x7fc00000u));
}

// acc / l of a finished row: zeros where it saw nothing, NaN where every score it saw was -inf.
__device__ __forceinline__ float row_factor(float l, bool seen) {
    return l == 0.0f ? (seen ? __builtin_nanf("") : 0.0f) : 1.0f / (l * kPScale);
}

// The kernel for many rows per sequence (attention_paged_tile.hip): its tiling, into a.t, and its launch of a.blocks
// workgroups.
void attn_paged_tile_form(const neko_hip_ctx* ctx, PagedAttnArgs& a);
int attn_paged_tile(neko_hip_ctx* ctx, const char* what, const PagedAttnArgs& a, int dtype);  // (of drafted trees where a.words > 0)

}  // namespace neko_hip
