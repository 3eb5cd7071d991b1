// Causal grouped-query attention over the paged 8-bit KV cache for gfx950: rows of few (token, head) pairs per
// sequence -- decoding -- one 16-row tile to a workgroup, the keys of a tile split over as many workgroups as fill the
// chip; and the merge of such splits.
//
// The query heads of a kv head share its K and V: (token, head) pairs are flattened into rows, 16 of them the columns
// of v_mfma_f32_16x16x32_f16. A wave takes 32 keys at a time, straight from the pages into registers (no other wave
// wants them): S^T = K Q^T with K's codes converted to f16 (exact), then O^T = V^T P^T. A contraction index may be
// permuted freely, so lane (c, g) of the first product reads 16 consecutive dimensions of key c, and of the second
// takes the weights where the first left them -- keys 4g .. 4g + 3 of both 16-key halves -- and reads of those eight
// keys' V rows the dimensions c * hd / 16 on, whose bytes v_perm pairs up by key.
//
// Scales. Page j has K scale 2^a and V scale 2^b for this head. 2^a joins the score's factor. 2^b goes into the
// exponent: with y_j = log2(weight) + b_j, O = sum 2^(y_j - m) code_j and l = sum 2^(y_j - m) 2^-b_j under one running
// maximum m of y, so no V code is ever scaled and weights rounded for the matrix cores are rounded relative to the
// largest term of O. m is an integer: rescaling by it is exact, and the exponent y_j - m comes from one fma. Weights
// are split into two f16 (24 bits of every weight above 2^-16 of the largest, 2^-39 of it below), f32 q as well, brought
// to [2^14, 2^15) first; l and O are f32.
//
// What bounds it: with many keys the reading of them, two sequences of 65521 tokens (32 / 8 heads of 128, f16) in 51 us,
// 5.3 TB/s of codes, and 5 for the merge; with fewer, launches and loads that wait for each other (32 ragged ones of up to
// 4096 tokens 18.1 us, one of 777 11.0). Of drafted trees, two of 7 tokens (28 rows) over 65500 53 us, 5.0 TB/s of codes, and
// 6 for the merge, one of 26 over 777 12.2.
#include <algorithm>
#include <atomic>

#include "attention_paged.h"

namespace neko_hip {
namespace {

constexpr int kTileRows = 16;
constexpr int kLeast = 8;           // tiles of 32 keys to a wave up to which a cache's keys are never split
constexpr int kFewRows = 32;        // flattened rows up to which a sequence is this kernel's
// Pairs of a query head's row and a key up to which the 16-row kernel alone is faster: it spreads them over more
// waves and starts sooner, the tiles convert a code once for 128 rows. 68 batches of 64 to 4000 rows, 8 to 32 heads
// of 64 to 256, each on both. f16: up to 8 million faster, half as long at a quarter of one (128 rows of 32 heads 7.3 us and
// 15.2), from 8 to 20 neither way by more than 1.3 times, slower past 30, 1.9 times as long at 67 (2048 rows 117 and 63).
// f32: faster up to 8 and mostly to 30 (1024 rows 45 and 59), level from there to 40, 1.2 times as long at 67.
template <typename TQ>
constexpr double kFewPairs = sizeof(TQ) == 2 ? 20e6 : 40e6;
// Drafted trees: two 16-row tiles to a workgroup where that is work enough, which halves what is loaded and converted, and
// sequences of more rows before the tiles of 128 are faster. 150 batches of 8 to 256 rows a sequence. f16 and 128
// dimensions: from 8 million pairs on faster (64 trees of 32 rows over 1500 keys 119 us one by one, 65 by two; 4 of 64 over
// 30000 189 and 87; 16 of 32 over 6000 68 and 52), and where the tiles one by one are more than are resident (16 of 128 rows
// over 300 20.4 and 15.6); slower below (one of 32 over 3000 16.7 and 17.2, 16 of 32 over 300 8.8 and 11.3). 64 dimensions
// have twice the waves: from 20 million (16 of 64 rows over 1500 32.7 and 35.3, 16 of 32 over 6000 60 and 45).
// The tiles of 128 against two of 16: f16, 64 trees of 64 rows over 1500 keys 133 us and 97, 4 of 96 over 30000 104 and
// 124; f32, whose conversion of q costs the tiles more, 4 of 96 over 30000 163 and 141, 64 of 128 over 1500 193 and 178.
template <typename TQ>
constexpr int kFewTreeRows = sizeof(TQ) == 2 ? 64 : 128;
template <int DH>
constexpr double kTwoPairs = DH <= 64 ? 20e6 : 8e6;
constexpr int kSpareRows = 256;     // flattened rows past one token to a sequence that still make a decoding batch

template <int N>
struct Words {
    uint32_t w[N];
};

// One wave's 32 keys: K as lane (c, g) of the first product wants it, V as of the second.
template <int DH>
struct KvTile {
    uint4v k[2][DH / 64];
    Words<DH / 64> v[2][4];
};

// Waves per SIMD that the kernel is compiled for. (At three, trees in f32 of 128 dimensions, one tile at a time, spill six or
// seven registers; 24 chains of up to 33 rows over up to 1021 tokens, 32 / 8 heads, take 33 us.)
template <typename TQ, int DH, int RT = 1>
constexpr int kResident = DH <= 64 ? (RT == 1 ? 4 : 3) : DH <= 128 ? (RT == 1 ? 3 : 2) : 1;

// Four dimensions, from d on, of a finished row.
template <typename TQ>
__device__ __forceinline__ void store_row(const PagedAttnArgs& a, const SeqRows& r, int kvh, int32_t row, int d, float4v x, float by) {
    const int32_t tok = static_cast<int32_t>(fast_div(static_cast<uint32_t>(row), a.by_group));
    const int head = kvh * a.t.group + (row - tok * a.t.group);
    TQ v[4];
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = from_f32<TQ>(by == 0.0f ? 0.0f : x[e] * by);
    __builtin_memcpy(static_cast<TQ*>(a.out) + static_cast<int64_t>(r.begin + tok) * a.os + static_cast<int64_t>(head) * a.p.hd + d, v, sizeof(v));
}

// TREE: rows of drafted trees (attention_paged.h). RT: 16-row tiles that a workgroup takes at once, each key's codes loaded
// and converted once for all.
template <typename TQ, int DH, int NW, bool MODS, bool TREE, int RT>
__global__ __launch_bounds__(64 * NW, (NW / 4 > kResident<TQ, DH, RT> ? NW / 4 : kResident<TQ, DH, RT>)) void attn_paged_kernel(PagedAttnArgs a) {
    constexpr bool kTwo = sizeof(TQ) == 4;
    constexpr int NU = DH / 64, NE = DH / 16, VW = DH / 64;
    constexpr int kRow = DH + 4;  // floats of a row in LDS
    extern __shared__ __align__(16) float o_sh[];  // [NW][16][kRow]
    __shared__ float m_sh[NW][16], l_sh[NW][16], seen_sh[NW][16];
    __shared__ half8 q_sh[RT][kTwo ? 2 : 1][2 * NU][64];
    __shared__ float sc_sh[RT][16];
    const int lane = static_cast<int>(threadIdx.x) & 63;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
    const int c = lane & 15, g4 = lane >> 4;
    int kvh;
    const uint32_t item = item_of(a, &kvh);
    // The item, by one wave for all: the search is issue-bound, and waves of a SIMD would do it in turn.
    __shared__ int32_t item_sh[16];
    if (wave == 0) {
        AttnItem f;
        const bool found = attn_find<false, TREE>(a.p, a.t, item, &f);
        if (found) {
            const SeqRows r = paged_seq(a.p, f.s);
            const TileKeys k = TREE ? tree_tile_keys(a, r, f) : tile_keys(a, r, f);
            if (lane == 0) {
                const int32_t x[14] = {f.s,      f.tile,   f.splits, static_cast<int32_t>(f.block), r.begin, r.n, r.len, k.lo_min,
                                       k.lo_max, k.hi_min, k.hi_max, k.k0, k.k1, 1};
#pragma unroll
                for (int i = 0; i < 14; i++) item_sh[i] = x[i];
            }
        } else if (lane == 0) {
            item_sh[13] = 0;
        }
    }
    __syncthreads();
    auto shared_at = [&](int i) { return __builtin_amdgcn_readfirstlane(item_sh[i]); };
    if (!shared_at(13)) return;
    AttnItem it;
    it.s = shared_at(0);
    it.tile = shared_at(1);
    it.splits = shared_at(2);
    it.block = static_cast<uint32_t>(shared_at(3));
    const SeqRows r = {shared_at(4), shared_at(5), shared_at(6)};
    const TileKeys tk = {shared_at(7), shared_at(8), shared_at(9), shared_at(10), shared_at(11), shared_at(12)};
    const int hd = a.p.hd;

    // This lane's rows (those past the last repeat it and are not written).
    const int32_t n_rows = r.n * a.t.group;
    int32_t tok[RT], depth[RT], pos[RT], hi[RT], lo[RT];
    int head[RT];
#pragma unroll
    for (int t = 0; t < RT; t++) {
        const int32_t row = min(((it.tile * RT + t) << 4) + c, n_rows - 1);
        tok[t] = static_cast<int32_t>(fast_div(static_cast<uint32_t>(row), a.by_group));
        head[t] = kvh * a.t.group + (row - tok[t] * a.t.group);
        depth[t] = TREE ? tree_depth(a, r, tok[t]) : tok[t];
        pos[t] = r.len - r.n + depth[t];
        hi[t] = TREE ? tk.hi_min : min(pos[t] + 1, min(r.len, paged_reach(a.p)));
        lo[t] = key_lo(pos[t], a.t.window);
    }

    // q as the B operands of the first product, the same for all waves, by one of them: in LDS, so that each
    // wave's registers have room for other things (168 of them at three waves per SIMD). f32 rows are brought to
    // [2^14, 2^15) and split; sc_sh then undoes that. A scale's sign goes into q; a scale of 0 weights all alike.
    if (wave >= 1 && wave <= RT) {
        const int t = wave - 1, mine = RT == 1 ? 0 : t;
        const int32_t my_tok = RT == 1 || t == 0 ? tok[0] : tok[RT - 1];
        const int my_head = RT == 1 || t == 0 ? head[0] : head[RT - 1];
        const TQ* qr = static_cast<const TQ*>(a.q) + static_cast<int64_t>(r.begin + my_tok) * a.qs + static_cast<int64_t>(my_head) * hd;
        const float sign = a.scale == 0.0f ? 0.0f : a.scale < 0.0f ? -1.0f : 1.0f;
        TQ x[2 * NU][8];
#pragma unroll
        for (int u = 0; u < 2 * NU; u++) {
            const int d = u / 2 * 64 + g4 * 16 + u % 2 * 8;
#pragma unroll
            for (int e = 0; e < 8; e++) x[u][e] = static_cast<TQ>(0.0f);
            if (d < hd) __builtin_memcpy(x[u], qr + d, sizeof(x[u]));
        }
        if constexpr (kTwo) {
            float mx = 0.0f;
#pragma unroll
            for (int u = 0; u < 2 * NU; u++)
#pragma unroll
                for (int e = 0; e < 8; e++) mx = fmaxf(mx, fabsf(x[u][e]));
            mx = swap32_max(swap16_max(mx));
            const int ex = mx > 0.0f && mx < __builtin_inff() ? 15 - __builtin_amdgcn_frexp_expf(mx) : 0;
            const int e1 = ex / 2, e2 = ex - e1;  // two factors of which each is a normal float
            sc_sh[mine][c] = ldexpf(a.scale == 0.0f ? 1.0f : fabsf(a.scale), -ex);
#pragma unroll
            for (int u = 0; u < 2 * NU; u++) {
                half8 y, z;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float v = ldexpf(ldexpf(x[u][e], e1), e2) * sign;
                    y[e] = static_cast<half_t>(v);
                    z[e] = static_cast<half_t>(v - to_f32(y[e]));
                }
                q_sh[mine][0][u][lane] = y;
                q_sh[mine][1][u][lane] = z;
            }
        } else {
#pragma unroll
            for (int u = 0; u < 2 * NU; u++) {
                half8 y;
                __builtin_memcpy(&y, x[u], sizeof(y));
                if (sign != 1.0f) y *= static_cast<half_t>(sign);
                q_sh[mine][0][u][lane] = y;
            }
        }
    }
    float slope[RT];
#pragma unroll
    for (int t = 0; t < RT; t++) slope[t] = MODS && a.slopes ? a.slopes[head[t]] : 0.0f;
    const float inv_cap = MODS && a.softcap > 0.0f ? fminf(1.0f / a.softcap, 0x1.fffffep127f) : 0.0f;

    // This wave's tiles of 32 keys, from key kw on.
    const int nt = tk.k1 > tk.k0 ? (tk.k1 - tk.k0 + 31) / 32 : 0;
    const int per = (nt + NW - 1) / NW;
    const int32_t kw = tk.k0 + 32 * per * wave;
    const int n = clamp_i32(nt - per * wave, 0, per);

    // Pages and scales of the next 64 blocks of 16 keys, one to a lane.
    int32_t page = -1;
    int ke = 0, ve = 0;
    auto look_up = [&](int tile) {
        const int32_t at = kw + 32 * tile + 16 * lane;
        page = -1;
        ke = ve = 0;
        if (lane < 2 * (n - tile) && at < tk.k1) page = paged_page(a.p, it.s, at);
        if (page >= 0) {
            const int64_t i = static_cast<int64_t>(page) * a.p.n_kv + kvh;
            ke = scale_exp(a.p.ks[i]);
            ve = scale_exp(a.p.vs[i]);
        }
    };
    // Offsets in a block of 16 keys. Dimensions past the head's end read its first ones, against zeros in q.
    uint32_t koff[NU];
#pragma unroll
    for (int u = 0; u < NU; u++) koff[u] = static_cast<uint32_t>(c * hd + (u * 64 + g4 * 16 < hd ? u * 64 + g4 * 16 : 0));
    const uint32_t voff = static_cast<uint32_t>(4 * g4 * hd + (c * VW * 4 < hd ? c * VW * 4 : 0));
    const uint8_t* k_head = a.p.k + kvh * a.p.head_bytes;
    const uint8_t* v_head = a.p.v + kvh * a.p.head_bytes;
    auto load = [&](int tile, KvTile<DH>& t) __attribute__((always_inline)) {
#pragma unroll
        for (int b = 0; b < 2; b++) {
            const int id = __builtin_amdgcn_readlane(page, 2 * (tile & 31) + b);
            // A block without a page reads page 0; its keys are masked. Every slot of a page may be read.
            const int32_t slot = (kw + 32 * tile + 16 * b) & ((1 << a.p.page_log2) - 1);
            const uint64_t at = static_cast<uint64_t>(static_cast<uint32_t>(id < 0 ? 0 : id)) * a.p.page_bytes + static_cast<uint32_t>(slot * hd);
            const uint8_t* kp = k_head + at;
            const uint8_t* vp = v_head + at;
#pragma unroll
            for (int u = 0; u < NU; u++) t.k[b][u] = *reinterpret_cast<const uint4v*>(kp + koff[u]);
#pragma unroll
            for (int i = 0; i < 4; i++) t.v[b][i] = *reinterpret_cast<const Words<VW>*>(vp + i * hd + voff);
        }
    };

    float4v o[RT][NE] = {};
    float m[RT], l[RT];
    bool seen[RT];
#pragma unroll
    for (int t = 0; t < RT; t++) {
        m[t] = -__builtin_inff();
        l[t] = 0.0f;
        seen[t] = false;
    }
    // acc += V^T B of one tile, four dimensions of each lane: x, a word of each key's row.
    auto product = [&](const uint32_t (&x)[2][4], const half8 (&bh)[RT], const half8 (&bl)[RT], int w) __attribute__((always_inline)) {
        half2v y[4][2][2];  // [dimension][block][key pair]
#pragma unroll
        for (int b = 0; b < 2; b++) {
            const uint32_t t0 = __builtin_amdgcn_perm(x[b][1], x[b][0], 0x05010400u);
            const uint32_t t1 = __builtin_amdgcn_perm(x[b][3], x[b][2], 0x05010400u);
            const uint32_t t2 = __builtin_amdgcn_perm(x[b][1], x[b][0], 0x07030602u);
            const uint32_t t3 = __builtin_amdgcn_perm(x[b][3], x[b][2], 0x07030602u);
            y[0][b][0] = f16_of_fp8<false>(t0);
            y[0][b][1] = f16_of_fp8<false>(t1);
            y[1][b][0] = f16_of_fp8<true>(t0);
            y[1][b][1] = f16_of_fp8<true>(t1);
            y[2][b][0] = f16_of_fp8<false>(t2);
            y[2][b][1] = f16_of_fp8<false>(t3);
            y[3][b][0] = f16_of_fp8<true>(t2);
            y[3][b][1] = f16_of_fp8<true>(t3);
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const half8 A = {y[e][0][0][0], y[e][0][0][1], y[e][0][1][0], y[e][0][1][1],
                             y[e][1][0][0], y[e][1][0][1], y[e][1][1][0], y[e][1][1][1]};
#pragma unroll
            for (int t = 0; t < RT; t++) {
                o[t][4 * w + e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(A, bl[t], o[t][4 * w + e], 0, 0, 0);
                o[t][4 * w + e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(A, bh[t], o[t][4 * w + e], 0, 0, 0);
            }
        }
    };
    auto step = [&](int tile, KvTile<DH>& t, int32_t pages, int kes, int ves) __attribute__((always_inline)) {
        const int32_t j0 = kw + 32 * tile;
        int ke2[2], ve2[2];
        bool ok[2];
#pragma unroll
        for (int b = 0; b < 2; b++) {
            const int idx = 2 * (tile & 31) + b;
            ke2[b] = __builtin_amdgcn_readlane(kes, idx);
            ve2[b] = __builtin_amdgcn_readlane(ves, idx);
            ok[b] = __builtin_amdgcn_readlane(pages, idx) >= 0;
        }
        float4v s[RT][2] = {};
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
            for (int u = 0; u < NU; u++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    half8 A;
#pragma unroll
                    for (int w = 0; w < 2; w++) {
                        const half2v x0 = f16_of_fp8<false>(t.k[b][u][2 * h + w]), x1 = f16_of_fp8<true>(t.k[b][u][2 * h + w]);
                        A[4 * w] = x0[0];
                        A[4 * w + 1] = x0[1];
                        A[4 * w + 2] = x1[0];
                        A[4 * w + 3] = x1[1];
                    }
#pragma unroll
                    for (int rt = 0; rt < RT; rt++) {
                        if constexpr (kTwo) s[rt][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(A, q_sh[rt][1][2 * u + h][lane], s[rt][b], 0, 0, 0);
                        s[rt][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(A, q_sh[rt][0][2 * u + h][lane], s[rt][b], 0, 0, 0);
                    }
                }
        // Keys that some row of the tile does not see.
        const bool partial = j0 < tk.lo_max || j0 + 32 > tk.hi_min || !ok[0] || !ok[1];
        half8 ph[RT], pl[RT];
        uint32_t sees[RT];  // (TREE) the tile's keys that the row sees
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
        const float sc = kTwo ? sc_sh[rt][c] : a.scale == 0.0f ? 1.0f : fabsf(a.scale);
        float f[2];  // score -> exponent of 2
#pragma unroll
        for (int b = 0; b < 2; b++) {
            f[b] = sc * exp2i(ke2[b]);
            if constexpr (!MODS) f[b] *= kAttnLog2e;
            f[b] = fminf(fmaxf(f[b], 0x1p-120f), 0x1p120f);  // (never 0 or infinite: masked scores are -inf)
        }
        if constexpr (MODS) {
#pragma unroll
            for (int b = 0; b < 2; b++)
#pragma unroll
                for (int i = 0; i < 4; i++) s[rt][b][i] *= f[b];
            if (a.softcap > 0.0f) {
#pragma unroll
                for (int b = 0; b < 2; b++)
#pragma unroll
                    for (int i = 0; i < 4; i++) s[rt][b][i] = cap_score(s[rt][b][i], a.softcap, inv_cap);
            }
            if (a.slopes) {
                const bool in_tree = TREE && j0 + 32 > tk.hi_min;
#pragma unroll
                for (int b = 0; b < 2; b++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        int32_t j = j0 + 16 * b + 4 * g4 + i;
                        if (in_tree) j = tree_key_place(a, r, j);
                        s[rt][b][i] = __builtin_fmaf(slope[rt], static_cast<float>(j - pos[rt]), s[rt][b][i]);
                    }
            }
            f[0] = f[1] = kAttnLog2e;
        }
        sees[rt] = 0;
        bool any_visible = true;
        if (partial) {
            any_visible = false;
            if constexpr (TREE) sees[rt] = tree_sees(a, r, tok[rt], depth[rt], lo[rt], hi[rt], j0) & ((ok[0] ? 0xffffu : 0u) | (ok[1] ? 0xffff0000u : 0u));
            // Visible: lo <= j < hi, as one unsigned comparison; no key of a block without a page. Likewise what any row sees.
            const uint32_t many = hi[rt] > lo[rt] ? static_cast<uint32_t>(hi[rt] - lo[rt]) : 0u;
            const uint32_t many_any = tk.hi_max > tk.lo_min ? static_cast<uint32_t>(tk.hi_max - tk.lo_min) : 0u;
#pragma unroll
            for (int b = 0; b < 2; b++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int32_t j = j0 + 16 * b + 4 * g4 + i;
                    const bool vis = TREE ? (sees[rt] >> (16 * b + 4 * g4 + i) & 1u) != 0 : static_cast<uint32_t>(j - lo[rt]) < (ok[b] ? many : 0u);
                    s[rt][b][i] = vis ? s[rt][b][i] : -__builtin_inff();
                    any_visible |= vis;
                    if (rt > 0) continue;
                    // What no row sees may be anything, codes of no token included.
                    const bool held = static_cast<uint32_t>(j - tk.lo_min) < (ok[b] ? many_any : 0u);
#pragma unroll
                    for (int w = 0; w < VW; w++) t.v[b][i].w[w] = held ? t.v[b][i].w[w] : 0u;
                }
        }
        seen[rt] = seen[rt] || any_visible;
        float top = -__builtin_inff();
#pragma unroll
        for (int b = 0; b < 2; b++) {
            const float mx = fmaxf(fmaxf(s[rt][b][0], s[rt][b][1]), fmaxf(s[rt][b][2], s[rt][b][3]));
            top = fmaxf(top, __builtin_fmaf(mx, f[b], static_cast<float>(ve2[b])));
        }
        top = ceilf(swap32_max(swap16_max(top)));
        if (__any(top > m[rt])) {
            const float mn = fmaxf(m[rt], top);
            const float corr = __builtin_amdgcn_exp2f(m[rt] - (mn == -__builtin_inff() ? 0.0f : mn));
            m[rt] = mn;
            l[rt] *= corr;
#pragma unroll
            for (int e = 0; e < NE; e++)
#pragma unroll
                for (int i = 0; i < 4; i++) o[rt][e][i] *= corr;
        }
        const float ms = m[rt] == -__builtin_inff() ? 0.0f : m[rt];
        float base[2] = {static_cast<float>(ve2[0]) - ms, static_cast<float>(ve2[1]) - ms};
        if (__any(fabsf(ms) >= kFarMax)) {  // exponents in place of scores
#pragma unroll
            for (int b = 0; b < 2; b++) {
#pragma unroll
                for (int i = 0; i < 4; i++) s[rt][b][i] = exponent_of(s[rt][b][i], f[b], static_cast<float>(ve2[b]), ms);
                f[b] = 1.0f;
                base[b] = 0.0f;
            }
        }
#pragma unroll
        for (int b = 0; b < 2; b++) {
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[rt][b][i], f[b], base[b]));
                sum += p;
                const float y = p * kPScale;
                ph[rt][4 * b + i] = static_cast<half_t>(y);
                pl[rt][4 * b + i] = static_cast<half_t>(y - to_f32(ph[rt][4 * b + i]));
            }
            l[rt] = __builtin_fmaf(sum, exp2i(-ve2[b]), l[rt]);
        }
        }
        // A NaN code times a weight of zero is NaN, so where rows see different keys NaN codes are taken out, noted by
        // key and lane in this wave's part of the LDS that is free until the end, and put into the dimensions of the
        // rows that do see them.
        uint16_t* nan_at = reinterpret_cast<uint16_t*>(o_sh + wave * kTileRows * kRow);  // [32 keys][16]
        bool mend = false;
        if (partial && (TREE || tk.hi_min != tk.hi_max || tk.lo_min != tk.lo_max)) {
            uint32_t any = 0;
#pragma unroll
            for (int b = 0; b < 2; b++)
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int w = 0; w < VW; w++) any |= nan_codes(t.v[b][i].w[w]);
            mend = __any(any != 0);
            if (mend) {
#pragma unroll
                for (int b = 0; b < 2; b++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        uint32_t at = 0;
#pragma unroll
                        for (int w = 0; w < VW; w++) {
                            const uint32_t nan = nan_codes(t.v[b][i].w[w]) >> 7;
                            t.v[b][i].w[w] &= ~(nan * 0xffu);
                            at |= ((nan * 0x01020408u) >> 24) << (4 * w);
                        }
                        nan_at[(16 * b + 4 * g4 + i) * 16 + c] = static_cast<uint16_t>(at);
                    }
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            }
        }
#pragma unroll
        for (int w = 0; w < VW; w++) {
            uint32_t x[2][4];
#pragma unroll
            for (int b = 0; b < 2; b++)
#pragma unroll
                for (int i = 0; i < 4; i++) x[b][i] = t.v[b][i].w[w];
            product(x, ph, pl, w);
        }
        if (mend) {
#pragma unroll 1
            for (int k = 0; k < 32; k++) {
#pragma unroll
                for (int rt = 0; rt < RT; rt++) {
                    if (TREE ? (sees[rt] >> k & 1u) == 0 : j0 + k < lo[rt] || j0 + k >= hi[rt]) continue;  // (a block without a page has no NaN left)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const uint32_t at = nan_at[k * 16 + 4 * g4 + i];
#pragma unroll
                        for (int e = 0; e < NE; e++)
                            o[rt][e][i] = nan_if(o[rt][e][i], at, e);
                    }
                }
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
    };

    if (n > 0) look_up(0);
    KvTile<DH> t, next;
    if (n > 0) load(0, t);
    __syncthreads();  // q is there
    for (int i = 0; i < n; i++) {
        asm volatile("" ::: "memory");  // (q is read again for each tile)
        const int32_t page_now = page;
        const int ke_now = ke, ve_now = ve;
        if (i + 1 < n) {
            if (((i + 1) & 31) == 0) look_up(i + 1);
            load(i + 1, next);
        }
        step(i, t, page_now, ke_now, ve_now);
        t = next;
    }

    constexpr int LPR = DH / 4;  // threads to a row, four dimensions each
    const uint32_t block = it.block * static_cast<uint32_t>(a.p.n_kv) + kvh;
    if (it.splits > 1 && block >= a.blocks) return;
#pragma unroll
    for (int t = 0; t < RT; t++) {
        if (t > 0) __syncthreads();  // (the LDS of the tile before)
        if (TREE && depth[t] < 0) {  // (tiles that all others see whole are not masked for a row that sees nothing)
            m[t] = -__builtin_inff();
            l[t] = 0.0f;
            seen[t] = false;
        }
        // The waves' results meet in LDS.
        l[t] = swap32_sum(swap16_sum(l[t]));
        const float any_seen = swap32_max(swap16_max(seen[t] ? 1.0f : 0.0f));
        if (g4 == 0) {
            m_sh[wave][c] = m[t];
            l_sh[wave][c] = l[t];
            seen_sh[wave][c] = any_seen;
        }
        const int32_t row0 = (it.tile * RT + t) << 4;
        const int rows_here = min(kTileRows, n_rows - row0);
        if (c < rows_here) {
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int e = 0; e < NE; e += 4)
                    *reinterpret_cast<float4v*>(o_sh + (wave * kTileRows + c) * kRow + (4 * g4 + i) * NE + e) =
                        float4v{o[t][e][i], o[t][e + 1][i], o[t][e + 2][i], o[t][e + 3][i]};
        }
        __syncthreads();
        for (int i = static_cast<int>(threadIdx.x) / LPR; i < rows_here; i += 64 * NW / LPR) {
            const int d = static_cast<int>(threadIdx.x) % LPR * 4;
            float mm = -__builtin_inff(), ll = 0.0f, ss = 0.0f;
#pragma unroll
            for (int w = 0; w < NW; w++) mm = fmaxf(mm, m_sh[w][i]);
            const float ms = mm == -__builtin_inff() ? 0.0f : mm;
            float4v x = {};
#pragma unroll 4
            for (int w = 0; w < NW; w++) {
                const float f = __builtin_amdgcn_exp2f(m_sh[w][i] - ms);
                const float4v y = *reinterpret_cast<const float4v*>(o_sh + (w * kTileRows + i) * kRow + d);
                ll = __builtin_fmaf(l_sh[w][i], f, ll);
                ss = fmaxf(ss, seen_sh[w][i]);
#pragma unroll
                for (int e = 0; e < 4; e++) x[e] = __builtin_fmaf(y[e], f, x[e]);
            }
            if (it.splits > 1) {
                const int64_t at = (static_cast<int64_t>(block) * RT + t) * kTileRows + i;
                *reinterpret_cast<float4v*>(a.part + at * DH + d) = x;
                if (d == 0) *reinterpret_cast<float4v*>(a.ml + at * 4) = float4v{mm, ll, ss, 0.0f};
            } else if (d < hd) {
                store_row<TQ>(a, r, kvh, row0 + i, d, x, row_factor(ll, ss > 0.0f));
            }
        }
    }
}

// Joins the splits of one tile, eight rows of 128 dimensions to a workgroup: DH / 4 lanes to a row, four dimensions
// each, the partial results of eight splits asked for at once.
template <typename TQ, int DH, bool TREE>
__global__ __launch_bounds__(256) void attn_paged_merge(PagedAttnArgs a) {
    constexpr int LPR = DH / 4, RPB = 256 / LPR, AHEAD = 8;
    int kvh;
    const uint32_t item = item_of(a, &kvh);
    AttnItem it;
    if (!attn_find<true, TREE>(a.p, a.t, item, &it)) return;
    const SeqRows r = paged_seq(a.p, it.s);
    const int d = static_cast<int>(threadIdx.x) % LPR * 4;
    if ((static_cast<uint64_t>(it.block) + static_cast<uint64_t>(it.splits)) * static_cast<uint32_t>(a.p.n_kv) > a.blocks) return;
    for (int i = static_cast<int>(blockIdx.y) * RPB + static_cast<int>(threadIdx.x) / LPR; i < 1 << a.t.tile_log2; i += static_cast<int>(gridDim.y) * RPB) {
        const int32_t row = (it.tile << a.t.tile_log2) + i;
        const uint32_t n_kv = static_cast<uint32_t>(a.p.n_kv);
        if (row >= r.n * a.t.group) return;
        const int64_t first = (static_cast<int64_t>(it.block * n_kv + kvh) << a.t.tile_log2) + i, step = static_cast<int64_t>(n_kv) << a.t.tile_log2;
        float m = -__builtin_inff(), l = 0.0f, ss = 0.0f;
        float4v x = {};
        for (int k0 = 0; k0 < it.splits; k0 += AHEAD) {
            float4v s[AHEAD], p[AHEAD];
#pragma unroll
            for (int k = 0; k < AHEAD; k++) {
                const int64_t at = first + min(k0 + k, it.splits - 1) * step;
                s[k] = *reinterpret_cast<const float4v*>(a.ml + at * 4);
                p[k] = *reinterpret_cast<const float4v*>(a.part + at * DH + d);
            }
            float mn = m;
#pragma unroll
            for (int k = 0; k < AHEAD; k++) mn = fmaxf(mn, s[k][0]);
            const float ms = mn == -__builtin_inff() ? 0.0f : mn, corr = __builtin_amdgcn_exp2f(m - ms);
            m = mn;
            l *= corr;
#pragma unroll
            for (int e = 0; e < 4; e++) x[e] *= corr;
#pragma unroll
            for (int k = 0; k < AHEAD; k++) {
                if (k0 + k < it.splits) {
                    const float f = __builtin_amdgcn_exp2f(s[k][0] - ms);
                    l = __builtin_fmaf(s[k][1], f, l);
                    ss = fmaxf(ss, s[k][2]);
#pragma unroll
                    for (int e = 0; e < 4; e++) x[e] = __builtin_fmaf(p[k][e], f, x[e]);
                }
            }
        }
        if (d < a.p.hd) store_row<TQ>(a, r, kvh, row, d, x, row_factor(l, ss > 0.0f));
        if (!TREE) break;
    }
}

// Workgroups of a launch and the bytes of its partial results, from its tiling.
struct Grid {
    int64_t blocks;
    size_t bytes;
};
Grid grid_of(const PagedAttnArgs& a, int dh) {
    Grid g;
    g.blocks = attn_blocks_bound(a.t, a.p.rows, a.p.n_seq, a.p.n_kv) * a.p.n_kv;
    g.bytes = attn_may_split(a.t, a.p) ? (static_cast<size_t>(g.blocks) << a.t.tile_log2) * (dh + 4) * sizeof(float) : 0;
    return g;
}

// The tiling of the 16-row kernel (tile_log2 is set) with `waves` waves to a workgroup, `resident` workgroups to a CU.
void few_form(const neko_hip_ctx* ctx, PagedAttnArgs& a, int waves, int resident) {
    a.t.unit_log2 = 5 + __builtin_ctz(static_cast<unsigned>(waves));
    a.t.least = paged_reach(a.p) <= (kLeast << a.t.unit_log2) ? kLeast : kLeast / 2;
    a.t.target = resident * ctx->cu_count;
    attn_form(a);
}

template <typename TQ, int DH, int NW, bool MODS, bool TREE, int RT>
int launch_few(neko_hip_ctx* ctx, const char* what, const PagedAttnArgs& a) {
    static std::atomic<uint64_t> allowed{0};
    constexpr size_t lds = NW * kTileRows * (DH + 4) * sizeof(float);
    if (lds + 4096 + RT * (sizeof(TQ) == 4 ? 2 : 1) * DH * 32 > 64 * 1024)
        if (int rc = allow_lds(ctx, reinterpret_cast<const void*>(&attn_paged_kernel<TQ, DH, NW, MODS, TREE, RT>), lds, allowed)) return rc;
    hipLaunchKernelGGL((attn_paged_kernel<TQ, DH, NW, MODS, TREE, RT>), dim3(a.blocks), dim3(64 * NW), lds, ctx->stream, a);
    return after_launch(ctx, what);
}

template <typename TQ, int DH>
int launch_dims(neko_hip_ctx* ctx, const char* what, PagedAttnArgs a, int dtype) {
    // Sequences of up to few_rows rows on the 16-row kernel, the rest on the tiles. Which a batch has is known on the
    // device alone, so both are launched, except where there is one sequence, where there are no more rows than a
    // padded decoding batch has, or where all there can be is little: then the 16-row kernel takes whatever there is.
    const int64_t most = static_cast<int64_t>(a.p.rows) * a.t.group;
    const int64_t reach = paged_reach(a.p), per_row = std::max(reach / 2, reach - a.p.rows / (2 * a.p.n_seq));
    const double pairs = static_cast<double>(a.p.rows) * a.n_head * static_cast<double>(a.t.window > 0 ? std::min<int64_t>(per_row, a.t.window) : per_row);
    // (f32 of 256 dimensions: 256 bytes of a lane's registers spill; f16 of 256 with a cap or bias 36, f32 of 128 with one 8)
    constexpr bool kTwoFit = sizeof(TQ) == 2 || DH <= 128;
    const int few_rows = a.words > 0 && kTwoFit ? kFewTreeRows<TQ> : kFewRows;
    const int64_t some = a.words > 0 ? static_cast<int64_t>(a.p.n_seq) * few_rows : static_cast<int64_t>(a.p.n_seq) * a.t.group + kSpareRows;
    const bool many = pairs > kFewPairs<TQ> && most > (a.p.n_seq == 1 ? few_rows : some);
    const bool few = a.p.n_seq > 1 || !many;
    constexpr int kMostWaves = DH <= 128 ? 8 : 4;
    PagedAttnArgs f = a, t = a;
    // Few items: many waves to each, whose results meet in LDS.
    const bool two = kTwoFit && a.words > 0 && most > 16 * static_cast<int64_t>(a.p.n_seq) &&
                     (pairs > kTwoPairs<DH> || most / 16 * a.p.n_kv > kResident<TQ, 128> * ctx->cu_count);
    f.t.tile_log2 = two ? 5 : 4;
    const int64_t items = attn_tiles_bound(f.t, a.p.rows, a.p.n_seq) * a.p.n_kv;
    const bool wide = items <= (two ? ctx->cu_count / 4 : ctx->cu_count);
    const int resident = two ? kResident<TQ, DH, 2> : kResident<TQ, DH>;
    few_form(ctx, f, wide ? kMostWaves : 4, wide ? resident * 4 / kMostWaves : resident);
    f.t.min_rows = 1;
    f.t.max_rows = many ? few_rows : 0x7fffffff;
    attn_paged_tile_form(ctx, t);
    t.t.min_rows = few ? few_rows + 1 : 1;
    t.t.max_rows = 0x7fffffff;
    const Grid fg = few ? grid_of(f, DH) : Grid{}, tg = many ? grid_of(t, DH) : Grid{};
    NEKO_REQUIRE(ctx, fg.blocks <= 0x7fffffff && tg.blocks <= 0x7fffffff, "%s: grid too large", what);
    void* ws = nullptr;
    if (fg.bytes + tg.bytes)
        if (int rc = workspace(ctx, fg.bytes + tg.bytes, &ws)) return rc;
    const bool mods = a.softcap > 0.0f || a.slopes;
    auto place = [](PagedAttnArgs& x, const Grid& g, void* at) {
        x.blocks = static_cast<uint32_t>(g.blocks);
        x.part = static_cast<float*>(at);
        x.ml = x.part + (g.blocks << x.t.tile_log2) * DH;
    };
    auto merge = [&](const PagedAttnArgs& x) {
        if (!attn_may_split(x.t, x.p)) return NEKO_OK;
        const int64_t tiles = attn_split_tiles_bound(x.t, x.p.rows, x.p.n_seq, x.p.n_kv) * x.p.n_kv;
        // Of trees, of whose tiles each workgroup searches longer (attention_paged.h), no more than are resident at once, which
        // go on with a tile's next rows (16 trees of up to 64 rows over up to 8192 keys 15 us, now 11).
        const int64_t parts = (DH << x.t.tile_log2) / 1024, wanted = x.words > 0 ? std::max<int64_t>(4, (6 * ctx->cu_count + tiles - 1) / tiles) : parts;
        const dim3 grid(static_cast<uint32_t>(tiles), static_cast<uint32_t>(std::min(parts, wanted)));
        if (x.words > 0) hipLaunchKernelGGL((attn_paged_merge<TQ, DH, true>), grid, dim3(256), 0, ctx->stream, x);
        else hipLaunchKernelGGL((attn_paged_merge<TQ, DH, false>), grid, dim3(256), 0, ctx->stream, x);
        return after_launch(ctx, what);
    };
    if (many) {
        place(t, tg, static_cast<char*>(ws) + fg.bytes);
        if (int rc = attn_paged_tile(ctx, what, t, dtype)) return rc;
        if (int rc = merge(t)) return rc;
    }
    if (few) {
        place(f, fg, ws);
        int rc = NEKO_OK;
        auto by_form = [&](auto tree, auto tiles) {
            constexpr bool TREE = decltype(tree)::value;
            constexpr int RT = decltype(tiles)::value;
            if (wide) return mods ? launch_few<TQ, DH, kMostWaves, true, TREE, RT>(ctx, what, f) : launch_few<TQ, DH, kMostWaves, false, TREE, RT>(ctx, what, f);
            return mods ? launch_few<TQ, DH, 4, true, TREE, RT>(ctx, what, f) : launch_few<TQ, DH, 4, false, TREE, RT>(ctx, what, f);
        };
        constexpr std::integral_constant<int, 1> one{};
        if constexpr (kTwoFit) {
            if (two) rc = by_form(std::true_type{}, std::integral_constant<int, 2>{});
        }
        if (!two) rc = a.words > 0 ? by_form(std::true_type{}, one) : by_form(std::false_type{}, one);
        if (rc) return rc;
        if (int rc2 = merge(f)) return rc2;
    }
    return NEKO_OK;
}

template <typename TQ>
int launch_typed(neko_hip_ctx* ctx, const char* what, const PagedAttnArgs& a, int dtype) {
    if (a.p.hd <= 64) return launch_dims<TQ, 64>(ctx, what, a, dtype);
    if (a.p.hd <= 128) return launch_dims<TQ, 128>(ctx, what, a, dtype);
    return launch_dims<TQ, 256>(ctx, what, a, dtype);
}

}  // namespace
}  // namespace neko_hip

using namespace neko_hip;

// `tree`: null for rows in a line.
static int attention(neko_hip_ctx* ctx, const char* what, const void* q, int64_t q_stride, int64_t rows, const neko_paged_kv* kv,
                     const neko_paged_batch* batch, const neko_paged_tree* tree, int n_head, float scale, float softcap,
                     int64_t window, const float* slopes, void* out, int64_t out_stride, int dtype) {
    NEKO_REQUIRE(ctx, valid_dtype(dtype), "%s: bad dtype %d", what, dtype);
    NEKO_REQUIRE(ctx, rows >= 0, "%s: rows=%lld", what, (long long)rows);
    PagedAttnArgs a{};
    if (int rc = paged_args(ctx, what, kv, batch, rows, &a.p)) return rc;
    NEKO_REQUIRE(ctx, n_head > 0 && n_head % kv->n_kv == 0, "%s: n_head=%d must be a positive multiple of n_kv=%d", what, n_head,
                 kv->n_kv);
    NEKO_REQUIRE(ctx, std::isfinite(scale) && std::isfinite(softcap) && softcap >= 0.0f && window >= 0,
                 "%s: scale=%g softcap=%g window=%lld (finite, the latter two not negative)", what, scale, softcap, (long long)window);
    NEKO_REQUIRE(ctx, rows * n_head <= 0x3fffffff, "%s: too many rows x heads", what);
    NEKO_REQUIRE(ctx, !tree || (tree->words > 0 && tree->words <= 32 && tree->mask_stride >= tree->words && tree->mask_stride <= (int64_t(1) << 32)),
                 "%s: masks of %d words (1..32), row stride %lld", what, tree->words, (long long)tree->mask_stride);
    if (rows == 0) return NEKO_OK;
    NEKO_REQUIRE(ctx, q && out, "%s: null pointer", what);
    const int64_t width = static_cast<int64_t>(n_head) * kv->hd;
    NEKO_REQUIRE(ctx, q_stride >= width && out_stride >= width, "%s: q / out row strides (%lld, %lld) below n_head*hd = %lld", what,
                 (long long)q_stride, (long long)out_stride, (long long)width);
    const size_t esz = dtype_size(dtype);
    NEKO_REQUIRE(ctx, aligned(q, esz) && aligned(out, esz), "%s: misaligned rows", what);
    const size_t sq = rows_span(rows, width, q_stride, esz), so = rows_span(rows, width, out_stride, esz);
    NEKO_REQUIRE(ctx, sq != 0 && so != 0, "%s: q / out rows span more than 2^62 bytes", what);
    NEKO_REQUIRE(ctx, !overlaps(out, so, q, sq) && !paged_overlaps(*kv, out, so), "%s: out may not overlap q or the cache", what);
    if (tree) {
        NEKO_REQUIRE(ctx, tree->depth && tree->mask && aligned(tree->depth, 4) && aligned(tree->mask, 4), "%s: null or misaligned depth or mask", what);
        const size_t sm = rows_span(rows, tree->words, tree->mask_stride, 4), sd = static_cast<size_t>(rows) * 4;
        NEKO_REQUIRE(ctx, sm != 0 && !overlaps(out, so, tree->mask, sm) && !overlaps(out, so, tree->depth, sd),
                     "%s: out may not overlap depth or mask", what);
        a.depth = tree->depth;
        a.mask = tree->mask;
        a.mask_stride = tree->mask_stride;
        a.words = tree->words;
        a.tree_rows = static_cast<int32_t>(std::min<int64_t>(rows, 32 * static_cast<int64_t>(tree->words)));
    }
    a.q = q;
    a.qs = q_stride;
    a.out = out;
    a.os = out_stride;
    a.n_head = n_head;
    a.t.group = n_head / kv->n_kv;
    a.t.window = window < (1 << 30) ? static_cast<int32_t>(window) : 0;
    a.by_group = make_fast_div(static_cast<uint32_t>(a.t.group));
    a.by_kv = make_fast_div(static_cast<uint32_t>(kv->n_kv));
    a.scale = scale;
    a.softcap = softcap;
    a.slopes = slopes;
    return dtype == NEKO_DT_F16 ? launch_typed<half_t>(ctx, what, a, dtype) : launch_typed<float>(ctx, what, a, dtype);
}

extern "C" int neko_hip_attention_paged(neko_hip_ctx* ctx, const void* q, int64_t q_stride, int64_t rows,
                                        const neko_paged_kv* kv, const neko_paged_batch* batch, int n_head, float scale,
                                        float softcap, int64_t window, const float* slopes, void* out, int64_t out_stride,
                                        int dtype) {
    NEKO_ENTER(ctx);
    return attention(ctx, "neko_hip_attention_paged", q, q_stride, rows, kv, batch, nullptr, n_head, scale, softcap, window, slopes,
                     out, out_stride, dtype);
}

extern "C" int neko_hip_attention_tree_paged(neko_hip_ctx* ctx, const void* q, int64_t q_stride, int64_t rows,
                                             const neko_paged_kv* kv, const neko_paged_batch* batch, const neko_paged_tree* tree,
                                             int n_head, float scale, float softcap, int64_t window, const float* slopes,
                                             void* out, int64_t out_stride, int dtype) {
    const char* what = "neko_hip_attention_tree_paged";
    NEKO_ENTER(ctx);
    NEKO_REQUIRE(ctx, tree, "%s: null tree", what);
    return attention(ctx, what, q, q_stride, rows, kv, batch, tree, n_head, scale, softcap, window, slopes, out, out_stride, dtype);
}
