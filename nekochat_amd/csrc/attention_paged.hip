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
#include <algorithm>

#include "attention_paged.h"

namespace neko_hip {
namespace {

constexpr int kWaves = 4;
constexpr int kTileRows = 16;
constexpr int kUnit = 32 * kWaves;  // keys of a split: a whole tile for every wave
constexpr int kFewRows = 32;        // flattened rows up to which a sequence is this kernel's

template <int N>
struct Words {
    uint32_t w[N];
};

// One wave's 32 keys: K as lane (c, g) of the first product wants it, V as of the second.
template <int DH>
struct KvTile {
    uint4v k[2][DH / 64];
    Words<DH / 64> v[2][4];
    int ke[2], ve[2];  // scale exponents of the two 16-key blocks
    bool ok[2];        // whether they have a page
};

template <typename TQ, int DH, bool MODS>
__global__ __launch_bounds__(256) void attn_paged_kernel(PagedAttnArgs a) {
    constexpr bool kTwo = sizeof(TQ) == 4;
    constexpr int NU = DH / 64, NE = DH / 16, VW = DH / 64;
    __shared__ float m_sh[kWaves][16], l_sh[kWaves][16], seen_sh[kWaves][16];
    __shared__ float o_sh[kWaves][4][DH <= 128 ? NE : NE / 2][64];
    const int lane = static_cast<int>(threadIdx.x) & 63;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
    const int c = lane & 15, g4 = lane >> 4;
    const int kvh = static_cast<int>(blockIdx.x % static_cast<uint32_t>(a.p.n_kv));
    AttnItem it;
    if (!attn_find<false>(a.p, a.t, blockIdx.x / static_cast<uint32_t>(a.p.n_kv), &it)) return;
    const SeqRows r = paged_seq(a.p, it.s);
    const TileKeys tk = tile_keys(a, r, it);
    const int hd = a.p.hd;

    // This lane's row (rows past the last repeat it and are not written).
    const int32_t n_rows = r.n * a.t.group;
    const int32_t row = min(it.tile * kTileRows + c, n_rows - 1);
    const int32_t tok = row / a.t.group;
    const int head = kvh * a.t.group + (row - tok * a.t.group);
    const int32_t pos = r.len - r.n + tok;
    const int32_t hi = min(pos + 1, min(r.len, paged_reach(a.p))), lo = key_lo(pos, a.window);

    half8 qh[2 * NU], ql[kTwo ? 2 * NU : 1];
    // Of the scores, in natural units; a scale of 0 weights all alike.
    float sc = a.scale == 0.0f ? 1.0f : fabsf(a.scale);
    {
        const TQ* qr = static_cast<const TQ*>(a.q) + static_cast<int64_t>(r.begin + tok) * a.qs + static_cast<int64_t>(head) * hd;
        const float sign = a.scale == 0.0f ? 0.0f : a.scale < 0.0f ? -1.0f : 1.0f;
        float x[NU][16];
#pragma unroll
        for (int u = 0; u < NU; u++) {
            const int d = u * 64 + g4 * 16;
            TQ v[16];
            if (d < hd) __builtin_memcpy(v, qr + d, sizeof(v));
#pragma unroll
            for (int e = 0; e < 16; e++) x[u][e] = d < hd ? to_f32(v[e]) * sign : 0.0f;
        }
        if constexpr (kTwo) {
            float mx = 0.0f;
#pragma unroll
            for (int u = 0; u < NU; u++)
#pragma unroll
                for (int e = 0; e < 16; e++) mx = fmaxf(mx, fabsf(x[u][e]));
            mx = swap32_max(swap16_max(mx));
            const int ex = mx > 0.0f && mx < __builtin_inff() ? 15 - __builtin_amdgcn_frexp_expf(mx) : 0;
            const int e1 = ex / 2, e2 = ex - e1;  // two factors of which each is a normal float
            sc = ldexpf(sc, -ex);
#pragma unroll
            for (int u = 0; u < NU; u++)
#pragma unroll
                for (int e = 0; e < 16; e++) x[u][e] = ldexpf(ldexpf(x[u][e], e1), e2);
        }
#pragma unroll
        for (int u = 0; u < NU; u++)
#pragma unroll
            for (int e = 0; e < 16; e++) {
                qh[2 * u + e / 8][e % 8] = static_cast<half_t>(x[u][e]);
                if constexpr (kTwo) ql[2 * u + e / 8][e % 8] = static_cast<half_t>(x[u][e] - to_f32(qh[2 * u + e / 8][e % 8]));
            }
    }
    const float slope = MODS && a.slopes ? a.slopes[head] : 0.0f;
    const float inv_cap = MODS && a.softcap > 0.0f ? 1.0f / a.softcap : 0.0f;

    // This wave's tiles of 32 keys, from key kw on.
    const int nt = tk.k1 > tk.k0 ? (tk.k1 - tk.k0 + 31) / 32 : 0;
    const int per = (nt + kWaves - 1) / kWaves;
    const int32_t kw = tk.k0 + 32 * per * wave;
    const int n = clamp_i32(nt - per * wave, 0, per);

    // Pages and scales of the next 64 blocks of 16 keys, one to a lane.
    int32_t page = -1;
    int ke = 0, ve = 0;
    auto look_up = [&](int tile) {
        const int32_t at = kw + 32 * tile + 16 * lane;
        page = -1;
        ke = ve = 0;
        if (at < tk.k1) page = paged_page(a.p, it.s, at);
        if (page >= 0) {
            const int64_t i = static_cast<int64_t>(page) * a.p.n_kv + kvh;
            ke = scale_exp(a.p.ks[i]);
            ve = scale_exp(a.p.vs[i]);
        }
    };
    const int dk = g4 * 16, dv = c * VW * 4;
    auto load = [&](int tile, KvTile<DH>& t) {
#pragma unroll
        for (int b = 0; b < 2; b++) {
            const int idx = 2 * (tile & 31) + b;
            const int id = __builtin_amdgcn_readlane(page, idx);
            t.ke[b] = __builtin_amdgcn_readlane(ke, idx);
            t.ve[b] = __builtin_amdgcn_readlane(ve, idx);
            t.ok[b] = id >= 0;
            // A block without a page reads page 0; its keys are masked. Every slot of a page may be read.
            const int32_t slot = (kw + 32 * tile + 16 * b) & ((1 << a.p.page_log2) - 1);
            const int64_t at = ((static_cast<int64_t>(id < 0 ? 0 : id) * a.p.n_kv + kvh) << a.p.page_log2) + slot;
            const uint8_t* kp = a.p.k + at * hd;
            const uint8_t* vp = a.p.v + at * hd;
#pragma unroll
            for (int u = 0; u < NU; u++) {
                // Dimensions past the head's end read its first ones, against zeros in q.
                const int d = u * 64 + dk;
                t.k[b][u] = *reinterpret_cast<const uint4v*>(kp + (c * hd + (d < hd ? d : 0)));
            }
#pragma unroll
            for (int i = 0; i < 4; i++)
                t.v[b][i] = *reinterpret_cast<const Words<VW>*>(vp + ((4 * g4 + i) * hd + (dv < hd ? dv : 0)));
        }
    };

    float4v o[NE] = {};
    float m = -__builtin_inff(), l = 0.0f;
    bool seen = false;
    // O^T += V^T B of one tile.
    auto product = [&](const Words<VW> (&v)[2][4], half8 bh, half8 bl, bool two, float4v* acc) __attribute__((always_inline)) {
#pragma unroll
        for (int w = 0; w < VW; w++) {
            half2v x[4][2][2];  // [dimension][block][key pair]
#pragma unroll
            for (int b = 0; b < 2; b++) {
                const uint32_t t0 = __builtin_amdgcn_perm(v[b][1].w[w], v[b][0].w[w], 0x05010400u);
                const uint32_t t1 = __builtin_amdgcn_perm(v[b][3].w[w], v[b][2].w[w], 0x05010400u);
                const uint32_t t2 = __builtin_amdgcn_perm(v[b][1].w[w], v[b][0].w[w], 0x07030602u);
                const uint32_t t3 = __builtin_amdgcn_perm(v[b][3].w[w], v[b][2].w[w], 0x07030602u);
                x[0][b][0] = f16_of_fp8<false>(t0);
                x[0][b][1] = f16_of_fp8<false>(t1);
                x[1][b][0] = f16_of_fp8<true>(t0);
                x[1][b][1] = f16_of_fp8<true>(t1);
                x[2][b][0] = f16_of_fp8<false>(t2);
                x[2][b][1] = f16_of_fp8<false>(t3);
                x[3][b][0] = f16_of_fp8<true>(t2);
                x[3][b][1] = f16_of_fp8<true>(t3);
            }
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const half8 A = {x[e][0][0][0], x[e][0][0][1], x[e][0][1][0], x[e][0][1][1],
                                 x[e][1][0][0], x[e][1][0][1], x[e][1][1][0], x[e][1][1][1]};
                if (two) acc[4 * w + e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(A, bl, acc[4 * w + e], 0, 0, 0);
                acc[4 * w + e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(A, bh, acc[4 * w + e], 0, 0, 0);
            }
        }
    };
    auto step = [&](int tile, KvTile<DH>& t) __attribute__((always_inline)) {
        const int32_t j0 = kw + 32 * tile;
        float4v s[2] = {};
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
                    if constexpr (kTwo) s[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(A, ql[2 * u + h], s[b], 0, 0, 0);
                    s[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(A, qh[2 * u + h], s[b], 0, 0, 0);
                }
        float f[2];  // score -> exponent of 2
#pragma unroll
        for (int b = 0; b < 2; b++) {
            f[b] = sc * exp2i(t.ke[b]);
            if constexpr (!MODS) f[b] *= kAttnLog2e;
            f[b] = fminf(fmaxf(f[b], 0x1p-120f), 0x1p120f);  // (never 0 or infinite: masked scores are -inf)
        }
        if constexpr (MODS) {
#pragma unroll
            for (int b = 0; b < 2; b++) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    float x = s[b][i] * f[b];
                    if (a.softcap > 0.0f) x = cap_score(x, a.softcap, inv_cap);
                    if (a.slopes) x = __builtin_fmaf(slope, static_cast<float>(j0 + 16 * b + 4 * g4 + i - pos), x);
                    s[b][i] = x;
                }
                f[b] = kAttnLog2e;
            }
        }
        // Keys that some row of the tile does not see.
        const bool partial = j0 < tk.lo_max || j0 + 32 > tk.hi_min || !t.ok[0] || !t.ok[1];
        uint32_t visible = 0xff;
        if (partial) {
#pragma unroll
            for (int b = 0; b < 2; b++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int32_t j = j0 + 16 * b + 4 * g4 + i;
                    const bool vis = t.ok[b] && j >= lo && j < hi;
                    if (!vis) {
                        s[b][i] = -__builtin_inff();
                        visible &= ~(1u << (4 * b + i));
                    }
                    // What no row sees may be anything, codes of no token included.
                    if (!(t.ok[b] && j >= tk.lo_min && j < tk.hi_max)) t.v[b][i] = Words<VW>{};
                }
        }
        seen = seen || visible != 0;
        float top = -__builtin_inff();
#pragma unroll
        for (int b = 0; b < 2; b++) {
            const float mx = fmaxf(fmaxf(s[b][0], s[b][1]), fmaxf(s[b][2], s[b][3]));
            top = fmaxf(top, __builtin_fmaf(mx, f[b], static_cast<float>(t.ve[b])));
        }
        top = ceilf(swap32_max(swap16_max(top)));
        if (__any(top > m)) {
            const float mn = fmaxf(m, top);
            const float corr = __builtin_amdgcn_exp2f(m - (mn == -__builtin_inff() ? 0.0f : mn));
            m = mn;
            l *= corr;
#pragma unroll
            for (int e = 0; e < NE; e++)
#pragma unroll
                for (int i = 0; i < 4; i++) o[e][i] *= corr;
        }
        const float ms = m == -__builtin_inff() ? 0.0f : m;
        half8 ph, pl;
#pragma unroll
        for (int b = 0; b < 2; b++) {
            const float base = static_cast<float>(t.ve[b]) - ms;
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][i], f[b], base));
                sum += p;
                const float y = p * kPScale;
                ph[4 * b + i] = static_cast<half_t>(y);
                pl[4 * b + i] = static_cast<half_t>(y - to_f32(ph[4 * b + i]));
            }
            l = __builtin_fmaf(sum, exp2i(-t.ve[b]), l);
        }
        // A NaN code times a weight of zero is NaN, so where rows see different keys NaN codes are taken out and
        // put into the dimensions of the rows that do see them.
        if (partial && (tk.hi_min != tk.hi_max || tk.lo_min != tk.lo_max)) {
            uint32_t any = 0;
#pragma unroll
            for (int b = 0; b < 2; b++)
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int w = 0; w < VW; w++) any |= nan_codes(t.v[b][i].w[w]);
            if (__any(any != 0)) {
                Words<VW> bad[2][4];
                half8 sees;
#pragma unroll
                for (int b = 0; b < 2; b++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        sees[4 * b + i] = static_cast<half_t>((visible >> (4 * b + i)) & 1u ? 1.0f : 0.0f);
#pragma unroll
                        for (int w = 0; w < VW; w++) {
                            const uint32_t x = nan_codes(t.v[b][i].w[w]) >> 7;
                            bad[b][i].w[w] = x * 0x38u;  // the code of 1
                            t.v[b][i].w[w] &= ~(x * 0xffu);
                        }
                    }
                float4v count[NE] = {};
                product(bad, sees, sees, false, count);
#pragma unroll
                for (int e = 0; e < NE; e++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (count[e][i] > 0.0f) o[e][i] = __builtin_nanf("");
            }
        }
        product(t.v, ph, pl, true, o);
    };

    if (n > 0) {
        KvTile<DH> t0, t1;
        look_up(0);
        load(0, t0);
        for (int i = 0; i < n; i += 2) {
            // (32 tiles to a look-up, an even number, so only even tiles begin one)
            if (i + 1 < n) load(i + 1, t1);
            step(i, t0);
            if (i + 2 < n) {
                if (((i + 2) & 31) == 0) look_up(i + 2);
                load(i + 2, t0);
            }
            if (i + 1 < n) step(i + 1, t1);
        }
    }

    // The waves' results meet: every wave puts its own in LDS and joins a quarter of the dimensions, those of
    // accumulator element `wave`.
    l = swap32_sum(swap16_sum(l));
    const float any_seen = swap32_max(swap16_max(seen ? 1.0f : 0.0f));
    if (g4 == 0) {
        m_sh[wave][c] = m;
        l_sh[wave][c] = l;
        seen_sh[wave][c] = any_seen;
    }
    constexpr int NH = DH <= 128 ? NE : NE / 2;  // dimensions' blocks in LDS at once
    float res[NE];
    float f[kWaves], mm = -__builtin_inff(), ll = 0.0f, ss = 0.0f;
#pragma unroll
    for (int half = 0; half < NE / NH; half++) {
        if (half) __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int e = 0; e < NH; e++) o_sh[wave][i][e][lane] = o[half * NH + e][i];
        __syncthreads();
        if (half == 0) {
#pragma unroll
            for (int w = 0; w < kWaves; w++) mm = fmaxf(mm, m_sh[w][c]);
            const float ms = mm == -__builtin_inff() ? 0.0f : mm;
#pragma unroll
            for (int w = 0; w < kWaves; w++) {
                f[w] = __builtin_amdgcn_exp2f(m_sh[w][c] - ms);
                ll = __builtin_fmaf(l_sh[w][c], f[w], ll);
                ss = fmaxf(ss, seen_sh[w][c]);
            }
        }
#pragma unroll
        for (int e = 0; e < NH; e++) {
            float x = 0.0f;
#pragma unroll
            for (int w = 0; w < kWaves; w++) x = __builtin_fmaf(o_sh[w][wave][e][lane], f[w], x);
            res[half * NH + e] = x;
        }
    }
    if (it.tile * kTileRows + c >= n_rows) return;
    const int d = (4 * g4 + wave) * NE;  // this lane's dimensions: row 4 g4 + wave of every block e
    if (it.splits == 1) {
        const float by = row_factor(ll, ss > 0.0f);
        if (d < hd) {
            TQ* out = static_cast<TQ*>(a.out) + static_cast<int64_t>(r.begin + tok) * a.os + static_cast<int64_t>(head) * hd + d;
            TQ v[NE];
#pragma unroll
            for (int e = 0; e < NE; e++) v[e] = from_f32<TQ>(by == 0.0f ? 0.0f : res[e] * by);
            __builtin_memcpy(out, v, sizeof(v));
        }
        return;
    }
    const uint32_t block = it.block * static_cast<uint32_t>(a.p.n_kv) + kvh;
    if (block >= a.blocks) return;
    const int64_t at = static_cast<int64_t>(block) * kTileRows + c;
#pragma unroll
    for (int e = 0; e < NE; e += 4) *reinterpret_cast<float4v*>(a.part + at * DH + d + e) = float4v{res[e], res[e + 1], res[e + 2], res[e + 3]};
    if (g4 == 0 && wave == 0) *reinterpret_cast<float4v*>(a.ml + at * 4) = float4v{mm, ll, ss, 0.0f};
}

// Joins the splits of one tile: DH / 4 lanes to a row, four dimensions each.
template <typename TQ, int DH>
__global__ __launch_bounds__(256) void attn_paged_merge(PagedAttnArgs a) {
    const int kvh = static_cast<int>(blockIdx.x % static_cast<uint32_t>(a.p.n_kv));
    AttnItem it;
    if (!attn_find<true>(a.p, a.t, blockIdx.x / static_cast<uint32_t>(a.p.n_kv), &it)) return;
    if (it.splits == 1) return;
    const SeqRows r = paged_seq(a.p, it.s);
    const int32_t n_rows = r.n * a.t.group;
    constexpr int LPR = DH / 4, RPP = 256 / LPR;
    const int d = static_cast<int>(threadIdx.x) % LPR * 4;
    const uint32_t n_kv = static_cast<uint32_t>(a.p.n_kv), block0 = it.block * n_kv + kvh;
    if (static_cast<uint64_t>(it.block) * n_kv + static_cast<uint64_t>(it.splits) * n_kv > a.blocks) return;
    for (int i = static_cast<int>(threadIdx.x) / LPR; i < a.t.tile_rows; i += RPP) {
        const int32_t row = it.tile * a.t.tile_rows + i;
        if (row >= n_rows) return;
        const int64_t first = static_cast<int64_t>(block0) * a.t.tile_rows + i, step = static_cast<int64_t>(n_kv) * a.t.tile_rows;
        float m = -__builtin_inff(), ss = 0.0f, l = 0.0f;
        for (int k = 0; k < it.splits; k++) m = fmaxf(m, a.ml[(first + k * step) * 4]);
        const float ms = m == -__builtin_inff() ? 0.0f : m;
        float4v x = {};
        for (int k = 0; k < it.splits; k++) {
            const float4v s = *reinterpret_cast<const float4v*>(a.ml + (first + k * step) * 4);
            const float4v p = *reinterpret_cast<const float4v*>(a.part + (first + k * step) * DH + d);
            const float f = __builtin_amdgcn_exp2f(s[0] - ms);
            l = __builtin_fmaf(s[1], f, l);
            ss = fmaxf(ss, s[2]);
#pragma unroll
            for (int e = 0; e < 4; e++) x[e] = __builtin_fmaf(p[e], f, x[e]);
        }
        if (d >= a.p.hd) continue;
        const float by = row_factor(l, ss > 0.0f);
        const int32_t tok = row / a.t.group;
        const int head = kvh * a.t.group + (row - tok * a.t.group);
        TQ v[4];
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = from_f32<TQ>(by == 0.0f ? 0.0f : x[e] * by);
        __builtin_memcpy(static_cast<TQ*>(a.out) + static_cast<int64_t>(r.begin + tok) * a.os + static_cast<int64_t>(head) * a.p.hd + d, v, sizeof(v));
    }
}

// Workgroups and tiles of a launch, from its tiling.
struct Grid {
    int64_t blocks, tiles;
    size_t bytes;  // of partial results
};
Grid grid_of(const PagedAttnArgs& a, int dh) {
    Grid g;
    g.blocks = attn_blocks_bound(a.t, a.p.rows, a.p.n_seq, a.p.n_kv) * a.p.n_kv;
    g.tiles = attn_tiles_bound(a.t, a.p.rows, a.p.n_seq) * a.p.n_kv;
    g.bytes = static_cast<size_t>(g.blocks) * a.t.tile_rows * (dh + 4) * sizeof(float);
    return g;
}

template <typename TQ, int DH>
int launch_dims(neko_hip_ctx* ctx, const char* what, PagedAttnArgs a, int dtype) {
    // Sequences of up to kFewRows rows on the 16-row kernel, the rest on the tiles. Which a batch has is known on the
    // device alone, so both are launched, except where no sequence can be the other's: one sequence, or as many rows
    // as sequences (then any that has more than one is the 16-row kernel's too).
    const int64_t most = static_cast<int64_t>(a.p.rows) * a.t.group;
    const bool few = a.p.n_seq > 1 || most <= kFewRows;
    const bool many = most > kFewRows && a.p.rows > a.p.n_seq;
    PagedAttnArgs f = a, t = a;
    f.t.tile_rows = kTileRows;
    f.t.unit = kUnit;
    f.t.target = 4 * ctx->cu_count;
    f.t.min_rows = 1;
    f.t.max_rows = many ? kFewRows : 0x7fffffff;
    attn_paged_tile_form(ctx, t);
    t.t.min_rows = few ? kFewRows + 1 : 1;
    t.t.max_rows = 0x7fffffff;
    const Grid fg = few ? grid_of(f, DH) : Grid{}, tg = many ? grid_of(t, DH) : Grid{};
    NEKO_REQUIRE(ctx, fg.blocks <= 0x7fffffff && tg.blocks <= 0x7fffffff, "%s: grid too large", what);
    void* ws = nullptr;
    if (int rc = workspace(ctx, fg.bytes + tg.bytes, &ws)) return rc;
    const bool mods = a.softcap > 0.0f || a.slopes;
    auto place = [](PagedAttnArgs& x, const Grid& g, void* at) {
        x.blocks = static_cast<uint32_t>(g.blocks);
        x.part = static_cast<float*>(at);
        x.ml = x.part + g.blocks * x.t.tile_rows * DH;
    };
    auto merge = [&](const PagedAttnArgs& x, const Grid& g) {
        if (paged_reach(x.p) <= x.t.unit) return NEKO_OK;  // lengths within one unit are never split
        hipLaunchKernelGGL((attn_paged_merge<TQ, DH>), dim3(static_cast<uint32_t>(g.tiles)), dim3(256), 0, ctx->stream, x);
        return after_launch(ctx, what);
    };
    if (many) {
        place(t, tg, static_cast<char*>(ws) + fg.bytes);
        if (int rc = attn_paged_tile(ctx, what, t, dtype)) return rc;
        if (int rc = merge(t, tg)) return rc;
    }
    if (few) {
        place(f, fg, ws);
        if (mods) hipLaunchKernelGGL((attn_paged_kernel<TQ, DH, true>), dim3(f.blocks), dim3(256), 0, ctx->stream, f);
        else hipLaunchKernelGGL((attn_paged_kernel<TQ, DH, false>), dim3(f.blocks), dim3(256), 0, ctx->stream, f);
        if (int rc = after_launch(ctx, what)) return rc;
        if (int rc = merge(f, fg)) return rc;
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

extern "C" int neko_hip_attention_paged(neko_hip_ctx* ctx, const void* q, int64_t q_stride, int64_t rows,
                                        const neko_paged_kv* kv, const neko_paged_batch* batch, int n_head, float scale,
                                        float softcap, int64_t window, const float* slopes, void* out, int64_t out_stride,
                                        int dtype) {
    const char* what = "neko_hip_attention_paged";
    NEKO_ENTER(ctx);
    NEKO_REQUIRE(ctx, valid_dtype(dtype), "%s: bad dtype %d", what, dtype);
    NEKO_REQUIRE(ctx, rows >= 0, "%s: rows=%lld", what, (long long)rows);
    PagedAttnArgs a{};
    if (int rc = paged_args(ctx, what, kv, batch, rows, &a.p)) return rc;
    NEKO_REQUIRE(ctx, n_head > 0 && n_head % kv->n_kv == 0, "%s: n_head=%d must be a positive multiple of n_kv=%d", what, n_head,
                 kv->n_kv);
    NEKO_REQUIRE(ctx, std::isfinite(scale) && std::isfinite(softcap) && softcap >= 0.0f && window >= 0,
                 "%s: scale=%g softcap=%g window=%lld (finite, the latter two not negative)", what, scale, softcap, (long long)window);
    NEKO_REQUIRE(ctx, rows * n_head <= 0x3fffffff, "%s: too many rows x heads", what);
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
    a.q = q;
    a.qs = q_stride;
    a.out = out;
    a.os = out_stride;
    a.n_head = n_head;
    a.t.group = n_head / kv->n_kv;
    a.window = window < (1 << 30) ? static_cast<int32_t>(window) : 0;
    a.t.window = a.window;
    a.scale = scale;
    a.softcap = softcap;
    a.slopes = slopes;
    return dtype == NEKO_DT_F16 ? launch_typed<half_t>(ctx, what, a, dtype) : launch_typed<float>(ctx, what, a, dtype);
}
