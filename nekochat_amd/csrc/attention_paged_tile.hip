// Paged attention for many rows per sequence -- prompts and chunks of them -- on the matrix cores of gfx950.
//
// Formulas and scales as in attention_paged.hip. A workgroup's waves hold 32 flattened (token, head) rows each, the
// columns of v_mfma_f32_32x32x16_f16, and share tiles of keys in LDS, converted to f16 once on the way in: a code is
// converted once per 128 rows instead of once per wave, and the pipeline needs one barrier a tile (tile t + 1 is
// written while t is read, and t + 2 is on its way from the pages in registers). S^T = K Q^T leaves a lane with the
// scores of one row and, by the permutation that the contraction index is free to take, exactly the B operand of
// O^T = V^T P^T; V^T comes from LDS by transposing reads. Eight consecutive scores of a lane are of one 16-key block,
// hence of one page: its scales are the same for all lanes.
//
// What bounds it: issue. 8192 tokens of 32 / 8 heads of 128 in f16 take 605 us, 908 TFLOP/s, with the matrix units busy
// 43% and the vector units 61% of the cycles; two workgroups to a CU, so that one's vector work runs beside the
// other's products. Of drafted trees (16 of up to 64 rows over up to 8192 tokens, 74 us, 478 TFLOP/s) the start of a
// workgroup and its 66 KB of partial results too: some 20 tiles of keys each.
//
// Precision: f16 calls round each weight to f16 (2^-11 of it, the largest term of O being 1; as large as the rounding
// of the result) and sum the weights before that, in f32: those of a page of small values may carry the sum and be
// nothing in O. f32 calls split weights and q into two f16 each.
#include <algorithm>
#include <atomic>

#include "attention_paged.h"

namespace neko_hip {
namespace {

typedef short short4v __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(1))) uint8_t Global;

// LDS by its address: through a pointer every place that is not the array's start plus a constant costs an addition of it.
template <typename T>
__device__ __forceinline__ __attribute__((address_space(3))) T* lds_at(uint32_t at) {
    return (__attribute__((address_space(3))) T*)(uintptr_t)at;
}

// The slot of 16-byte chunk c of tile row `row` in LDS: the 16 rows of a ds_read_b128 pass at one chunk of K, and
// the 4 rows x 4 chunks of half a transposing read of V, fall on distinct banks.
template <int DH>
__device__ __forceinline__ int k_slot(int row, int c) {
    return DH >= 128 ? c ^ (row & 15) : c ^ ((row >> 1) & 7);
}
template <int DH>
__device__ __forceinline__ int v_slot(int row, int c) {
    return DH >= 128 ? c ^ ((row & 3) << 2) : c ^ ((row & 2) << 1);
}

template <typename TQ, int DH>
struct TileForm {
    static constexpr int waves = 4, rows = 32 * waves;
    // (fewer where registers are short: both planes of f32 q, 256 dimensions)
    static constexpr int keys = DH <= (sizeof(TQ) == 2 ? 128 : 64) ? 64 : 32;
    static constexpr int blocks = keys / kBlockKeys;  // pages' parts of a tile
    static constexpr int units = blocks / 2;          // blocks that a wave brings in, of K or V
    static constexpr int half_bytes = keys * DH * 2;
    static constexpr int tiles = 4 * half_bytes;       // two buffers of K and V
    static constexpr int lds = tiles + 2 * 4 * (waves + keys * (DH / 32));  // and what is noted of NaN values
    static constexpr int window = 64 / blocks;         // tiles of a page look-up
    static constexpr int rpi = 64 * 16 / DH;           // rows of a load instruction
    static constexpr int loads = kBlockKeys / rpi;     // load instructions of a unit
};

// The largest of three, NaN if one is (v_maximum3_f32; fmaxf first quiets operands that may be signalling NaNs, an
// instruction each). A row with a NaN score is NaN whatever its maximum.
__device__ __forceinline__ float max3(float a, float b, float c) {
    return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c);
}

// A block's exponents in one scalar.
__device__ __forceinline__ int pack_block(int ke, int ve) { return (ke + 128) | (ve + 128) << 8; }
__device__ __forceinline__ int block_ke(int x) { return (x & 255) - 128; }
__device__ __forceinline__ int block_ve(int x) { return ((x >> 8) & 255) - 128; }

// (f16 rows of 64 dimensions: three workgroups to a CU, at which four registers are spilled with a cap, of trees 20; 4 prompts of 2048
// tokens, 12 heads, 151 us, at two 175)
// TREE: rows of drafted trees (attention_paged.h).
template <typename TQ, int DH, bool MODS, bool TREE>
__global__ __launch_bounds__(256, DH <= 64 && sizeof(TQ) == 2 ? 3 : DH <= 128 ? 2 : 1) void attn_paged_tile_kernel(PagedAttnArgs a) {
    typedef TileForm<TQ, DH> C;
    constexpr bool kTwo = sizeof(TQ) == 4;
    constexpr int NS = DH / 16, ND = DH / 32, KB = C::keys / 32;
    extern __shared__ __align__(512) uint8_t tile_lds[];  // (places in a row are exclusive-ors of these address bits)
    const uint32_t lds0 = static_cast<uint32_t>((uintptr_t)(__attribute__((address_space(3))) uint8_t*)tile_lds);
    auto nan_sh = reinterpret_cast<uint32_t(*)[C::waves]>(tile_lds + C::tiles);  // whether a wave took NaN values out of the tile,
    auto nan_bits = reinterpret_cast<uint32_t(*)[C::keys][DH / 32]>(tile_lds + C::tiles + 2 * 4 * C::waves);  // and where
    const int lane = static_cast<int>(threadIdx.x) & 63;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
    const int l32 = lane & 31, h = lane >> 5;
    int kvh;
    const uint32_t item = item_of(a, &kvh);
    AttnItem it;
    if (!attn_find<false, TREE>(a.p, a.t, item, &it)) return;
    const SeqRows r = paged_seq(a.p, it.s);
    const TileKeys tk = TREE ? tree_tile_keys(a, r, it) : tile_keys(a, r, it);
    const int hd = a.p.hd;
    const int32_t reach = min(r.len, paged_reach(a.p));

    // This lane's row, and the keys that this wave's rows see (rows past the last repeat it).
    const int32_t n_rows = r.n * a.t.group, row0 = it.tile * C::rows + 32 * wave;
    const int32_t row = min(row0 + l32, n_rows - 1);
    const int32_t tok = static_cast<int32_t>(fast_div(static_cast<uint32_t>(row), a.by_group));
    const int head = kvh * a.t.group + (row - tok * a.t.group);
    const int32_t depth = TREE ? tree_depth(a, r, tok) : tok;
    const int32_t pos = r.len - r.n + depth;
    const int32_t hi = TREE ? tk.hi_min : min(pos + 1, reach), lo = key_lo(pos, a.t.window);
    const int32_t w_first = r.len - r.n + static_cast<int32_t>(fast_div(static_cast<uint32_t>(min(row0, n_rows - 1)), a.by_group));
    const int32_t w_last = r.len - r.n + static_cast<int32_t>(fast_div(static_cast<uint32_t>(min(row0 + 31, n_rows - 1)), a.by_group));
    const int32_t w_lo_min = TREE ? tk.lo_min : key_lo(w_first, a.t.window), w_lo_max = TREE ? tk.lo_max : key_lo(w_last, a.t.window);
    const int32_t w_hi_min = TREE ? tk.hi_min : min(w_first + 1, reach), w_hi_max = TREE ? tk.hi_max : min(w_last + 1, reach);

    // q: dimensions 16 s + 8 h .. + 7 of the row as the B operand of step s.
    half8 qh[NS], ql[kTwo ? NS : 1];
    float sc = a.scale == 0.0f ? 1.0f : fabsf(a.scale);
    {
        const TQ* qr = static_cast<const TQ*>(a.q) + static_cast<int64_t>(r.begin + tok) * a.qs + static_cast<int64_t>(head) * hd;
        const float sign = a.scale == 0.0f ? 0.0f : a.scale < 0.0f ? -1.0f : 1.0f;
        float x[NS][8];
#pragma unroll
        for (int s = 0; s < NS; s++) {
            const int d = 16 * s + 8 * h;
            TQ v[8];
            if (d < hd) __builtin_memcpy(v, qr + d, sizeof(v));
#pragma unroll
            for (int e = 0; e < 8; e++) x[s][e] = d < hd ? to_f32(v[e]) * sign : 0.0f;
        }
        if constexpr (kTwo) {
            float mx = 0.0f;
#pragma unroll
            for (int s = 0; s < NS; s++)
#pragma unroll
                for (int e = 0; e < 8; e++) mx = fmaxf(mx, fabsf(x[s][e]));
            mx = swap32_max(mx);
            const int ex = mx > 0.0f && mx < __builtin_inff() ? 15 - __builtin_amdgcn_frexp_expf(mx) : 0;
            const int e1 = ex / 2, e2 = ex - e1;
            sc = ldexpf(sc, -ex);
#pragma unroll
            for (int s = 0; s < NS; s++)
#pragma unroll
                for (int e = 0; e < 8; e++) x[s][e] = ldexpf(ldexpf(x[s][e], e1), e2);
        }
#pragma unroll
        for (int s = 0; s < NS; s++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                qh[s][e] = static_cast<half_t>(x[s][e]);
                if constexpr (kTwo) ql[s][e] = static_cast<half_t>(x[s][e] - to_f32(qh[s][e]));
            }
    }
    const float slope = MODS && a.slopes ? a.slopes[head] : 0.0f;
    const float inv_cap = MODS && a.softcap > 0.0f ? fminf(1.0f / a.softcap, 0x1.fffffep127f) : 0.0f;

    // Waves 0 and 1 bring in K, 2 and 3 V: half of a tile's blocks each.
    const bool is_v = wave >= C::waves / 2;
    const int block0 = (wave & 1) * C::units;

    // The next 64 blocks of 16 keys, one to a lane: where this wave's operand of it stands, and its exponents. Those
    // after them are asked for half a window ahead.
    const int nt = tk.k1 > tk.k0 ? (tk.k1 - tk.k0 + C::keys - 1) / C::keys : 0;
    uint32_t from_lo = 0, from_hi = 0;
    int32_t next_page = -1;
    int exps = pack_block(0, 0);
    uint64_t exps_ok = 0;  // which of them have a page
    float next_ks = 1.0f, next_vs = 1.0f;
    auto ask_pages = [&](int tile) __attribute__((always_inline)) {
        const int32_t at = tk.k0 + C::keys * tile + kBlockKeys * lane;
        next_page = -1;
        if (tile < nt && at < tk.k1) next_page = paged_page(a.p, it.s, at);
    };
    auto ask_scales = [&]() __attribute__((always_inline)) {
        const int64_t i = static_cast<int64_t>(next_page < 0 ? 0 : next_page) * a.p.n_kv + kvh;
        next_ks = a.p.ks[i];
        next_vs = a.p.vs[i];
    };
    auto take_pages = [&](int tile) __attribute__((always_inline)) {
        const uint8_t* head_base = (is_v ? a.p.v : a.p.k) + kvh * a.p.head_bytes;
        const int32_t slot = (tk.k0 + C::keys * tile + kBlockKeys * lane) & ((1 << a.p.page_log2) - 1);
        // (a block without a page reads page 0 and is masked; every slot of a page may be read)
        const uint64_t at = reinterpret_cast<uint64_t>(head_base) + static_cast<uint64_t>(static_cast<uint32_t>(next_page < 0 ? 0 : next_page)) * a.p.page_bytes +
                            static_cast<uint32_t>(slot * hd);
        from_lo = static_cast<uint32_t>(at);
        from_hi = static_cast<uint32_t>(at >> 32);
        exps = next_page < 0 ? pack_block(0, 0) : pack_block(scale_exp(next_ks), scale_exp(next_vs));
        exps_ok = __ballot(next_page >= 0);
    };
    // Of the blocks of the window that is being multiplied: score -> exponent of 2 (with a cap or a bias: -> natural
    // units; f32: without the row's own factor), the value scale's exponent and its inverse, and which have a page.
    float now_f = 0.0f, now_ve = 0.0f, now_inv = 0.0f;
    uint64_t now_ok = 0;
    auto use_window = [&]() __attribute__((always_inline)) {
        now_f = exp2i(block_ke(exps)) * (kTwo ? 1.0f : sc) * (MODS ? 1.0f : kAttnLog2e);
        if constexpr (!kTwo) now_f = fminf(fmaxf(now_f, 0x1p-120f), 0x1p120f);  // (never 0 or infinite: masked scores are -inf)
        now_ve = static_cast<float>(block_ve(exps));
        now_inv = exp2i(-block_ve(exps));
        now_ok = exps_ok;
    };
    // Tiles of which every row of the workgroup sees every key, as far as the keys have pages.
    const int inner0 = tk.lo_max > tk.k0 ? (tk.lo_max - tk.k0 + C::keys - 1) / C::keys : 0;
    const int inner1 = tk.hi_min > tk.k0 ? (tk.hi_min - tk.k0) / C::keys : 0;
    constexpr uint64_t kTileBits = (1ull << C::blocks) - 1;

    // Lane (row, 16-byte chunk) of a load instruction. Dimensions past the head's end: any of its own, against zeros in q.
    const int lr = lane / (DH / 16), lc = lane % (DH / 16);
    const uint32_t src = static_cast<uint32_t>(lr * hd + (lc * 16 < hd ? lc * 16 : 0));
    struct Raw {
        uint4v x[C::units][C::loads];
    };
    Raw raw;
    int raw_bad = 0;  // -1: not all its blocks have pages
    auto load = [&](int tile) __attribute__((always_inline)) {
        const int at = tile % C::window * C::blocks;
        uint32_t off = src;  // (opaque: a scalar base and this, not a sum of 64 bits that was widened outside the loop)
        asm volatile("" : "+v"(off));
        raw_bad = ((exps_ok >> at) & kTileBits) == kTileBits ? 0 : -1;
#pragma unroll
        for (int i = 0; i < C::units; i++) {
            const uint32_t lo32 = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(from_lo), at + block0 + i));
            const uint32_t hi32 = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(from_hi), at + block0 + i));
            // (in global memory: through a flat load the compiler would wait for these with the next read of LDS)
            const Global* from = reinterpret_cast<const Global*>(static_cast<uint64_t>(hi32) << 32 | lo32);
#pragma unroll
            for (int n = 0; n < C::loads; n++)
                raw.x[i][n] = *reinterpret_cast<const __attribute__((address_space(1))) uint4v*>(from + (n * C::rpi * hd + off));
        }
    };
    // Where this wave's codes go in LDS: piece (i, n, p) at (dst ^ 16 p ^ n dst_n) + rows, as the slots' exclusive-ors allow.
    uint32_t dst;
    {
        const int row = block0 * kBlockKeys + lr, c = 2 * lc;
        dst = lds0 + static_cast<uint32_t>((is_v ? C::half_bytes : 0) + row * DH * 2 + 16 * (is_v ? v_slot<DH>(row, c) : k_slot<DH>(row, c)));
    }
    const uint32_t dst_n = is_v || DH < 128 ? 0u : static_cast<uint32_t>(C::rpi) * 16u;
    // The tile in `raw`: a NaN value times a weight of zero is NaN, so in tiles of which some row does not see all, values
    // that no row sees become zeros (they may be codes of no token), and NaN values are taken out and noted.
    auto mend = [&](int tile, int buf) __attribute__((always_inline)) {
        const int32_t j0 = tk.k0 + C::keys * tile;
        const int at0 = tile % C::window * C::blocks + block0;
        {
            bool any = false;
            if (is_v) {
                uint32_t bad = 0;
#pragma unroll
                for (int i = 0; i < C::units; i++)
#pragma unroll
                    for (int n = 0; n < C::loads; n++) {
                        const int row = (block0 + i) * kBlockKeys + n * C::rpi + lr;
                        const bool held = ((exps_ok >> (at0 + i)) & 1) != 0 && j0 + row >= tk.lo_min && j0 + row < tk.hi_max;
                        uint32_t at = 0;  // a bit for each NaN code
#pragma unroll
                        for (int w = 0; w < 4; w++) {
                            const uint32_t y = held ? raw.x[i][n][w] : 0u, nan = nan_codes(y) >> 7;
                            raw.x[i][n][w] = y & ~(nan * 0xffu);
                            at |= ((nan * 0x01020408u) >> 24) << (4 * w);
                        }
                        reinterpret_cast<uint16_t*>(nan_bits[buf][row])[lc] = static_cast<uint16_t>(at);
                        bad |= at;
                    }
                any = __any(bad != 0);
            }
            if (lane == 0) nan_sh[buf][wave] = any;
        }
    };
    // Eight codes of each lane, converted, to LDS: piece k of kPieces.
    constexpr int kPieces = C::units * C::loads * 2;
    auto store_piece = [&](int k, int buf) __attribute__((always_inline)) {
        const int i = k / (2 * C::loads), n = k / 2 % C::loads, p = k % 2;
        half8 y;
#pragma unroll
        for (int w = 0; w < 2; w++) {
            const uint32_t x = raw.x[i][n][2 * p + w];
            const half2v y0 = f16_of_fp8<false>(x), y1 = f16_of_fp8<true>(x);
            y[4 * w] = y0[0];
            y[4 * w + 1] = y0[1];
            y[4 * w + 2] = y1[0];
            y[4 * w + 3] = y1[1];
        }
        *lds_at<half8>(buf * 2 * C::half_bytes + (i * kBlockKeys + n * C::rpi) * DH * 2 + (dst ^ (16u * p) ^ (static_cast<uint32_t>(n) * dst_n))) = y;
    };
    auto store = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < kPieces; k++) store_piece(k, buf);
    };

    float16v o[ND] = {};
    float m = -__builtin_inff(), l = 0.0f;
    int seen = 0;
    // Fragments: K, 8 dimensions of key 32 b + l32 for step d; V, by transposing reads, of eight keys for 32 dimensions.
    // The slots make their places k_at ^ 32 d and v_at ^ 64 d, one register each instead of one for every d.
    uint32_t k_lane = lds0 + static_cast<uint32_t>(l32 * DH * 2 + 16 * k_slot<DH>(l32, h)), v_lane;
    {
        const int tq = lane & 15, row = 4 * h + (tq >> 2);
        v_lane = lds0 + static_cast<uint32_t>(C::half_bytes + row * DH * 2 + 16 * v_slot<DH>(row, 2 * ((lane >> 4) & 1) + ((tq & 3) >> 1)) + 8 * (tq & 1));
    }
    auto k_frag = [&](uint32_t k_at, int b, int d) __attribute__((always_inline)) {
        return *lds_at<half8>(32 * b * DH * 2 + (k_at ^ (32u * d)));
    };
    auto v_frag = [&](uint32_t v_at, int d, int b, int i) __attribute__((always_inline)) {
        const uint32_t p0 = (32 * b + 16 * i) * DH * 2 + (v_at ^ (64u * d));
        const short4v a0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds_at<short4v>(p0));
        const short4v a1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds_at<short4v>(p0 + 8 * DH * 2));
        return __builtin_bit_cast(half8, __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    // `whole`: every row of the workgroup sees all of the tile's keys.
    auto step = [&](int tile, int buf, bool whole) __attribute__((always_inline)) {
        const int32_t j0 = tk.k0 + C::keys * tile;
        const int at = tile % C::window * C::blocks;
        if (!whole && (j0 >= w_hi_max || j0 + C::keys <= w_lo_min)) {  // nothing for this wave's rows
            store(buf ^ 1);
            return;
        }
        // (opaque, so that the places are made from these for each tile and not kept)
        uint32_t k_at = k_lane, v_at = v_lane;
        asm volatile("" : "+v"(k_at), "+v"(v_at));
        k_at += static_cast<uint32_t>(buf * 2 * C::half_bytes);
        v_at += static_cast<uint32_t>(buf * 2 * C::half_bytes);
        // Fragments are asked for eight products ahead (64 dimensions: four); left to itself the compiler puts each
        // read just before its use and waits for it there (a tile's 16 products took 1200 cycles, half of them waits).
        float16v s[KB];
        constexpr int kAhead = 8 < NS ? 8 : NS;
        half8 A[kAhead];
#pragma unroll
        for (int d = 0; d < kAhead; d++) A[d] = k_frag(k_at, 0, d);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int b = 0; b < KB; b++) {
            s[b] = float16v{};
#pragma unroll
            for (int d = 0; d < NS; d++) {
                const int u = b * NS + d, a = u % kAhead, next = u + kAhead;
                if constexpr (kTwo) s[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(A[a], ql[d], s[b], 0, 0, 0);
                s[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(A[a], qh[d], s[b], 0, 0, 0);
                if (next < KB * NS) A[a] = k_frag(k_at, next / NS, next % NS);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        // The first values, on their way while the weights are made.
        constexpr int kSteps = KB * ND, kVAhead = kSteps < 3 ? kSteps : 3;
        half8 V[kVAhead][2];
#pragma unroll
        for (int u = 0; u < kVAhead - 1; u++)
#pragma unroll
            for (int i = 0; i < 2; i++) V[u][i] = v_frag(v_at, u % ND, u / ND, i);
        __builtin_amdgcn_sched_barrier(0);
        auto lane_of = [&](float v, int b) __attribute__((always_inline)) {
            return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), at + b));
        };
        float f[C::blocks], ve[C::blocks];
#pragma unroll
        for (int b = 0; b < C::blocks; b++) {
            f[b] = lane_of(now_f, b);
            ve[b] = lane_of(now_ve, b);
            if constexpr (kTwo) f[b] = fminf(fmaxf(f[b] * sc, 0x1p-120f), 0x1p120f);
        }
        if constexpr (MODS) {
#pragma unroll
            for (int b = 0; b < KB; b++)
                unrolled<16>([&](auto ec) {
                    constexpr int e = decltype(ec)::value;
                    s[b][e] *= f[2 * b + e / 8];
                });
            if (a.softcap > 0.0f) {
#pragma unroll
                for (int b = 0; b < KB; b++)
                    unrolled<16>([&](auto ec) { s[b][decltype(ec)::value] = cap_score(s[b][decltype(ec)::value], a.softcap, inv_cap); });
            }
            if (a.slopes) {
                const int32_t away = j0 + 4 * h - pos;
                const bool in_tree = TREE && j0 + C::keys > tk.hi_min;
#pragma unroll
                for (int b = 0; b < KB; b++)
                    unrolled<16>([&](auto ec) {
                        constexpr int e = decltype(ec)::value;
                        int32_t by = away + 32 * b + 8 * (e >> 2) + (e & 3);
                        if (in_tree) by = tree_key_place(a, r, by + pos) - pos;
                        s[b][e] = __builtin_fmaf(slope, static_cast<float>(by), s[b][e]);
                    });
            }
#pragma unroll
            for (int b = 0; b < C::blocks; b++) f[b] = kAttnLog2e;
        }
        if (!whole && (j0 < w_lo_max || j0 + C::keys > w_hi_min || ((now_ok >> at) & kTileBits) != kTileBits)) {
            // Visible: lo <= j < hi, as one unsigned comparison of the distance from the first key seen; no key of a block
            // without a page.
            const uint32_t first = static_cast<uint32_t>(j0 + 4 * h - lo), many = hi > lo ? static_cast<uint32_t>(hi - lo) : 0u;
#pragma unroll
            for (int b = 0; b < KB; b++)
                unrolled<2>([&](auto ic) {
                    constexpr int i = decltype(ic)::value;
                    if constexpr (TREE) {
                        uint32_t sees = tree_sees(a, r, tok, depth, lo, hi, j0 + 32 * b) >> (16 * i) & 0xffffu;
                        sees = (now_ok >> (at + 2 * b + i)) & 1u ? sees : 0u;
                        seen |= static_cast<int>(sees != 0);
                        sees >>= 4 * h;
                        unrolled<8>([&](auto ec) {
                            constexpr int e = 8 * i + decltype(ec)::value;
                            s[b][e] = sees >> (8 * ((e >> 2) & 1) + (e & 3)) & 1u ? s[b][e] : -__builtin_inff();
                        });
                        return;
                    }
                    const uint32_t most = (now_ok >> (at + 2 * b + i)) & 1u ? many : 0u;
                    const int32_t from = j0 + 32 * b + 16 * i;
                    seen |= static_cast<int>(most != 0) & static_cast<int>(max(from, lo) < min(from + 16, hi));
                    unrolled<8>([&](auto ec) {
                        constexpr int e = 8 * i + decltype(ec)::value;
                        const bool vis = first + static_cast<uint32_t>(32 * b + 8 * (e >> 2) + (e & 3)) < most;
                        s[b][e] = vis ? s[b][e] : -__builtin_inff();
                    });
                    __builtin_amdgcn_sched_barrier(0);  // (else all comparisons first, their masks in scalar registers that the loop has use for)
                });
        } else {
            seen = 1;
        }
        float top = -__builtin_inff();
#pragma unroll
        for (int b = 0; b < KB; b++)
            unrolled<2>([&](auto ic) {
                constexpr int i = decltype(ic)::value;
                float mx = max3(s[b][8 * i], s[b][8 * i + 1], s[b][8 * i + 2]);
                mx = max3(mx, s[b][8 * i + 3], s[b][8 * i + 4]);
                mx = max3(mx, s[b][8 * i + 5], s[b][8 * i + 6]);
                mx = max3(mx, s[b][8 * i + 7], s[b][8 * i + 7]);
                top = fmaxf(top, __builtin_fmaf(mx, f[2 * b + i], ve[2 * b + i]));
            });
        top = ceilf(swap32_max(top));
        if (__any(top > m)) {
            const float mn = fmaxf(m, top);
            const float corr = __builtin_amdgcn_exp2f(m - (mn == -__builtin_inff() ? 0.0f : mn));
            m = mn;
            l *= corr;
#pragma unroll
            for (int d = 0; d < ND; d++)
                unrolled<16>([&](auto ec) { o[d][decltype(ec)::value] *= corr; });
        }
        const float ms = m == -__builtin_inff() ? 0.0f : m;
        half8 ph[KB][2], pl[KB][2];
        float sums[KB][2] = {}, base[C::blocks];
        // (f16: the offset joins the exponent; its rounding, 2^-21 of the weight, is nothing beside the weight's)
#pragma unroll
        for (int b = 0; b < C::blocks; b++) base[b] = ve[b] - (kTwo ? ms : ms - static_cast<float>(kPOffset));
        if (__any(fabsf(ms) >= kFarMax)) {  // exponents in place of scores
#pragma unroll
            for (int b = 0; b < KB; b++)
                unrolled<16>([&](auto ec) {
                    constexpr int e = decltype(ec)::value;
                    s[b][e] = exponent_of(s[b][e], f[2 * b + e / 8], ve[2 * b + e / 8], ms);
                });
#pragma unroll
            for (int b = 0; b < C::blocks; b++) {
                f[b] = 1.0f;
                base[b] = kTwo ? 0.0f : static_cast<float>(kPOffset);
            }
        }
        // Weights of elements e0 .. e0 + n - 1 of group b, their parts for the matrix cores and their sums.
        auto weights = [&](auto bc, auto e0c, auto nc) __attribute__((always_inline)) {
            constexpr int b = decltype(bc)::value;
            unrolled<decltype(nc)::value>([&](auto ec) {
                constexpr int e = decltype(e0c)::value + decltype(ec)::value, i = e / 8;
                if constexpr (kTwo) {
                    const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][e], f[2 * b + i], base[2 * b + i]));
                    const float y = p * kPScale;
                    ph[b][i][e % 8] = static_cast<half_t>(y);
                    pl[b][i][e % 8] = static_cast<half_t>(y - to_f32(ph[b][i][e % 8]));
                    sums[b][i] += p;
                } else {
                    const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][e], f[2 * b + i], base[2 * b + i]));
                    ph[b][i][e % 8] = static_cast<half_t>(p);
                    sums[b][i] += p;
                }
            });
        };
        // The matrix cores take the first group's weights while the second's are made, and the second's while the next
        // tile's codes are converted: with each of these by itself, 16 products and 110 vector operations of a tile ran
        // one after the other (678 us for a prompt of 8192 tokens).
        weights(std::integral_constant<int, 0>{}, std::integral_constant<int, 0>{}, std::integral_constant<int, 16>{});
        unrolled<kSteps>([&](auto uc) {
            constexpr int u = decltype(uc)::value, b = u / ND, d = u % ND, v = u % kVAhead, ahead = u + kVAhead - 1;
            if constexpr (ahead < kSteps) {
#pragma unroll
                for (int i = 0; i < 2; i++) V[ahead % kVAhead][i] = v_frag(v_at, ahead % ND, ahead / ND, i);
            }
#pragma unroll
            for (int i = 0; i < 2; i++) {
                if constexpr (kTwo) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(V[v][i], pl[b][i], o[d], 0, 0, 0);
                o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(V[v][i], ph[b][i], o[d], 0, 0, 0);
            }
            if constexpr (b + 1 < KB) {
                weights(std::integral_constant<int, b + 1>{}, std::integral_constant<int, 16 / ND * d>{}, std::integral_constant<int, 16 / ND>{});
            } else {
                constexpr int n = kPieces / ND;
                unrolled<n>([&](auto kc) { store_piece(n * d + decltype(kc)::value, buf ^ 1); });
            }
            // (the sums here, not after the branch below, where the matrix cores have nothing to do)
            if constexpr (d == ND - 1 && b + 1 == KB) {
#pragma unroll
                for (int x = 0; x < KB; x++) asm volatile("" : "+v"(sums[x][0]), "+v"(sums[x][1]));
            }
            __builtin_amdgcn_sched_barrier(0);
        });
#pragma unroll
        for (int b = 0; b < C::blocks; b++) l = __builtin_fmaf(sums[b / 2][b % 2], lane_of(now_inv, b), l);
        // NaN values taken out of the tile, put into the dimensions of the rows that see them.
        if (!whole) {
            uint32_t any = 0;
#pragma unroll
            for (int w = 0; w < C::waves; w++) any |= nan_sh[buf][w];
            if (__builtin_amdgcn_readfirstlane(any) != 0) {
#pragma unroll 1
                for (int k = 0; k < C::keys; k++) {
                    if (TREE ? (tree_sees(a, r, tok, depth, lo, hi, j0 + k) & 1u) == 0 : j0 + k < lo || j0 + k >= hi) continue;
#pragma unroll
                    for (int d = 0; d < ND; d++) {
                        const uint32_t bits = nan_bits[buf][k][d] >> (4 * h);
                        unrolled<16>([&](auto ec) {
                            constexpr int e = decltype(ec)::value;
                            o[d][e] = nan_if(o[d][e], bits, 8 * (e >> 2) + (e & 3));
                        });
                    }
                }
            }
        }
    };

    if (nt > 0) {
        // (as signs: conditions would be kept as lane masks) below 0: some row does not see all of the tile.
        auto outer = [&](int tile) __attribute__((always_inline)) { return (tile - inner0) | (inner1 - 1 - tile); };
        ask_pages(0);
        ask_scales();
        take_pages(0);
        ask_pages(C::window);
        load(0);
        int part = outer(0) | raw_bad;  // of the tile that is multiplied next
        if (part < 0) mend(0, 0);
        store(0);
        use_window();
        if (nt > 1) load(1);
        __syncthreads();
        for (int t = 0; t < nt; t++) {
            const int buf = t & 1;
            // Tile t + 1 is in `raw`: mended here, stored in the step (past the last, nothing of use). That buffer's
            // readers passed the barrier.
            const int next_part = outer(t + 1) | raw_bad;
            if (next_part < 0 && t + 1 < nt) mend(t + 1, buf ^ 1);
            step(t, buf, part >= 0);
            part = next_part;
            if ((t + 1) % C::window == 0) use_window();
            if (t + 2 < nt) {
                const int at = (t + 2) % C::window;
                if (at % (C::window / 2) == 0) {
                    if (at == 0) {
                        take_pages(t + 2);
                        ask_pages(t + 2 + C::window);
                    } else {
                        ask_scales();
                    }
                }
                load(t + 2);
            }
            __syncthreads();
        }
    }

    if (TREE && depth < 0) {  // (tiles that all others see whole are not masked for a row that sees nothing)
        m = -__builtin_inff();
        l = 0.0f;
        seen = 0;
    }
    l = swap32_sum(l);
    const bool any_seen = swap32_max(seen != 0 ? 1.0f : 0.0f) > 0.0f;
    if (row0 + l32 >= n_rows) return;
    const float l_by = kTwo ? 1.0f : 1.0f / kPScale;  // f16: the sum is of the weights times 2^kPOffset
    if (it.splits == 1) {
        const float by = row_factor(l * l_by, any_seen);
        TQ* out = static_cast<TQ*>(a.out) + static_cast<int64_t>(r.begin + tok) * a.os + static_cast<int64_t>(head) * hd;
#pragma unroll
        for (int d = 0; d < ND; d++)
            unrolled<4>([&](auto gc) {
                constexpr int g = decltype(gc)::value;
                const int at = 32 * d + 8 * g + 4 * h;
                TQ v[4];
                unrolled<4>([&](auto ec) {
                    constexpr int e = decltype(ec)::value;
                    v[e] = from_f32<TQ>(by == 0.0f ? 0.0f : o[d][4 * g + e] * by);
                });
                if (at < hd) __builtin_memcpy(out + at, v, sizeof(v));
            });
        return;
    }
    const uint32_t block = it.block * static_cast<uint32_t>(a.p.n_kv) + kvh;
    if (block >= a.blocks) return;
    const int64_t at = static_cast<int64_t>(block) * C::rows + 32 * wave + l32;
#pragma unroll
    for (int d = 0; d < ND; d++)
        unrolled<4>([&](auto gc) {
            constexpr int g = decltype(gc)::value;
            *reinterpret_cast<float4v*>(a.part + at * DH + 32 * d + 8 * g + 4 * h) =
                float4v{o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]};
        });
    if (h == 0) *reinterpret_cast<float4v*>(a.ml + at * 4) = float4v{m, l * l_by, any_seen ? 1.0f : 0.0f, 0.0f};
}

template <typename TQ, int DH, bool MODS, bool TREE>
int launch_tiles(neko_hip_ctx* ctx, const char* what, const PagedAttnArgs& a) {
    typedef TileForm<TQ, DH> C;
    static std::atomic<uint64_t> allowed{0};
    const void* kernel = reinterpret_cast<const void*>(&attn_paged_tile_kernel<TQ, DH, MODS, TREE>);
    if (C::lds > 64 * 1024)
        if (int rc = allow_lds(ctx, kernel, C::lds, allowed)) return rc;
    hipLaunchKernelGGL((attn_paged_tile_kernel<TQ, DH, MODS, TREE>), dim3(a.blocks), dim3(64 * C::waves), C::lds, ctx->stream, a);
    return after_launch(ctx, what);
}

template <typename TQ, bool MODS, bool TREE>
int launch_dims(neko_hip_ctx* ctx, const char* what, const PagedAttnArgs& a) {
    if (a.p.hd <= 64) return launch_tiles<TQ, 64, MODS, TREE>(ctx, what, a);
    if (a.p.hd <= 128) return launch_tiles<TQ, 128, MODS, TREE>(ctx, what, a);
    return launch_tiles<TQ, 256, MODS, TREE>(ctx, what, a);
}

}  // namespace

void attn_paged_tile_form(const neko_hip_ctx* ctx, PagedAttnArgs& a) {
    a.t.tile_log2 = 7;  // TileForm::rows
    a.t.unit_log2 = 6;  // a whole number of tiles of either size
    a.t.target = 2 * ctx->cu_count;
    a.t.least = 1;
    attn_form(a);
}

int attn_paged_tile(neko_hip_ctx* ctx, const char* what, const PagedAttnArgs& a, int dtype) {
    const bool mods = a.softcap > 0.0f || a.slopes;
    auto by_form = [&](auto tree) {
        constexpr bool TREE = decltype(tree)::value;
        if (dtype == NEKO_DT_F16) return mods ? launch_dims<half_t, true, TREE>(ctx, what, a) : launch_dims<half_t, false, TREE>(ctx, what, a);
        return mods ? launch_dims<float, true, TREE>(ctx, what, a) : launch_dims<float, false, TREE>(ctx, what, a);
    };
    return a.words > 0 ? by_form(std::true_type{}) : by_form(std::false_type{});
}

}  // namespace neko_hip
