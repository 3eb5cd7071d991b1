// Appending to a paged 8-bit KV cache for gfx950: the q / k heads of each new row normed (optionally) and rotated
// -- q to its own rows, k and v as E4M3 codes into the pages of the row's sequence, under one power-of-two scale for
// each page and kv head.
//
// Formulas. x' = x / sqrt(mean(x^2) + eps) * w per head (the sum in double, the scale rounded to float); rotation of
// the pairs (x_i, x_{i + rot/2}) or (x_2i, x_2i+1) by the position's angles; k' rounded to the activations' type. Page
// scale 2^e, e the smallest with amax <= 448 * 2^e over the page's tokens of that head; code = e4m3(x * 2^-e), nearest
// even. A page that already holds tokens keeps its scale or raises it; raising it re-rounds the earlier codes, which
// moves only those that leave E4M3's normal range (a power of two just lowers the exponent), so a sequence appended
// token by token and one appended at once differ at most there. A scale that were amax / 448 itself would re-round
// every code of the page each time its largest value grows.
//
// A wave takes 16 tokens of one page, one kv head and one of k and v, all in registers between the maximum and the
// codes: one pass over the data. Larger pages take several waves, whose maxima meet in LDS. The q heads are waves of
// the same launch, four rows (128 dimensions) by four heads each, so the angles are loaded once per row. Lanes: head
// size / 8 lanes to a row, each with two quads that rotate into each other, so the rotation needs no exchange. What
// bounds it: memory, 8192 rows of 32 / 8 heads of 128 in f16 in 45.2 us, 4.1 TB/s; a few rows the launch and three loads
// that need each other (64 decoded tokens 5.5 us).
#include <algorithm>

#include "internal.h"
#include "paged_device.h"

namespace neko_hip {
namespace {

// q heads of a wave: their values in flight set the kernel's registers (8: 98 and five waves per SIMD, a prefill of
// 8192 rows 51.9 us and 64 decoded tokens 7.1; 4: 45.2 and 5.5; 2: 50.1 and 5.9).
constexpr int kHeadsPerWave = 4;
constexpr int kWaveTokens = 16;   // tokens of a page that one wave holds

struct AppendArgs {
    Paged p;
    const void* qkv;
    int64_t stride;
    void* q_out;
    int64_t q_stride;
    const float* wqk;
    const float* cs;
    int32_t n_pos;  // positions from there on are left alone
    int32_t rot;
    int32_t inter;
    int32_t n_q;
    float eps;
    uint32_t kv_ratio;     // 2^32 times the share of workgroups that are the pages', rounded up
    uint32_t kv_parts;     // (segment, k or v, kv head) parts of those
    uint32_t by_row;       // segments are looked for at each row instead of in the slots
    uint32_t q_groups;     // waves along the heads of the q part
    uint32_t q_waves;
};

// Where a lane's two quads stand in a head, and whether they rotate.
struct Quads {
    int a, b;
    bool turns;
};
__device__ __forceinline__ Quads quads_of(int sub, int rot, bool inter) {
    const int turning = rot / 8;
    Quads q;
    q.turns = sub < turning;
    if (inter || !q.turns) {  // (past the rotated part, 8 * sub = rot + 8 * (sub - turning))
        q.a = 8 * sub;
        q.b = q.a + 4;
    } else {
        q.a = 4 * sub;
        q.b = rot / 2 + 4 * sub;
    }
    return q;
}

template <typename T>
__device__ __forceinline__ void load_quad(const T* p, float* x) {
    T v[4];
    __builtin_memcpy(v, p, sizeof(v));  // (rows of any alignment)
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = to_f32(v[i]);
}
template <typename T>
__device__ __forceinline__ void store_quad(T* p, const float* x) {
    T v[4];
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = from_f32<T>(x[i]);
    // Past the caches: a prefill's q is larger than they are (8192 rows 54.3 -> 52.2 us).
    typedef T Q __attribute__((ext_vector_type(4), aligned(sizeof(T))));
    __builtin_nontemporal_store(Q{v[0], v[1], v[2], v[3]}, reinterpret_cast<Q*>(p));
}

// The head's norm over its LPR lanes; lanes past the head's end hold zeros.
template <int LPR>
__device__ __forceinline__ void norm_head(float* x, const float* w, int hd, float eps) {
    double ss = 0.0;
#pragma unroll
    for (int i = 0; i < 8; i++) ss = __builtin_fma(static_cast<double>(x[i]), static_cast<double>(x[i]), ss);
    ss = group_sum_f64<LPR>(ss);
    const float r = rsqrt_to_float(ss * (1.0 / hd) + static_cast<double>(eps));
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = x[i] * r * w[i];
}

// cs: (cos, sin) of the lane's four pairs.
__device__ __forceinline__ void rotate(float* x, const float* cs, bool inter) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int ia = inter ? 2 * i : i, ib = inter ? 2 * i + 1 : i + 4;
        const float a = x[ia], b = x[ib], c = cs[2 * i], s = cs[2 * i + 1];
        x[ia] = a * c - b * s;
        x[ib] = a * s + b * c;
    }
}

// Tokens [a, b) of one page, kv head `g`, of k or v: wave `w` of NW holds slots 16 w .. 16 w + 15.
template <typename T, int LPR, int NW>
__device__ __forceinline__ void append_page(const AppendArgs& a, const Segment& seg, int g, bool is_k, int w, uint32_t* sh) {
    constexpr int RPL = 64 / LPR;                                           // rows of a load
    constexpr int IT = RPL >= kWaveTokens ? 1 : kWaveTokens / RPL;          // loads
    const int lane = static_cast<int>(threadIdx.x) & 63;
    const int sub = lane % LPR, hd = a.p.hd;
    const bool in_head = 8 * sub < hd;
    const bool inter = a.inter != 0;
    const Quads d = quads_of(sub, is_k ? a.rot : 0, inter);
    const T* base = static_cast<const T*>(a.qkv) + static_cast<int64_t>(a.n_q + (is_k ? 0 : a.p.n_kv) + g) * hd;
    float wt[8];
    const bool norm = is_k && a.wqk != nullptr;
    if (norm && in_head) {
        __builtin_memcpy(wt, a.wqk + hd + d.a, 16);
        __builtin_memcpy(wt + 4, a.wqk + hd + d.b, 16);
    }
    float x[IT][8];
    bool mine[IT];
#pragma unroll
    for (int it = 0; it < IT; it++) {
        const int in_wave = it * RPL + lane / LPR;
        const int slot = w * kWaveTokens + in_wave;
        mine[it] = in_head && in_wave < kWaveTokens && slot >= seg.a && slot < seg.b;
#pragma unroll
        for (int i = 0; i < 8; i++) x[it][i] = 0.0f;
        if (mine[it]) {
            const T* row = base + static_cast<int64_t>(seg.row0 + slot) * a.stride;
            load_quad(row + d.a, x[it]);
            load_quad(row + d.b, x[it] + 4);
        }
    }
    uint32_t top = 0;
#pragma unroll
    for (int it = 0; it < IT; it++) {
        if (is_k) {
            if (norm) norm_head<LPR>(x[it], wt, hd, a.eps);
            if (d.turns && mine[it]) {
                float cs[8];
                const int slot = w * kWaveTokens + it * RPL + lane / LPR;
                __builtin_memcpy(cs, a.cs + static_cast<int64_t>(seg.pos0 + slot) * a.rot + 8 * sub, 32);
                rotate(x[it], cs, inter);
            }
            if constexpr (sizeof(T) == 2) {  // as a row of this type would hold it
#pragma unroll
                for (int i = 0; i < 8; i++) x[it][i] = to_f32(f16_rne(x[it][i]));
            }
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint32_t m = __builtin_bit_cast(uint32_t, x[it][i]) & 0x7fffffffu;
            if (mine[it] && m < 0x7f800000u) top = top > m ? top : m;  // the page's scale is that of its finite values
        }
    }
    top = wave_max_u32(top);
    float* scale = (is_k ? a.p.ks : a.p.vs) + static_cast<int64_t>(seg.page) * a.p.n_kv + g;
    const int had = seg.a > 0 ? scale_exp(*scale) : -kScaleMax;
    if constexpr (NW > 1) {
        if (lane == 0) sh[w] = top;
        __syncthreads();  // also between every wave's read of the scale and its store below
#pragma unroll
        for (int i = 0; i < NW; i++) top = top > sh[i] ? top : sh[i];
    }
    const int need = need_exp(top);
    const int e = need > had ? need : had;
    uint8_t* page = (is_k ? a.p.k : a.p.v) + static_cast<uint64_t>(seg.page) * a.p.page_bytes + g * a.p.head_bytes;
    if (seg.a > 0 && e > had) {  // the tokens that were there, under the new scale
        const float down = exp2i(had - e < -126 ? -126 : had - e);
#pragma unroll 1
        for (int it = 0; it < IT; it++) {
            const int in_wave = it * RPL + lane / LPR;
            const int slot = w * kWaveTokens + in_wave;
            if (in_head && in_wave < kWaveTokens && slot < seg.a) {
                uint2v* at = reinterpret_cast<uint2v*>(page + slot * hd + 8 * sub);
                uint2v c = *at;
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const half2v lo = f16_of_fp8<false>(c[h]), hi = f16_of_fp8<true>(c[h]);
                    const float y[4] = {to_f32(lo[0]), to_f32(lo[1]), to_f32(hi[0]), to_f32(hi[1])};
                    const uint32_t r = fp8_of_f32(y, down);
                    c[h] = r;
                }
                *at = c;
            }
        }
    }
    const float by = exp2i(-e);
#pragma unroll
    for (int it = 0; it < IT; it++) {
        if (mine[it]) {
            const int slot = w * kWaveTokens + it * RPL + lane / LPR;
            *reinterpret_cast<uint32_t*>(page + slot * hd + d.a) = fp8_of_f32(x[it], by);
            *reinterpret_cast<uint32_t*>(page + slot * hd + d.b) = fp8_of_f32(x[it] + 4, by);
        }
    }
    if (w == 0 && lane == 0) *scale = exp2i(e);
}

// The q heads [h0, h0 + kHeadsPerWave) of rows r0 .. r0 + 64 / LPR - 1.
template <typename T, int LPR>
__device__ __forceinline__ void append_q(const AppendArgs& a, uint32_t wave) {
    constexpr int RPL = 64 / LPR;
    const int lane = static_cast<int>(threadIdx.x) & 63;
    const int sub = lane % LPR, hd = a.p.hd;
    const uint32_t tile = wave / a.q_groups;  // (the groups of a row's heads by waves that run together)
    const int32_t r0 = static_cast<int32_t>(tile) * RPL;
    const int h0 = static_cast<int>(wave - tile * a.q_groups) * kHeadsPerWave;
    const int32_t row = r0 + lane / LPR;
    const bool in_head = 8 * sub < hd;
    const bool inter = a.inter != 0;
    const Quads d = quads_of(sub, a.rot, inter);
    const bool inside = in_head && row < a.p.rows;
    const T* in = static_cast<const T*>(a.qkv) + static_cast<int64_t>(inside ? row : 0) * a.stride;
    float x[kHeadsPerWave][8];
#pragma unroll
    for (int h = 0; h < kHeadsPerWave; h++) {
#pragma unroll
        for (int i = 0; i < 8; i++) x[h][i] = 0.0f;
        if (inside && h0 + h < a.n_q) {
            load_quad(in + (h0 + h) * hd + d.a, x[h]);
            load_quad(in + (h0 + h) * hd + d.b, x[h] + 4);
        }
    }
    // The sequence of each row: that of the wave's first, then past the sequences that end before it.
    const int32_t s = paged_seq_from(a.p, wave_last(a.p.n_seq, r0, [&](int32_t i) { return clamp_i32(a.p.row_start[i], 0, a.p.rows); }), row);
    const SeqRows r = paged_seq(a.p, s);
    const int32_t pos = r.len - r.n + (row - r.begin);
    const bool mine = inside && row >= r.begin && row < r.begin + r.n && pos >= 0 && pos < a.n_pos;
    float cs[8], wt[8];
    if (mine && d.turns) __builtin_memcpy(cs, a.cs + static_cast<int64_t>(pos) * a.rot + 8 * sub, 32);
    if (a.wqk != nullptr && in_head) {
        __builtin_memcpy(wt, a.wqk + d.a, 16);
        __builtin_memcpy(wt + 4, a.wqk + d.b, 16);
    }
    T* out = static_cast<T*>(a.q_out) + static_cast<int64_t>(inside ? row : 0) * a.q_stride;
#pragma unroll
    for (int h = 0; h < kHeadsPerWave; h++) {
        if (a.wqk != nullptr) norm_head<LPR>(x[h], wt, hd, a.eps);
        if (mine && h0 + h < a.n_q) {
            if (d.turns) rotate(x[h], cs, inter);
            store_quad(out + (h0 + h) * hd + d.a, x[h]);
            store_quad(out + (h0 + h) * hd + d.b, x[h] + 4);
        }
    }
}

// NW waves to a page's part; a workgroup has four such parts where they are one wave each.
template <int NW>
constexpr int kParts = NW == 1 ? 4 : 1;

template <typename T, int LPR, int NW>
__global__ __launch_bounds__(64 * NW * kParts<NW>) void append_kernel(AppendArgs a) {
    __shared__ uint32_t sh[NW];
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6), w = wave % NW;
    // Workgroups of the pages and of q in turn, in the ratio of their numbers (umulhi(b, ratio) of the first b are the
    // pages'): one after the other they took 20 and 36 us of a prefill of 8192 rows, one short of memory requests, the
    // other short of nothing else.
    const uint32_t kv_block = __umulhi(blockIdx.x, a.kv_ratio);
    if (__umulhi(blockIdx.x + 1, a.kv_ratio) == kv_block) {
        const uint32_t q_wave = (blockIdx.x - kv_block) * (NW * kParts<NW>) + wave;
        if (q_wave < a.q_waves) append_q<T, LPR>(a, q_wave);
        return;
    }
    // Kv heads fastest, so that with eight of them an XCD writes the pages' parts that its attention reads.
    const uint32_t units = 2u * a.p.n_kv;
    const uint32_t part = kv_block * kParts<NW> + wave / NW;
    if (part >= a.kv_parts) return;
    const int32_t at = static_cast<int32_t>(part / units);
    const int g = static_cast<int>(part % units) % a.p.n_kv;
    const bool is_k = static_cast<int>(part % units) < a.p.n_kv;
    int32_t s, i;
    if (a.by_row) {
        // A segment begins at a sequence's first row and at the first row of each page.
        s = wave_last(a.p.n_seq, at, [&](int32_t j) { return clamp_i32(a.p.row_start[j], 0, a.p.rows); });
        const SeqRows r = paged_seq(a.p, s);
        const int32_t first = r.len - r.n, begin = first < 0 ? 0 : first, pos = first + (at - r.begin);
        if (at < r.begin || at >= r.begin + r.n || pos < begin) return;
        if (pos != begin && (pos & ((1 << a.p.page_log2) - 1)) != 0) return;
        i = (pos >> a.p.page_log2) - (begin >> a.p.page_log2);
    } else {
        s = wave_last(a.p.n_seq, at, [&](int32_t j) { return segment_slot(a.p, j); });
        i = at - segment_slot(a.p, s);
    }
    const Segment seg = paged_segment(a.p, s, i, a.n_pos);
    if (seg.page < 0) return;
    append_page<T, LPR, NW>(a, seg, g, is_k, w, sh);
}

template <typename T, int LPR>
void launch_pages(neko_hip_ctx* ctx, const AppendArgs& a, uint32_t grid) {
    switch (a.p.page_log2) {
        case 4: hipLaunchKernelGGL((append_kernel<T, LPR, 1>), dim3(grid), dim3(64 * kParts<1>), 0, ctx->stream, a); break;
        case 5: hipLaunchKernelGGL((append_kernel<T, LPR, 2>), dim3(grid), dim3(128), 0, ctx->stream, a); break;
        case 6: hipLaunchKernelGGL((append_kernel<T, LPR, 4>), dim3(grid), dim3(256), 0, ctx->stream, a); break;
        case 7: hipLaunchKernelGGL((append_kernel<T, LPR, 8>), dim3(grid), dim3(512), 0, ctx->stream, a); break;
        default: hipLaunchKernelGGL((append_kernel<T, LPR, 16>), dim3(grid), dim3(1024), 0, ctx->stream, a); break;
    }
}

int launch_append(neko_hip_ctx* ctx, const char* what, AppendArgs a, int dtype) {
    const int lpr = a.p.hd <= 16 ? 2 : a.p.hd <= 32 ? 4 : a.p.hd <= 64 ? 8 : a.p.hd <= 128 ? 16 : 32;
    const int nw = 1 << (a.p.page_log2 - 4);
    // The slots of the segments, or the rows where those are fewer (a decode step).
    const int64_t slots = segment_slots(a.p.rows, a.p.n_seq, a.p.page_log2);
    a.by_row = a.p.rows <= slots;
    const int64_t parts = std::min<int64_t>(slots, a.p.rows) * 2 * a.p.n_kv;
    const int per_block = nw == 1 ? kParts<1> : 1;
    const int64_t kv = (parts + per_block - 1) / per_block;
    const int64_t tiles = (static_cast<int64_t>(a.p.rows) * lpr + 63) / 64;
    const int64_t waves = tiles * ((a.n_q + kHeadsPerWave - 1) / kHeadsPerWave);
    const int64_t grid = kv + (waves + nw * per_block - 1) / (nw * per_block);
    NEKO_REQUIRE(ctx, grid <= 0x7fffffff && parts <= 0x7fffffff, "%s: grid too large", what);
    a.kv_parts = static_cast<uint32_t>(parts);
    a.kv_ratio = static_cast<uint32_t>((static_cast<uint64_t>(kv) << 32) / static_cast<uint64_t>(grid) + 1);
    a.q_groups = static_cast<uint32_t>((a.n_q + kHeadsPerWave - 1) / kHeadsPerWave);
    a.q_waves = static_cast<uint32_t>(waves);
    const uint32_t n = static_cast<uint32_t>(grid);
    auto pick = [&](auto t) {
        typedef decltype(t) T;
        switch (lpr) {
            case 2: launch_pages<T, 2>(ctx, a, n); break;
            case 4: launch_pages<T, 4>(ctx, a, n); break;
            case 8: launch_pages<T, 8>(ctx, a, n); break;
            case 16: launch_pages<T, 16>(ctx, a, n); break;
            default: launch_pages<T, 32>(ctx, a, n); break;
        }
    };
    if (dtype == NEKO_DT_F16) pick(half_t{});
    else pick(float{});
    return after_launch(ctx, what);
}

}  // namespace

int paged_args(neko_hip_ctx* ctx, const char* what, const neko_paged_kv* kv, const neko_paged_batch* batch, int64_t rows,
               Paged* p) {
    NEKO_REQUIRE(ctx, kv && batch, "%s: null cache or batch", what);
    NEKO_REQUIRE(ctx, kv->k_pages && kv->v_pages && kv->k_scales && kv->v_scales, "%s: null cache pointer", what);
    NEKO_REQUIRE(ctx, kv->hd >= 16 && kv->hd <= 256 && kv->hd % 16 == 0, "%s: head size %d (a multiple of 16, 16..256)", what,
                 kv->hd);
    NEKO_REQUIRE(ctx, kv->page_size >= 16 && kv->page_size <= 256 && (kv->page_size & (kv->page_size - 1)) == 0,
                 "%s: page size %d (a power of two, 16..256)", what, kv->page_size);
    NEKO_REQUIRE(ctx, kv->n_kv > 0 && kv->n_kv <= 4095, "%s: n_kv=%d (1..4095)", what, kv->n_kv);
    NEKO_REQUIRE(ctx, kv->n_pages > 0 && kv->n_pages <= 0x7fffffff, "%s: n_pages=%lld", what, (long long)kv->n_pages);
    NEKO_REQUIRE(ctx, aligned(kv->k_pages, 16) && aligned(kv->v_pages, 16) && aligned(kv->k_scales, 4) && aligned(kv->v_scales, 4),
                 "%s: pages must be 16-byte aligned, scales 4-byte", what);
    NEKO_REQUIRE(ctx, batch->n_seq > 0 && batch->n_seq <= (1 << 24), "%s: n_seq=%lld (1..2^24)", what, (long long)batch->n_seq);
    NEKO_REQUIRE(ctx, batch->page_table && batch->row_start && batch->kv_len, "%s: null batch pointer", what);
    NEKO_REQUIRE(ctx, batch->max_pages > 0 && batch->max_pages <= 0x7fffffff && batch->table_stride >= batch->max_pages &&
                 batch->table_stride <= (int64_t(1) << 32),
                 "%s: page table of %lld columns, row stride %lld", what, (long long)batch->max_pages, (long long)batch->table_stride);
    NEKO_REQUIRE(ctx, rows <= 0x3fffffff, "%s: rows=%lld too many", what, (long long)rows);
    const size_t codes = paged_code_bytes(*kv), scales = paged_scale_bytes(*kv);
    NEKO_REQUIRE(ctx, !overlaps(kv->k_pages, codes, kv->v_pages, codes) && !overlaps(kv->k_scales, scales, kv->v_scales, scales) &&
                 !overlaps(kv->k_pages, codes, kv->k_scales, scales) && !overlaps(kv->k_pages, codes, kv->v_scales, scales) &&
                 !overlaps(kv->v_pages, codes, kv->k_scales, scales) && !overlaps(kv->v_pages, codes, kv->v_scales, scales),
                 "%s: the cache's arrays may not overlap", what);
    p->k = static_cast<uint8_t*>(kv->k_pages);
    p->v = static_cast<uint8_t*>(kv->v_pages);
    p->ks = kv->k_scales;
    p->vs = kv->v_scales;
    p->table = batch->page_table;
    p->row_start = batch->row_start;
    p->kv_len = batch->kv_len;
    p->table_stride = batch->table_stride;
    p->n_pages = kv->n_pages;
    p->max_pages = static_cast<int32_t>(batch->max_pages);
    p->n_seq = static_cast<int32_t>(batch->n_seq);
    p->rows = static_cast<int32_t>(rows);
    p->page_log2 = __builtin_ctz(static_cast<unsigned>(kv->page_size));
    p->n_kv = kv->n_kv;
    p->hd = kv->hd;
    p->head_bytes = static_cast<uint32_t>(kv->page_size * kv->hd);
    p->page_bytes = p->head_bytes * static_cast<uint32_t>(kv->n_kv);
    return NEKO_OK;
}

bool paged_overlaps(const neko_paged_kv& kv, const void* p, size_t bytes) {
    const size_t codes = paged_code_bytes(kv), scales = paged_scale_bytes(kv);
    return overlaps(p, bytes, kv.k_pages, codes) || overlaps(p, bytes, kv.v_pages, codes) ||
           overlaps(p, bytes, kv.k_scales, scales) || overlaps(p, bytes, kv.v_scales, scales);
}

}  // namespace neko_hip

using namespace neko_hip;

extern "C" int neko_hip_qk_norm_rope_paged(neko_hip_ctx* ctx, const void* qkv, int64_t row_stride, int64_t rows, int n_q,
                                           const neko_paged_kv* kv, const neko_paged_batch* batch, const float* wqk,
                                           const float* cs, int64_t n_pos, int rot_dim, int interleaved, float eps,
                                           void* q_out, int64_t q_out_stride, int dtype) {
    const char* what = "neko_hip_qk_norm_rope_paged";
    NEKO_ENTER(ctx);
    NEKO_REQUIRE(ctx, valid_dtype(dtype), "%s: bad dtype %d", what, dtype);
    NEKO_REQUIRE(ctx, rows >= 0 && n_q > 0 && n_q <= 65536, "%s: bad shape rows=%lld n_q=%d", what, (long long)rows, n_q);
    AppendArgs a{};
    if (int rc = paged_args(ctx, what, kv, batch, rows, &a.p)) return rc;
    NEKO_REQUIRE(ctx, rot_dim >= 0 && rot_dim <= kv->hd && rot_dim % 8 == 0, "%s: rot_dim=%d (a multiple of 8, up to the head size %d)",
                 what, rot_dim, kv->hd);
    NEKO_REQUIRE(ctx, rot_dim == 0 || (cs && n_pos >= 0), "%s: a rotation needs a cos/sin table", what);
    if (rows == 0 || (rot_dim > 0 && n_pos == 0)) return NEKO_OK;
    NEKO_REQUIRE(ctx, qkv && q_out, "%s: null pointer", what);
    const int64_t q_width = static_cast<int64_t>(n_q) * kv->hd, width = q_width + 2LL * kv->n_kv * kv->hd;
    NEKO_REQUIRE(ctx, row_stride >= width && q_out_stride >= q_width, "%s: row strides (%lld, %lld) below the rows' widths (%lld, %lld)",
                 what, (long long)row_stride, (long long)q_out_stride, (long long)width, (long long)q_width);
    const size_t esz = dtype_size(dtype);
    NEKO_REQUIRE(ctx, aligned(qkv, esz) && aligned(q_out, esz), "%s: misaligned rows", what);
    const size_t s_in = rows_span(rows, width, row_stride, esz), s_out = rows_span(rows, q_width, q_out_stride, esz);
    NEKO_REQUIRE(ctx, s_in != 0 && s_out != 0, "%s: rows span more than 2^62 bytes", what);
    NEKO_REQUIRE(ctx, (q_out == qkv && (rows == 1 || q_out_stride == row_stride)) || !overlaps(q_out, s_out, qkv, s_in),
                 "%s: q_out is the q columns of qkv itself or disjoint from qkv", what);
    NEKO_REQUIRE(ctx, !paged_overlaps(*kv, qkv, s_in) && !paged_overlaps(*kv, q_out, s_out), "%s: the cache may not overlap qkv or q_out",
                 what);
    a.qkv = qkv;
    a.stride = row_stride;
    a.q_out = q_out;
    a.q_stride = q_out_stride;
    a.wqk = wqk;
    a.cs = cs;
    a.n_pos = rot_dim > 0 && n_pos < (1 << 30) ? static_cast<int32_t>(n_pos) : 1 << 30;
    a.rot = rot_dim;
    a.inter = interleaved != 0;
    a.n_q = n_q;
    a.eps = eps;
    return launch_append(ctx, what, a, dtype);
}
