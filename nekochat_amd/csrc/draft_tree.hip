// Drafted trees over the paged 8-bit KV cache: the path that sampled tokens take from a tree's root, and the path's tokens
// moved together in the pages.
//
// Accept. at = the root; while a child of `at` holds the token sampled at `at`, the first such child is the next. Where row 0
// is no root, or the length is short of the rows, all rows are padding: nothing of them was appended, and there is no path. A
// wave to a sequence: parents, tokens and samples of up to 256 rows stay in its registers, so a step is two lane reads and a
// ballot for each 64 rows, no load.
//
// Keep. The cached value of slot base + path[k] goes to slot base + k, as if the append had made it there: under the
// page's power of two, the smallest that holds the largest finite magnitude, at least the old one where earlier tokens
// stay in the page (which are rounded again where it grows). A wave to a (sequence, kv head, k or v) takes the pages in
// order. Paths increase, so a token's source lies behind every slot that is written before it is read, and a page's
// scale changes only after all tokens that come from it.
//
// What bounds both: the launch and loads that need each other. Accept: one tree of 26 rows 3.9 us, 256 of up to 64 4.0.
// Keep, 8 kv heads of 128: one tree of 26 3.8 us, 64 of up to 61 (2.6 MB) 5.1.
#include <algorithm>

#include "internal.h"
#include "paged_device.h"

namespace neko_hip {
namespace {

struct AcceptArgs {
    const int32_t* tokens;
    const int32_t* sampled;
    const int32_t* parents;
    int32_t* path;
    int32_t* count;
    int32_t* next;
    int32_t* new_len;
    Paged p;  // rows, row_start, kv_len, n_seq
    int32_t max_path;
};

constexpr int kAcceptHeld = 4;  // rows of a lane that stay in registers

__global__ __launch_bounds__(64) void accept_kernel(AcceptArgs a) {
    const int32_t s = static_cast<int32_t>(blockIdx.x), lane = static_cast<int32_t>(threadIdx.x);
    const SeqRows r = paged_seq(a.p, s);
    int32_t parent[kAcceptHeld], token[kAcceptHeld], sampled[kAcceptHeld];
#pragma unroll
    for (int k = 0; k < kAcceptHeld; k++) {
        const int32_t i = 64 * k + lane;
        const bool in = i < r.n;
        parent[k] = in ? a.parents[r.begin + i] : -1;
        token[k] = in ? a.tokens[r.begin + i] : -1;
        sampled[k] = in ? a.sampled[r.begin + i] : -1;
    }
    int32_t* path = a.path + static_cast<int64_t>(s) * a.max_path;
    int32_t at = 0, count = 0, last = -1;
    const bool root = r.n > 0 && r.len >= r.n && __builtin_amdgcn_readfirstlane(parent[0]) == -1;
    while (root) {
        if (lane == 0) path[count] = at;
        count++;
        // The token sampled at `at`, and the first child that holds it.
        int32_t want = -1, below = -1;
        if (r.n <= 64 * kAcceptHeld) {
#pragma unroll
            for (int k = 0; k < kAcceptHeld; k++)
                if (at >> 6 == k) want = __builtin_amdgcn_readlane(sampled[k], at & 63);
#pragma unroll
            for (int k = 0; k < kAcceptHeld; k++) {
                const uint64_t hit = __ballot(parent[k] == at && token[k] == want && 64 * k + lane > at && 64 * k + lane < r.n);
                if (below < 0 && hit) below = 64 * k + __builtin_ctzll(hit);
            }
        } else {
            want = a.sampled[r.begin + at];
            for (int32_t i0 = at + 1; i0 < r.n && below < 0; i0 += 64) {
                const int32_t i = i0 + lane;
                const uint64_t hit = __ballot(i < r.n && a.parents[r.begin + i] == at && a.tokens[r.begin + i] == want);
                if (hit) below = i0 + __builtin_ctzll(hit);
            }
        }
        last = want;
        if (want < 0 || below < 0 || count == a.max_path) break;
        at = below;
    }
    for (int32_t i = count + lane; i < a.max_path; i += 64) path[i] = -1;
    if (lane == 0) {
        a.count[s] = count;
        a.next[s] = last;
        const int32_t len = r.len - r.n + count;
        a.new_len[s] = len < 0 ? 0 : len;
    }
}

struct KeepArgs {
    Paged p;
    const int32_t* path;
    const int32_t* count;
    int64_t path_stride;
    int32_t max_path;
};

__device__ __forceinline__ float max_value(uint32_t code) { return to_f32(f16_of_fp8<false>(code)[0]); }

// LPT: lanes to a token, 16 dimensions each.
template <int LPT>
__global__ __launch_bounds__(64) void keep_kernel(KeepArgs a) {
    constexpr int TPB = 64 / LPT;  // tokens of a step
    const int lane = static_cast<int>(threadIdx.x);
    const uint32_t parts = 2u * static_cast<uint32_t>(a.p.n_kv);
    const int32_t s = static_cast<int32_t>(blockIdx.x / parts);
    const int part = static_cast<int>(blockIdx.x % parts);
    const bool is_k = part < a.p.n_kv;
    const int g = is_k ? part : part - a.p.n_kv;
    const SeqRows r = paged_seq(a.p, s);
    const int32_t base = r.len - r.n, most = r.n < a.max_path ? r.n : a.max_path;
    const int32_t c = clamp_i32(a.count[s], 0, most);
    const int32_t* path = a.path + s * a.path_stride;
    if (base < 0) return;
    // The first token that moves.
    int32_t k0 = c;
    for (int32_t i0 = 0; i0 < c && k0 == c; i0 += 64) {
        const uint64_t moves = __ballot(i0 + lane < c && path[i0 + lane < c ? i0 + lane : 0] > i0 + lane);
        if (moves) k0 = i0 + __builtin_ctzll(moves);
    }
    const int hd = a.p.hd, sub = lane % LPT, in_step = lane / LPT;
    uint8_t* codes = (is_k ? a.p.k : a.p.v) + static_cast<uint64_t>(g) * a.p.head_bytes;
    float* scales = is_k ? a.p.ks : a.p.vs;
    const int32_t size = 1 << a.p.page_log2;
    for (int32_t from = k0; from < c;) {
        const int32_t pos0 = (base + from) & ~(size - 1), to = pos0 + size - base < c ? pos0 + size - base : c;  // this page's tokens
        const int32_t page = paged_page(a.p, s, pos0);
        // Token k's codes, 16 to a lane, and its scale's exponent; false where it does not move.
        auto get = [&](int32_t k, uint4v* x, int* e) {
            const int32_t src = k < to ? path[k] : -1;
            if (src <= k || src >= r.n || 16 * sub >= hd) return false;
            const int32_t id = paged_page(a.p, s, base + src);
            if (id < 0) return false;
            *x = *reinterpret_cast<const uint4v*>(codes + static_cast<uint64_t>(id) * a.p.page_bytes + ((base + src) & (size - 1)) * hd + 16 * sub);
            *e = scale_exp(scales[static_cast<int64_t>(id) * a.p.n_kv + g]);
            return true;
        };
        if (page >= 0) {
            uint32_t top = 0;
            bool any = false;
            uint4v first_x = {};
            int first_e = 0;
            bool first_is = false;
            for (int32_t k = from; k < to; k += TPB) {
                uint4v x = {};
                int e = 0;
                const bool is = get(k + in_step, &x, &e);
                if (k == from) {
                    first_x = x;
                    first_e = e;
                    first_is = is;
                }
                if (is) {
                    any = true;
                    uint32_t m = 0;
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const uint32_t code = (x[i / 4] >> (8 * (i % 4))) & 0x7fu;
                        m = code != 0x7fu && code > m ? code : m;
                    }
                    const uint32_t bits = __builtin_bit_cast(uint32_t, max_value(m) * exp2i(e));
                    top = top > bits ? top : bits;
                }
            }
            if (__any(any)) {
                top = wave_max_u32(top);
                float* scale = scales + static_cast<int64_t>(page) * a.p.n_kv + g;
                const int32_t old = base + from - pos0;  // tokens that stay before them
                const int had = old > 0 ? scale_exp(*scale) : -kScaleMax, need = need_exp(top), e = need > had ? need : had;
                uint8_t* at = codes + static_cast<uint64_t>(page) * a.p.page_bytes;
                auto again = [&](uint4v x, float by) {
                    uint4v y;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const half2v lo = f16_of_fp8<false>(x[i]), hi = f16_of_fp8<true>(x[i]);
                        const float v[4] = {to_f32(lo[0]), to_f32(lo[1]), to_f32(hi[0]), to_f32(hi[1])};
                        y[i] = fp8_of_f32(v, by);
                    }
                    return y;
                };
                if (e > had) {
                    const float by = exp2i(had - e < -126 ? -126 : had - e);
                    for (int32_t i = in_step; i < old; i += TPB)
                        if (16 * sub < hd) {
                            uint4v* x = reinterpret_cast<uint4v*>(at + i * hd + 16 * sub);
                            *x = again(*x, by);
                        }
                }
                for (int32_t k = from; k < to; k += TPB) {
                    uint4v x = first_x;
                    int from_e = first_e;
                    const bool is = k == from ? first_is : get(k + in_step, &x, &from_e);
                    // (2^-126 for less: its product with a code is below half the smallest one all the same)
                    if (is) *reinterpret_cast<uint4v*>(at + (base + k + in_step - pos0) * hd + 16 * sub) = again(x, exp2i(clamp_i32(from_e - e, -126, 126)));
                }
                if (lane == 0) *scale = exp2i(e);
            }
        }
        from = to;
    }
}

template <int LPT>
void launch_keep(neko_hip_ctx* ctx, const KeepArgs& a) {
    hipLaunchKernelGGL((keep_kernel<LPT>), dim3(static_cast<uint32_t>(a.p.n_seq) * 2u * static_cast<uint32_t>(a.p.n_kv)), dim3(64), 0, ctx->stream, a);
}

}  // namespace
}  // namespace neko_hip

using namespace neko_hip;

extern "C" int neko_hip_accept_tree(neko_hip_ctx* ctx, const int32_t* tokens, const int32_t* sampled, const int32_t* parents,
                                    int64_t rows, const int32_t* row_start, const int32_t* kv_len, int64_t n_seq, int32_t* path,
                                    int64_t max_path, int32_t* count, int32_t* next, int32_t* new_len) {
    const char* what = "neko_hip_accept_tree";
    NEKO_ENTER(ctx);
    NEKO_REQUIRE(ctx, rows >= 0 && rows <= 0x3fffffff, "%s: rows=%lld", what, (long long)rows);
    NEKO_REQUIRE(ctx, n_seq > 0 && n_seq <= (1 << 24), "%s: n_seq=%lld (1..2^24)", what, (long long)n_seq);
    NEKO_REQUIRE(ctx, max_path > 0 && max_path <= 0x3fffffff, "%s: max_path=%lld", what, (long long)max_path);
    NEKO_REQUIRE(ctx, row_start && kv_len && path && count && next && new_len && (rows == 0 || (tokens && sampled && parents)),
                 "%s: null pointer", what);
    const struct {
        const void* p;
        size_t bytes;
    } in[] = {{tokens, static_cast<size_t>(rows) * 4}, {sampled, static_cast<size_t>(rows) * 4}, {parents, static_cast<size_t>(rows) * 4},
              {row_start, static_cast<size_t>(n_seq + 1) * 4}, {kv_len, static_cast<size_t>(n_seq) * 4}},
      out[] = {{path, static_cast<size_t>(n_seq) * static_cast<size_t>(max_path) * 4}, {count, static_cast<size_t>(n_seq) * 4},
               {next, static_cast<size_t>(n_seq) * 4}, {new_len, static_cast<size_t>(n_seq) * 4}};
    for (const auto& o : out) {
        NEKO_REQUIRE(ctx, aligned(o.p, 4), "%s: misaligned pointer", what);
        for (const auto& i : in)
            NEKO_REQUIRE(ctx, aligned(i.p, 4) && !overlaps(o.p, o.bytes, i.p, i.bytes), "%s: an output overlaps an input, or a misaligned pointer", what);
        for (const auto& q : out)
            NEKO_REQUIRE(ctx, &q == &o || !overlaps(o.p, o.bytes, q.p, q.bytes), "%s: the outputs may not overlap", what);
    }
    AcceptArgs a{};
    a.tokens = tokens;
    a.sampled = sampled;
    a.parents = parents;
    a.path = path;
    a.count = count;
    a.next = next;
    a.new_len = new_len;
    a.p.row_start = row_start;
    a.p.kv_len = kv_len;
    a.p.n_seq = static_cast<int32_t>(n_seq);
    a.p.rows = static_cast<int32_t>(rows);
    a.max_path = static_cast<int32_t>(max_path);
    hipLaunchKernelGGL(accept_kernel, dim3(static_cast<uint32_t>(n_seq)), dim3(64), 0, ctx->stream, a);
    return after_launch(ctx, what);
}

extern "C" int neko_hip_keep_paged(neko_hip_ctx* ctx, const neko_paged_kv* kv, const neko_paged_batch* batch, const int32_t* path,
                                   int64_t path_stride, int64_t max_path, const int32_t* count) {
    const char* what = "neko_hip_keep_paged";
    NEKO_ENTER(ctx);
    KeepArgs a{};
    if (int rc = paged_args(ctx, what, kv, batch, 0x3fffffff, &a.p)) return rc;  // (the rows themselves are not looked at)
    NEKO_REQUIRE(ctx, path && count && aligned(path, 4) && aligned(count, 4), "%s: null or misaligned path or count", what);
    NEKO_REQUIRE(ctx, max_path > 0 && max_path <= 0x3fffffff && path_stride >= max_path && path_stride <= (int64_t(1) << 32),
                 "%s: paths of %lld entries, row stride %lld", what, (long long)max_path, (long long)path_stride);
    const size_t paths = rows_span(batch->n_seq, max_path, path_stride, 4);
    NEKO_REQUIRE(ctx, paths != 0 && !paged_overlaps(*kv, path, paths) && !paged_overlaps(*kv, count, static_cast<size_t>(batch->n_seq) * 4),
                 "%s: the cache may not overlap path or count", what);
    NEKO_REQUIRE(ctx, batch->n_seq * 2 * kv->n_kv <= 0x7fffffff, "%s: grid too large", what);
    a.path = path;
    a.count = count;
    a.path_stride = path_stride;
    a.max_path = static_cast<int32_t>(max_path);
    if (kv->hd <= 16) launch_keep<1>(ctx, a);
    else if (kv->hd <= 32) launch_keep<2>(ctx, a);
    else if (kv->hd <= 64) launch_keep<4>(ctx, a);
    else if (kv->hd <= 128) launch_keep<8>(ctx, a);
    else launch_keep<16>(ctx, a);
    return after_launch(ctx, what);
}
