// The paged 8-bit KV cache: its launch arguments, and the index arithmetic that the append and attention
// kernels share. Everything on the device side of a batch -- page ids, row ranges, lengths -- is data that no
// host check has seen, so each value is brought into range here before it forms an address: a page id outside
// the cache is a page that holds nothing, a row range is cut to the call's rows, a length to the table's reach.
// The functions without wave operations compile for the host too and are tested there.
#pragma once

#ifdef __HIPCC__
#include "device.h"
#define NEKO_HD __host__ __device__ __forceinline__
#else
#include <cstdint>
#include <cstring>
#define NEKO_HD inline
#endif

namespace neko_hip {

// Scales are powers of two within 2^+-kScaleMax; an E4M3 code reaches kCodeMax = 1.75 * 2^8.
constexpr int kScaleMax = 64;
constexpr int kBlockKeys = 16;  // the smallest page; every page is a whole number of such blocks

struct Paged {
    uint8_t* k;  // [n_pages][n_kv][page][hd] E4M3 codes
    uint8_t* v;
    float* ks;  // [n_pages][n_kv]
    float* vs;
    const int32_t* table;  // page ids of sequence s: table[s * table_stride ..], max_pages of them
    const int32_t* row_start;
    const int32_t* kv_len;
    int64_t table_stride;
    int64_t n_pages;
    int32_t max_pages;
    int32_t n_seq;
    int32_t rows;
    int32_t page_log2;
    int32_t n_kv;
    int32_t hd;
    uint32_t head_bytes;  // of one kv head's tokens of a page: page * hd
    uint32_t page_bytes;  // n_kv * head_bytes (paged_args: below 2^28)
};

struct SeqRows {
    int32_t begin, n;  // this call's rows of the sequence
    int32_t len;       // its length with them, as given: row i stands at position len - n + i
};

NEKO_HD int32_t clamp_i32(int32_t v, int32_t lo, int32_t hi) { return v < lo ? lo : v > hi ? hi : v; }

NEKO_HD SeqRows paged_seq(const Paged& p, int32_t s) {
    SeqRows r;
    r.begin = clamp_i32(p.row_start[s], 0, p.rows);
    r.n = clamp_i32(p.row_start[s + 1], r.begin, p.rows) - r.begin;
    // (2^30: positions and the keys of a tile past them stay in 32 bits)
    r.len = clamp_i32(p.kv_len[s], 0, 1 << 30);
    return r;
}

// The last sequence from s on that begins at or before `row`, s being one: it or one of the next few, or by halves
// (a batch padded with places that are idle: one after the other, 255 of those took 29 us).
NEKO_HD int32_t paged_seq_from(const Paged& p, int32_t s, int32_t row) {
    for (int k = 0; k < 4; k++) {
        if (s + 1 >= p.n_seq || clamp_i32(p.row_start[s + 1], 0, p.rows) > row) return s;
        s++;
    }
    int32_t past = p.n_seq;
    while (past - s > 1) {
        const int32_t mid = s + (past - s) / 2;
        if (clamp_i32(p.row_start[mid], 0, p.rows) <= row) s = mid;
        else past = mid;
    }
    return s;
}

// Keys that the table reaches: positions below this have an entry.
NEKO_HD int32_t paged_reach(const Paged& p) {
    const int64_t n = static_cast<int64_t>(p.max_pages) << p.page_log2;
    return n < (1 << 30) ? static_cast<int32_t>(n) : 1 << 30;
}

// The page that holds position `pos` of sequence s; -1 where there is none.
NEKO_HD int32_t paged_page(const Paged& p, int32_t s, int32_t pos) {
    const int32_t i = pos >> p.page_log2;
    if (pos < 0 || i >= p.max_pages) return -1;
    const int32_t id = p.table[s * p.table_stride + i];
    return id < 0 || id >= p.n_pages ? -1 : id;
}

// Exponent of a scale, from its bits (a scale that is no power of two counts as the one below it).
NEKO_HD int scale_exp(float s) {
    uint32_t b;
#ifdef __HIPCC__
    b = __builtin_bit_cast(uint32_t, s);
#else
    std::memcpy(&b, &s, 4);
#endif
    const int e = static_cast<int>((b >> 23) & 255u) - 127;
    return e < -kScaleMax ? -kScaleMax : e > kScaleMax ? kScaleMax : e;
}

// The smallest exponent e, within +-kScaleMax, with amax <= 448 * 2^e, of the bits of a finite amax >= 0:
// amax = 1.f * 2^x is at most 1.75 * 2^x or needs one more.
NEKO_HD int need_exp(uint32_t amax_bits) {
    const int x = static_cast<int>(amax_bits >> 23) - 127;
    const int e = x - 8 + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return e < -kScaleMax ? -kScaleMax : e > kScaleMax ? kScaleMax : e;
}

// ---- append: page segments. A segment is the new rows of one sequence that fall into one page. Sequence s
// gets the slots from floor(begin / page) + 2 s on: its segments number at most floor(n / page) + 2, and
// floor(a + b) >= floor(a) + floor(b) keeps the slots of the next sequence past them.
NEKO_HD int32_t segment_slot(const Paged& p, int32_t s) { return (clamp_i32(p.row_start[s], 0, p.rows) >> p.page_log2) + 2 * s; }
NEKO_HD int64_t segment_slots(int64_t rows, int64_t n_seq, int page_log2) { return (rows >> page_log2) + 2 * n_seq; }

struct Segment {
    int32_t page;    // -1: nothing to do
    int32_t a, b;    // slots [a, b) of the page are new
    int32_t row0;    // row of slot 0 (slots below a: not a row of this call)
    int32_t pos0;    // position of slot 0
};

// Segment i of sequence s; `limit`: positions from there on are not written.
NEKO_HD Segment paged_segment(const Paged& p, int32_t s, int32_t i, int32_t limit) {
    const SeqRows r = paged_seq(p, s);
    const int32_t first = r.len - r.n;  // position of the first row; below 0 where the length is short of the rows
    const int32_t begin = first < 0 ? 0 : first;
    const int32_t end = r.len < limit ? r.len : limit;
    Segment g;
    const int64_t j = static_cast<int64_t>(begin >> p.page_log2) + i;
    g.page = -1;
    g.a = g.b = 0;
    g.pos0 = 0;
    g.row0 = 0;
    if (i < 0 || begin >= end || (j << p.page_log2) >= end) return g;
    g.pos0 = static_cast<int32_t>(j << p.page_log2);
    g.page = paged_page(p, s, g.pos0);
    g.a = begin > g.pos0 ? begin - g.pos0 : 0;
    const int32_t size = 1 << p.page_log2;
    g.b = end - g.pos0 < size ? end - g.pos0 : size;
    g.row0 = r.begin + (g.pos0 - first);
    return g;
}

// ---- attention: row tiles and key splits. The rows of a sequence times the query heads of a kv head are cut
// into tiles of `tile_rows`; a tile's keys into splits of `chunk` keys, so that the launch has about `target`
// workgroups whatever the lengths are, which only the device knows.
struct AttnTiling {
    int32_t group;       // query heads per kv head
    int32_t tile_log2;   // flattened (token, head) rows of a tile
    int32_t unit_log2;   // keys that a split is a multiple of
    int32_t target;      // workgroups that are resident at once
    int32_t least;       // units of a split, at least
    int32_t window;      // 0: none
    int32_t span;        // with a window: the keys that a tile spans at most (attn_set)
    // Sequences with min_rows <= flattened rows <= max_rows are this launch's.
    int32_t min_rows, max_rows;
};

// The derived fields. A tile spans its first token's window and its further tokens, from a multiple of 32.
NEKO_HD void attn_set(AttnTiling& t) {
    const int64_t span = static_cast<int64_t>(t.window) + ((1 << t.tile_log2) / t.group + 2) + 32;
    t.span = span < (1 << 30) ? static_cast<int32_t>(span) : 1 << 30;
}

NEKO_HD int32_t attn_tiles(const AttnTiling& t, const SeqRows& r) {
    const int32_t rows = r.n * t.group;  // rows * n_head <= 2^30
    if (rows < t.min_rows || rows > t.max_rows) return 0;
    return (rows + (1 << t.tile_log2) - 1) >> t.tile_log2;
}

// Units of keys that a tile of this sequence spans at most: all of them, or the window's.
NEKO_HD int32_t attn_units(const AttnTiling& t, int32_t reach, const SeqRows& r) {
    int32_t keys = r.len < reach ? r.len : reach;
    if (t.window > 0 && t.span < keys) keys = t.span;
    return (keys + (1 << t.unit_log2) - 1) >> t.unit_log2;
}

// Units per split, at most, from the launch's tiles and its work, the sum over its tiles of their units (whole
// numbers, both over all kv heads): as many workgroups as are resident at once, or, where the tiles alone are half of
// those, half, so that only what is longer than average is split. (f32's rounding may leave a chunk short of work /
// wanted by 2^-22 of it: the one workgroup more in attn_blocks_bound.) Measured (512 resident): 509 rows of 32 heads over 8190
// keys, 128 tiles, in four splits 106 us, in three (what is free beside one for each tile) 123; a prompt of 1400, 350 tiles,
// with half as many wanted 50.3, with all 63.6.
NEKO_HD int32_t attn_chunk(const AttnTiling& t, double work, int64_t tiles) {
    const int32_t wanted = 2 * tiles >= t.target ? (t.target + 1) / 2 : t.target;
    const float c = static_cast<float>(work) / static_cast<float>(wanted);
    const int32_t n = (c < 1e9f ? static_cast<int32_t>(c) : 1000000000) + 1;
    return n < t.least ? t.least : n;
}

// ceil(units / chunk) without an integer division: the quotient by a reciprocal is off by one at most for the fewer
// than 2^20 splits that there are, and put right.
NEKO_HD int32_t attn_splits(int32_t units, int32_t chunk) {
    if (units <= chunk) return 1;
    int32_t q = static_cast<int32_t>(static_cast<float>(units) * (1.0f / static_cast<float>(chunk)));
    const int32_t left = units - q * chunk;
    if (left > 0) q++;
    if (left > chunk) q++;
    if (left <= -chunk) q--;
    return q;
}

// Workgroups per kv head that the splits above can come to: sum of tiles * splits <= work / (n_kv * chunk) +
// sum of tiles, and the tiles number at most rows * group / tile_rows + n_seq. Tiles that are split have more than
// chunk units each, so they number at most work / (n_kv * chunk) <= target / n_kv.
NEKO_HD int64_t attn_tiles_bound(const AttnTiling& t, int64_t rows, int64_t n_seq) {
    const int64_t tiles = ((rows * t.group) >> t.tile_log2) + (rows < n_seq ? rows : n_seq);
    return tiles < rows * t.group ? tiles : rows * t.group;
}
NEKO_HD int64_t attn_blocks_bound(const AttnTiling& t, int64_t rows, int64_t n_seq, int n_kv) {
    return attn_tiles_bound(t, rows, n_seq) + (t.target + n_kv - 1) / n_kv + 1;
}

NEKO_HD int64_t attn_split_tiles_bound(const AttnTiling& t, int64_t rows, int64_t n_seq, int n_kv) {
    const int64_t tiles = attn_tiles_bound(t, rows, n_seq), most = (t.target + n_kv - 1) / n_kv + 1;
    return tiles < most ? tiles : most;
}
// Whether a launch plans for splits: a workspace for their partial results and the merge. One sequence with as many
// tiles as wanted would not be split (chunk >= units), unless some of the call's rows are not its own.
NEKO_HD bool attn_may_split(const AttnTiling& t, const Paged& p) {
    if (paged_reach(p) <= static_cast<int64_t>(t.least) << t.unit_log2) return false;
    if (p.n_seq > 1) return true;
    const int64_t tiles = (static_cast<int64_t>(p.rows) * t.group + (1 << t.tile_log2) - 1) >> t.tile_log2;
    return tiles * p.n_kv < t.target;
}
// The chunk of a launch, as the device takes it: more than any tile has where no splits are planned, so that what only
// the device knows -- rows behind the last sequence, which leave fewer tiles than the call's rows make -- cannot ask for
// splits that have no place. (Such a call takes no longer than one whose rows are all the sequence's.) `sums`: the work
// and the tiles of attn_chunk.
constexpr int32_t kUnsplit = 1 << 30;
template <typename F>
NEKO_HD int32_t attn_plan(const AttnTiling& t, const Paged& p, F&& sums) {
    if (!attn_may_split(t, p)) return kUnsplit;
    double work;
    int64_t tiles;
    sums(work, tiles);
    return attn_chunk(t, work, tiles);
}

}  // namespace neko_hip
