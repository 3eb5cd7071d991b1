// The paged cache's index arithmetic (nekochat_amd/csrc/paged.h) as the kernels compile it, on the host: what
// tests/test_paged_index.py asks of it, for batches that no host check has looked at.
#include "../../nekochat_amd/csrc/paged.h"

#include <vector>

using namespace neko_hip;

extern "C" {

struct Batch {
    const int32_t* table;
    const int32_t* row_start;
    const int32_t* kv_len;
    int64_t table_stride, n_pages;
    int32_t max_pages, n_seq, rows, page_log2, n_kv, hd;
};

static Paged paged(const Batch* b) {
    Paged p{};
    p.table = b->table;
    p.row_start = b->row_start;
    p.kv_len = b->kv_len;
    p.table_stride = b->table_stride;
    p.n_pages = b->n_pages;
    p.max_pages = b->max_pages;
    p.n_seq = b->n_seq;
    p.rows = b->rows;
    p.page_log2 = b->page_log2;
    p.n_kv = b->n_kv;
    p.hd = b->hd;
    return p;
}

int check_need_exp(uint32_t bits) { return need_exp(bits); }
int check_scale_exp(float s) { return scale_exp(s); }
int check_page(const Batch* b, int32_t s, int32_t pos) { return paged_page(paged(b), s, pos); }
void check_seq(const Batch* b, int32_t s, int32_t* out) {
    const SeqRows r = paged_seq(paged(b), s);
    out[0] = r.begin;
    out[1] = r.n;
    out[2] = r.len;
}

// Every segment that the slots of the append's launch reach: (sequence, page, a, b, row of slot 0, position of slot 0)
// each; their number, or -1 past `room`.
int64_t check_segments(const Batch* b, int32_t limit, int32_t* out, int64_t room) {
    const Paged p = paged(b);
    int64_t n = 0;
    const int64_t slots = segment_slots(p.rows, p.n_seq, p.page_log2);
    for (int64_t at = 0; at < slots; at++) {
        int32_t s = 0;  // the last whose first slot is at or before this one
        while (s + 1 < p.n_seq && segment_slot(p, s + 1) <= at) s++;
        const Segment g = paged_segment(p, s, static_cast<int32_t>(at) - segment_slot(p, s), limit);
        if (g.page < 0) continue;
        if (n == room) return -1;
        const int32_t row[6] = {s, g.page, g.a, g.b, g.row0, g.pos0};
        for (int i = 0; i < 6; i++) out[6 * n + i] = row[i];
        n++;
    }
    return n;
}

// The attention launch's workgroups per kv head and the bounds that the host sizes the grid and workspace by.
void check_blocks(const Batch* b, const AttnTiling* given, int64_t* out) {
    const Paged p = paged(b);
    AttnTiling t = *given;
    attn_set(t);
    const int32_t reach = paged_reach(p);
    double work = 0;
    int64_t all = 0;
    for (int32_t s = 0; s < p.n_seq; s++) {
        const SeqRows r = paged_seq(p, s);
        work += static_cast<double>(attn_tiles(t, r)) * attn_units(t, reach, r);
        all += attn_tiles(t, r);
    }
    const int32_t chunk = attn_chunk(t, work * p.n_kv, all * p.n_kv);
    int64_t tiles = 0, blocks = 0, uncovered = 0, split = 0;
    for (int32_t s = 0; s < p.n_seq; s++) {
        const SeqRows r = paged_seq(p, s);
        const int64_t n = attn_tiles(t, r), units = attn_units(t, reach, r), splits = attn_splits(static_cast<int32_t>(units), chunk);
        tiles += n;
        blocks += n * splits;
        if (n && splits * chunk < units) uncovered++;
        if (splits > 1) split += n;
    }
    out[0] = tiles;
    out[1] = blocks;
    out[2] = attn_tiles_bound(t, p.rows, p.n_seq);
    out[3] = attn_blocks_bound(t, p.rows, p.n_seq, p.n_kv);
    out[4] = uncovered;
    out[5] = split;
    out[6] = attn_may_split(t, p) ? attn_split_tiles_bound(t, p.rows, p.n_seq, p.n_kv) : 0;
}

// The same of a launch as it is planned: what the device splits beside what the host has made room for: tiles, blocks,
// tiles that are split, units of keys that no split covers; whether splits are planned, the most blocks and split tiles.
void check_plan(const Batch* b, const AttnTiling* given, int64_t* out) {
    const Paged p = paged(b);
    AttnTiling t = *given;
    attn_set(t);
    const int32_t reach = paged_reach(p);
    const int32_t chunk = attn_plan(t, p, [&](double& work, int64_t& n) {
        work = 0;
        n = 0;
        for (int32_t s = 0; s < p.n_seq; s++) {
            const SeqRows r = paged_seq(p, s);
            work += static_cast<double>(attn_tiles(t, r)) * attn_units(t, reach, r);
            n += attn_tiles(t, r);
        }
        work *= p.n_kv;
        n *= p.n_kv;
    });
    for (int i = 0; i < 4; i++) out[i] = 0;
    for (int32_t s = 0; s < p.n_seq; s++) {
        const SeqRows r = paged_seq(p, s);
        const int64_t n = attn_tiles(t, r), units = attn_units(t, reach, r), splits = attn_splits(static_cast<int32_t>(units), chunk);
        out[0] += n;
        out[1] += n * splits;
        if (splits > 1) out[2] += n;
        if (n && splits * chunk < units) out[3] += units - splits * chunk;
    }
    out[4] = attn_may_split(t, p);
    out[5] = attn_blocks_bound(t, p.rows, p.n_seq, p.n_kv);
    out[6] = attn_split_tiles_bound(t, p.rows, p.n_seq, p.n_kv);
}

int check_seq_from(const Batch* b, int32_t s, int32_t row) { return paged_seq_from(paged(b), s, row); }
int check_splits(int32_t units, int32_t chunk) { return attn_splits(units, chunk); }

}  // extern "C"
