"""GPU tests of drafted trees over the paged 8-bit KV cache (neko_hip_qk_norm_rope_tree_paged, neko_hip_attention_tree_paged,
neko_hip_accept_tree, neko_hip_keep_paged) against a plain evaluation in 64 bits (tests/tree_oracle.py).

Tolerances. u = 2^-24, half a step of f32, and h = 2^-11, of f16.
  append: q as at most eight f32 roundings of values of size z = |x_a| + |x_b| (the pair) and one to its type; scales
    equal; codes within half a step of E4M3 (2^-4 of the value, or 2^-10 where subnormal) besides what precedes them.
  attention: as over rows in a line. A weight's relative error is its exponent's, the score's -- hd products in any order,
    hd u s with s the largest sum of |q k|, and 4 u s for scaling, cap and bias -- and 8 u of its own; errors e of all
    weights move the quotient by at most 2 e a, a = sum w |v| / sum w; sums over n keys, 32 to a product, by 2 (n / 32 + 64)
    u a. f16 results are rounded once (h |out|), and f16 calls of many rows round each weight to f16 (h a).
  accept: equal. keep: equal, codes and scales: a code times a power of two is exact in f32, its rounding to E4M3 torch's.
"""
import threading

import numpy as np
import pytest
import torch

import paged_oracle as P
import tree_oracle as T
from nekochat_amd import NekoError, ops

pytestmark = pytest.mark.gpu

U, H16 = T.U, T.H16
DT = {"f16": torch.float16, "f32": torch.float32}


def _case(msg):
    print(f"[case] {msg}", flush=True)


def _cache_on(cache, dev):
    return ops.PagedKV(*(t.clone().to(dev) for t in cache))


def _parts(cache):
    return tuple(x.cpu() for x in (cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales))


def _same(a, b):
    return torch.equal(a.view(torch.uint8) if a.dtype == P.F8 else a, b.view(torch.uint8) if b.dtype == P.F8 else b)


def _trees(kind, seed):
    rng = np.random.default_rng(seed)
    tree = lambda n, reach=9, padding=0: T.random_parents(n, reach, rng, padding)  # noqa: E731
    if kind == "small":  # one row, chains, a forest, padding; contexts from nothing on; idle places
        return [([-1], 0), (tree(5), 0), (tree(4, 1), 33), ([], 40), (tree(7, padding=3), 100), ([-1, -1, 0, 1, 1], 16), ([], 0),
                ([-2, -2], 20), (tree(9), 333), ([-1], 700)]
    if kind == "large":  # more rows than one word has bits, ends inside blocks and pages
        return [(tree(64), 200), (tree(33, 1), 31), ([], 5), (tree(40, padding=24), 350), (tree(70, 20), 65), (tree(2), 500)]
    return [(tree(300, 40), 250), (tree(130, 130), 1)]


# ------------------------------------------------------------------ attention

def _wide(t, H, page):
    """Free places in a row of the page table: with so many the batch could be large, and its longer trees run on the tiles
    of 128 rows; without, one of this size runs on the 16-row kernel alone."""
    return int(60e6) // (t.batch.row_start[-1] * H * page) + 1


def _check(dev, H, KV, hd, dtype, t, seed, cache=None, scale=None, what="", q=None, unaligned=0, mask=None, **kw):
    page, dt, b = t.batch.page, DT[dtype], t.batch
    g = torch.Generator().manual_seed(seed)
    q = torch.randn((b.rows, H * hd), generator=g).to(dt) if q is None else q
    cache = cache or P.random_cache(b.n_pages, KV, page, hd, seed + 1)
    scale = 1 / np.sqrt(hd) if scale is None else scale
    buf = torch.full((b.rows, H * hd + unaligned), 7.0, dtype=dt, device=dev)
    out = buf[:, unaligned // 2: unaligned // 2 + H * hd]
    dq = q.to(dev)
    if unaligned:
        dq = torch.cat([torch.zeros((b.rows, unaligned // 2), dtype=dt, device=dev), dq], 1)[:, unaligned // 2:]
    table, start, length, depth = t.tensors(dev)
    slopes = kw.get("slopes")
    ops.attention_tree_paged(dq, _cache_on(cache, dev), table, start, length, depth, (t.mask() if mask is None else mask).to(dev), H, scale=scale,
                             out=out, **{**kw, "slopes": None if slopes is None else slopes.to(dev)})
    torch.cuda.synchronize()
    want, a, s = T.attention(q, cache, t, H, float(np.float32(scale)), **kw)
    got, total = out.cpu().double(), int(b.row_start[-1])
    assert torch.equal(got[total:], torch.full_like(got[total:], 7.0)), "rows of no sequence were written"
    got, want, a, s = got[:total], want[:total], a[:total], s[:total]
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    ok = ~torch.isnan(want)
    over = torch.where(ok, (got - want).abs() - T.bar(want, a, s, max(n for _, n in b.seqs), hd, dtype), -1.0)
    print(f"{what} {H}/{KV}/{hd} page {page} {dtype}: worst past the bar {float(over.max()):.2e}", flush=True)
    assert float(over.max()) <= 0
    return got


def _made(kind, page, seed, H, wide, pad=2):
    trees = _trees(kind, seed)
    t = T.Trees(trees, page, seed, pad=pad)
    return T.Trees(trees, page, seed, pad=pad, slack=_wide(t, H, page)) if wide else t


@pytest.mark.parametrize("H,KV,hd,page,dtype", [
    (8, 2, 128, 16, "f16"), (8, 2, 128, 32, "f32"), (6, 6, 64, 64, "f32"), (4, 4, 64, 16, "f16"), (8, 1, 256, 16, "f16"),
    (3, 1, 256, 128, "f32"), (5, 1, 80, 16, "f16"), (2, 2, 16, 16, "f32"), (20, 1, 128, 256, "f16"), (2, 1, 144, 32, "f32"),
])
@pytest.mark.parametrize("kind,wide", [("small", False), ("small", True), ("large", False), ("large", True)])
def test_attention(dev, H, KV, hd, page, dtype, kind, wide):
    _case(f"attention of {kind} trees, wide {wide}, {H}/{KV}/{hd} page {page} {dtype}")
    _check(dev, H, KV, hd, dtype, _made(kind, page, hd + page, H, wide), hd, what=f"{kind} {wide}")


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("kw", [{"window": 1}, {"window": 4}, {"window": 37}, {"window": 300}, {"softcap": 3.0},
                                {"slopes": True}, {"slopes": True, "window": 3}, {"slopes": True, "softcap": 5.0, "window": 40}])
def test_attention_cap_window_slopes(dev, kw, wide, dtype):
    """Distances are between places, not slots: windows that end inside the tree and before it, a bias along it."""
    _case(f"attention of trees, {kw}, wide {wide} {dtype}")
    H = 4
    if kw.get("slopes"):
        kw = {**kw, "slopes": torch.tensor([0.5, 0.1, 0.03, 0.0])}
    for kind in ("small", "large"):
        _check(dev, H, 2, 64, dtype, _made(kind, 16, 7, H, wide), 8, what=kind, **kw)


@pytest.mark.parametrize("hd,dtype", [(64, "f16"), (128, "f16"), (128, "f32"), (256, "f32")])
def test_attention_more_rows_than_two_words(dev, hd, dtype):
    _case(f"attention of trees of 300 rows, {hd} {dtype}")
    for wide in (False, True):
        _check(dev, 4, 2, hd, dtype, _made("huge", 16, 5, 4, wide), 6, what="huge")


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("trees", [[(7, 5000)], [(1, 4097), (3, 2)], [(64, 4000)], [(20, 2050), (0, 0), (20, 3)]])
def test_attention_split_keys(dev, trees, dtype):
    """Keys split over workgroups, the tree in the last split or at the edge of one."""
    _case(f"attention of trees, split keys, {trees} {dtype}")
    rng = np.random.default_rng(1)
    trees = [(T.random_parents(n, 5, rng) if n else [], ctx) for n, ctx in trees]
    _check(dev, 8, 2, 128, dtype, T.Trees(trees, 16, 11), 11, what=str(len(trees)))
    t = T.Trees(trees, 16, 11, slack=_wide(T.Trees(trees, 16, 11), 8, 16))
    _check(dev, 8, 2, 128, dtype, t, 11, what=str(len(trees)))


@pytest.mark.parametrize("hd,dtype,window", [(128, "f16", 0), (64, "f32", 11), (128, "f32", 0), (256, "f16", 0)])
@pytest.mark.parametrize("seqs,most", [(24, 24), (70, 9)])
def test_attention_many_trees(dev, seqs, most, hd, dtype, window):
    """More 16-row tiles than are resident, of more sequences than a wave has lanes too."""
    _case(f"attention of {seqs} trees, {hd} {dtype} window {window}")
    rng = np.random.default_rng(seqs)
    trees = [(T.random_parents(n, 4, rng, 1 if n > 4 and s % 5 == 0 else 0), int(rng.integers(0, 90)))
             for s, n in enumerate(int(rng.integers(0 if i % 7 == 6 else most - 4, most + 1)) for i in range(seqs))]
    _check(dev, 32, 8, hd, dtype, T.Trees([t if t[0] else ([], 0) for t in trees], 16, seqs), seqs, what="many", window=window)


@pytest.mark.parametrize("hd,dtype,wide", [(64, "f16", False), (128, "f32", False), (128, "f16", True)])
def test_attention_trees_of_most_rows(dev, hd, dtype, wide):
    """32 words of mask."""
    _case(f"attention of trees of 1024 rows, {hd} {dtype} wide {wide}")
    rng = np.random.default_rng(1024)
    trees = [(T.random_parents(1024, 30, rng), 37), ([-1], 3), (list(range(-1, 998)), 5)]
    t = T.Trees(trees, 16, 7)
    if wide:
        t = T.Trees(trees, 16, 7, slack=_wide(t, 2, 16))
    assert t.words == 32
    _check(dev, 2, 1, hd, dtype, t, 9, what="1024 rows")


@pytest.mark.parametrize("wide", [False, True])
def test_attention_any_mask(dev, wide):
    """Masks that are no tree's: rows that see nothing of it, not themselves, later rows; bits past the sequence's rows;
    fewer bits than rows; rows that see nothing at all."""
    _case(f"attention, any mask, wide {wide}")
    rng = np.random.default_rng(3)
    for words, window in ((1, 0), (2, 0), (3, 5)):
        t = _made("large", 16, 9, 4, wide)
        t.words = words
        noise = torch.from_numpy(rng.integers(-2**31, 2**31, (t.rows, words), dtype=np.int64).astype(np.int32))
        noise[::5] = 0
        start = t.batch.row_start
        for s, (n, _) in enumerate(t.batch.seqs):
            for i in range(n):
                r = int(start[s]) + i
                bits = noise[r].numpy().view(np.uint32)
                t.sees[r] = {k for k in range(min(n, 32 * words)) if bits[k // 32] >> (k % 32) & 1}
        _check(dev, 4, 2, 64, "f32", t, 10, mask=noise, window=window)
    t = T.Trees([([-1, 0, 0], 0), ([-1] * 40, 0)], 16, 2, slack=3000 if wide else 1)
    t.sees = [{0}, set(), {0, 2}] + [set()] * 40
    got = _check(dev, 4, 2, 64, "f32", t, 12)
    assert bool((got[1] == 0).all()) and bool((got[3:] == 0).all()) and bool((got[2] != 0).any())


def test_attention_mask_and_rows_of_any_stride(dev):
    _case("attention of trees, strides")
    t = _made("large", 32, 3, 4, False)
    wide = torch.full((t.rows, t.words + 3), -1, dtype=torch.int32)
    wide[:, 2: 2 + t.words] = t.mask()
    for dtype in ("f16", "f32"):
        q = torch.randn((t.rows, 256), generator=torch.Generator().manual_seed(4)).to(DT[dtype])
        dw = wide.to(dev)

        class View:  # the columns of a wider mask, on the device
            def to(self, _):
                return dw[:, 2: 2 + t.words]

        _check(dev, 4, 2, 64, dtype, t, 4, q=q, mask=View(), unaligned=6)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("wide", [False, True])
def test_attention_of_chains_is_that_of_rows_in_a_line(dev, wide, dtype):
    """A tree without branches: attention_paged's rows, within both calls' roundings."""
    _case(f"attention of chains, wide {wide} {dtype}")
    trees = [(list(range(-1, n - 1)), ctx) for n, ctx in ((1, 50), (17, 100), (64, 0), (50, 333))]
    t = T.Trees(trees, 16, 4, slack=3000 if wide else 1)
    H, hd = 4, 128
    cache = P.random_cache(t.batch.n_pages, 2, 16, hd, 5)
    q = torch.randn((t.rows, H * hd), generator=torch.Generator().manual_seed(6)).to(DT[dtype])
    table, start, length, depth = t.tensors(dev)
    dc = _cache_on(cache, dev)
    for kw in ({}, {"window": 30}, {"slopes": torch.tensor([0.1, 0.2, 0.3, 0.0], device=dev)}):
        a = ops.attention_paged(q.to(dev), dc, table, start, length, H, **kw)
        b = ops.attention_tree_paged(q.to(dev), dc, table, start, length, depth, t.mask().to(dev), H, **kw)
        torch.cuda.synchronize()
        want, size, s = P.attention(q, cache, t.batch, H, float(np.float32(hd ** -0.5)), **{k: v if k == "window" else v.cpu() for k, v in kw.items()})
        bar = 2 * T.bar(want, size, s, 400, hd, dtype)
        assert float(((a - b).abs().cpu().double() - bar).max()) <= 0


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("hd,dtype", [(64, "f32"), (128, "f16"), (128, "f32"), (256, "f32"), (80, "f16")])
def test_attention_nan_where_it_is_seen_only(dev, hd, dtype, wide):
    """NaN in a token, of the context or drafted, reaches the rows that see it and no others; free slots, padding's slots
    and those past the length may hold anything."""
    _case(f"attention of trees, NaN tokens, {hd} {dtype} wide {wide}")
    rng = np.random.default_rng(6)
    trees = [(T.random_parents(6, 3, rng), 50), ([-1, 0, 0, 1, 1, 2, 2, 3, -2, -2], 75), (T.random_parents(60, 6, rng), 90), (T.random_parents(20, 9, rng), 120)]
    page, KV, H = 16, 2, 4
    t = T.Trees(trees, page, 61)
    if wide:
        t = T.Trees(trees, page, 61, slack=_wide(t, H, page))
    b = t.batch
    cache = P.random_cache(b.n_pages, KV, page, hd, 62)
    kb, vb = cache[0].view(torch.uint8), cache[1].view(torch.uint8)

    def at(s, j):
        return int(b.table[s, j // page]), slice(None), j % page

    for pg in b.free:
        kb[pg], vb[pg] = 0x7F, 0xFF
    for s, (_, length) in enumerate(b.seqs):
        if length % page:
            kb[b.table[s, length // page], :, length % page:] = 0xFF
            vb[b.table[s, length // page], :, length % page:] = 0x7F
    for j in (75 + 8, 75 + 9):  # padding
        kb[at(1, j)], vb[at(1, j)] = 0xFF, 0x7F
    vb[at(1, 75 + 1)] = 0x7F  # drafted: row 1 and those below it
    vb[int(b.table[2, 33 // page]), 1, 33 % page, hd - 1] = 0xFF  # context: every row, one dimension
    kb[int(b.table[2, (90 + 7) // page]), 0, (90 + 7) % page, 3] = 0x7F
    vb[int(b.table[3, 125 // page]), 0, 125 % page, 0] = 0x7F
    got = _check(dev, H, KV, hd, dtype, t, 63, cache=cache)
    rows = torch.isnan(got).any(1)
    assert rows[6: 16].tolist() == [False, True, False, True, True, False, False, True, False, False]
    assert bool((got[14:16] == 0).all()) and not bool(rows[:6].any())


@pytest.mark.parametrize("wide", [False, True])
def test_attention_bad_pages_lengths_and_depths(dev, wide):
    """Pages outside the cache hold nothing; a length short of the rows, and depths outside the tree, see nothing."""
    _case(f"attention of trees, bad pages, lengths and depths, wide {wide}")
    rng = np.random.default_rng(8)
    trees = [(T.random_parents(n, 4, rng), ctx) for n, ctx in ((5, 55), (40, 50), (3, 20), (40, 8))]
    t = T.Trees(trees, 16, 81)
    if wide:
        t = T.Trees(trees, 16, 81, slack=_wide(t, 4, 16))
    b = t.batch
    b.table[0, 1] = b.n_pages + 5
    b.table[1, 3:] = -1
    b.table[2, 0] = -2**31
    b.seqs[3] = (40, 30)  # fewer tokens than rows
    b.kv_len[3] = 30
    r = int(b.row_start[1])
    for i, d in ((3, -1), (4, 40), (5, 2**31 - 1), (6, -2**31)):
        t.depth[r + i] = d
    for row in range(r, r + 40):
        t.sees[row] -= {3, 4, 5, 6}
    got = _check(dev, 4, 2, 64, "f32", t, 82)
    assert bool((got[r + 3: r + 7] == 0).all()) and bool((got[int(b.row_start[3]):] == 0).all())


def test_attention_not_finite_queries(dev):
    _case("attention of trees, q not finite")
    H, hd = 4, 64
    for wide in (False, True):
        for dtype in ("f16", "f32"):
            t = _made("large", 16, 71, H, wide)
            q = torch.randn((t.rows, H * hd), generator=torch.Generator().manual_seed(1)).to(DT[dtype])
            q[1, 3], q[2, hd + 1] = float("nan"), float("inf")
            r = t.depth.index(-1)  # padding: nothing of it comes out
            q[r] = float("nan")
            got = _check(dev, H, 2, hd, dtype, t, 72, q=q)
            bad = torch.isnan(got).reshape(-1, H, hd)
            assert bool(bad[1, 0].all()) and bool(bad[2, 1].all()) and int(bad.sum()) == 2 * hd


# ------------------------------------------------------------------ append

@pytest.mark.parametrize("n_q,n_kv,hd,page,dtype,rot,inter,norm", [
    (4, 2, 128, 16, "f16", 128, False, True), (4, 2, 128, 16, "f32", 128, False, True), (9, 1, 128, 32, "f16", 128, True, False),
    (3, 3, 64, 64, "f32", 32, True, False), (2, 1, 256, 128, "f32", 64, False, True), (5, 5, 80, 64, "f16", 40, False, False),
    (4, 4, 16, 16, "f16", 16, False, True), (4, 2, 32, 256, "f32", 8, True, True), (2, 2, 64, 16, "f16", 0, False, False),
])
@pytest.mark.parametrize("kind", ["small", "large"])
def test_append(dev, n_q, n_kv, hd, page, dtype, rot, inter, norm, kind):
    _case(f"append of {kind} trees {n_q}/{n_kv}/{hd} page {page} {dtype} rot {rot}")
    t = T.Trees(_trees(kind, hd), page, hd, pad=2)
    b, dt = t.batch, DT[dtype]
    g = torch.Generator().manual_seed(page)
    qkv = torch.randn((b.rows, (n_q + 2 * n_kv) * hd), generator=g).to(dt)
    cache = P.random_cache(b.n_pages, n_kv, page, hd, 5)
    cs = torch.from_numpy(ops.rope_table(1e4, rot, int(max(b.kv_len)))) if rot else None
    wqk = torch.randn(2 * hd, generator=g) * 0.2 + 1.0 if norm else None
    dc = _cache_on(cache, dev)
    table, start, length, depth = t.tensors(dev)
    out = torch.full((b.rows, n_q * hd), 7.0, dtype=dt, device=dev)
    ops.qk_norm_rope_tree_paged(qkv.to(dev), n_q, dc, table, start, length, depth, None if cs is None else cs.to(dev), 1e-6,
                                wqk=None if wqk is None else wqk.to(dev), interleaved=inter, q_out=out)
    torch.cuda.synchronize()
    got_q, parts = out.cpu().double().reshape(b.rows, n_q, hd), _parts(dc)
    values = ({}, {})
    for row, s, pos, pg, slot in b.places():
        n, total = b.seqs[s]
        if t.depth[row] < 0:
            assert bool((got_q[row] == 7.0).all())
            continue
        x = qkv[row].double().reshape(n_q + 2 * n_kv, hd)
        qk, v = x[: n_q + n_kv], x[n_q + n_kv:]
        if wqk is not None:
            w = wqk.double().reshape(2, hd)
            qk = qk / torch.sqrt(qk.square().mean(-1, keepdim=True) + 1e-6) * torch.cat([w[:1].expand(n_q, hd), w[1:].expand(n_kv, hd)])
        y, z = P.turned(qk, cs, total - n + t.depth[row], rot, inter)
        bar = 8 * U * z[:n_q] + (H16 * y[:n_q].abs() + 2.0 ** -25 if dtype == "f16" else 0.0)
        assert float(((got_q[row] - y[:n_q]).abs() - bar).max()) <= 0, row
        values[0].setdefault(pg, {})[slot] = (y[n_q:], z[n_q:])
        values[1].setdefault(pg, {})[slot] = (v, v.abs())
    assert bool((got_q[int(b.row_start[-1]):] == 7.0).all())
    firsts = {int(b.table[s, (total - n) // page]): (total - n) % page for s, (n, total) in enumerate(b.seqs) if n}
    for which in range(2):
        codes, scales = parts[which], parts[2 + which]
        for pg in range(b.n_pages):
            if pg not in values[which]:
                assert _same(codes[pg], cache[which][pg]) and torch.equal(scales[pg], cache[2 + which][pg]), f"page {pg} changed"
                continue
            at = values[which][pg]
            first = firsts.get(pg, 0)
            new = torch.stack([x for x, _ in at.values()]).to(dt).double().abs().amax((0, 2))
            want = torch.tensor([P.need_scale(float(m)) for m in new])
            if first:
                want = torch.maximum(want, cache[2 + which][pg])
            assert torch.equal(scales[pg], want), f"scales of page {pg}"
            for slot in range(page):
                if slot in at:
                    x, z = at[slot]
                    y = x / want.double()[:, None]
                    before = (8 * U * z + (H16 * x.abs() if dtype == "f16" and which == 0 else 0)) / want.double()[:, None]
                    bar = torch.maximum(y.abs() * 2.0 ** -4, torch.tensor(2.0 ** -10, dtype=torch.float64)) * (1 + 2.0 ** -20) + before * 1.07
                    assert bool(((codes[pg, :, slot].float().double() - y).abs() <= bar).all()), f"codes of {(pg, slot)}"
                else:
                    old = cache[which][pg, :, slot]
                    if slot < first:
                        old = (old.float() * (cache[2 + which][pg] / want)[:, None]).to(P.F8)
                    assert _same(codes[pg, :, slot], old), f"slot {(pg, slot)} changed"


def test_append_of_chains_is_that_of_rows_in_a_line(dev):
    """Bit for bit, the q columns of the rows themselves as output, rows at odd elements."""
    _case("append of chains")
    n_q, n_kv, hd = 4, 2, 64
    trees = [(list(range(-1, n - 1)), ctx) for n, ctx in ((1, 50), (17, 100), (64, 0), (0, 9), (50, 33))]
    for page, dtype in ((16, "f16"), (64, "f32")):
        t = T.Trees(trees, page, 4, pad=1)
        table, start, length, depth = t.tensors(dev)
        wide = torch.randn((t.rows, (n_q + 2 * n_kv) * hd + 5), generator=torch.Generator().manual_seed(3)).to(DT[dtype]).to(dev)
        cs = torch.from_numpy(ops.rope_table(1e4, hd, 200)).to(dev)
        got = []
        for tree in (False, True):
            cache, x = _cache_on(P.random_cache(t.batch.n_pages, n_kv, page, hd, 5), dev), wide.clone()
            rows = x[:, 3: 3 + (n_q + 2 * n_kv) * hd]
            args = (cs, 1e-6)
            if tree:
                ops.qk_norm_rope_tree_paged(rows, n_q, cache, table, start, length, depth, *args, q_out=rows[:, : n_q * hd])
            else:
                ops.qk_norm_rope_paged(rows, n_q, cache, table, start, length, *args, q_out=rows[:, : n_q * hd])
            torch.cuda.synchronize()
            got.append((x.cpu(), *_parts(cache)))
        assert all(_same(a, b) for a, b in zip(*got))


def test_append_places_past_the_angles_and_bad_depths(dev):
    """Rows at places without angles, with depths outside the tree, or of a length short of the rows are left alone."""
    _case("append of trees, bad places")
    n_q, n_kv, hd, page = 2, 1, 64, 16
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=dev)
    start, length = torch.tensor([0, 20, 30], dtype=torch.int32, device=dev), torch.tensor([28, 6], dtype=torch.int32, device=dev)
    depth = list(range(20)) + list(range(10))
    depth[3], depth[4], depth[5] = -1, 20, 2**31 - 1
    qkv = torch.randn((31, (n_q + 2 * n_kv) * hd), generator=torch.Generator().manual_seed(2)).to(dev)
    cache = _cache_on(P.random_cache(4, n_kv, page, hd, 4), dev)
    was = cache.k_pages.view(torch.uint8).clone()
    out = torch.full((31, n_q * hd), 7.0, device=dev)
    cs = torch.from_numpy(ops.rope_table(1e4, hd, 20)).to(dev)  # places 8 .. 19 of 8 .. 27
    ops.qk_norm_rope_tree_paged(qkv, n_q, cache, table, start, length, torch.tensor(depth + [0], dtype=torch.int32, device=dev), cs, 1e-6, q_out=out)
    torch.cuda.synchronize()
    written = (out != 7.0).any(1).cpu().tolist()
    want = [i < 12 and i not in (3, 4, 5) for i in range(20)] + [False] * 11
    assert written == want
    same = (cache.k_pages.view(torch.uint8) == was).all(3)[:, 0].cpu()
    for i in range(20):
        slot = 8 + i
        assert bool(same[slot // 16, slot % 16]) == (not want[i]), i
    assert bool(same[2:].all())


# ------------------------------------------------------------------ accept

def _drafts(trees, rng, agree=0.6):
    tokens, sampled = [], []
    for p, _ in trees:
        tok = rng.integers(0, 6, len(p)).tolist()  # (few tokens, so that siblings are often alike)
        got = rng.integers(-1, 6, len(p)).tolist()
        for i in range(len(p) - 1, 0, -1):
            if p[i] >= 0 and rng.random() < agree:
                got[p[i]] = tok[i]
        tokens += tok
        sampled += got
    return tokens, sampled


@pytest.mark.parametrize("sizes,most", [([1], 1), ([5, 0, 33, 1], 40), ([64, 65, 63], 64), ([200, 256, 257, 1000], 300), ([9] * 300, 9), ([40, 300], 3), ([40, 300], 1)])
def test_accept(dev, sizes, most):
    _case(f"accept, {sizes[:4]} rows, paths of {most}")
    rng = np.random.default_rng(len(sizes) + most)
    for turn in range(3):
        trees = [(T.random_parents(n, 1 if turn == 2 else 6, rng, n // 5) if n else [], int(rng.integers(0, 50))) for n in sizes]
        tokens, sampled = _drafts(trees, rng, 0.97 if turn else 0.6)
        start = np.cumsum([0] + [len(p) for p, _ in trees])
        cuda = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
        parents = [x for p, _ in trees for x in p]
        path, count, after, new_len = ops.accept_tree(cuda(tokens + [1]), cuda(sampled + [2]), cuda(parents + [-1]), cuda(start.tolist()),
                                                      cuda([ctx + len(p) for p, ctx in trees]), most)
        torch.cuda.synchronize()
        for s, (p, ctx) in enumerate(trees):
            a, b = start[s], start[s + 1]
            want, last = T.walk(p, tokens[a:b], sampled[a:b], most)
            assert path[s].tolist() == want + [-1] * (most - len(want))
            assert (count[s].item(), after[s].item(), new_len[s].item()) == (len(want), last, ctx + len(want))


def test_accept_odd_batches(dev):
    """Row ranges that run backwards or past the rows, lengths below the rows, parents that are nonsense."""
    _case("accept, odd batches")
    cuda = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    n = 40
    rng = np.random.default_rng(1)
    tok = cuda(rng.integers(0, 2, n).tolist())
    par = cuda(rng.integers(-2**31, 2**31, n).tolist())
    path, count, after, new_len = ops.accept_tree(tok, tok, par, cuda([-5, 30, 10, 2**31 - 1, 3]), cuda([7, -4, 2**31 - 1, 5]), 50)
    torch.cuda.synchronize()
    assert count.tolist()[1] == 0 and count.tolist()[3] == 0 and after[1].item() == -1 and bool((path[1] == -1).all())
    assert count[0].item() >= 1 and min(new_len.tolist()) >= 0


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 256, 257, 1000])
def test_accept_of_padding(dev, n):
    """Trees that are padding as a whole -- a first row that is no root, a length short of the rows -- have no path, no token
    after it and the length that they had before, though all their tokens agree; the trees between them are walked."""
    _case(f"accept of padding, {n} rows")
    chain = list(range(-1, n - 1))
    trees = [  # (parents, kv_len, rows of the path)
        (chain, n + 5, n), ([-2] * n, n + 7, 0), ([-2] + chain[1:], n + 30, 0), ([0] + chain[1:], n, 0), ([2**31 - 1] + chain[1:], n + 1, 0),
        ([-2**31] + [-1] * (n - 1), n + 2, 0), (chain, n - 1, 0), (chain, 0, 0), (chain, -2**31, 0), ([], 9, 0), (chain, n, n),
    ]
    cuda = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    start = np.cumsum([0] + [len(p) for p, _, _ in trees]).tolist()
    tokens = cuda([7] * start[-1])
    path, count, after, new_len = ops.accept_tree(tokens, tokens, cuda([x for p, _, _ in trees for x in p]), cuda(start), cuda([k for _, k, _ in trees]), n)
    torch.cuda.synchronize()
    for s, (p, length, rows) in enumerate(trees):
        assert path[s].tolist() == list(range(rows)) + [-1] * (n - rows), s
        assert (count[s].item(), after[s].item(), new_len[s].item()) == (rows, 7 if rows else -1, max(0, length - len(p)) + rows), s


def test_accept_odd_batches_by_the_rules(dev):
    """The batch of test_accept_odd_batches: what is no sequence, or shorter than its rows, has no path."""
    _case("accept, odd batches by the rules")
    cuda = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    n = 40
    rng = np.random.default_rng(1)
    tok = cuda(rng.integers(0, 2, n).tolist())
    par = cuda(rng.integers(-2**31, 2**31, n).tolist())
    path, count, after, new_len = ops.accept_tree(tok, tok, par, cuda([-5, 30, 10, 2**31 - 1, 3]), cuda([7, -4, 2**31 - 1, 5]), 50)
    torch.cuda.synchronize()
    # rows 0 .. 29 of a length of 7; none, of a length that is read as 0; rows 10 .. 39, of 2^30; none, of 5
    assert par[10].item() != -1
    assert count.tolist() == [0] * 4 and after.tolist() == [-1] * 4 and bool((path == -1).all())
    assert new_len.tolist() == [0, 0, 2**30 - 30, 5]


def test_captured_idle_place(dev):
    """A place of a captured step that is padding for some turns: its length and its tokens stay, the next tree goes on from
    them, and the text of the other places is as if it had never been idle."""
    _case("a captured step with a place that is idle for some turns")
    H, KV, hd, page, S, N = 4, 2, 64, 16, 2, 6
    table = torch.arange(S * 4, dtype=torch.int32, device=dev).reshape(S, 4)
    cs = torch.from_numpy(ops.rope_table(1e4, hd, 64)).to(dev)
    ints = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=dev)  # noqa: E731
    cache = ops.PagedKV.empty(S * 4, page, KV, hd, dev)
    start, length, depth, mask, parents, tokens, sampled = ints(S + 1), ints(S), ints(S * N), ints(S * N, 1), ints(S * N), ints(S * N), ints(S * N)
    rows = torch.zeros((S * N, (H + 2 * KV) * hd), dtype=torch.float16, device=dev)

    def fill(trees, seed):
        t = T.Trees(trees, page, 1, words=1)
        start.copy_(torch.from_numpy(t.batch.row_start))
        length.copy_(torch.from_numpy(t.batch.kv_len))
        depth.copy_(torch.tensor(t.depth, dtype=torch.int32))
        mask.copy_(t.mask())
        parents.copy_(torch.tensor(t.parents, dtype=torch.int32))
        rows.copy_(torch.randn(rows.shape, generator=torch.Generator().manual_seed(seed)).half())

    def step():
        q = ops.qk_norm_rope_tree_paged(rows, H, cache, table, start, length, depth, cs, 1e-6)
        out = ops.attention_tree_paged(q, cache, table, start, length, depth, mask, H)
        path, count, after, new_len = ops.accept_tree(tokens, sampled, parents, start, length, N)
        ops.keep_paged(cache, table, start, length, path, count)
        return out, path, count, after, new_len

    tree, idle = [-1, 0, 0, 2, -2, -2], [-2] * N  # (all tokens alike: the path is rows 0 and 1)
    lens = [0, 0]
    fill([(tree, 0), (tree, 0)], 0)
    stream = torch.cuda.Stream(dev)
    with torch.cuda.stream(stream):
        step()  # the workspace
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out, path, count, after, new_len = step()
    for turn, busy in enumerate([(1, 1), (1, 0), (0, 0), (1, 0), (1, 1)]):
        fill([(tree if b else idle, n) for b, n in zip(busy, lens)], 10 + turn)
        before = _parts(cache)
        graph.replay()
        torch.cuda.synchronize()
        assert count.tolist() == [2 * b for b in busy] and path.tolist() == [[0, 1, -1, -1, -1, -1] if b else [-1] * N for b in busy], turn
        assert after.tolist() == [0 if b else -1 for b in busy] and new_len.tolist() == [n + 2 * b for b, n in zip(busy, lens)], turn
        now = _parts(cache)
        for s in range(S):
            ids = table[s].tolist()
            if not busy[s]:
                assert all(_same(x[ids], y[ids]) for x, y in zip(before, now)), turn
                assert not bool(out[s * N: (s + 1) * N].any())
        lens = new_len.tolist()
    assert lens == [8, 4]


# ------------------------------------------------------------------ keep

def _paths(trees, rng, most, stay=0.1):
    path, count = torch.full((len(trees), most), -1, dtype=torch.int32), []
    for s, (p, _) in enumerate(trees):
        walk = [0] if p else []
        while p and len(walk) < most:
            below = [i for i, x in enumerate(p) if x == walk[-1] and i]
            if not below or rng.random() < stay:
                break
            walk.append(below[int(rng.integers(0, len(below)))])
        path[s, : len(walk)] = torch.tensor(walk, dtype=torch.int32)
        count.append(len(walk))
    return path, torch.tensor(count, dtype=torch.int32)


def _check_keep(dev, t, cache, path, count):
    dc = _cache_on(cache, dev)
    ops.keep_paged(dc, *t.batch.tensors(dev), path.to(dev), count.to(dev))
    torch.cuda.synchronize()
    want, got, b = T.keep(cache, t, path, count), _parts(dc), t.batch
    # Slots behind the path may hold anything.
    page, past = b.page, set()
    for s, (n, length) in enumerate(b.seqs):
        for j in range(max(0, length - n + max(0, min(int(count[s]), n))), b.table.shape[1] * page):
            id_ = int(b.table[s, j // page])
            if 0 <= id_ < b.n_pages:
                past.add((id_, j % page))
    for which in range(2):
        assert torch.equal(got[2 + which], want[2 + which]), "scales"
        for pg in range(b.n_pages):
            for slot in range(page):
                if (pg, slot) not in past:
                    x, y = got[which][pg, :, slot], want[which][pg, :, slot]
                    nan = torch.isnan(y.float())
                    assert torch.equal(torch.isnan(x.float()), nan) and torch.equal(x.float()[~nan], y.float()[~nan]), (which, pg, slot)
    return got


@pytest.mark.parametrize("n_kv,hd,page", [(2, 128, 16), (1, 64, 32), (3, 256, 16), (2, 80, 64), (1, 16, 16), (2, 32, 128), (1, 144, 256), (5, 48, 16)])
@pytest.mark.parametrize("kind", ["small", "large", "huge"])
def test_keep(dev, n_kv, hd, page, kind):
    """Trees of any size behind contexts that end anywhere in a page; scales that differ widely from page to page, so that
    a page's grows, and tokens that are rounded again."""
    _case(f"keep, {kind} trees, {n_kv}/{hd} page {page}")
    rng = np.random.default_rng(hd + page)
    for spread in (0.3, 3.0):
        trees = _trees(kind, hd)
        t = T.Trees(trees, page, hd)
        cache = P.random_cache(t.batch.n_pages, n_kv, page, hd, 5, spread)
        _check_keep(dev, t, cache, *_paths(trees, rng, max(len(p) for p, _ in trees), stay=0.02))


def test_keep_long_paths(dev):
    """Paths over many pages, every token but the first one or two slots on; each page is a source before it is written."""
    _case("keep, long paths")
    trees = [([-1] + [max(0, i - 2) for i in range(1, 500)], ctx) for ctx in (0, 5, 16, 1000)]
    for page, step in ((16, 1), (32, 2), (64, 3)):
        t = T.Trees(trees, page, page)
        cache = P.random_cache(t.batch.n_pages, 2, page, 64, 6, 2.0)
        n = (499 - 1) // step
        path = torch.tensor([[0] + [1 + step * (k + 1) if step > 1 else k + 2 for k in range(n - 1)]] * 4, dtype=torch.int32)
        path = path[:, : int((path[0] < 500).sum())].contiguous()
        _check_keep(dev, t, cache, path, torch.tensor([path.shape[1], 1, 40, path.shape[1]], dtype=torch.int32))


def test_keep_nothing_to_move(dev):
    """Paths that are in place, counts of 0 and below, past the rows and the path: nothing changes, or what is there does."""
    _case("keep, nothing to move")
    trees = [(list(range(-1, 9)), 20), (list(range(-1, 9)), 31), ([-1, 0, 0, 1], 7), ([-1, 0, 0, 1], 40)]
    t = T.Trees(trees, 16, 3)
    cache = P.random_cache(t.batch.n_pages, 2, 16, 64, 4)
    path = torch.tensor([list(range(10)), [0, 2, 4, 6, 8, 9, -1, -1, -1, -1], [0, 2] + [-1] * 8, [0, 2] + [-1] * 8], dtype=torch.int32)
    dc = _cache_on(cache, dev)
    ops.keep_paged(dc, *t.batch.tensors(dev), path.to(dev), torch.tensor([10, 0, 1, -3], dtype=torch.int32, device=dev))
    torch.cuda.synchronize()
    assert all(_same(a, b) for a, b in zip(_parts(dc), cache))
    _check_keep(dev, t, cache, path, torch.tensor([99, 2**31 - 1, 2, 10], dtype=torch.int32))


def test_keep_nan_bad_pages_and_odd_paths(dev):
    """NaN codes move as NaN and set no scale; tokens from or to pages outside the cache stay; entries that are not behind
    their slot, or past the tree, do not move; a length short of the rows moves nothing."""
    _case("keep, NaN, bad pages, odd paths")
    trees = [([-1] + [0] * 19, 12), ([-1] + [0] * 39, 30), ([-1] + [0] * 39, 5), ([-1] + [0] * 9, 8)]
    t = T.Trees(trees, 16, 5)
    b = t.batch
    cache = P.random_cache(b.n_pages, 2, 16, 64, 6, 2.0)
    for codes in cache[:2]:
        codes.view(torch.uint8)[int(b.table[0, 1]), 0, 3] = 0x7F
        codes.view(torch.uint8)[int(b.table[0, 1]), 1, 4, 7] = 0xFF
    b.table[1, 2] = b.n_pages + 3
    b.seqs[3], b.kv_len[3] = (10, 6), 6
    path = torch.tensor([[0, 7, 8, 9, 15, 19, -1, -1, -1], [0, 4, 9, 20, 25, 30, 35, 36, 37], [0, 1, 2, 40, 41, 1, 3, 2**31 - 1, -2**31],
                         [0, 2, 3, 4, 5, 6, 7, 8, 9]], dtype=torch.int32)
    _check_keep(dev, t, cache, path, torch.tensor([6, 9, 9, 9], dtype=torch.int32))


def test_keep_paths_of_any_stride(dev):
    _case("keep, strides")
    rng = np.random.default_rng(2)
    trees = _trees("large", 3)
    t = T.Trees(trees, 16, 3)
    cache = P.random_cache(t.batch.n_pages, 2, 16, 64, 5)
    path, count = _paths(trees, rng, 20)
    wide = torch.full((len(trees), 29), 3, dtype=torch.int32)
    wide[:, 4:24] = path
    a, b = _cache_on(cache, dev), _cache_on(cache, dev)
    ops.keep_paged(a, *t.batch.tensors(dev), path.to(dev), count.to(dev))
    ops.keep_paged(b, *t.batch.tensors(dev), wide.to(dev)[:, 4:24], count.to(dev))
    torch.cuda.synchronize()
    assert all(_same(x, y) for x, y in zip(_parts(a), _parts(b)))


# ------------------------------------------------------------------ together

class Drafter:
    """A toy model of one layer over the operators: rows' embeddings to qkv, attention to logits; trees of random tokens of
    which most agree with what the model would say."""

    def __init__(self, dev, H, KV, hd, vocab, seed):
        g = torch.Generator().manual_seed(seed)
        self.dev, self.H, self.KV, self.hd, self.vocab = dev, H, KV, hd, vocab
        self.embed = torch.randn((vocab, (H + 2 * KV) * hd), generator=g).half().to(dev)
        self.head = (torch.randn((H * hd, vocab), generator=g) * 0.3).to(dev)
        self.cs = torch.from_numpy(ops.rope_table(1e4, hd, 512)).to(dev)

    def logits(self, out):
        return out.float() @ self.head


def _step(m, cache, batch, tokens, depth, mask, parents, u, settings, most):
    table, start, length = batch
    q = ops.qk_norm_rope_tree_paged(m.embed[tokens.long()], m.H, cache, table, start, length, depth, m.cs, 1e-6)
    out = ops.attention_tree_paged(q, cache, table, start, length, depth, mask, m.H)
    logits = m.logits(out)
    sampled = ops.sample(logits, u, **settings)
    path, count, after, new_len = ops.accept_tree(tokens, sampled, parents, start, length, most)
    ops.keep_paged(cache, table, start, length, path, count)
    return q, out, logits, sampled, path, count, after, new_len


def test_pages_past_32_bits(dev):
    """A step over pages whose codes stand past 4 GiB of the cache's start: bit for bit the one over the same pages at its start."""
    _case("pages past 32 bits")
    H, KV, hd, page, first = 8, 2, 128, 16, (1 << 32) // 4096 + 3
    rng = np.random.default_rng(32)
    t = T.Trees([(T.random_parents(20, 5, rng, 2), 45), (T.random_parents(9, 3, rng), 0), (T.random_parents(40, 6, rng), 130)], page, 3)
    n = t.batch.n_pages
    small = _cache_on(P.random_cache(n, KV, page, hd, 4), dev)
    large = ops.PagedKV.empty(first + n, page, KV, hd, dev)
    assert large.k_pages[first:].data_ptr() - large.k_pages.data_ptr() > 1 << 32
    for x, y in zip((large.k_pages, large.v_pages, large.k_scales, large.v_scales), (small.k_pages, small.v_pages, small.k_scales, small.v_scales)):
        x[first:].view(torch.uint8).copy_(y.view(torch.uint8))
    g = torch.Generator().manual_seed(5)
    qkv = torch.randn((t.rows, (H + 2 * KV) * hd), generator=g).half().to(dev)
    table, start, length, depth = t.tensors(dev)
    cs = torch.from_numpy(ops.rope_table(1e4, hd, 300)).to(dev)
    count = torch.tensor([4, 3, 5], dtype=torch.int32, device=dev)
    path = torch.tensor([[0, 3, 7, 18, -1], [0, 2, 8, -1, -1], [0, 1, 20, 30, 39]], dtype=torch.int32, device=dev)
    got = []
    for cache, tab in ((small, table), (large, torch.where(table >= 0, table + first, table))):
        q = torch.zeros((t.rows, H * hd), dtype=torch.float16, device=dev)
        ops.qk_norm_rope_tree_paged(qkv, H, cache, tab, start, length, depth, cs, 1e-6, q_out=q)
        out = ops.attention_tree_paged(q, cache, tab, start, length, depth, t.mask().to(dev), H)
        ops.keep_paged(cache, tab, start, length, path, count)
        torch.cuda.synchronize()
        got.append((q.cpu(), out.cpu(), *(x[-n:].cpu() for x in (cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales))))
    assert all(_same(a, b) for a, b in zip(*got))
    # The pages before them are as an empty cache has them.
    assert bool((large.k_scales[:first] == 1).all()) and not bool(large.k_pages[:first].view(torch.uint8).any())


def test_speculative_steps(dev):
    """Five steps of three users, each operator on what the ones before it left, against 64 bits; and the text that comes
    out is the one that single greedy tokens give, as far as those are sure of themselves."""
    _case("speculative steps")
    H, KV, hd, page, vocab = 8, 2, 64, 16, 50
    m = Drafter(dev, H, KV, hd, vocab, 1)
    rng = np.random.default_rng(2)
    contexts = [21, 0, 40]
    table = np.array([[3, 0, 9, 1, 12, -1], [5, 2, 11, 13, 14, -1], [7, 4, 8, 10, 6, 15]], np.int32)
    cache = ops.PagedKV.empty(16, page, KV, hd, dev)
    cuda = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    # Prompts, by the append that is there.
    prompt = torch.from_numpy(rng.integers(0, vocab, sum(contexts))).to(dev)
    ops.qk_norm_rope_paged(m.embed[prompt], H, cache, torch.from_numpy(table).to(dev), cuda(np.cumsum([0] + contexts).tolist()), cuda(contexts),
                           m.cs, 1e-6)
    lens, roots = list(contexts), rng.integers(0, vocab, 3).tolist()
    for turn in range(5):
        trees = [(T.random_parents(int(rng.integers(1, 13)), 4, rng, int(rng.integers(0, 3))), n) for n in lens]
        t = T.Trees(trees, page, 1)
        t.batch.table, t.batch.n_pages = table, 16
        tokens = rng.integers(0, 6, t.rows)  # (few of them, so that some agree)
        tokens[t.batch.row_start[:-1]] = roots
        m.head[:, 6:] = -abs(m.head[:, 6:])  # (likewise)
        tab, start, length, depth = t.tensors(dev)
        before = _parts(cache)
        u = torch.rand(t.rows, generator=torch.Generator().manual_seed(turn))
        settings = {"temperature": torch.full((t.rows,), 0.0 if turn % 2 else 0.7, device=dev), "top_k": torch.full((t.rows,), 9, dtype=torch.int32, device=dev)}
        q, out, logits, sampled, path, count, after, new_len = _step(m, cache, (tab, start, length), cuda(tokens.tolist()), depth, t.mask().to(dev),
                                                                     cuda(t.parents), u.to(dev), settings, 13)
        torch.cuda.synchronize()
        # What the append left, by doing it alone; attention, samples, path and the kept tokens from there.
        again = _cache_on(before, dev)
        ops.qk_norm_rope_tree_paged(m.embed[torch.from_numpy(tokens).to(dev)], H, again, tab, start, length, depth, m.cs, 1e-6)
        torch.cuda.synchronize()
        held = _parts(again)
        want, a, s = T.attention(q.cpu(), held, t, H, float(np.float32(hd ** -0.5)))
        assert float(((out.cpu().double() - want).abs() - T.bar(want, a, s, max(lens) + 20, hd, "f16"))[: t.rows].max()) <= 0
        for r in range(t.rows):
            tok, near, _ = T.sample(logits[r].cpu().double().numpy(), float(u[r]), temperature=float(settings["temperature"][r]), top_k=9)
            assert sampled[r].item() == tok and near > 1e-9
        roots = []
        for i, (p, n) in enumerate(trees):
            x, y = int(t.batch.row_start[i]), int(t.batch.row_start[i + 1])
            walk, last = T.walk(p, tokens[x:y].tolist(), sampled[x:y].tolist(), 13)
            assert path[i, : len(walk)].tolist() == walk and count[i].item() == len(walk) and after[i].item() == last
            lens[i] = n + len(walk)
            assert new_len[i].item() == lens[i]
            roots.append(last)
        kept = T.keep(held, t, path.cpu(), count.cpu())
        now = _parts(cache)
        for i in range(3):
            for j in range(lens[i]):
                pg, slot = int(table[i, j // page]), j % page
                assert all(_same(x[pg, :, slot], y[pg, :, slot]) for x, y in zip(now[:2], kept[:2])), (turn, i, j)
        assert torch.equal(now[2], kept[2]) and torch.equal(now[3], kept[3])


def test_captured_steps_follow_the_batch(dev):
    """One captured step of all five operators, replayed as trees, lengths and tokens change on the device, against eager
    calls on a copy of the cache."""
    _case("a captured speculative step")
    H, KV, hd, page, vocab, S, N = 8, 2, 64, 16, 60, 3, 12
    m = Drafter(dev, H, KV, hd, vocab, 3)
    rng = np.random.default_rng(4)
    table = torch.arange(S * 8, dtype=torch.int32, device=dev).reshape(S, 8)
    cache, other = (ops.PagedKV.empty(S * 8, page, KV, hd, dev) for _ in range(2))
    ints = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=dev)  # noqa: E731
    start, length, depth, mask, parents, tokens = ints(S + 1), ints(S), ints(S * N), ints(S * N, 1), ints(S * N), ints(S * N)
    u = torch.zeros(S * N, device=dev)
    settings = {"temperature": torch.full((S * N,), 0.8, device=dev), "top_p": torch.full((S * N,), 0.9, device=dev)}
    lens = [0, 17, 30]

    def fill(turn):
        trees = [(T.random_parents(N - i, 4, rng, i) if turn != 2 or i else [-2] * N, n) for i, n in enumerate(lens)]
        t = T.Trees(trees, page, 1, words=1)
        start.copy_(torch.from_numpy(t.batch.row_start))
        length.copy_(torch.from_numpy(t.batch.kv_len))
        depth.copy_(torch.tensor(t.depth, dtype=torch.int32))
        mask.copy_(t.mask())
        parents.copy_(torch.tensor(t.parents, dtype=torch.int32))
        tokens.copy_(torch.from_numpy(rng.integers(0, 5, S * N).astype(np.int32)))
        u.copy_(torch.rand(S * N, generator=torch.Generator().manual_seed(turn)))

    def step(c):
        q = ops.qk_norm_rope_tree_paged(rows, H, c, table, start, length, depth, m.cs, 1e-6)
        out = ops.attention_tree_paged(q, c, table, start, length, depth, mask, H)
        sampled = ops.sample(out, u, **settings)  # (the rows themselves as logits: no product of a library in the graph)
        path, count, after, new_len = ops.accept_tree(tokens, sampled, parents, start, length, N)
        ops.keep_paged(c, table, start, length, path, count)
        return out, sampled, path, count, after, new_len

    rows = torch.zeros((S * N, (H + 2 * KV) * hd), dtype=torch.float16, device=dev)
    stream = torch.cuda.Stream(dev)
    fill(0)
    with torch.cuda.stream(stream):
        step(cache)  # the workspace
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        held = step(cache)
    for turn in range(4):
        fill(turn)
        rows.copy_(torch.randn(rows.shape, generator=torch.Generator().manual_seed(50 + turn)).half())
        for x, y in ((cache.k_pages, other.k_pages), (cache.v_pages, other.v_pages)):
            y.view(torch.uint8).copy_(x.view(torch.uint8))
        other.k_scales.copy_(cache.k_scales)
        other.v_scales.copy_(cache.v_scales)
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in held]
        want = step(other)
        torch.cuda.synchronize()
        assert all(_same(a, b) for a, b in zip(got, want)), turn
        assert all(_same(a, b) for a, b in zip(_parts(cache), _parts(other))), turn
        lens = got[5].tolist()
        assert lens == [a + b for a, b in zip([int(x) for x in (length - (start[1:] - start[:-1])).tolist()], got[3].tolist())]


def test_two_threads_and_another_stream(dev):
    _case("trees, two threads")
    H, KV, hd = 4, 2, 64
    jobs = []
    for i in range(2):
        t = T.Trees(_trees("large", 20 + i), 16, 21 + i)
        cache = _cache_on(P.random_cache(t.batch.n_pages, KV, 16, hd, 22), dev)
        q = torch.randn((t.rows, H * hd), generator=torch.Generator().manual_seed(i)).half().to(dev)
        jobs.append((q, cache, *t.tensors(dev), t.mask().to(dev), H))
    want = [ops.attention_tree_paged(*j).cpu() for j in jobs]
    got, failed = [None, None], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream(dev)):
                for _ in range(20):
                    out = ops.attention_tree_paged(*jobs[i])
                got[i] = out.cpu()
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [x.start() for x in threads]
    [x.join() for x in threads]
    assert not failed and all(torch.equal(a, b) for a, b in zip(got, want))


# ------------------------------------------------------------------ refusals

def test_refusals(dev):
    _case("trees, refusals")
    H, KV, hd = 4, 2, 64
    t = T.Trees([([-1, 0, 0], 20)], 16, 1)
    table, start, length, depth = t.tensors(dev)
    mask = t.mask().to(dev)
    cache = _cache_on(P.random_cache(t.batch.n_pages, KV, 16, hd, 2), dev)
    q = torch.zeros((3, H * hd), device=dev)
    qkv = torch.zeros((3, (H + 2 * KV) * hd), device=dev)
    path, count = torch.zeros((1, 3), dtype=torch.int32, device=dev), torch.ones(1, dtype=torch.int32, device=dev)
    att = lambda q=q, depth=depth, mask=mask, H=H, **kw: ops.attention_tree_paged(q, cache, table, start, length, depth, mask, H, **kw)  # noqa: E731
    app = lambda qkv=qkv, depth=depth, **kw: ops.qk_norm_rope_tree_paged(qkv, H, cache, table, start, length, depth, None, 1e-6, **kw)  # noqa: E731
    acc = lambda a=depth, b=depth, c=depth, d=start, e=length, n=3: ops.accept_tree(a, b, c, d, e, n)  # noqa: E731
    att(), app(), acc()
    bad = [
        lambda: att(depth=None), lambda: att(depth=depth[:2]), lambda: att(depth=depth.float()), lambda: att(depth=depth.cpu()),
        lambda: att(mask=mask[:2]), lambda: att(mask=mask.float()), lambda: att(mask=mask[0]), lambda: att(mask=mask.cpu()),
        lambda: att(mask=torch.zeros((3, 33), dtype=torch.int32, device=dev)), lambda: att(mask=mask[:, :0]),
        lambda: att(mask=torch.zeros((2, 3), dtype=torch.int32, device=dev).t()), lambda: att(H=3), lambda: att(q=q.double()),
        lambda: att(window=-1), lambda: att(softcap=-1.0), lambda: att(scale=float("nan")), lambda: att(out=q),
        lambda: att(out=torch.zeros((2, H * hd), device=dev)),
        lambda: app(depth=None), lambda: app(depth=depth[1:]), lambda: app(depth=depth.long()), lambda: app(qkv=qkv[:, 1:]),
        lambda: app(q_out=qkv[:, hd: hd + H * hd]),
        lambda: acc(a=depth[:2]), lambda: acc(b=depth[:2]), lambda: acc(c=depth.float()), lambda: acc(d=start[:1]), lambda: acc(n=0),
        lambda: acc(e=length.cpu()), lambda: acc(e=length[:0]),
        lambda: ops.keep_paged(cache, table, start, length, path.float(), count), lambda: ops.keep_paged(cache, table, start, length, path[0], count),
        lambda: ops.keep_paged(cache, table, start, length, path, count.long()), lambda: ops.keep_paged(cache, table, start, length, path[:, :0], count),
        lambda: ops.keep_paged(cache, table, start, length, path.cpu(), count), lambda: ops.keep_paged(cache, table, start[:1], length, path, count),
        lambda: ops.keep_paged(cache, table, start, length, cache.k_pages.view(torch.int32).reshape(-1)[:3][None], count),
        lambda: ops.keep_paged(cache, table, start, length, path, cache.k_scales.view(torch.int32).reshape(-1)[:1]),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(NekoError):
            f()
            print("accepted:", i)
    assert ops.attention_tree_paged(q[:0], cache, table, start, length, depth[:0], mask[:0], H).shape == (0, H * hd)
