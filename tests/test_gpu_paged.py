"""GPU tests of the paged 8-bit KV cache: neko_hip_qk_norm_rope_paged and neko_hip_attention_paged against a plain
evaluation in 64 bits (tests/paged_oracle.py).

Tolerances, derived from the operators' arithmetic. u = 2^-24, half a step of f32, and h = 2^-11, of f16.
  q (append): norm and rotation are at most eight f32 roundings of values of size z = |x_a| + |x_b| (the pair), and one
    of the result to its type: 8 u z + h |q| for f16.
  scales: equal. Codes: half a step of E4M3, 2^-4 |y| or 2^-10 where subnormal, of y = value / scale, besides what
    precedes it (8 u z and, in f16, the row's own rounding h |k|).
  attention: a weight's relative error is that of its exponent, the score, plus that of the exponential and of the
    weight's own two-part rounding (8 u together). A score is a sum of hd products, in any order: hd u s with s the
    largest sum of |q k|, some 4 u s for scaling, cap and bias. Relative errors e of all weights move the
    quotient by at most 2 e a, a = sum w |v| / sum w; the sums over n keys, 32 to a product, n / 32 + 64 roundings
    each, by 2 (n / 32 + 64) u a. f16 results are rounded once (h |out|), and f16 calls of many rows round each
    weight to f16 (h a).
"""
import numpy as np
import pytest
import torch

import paged_oracle as P
from nekochat_amd import NekoError, ops

pytestmark = pytest.mark.gpu

U, H16 = 2.0 ** -24, 2.0 ** -11
DT = {"f16": torch.float16, "f32": torch.float32}


def _case(msg):
    print(f"[case] {msg}", flush=True)


def _cache_on(cache, dev):
    return ops.PagedKV(*(t.clone().to(dev) for t in cache))


def _bytes(t):
    return t.cpu().view(torch.uint8)


def _rope(n_pos, rot):
    if not rot:
        return None
    return torch.from_numpy(ops.rope_table(1e4, rot, n_pos))


# ------------------------------------------------------------------ append

RAGGED = [(1, 1), (3, 3), (0, 0), (5, 40), (1, 33), (1, 17), (33, 70), (0, 20), (16, 32), (1, 96)]


def _check_append(dev, n_q, n_kv, hd, page, dtype, seqs, rot, inter, norm, seed, pad=2, extra=0, in_place=False, std=1.0):
    b = P.Batch(seqs, page, seed, pad=pad)
    dt = DT[dtype]
    g = torch.Generator().manual_seed(seed)
    qkv = (torch.randn((b.rows, (n_q + 2 * n_kv) * hd + extra), generator=g) * std).to(dt)
    cache = P.random_cache(b.n_pages, n_kv, page, hd, seed + 1)
    cs = _rope(max(b.kv_len) + 1, rot)
    wqk = torch.randn(2 * hd, generator=g) * 0.2 + 1.0 if norm else None
    dc = _cache_on(cache, dev)
    dq = qkv.to(dev)
    rows = dq[:, 1: 1 + (n_q + 2 * n_kv) * hd] if extra else dq
    src = qkv[:, 1: 1 + (n_q + 2 * n_kv) * hd] if extra else qkv
    out = rows[:, : n_q * hd] if in_place else torch.full((b.rows, n_q * hd), 7.0, dtype=dt, device=dev)
    before = out.cpu().clone()
    ops.qk_norm_rope_paged(rows, n_q, dc, *b.tensors(dev), None if cs is None else cs.to(dev), 1e-6,
                           wqk=None if wqk is None else wqk.to(dev), interleaved=inter, q_out=out)
    torch.cuda.synchronize()
    q, size, new, scales = P.append(src, n_q, n_kv, hd, b, cache, cs, 1e-6, wqk, inter, dt)
    got = out.cpu().double().reshape(b.rows, n_q, hd)
    written = ~torch.isnan(q[:, 0, 0])
    bar = 8 * U * size + (H16 * q.abs() + 2.0 ** -25 if dt == torch.float16 else 0.0)
    over = ((got - q).abs() - bar)[written].max()
    assert float(over) <= 0, f"q off by {float(over):.3g} past the bar"
    assert torch.equal(out.cpu()[~written], before[~written]), "rows of no sequence were written"
    if not in_place:
        assert torch.equal(dq.cpu(), qkv), "qkv was written"
    for which, (codes, had_codes, want, had) in enumerate(
            ((dc.k_pages, cache[0], new[0], cache[2]), (dc.v_pages, cache[1], new[1], cache[3]))):
        got_scale = (dc.k_scales, dc.v_scales)[which].cpu()
        assert torch.equal(got_scale, scales[which]), "scales"
        values = codes.cpu().float().double()
        touched = torch.zeros(codes.shape[:3:2], dtype=torch.bool)  # [page, slot]
        for (pg, slot), x in want.items():
            touched[pg, slot] = True
            y = x / got_scale[pg].double()[:, None]
            z = (8 * U * np.sqrt(2) * x.abs().amax(-1, keepdim=True) * 2 + (H16 * x.abs() if dt == torch.float16 and which == 0 else 0)) / got_scale[pg].double()[:, None]
            err = (values[pg, :, slot] - y).abs()
            assert bool((err <= torch.maximum(y.abs() * 2.0 ** -4, torch.tensor(2.0 ** -10, dtype=torch.float64)) * (1 + 2.0 ** -20) + z * 1.07).all()), f"codes of {(pg, slot)}"
        first = {}
        for pg, slot in want:
            first[pg] = min(first.get(pg, page), slot)
        for pg in range(b.n_pages):
            for slot in range(page):
                if touched[pg, slot]:
                    continue
                now = _bytes(codes[pg, :, slot])
                old = had_codes[pg, :, slot]
                if pg in first and slot < first[pg]:  # earlier tokens: the same values under the page's scale
                    ratio = (had[pg] / got_scale[pg])[:, None]
                    old = (old.float() * ratio).to(P.F8)
                assert torch.equal(now, old.view(torch.uint8)), f"slot {(pg, slot)} changed"
    return dc, out


@pytest.mark.parametrize("n_q,n_kv,hd,page,dtype,rot,inter,norm", [
    (4, 2, 128, 16, "f16", 128, False, True),    # the Qwen3 form
    (4, 2, 128, 16, "f32", 128, False, True),
    (9, 1, 128, 32, "f16", 128, True, False),    # more heads than a wave takes, one kv head
    (3, 3, 64, 32, "f32", 32, True, False),      # half of each head, interleaved
    (3, 3, 64, 64, "f16", 32, False, True),      # half of each head, in halves
    (2, 1, 256, 16, "f16", 256, False, True),
    (2, 1, 256, 128, "f32", 64, True, True),
    (5, 5, 80, 64, "f16", 40, False, False),     # lanes past the head
    (5, 5, 80, 16, "f32", 80, False, True),
    (4, 4, 16, 16, "f16", 16, False, True),
    (4, 2, 32, 256, "f32", 8, True, True),
    (4, 2, 48, 128, "f16", 0, False, True),      # no rotation
    (2, 2, 64, 16, "f16", 0, False, False),      # a plain store (GPT-2)
])
def test_append(dev, n_q, n_kv, hd, page, dtype, rot, inter, norm):
    _case(f"append {n_q}/{n_kv}/{hd} page {page} {dtype} rot {rot} inter {inter} norm {norm}")
    _check_append(dev, n_q, n_kv, hd, page, dtype, RAGGED, rot, inter, norm, seed=hd + page)


@pytest.mark.parametrize("page", [16, 64])
def test_append_unaligned_rows_and_in_place(dev, page):
    _case(f"append, rows at odd elements, page {page}")
    _check_append(dev, 4, 2, 128, page, "f16", RAGGED, 128, False, True, seed=5, extra=3)
    _check_append(dev, 4, 2, 64, page, "f32", RAGGED, 64, True, True, seed=6, extra=5)
    _case("append, q in place")
    _check_append(dev, 4, 2, 128, page, "f16", RAGGED, 128, False, True, seed=7, in_place=True)


def test_append_one_row_in_place_at_any_stride(dev):
    """One row has no stride to speak of: a view of it is its own q columns whatever strides the tensors name."""
    _case("append, one row in place, odd strides")
    n_q, n_kv, hd = 4, 2, 64
    width = (n_q + 2 * n_kv) * hd
    row = torch.randn(width, generator=torch.Generator().manual_seed(1)).half().to(dev)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)
    batch = (torch.zeros((1, 1), dtype=torch.int32, device=dev), i32(0, 1), i32(1))
    cs = _rope(4, hd).to(dev)
    want = ops.qk_norm_rope_paged(row[None], n_q, ops.PagedKV.empty(1, 16, n_kv, hd, dev), *batch, cs, 1e-6)
    for stride in (1, 5, width):
        x = row.clone().as_strided((1, width), (stride, 1))
        got = ops.qk_norm_rope_paged(x, n_q, ops.PagedKV.empty(1, 16, n_kv, hd, dev), *batch, cs, 1e-6, q_out=x[:, : n_q * hd])
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(x[:, n_q * hd:], row[None, n_q * hd:])


@pytest.mark.parametrize("n_seq,dtype", [(1, "f16"), (70, "f16"), (300, "f32")])
def test_append_many_sequences(dev, n_seq, dtype):
    """More sequences than one search step holds, idle places in rows, one sequence alone."""
    _case(f"append, {n_seq} sequences")
    rng = np.random.default_rng(n_seq)
    seqs = []
    for _ in range(n_seq):
        length = int(rng.integers(1, 40))
        seqs.append((int(rng.choice([0, 0, 1, 1, min(length, 2)])) if n_seq > 1 else 1, length))
    _check_append(dev, 2, 1, 64, 16, dtype, seqs, 64, False, True, seed=n_seq)


@pytest.mark.parametrize("n_seq", [65, 700])
def test_append_padded_batch(dev, n_seq):
    """Few sequences among many idle places, the rows padded to the places: searches that skip all of them."""
    _case(f"append, idle places, {n_seq}")
    seqs = [(0, 5)] * n_seq
    seqs[3], seqs[n_seq // 2], seqs[-1] = (1, 20), (2, 33), (1, 1)
    _check_append(dev, 2, 1, 64, 16, "f16", seqs, 64, False, True, seed=1, pad=n_seq - 4)
    seqs[-1], seqs[0] = (0, 0), (1, 17)
    _check_append(dev, 2, 1, 128, 32, "f32", seqs, 64, False, True, seed=2, pad=n_seq - 4)


def test_append_long_prompt(dev):
    """Slots of page segments instead of rows: one prompt of many pages beside single tokens."""
    _case("append, a long prompt")
    _check_append(dev, 2, 1, 64, 16, "f16", [(1, 5), (300, 300), (1, 64), (130, 137)], 64, False, True, seed=1)


def test_append_q_equals_the_unpaged_op(dev):
    """The q rows are those of qk_norm_rope bit for bit, for the layout that it knows."""
    _case("append against qk_norm_rope")
    n_q, n_kv, hd, rows = 8, 2, 128, 37
    g = torch.Generator().manual_seed(2)
    for dt in DT.values():
        qkv = torch.randn((rows, (n_q + 2 * n_kv) * hd), generator=g).to(dt).to(dev)
        cs, wqk = _rope(rows, hd).to(dev), (torch.randn(2 * hd, generator=g) * 0.1 + 1).to(dev)
        cache = ops.PagedKV.empty(4, 16, n_kv, hd, dev)
        table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device=dev)
        q = ops.qk_norm_rope_paged(qkv, n_q, cache, table, torch.tensor([0, rows], dtype=torch.int32, device=dev),
                                   torch.tensor([rows], dtype=torch.int32, device=dev), cs, 1e-6, wqk=wqk)
        want = ops.qk_norm_rope(qkv.clone(), n_q, n_kv, hd, cs, 1e-6, wqk=wqk)
        torch.cuda.synchronize()
        assert torch.equal(q, want[:, : n_q * hd])
        # ... and the k codes those of its k heads, which the page's scale brings to 448 or below.
        k = want[:, n_q * hd: (n_q + n_kv) * hd].float().reshape(rows, n_kv, hd)
        for j, page in enumerate((2, 0, 1)):
            part = k[16 * j: 16 * j + 16]
            for h in range(n_kv):
                s = P.need_scale(float(part[:, h].abs().max()))
                assert float(cache.k_scales[page, h]) == s
                assert torch.equal(cache.k_pages[page, h, : len(part)].view(torch.uint8), (part[:, h] / s).to(P.F8).view(torch.uint8))


@pytest.mark.parametrize("page", [16, 32])
def test_append_token_by_token(dev, page):
    """A sequence appended token by token, its scales raised on the way by ever larger tokens, ends with the scales of
    one appended at once, and with its codes but where a raised scale rounded a code of the subnormal range again."""
    _case(f"append token by token, page {page}")
    n_q, n_kv, hd, n = 2, 2, 64, 45
    g = torch.Generator().manual_seed(3)
    qkv = (torch.randn((n, (n_q + 2 * n_kv) * hd), generator=g) * torch.exp(torch.rand((n, 1), generator=g) * 6 - 3)).half().to(dev)
    table = torch.tensor([[3, 0, 2, 1]], dtype=torch.int32, device=dev)[:, : -(-n // page)].contiguous()
    caches = [ops.PagedKV.empty(4, page, n_kv, hd, dev) for _ in range(2)]
    cs = _rope(n, hd).to(dev)

    def go(cache, a, b):
        return ops.qk_norm_rope_paged(qkv[a:b], n_q, cache, table, torch.tensor([0, b - a], dtype=torch.int32, device=dev),
                                      torch.tensor([b], dtype=torch.int32, device=dev), cs, 1e-6)

    whole = go(caches[0], 0, n)
    parts = torch.cat([go(caches[1], i, i + 1) for i in range(n)])
    torch.cuda.synchronize()
    assert torch.equal(whole, parts)
    assert torch.equal(caches[0].k_scales, caches[1].k_scales) and torch.equal(caches[0].v_scales, caches[1].v_scales)
    for a, b in ((caches[0].k_pages, caches[1].k_pages), (caches[0].v_pages, caches[1].v_pages)):
        a, b = a.float(), b.float()
        # At most one more rounding to the subnormal step for each raise; values above 2^-6 keep theirs.
        off = (a - b).abs()
        assert float(off.max()) <= 2.0 ** -9 and float(off[a.abs() > 2.0 ** -5].max()) == 0.0
    # The same call again changes nothing.
    was = [t.clone() for t in (caches[0].k_pages.view(torch.uint8), caches[0].v_pages.view(torch.uint8), caches[0].k_scales)]
    go(caches[0], 30, n)
    torch.cuda.synchronize()
    assert torch.equal(was[0], caches[0].k_pages.view(torch.uint8)) and torch.equal(was[1], caches[0].v_pages.view(torch.uint8))
    assert torch.equal(was[2], caches[0].k_scales)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_append_not_finite_and_extreme(dev, dtype):
    """Infinities and NaN become NaN codes and leave the page's scale to the finite values; zeros, the smallest and the
    largest values."""
    _case(f"append, not finite, {dtype}")
    n_kv, hd, n = 1, 64, 6
    x = torch.randn((n, 3 * hd), generator=torch.Generator().manual_seed(1))
    x[1, hd + 3], x[2, hd + 5], x[3, 2 * hd + 1] = float("inf"), float("nan"), -float("inf")
    x[4, hd:] = 0.0
    dt = DT[dtype]
    x = x.to(dt)
    table = torch.zeros((1, 1), dtype=torch.int32, device=dev)

    def go(x):
        cache = ops.PagedKV.empty(1, 16, n_kv, hd, dev)
        m = x.shape[0]
        ops.qk_norm_rope_paged(x.to(dev), 1, cache, table, torch.tensor([0, m], dtype=torch.int32, device=dev),
                               torch.tensor([m], dtype=torch.int32, device=dev), None, 1e-6)
        torch.cuda.synchronize()
        return cache

    cache = go(x)
    for codes, scale, part in ((cache.k_pages, cache.k_scales, x[:, hd: 2 * hd]), (cache.v_pages, cache.v_scales, x[:, 2 * hd:])):
        part = part.double()
        s = P.need_scale(float(part[torch.isfinite(part)].abs().max()))
        assert float(scale[0, 0]) == s
        got = codes[0, 0, :n].float().cpu()
        assert torch.equal(torch.isnan(got), ~torch.isfinite(part))
        ok = torch.isfinite(part)
        assert torch.equal(got[ok], (part / s).float().to(P.F8).float()[ok])
    big = torch.finfo(dt).max
    for value, scale in ((0.0, 2.0 ** -64), (448.0, 1.0), (449.0, 2.0), (float(torch.finfo(dt).tiny), None), (big, None)):
        y = torch.zeros((1, 3 * hd), dtype=dt)
        y[0, hd:] = value
        cache = go(y)
        want = P.need_scale(value if value == 0 else float(y[0, hd]))
        assert scale is None or want == scale
        assert float(cache.k_scales[0, 0]) == want and float(cache.v_scales[0, 0]) == want
        got = cache.k_pages[0, 0, 0].float().cpu()
        if float(y[0, hd]) > 448 * 2.0 ** 64:
            assert bool(torch.isnan(got).all())
        else:
            assert torch.equal(got, (y[0, hd: 2 * hd].double() / want).float().to(P.F8).float())


def test_append_every_f16_value(dev):
    """Every finite f16 value under its own scale: the conversion's rounding is E4M3's, nearest even."""
    _case("append, every f16 value")
    hd, n = 64, 1024
    bits = torch.arange(n * hd, dtype=torch.int32).to(torch.int16).view(torch.float16).reshape(n, hd)
    x = torch.cat([torch.zeros_like(bits), bits, bits.flip(0)], 1).to(dev)
    cache = ops.PagedKV.empty(n // 16, 16, 1, hd, dev)
    ops.qk_norm_rope_paged(x, 1, cache, torch.arange(n // 16, dtype=torch.int32, device=dev)[None],
                           torch.tensor([0, n], dtype=torch.int32, device=dev), torch.tensor([n], dtype=torch.int32, device=dev), None, 0.0)
    torch.cuda.synchronize()
    for codes, scales, src in ((cache.k_pages, cache.k_scales, bits), (cache.v_pages, cache.v_scales, bits.flip(0))):
        y = src.double().reshape(-1, 16, hd) / scales.cpu().double()[:, :, None]
        got, ok = codes.float().cpu()[:, 0], torch.isfinite(y)
        assert torch.equal(got[ok], y.float().to(P.F8).float()[ok]) and bool(torch.isnan(got[~ok]).all())


def test_append_bad_pages_and_positions(dev):
    """Tokens whose page id is outside the cache, whose position is negative, past the table or past the angles are not
    stored, and nothing else changes; q rows within the angles are still written."""
    _case("append, bad pages and positions")
    n_q, n_kv, hd, page = 2, 1, 64, 16
    g = torch.Generator().manual_seed(9)
    n_pages = 5
    table = torch.tensor([[99, 1], [-7, 2], [3, 2**31 - 1], [0, 4]], dtype=torch.int32, device=dev)
    # sequence 0: page 0 is bad; 1: length short of the rows (positions -3 .. 1, page id bad); 2: a bad second page;
    # 3: past the table.
    starts = torch.tensor([0, 20, 25, 45, 85], dtype=torch.int32, device=dev)
    lens = torch.tensor([20, 2, 20, 40], dtype=torch.int32, device=dev)
    qkv = torch.randn((88, (n_q + 2 * n_kv) * hd), generator=g).to(dev)
    cache = _cache_on(P.random_cache(n_pages, n_kv, page, hd, 4), dev)
    was = [t.clone() for t in (cache.k_pages.view(torch.uint8), cache.k_scales)]
    cs = _rope(30, hd).to(dev)
    out = torch.full((88, n_q * hd), 7.0, device=dev)
    ops.qk_norm_rope_paged(qkv, n_q, cache, table, starts, lens, cs, 1e-6, q_out=out)
    torch.cuda.synchronize()
    untouched = (out == 7.0).all(1).cpu()
    want = torch.zeros(88, dtype=torch.bool)
    want[20:23] = True   # negative positions
    want[75:] = True     # sequence 3 from position 30 on (its rows stand at 0 .. 39), and rows of no sequence
    assert torch.equal(untouched, want)
    k = cache.k_pages.view(torch.uint8)
    assert torch.equal(k[2], was[0][2]), "page of no token"
    stored = {1: range(0, 4), 3: range(0, 16), 0: range(0, 16), 4: range(0, 14)}
    for pg in range(n_pages):
        for slot in range(page):
            same = torch.equal(k[pg, :, slot], was[0][pg, :, slot])
            assert same == (slot not in stored.get(pg, ())), (pg, slot)


# ------------------------------------------------------------------ attention

def _bar(out, a, s, n_keys, hd, dtype):
    e = (hd + 4) * U * s + 8 * U + (n_keys / 32 + 64) * U
    bar = 2 * e * a
    if dtype == "f16":
        bar = bar + H16 * out.abs() + 2.0 ** -25 + H16 * a
    return bar + 2 * U * out.abs()


def _wide(seqs, H, page):
    """Free places in a row of the page table: with so many the batch could be large, and its longer sequences run on
    the tiles of 128 rows; without, one of this size runs on the 16-row kernel alone."""
    return int(60e6) // (sum(n for n, _ in seqs) * H * page) + 1


def _check_attention(dev, H, KV, hd, page, dtype, seqs, seed, pad=2, cache=None, scale=None, what="", q=None, batch=None, unaligned=0, wide=False, **kw):
    b = batch or P.Batch(seqs, page, seed, pad=pad, slack=_wide(seqs, H, page) if wide else 1)
    dt = DT[dtype]
    g = torch.Generator().manual_seed(seed)
    if q is None:
        q = torch.randn((b.rows, H * hd), generator=g).to(dt)
    cache = cache or P.random_cache(b.n_pages, KV, page, hd, seed + 1)
    dc = _cache_on(cache, dev)
    scale = 1 / np.sqrt(hd) if scale is None else scale
    wide = torch.full((b.rows, H * hd + unaligned), 7.0, dtype=dt, device=dev)
    out = wide[:, unaligned // 2: unaligned // 2 + H * hd]
    dq = q.to(dev)
    if unaligned:
        dq = torch.cat([torch.zeros((b.rows, unaligned // 2), dtype=dt, device=dev), dq], 1)[:, unaligned // 2:]
    slopes = kw.get("slopes")
    ops.attention_paged(dq, dc, *b.tensors(dev), H, scale=scale, out=out, **{**kw, "slopes": None if slopes is None else slopes.to(dev)})
    torch.cuda.synchronize()
    want, a, s = P.attention(q, cache, b, H, float(np.float32(scale)), **kw)
    got = out.cpu().double()
    total = int(b.row_start[-1])
    assert torch.equal(got[total:], torch.full_like(got[total:], 7.0)), "rows of no sequence were written"
    got, want, a, s = got[:total], want[:total], a[:total], s[:total]
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    ok = ~torch.isnan(want)
    over = torch.where(ok, (got - want).abs() - _bar(want, a, s, max(n for _, n in b.seqs), hd, dtype), -1.0)
    rel = float((got - want)[ok].norm() / want[ok].norm().clamp(min=1e-300))
    print(f"{what or 'attention'} {H}/{KV}/{hd} page {page} {dtype}: rel {rel:.2e}, worst past the bar {float(over.max()):.2e}", flush=True)
    assert float(over.max()) <= 0
    if dtype == "f32":
        assert float(((got - want).abs() / (1 + a))[ok].max()) <= 2e-6 * max(1.0, float(s.max()) / 8)
    return got


DECODE = [(1, 1), (1, 16), (1, 17), (0, 0), (1, 200), (1, 333), (2, 65), (0, 9), (4, 130), (1, 700)]
PROMPT = [(70, 70), (1, 40), (130, 300), (5, 5), (0, 0), (33, 600)]


@pytest.mark.parametrize("H,KV,hd,page,dtype", [
    (8, 2, 128, 16, "f16"), (8, 2, 128, 32, "f32"), (6, 6, 64, 64, "f32"), (4, 4, 64, 16, "f16"), (8, 1, 256, 16, "f16"),
    (3, 1, 256, 128, "f32"), (5, 1, 80, 16, "f16"), (10, 2, 80, 64, "f32"), (2, 2, 16, 16, "f32"), (20, 1, 128, 256, "f16"),
    (4, 2, 48, 32, "f16"), (2, 1, 144, 32, "f32"), (7, 1, 32, 16, "f16"),
])
@pytest.mark.parametrize("form", ["decode", "prompt", "wide"])
def test_attention(dev, H, KV, hd, page, dtype, form):
    _case(f"attention {form} {H}/{KV}/{hd} page {page} {dtype}")
    _check_attention(dev, H, KV, hd, page, dtype, DECODE if form == "decode" else PROMPT, seed=hd + page, what=form, wide=form == "wide")


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("seqs", [[(1, 5000)], [(1, 1)], [(1, 4097), (1, 3)], [(3, 2050)], [(40, 4001)]])
def test_attention_split_keys(dev, seqs, dtype):
    """Few rows over long caches: keys split over workgroups and joined."""
    _case(f"attention, split keys, {seqs} {dtype}")
    _check_attention(dev, 8, 2, 128, 16, dtype, seqs, seed=11, what=str(seqs))
    _check_attention(dev, 8, 2, 128, 16, dtype, seqs, seed=11, what=str(seqs), wide=True)


def test_attention_many_sequences(dev):
    _case("attention, 150 sequences")
    rng = np.random.default_rng(4)
    seqs = [(int(rng.choice([0, 1, 1, 2])), int(rng.integers(2, 120))) for _ in range(150)]
    _check_attention(dev, 4, 2, 64, 16, "f32", seqs, seed=12)


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("n_seq", [64, 65, 513, 1100])
def test_attention_sequences_past_one_search(dev, n_seq, wide):
    """Batches that a search passes over in one step and in several, most places idle, some sequences long enough to be
    split, prompts and a padded end among them."""
    _case(f"attention, {n_seq} places, wide {wide}")
    rng = np.random.default_rng(n_seq)
    seqs = [(int(rng.random() < 0.2), int(rng.integers(1, 40))) for _ in range(n_seq)]
    for at, s in ((0, (1, 1500)), (9, (0, 0)), (n_seq // 2, (70, 300)), (n_seq // 2 + 1, (2, 900)), (n_seq - 3, (1, 1999)), (n_seq - 1, (0, 3))):
        seqs[at] = s
    _check_attention(dev, 4, 2, 64, 16, "f16", seqs, seed=13, pad=n_seq + 150 if wide else 7, wide=wide)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("rows,own,length,reach", [
    (2048, 150, 150, 4000), (2048, 150, 600, 4000), (2048, 1, 1100, 4000), (2048, 500, 500, 4000),  # the tiles
    (512, 1, 1100, 1104), (512, 33, 1104, 1104),                                                    # the 16-row kernel
])
def test_attention_one_sequence_in_a_buffer_of_many_rows(dev, rows, own, length, reach, dtype):
    """Rows behind the only sequence's, more than it has: the launch is planned by the call's rows."""
    _case(f"attention, {own} of {rows} rows, length {length}, {dtype}")
    H, KV, hd, page = 32, 8, 64, 16
    b = P.Batch([(own, length)], page, 17, pad=rows - own, slack=reach // page - -(-length // page))
    _check_attention(dev, H, KV, hd, page, dtype, b.seqs, 17, batch=b, what=f"{own} of {rows}")


def test_attention_smallest_cap(dev):
    """A cap whose inverse is past the largest number caps every score to next to nothing: all keys alike."""
    _case("attention, a cap of 1e-39")
    for seqs, wide in (([(1, 40), (3, 9)], False), ([(70, 90)], True)):
        H, KV, hd, page = 4, 2, 64, 16
        b = P.Batch(seqs, page, 3, slack=_wide(seqs, H, page) if wide else 1)
        cache = P.random_cache(b.n_pages, KV, page, hd, 4)
        q = torch.randn((b.rows, H * hd), generator=torch.Generator().manual_seed(5))
        q[0] = 0.0  # and scores of zero stay
        dc = _cache_on(cache, dev)
        got = ops.attention_paged(q.to(dev), dc, *b.tensors(dev), H, softcap=1e-39)
        torch.cuda.synchronize()
        want, a, s = P.attention(q, cache, b, H, 0.0)
        assert float(((got.cpu().double() - want).abs() - _bar(want, a, s, 90, hd, "f32")).max()) <= 0


@pytest.mark.parametrize("form", ["decode", "prompt", "wide"])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("kw", [dict(softcap=5.0), dict(window=1), dict(window=37), dict(window=10000), dict(slopes=True),
                                dict(softcap=2.0, window=50, slopes=True)])
def test_attention_cap_window_slopes(dev, kw, dtype, form):
    _case(f"attention {form} {kw} {dtype}")
    H, KV, hd = 6, 2, 64
    if kw.get("slopes"):
        kw = {**kw, "slopes": 2.0 ** -torch.arange(1, H + 1).float()}
    _check_attention(dev, H, KV, hd, 16, dtype, DECODE if form == "decode" else PROMPT, seed=21, what=form, wide=form == "wide", **kw)


@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0, 1e-20])
@pytest.mark.parametrize("seqs", [DECODE, PROMPT])
def test_attention_scales_of_scores(dev, scale, seqs):
    """A zero scale weights all keys alike, a negative one turns the order, a large one leaves one key."""
    _case(f"attention, scale {scale}")
    for wide in (False, True):
        _check_attention(dev, 4, 2, 64, 16, "f32", seqs, seed=31, scale=scale, wide=wide)
        _check_attention(dev, 4, 2, 128, 16, "f16", seqs, seed=32, scale=scale, wide=wide)


def _check_one_winner(dev, H, KV, hd, dtype, seqs, seed, cache, batch, q, scale, **kw):
    """Rows whose weights are 1 or nothing (one key seen, or scores further apart than their roundings), up to equal ones:
    no score's rounding reaches the result, so the bar is _bar's without them."""
    dc = _cache_on(cache, dev)
    slopes = kw.get("slopes")
    got = ops.attention_paged(q.to(dev), dc, *batch.tensors(dev), H, scale=scale,
                              **{**kw, "slopes": None if slopes is None else slopes.to(dev)})
    torch.cuda.synchronize()
    want, a, _ = P.attention(q, cache, batch, H, float(np.float32(scale)), **kw)
    got = got.cpu().double()
    assert bool(torch.isfinite(got).all()), "not finite"
    n = max(n for _, n in seqs)
    bar = 2 * (8 + n / 32 + 64) * U * a + (H16 * want.abs() + H16 * a + 2.0 ** -25 if dtype == "f16" else 0.0)
    over = float(((got - want).abs() - bar).max())
    assert over <= 0, f"off by {over:.3g} past the bar"


FORMS = {"decode": (DECODE, False), "prompt": (PROMPT, False), "wide": (PROMPT, True), "split": ([(1, 5000), (2, 40)], False)}


@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_one_key_of_any_score(dev, hd, dtype, form):
    """A row that sees one key gives its value, whatever the score: past 2^24 a score's rounding is a whole exponent."""
    _case(f"attention {form}, one key, hd {hd} {dtype}")
    seqs, wide = FORMS[form]
    H, KV, page = 4, 2, 16
    b = P.Batch(seqs, page, 23, slack=_wide(seqs, H, page) if wide else 1)
    cache = P.random_cache(b.n_pages, KV, page, hd, 24)
    q = torch.randn((b.rows, H * hd), generator=torch.Generator().manual_seed(25)).to(DT[dtype])
    for scale in (1e5, 1e6, -1e6, 1e7, 1e8, -1e9, 1e12):
        _check_one_winner(dev, H, KV, hd, dtype, seqs, 23, cache, b, q, scale, window=1)
    _check_one_winner(dev, H, KV, hd, dtype, seqs, 23, cache, b, q, 1e7, window=1, softcap=1e10, slopes=torch.full((H,), 3.0))


@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_scores_far_apart(dev, hd, dtype, form):
    """Many keys with scores of 1e7 to 1e11 of either sign, at least 1e6 apart or equal: the mean of the largest's values."""
    _case(f"attention {form}, scores far apart, hd {hd} {dtype}")
    seqs, wide = FORMS[form]
    H, KV, page = 4, 2, 16
    b = P.Batch(seqs, page, 26, slack=_wide(seqs, H, page) if wide else 1)
    g = torch.Generator().manual_seed(27)
    cache = list(P.random_cache(b.n_pages, KV, page, hd, 28))
    keys = torch.zeros(cache[0].shape)
    keys[..., 0] = 2.0 ** torch.randint(0, 5, keys.shape[:3], generator=g)  # score: q_0 times 1, 2, 4, 8 or 16
    cache[0], cache[2] = keys.to(P.F8), torch.ones_like(cache[2])
    cache[3] = torch.full_like(cache[3], 2.0 ** -7)  # (equal scores weigh alike where they are rounded alike)
    cache = tuple(cache)
    q = torch.zeros((b.rows, H, hd))
    q[..., 0] = torch.randint(1000, 2000, (b.rows, H), generator=g).float()
    q[::3] *= -1.0
    q = q.reshape(b.rows, -1).to(DT[dtype])
    for scale in (1e3, 1e4, -1e5, 1e6, 3e6):
        _check_one_winner(dev, H, KV, hd, dtype, seqs, 26, cache, b, q, scale)
    _check_one_winner(dev, H, KV, hd, dtype, seqs, 26, cache, b, q, 1e4, softcap=1e9, window=40)
    # A bias that favours far keys: q of zeros, scores slope * distance.
    _check_one_winner(dev, H, KV, hd, dtype, seqs, 26, cache, b, torch.zeros_like(q), 1.0, slopes=-torch.tensor([1e6, 3e6, 1e7, 1e8]))
    _check_one_winner(dev, H, KV, hd, dtype, seqs, 26, cache, b, torch.zeros_like(q), 1.0, slopes=-torch.tensor([1e6, 3e6, 1e7, 1e8]), window=20)


@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_attention_rows_beside_large_scores(dev, dtype, form):
    """Rows of ordinary scores are as exact as ever beside rows of huge ones, which stay within their values."""
    _case(f"attention {form}, rows beside large scores, {dtype}")
    seqs, wide = FORMS[form]
    H, KV, hd, page = 4, 2, 128, 16
    b = P.Batch(seqs, page, 29, slack=_wide(seqs, H, page) if wide else 1)
    cache = P.random_cache(b.n_pages, KV, page, hd, 30)
    q = torch.randn((b.rows, H, hd), generator=torch.Generator().manual_seed(31))
    big = torch.rand((b.rows, H, 1), generator=torch.Generator().manual_seed(32)) < 0.4
    q = torch.where(big, q * 1e4, q * 1e-3).reshape(b.rows, -1).to(DT[dtype])
    dc = _cache_on(cache, dev)
    got = ops.attention_paged(q.to(dev), dc, *b.tensors(dev), H, scale=1e3)
    torch.cuda.synchronize()
    want, a, s = P.attention(q, cache, b, H, 1e3)
    got, big = got.cpu().double(), big.expand(-1, -1, hd).reshape(b.rows, -1)
    assert bool(torch.isfinite(got).all())
    most = float((cache[1].float() * cache[3][..., None, None]).abs().max())
    over = torch.where(big, got.abs() - 1.01 * most, (got - want).abs() - _bar(want, a, s, max(n for _, n in seqs), hd, dtype))
    assert float(over.max()) <= 0


@pytest.mark.parametrize("seqs", [DECODE, PROMPT, [(1, 3), (1, 5), (7, 9)]])
def test_attention_f16_weights_of_few_rows_are_not_rounded(dev, seqs):
    """f16 calls on the 16-row kernel keep 24 bits of each weight: f32's bar and the result's own rounding, where values
    cancel. Weights of one f16 miss it: near-equal scores, so that nothing else is large, and sums near zero beside a."""
    _case(f"attention, f16 weights, {len(seqs)} sequences")
    H, KV, hd, page = 8, 2, 64, 16
    b = P.Batch(seqs, page, 33)
    cache = P.random_cache(b.n_pages, KV, page, hd, 34)
    q = torch.randn((b.rows, H * hd), generator=torch.Generator().manual_seed(35)).half()
    got = ops.attention_paged(q.to(dev), _cache_on(cache, dev), *b.tensors(dev), H, scale=0.02)
    torch.cuda.synchronize()
    want, a, s = P.attention(q, cache, b, H, float(np.float32(0.02)))
    bar = _bar(want, a, s, max(n for _, n in seqs), hd, "f32") + H16 * want.abs() + 2.0 ** -25
    assert float(((got.cpu().double() - want).abs() - bar).max()) <= 0


@pytest.mark.parametrize("seqs,wide", [(DECODE, False), (PROMPT, False), (PROMPT, True)])
def test_attention_pages_of_far_apart_scales(dev, seqs, wide):
    """Value pages whose scales lie 2^50 apart, each row's result as exact as if they did not; keys likewise small."""
    _case("attention, far apart scales")
    b = P.Batch(seqs, 16, 41, slack=_wide(seqs, 4, 16) if wide else 1)
    cache = P.random_cache(b.n_pages, 2, 16, 64, 42)
    e = torch.from_numpy(np.random.default_rng(1).integers(-25, 26, (b.n_pages, 2)).astype(np.float32))
    cache = (cache[0], cache[1], cache[2] * 2.0 ** -3, cache[3] * torch.exp2(e))
    for dtype in ("f32", "f16"):
        if dtype == "f16":
            cache = (cache[0], cache[1], cache[2], cache[3] * 2.0 ** -20)
        _check_attention(dev, 4, 2, 64, 16, dtype, seqs, seed=41, cache=cache, batch=b)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_attention_unaligned_rows(dev, dtype):
    _case(f"attention, rows at odd elements, {dtype}")
    for seqs, wide in ((DECODE, False), (PROMPT, False), (PROMPT, True)):
        _check_attention(dev, 4, 2, 64, 32, dtype, seqs, seed=51, unaligned=6, wide=wide)


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("window", [0, 30])
@pytest.mark.parametrize("hd,dtype", [(64, "f32"), (128, "f16"), (128, "f32"), (256, "f32"), (80, "f16")])
def test_attention_nan_where_it_is_seen_only(dev, hd, dtype, window, wide):
    """NaN in a cached token, key or value, reaches the rows that see it -- a value's only its own dimension -- and no
    others; free slots, pages of others and slots past the length may hold anything."""
    _case(f"attention, NaN tokens, hd {hd} {dtype} window {window}")
    seqs = [(1, 50), (6, 75), (90, 90), (3, 40), (1, 120)]
    page, KV = 16, 2
    b = P.Batch(seqs, page, 61, slack=_wide(seqs, 4, page) if wide else 1)
    cache = P.random_cache(b.n_pages, KV, page, hd, 62)
    kb, vb = cache[0].view(torch.uint8), cache[1].view(torch.uint8)
    for pg in b.free:
        kb[pg], vb[pg] = 0x7F, 0xFF
    for s, (_, length) in enumerate(seqs):
        if length % page:
            kb[b.table[s, length // page], :, length % page:] = 0xFF
            vb[b.table[s, length // page], :, length % page:] = 0x7F

    def at(s, j):
        return int(b.table[s, j // page]), j % page

    pg, slot = at(1, 72)  # of positions 69 .. 74
    vb[pg, 0, slot, 5] = 0x7F
    pg, slot = at(2, 33)
    vb[pg, 1, slot, hd - 1] = 0xFF
    vb[pg, 1, slot, 0] = 0x7F
    pg, slot = at(2, 60)
    kb[pg, 0, slot, 3] = 0x7F
    pg, slot = at(3, 39)
    vb[pg, :, slot] = 0x7F
    got = _check_attention(dev, 4, KV, hd, page, dtype, seqs, 63, cache=cache, batch=b, window=window)
    assert bool(torch.isnan(got).any()) and not bool(torch.isnan(got[0]).any())


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_attention_not_finite_queries(dev, dtype):
    """NaN and infinities in q reach their own head's row alone."""
    _case(f"attention, q not finite, {dtype}")
    for seqs, wide in (([(1, 60), (5, 40)], False), ([(80, 80)], False), ([(80, 80)], True)):
        b = P.Batch(seqs, 16, 71, slack=_wide(seqs, 4, 16) if wide else 1)
        H, hd = 4, 64
        q = torch.randn((b.rows, H * hd), generator=torch.Generator().manual_seed(1)).to(DT[dtype])
        q[1, 3] = float("nan")
        q[2, hd + 1] = float("inf")
        got = _check_attention(dev, H, 2, hd, 16, dtype, seqs, 72, batch=b, q=q)
        bad = torch.isnan(got).reshape(-1, H, hd)
        assert bool(bad[1, 0].all()) and bool(bad[2, 1].all()) and int(bad.sum()) == 2 * hd


def test_attention_bad_pages_and_empty_rows(dev):
    """Pages outside the cache hold nothing; rows that see nothing -- all pages bad, a negative position -- give zeros."""
    _case("attention, bad pages, empty rows")
    H, KV, hd, page = 4, 2, 64, 16
    for n, wide in ((1, False), (40, False), (40, True)):
        seqs = [(n, 60), (n, 50), (1, 20), (2, 20)]
        b = P.Batch(seqs, page, 81, slack=_wide(seqs, H, page) if wide else 1)
        b.table[0, 1] = b.n_pages + 5
        b.table[1, :] = -1
        b.table[2, 1] = -2**31
        got = _check_attention(dev, H, KV, hd, page, "f32", seqs, 82, batch=b)
        assert bool((got[n: 2 * n] == 0).all())
    # A length short of the rows: positions -3 .. 2; and one past the table's reach.
    for rows in (6, 40):
        cache = P.random_cache(3, KV, page, hd, 5)
        dc = _cache_on(cache, dev)
        q = torch.randn((2 * rows, H * hd), generator=torch.Generator().manual_seed(3)).to(dev)
        table = torch.tensor([[0, 1], [2, 1]], dtype=torch.int32, device=dev)
        out = ops.attention_paged(q, dc, table, torch.tensor([0, rows, 2 * rows], dtype=torch.int32, device=dev),
                                  torch.tensor([3, 32 + rows], dtype=torch.int32, device=dev), H)
        torch.cuda.synchronize()
        assert bool((out[: rows - 3] == 0).all()) and bool((out[rows - 3:] != 0).any(1).all())
        # Rows past the reach (positions 32 ..) see its 32 keys: those of a sequence of 32 that asks with them.
        want = ops.attention_paged(q[rows:].reshape(rows, -1).contiguous(), dc, table[1:].expand(rows, 2).contiguous(),
                                   torch.arange(rows + 1, dtype=torch.int32, device=dev),
                                   torch.full((rows,), 32, dtype=torch.int32, device=dev), H)
        torch.cuda.synchronize()
        assert float((out[rows:] - want).abs().max()) <= 4e-6


def test_attention_cache_past_4_gib(dev):
    """Pages whose bytes lie past 2^32 from the cache's start."""
    _case("a cache past 4 GiB")
    KV, hd, page = 8, 128, 64
    n_pages = (1 << 32) // (KV * hd * page) + 100
    b = P.Batch([(3, 130)], page, 91, free=1)
    cache = P.random_cache(b.n_pages, KV, page, hd, 92)
    big = ops.PagedKV(*(torch.empty((n_pages, KV, page, hd), dtype=torch.uint8, device=dev).view(P.F8) for _ in range(2)),
                      *(torch.ones((n_pages, KV), device=dev) for _ in range(2)))
    shift = n_pages - b.n_pages
    for i in range(b.n_pages):
        big.k_pages[shift + i].view(torch.uint8).copy_(cache[0][i].view(torch.uint8))
        big.v_pages[shift + i].view(torch.uint8).copy_(cache[1][i].view(torch.uint8))
    big.k_scales[shift:], big.v_scales[shift:] = cache[2].to(dev), cache[3].to(dev)
    small = _cache_on(cache, dev)
    table, start, length = b.tensors(dev)
    far = torch.where(table >= 0, table + shift, table)
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn((b.rows, (16 + 2 * KV) * hd), generator=g).half().to(dev)
    cs = _rope(200, hd).to(dev)
    outs = []
    for c, t in ((small, table), (big, far)):
        q = ops.qk_norm_rope_paged(qkv, 16, c, t, start, length, cs, 1e-6)
        outs.append(ops.attention_paged(q, c, t, start, length, 16))
    torch.cuda.synchronize()
    assert torch.equal(outs[0], outs[1])
    for i in range(b.n_pages):
        assert torch.equal(big.k_pages[shift + i].view(torch.uint8), small.k_pages[i].view(torch.uint8))


# ------------------------------------------------------------------ together

def _serve(dev, cache, batch_of, qkv_of, steps, H, KV, hd, cs, wqk):
    outs = []
    for i in range(steps):
        t = batch_of(i)
        q = ops.qk_norm_rope_paged(qkv_of(i), H, cache, *t, cs, 1e-6, wqk=wqk)
        outs.append(ops.attention_paged(q, cache, *t, H))
    return outs


def test_serving_run(dev):
    """Two prompts in chunks and three decode steps, append and attention in turn; every step against 64 bits on the
    cache as it stands, and near attention over the f16 cache of the unquantised path."""
    _case("a serving run")
    H, KV, hd, page = 8, 2, 128, 16
    g = torch.Generator().manual_seed(1)
    cs, wqk = _rope(200, hd), torch.randn(2 * hd, generator=g) * 0.1 + 1
    table = np.array([[4, 9, 2, 7, 0, 11, -1], [1, 8, 3, -1, -1, -1, -1]], np.int32)
    cache = ops.PagedKV.empty(12, page, KV, hd, dev)
    kc = [torch.zeros((200, KV * hd), dtype=torch.float16, device=dev) for _ in range(2)]
    vc = [torch.zeros((200, KV * hd), dtype=torch.float16, device=dev) for _ in range(2)]
    lens = [0, 0]
    for new in ([50, 20], [27, 0], [1, 1], [1, 1], [1, 4]):
        qkv = torch.randn((sum(new), (H + 2 * KV) * hd), generator=g).half().to(dev)
        lens = [a + n for a, n in zip(lens, new)]
        b = P.Batch([(n, a) for n, a in zip(new, lens)], page, 1)
        b.table, b.n_pages = table, 12
        t = b.tensors(dev)
        q = ops.qk_norm_rope_paged(qkv, H, cache, *t, cs.to(dev), 1e-6, wqk=wqk.to(dev))
        out = ops.attention_paged(q, cache, *t, H)
        torch.cuda.synchronize()
        now = tuple(x.cpu() for x in (cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales))
        want, a, s = P.attention(q.cpu(), now, b, H, float(np.float32(1 / np.sqrt(hd))))
        assert float(((out.cpu().double() - want).abs() - _bar(want, a, s, max(lens), hd, "f16")).max()) <= 0
        at = 0
        for i, n in enumerate(new):
            if n:
                rows = qkv[at: at + n].clone()
                ops.qk_norm_rope_kv(rows, H, KV, hd, cs.to(dev), 1e-6, kc[i], vc[i], wqk=wqk.to(dev), pos0=lens[i] - n)
                full = ops.attention(rows[:, : H * hd], kc[i], vc[i], H, KV, hd, pos0=lens[i] - n)
                # 8 bits: each code within 2^-4 of its value, weights' exponents within 2^-4 |scores|: some percent.
                rel = float((out[at: at + n].float() - full.float()).norm() / full.float().norm())
                assert rel < 0.15, rel
            at += n


def test_captured_decode_follows_growing_lengths(dev):
    """One captured graph of append and attention, replayed as the lengths grow on the device, against eager calls;
    eager work of the same context between the replays."""
    _case("captured decode")
    H, KV, hd, page, S = 8, 2, 64, 16, 5
    g = torch.Generator().manual_seed(8)
    n_pages, width = 60, 10
    table = torch.randperm(n_pages, generator=g)[: S * width].reshape(S, width).int().to(dev)
    start = torch.arange(S + 1, dtype=torch.int32, device=dev)
    first = torch.tensor([3, 130, 15, 31, 64], dtype=torch.int32, device=dev)
    init = P.random_cache(n_pages, KV, page, hd, 9)
    cs = _rope(200, hd).to(dev)
    steps = [torch.randn((S, (H + 2 * KV) * hd), generator=g).half().to(dev) for _ in range(6)]

    eager = _cache_on(init, dev)
    want = []
    for i, x in enumerate(steps):
        length = first + i
        q = ops.qk_norm_rope_paged(x, H, eager, table, start, length, cs, 1e-6)
        want.append(ops.attention_paged(q, eager, table, start, length, H))
    torch.cuda.synchronize()

    cache, x, length = _cache_on(init, dev), torch.empty_like(steps[0]), first.clone()
    q, out = torch.zeros((S, H * hd), dtype=torch.float16, device=dev), torch.zeros((S, H * hd), dtype=torch.float16, device=dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.qk_norm_rope_paged(x, H, cache, table, start, length, cs, 1e-6, q_out=q)
        ops.attention_paged(q, cache, table, start, length, H, out=out)
    for i, rows in enumerate(steps):
        x.copy_(rows)
        length.copy_(first + i)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i]), f"replay {i}"
        ops.attention_paged(q, eager, table, start, first, H)  # the workspace is used in between
    assert torch.equal(cache.k_pages.view(torch.uint8), eager.k_pages.view(torch.uint8))
    assert torch.equal(cache.v_scales, eager.v_scales)


def test_captured_prompts_of_two_graphs(dev):
    """Chunks of prompts captured on the tiles and beside single tokens, in two graphs that share the context's workspace,
    replayed in turn with lengths and pages that change on the device; eager calls in between."""
    _case("two captured graphs")
    H, KV, hd, page = 8, 2, 64, 16
    g = torch.Generator().manual_seed(18)
    n_pages, width, chunk = 400, 6000, 130
    cs = _rope(2000, hd).to(dev)
    init = P.random_cache(n_pages, KV, page, hd, 19)
    # Graph 0: one sequence's chunk; graph 1: a chunk between two single tokens and an idle place.
    new = [[chunk], [1, chunk, 0, 1]]
    start = [torch.tensor(np.cumsum([0] + n), dtype=torch.int32, device=dev) for n in new]
    lengths = [[[chunk], [2 * chunk], [900]], [[700, chunk, 0, 33], [701, 1300, 0, 34], [17, 2 * chunk, 5, 1]]]

    def table(i, k):
        t = torch.full((len(new[i]), width), -1, dtype=torch.int32)
        order = torch.randperm(n_pages, generator=torch.Generator().manual_seed(10 * i + k))
        at = 0
        for s, n in enumerate(lengths[i][k]):
            used = -(-n // page)
            t[s, :used] = order[at: at + used].int()
            at += used
        return t.to(dev)

    rows = [[torch.randn((sum(n), (H + 2 * KV) * hd), generator=g).half().to(dev) for _ in range(3)] for n in new]

    def step(i, x, cache, t, length, q, out):
        ops.qk_norm_rope_paged(x, H, cache, t, start[i], length, cs, 1e-6, q_out=q)
        ops.attention_paged(q, cache, t, start[i], length, H, out=out)

    def buffers(i):
        return tuple(torch.zeros((sum(new[i]), H * hd), dtype=torch.float16, device=dev) for _ in range(2))

    len_of = lambda i, k: torch.tensor(lengths[i][k], dtype=torch.int32, device=dev)
    eager, want = _cache_on(init, dev), []
    for k in range(3):
        for i in range(2):
            q, out = buffers(i)
            step(i, rows[i][k], eager, table(i, k), len_of(i, k), q, out)
            want.append(out)
    torch.cuda.synchronize()

    cache = _cache_on(init, dev)
    held, graphs = [], []
    for i in range(2):
        x, t, length = torch.empty_like(rows[i][0]), table(i, 0), len_of(i, 0)
        q, out = buffers(i)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(i, x, cache, t, length, q, out)
        held.append((x, t, length, out))
        graphs.append(graph)
    for k in range(3):
        for i in range(2):
            x, t, length, out = held[i]
            x.copy_(rows[i][k])
            t.copy_(table(i, k))
            length.copy_(len_of(i, k))
            graphs[i].replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want[2 * k + i]), f"replay {k} of graph {i}"
            q, o = buffers(1 - i)
            ops.attention_paged(q, eager, table(1 - i, k), start[1 - i], len_of(1 - i, k), H, out=o)  # (the workspace, between)
    assert torch.equal(cache.k_pages.view(torch.uint8), eager.k_pages.view(torch.uint8))
    assert torch.equal(cache.v_pages.view(torch.uint8), eager.v_pages.view(torch.uint8))


def test_one_captured_graph_for_row_ranges_that_shrink(dev):
    """Graphs captured for a buffer of many rows, replayed as the one sequence of them fills fewer: on the tiles and on the
    16-row kernel, each replay as the eager call, eager calls in between."""
    _case("row ranges that shrink")
    H, KV, hd, page = 32, 8, 64, 16
    for rows, width, steps in ((2048, 250, [(2048, 2048), (500, 2600), (1, 2601), (64, 4000), (2048, 4000)]),
                               (512, 69, [(512, 600), (1, 1100), (40, 1104), (512, 1104)])):
        cache = _cache_on(P.random_cache(width, KV, page, hd, 1), dev)
        table = torch.randperm(width, generator=torch.Generator().manual_seed(2))[None].int().to(dev)
        q = torch.randn((rows, H * hd), generator=torch.Generator().manual_seed(3)).half().to(dev)
        start, length = (torch.zeros(n, dtype=torch.int32, device=dev) for n in (2, 1))
        call = lambda out: ops.attention_paged(q, cache, table, start, length, H, out=out)

        def set_to(n, total):
            start.copy_(torch.tensor([0, n], dtype=torch.int32))
            length.fill_(total)

        want = []
        for n, total in steps:
            set_to(n, total)
            want.append(call(torch.full_like(q, 7.0)))
            assert bool((want[-1][n:] == 7.0).all()) and bool((want[-1][:n] != 7.0).any(1).all())
        out = torch.empty_like(q)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call(out)
        for i in [1, 2, 0, 3, 1]:
            set_to(*steps[i])
            out.fill_(7.0)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want[i]), f"rows {steps[i]} of {rows}"
            call(torch.empty_like(q))


def test_two_threads(dev):
    """A context and a stream for each of two host threads, calls of both at once: split keys in each one's workspace."""
    _case("two threads")
    import threading

    H, KV, hd, page = 8, 2, 128, 16
    cases = []
    for i, seqs in enumerate(([(1, 5000), (1, 70)], [(2, 3000), (150, 200)])):
        b = P.Batch(seqs, page, 5 + i)
        dc, t = _cache_on(P.random_cache(b.n_pages, KV, page, hd, 6 + i), dev), b.tensors(dev)
        q = torch.randn((b.rows, H * hd), generator=torch.Generator().manual_seed(i)).to(dev)
        cases.append((q, dc, t, ops.attention_paged(q, dc, *t, H)))
    torch.cuda.synchronize()
    bad = []

    def work(case):
        try:
            q, dc, t, want = case
            with torch.cuda.stream(torch.cuda.Stream()):
                got = [ops.attention_paged(q, dc, *t, H) for _ in range(20)]
                torch.cuda.current_stream().synchronize()
            bad.extend(i for i, x in enumerate(got) if not torch.equal(x, want))
        except Exception as e:  # noqa: BLE001 -- reported below
            bad.append(e)

    threads = [threading.Thread(target=work, args=(c,)) for c in cases]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad, bad


def test_another_stream_and_prepared_calls(dev):
    _case("another stream, prepared calls")
    H, KV, hd = 8, 2, 128
    b = P.Batch([(1, 300), (2, 40), (70, 90)], 16, 3)
    cache = P.random_cache(b.n_pages, KV, 16, hd, 4)
    q = torch.randn((b.rows, H * hd), generator=torch.Generator().manual_seed(2)).to(dev)
    dc, t = _cache_on(cache, dev), b.tensors(dev)
    want = ops.attention_paged(q, dc, *t, H)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = ops.attention_paged(q, dc, *t, H)
    side.synchronize()
    assert torch.equal(got, want)
    out = torch.zeros_like(want)
    run, _ = ops.prepare(ops.attention_paged, q, dc, *t, H, out=out)
    for _ in range(3):
        out.zero_()
        run()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


# ------------------------------------------------------------------ refusals

@pytest.mark.parametrize("n_q", [0, -1, -8])
def test_append_refuses_heads_below_one(dev, n_q):
    _case(f"refusal of n_q {n_q}")
    cache, table = ops.PagedKV.empty(1, 16, 2, 64, dev), torch.zeros((1, 1), dtype=torch.int32, device=dev)
    start, length = torch.tensor([0, 1], dtype=torch.int32, device=dev), torch.ones(1, dtype=torch.int32, device=dev)
    with pytest.raises(NekoError):
        ops.qk_norm_rope_paged(torch.zeros((1, 512), device=dev), n_q, cache, table, start, length, None, 1e-6)


def test_refusals(dev):
    _case("refusals")
    H, KV, hd, page = 4, 2, 64, 16
    cache = ops.PagedKV.empty(4, page, KV, hd, dev)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)
    table, start, length = torch.zeros((1, 2), dtype=torch.int32, device=dev), i32(0, 1), i32(1)
    qkv = torch.zeros((1, (H + 2 * KV) * hd), device=dev)
    q = torch.zeros((1, H * hd), device=dev)
    cs = torch.zeros((8, hd), device=dev)
    good = dict(q=q, cache=cache, page_table=table, row_start=start, kv_len=length, n_head=H)
    ops.attention_paged(**good)
    for bad in (dict(n_head=3), dict(n_head=8), dict(page_table=table.long()), dict(row_start=i32(0)), dict(kv_len=i32(1, 1)),
                dict(kv_len=length.cpu()), dict(q=q.cpu()), dict(q=q.double()), dict(scale=float("nan")), dict(scale=float("inf")),
                dict(softcap=-1.0), dict(window=-1), dict(slopes=torch.zeros(2, device=dev)), dict(out=torch.zeros((1, 8), device=dev)),
                dict(out=q), dict(page_table=torch.zeros((1, 0), dtype=torch.int32, device=dev)),
                dict(page_table=torch.zeros((0, 2), dtype=torch.int32, device=dev), row_start=i32(0), kv_len=i32())):
        with pytest.raises(NekoError):
            ops.attention_paged(**{**good, **bad})
    good = dict(qkv=qkv, n_q=H, cache=cache, page_table=table, row_start=start, kv_len=length, cs=cs, eps=1e-6)
    ops.qk_norm_rope_paged(**good)
    for bad in (dict(n_q=5), dict(n_q=0), dict(cs=torch.zeros((8, 12), device=dev)), dict(cs=torch.zeros((8, 72), device=dev)),
                dict(cs=cs.half()), dict(wqk=torch.zeros(hd, device=dev)), dict(qkv=qkv.cpu()), dict(row_start=start.long()),
                dict(q_out=torch.zeros((1, 8), device=dev)), dict(q_out=qkv[:, hd: hd + H * hd])):
        with pytest.raises(NekoError):
            ops.qk_norm_rope_paged(**{**good, **bad})
    for shape in ((2, KV, 24, hd), (2, KV, 8, hd), (2, KV, 512, hd), (2, KV, 16, 40), (2, KV, 16, 272)):
        odd = ops.PagedKV.empty(*(shape[i] for i in (0, 2, 1, 3)), dev)
        with pytest.raises(NekoError):
            ops.attention_paged(torch.zeros((1, H * shape[3]), device=dev), odd, table, start, length, H)
    with pytest.raises(NekoError):
        ops.PagedKV(cache.k_pages, cache.v_pages[:2], cache.k_scales, cache.v_scales)
    with pytest.raises(NekoError):
        ops.PagedKV(cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales.half())
    twice = ops.PagedKV(cache.k_pages, cache.k_pages, cache.k_scales, cache.v_scales)
    with pytest.raises(NekoError):
        ops.attention_paged(q, twice, table, start, length, H)
    # No rows is nothing to do.
    none = ops.attention_paged(q[:0], cache, table, i32(0, 0), i32(0), H)
    assert none.shape == (0, H * hd)
    assert ops.qk_norm_rope_paged(qkv[:0], H, cache, table, i32(0, 0), i32(0), cs, 1e-6).shape == (0, H * hd)
