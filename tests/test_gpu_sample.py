"""GPU tests of neko_hip_sample against an evaluation in 64 bits (tests/tree_oracle.py).

Tolerance: the tokens are equal. The kernel's weights are e^x in double and so is its running sum: a row whose u falls nearer
to a border than V * 2^-44 of the sum could go either way. What top-p compares is a sum over bins of weights that are held to
2^-30 of themselves or better, and a total like it, 2^-28 of the sum at most: a cut nearer to a border than 2^-27 could be
before or after a token. The oracle says how near each was; in such rows, which random numbers hardly ever make, both sides
are right. Where all weights are 1 every sum is exact, and the tokens are equal however near.
"""
import threading

import numpy as np
import pytest
import torch

import tree_oracle as T
from nekochat_amd import NekoError, ops

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "f32": torch.float32}


def _case(msg):
    print(f"[case] {msg}", flush=True)


def _check(dev, x, u, exact_ties=False, **kw):
    """x: a CPU tensor of logits; kw: per-row settings, as CPU tensors. exact_ties: weights and sums that are whole numbers,
    whose borders are met exactly."""
    got = ops.sample(x.to(dev), u.to(dev), **{k: v.to(dev) for k, v in kw.items()})
    torch.cuda.synchronize()
    got = got.cpu().tolist()
    rows = x.float().double().numpy()
    for r in range(len(rows)):
        mine = {k: float(v[r]) if v.dtype != torch.int32 else int(v[r]) for k, v in kw.items()}
        want, near, near_p = T.sample(rows[r], float(u[r]), **mine)
        by, by_p = (x.shape[1] * 2.0 ** -44 if near <= x.shape[1] * 2.0 ** -44 else 0.0), (2.0 ** -27 if near_p <= 2.0 ** -27 else 0.0)
        if not exact_ties and (by or by_p):
            right = {T.sample(rows[r], float(u[r]), shift=i * by, shift_p=j * by_p, **mine)[0] for i in (-1, 1) for j in (-1, 1)}
            assert got[r] in right, f"row {r}: {got[r]}, not of {right}"
            continue
        assert got[r] == want, f"row {r}: {got[r]}, not {want} ({ {k: v[r].item() for k, v in kw.items()} }, u {float(u[r])})"
    return got


def _settings(rows, vocab, g, mode):
    f = lambda lo, hi: torch.rand(rows, generator=g) * (hi - lo) + lo  # noqa: E731
    kw = {"temperature": f(0.3, 1.7)}
    if mode in ("k", "all"):
        kw["top_k"] = torch.randint(1, max(2, min(vocab, 300)), (rows,), generator=g, dtype=torch.int32)
    if mode in ("p", "all"):
        kw["top_p"] = f(0.05, 0.999)
    if mode in ("min_p", "all"):
        kw["min_p"] = f(0.0, 0.3)
    return kw


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("vocab", [1, 2, 7, 63, 2047, 2049, 50257, 151936])
@pytest.mark.parametrize("mode", ["none", "k", "p", "min_p", "all"])
def test_sample(dev, vocab, dtype, mode):
    _case(f"sample, vocabulary {vocab} {dtype} {mode}")
    rows = 40 if vocab < 10000 else 6
    g = torch.Generator().manual_seed(vocab + len(mode))
    x = (torch.randn((rows, vocab), generator=g) * 3).to(DT[dtype])
    _check(dev, x, torch.rand(rows, generator=g), **_settings(rows, vocab, g, mode))


def test_sample_many_rows(dev):
    """So many rows that each is one workgroup's."""
    _case("sample, 1500 rows")
    g = torch.Generator().manual_seed(3)
    x = (torch.randn((1500, 5000), generator=g) * 2).half()
    _check(dev, x, torch.rand(1500, generator=g), **_settings(1500, 5000, g, "all"))


def test_sample_the_largest_vocabulary(dev):
    """As many tokens as a call takes, in more rows than one set of launches does at once: all rows' logits are alike, so a
    row's token is that of a call of its own.

    Which token's share of the running sum u falls into is checked to b = V 2^-44 / S + 2^-26 of the sum S (in weights of the
    largest): listed tokens' weights are rounded to units of 2^-44, by half of one each, and doubles' sums by less than 2^-40
    of S; the cut of top-p is within 2^-27 of S, by which the running sum moves and what u is compared with too."""
    _case("sample, vocabulary 2^24, 50 rows")
    g = torch.Generator().manual_seed(24)
    vocab, rows = 1 << 24, 50
    x = (torch.randn((1, vocab), generator=g) * 2).half()
    u = torch.rand(rows, generator=g)
    u[49] = u[46] = u[0]
    dx, l = x.to(dev).expand(rows, vocab).contiguous(), x[0].double().numpy()
    w = np.exp(l - l.max())
    order = np.argsort(-l, kind="stable")
    for kw in ({"top_p": 0.9}, {"top_k": 50, "top_p": 0.95}, {"min_p": 0.01}):
        make = lambda n: {k: torch.full((n,), v, dtype=torch.int32 if k == "top_k" else torch.float32).to(dev) for k, v in kw.items()}  # noqa: E731
        got = ops.sample(dx, u.to(dev), **make(rows)).tolist()
        print(kw, got[:4], flush=True)
        alone = []
        for r in range(rows):
            alone += ops.sample(dx[:1], u[r:r + 1].to(dev), **make(1)).tolist()
        assert got == alone and got[0] == got[46] == got[49]
        stays = order[: kw.get("top_k", vocab)]
        cum = np.cumsum(w[stays])
        if "top_p" in kw:
            stays = stays[: int(np.searchsorted(cum, float(np.float32(kw["top_p"])) * cum[-1])) + 1]
        stays = np.sort(stays[w[stays] >= float(np.float32(kw.get("min_p", 0.0)))])
        cum = np.cumsum(w[stays])
        for r, token in enumerate(got):
            at = int(np.searchsorted(stays, token))
            near = vocab * 2.0 ** -44 / cum[-1] + 2.0 ** -26
            before, after = (cum[at - 1] if at else 0.0) / cum[-1], (cum[at] if at < len(cum) else cum[-1]) / cum[-1]
            if at == len(stays) or stays[at] != token:  # (right at the cut)
                assert abs(after - before) <= near
                after = before
            assert before - near <= float(u[r]) <= after + near, (r, token, before, float(u[r]), after)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_sample_settings_that_cut_nothing(dev, dtype):
    """Settings at and past their ends, and not numbers."""
    _case(f"sample, settings that cut nothing or all, {dtype}")
    nan, inf = float("nan"), float("inf")
    k = [0, -5, 1000, 2**31 - 1, 1, 2, 999]
    p = [1.0, 2.0, nan, inf, 0.0, -1.0, 1e-30]
    m = [0.0, -1.0, nan, 1.0, 2.0, inf, 1e-30]
    t = [1.0, 0.0, -2.0, nan, inf, 1e-30, 1e30]
    g = torch.Generator().manual_seed(2)
    n = 7
    base = torch.randn((n, 1000), generator=g).to(DT[dtype])
    ints = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    u = torch.rand(n, generator=g)
    _check(dev, base, u, top_k=ints(k))
    _check(dev, base, u, top_p=torch.tensor(p))
    _check(dev, base, u, min_p=torch.tensor(m))
    _check(dev, base, u, temperature=torch.tensor(t))
    for i in range(n):
        _check(dev, base, u, top_k=ints(k), top_p=torch.tensor(p[i:] + p[:i]), min_p=torch.tensor(m), temperature=torch.tensor(t[i:] + t[:i]))


def test_sample_u_at_its_ends(dev):
    _case("sample, u at its ends")
    x = torch.zeros((8, 16))  # sixteen weights of 1: borders at every sixteenth
    u = torch.tensor([0.0, -0.0, -3.0, float("nan"), 1.0, float("inf"), 1 - 2.0 ** -24, 0.5])
    got = _check(dev, x, u, exact_ties=True)
    assert got == [0, 0, 0, 0, 15, 15, 15, 8]


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("vocab", [5, 300, 4097, 30000])
def test_sample_equal_logits(dev, vocab, dtype):
    """Nothing but ties: weights of exactly 1, so every cut is at a whole number of tokens, and the lowest indices stay.
    30000 of them are more than one list holds."""
    _case(f"sample, {vocab} equal logits {dtype}")
    k = [1, 2, 3, vocab // 2, vocab - 1, 0]
    n = len(k)
    x = torch.full((n, vocab), 2.5).to(DT[dtype])
    x[:, ::3] = -1.5 if vocab > 10 else 2.5
    # u a multiple of 2^-10 and sums below 2^15 make every product exact
    u = torch.tensor([0.0, 0.25, 0.5, 0.75, 0.875, 0.9375])
    # (with the others kept, weights of e^-4 among those of 1: one in three, so u = 15/16 of 30000 tokens is the border behind
    # the 28125th in exact arithmetic, 15/16 (20000 + 10000 e^-4) = 18750 + 9375 e^-4, and rounded sums fall to either side)
    _check(dev, x, u, top_k=torch.tensor(k, dtype=torch.int32))
    zero = torch.zeros((n, vocab)).to(DT[dtype])
    zero[:, 1::2] = -0.0  # equal to zero
    _check(dev, zero, u, exact_ties=True, top_k=torch.tensor(k, dtype=torch.int32))
    _check(dev, zero, u, exact_ties=True, top_p=torch.tensor([0.5, 0.25, 0.125, 0.0625, 0.75, 2.0 ** -20]))
    _check(dev, zero, u, exact_ties=True, top_k=torch.tensor(k, dtype=torch.int32), top_p=torch.tensor([0.5, 0.25, 0.125, 0.0625, 0.75, 0.875]))


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("temperature", [1.0, 1e4])
def test_sample_crowded_values(dev, dtype, temperature):
    """More tokens within one bin than are sorted at once: close values, a few of them often, and at a high temperature."""
    _case(f"sample, crowded values {dtype} at {temperature}")
    g = torch.Generator().manual_seed(5)
    rows, vocab = 6, 40000
    x = (torch.randint(0, 50, (rows, vocab), generator=g) * 2.0 ** -10 + 1.0).to(DT[dtype])
    x[1::2] = (torch.rand((3, vocab), generator=g) * 0.01 + 3.0).to(DT[dtype])
    t = torch.full((rows,), temperature)
    u = torch.rand(rows, generator=g)
    _check(dev, x, u, temperature=t, top_k=torch.tensor([1, 100, 5000, 20000, 39999, 7], dtype=torch.int32))
    _check(dev, x, u, temperature=t, top_p=torch.tensor([0.1, 0.3, 0.5, 0.7, 0.9, 0.99]))
    _check(dev, x, u, temperature=t, top_k=torch.tensor([30000, 100, 5000, 20000, 39999, 7], dtype=torch.int32),
           top_p=torch.tensor([0.1, 0.3, 0.5, 0.7, 0.9, 0.99]))


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("vocab", [9, 6000])
def test_sample_masked_and_not_finite(dev, vocab, dtype):
    """-inf and NaN are never chosen; where the largest is +inf only those that are; nothing to choose from gives -1."""
    _case(f"sample, masks, infinities and NaN, vocabulary {vocab} {dtype}")
    g = torch.Generator().manual_seed(6)
    nan, inf = float("nan"), float("inf")
    x = torch.randn((8, vocab), generator=g)
    x[0] = -inf
    x[1] = nan
    x[2, : vocab - 1] = -inf
    x[3, 2:] = nan
    x[4, 3] = x[4, 5] = inf
    x[5] = -inf
    x[5, 1::2] = nan
    x[6, ::2] = -inf
    x[7] = -3e38 if dtype == "f32" else -65504.0
    x[7, 4] = 3e38 if dtype == "f32" else 65504.0
    x = x.to(DT[dtype])
    u = torch.rand(8, generator=g)
    for kw in ({}, {"top_k": torch.full((8,), 3, dtype=torch.int32)}, {"top_p": torch.full((8,), 0.7)}, {"temperature": torch.zeros(8)},
               {"top_k": torch.full((8,), 4, dtype=torch.int32), "top_p": torch.full((8,), 0.6), "min_p": torch.full((8,), 0.1)},
               {"temperature": torch.full((8,), inf), "top_p": torch.full((8,), 0.6)}):
        got = _check(dev, x, u, exact_ties=True, **kw)
        assert got[0] == got[1] == got[5] == -1 and got[2] == vocab - 1 and got[3] in (0, 1) and got[4] in (3, 5) and got[6] % 2 == 1


def test_sample_frequencies(dev):
    """What comes out over an even grid of u is the weights' distribution: counts within one of their shares."""
    _case("sample, frequencies")
    x = torch.tensor([0.0, 1.0, -1.0, 2.0, 0.5])
    n = 4096
    got = ops.sample(x.repeat(n, 1).to(dev), ((torch.arange(n) + 0.5) / n).to(dev))
    torch.cuda.synchronize()
    counts = torch.bincount(got.cpu().long(), minlength=5).double()
    assert float((counts - n * torch.softmax(x.double(), 0)).abs().max()) <= 1


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_sample_rows_at_any_element(dev, dtype):
    """Logits as columns of a wider tensor that begin at odd elements; one row of any stride."""
    _case(f"sample, rows at odd elements {dtype}")
    g = torch.Generator().manual_seed(8)
    wide = torch.randn((9, 3005), generator=g).to(DT[dtype])
    u, kw = torch.rand(9, generator=g), _settings(9, 3001, g, "all")
    want = _check(dev, wide[:, 3:3004].contiguous(), u, **kw)
    on = {k: v.to(dev) for k, v in kw.items()}
    got = ops.sample(wide.to(dev)[:, 3:3004], u.to(dev), **on)
    one = ops.sample(wide.to(dev)[4:5, 3:3004], u.to(dev)[4:5], **{k: v[4:5] for k, v in on.items()})
    torch.cuda.synchronize()
    assert got.cpu().tolist() == want and one.item() == want[4]


def test_sample_same_in_every_batch_and_again(dev):
    """A row's token does not depend on the rows beside it, nor on when it is drawn."""
    _case("sample, the same row in several batches")
    g = torch.Generator().manual_seed(9)
    x, u = (torch.randn((300, 20000), generator=g) * 2).to(dev), torch.rand(300, generator=g).to(dev)
    kw = {k: v.to(dev) for k, v in _settings(300, 20000, g, "all").items()}
    whole = ops.sample(x, u, **kw)
    again = ops.sample(x, u, **kw)
    parts = torch.cat([ops.sample(x[a:b], u[a:b], **{k: v[a:b] for k, v in kw.items()}) for a, b in ((0, 1), (1, 8), (8, 300))])
    torch.cuda.synchronize()
    assert torch.equal(whole, again) and torch.equal(whole, parts)


def test_sample_captured(dev):
    """A captured graph follows new logits, settings and numbers, beside eager calls of other sizes."""
    _case("sample, captured")
    g = torch.Generator().manual_seed(10)
    x, u = torch.empty((5, 30001), dtype=torch.float16, device=dev), torch.empty(5, device=dev)
    kw = {k: v.to(dev) for k, v in _settings(5, 30001, g, "all").items()}
    out = torch.empty(5, dtype=torch.int32, device=dev)

    def fill(i):
        x.copy_((torch.randn((5, 30001), generator=g) * (1 + i)).half())
        u.copy_(torch.rand(5, generator=g))
        for k, v in _settings(5, 30001, g, "all").items():
            kw[k].copy_(v)

    stream = torch.cuda.Stream(dev)
    fill(0)
    with torch.cuda.stream(stream):
        ops.sample(x, u, out=out, **kw)  # the workspace
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        ops.sample(x, u, out=out, **kw)
    for i in range(4):
        fill(i)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        want = ops.sample(x, u, **kw)
        ops.sample(torch.randn((200, 777), device=dev), torch.rand(200, device=dev), top_p=torch.full((200,), 0.5, device=dev))
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_sample_two_threads(dev):
    _case("sample, two threads")
    g = torch.Generator().manual_seed(11)
    jobs = [((torch.randn((20, 9000), generator=g) * 2).to(dev), torch.rand(20, generator=g).to(dev),
             {k: v.to(dev) for k, v in _settings(20, 9000, g, "all").items()}) for _ in range(2)]
    want = [ops.sample(x, u, **kw).cpu() for x, u, kw in jobs]
    got, failed = [None, None], []

    def work(i):
        try:
            x, u, kw = jobs[i]
            with torch.cuda.stream(torch.cuda.Stream(dev)):
                for _ in range(20):
                    out = ops.sample(x, u, **kw)
                got[i] = out.cpu()
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not failed and all(torch.equal(a, b) for a, b in zip(got, want))


def test_sample_refuses(dev):
    _case("sample, refusals")
    x, u = torch.zeros((4, 10), device=dev), torch.zeros(4, device=dev)
    bad = [
        lambda: ops.sample(x.double(), u), lambda: ops.sample(x.cpu(), u), lambda: ops.sample(x.t(), u), lambda: ops.sample(x[0], u),
        lambda: ops.sample(x, u[:3]), lambda: ops.sample(x, u.half()), lambda: ops.sample(x, u.cpu()), lambda: ops.sample(x, None),
        lambda: ops.sample(x[:, :0], u), lambda: ops.sample(x, u, top_k=u), lambda: ops.sample(x, u, temperature=u[:1]),
        lambda: ops.sample(x, u, min_p=torch.zeros((4, 1), device=dev)), lambda: ops.sample(x, u, out=torch.zeros(4, device=dev)),
        lambda: ops.sample(x, u, top_p=torch.zeros(8, device=dev)[::2]),
        lambda: ops.sample(x, u, out=u.view(torch.int32)), lambda: ops.sample(x, u, out=x.view(torch.int32).reshape(-1)[:4]),
    ]
    for f in bad:
        with pytest.raises(NekoError):
            f()
    assert ops.sample(x[:0], u[:0]).shape == (0,)


# ------------------------------------------------------------------ the stated accuracy

def _kept_of_ties(vocab, top, p):
    """One logit of `top` at index 0 over vocab - 1 zeros, temperature 1: how many tokens top-p keeps, and a zero's weight."""
    w = np.exp(-np.longdouble(top))
    total = 1 + (vocab - 1) * w
    return max(1, 1 + int(np.ceil((np.longdouble(np.float32(p)) * total - 1) / w))), w


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("vocab,top,p", [(1 << 20, 20.0, 0.999), (1 << 20, 14.0, 0.8), (1 << 22, 20.0, 0.995), (1 << 24, 20.0, 0.99), (1 << 24, 24.0, 0.9999)])
def test_sample_ties_far_below_the_largest(dev, vocab, top, p, dtype):
    """Weights far below the row's largest, alike and many, so that each one's rounding adds up: the cut of top-p is within
    2^-27 of the weights' sum S of the exact one, and the token's share of the running sum within V 2^-44 / S besides.

    The running sum up to zero i (index i) is 1 + i w. Moving the cut by c moves the kept sum by c, hence what u is compared
    with; with both bounds the token is within (2^-27 + V 2^-44 / S) S / w of the exact one, and one for the rounding to whole
    tokens."""
    _case(f"sample, {vocab} tokens, one of {top} over zeros, top-p {p} {dtype}")
    x = torch.zeros((1, vocab), dtype=DT[dtype], device=dev)
    x[0, 0] = top
    us = [1 - 2.0 ** -24, 0.9999, 0.99, 0.97, 0.5]
    n, w = _kept_of_ties(vocab, top, p)
    assert 2 < n < vocab - 1
    total, kept = 1 + (vocab - 1) * w, 1 + (n - 1) * w
    rows = x.expand(len(us), vocab)[: len(us)].contiguous()
    for k in (0, vocab - 7):
        kw = {"top_p": torch.full((len(us),), p, device=dev)}
        if k:
            kw["top_k"] = torch.full((len(us),), k, dtype=torch.int32, device=dev)
            n, _ = _kept_of_ties(k, top, p)
            total, kept = 1 + (k - 1) * w, 1 + (n - 1) * w
        got = ops.sample(rows, torch.tensor(us, device=dev), **kw).tolist()
        off = float((2.0 ** -27 * total + vocab * np.longdouble(2.0) ** -44) / w) + 1
        for u, token in zip(us, got):
            want = max(0, int(np.floor((np.longdouble(np.float32(u)) * kept - 1) / w)) + 1)
            print(f"k {k} u {u:.8f}: {token}, exactly {want}, bound {off:.1f}", flush=True)
            assert abs(token - want) <= off and 0 <= token < n + off


@pytest.mark.parametrize("scale", [2.0 ** 20, -(2.0 ** 20), 2.0 ** 14])
def test_sample_logits_far_from_zero(dev, scale):
    """Logits whose size is large against their differences: weights go by the differences, so a u that is V 2^-44 or more
    from a border is on its own side of it. u is the number of f32 next to a border, in rows where that is V 2^-44 to 2^-34
    from it."""
    _case(f"sample, logits about {scale}")
    rng = np.random.default_rng(13)
    vocab, rows = 16, 60000
    step = abs(scale) * 2.0 ** -23
    l = scale + np.floor(rng.random((rows, vocab)) * 4 / step) * step
    t = (rng.random(rows) * 1.4 + 0.3).astype(np.float32) * np.float32(1.0 if abs(scale) > 2.0 ** 15 else 0.01)
    l = (scale + (l - scale) * (1.0 if abs(scale) > 2.0 ** 15 else 2.0 ** -6)).astype(np.float32)
    x = l.astype(np.longdouble)
    cum = np.cumsum(np.exp((x - x.max(1, keepdims=True)) / t.astype(np.longdouble)[:, None]), 1)
    cum /= cum[:, -1:]
    border = cum[np.arange(rows), rng.integers(0, vocab - 1, rows)]
    u = border.astype(np.float32)
    away = np.abs(u.astype(np.longdouble) - border)
    take = (away > vocab * 2.0 ** -44) & (away < 2.0 ** -34) & (u < 1)
    l, t, u, cum = l[take], t[take], u[take], cum[take]
    assert len(l) > 20
    want = (cum <= u.astype(np.longdouble)[:, None]).sum(1)
    got = ops.sample(torch.from_numpy(l).to(dev), torch.from_numpy(u).to(dev), temperature=torch.from_numpy(t).to(dev)).cpu().numpy()
    print(f"{int((got != want).sum())} of {len(l)} on the wrong side", flush=True)
    assert np.array_equal(got, want)


# (temperature, logit, min_p), f32: e^x is within 1.1 * 2^-53 of min_p, relative, for x = logit * (1 / temperature) in double, whose
# two roundings move the weight by 2 |x| 2^-53 from the exact one; |x| < 10.
NEXT_TO_MIN_P = """
0x1.016486p+0 -0x1.b05ba4p+0 0x1.7dc912p-3; 0x1.035c18p+0 -0x1.52dc34p+1 0x1.2c47a2p-4;
0x1.052658p+0 -0x1.7b8588p-3 0x1.aaf31p-1; 0x1.0885a4p+0 -0x1.d5764p-6 0x1.f1ff3cp-1;
0x1.09015p+0 -0x1.2aaaep+1 0x1.adf856p-4; 0x1.099ec8p+0 -0x1.9785p-4 0x1.d12f74p-1;
0x1.0b7eep-1 -0x1.1cd438p+1 0x1.cf21ep-7; 0x1.13721ep+0 -0x1.3a274p-1 0x1.217906p-1;
0x1.1d49cap-1 -0x1.a35572p+0 0x1.b13284p-5; 0x1.224188p-1 -0x1.53f88ap+1 0x1.2e80aep-7;
0x1.2449ecp-1 -0x1.db5c6cp-2 0x1.c617c2p-2; 0x1.24635ap+0 -0x1.174b68p+1 0x1.2f22d4p-3;
0x1.2b79bcp+0 -0x1.13571cp-2 0x1.96dc84p-1; 0x1.2ee9eap+0 -0x1.f3cce8p+0 0x1.8953dep-3;
0x1.30546ap+0 -0x1.c1c278p+0 0x1.d3324p-3; 0x1.3511d8p+0 -0x1.e559f8p+0 0x1.a9ec12p-3;
0x1.39997cp-2 -0x1.525d06p+1 0x1.7609f2p-13; 0x1.3b01dp-1 -0x1.f7ecc8p-2 0x1.cc2d0cp-2;
0x1.3ea258p+0 -0x1.1e49dcp+0 0x1.a0f538p-2; 0x1.4613ap-1 -0x1.26318p-3 0x1.989d02p-1;
0x1.49473p-1 -0x1.c49f46p-1 0x1.03039ap-2; 0x1.51876p-1 -0x1.f62d0cp+0 0x1.a1eda2p-5;
0x1.540ab2p-1 -0x1.22f8f4p+1 0x1.0b3c28p-5; 0x1.54da58p-1 -0x1.dbdf3ap+0 0x1.f60918p-5;
0x1.55ecfcp-1 -0x1.6db14p-1 0x1.5f69dap-2; 0x1.5bbdbp+0 -0x1.6bd52p+1 0x1.f9552ep-4;
0x1.671792p-1 -0x1.c469c4p+0 0x1.49a428p-4; 0x1.6bff12p+0 -0x1.c39caap-1 0x1.13549ep-1;
0x1.6ddbaep+0 -0x1.787ad2p+1 0x1.05881p-3; 0x1.73c9d8p+0 -0x1.4c3044p+1 0x1.56f85p-3;
0x1.881daep+0 -0x1.66b916p+1 0x1.48a1fap-3; 0x1.8f856ap-2 -0x1.9191a4p+0 0x1.25fe64p-6;
0x1.967af2p+0 -0x1.90a1cp-1 0x1.38c92ap-1; 0x1.96f7a6p+0 -0x1.b3c7p+0 0x1.5ef674p-2;
0x1.98b76p+0 -0x1.8fc798p-1 0x1.39f516p-1; 0x1.9de7acp-2 -0x1.fb091p+0 0x1.e802bep-8;
0x1.ad0318p+0 -0x1.e9601ep+0 0x1.4743b4p-2; 0x1.b1e97ep+0 -0x1.43890cp+0 0x1.e5d318p-2;
0x1.b1f75p+0 -0x1.49883p+0 0x1.df33b4p-2; 0x1.c2c88ep-2 -0x1.aebffp-1 0x1.2eee28p-3;
0x1.d0715ep-1 -0x1.f8a67ap-1 0x1.5977d8p-2; 0x1.db724ap-2 -0x1.49f5bcp+0 0x1.fe419p-5;
0x1.dc5d3ap-1 -0x1.7fe036p+1 0x1.4634fep-5; 0x1.dcb15ep-1 -0x1.f5e4bcp+0 0x1.f2b71p-4;
0x1.debcep-1 -0x1.4f1e76p+0 0x1.f90676p-3; 0x1.ef5f9cp-1 -0x1.bc8c16p-1 0x1.a16978p-2;
0x1.f96f04p-2 -0x1.28b588p+0 0x1.875a84p-4;
"""


def test_sample_min_p_next_to_a_weight(dev):
    """Weights within (1.1 + 2 * 10) 2^-53 < 2^-48 of min_p, each in a block of its own behind the largest's: whichever side they fall to, a token is
    chosen, and one that may stay. u asks for the last token that stays."""
    _case("sample, min_p next to a weight")
    rows = [[float.fromhex(v) for v in r.split()] for r in NEXT_TO_MIN_P.replace("\n", " ").split(";") if r.strip()]
    n, vocab = len(rows), 5000
    x = torch.full((n, vocab), -float("inf"))
    x[:, 0] = 0.0
    t, x[:, 4099], m = (torch.tensor([r[i] for r in rows]) for i in range(3))
    exact = np.exp(x[:, 4099].numpy().astype(np.longdouble) / t.numpy().astype(np.longdouble))
    assert float(np.abs(exact / m.numpy().astype(np.longdouble) - 1).max()) <= 2.0 ** -48
    out = torch.full((n,), -7, dtype=torch.int32, device=dev)
    ops.sample(x.to(dev), torch.full((n,), 0.99, device=dev), temperature=t.to(dev), min_p=m.to(dev), out=out)
    got = out.tolist()
    print(got, flush=True)
    assert set(got) <= {0, 4099}


def test_sample_min_p_of_one(dev):
    """min_p = 1 where weights are 1 or the number below it, each in a block of its own: a token is chosen, one whose weight is
    1 but for the rounding of its exponential (2^-52)."""
    _case("sample, min_p of 1, weights next to 1")
    g = torch.Generator().manual_seed(12)
    vocab, rows = 30 * 2048, 64
    for temperature, scale in ((1e15, 8.0), (1e16, 8.0), (3e16, 8.0), (1e17, 8.0), (1e18, 8.0), (1.0, 1e-16), (0.7, 3e-16)):
        x = torch.full((rows, vocab), -float("inf"))
        x[:, 700::2048] = torch.rand((rows, 30), generator=g) * scale
        u = torch.rand(rows, generator=g)
        out = torch.full((rows,), -7, dtype=torch.int32, device=dev)
        ops.sample(x.to(dev), u.to(dev), temperature=torch.full((rows,), temperature, device=dev), min_p=torch.ones(rows, device=dev), out=out)
        got = out.cpu().long()
        assert bool(((got >= 0) & (got < vocab)).all()), (temperature, got.tolist())
        l = x.numpy().astype(np.longdouble)
        chosen = np.exp((l[np.arange(rows), got.numpy()] - l.max(1)) / np.longdouble(np.float32(temperature)))
        assert float((1 - chosen).max()) <= 2.0 ** -52, temperature


def test_sample_top_p_of_logits_far_from_zero(dev):
    """Small temperatures, logits 2^27 times as large: one of 1000 and 30000 of the next f32 below it, 8 to 9 temperatures away.
    The cut of top-p is where the weights by the difference put it, when those are more than 2^-27 of the sum from a border:
    u = 1 - 2^-24 asks for the last token that stays, whose weight is e^-9 / 5 or e^-8 / 11 > 2^-24 of the kept ones'."""
    _case("sample, top-p of logits far from zero")
    rng = np.random.default_rng(14)
    rows, ties = 2000, 30000
    low = np.nextafter(np.float32(1000.0), np.float32(0.0))
    t = (float(np.float32(1000.0) - low) / (8 + rng.random(rows))).astype(np.float32)
    w = np.exp((np.longdouble(low) - 1000) / t.astype(np.longdouble))
    j = rng.integers(1, ties, rows)  # ties kept up to the border
    border = (1 + j * w) / (1 + ties * w)
    p = border.astype(np.float32)
    off = p.astype(np.longdouble) - border
    take = (np.abs(off) > 1.25 * 2.0 ** -27) & (np.abs(off) < 2.0 ** -25)
    t, j, p, off = t[take], j[take], p[take], off[take]
    n = len(t)
    assert n > 500
    x = torch.full((n, ties + 1), float(low), device=dev)
    x[:, 0] = 1000.0
    want = j + (off > 0)
    got = ops.sample(x, torch.full((n,), 1 - 2.0 ** -24, device=dev), temperature=torch.from_numpy(t).to(dev), top_p=torch.from_numpy(p).to(dev)).cpu().numpy()
    print(f"{int((got != want).sum())} of {n} cut elsewhere", flush=True)
    assert np.array_equal(got, want)


@pytest.mark.parametrize("vocab", [7, 300, 6000, 30000])
def test_sample_largest_logits_far_from_all_others(dev, vocab):
    """Logits so large against the temperature that only those equal to the largest weigh anything, in several parts of the
    row: whole numbers of tokens, cuts and borders met exactly."""
    _case(f"sample, ties far from all others, vocabulary {vocab}")
    x = torch.full((6, vocab), -1.0)
    x[:, ::2] = torch.tensor([1e30, 1e30, -1.0, 65504.0, 3e38, 1e-3])[:, None]
    x[2, 1::2] = -3e38
    t = torch.tensor([0.5, 1e3, 1e-30, 1e-20, 1e-30, 1e-25])
    u = torch.tensor([0.0, 0.25, 0.5, 0.75, 0.875, 0.9375])
    half = (vocab + 1) // 2
    k = torch.tensor([1, 2, half, half + 1, vocab - 1, 0], dtype=torch.int32)
    p = torch.tensor([0.5, 0.25, 0.125, 0.75, 0.0625, 0.875])
    _check(dev, x, u, exact_ties=True, temperature=t, top_p=p)
    _check(dev, x, u, exact_ties=True, temperature=t, top_k=k)
    _check(dev, x, u, exact_ties=True, temperature=t, top_k=k, top_p=p, min_p=torch.full((6,), 0.5))


def test_sample_captured_in_the_workspace_of_the_other_type(dev):
    """The workspace goes by rows, vocabulary and settings, not by the type: a call of one type has made room for the other's."""
    _case("sample, captured after a call of the other type")
    for first, then in ((torch.float32, torch.float16), (torch.float16, torch.float32)):
        x = (torch.randn((130, 151936), generator=torch.Generator().manual_seed(15)) * 2).to(dev)
        u, p = torch.rand(130, generator=torch.Generator().manual_seed(16)).to(dev), torch.full((130,), 0.9, device=dev)
        out = torch.empty(130, dtype=torch.int32, device=dev)
        a, b = x.to(first), x.to(then)
        del x

        def work():  # (a thread's context and workspace are its own)
            stream = torch.cuda.Stream(dev)
            with torch.cuda.stream(stream):
                ops.sample(a, u, top_p=p)
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
                ops.sample(b, u, top_p=p, out=out)
            graph.replay()
            torch.cuda.synchronize()
            got.append((out.clone(), ops.sample(b, u, top_p=p)))

        got = []
        t = threading.Thread(target=work)
        t.start()
        t.join()
        torch.cuda.synchronize()
        assert len(got) == 1 and torch.equal(*got[0])
