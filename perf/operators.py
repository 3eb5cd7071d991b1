"""The measured operators of serving many sequences from a paged 8-bit KV cache.

  append     one call of ops.qk_norm_rope_paged: the q / k heads of new rows normed and rotated, k and v rounded to
             8 bits and written to the sequences' pages with one power-of-two scale for each page and head
  attention  one call of ops.attention_paged: causal grouped-query attention of new rows over those pages

A batch is a list of sequences, each with some new rows (none to all of its length); the rows stand one sequence after
another. Calls are validated once with ops.prepare and re-issued, as a serving loop does.
"""
import math
import random

import torch

own = False

EPS = 1e-6
THETA = 1e6
DT = {"f16": torch.float16, "f32": torch.float32}
F8 = torch.float8_e4m3fn

# Heads of the repository's configurations (query heads, kv heads, head size) and two generic ones.
HEADS = {
    "qwen3_4b": (32, 8, 128),
    "qwen3_0.6b": (16, 8, 128),
    "gpt2": (12, 12, 64),
    "one_kv_256": (8, 1, 256),
    "odd_80": (20, 4, 80),
}

# Fields of a case: heads; seqs sequences of at most ctx tokens, of which at most new are this call's rows; how
# ("even": all alike; "ragged": each its own; "mixed": one prompt chunk of new rows beside single tokens); pick (which
# ragged lengths); page size; dtype of the activations; pad rows behind the last sequence. Attention: cap (scores capped
# at this magnitude by a tanh, 0: none), window (keys a row sees, 0: all before it), slopes (a bias by distance).
# Append: norm, rot (rotated dimensions, 0: none), inter (pairs interleaved rather than split in halves).


def _attn(name, heads, seqs, new, ctx, how, page, dtype, pick=1, pad=0, cap=0.0, window=0, slopes=0):
    return {"name": name, "kind": "attention", "heads": heads, "seqs": seqs, "new": new, "ctx": ctx, "how": how, "page": page,
            "dtype": dtype, "pick": pick, "pad": pad, "cap": cap, "window": window, "slopes": slopes}


def _app(name, heads, seqs, new, ctx, how, page, dtype, pick=1, pad=0, norm=1, rot=128, inter=0):
    return {"name": name, "kind": "append", "heads": heads, "seqs": seqs, "new": new, "ctx": ctx, "how": how, "page": page,
            "dtype": dtype, "pick": pick, "pad": pad, "norm": norm, "rot": rot, "inter": inter}


def listed():
    return [
        # One user, one token, a short chat: the smallest attention call, where latency counts.
        _attn("attn_decode_one", "qwen3_0.6b", 1, 1, 777, "even", 16, "f16"),
        # A decode step of 32 users of ragged lengths, as a server runs all the time; the batch padded to 40 rows.
        _attn("attn_decode_batch", "qwen3_4b", 32, 1, 4096, "ragged", 16, "f16", pad=8),
        # Two users far into long documents.
        _attn("attn_decode_long", "qwen3_4b", 2, 1, 65521, "even", 64, "f16"),
        # 64 short sequences with f32 activations (what the C++ engine passes) and a bias by distance.
        _attn("attn_decode_f32", "gpt2", 64, 1, 1021, "ragged", 32, "f32", pick=2, slopes=1),
        # A prompt's chunk taken along with a running decode batch.
        _attn("attn_mixed", "qwen3_4b", 24, 509, 8190, "mixed", 16, "f16"),
        # A long prompt in one call: the largest.
        _attn("attn_prefill_8k", "qwen3_4b", 1, 8192, 8192, "even", 16, "f16"),
        # Ragged prompts with capped scores and a sliding window, f32 activations.
        _attn("attn_window_f32", "qwen3_0.6b", 6, 2048, 2048, "ragged", 64, "f32", pick=15, cap=50.0, window=500),
        # The cache's side of one decode step: one user, and 64 in the middle of their pages.
        _app("append_one", "qwen3_0.6b", 1, 1, 777, "even", 16, "f16"),
        _app("append_decode", "qwen3_4b", 64, 1, 4096, "ragged", 16, "f16"),
        # A prefill of 4 x 2048 tokens.
        _app("append_prefill", "qwen3_4b", 4, 2048, 2048, "even", 16, "f16"),
        # Ragged chunks that begin and end inside pages: f32, no norm, half of each head rotated in interleaved pairs.
        _app("append_ragged", "gpt2", 9, 700, 1500, "ragged", 32, "f32", pick=4, norm=0, rot=32, inter=1),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    heads = rng.choice(["qwen3_4b", "qwen3_4b", "qwen3_0.6b", "gpt2", "one_kv_256", "odd_80"])
    kind = rng.choice(["attention", "attention", "append"])
    page, dtype, pick, pad = rng.choice([16, 16, 32, 64, 128]), rng.choice(["f16", "f16", "f32"]), rng.randint(1, 10**6), rng.choice([0, 0, rng.randint(1, 9)])
    how = rng.choice(["decode", "prompt", "ragged", "mixed"])
    if how == "decode":  # single tokens, or a few at once to be verified
        seqs = _log_int(rng, 1, 96)
        new, ctx, how = rng.choice([1, 1, 1, rng.randint(2, 8)]), _log_int(rng, 8, min(65536, 262144 // seqs)), rng.choice(["even", "ragged"])
    elif how == "prompt":
        seqs, new = 1, _log_int(rng, 9, 6000)
        ctx, how = new + rng.choice([0, 0, _log_int(rng, 1, 4096)]), "even"
    elif how == "ragged":
        seqs, new = rng.randint(2, 16), _log_int(rng, 9, 1024)
        ctx = max(new, _log_int(rng, 9, 4096))
    else:
        seqs, new = rng.randint(2, 32), _log_int(rng, 9, 700)
        ctx = max(new, _log_int(rng, 64, 8192))
    if kind == "attention":
        c = _attn("", heads, seqs, new, ctx, how, page, dtype, pick, pad, rng.choice([0.0, 0.0, 30.0]), rng.choice([0, 0, _log_int(rng, 1, 4096)]), rng.choice([0, 0, 1]))
    else:
        hd = HEADS[heads][2]
        c = _app("", heads, seqs, new, ctx, how, page, dtype, pick, pad, rng.randint(0, 1), rng.choice([hd, hd, hd // 2 // 8 * 8, 0]), rng.randint(0, 1))
    del c["name"]
    return c


def _seqs(c):
    """(new rows, length with them) of each sequence."""
    r = random.Random(c["pick"])
    got = []
    for i in range(c["seqs"]):
        if c["how"] == "even":
            n, length = c["new"], c["ctx"]
        elif c["how"] == "ragged":
            length = _log_int(r, max(1, c["ctx"] // 64), c["ctx"])
            n = c["new"] if c["new"] == 1 else _log_int(r, max(1, c["new"] // 16), c["new"])
            if i % 8 == 7:  # a place in the batch that no user has now
                n = length = 0
        else:
            length = _log_int(r, max(1, c["ctx"] // 16), c["ctx"])
            n = 1
            if i == c["seqs"] // 2:
                n, length = c["new"], c["ctx"]
        got.append((min(n, length), length))
    return got


# ------------------------------------------------------------------ inputs

def _rope_table(n_pos, rot):
    inv = THETA ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / max(rot, 1))
    a = torch.arange(n_pos, device="cuda", dtype=torch.float64)[:, None] * inv
    return torch.stack([a.cos(), a.sin()], -1).reshape(n_pos, rot).float()


def _pages(g, n_pages, kv, page, hd, std):
    """Pages of random tokens in 8 bits, with a spread of scales between pages and heads; per-channel sizes as keys have them."""
    k, s = [], []
    step = max(1, (1 << 26) // (kv * page * hd))
    channel = torch.randn((1, kv, 1, hd), generator=g, device="cuda").mul(0.5).exp()
    for i in range(0, n_pages, step):
        n = min(step, n_pages - i)
        x = torch.randn((n, kv, page, hd), generator=g, device="cuda") * channel * std
        x = x * torch.randn((n, kv, 1, 1), generator=g, device="cuda").mul(0.3).exp()
        m, e = torch.frexp(x.abs().amax((2, 3)))
        sc = torch.ldexp(torch.ones_like(m), e - 9 + (m > 0.875).int())
        k.append((x / sc[:, :, None, None]).to(F8))
        s.append(sc)
    return torch.cat(k), torch.cat(s)


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + 13)
    H, KV, hd = HEADS[c["heads"]]
    P, dt = c["page"], DT[c["dtype"]]
    seqs = _seqs(c)
    used = [-(-length // P) for _, length in seqs]
    n_pages = sum(used) + 3  # a few are free
    k_pages, k_scales = _pages(g, n_pages, KV, P, hd, 1.0)
    v_pages, v_scales = _pages(g, n_pages, KV, P, hd, 0.7)
    order = torch.randperm(n_pages, generator=g, device="cuda").int()
    width = max(max(used), 1)
    slot = torch.arange(width, device="cuda")[None, :]
    n_used = torch.tensor(used, device="cuda")[:, None]
    first = torch.cumsum(n_used, 0) - n_used
    table = torch.where(slot < n_used, order[(first + slot).clamp(max=n_pages - 1)], -1).int().contiguous()
    starts = [0]
    for n, _ in seqs:
        starts.append(starts[-1] + n)
    rows, total = starts[-1] + c["pad"], starts[-1]
    st = {"c": c, "H": H, "KV": KV, "hd": hd, "P": P, "rows": rows, "total": total, "k_pages": k_pages, "v_pages": v_pages,
          "k_scales": k_scales, "v_scales": v_scales, "table": table, "free": order[-1].long(), "max_new": max(n for n, _ in seqs),
          "max_len": max(length for _, length in seqs),
          "row_start": torch.tensor(starts, device="cuda", dtype=torch.int32),
          "kv_len": torch.tensor([length for _, length in seqs], device="cuda", dtype=torch.int32)}
    if c["kind"] == "attention":
        q = torch.randn((rows, H, hd), generator=g, device="cuda") * torch.randn((1, H, 1), generator=g, device="cuda").mul(0.3).exp()
        st["q"] = q.reshape(rows, H * hd).to(dt)
        st["out"] = torch.zeros((rows, H * hd), dtype=dt, device="cuda")
        st["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], device="cuda") if c["slopes"] else None
        st["scale"] = 1.0 / math.sqrt(hd)
    else:
        st["qkv"] = (torch.randn((rows, (H + 2 * KV) * hd), generator=g, device="cuda") * 1.5).to(dt)
        st["q_out"] = torch.zeros((rows, H * hd), dtype=dt, device="cuda")
        st["wqk"] = (torch.randn((2 * hd,), generator=g, device="cuda") * 0.1 + 1.0) if c["norm"] else None
        st["cs"] = _rope_table(st["max_len"], c["rot"]) if c["rot"] else None
    return st


# ------------------------------------------------------------------ plain forms

def _place(st):
    """Of each row: its sequence, its place among the sequence's new rows, its position."""
    start, length = st["row_start"].long(), st["kv_len"].long()
    row = torch.arange(st["total"], device="cuda")
    seq = torch.searchsorted(start[1:], row, right=True)
    i = row - start[seq]
    return seq, i, length[seq] - (start[seq + 1] - start[seq]) + i


def _plain_attention(st):
    c, H, KV, hd, P = st["c"], st["H"], st["KV"], st["hd"], st["P"]
    G, S, R = H // KV, st["table"].shape[0], st["max_new"]
    out, length = st["out"], st["kv_len"].long()
    if not st["total"]:
        return out
    seq, i, pos = _place(st)
    page = st["table"].long().clamp(min=0)

    def cached(codes, scales):  # [S, KV, keys, hd]
        x = codes.view(torch.uint8)[page].view(F8).float() * scales[page][..., None, None]
        return x.transpose(1, 2).reshape(S, KV, -1, hd)

    k, v = cached(st["k_pages"], st["k_scales"]), cached(st["v_pages"], st["v_scales"])
    inside = torch.arange(k.shape[2], device="cuda") < length[:, None]
    v = torch.where(inside[:, None, :, None], v, torch.zeros((), device="cuda"))
    q = torch.zeros((S, R, H, hd), device="cuda")
    q[seq, i] = st["q"][: st["total"]].float().reshape(-1, H, hd)
    p = torch.full((S, R), -1, device="cuda")
    p[seq, i] = pos
    q = q.reshape(S, R, KV, G, hd).permute(0, 2, 1, 3, 4).reshape(S, KV, R * G, hd)
    s = torch.matmul(q, k.transpose(2, 3)).reshape(S, KV, R, G, -1) * st["scale"]
    del k
    if c["cap"]:
        s = torch.tanh(s / c["cap"]) * c["cap"]
    away = torch.arange(s.shape[-1], device="cuda") - p[:, :, None]  # [S, R, keys]
    if st["slopes"] is not None:
        s = s + st["slopes"].reshape(KV, 1, G, 1) * away[:, None, :, None, :]
    sees = (away <= 0) & inside[:, None, :]
    if c["window"]:
        sees &= away > -c["window"]
    s = torch.where(sees[:, None, :, None, :], s, torch.full((), -math.inf, device="cuda"))
    m = s.amax(-1, keepdim=True)
    s = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.reshape(S, KV, R * G, -1), v).reshape(S, KV, R, G, hd) / torch.where(total == 0, 1.0, total)
    out[: st["total"]] = o.permute(0, 2, 1, 3, 4).reshape(S, R, H * hd)[seq, i].to(out.dtype)
    return out


def _rotated(x, cs, pos, rot, inter):
    """x [rows, heads, hd]: its first rot dimensions turned by the angles of pos."""
    if not rot:
        return x
    t = cs[pos][:, None, :]
    co, si = t[..., 0::2], t[..., 1::2]
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if inter else (x[..., : rot // 2], x[..., rot // 2: rot])
    y, z = a * co - b * si, b * co + a * si
    turned = torch.stack([y, z], -1).flatten(-2) if inter else torch.cat([y, z], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _need(amax):
    """The smallest power of two that brings amax to 448, the largest 8-bit value, or below."""
    m, e = torch.frexp(amax)
    e = torch.where(amax > 0, e - 9 + (m > 0.875).int(), -64).clamp(-64, 64)
    return torch.ldexp(torch.ones_like(amax), e)


def _plain_append(st):
    c, H, KV, hd, P, n = st["c"], st["H"], st["KV"], st["hd"], st["P"], st["total"]
    seq, i, pos = _place(st)
    dt = st["qkv"].dtype
    x = st["qkv"][:n].float().reshape(n, H + 2 * KV, hd)
    q, k, v = x[:, :H], x[:, H: H + KV], x[:, H + KV:]
    if st["wqk"] is not None:
        q, k = (t / torch.sqrt(t.square().mean(-1, keepdim=True) + EPS) * w for t, w in ((q, st["wqk"][:hd]), (k, st["wqk"][hd:])))
    st["q_out"][:n] = _rotated(q, st["cs"], pos, c["rot"], c["inter"]).to(dt).reshape(n, H * hd)
    k = _rotated(k, st["cs"], pos, c["rot"], c["inter"]).to(dt).float()
    page, slot = st["table"].long()[seq, pos // P], pos % P
    # Each sequence's first page of the call may hold earlier tokens, in the slots before `old`.
    start, length = st["row_start"].long(), st["kv_len"].long()
    p0 = length - (start[1:] - start[:-1])
    old = torch.where(length > p0, p0 % P, 0)
    first = st["table"].long().gather(1, (p0 // P).clamp(max=st["table"].shape[1] - 1)[:, None])[:, 0]
    first = torch.where(old > 0, first, st["free"])  # a page that stays as it is where there are none
    earlier = (torch.arange(P, device="cuda") < old[:, None])[:, None, :, None]
    for new, codes, scales in ((k, st["k_pages"], st["k_scales"]), (v, st["v_pages"], st["v_scales"])):
        bits = codes.view(torch.uint8)
        scale = _need(torch.zeros((codes.shape[0], KV), device="cuda").index_reduce_(0, page, new.abs().amax(-1), "amax"))
        scale[first] = torch.maximum(scale[first], scales[first])
        had = bits[first]
        again = (had.view(F8).float() * (scales[first] / scale[first])[:, :, None, None]).to(F8).view(torch.uint8)
        bits[first] = torch.where(earlier, again, had)
        bits[page, :, slot] = (new / scale[page][..., None]).to(F8).view(torch.uint8)
        scales[page] = scale[page]
    return st["q_out"], st["k_pages"], st["v_pages"], st["k_scales"], st["v_scales"]


def run(st):
    c = st["c"]
    if not own:
        return _plain_attention(st) if c["kind"] == "attention" else _plain_append(st)
    if "call" not in st:
        from nekochat_amd import ops

        cache = ops.PagedKV(st["k_pages"], st["v_pages"], st["k_scales"], st["v_scales"])
        batch = (cache, st["table"], st["row_start"], st["kv_len"])
        if c["kind"] == "attention":
            st["call"], _ = ops.prepare(ops.attention_paged, st["q"], *batch, st["H"], scale=st["scale"], softcap=c["cap"],
                                        window=c["window"], slopes=st["slopes"], out=st["out"])
        else:
            st["call"], _ = ops.prepare(ops.qk_norm_rope_paged, st["qkv"], st["H"], *batch, st["cs"], EPS, wqk=st["wqk"],
                                        interleaved=bool(c["inter"]), q_out=st["q_out"])
    st["call"]()
    if c["kind"] == "attention":
        return st["out"]
    return st["q_out"], st["k_pages"], st["v_pages"], st["k_scales"], st["v_scales"]


# ------------------------------------------------------------------ work

def work(c):
    H, KV, hd = HEADS[c["heads"]]
    size, seqs, w = 2 if c["dtype"] == "f16" else 4, _seqs(c), c.get("window", 0)
    rows, P = sum(n for n, _ in seqs), c["page"]
    small = 4 * (2 * len(seqs) + 1)
    if c["kind"] == "append":
        pages = sum(-(-length // P) - (length - n) // P for n, length in seqs if n)
        table = 0 if not c["rot"] else 4 * c["rot"] * max((length for n, length in seqs if n), default=0)
        # q, k, v read, q written, k and v codes written, a scale for each page and head, the table's angles at most once.
        return {"bytes": rows * (H + 2 * KV) * hd * size + rows * H * hd * size + 2 * rows * KV * hd + pages * (8 * KV + 4) +
                min(table, 4 * c["rot"] * rows) + small, "flops": 10 * rows * (H + KV) * hd}
    keys = pairs = pages = 0
    for n, length in seqs:
        if not n:
            continue
        begin = max(0, length - n - w + 1) if w else 0
        keys += length - begin
        pages += -(-length // P) - begin // P
        # row i sees the keys up to length - n + i, at most w of them
        lo, hi = length - n + 1, length
        if w and w < hi:
            full = hi - max(lo, w) + 1  # rows that see w keys
            pairs += full * w + sum(range(lo, max(lo, w)))
        else:
            pairs += (lo + hi) * n // 2
    return {"bytes": 2 * rows * H * hd * size + 2 * keys * KV * hd + pages * (8 * KV + 4) + small, "flops": 4 * hd * H * pairs}


# ------------------------------------------------------------------ 64 bits

def _value(codes):
    """The value of each E4M3 code, from its bits."""
    b = codes.view(torch.uint8).long()
    e, m = (b >> 3) & 15, b & 7
    mag = torch.where(e > 0, (8 + m).double() * 2.0 ** (e - 10).double(), m.double() * 2.0**-9)
    return torch.where(b > 127, -mag, mag)


def exact(c, seed):
    st = prepare(c, seed)
    H, KV, hd = HEADS[c["heads"]]
    P, G = c["page"], H // KV
    row = 0
    if c["kind"] == "attention":
        out = torch.zeros((st["rows"], H * hd), dtype=torch.float64, device="cuda")
        for s, (n, length) in enumerate(_seqs(c)):
            if not n:
                continue
            ids = st["table"][s, : -(-length // P)].long()
            at, pos = torch.arange(length, device="cuda")[None], torch.arange(length - n, length, device="cuda")[:, None]
            sees = at <= pos
            if c["window"]:
                sees = sees & (pos - at < c["window"])
            for h in range(H):
                g = h // G
                k, v = ((_value(codes[ids, g]) * scales[ids, g].double()[:, None, None]).reshape(-1, hd)[:length]
                        for codes, scales in ((st["k_pages"], st["k_scales"]), (st["v_pages"], st["v_scales"])))
                x = st["q"][row: row + n, h * hd: (h + 1) * hd].double() @ k.T * st["scale"]
                if c["cap"]:
                    x = c["cap"] * torch.tanh(x / c["cap"])
                if st["slopes"] is not None:
                    x = x - float(st["slopes"][h]) * (pos - at)
                w = torch.softmax(x.masked_fill_(~sees, -math.inf), -1)
                out[row: row + n, h * hd: (h + 1) * hd] = w @ v
            row += n
        return out

    rot, dt = c["rot"], DT[c["dtype"]]
    q_out = torch.zeros((st["rows"], H * hd), dtype=torch.float64, device="cuda")
    kc, vc, ks, vs = _value(st["k_pages"]), _value(st["v_pages"]), st["k_scales"].double(), st["v_scales"].double()
    for s, (n, length) in enumerate(_seqs(c)):
        if not n:
            continue
        x = st["qkv"][row: row + n].double().reshape(n, H + 2 * KV, hd)
        qk, v = x[:, : H + KV], x[:, H + KV:]
        if st["wqk"] is not None:
            w = st["wqk"].double().reshape(2, 1, hd).repeat_interleave(torch.tensor([H, KV], device="cuda"), 0).reshape(H + KV, hd)
            qk = qk * (qk.pow(2).sum(-1, keepdim=True) / hd + EPS).rsqrt() * w
        if rot:
            z = st["cs"][length - n: length].double().reshape(n, 1, rot // 2, 2)
            pairs = qk[..., :rot].reshape(n, H + KV, rot // 2, 2) if c["inter"] else qk[..., :rot].reshape(n, H + KV, 2, rot // 2).transpose(2, 3)
            turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * torch.view_as_complex(z.contiguous()))
            turned = turned if c["inter"] else turned.transpose(2, 3)
            qk = torch.cat([turned.reshape(n, H + KV, rot), qk[..., rot:]], -1)
        q_out[row: row + n] = qk[:, :H].reshape(n, H * hd)
        row += n
        for new, codes, scales in ((qk[:, H:], kc, ks), (v, vc, vs)):
            for j in range((length - n) // P, -(-length // P)):
                a, b = max(0, length - n - j * P), min(P, length - j * P)  # the new slots of page j
                part = new[j * P + a - (length - n): j * P + b - (length - n)]
                top = part.to(dt).double().abs().amax((0, 2))  # rounded to the activations' type first
                scale = 2.0 ** torch.ceil(torch.log2(top / 448)).clamp(-64, 64)
                page = int(st["table"][s, j])
                if a:
                    scale = torch.maximum(scale, scales[page])
                    codes[page, :, :a] *= (scales[page] / scale)[:, None, None]
                codes[page, :, a:b] = (part / scale[:, None]).transpose(0, 1)
                scales[page] = scale
    return q_out, kc, vc, ks, vs
