"""The measured operators of a step of speculative decoding over a paged 8-bit KV cache: a drafter proposes a small tree
of tokens for every sequence, the model looks at all of them at once, and what it agrees with stays.

  append     one call of ops.qk_norm_rope_tree_paged: the q / k heads of the drafted rows normed and turned by the angle
             of their place in the text (the depth in the tree, not the slot), k and v to the sequences' pages
  attention  one call of ops.attention_tree_paged: grouped-query attention of those rows over the whole context and, of
             the drafted tokens, each row's own ancestors
  sample     one call of ops.sample: a token of each row of logits, by temperature, top-k, top-p and min-p, from a given
             uniform number
  accept     one call of ops.accept_tree: the path that the sampled tokens take from each tree's root
  keep       one call of ops.keep_paged: the tokens of that path moved together in the pages

A batch is a list of sequences, each with the rows of its tree (none: an idle place), the rows one sequence after
another. Row 0 of a tree is its root, the last token that was decided; parents stand before their children. Calls are
validated once with ops.prepare and re-issued, as a serving loop does.
"""
import math
import random

import numpy as np
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

# Fields of a batch: heads; seqs sequences of at most ctx tokens before the tree and trees of at most nodes rows; how
# ("even": all alike; "ragged": each its own, some places idle, some trees padded to a fixed size); shape ("wide": several
# branches at each level; "chain": mostly one token after another); pick (which lengths and trees); page size; dtype of
# the activations; pad rows behind the last sequence. Attention: cap, window, slopes as in attention over a paged cache.
# Append: norm, rot (rotated dimensions), inter (pairs interleaved). Sample: rows, vocab, dtype, mode ("all": every filter
# in every row; "mixed": each row its own settings, some greedy or with no filter; "plain": temperature and top-p).


def _batch(name, kind, heads, seqs, nodes, ctx, how, shape, page, dtype, pick, pad=0, **more):
    return {"name": name, "kind": kind, "heads": heads, "seqs": seqs, "nodes": nodes, "ctx": ctx, "how": how, "shape": shape,
            "page": page, "dtype": dtype, "pick": pick, "pad": pad, **more}


def _attn(*a, cap=0.0, window=0, slopes=0, **k):
    return _batch(a[0], "attention", *a[1:], cap=cap, window=window, slopes=slopes, **k)


def _app(*a, norm=1, rot=128, inter=0, **k):
    return _batch(a[0], "append", *a[1:], norm=norm, rot=rot, inter=inter, **k)


def _sample(name, rows, vocab, dtype, mode, pick):
    return {"name": name, "kind": "sample", "rows": rows, "vocab": vocab, "dtype": dtype, "mode": mode, "pick": pick}


def listed():
    return [
        # One user's tree in a short chat: the smallest attention call, where latency counts.
        _attn("attn_tree_one", "qwen3_0.6b", 1, 26, 777, "even", "wide", 16, "f16", 1),
        # A server's verification step: ragged lengths, trees padded to 64 rows, the batch padded too. The largest.
        _attn("attn_tree_batch", "qwen3_4b", 16, 64, 8192, "ragged", "wide", 16, "f16", 3, pad=8),
        # A short draft far into two long documents.
        _attn("attn_tree_long", "qwen3_4b", 2, 7, 65500, "even", "chain", 64, "f16", 2),
        # f32 activations (what the C++ engine passes), a bias by distance and a sliding window.
        _attn("attn_tree_f32", "gpt2", 24, 33, 1021, "ragged", "chain", 32, "f32", 4, window=600, slopes=1),
        # The cache's side of a step: one user, and the server's batch.
        _app("append_tree_one", "qwen3_0.6b", 1, 26, 777, "even", "wide", 16, "f16", 1),
        _app("append_tree_batch", "qwen3_4b", 32, 64, 4096, "ragged", "wide", 16, "f16", 5, pad=3),
        # One token for one user, every filter on.
        _sample("sample_one", 1, 151936, "f16", "all", 1),
        # The rows of a verification step for users with settings of their own, f32 logits.
        _sample("sample_batch", 128, 151936, "f32", "mixed", 2),
        # The path through one tree, and through 256.
        _batch("accept_one", "accept", "qwen3_0.6b", 1, 26, 777, "even", "wide", 16, "f16", 1),
        _batch("accept_batch", "accept", "qwen3_0.6b", 256, 64, 4096, "ragged", "wide", 16, "f16", 6),
        # The accepted tokens of one tree moved together in the pages, and of 64 chains and trees.
        _batch("keep_one", "keep", "qwen3_0.6b", 1, 26, 777, "even", "wide", 16, "f16", 1),
        _batch("keep_batch", "keep", "qwen3_4b", 64, 61, 2048, "ragged", "wide", 32, "f16", 7),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "append", "sample", "sample", "accept", "keep"])
    pick = rng.randint(1, 10**6)
    if kind == "sample":
        rows = _log_int(rng, 1, 128)
        vocab = rng.choice([151936, 50257, _log_int(rng, 300, 151936), _log_int(rng, 300, 151936)])
        c = _sample("", rows, vocab, rng.choice(["f16", "f32"]), rng.choice(["all", "mixed", "mixed", "plain"]), pick)
        del c["name"]
        return c
    heads = rng.choice(["qwen3_4b", "qwen3_4b", "qwen3_0.6b", "gpt2", "one_kv_256", "odd_80"])
    page, dtype, pad = rng.choice([16, 16, 32, 64, 128]), rng.choice(["f16", "f16", "f32"]), rng.choice([0, 0, rng.randint(1, 9)])
    how, shape = rng.choice(["even", "ragged", "ragged"]), rng.choice(["wide", "chain"])
    seqs = _log_int(rng, 1, 32 if kind in ("attention", "append") else 200)
    nodes = _log_int(rng, 1, 100 if seqs <= 8 else 50)
    most = {"attention": min(65000, 4000000 // (seqs * max(nodes, 4))), "append": 130000 // seqs, "keep": 130000 // seqs, "accept": 65000}[kind]
    a = ("", heads, seqs, nodes, _log_int(rng, 8, max(9, most)), how, shape, page, dtype, pick, pad)
    if kind == "attention":
        c = _attn(*a, cap=rng.choice([0.0, 0.0, 30.0]), window=rng.choice([0, 0, _log_int(rng, 1, 4096)]), slopes=rng.choice([0, 0, 1]))
    elif kind == "append":
        hd = HEADS[heads][2]
        c = _app(*a, norm=rng.randint(0, 1), rot=rng.choice([hd, hd, hd // 2 // 8 * 8]), inter=rng.randint(0, 1))
    else:
        c = _batch(a[0], kind, *a[1:])
    del c["name"]
    return c


def _trees(c):
    """(parents of the tree's rows, tokens before it) of each sequence. -1: no parent; -2: a row that is padding."""
    r = random.Random(c["pick"])
    got = []
    for s in range(c["seqs"]):
        n, ctx, real = c["nodes"], c["ctx"], c["nodes"]
        if c["how"] == "ragged":
            ctx = _log_int(r, max(1, ctx // 32), ctx)
            if s % 8 == 7:  # a place in the batch that no user has now
                got.append(([], 0))
                continue
            if s % 3 == 1:  # a smaller tree in a place of the fixed size
                real = max(1, n * r.randint(5, 9) // 10)
            elif s % 3 == 2:
                n = real = max(1, n * r.randint(3, 10) // 10)
        reach = 2 if c["shape"] == "chain" else 9
        got.append(([-1] + [max(0, i - r.randint(1, reach)) for i in range(1, real)] + [-2] * (n - real), ctx))
    return got


def _path(parents, r):
    """The rows that stay: the root and a walk down from it."""
    p = [0]
    while True:
        below = [i for i, x in enumerate(parents) if x == p[-1]]
        if not below or (len(p) > 1 and r.random() < 0.15):
            return p
        p.append(r.choice(below))


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


def _prepare_sample(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + 17)
    R, V = c["rows"], c["vocab"]

    def uniform(lo, hi):
        return torch.rand((R,), generator=g, device="cuda") * (hi - lo) + lo

    # Rows between sure of themselves and undecided; a few likely tokens above the rest; some rows with most of the
    # vocabulary masked, as a grammar does.
    x = torch.randn((R, V), generator=g, device="cuda") * uniform(1.2, 3.0)[:, None]
    top = torch.randint(0, V, (R, 12), generator=g, device="cuda")
    x.scatter_add_(1, top, torch.rand((R, 12), generator=g, device="cuda") * 14.0)
    masked = (torch.rand((R, V), generator=g, device="cuda") < 0.9) & (torch.arange(R, device="cuda") % 5 == 4)[:, None]
    masked[:, 0] = False
    x = torch.where(masked, -math.inf, x).to(DT[c["dtype"]])
    st = {"c": c, "logits": x, "u": torch.rand((R,), generator=g, device="cuda"), "temperature": uniform(0.6, 1.2),
          "top_p": uniform(0.8, 0.99), "top_k": None, "min_p": None, "out": torch.zeros((R,), dtype=torch.int32, device="cuda")}
    if c["mode"] != "plain":
        st["top_k"] = torch.randint(1, 200, (R,), generator=g, device="cuda", dtype=torch.int32)
        st["min_p"] = uniform(0.0, 0.1)
    if c["mode"] == "mixed":
        way = torch.randint(0, 8, (R,), generator=g, device="cuda")
        st["temperature"] = torch.where(way == 0, 0.0, st["temperature"])
        st["top_k"] = torch.where(way % 2 == 0, 0, st["top_k"])
        st["top_p"] = torch.where((way == 1) | (way == 2), 1.0, st["top_p"])
        st["min_p"] = torch.where(way < 6, 0.0, st["min_p"])
    return st


def prepare(c, seed):
    if c["kind"] == "sample":
        return _prepare_sample(c, seed)
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + 13)
    H, KV, hd = HEADS[c["heads"]]
    P, dt, trees = c["page"], DT[c["dtype"]], _trees(c)
    starts, parents, depth, lengths = [0], [], [], []
    most = max(max(len(p) for p, _ in trees), 1)
    words = (most + 31) // 32
    bits = np.zeros((sum(len(p) for p, _ in trees) + c["pad"], words), np.uint32)
    for p, ctx in trees:
        up = []
        for i, x in enumerate(p):
            depth.append(-1 if x < -1 else 0 if x < 0 else depth[starts[-1] + x] + 1)
            up.append(0 if x < -1 else (up[x] if x >= 0 else 0) | 1 << i)
            for w in range(words):
                bits[starts[-1] + i, w] = up[i] >> (32 * w) & 0xFFFFFFFF
        parents += p
        starts.append(starts[-1] + len(p))
        lengths.append(ctx + len(p))
    total, rows = starts[-1], starts[-1] + c["pad"]
    cuda = lambda x, t=torch.int32: torch.tensor(x, dtype=t, device="cuda")  # noqa: E731
    st = {"c": c, "H": H, "KV": KV, "hd": hd, "P": P, "rows": rows, "total": total, "max_new": most, "row_start": cuda(starts), "kv_len": cuda(lengths),
          "parents": cuda(parents + [-2] * c["pad"]), "depth": cuda(depth + [-1] * c["pad"]), "mask": torch.from_numpy(bits.view(np.int32)).cuda()}
    r = random.Random(seed * 31 + c["pick"])
    if c["kind"] == "accept":
        # Drafted tokens with some siblings alike; most sampled tokens are one of the children's.
        drafted = [r.randint(0, 150000) for _ in range(rows)]
        sampled = [r.randint(0, 150000) for _ in range(rows)]
        for s, (p, _) in enumerate(trees):
            for i in range(len(p) - 1, 0, -1):
                if r.random() < 0.05:
                    drafted[starts[s] + i] = drafted[starts[s] + i - 1]
                if p[i] >= 0 and r.random() < 0.4:
                    sampled[starts[s] + p[i]] = drafted[starts[s] + i]
        st |= {"tokens": cuda(drafted), "sampled": cuda(sampled)}
        return st
    used = [-(-n // P) for n in lengths]
    n_pages = sum(used) + 3  # a few are free
    k_pages, k_scales = _pages(g, n_pages, KV, P, hd, 1.0)
    v_pages, v_scales = _pages(g, n_pages, KV, P, hd, 0.7)
    order = torch.randperm(n_pages, generator=g, device="cuda").int()
    width = max(max(used), 1)
    slot = torch.arange(width, device="cuda")[None, :]
    n_used = torch.tensor(used, device="cuda")[:, None]
    first = torch.cumsum(n_used, 0) - n_used
    st |= {"k_pages": k_pages, "v_pages": v_pages, "k_scales": k_scales, "v_scales": v_scales, "free": order[-1].long(),
           "table": torch.where(slot < n_used, order[(first + slot).clamp(max=n_pages - 1)], -1).int().contiguous()}
    if c["kind"] == "attention":
        q = torch.randn((rows, H, hd), generator=g, device="cuda") * torch.randn((1, H, 1), generator=g, device="cuda").mul(0.3).exp()
        st["q"] = q.reshape(rows, H * hd).to(dt)
        st["out"] = torch.zeros((rows, H * hd), dtype=dt, device="cuda")
        st["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], device="cuda") if c["slopes"] else None
        st["scale"] = 1.0 / math.sqrt(hd)
    elif c["kind"] == "append":
        st["qkv"] = (torch.randn((rows, (H + 2 * KV) * hd), generator=g, device="cuda") * 1.5).to(dt)
        st["q_out"] = torch.zeros((rows, H * hd), dtype=dt, device="cuda")
        st["wqk"] = (torch.randn((2 * hd,), generator=g, device="cuda") * 0.1 + 1.0) if c["norm"] else None
        st["cs"] = _rope_table(max(lengths) + 1, c["rot"])
    else:
        paths = [_path(p, r) if p else [] for p, _ in trees]
        st["path"] = cuda([p + [-1] * (most - len(p)) for p in paths])
        st["count"] = cuda([len(p) for p in paths])
    return st


# ------------------------------------------------------------------ plain forms

def _place(st):
    """Of each row: its sequence, its place among the sequence's rows, the tokens before the tree."""
    start, length = st["row_start"].long(), st["kv_len"].long()
    row = torch.arange(st["total"], device="cuda")
    seq = torch.searchsorted(start[1:], row, right=True)
    return seq, row - start[seq], length[seq] - (start[seq + 1] - start[seq])


def _ancestors(st):
    """[rows, most rows of a tree]: whether a row sees a drafted token, itself among them."""
    k = torch.arange(st["max_new"], device="cuda")
    return (st["mask"][: st["total"]][:, k // 32] >> (k % 32).int() & 1).bool()


def _plain_attention(st):
    c, H, KV, hd = st["c"], st["H"], st["KV"], st["hd"]
    G, S, R, total = H // KV, st["table"].shape[0], st["max_new"], st["total"]
    out, length = st["out"], st["kv_len"].long()
    if not total:
        return out
    seq, i, base = _place(st)
    page = st["table"].long().clamp(min=0)

    def cached(codes, scales):  # [S, KV, keys, hd]
        x = codes.view(torch.uint8)[page].view(F8).float() * scales[page][..., None, None]
        return x.transpose(1, 2).reshape(S, KV, -1, hd)

    k, v = cached(st["k_pages"], st["k_scales"]), cached(st["v_pages"], st["v_scales"])
    keys = torch.arange(k.shape[2], device="cuda")
    v = torch.where((keys < length[:, None])[:, None, :, None], v, torch.zeros((), device="cuda"))
    # The place in the text of each key: its slot, or for drafted tokens that of their depth. What each row sees of it.
    start = st["row_start"].long()
    before = length - (start[1:] - start[:-1])
    place = keys.expand(S, -1).clone()
    place[seq, base + i] = base + st["depth"][:total].clamp(min=0)
    real = st["depth"][:total] >= 0
    sees = torch.zeros((S, R, keys.numel()), dtype=torch.bool, device="cuda")
    sees[seq, i] = (keys < before[seq][:, None]) & real[:, None]
    row, node = torch.nonzero(_ancestors(st) & real[:, None], as_tuple=True)
    sees[seq[row], i[row], base[row] + node] = True
    away = torch.zeros((S, R, keys.numel()), dtype=torch.long, device="cuda")
    away[seq, i] = place[seq] - (base + st["depth"][:total])[:, None]
    if c["window"]:
        sees &= away > -c["window"]
    q = torch.zeros((S, R, H, hd), device="cuda")
    q[seq, i] = st["q"][:total].float().reshape(-1, H, hd)
    q = q.reshape(S, R, KV, G, hd).permute(0, 2, 1, 3, 4).reshape(S, KV, R * G, hd)
    s = torch.matmul(q, k.transpose(2, 3)).reshape(S, KV, R, G, -1) * st["scale"]
    del k
    if c["cap"]:
        s = torch.tanh(s / c["cap"]) * c["cap"]
    if st["slopes"] is not None:
        s = s + st["slopes"].reshape(KV, 1, G, 1) * away[:, None, :, None, :]
    s = torch.where(sees[:, None, :, None, :], s, torch.full((), -math.inf, device="cuda"))
    m = s.amax(-1, keepdim=True)
    s = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    den = s.sum(-1, keepdim=True)
    o = torch.matmul(s.reshape(S, KV, R * G, -1), v).reshape(S, KV, R, G, hd) / torch.where(den == 0, 1.0, den)
    out[:total] = o.permute(0, 2, 1, 3, 4).reshape(S, R, H * hd)[seq, i].to(out.dtype)
    return out


def _rotated(x, cs, pos, rot, inter):
    """x [rows, heads, hd]: its first rot dimensions turned by the angles of pos."""
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


def _store(new, codes, scales, page, slot, first, old):
    """Tokens `new` [n, KV, hd] to their pages and slots. first: each sequence's first page that gets any; its slots
    before `old` hold tokens that stay."""
    P = codes.shape[2]
    bits = codes.view(torch.uint8)
    scale = _need(torch.zeros_like(scales).index_reduce_(0, page, new.abs().amax(-1), "amax"))
    scale[first] = torch.maximum(scale[first], scales[first])
    had = bits[first]
    again = (had.view(F8).float() * (scales[first] / scale[first])[:, :, None, None]).to(F8).view(torch.uint8)
    earlier = (torch.arange(P, device="cuda") < old[:, None])[:, None, :, None]
    bits[first] = torch.where(earlier, again, had)
    bits[page, :, slot] = (new / scale[page][..., None]).to(F8).view(torch.uint8)
    scales[page] = scale[page]


def _plain_append(st):
    c, H, KV, hd, P, n = st["c"], st["H"], st["KV"], st["hd"], st["P"], st["total"]
    seq, i, base = _place(st)
    dt = st["qkv"].dtype
    real = st["depth"][:n] >= 0
    place = base + st["depth"][:n].clamp(min=0)
    x = st["qkv"][:n].float().reshape(n, H + 2 * KV, hd)
    q, k, v = x[:, :H], x[:, H: H + KV], x[:, H + KV:]
    if st["wqk"] is not None:
        q, k = (t / torch.sqrt(t.square().mean(-1, keepdim=True) + EPS) * w for t, w in ((q, st["wqk"][:hd]), (k, st["wqk"][hd:])))
    q = _rotated(q, st["cs"], place, c["rot"], c["inter"]).to(dt).reshape(n, H * hd)
    st["q_out"][:n] = torch.where(real[:, None], q, st["q_out"][:n])
    k = _rotated(k, st["cs"], place, c["rot"], c["inter"]).to(dt).float()
    pos = base + i
    page, slot = st["table"].long()[seq, pos // P][real], (pos % P)[real]
    # Each sequence's first page of the call may hold earlier tokens, in the slots before `old`.
    start, length = st["row_start"].long(), st["kv_len"].long()
    p0 = length - (start[1:] - start[:-1])
    old = torch.where(length > p0, p0 % P, 0)
    first = st["table"].long().gather(1, (p0 // P).clamp(max=st["table"].shape[1] - 1)[:, None])[:, 0]
    first = torch.where(old > 0, first, st["free"])  # a page that stays as it is where there are none
    _store(k[real], st["k_pages"], st["k_scales"], page, slot, first, old)
    _store(v[real], st["v_pages"], st["v_scales"], page, slot, first, old)
    return st["q_out"], st["k_pages"], st["v_pages"], st["k_scales"], st["v_scales"]


def _plain_sample(st):
    x = st["logits"].double()
    x = torch.where(torch.isnan(x), -math.inf, x)
    R, V = x.shape
    index = torch.arange(V, device="cuda")
    m = x.amax(-1, keepdim=True)
    best = torch.where(x == m, index, V).amin(-1)
    t = st["temperature"].double()[:, None]
    w = torch.where(x == m, 1.0, torch.exp((x - m) / torch.where(t > 0, t, 1.0)))
    w = torch.where(x == -math.inf, 0.0, w)
    s, order = torch.sort(x, dim=-1, descending=True, stable=True)
    ws = w.gather(1, order)
    kept = s > -math.inf
    if st["top_k"] is not None:
        k = st["top_k"].long()[:, None]
        kept &= (index < k) | (k <= 0)
    cum = torch.cumsum(torch.where(kept, ws, 0.0), -1)
    p = st["top_p"].double()[:, None]
    kept &= (torch.nn.functional.pad(cum, (1, 0))[:, :-1] < p * cum[:, -1:]) | (p >= 1) | (index == 0)
    if st["min_p"] is not None:
        kept &= ws >= st["min_p"].double().clamp(max=1.0)[:, None]
    w = torch.where(torch.zeros_like(kept).scatter_(1, order, kept), w, 0.0)
    cum = torch.cumsum(w, -1)
    token = torch.searchsorted(cum, st["u"].double()[:, None] * cum[:, -1:], right=True)[:, 0].clamp(max=V - 1)
    token = torch.where(t[:, 0] > 0, token, best)
    st["out"].copy_(torch.where(m[:, 0] == -math.inf, -1, token))
    return st["out"]


def _plain_accept(st):
    S, R, total = st["row_start"].numel() - 1, st["max_new"], st["total"]
    seq, i, base = _place(st)
    start, length = st["row_start"].long(), st["kv_len"].long()
    parent, token, sampled = (st[k][:total].long() for k in ("parents", "tokens", "sampled"))
    # A row goes on from its parent if it holds what was sampled there, the first of its parent's children that does.
    agrees = (parent >= 0) & (token == sampled[(start[seq] + parent).clamp(min=0, max=max(total - 1, 0))])
    by = torch.full((S, R), -1, device="cuda")
    by[seq, i] = torch.where(agrees, parent, -1)
    earlier = torch.arange(R, device="cuda") < i[:, None]
    good = (agrees & ~((by[seq] == parent[:, None]) & earlier).any(-1)) | (i == 0)
    # It is on the path if all of its ancestors are good.
    all_good = torch.zeros((S, R), dtype=torch.bool, device="cuda")
    all_good[seq, i] = good
    on = torch.zeros((S, R), dtype=torch.bool, device="cuda")
    anc = _ancestors(st)
    on[seq, i] = (~anc | all_good[seq]).all(-1) & anc.any(-1) & (anc[:, 0] | (i == 0))
    count = on.sum(-1)
    node = torch.arange(R, device="cuda")
    path = torch.sort(torch.where(on, node, R), -1).values
    path = torch.where(path < R, path, -1)
    last = (start[:-1] + path.gather(1, (count - 1).clamp(min=0)[:, None])[:, 0]).clamp(min=0, max=max(total - 1, 0))
    after = torch.where(count > 0, sampled[last] if total else -1, -1)
    return path.int(), count.int(), after.int(), (length - (start[1:] - start[:-1]) + count).int()


def _plain_keep(st):
    P, S = st["P"], st["row_start"].numel() - 1
    start, length = st["row_start"].long(), st["kv_len"].long()
    base = length - (start[1:] - start[:-1])
    path = st["path"].long()
    to = torch.arange(path.shape[1], device="cuda").expand(S, -1)
    moved = (to < st["count"][:, None]) & (path > to)
    seq = torch.arange(S, device="cuda")[:, None].expand_as(path)[moved]
    src, dst = base[seq] + path[moved], base[seq] + to[moved]
    table = st["table"].long()
    # The first token that moves; what stands before it in its page stays.
    p0 = base + torch.where(moved, to, path.shape[1]).amin(-1)
    some = moved.any(-1)
    old = torch.where(some, p0 % P, 0)
    first = torch.where(old > 0, table.gather(1, (p0 // P).clamp(max=table.shape[1] - 1)[:, None])[:, 0], st["free"])
    from_page, from_slot, page, slot = table[seq, src // P], src % P, table[seq, dst // P], dst % P
    for codes, scales in ((st["k_pages"], st["k_scales"]), (st["v_pages"], st["v_scales"])):
        x = codes.view(torch.uint8)[from_page, :, from_slot].view(F8).float() * scales[from_page][..., None]
        _store(x, codes, scales, page, slot, first, old)
    return st["k_pages"], st["v_pages"], st["k_scales"], st["v_scales"]


PLAIN = {"attention": _plain_attention, "append": _plain_append, "sample": _plain_sample, "accept": _plain_accept, "keep": _plain_keep}


def run(st):
    c = st["c"]
    if not own:
        return PLAIN[c["kind"]](st)
    if "call" not in st:
        from nekochat_amd import ops

        if c["kind"] == "sample":
            st["call"], st["got"] = ops.prepare(ops.sample, st["logits"], st["u"], temperature=st["temperature"], top_k=st["top_k"],
                                                top_p=st["top_p"], min_p=st["min_p"], out=st["out"])
        elif c["kind"] == "accept":
            st["call"], st["got"] = ops.prepare(ops.accept_tree, st["tokens"], st["sampled"], st["parents"], st["row_start"],
                                                st["kv_len"], st["max_new"])
        else:
            cache = ops.PagedKV(st["k_pages"], st["v_pages"], st["k_scales"], st["v_scales"])
            batch = (cache, st["table"], st["row_start"], st["kv_len"])
            st["got"] = (st["k_pages"], st["v_pages"], st["k_scales"], st["v_scales"])
            if c["kind"] == "attention":
                st["call"], st["got"] = ops.prepare(ops.attention_tree_paged, st["q"], *batch, st["depth"], st["mask"], st["H"],
                                                    scale=st["scale"], softcap=c["cap"], window=c["window"], slopes=st["slopes"],
                                                    out=st["out"])
            elif c["kind"] == "append":
                st["call"], _ = ops.prepare(ops.qk_norm_rope_tree_paged, st["qkv"], st["H"], *batch, st["depth"], st["cs"], EPS,
                                            wqk=st["wqk"], interleaved=bool(c["inter"]), q_out=st["q_out"])
                st["got"] = (st["q_out"], *st["got"])
            else:
                st["call"], _ = ops.prepare(ops.keep_paged, *batch, st["path"], st["count"])
    st["call"]()
    return st["got"]


# ------------------------------------------------------------------ work

def work(c):
    if c["kind"] == "sample":
        n = c["rows"] * c["vocab"]  # each logit read once; its weight is a difference, a quotient, an exponential, a sum
        return {"bytes": n * (2 if c["dtype"] == "f16" else 4) + 24 * c["rows"], "flops": 4 * n}
    H, KV, hd = HEADS[c["heads"]]
    size, trees, w, P = 2 if c["dtype"] == "f16" else 4, _trees(c), c.get("window", 0), c["page"]
    rows = sum(len(p) for p, _ in trees)
    real = sum(sum(x > -2 for x in p) for p, _ in trees)
    small = 4 * (2 * len(trees) + 1)
    words = (max(max(len(p) for p, _ in trees), 1) + 31) // 32
    if c["kind"] == "accept":  # three numbers of each row read; a path, a count, a token and a length written for each sequence
        return {"bytes": 12 * rows + small + 4 * len(trees) * (max(max(len(p) for p, _ in trees), 1) + 3), "flops": 0}
    if c["kind"] == "keep":  # about a token for each level of a tree, read and written
        levels = sum(_levels(p) for p, _ in trees)
        return {"bytes": 4 * levels * KV * hd + small + 4 * levels, "flops": 2 * levels * KV * hd}
    if c["kind"] == "append":
        pages = sum(-(-(ctx + len(p)) // P) - ctx // P for p, ctx in trees if p)
        # q, k, v read, q written, k and v codes written, a scale for each page and head, the angles of each level
        return {"bytes": real * (H + 2 * KV) * hd * size + real * H * hd * size + 2 * real * KV * hd + pages * (8 * KV + 4) +
                4 * c["rot"] * sum(_levels(p) for p, _ in trees) + 4 * rows + small, "flops": 10 * real * (H + KV) * hd}
    keys = pairs = pages = 0
    for p, ctx in trees:
        if not p:
            continue
        depth = []
        for x in p:
            depth.append(-1 if x < -1 else 0 if x < 0 else depth[x] + 1)
        begin = max(0, ctx - w + 1) if w else 0
        keys += ctx + len(p) - begin
        pages += -(-(ctx + len(p)) // P) - begin // P
        for d in depth:
            if d >= 0:
                pairs += min(ctx + d + 1, w) if w else ctx + d + 1
    return {"bytes": 2 * rows * H * hd * size + 2 * keys * KV * hd + pages * (8 * KV + 4) + rows * (4 + 4 * words) + small,
            "flops": 4 * hd * H * pairs}


def _levels(parents):
    depth = []
    for x in parents:
        depth.append(-1 if x < -1 else 0 if x < 0 else depth[x] + 1)
    return max(depth, default=-1) + 1


# ------------------------------------------------------------------ 64 bits

def _value(codes):
    """The value of each E4M3 code, from its bits."""
    b = codes.view(torch.uint8).long()
    e, m = (b >> 3) & 15, b & 7
    mag = torch.where(e > 0, (8 + m).double() * 2.0 ** (e - 10).double(), m.double() * 2.0**-9)
    return torch.where(b > 127, -mag, mag)


def _exact_sample(st):
    x = st["logits"].cpu().numpy().astype(np.float64)
    get = lambda k, none: np.full(len(x), none) if st[k] is None else st[k].cpu().numpy().astype(np.float64)  # noqa: E731
    t, k, p, mp, u = get("temperature", 1.0), get("top_k", 0), get("top_p", 1.0), get("min_p", 0.0), get("u", 0.0)
    got = []
    for r, row in enumerate(x):
        order = np.argsort(-row, kind="stable")
        order = order[row[order] > -np.inf]
        if t[r] <= 0:
            got.append(int(order[0]))
            continue
        if k[r] > 0:
            order = order[: int(k[r])]
        w = np.exp((row[order] - row[order[0]]) / t[r])
        if p[r] < 1:
            order = order[: 1 + int(np.searchsorted(np.cumsum(w), p[r] * w.sum(), side="left"))]
            w = w[: len(order)]
        order = np.sort(order[w >= min(mp[r], 1.0)])
        w = np.cumsum(np.exp((row[order] - row[order].max()) / t[r]))
        got.append(int(order[min(int(np.searchsorted(w, u[r] * w[-1], side="right")), len(order) - 1)]))
    return torch.tensor(got, dtype=torch.int32)


def _exact_accept(c, st):
    token, sampled = st["tokens"].tolist(), st["sampled"].tolist()
    path, count, after, new_len, row = [], [], [], [], 0
    for p, ctx in _trees(c):
        at, walk = 0, [0] if p else []
        while p:
            below = [i for i, x in enumerate(p) if x == at and i and token[row + i] == sampled[row + at]]
            if not below:
                break
            at = below[0]
            walk.append(at)
        path.append(walk + [-1] * (st["max_new"] - len(walk)))
        count.append(len(walk))
        after.append(sampled[row + at] if p else -1)
        new_len.append(ctx + len(walk))
        row += len(p)
    return tuple(torch.tensor(x, dtype=torch.int32) for x in (path, count, after, new_len))


def _exact_attention(c, st):
    H, KV, hd = HEADS[c["heads"]]
    P, G, row = c["page"], H // KV, 0
    out = torch.zeros((st["rows"], H * hd), dtype=torch.float64, device="cuda")
    for s, (p, ctx) in enumerate(_trees(c)):
        n, length = len(p), ctx + len(p)
        if not n:
            continue
        place, up = list(range(ctx)), []
        for i, x in enumerate(p):
            up.append([] if x < -1 else (up[x] if x >= 0 else []) + [i])
            place.append(ctx + len(up[i]) - 1)
        place = torch.tensor(place, device="cuda")
        sees = torch.zeros((n, length), dtype=torch.bool)
        for i, x in enumerate(up):
            sees[i, :ctx] = bool(x)
            sees[i, [ctx + j for j in x]] = True
        sees = sees.cuda()
        away = place[ctx:, None] - place[None]
        if c["window"]:
            sees = sees & (away < c["window"])
        ids = st["table"][s, : -(-length // P)].long()
        some = sees.any(-1, keepdim=True)
        for h in range(H):
            g = h // G
            k, v = ((_value(codes[ids, g]) * scales[ids, g].double()[:, None, None]).reshape(-1, hd)[:length]
                    for codes, scales in ((st["k_pages"], st["k_scales"]), (st["v_pages"], st["v_scales"])))
            x = st["q"][row: row + n, h * hd: (h + 1) * hd].double() @ k.T * st["scale"]
            if c["cap"]:
                x = c["cap"] * torch.tanh(x / c["cap"])
            if st["slopes"] is not None:
                x = x - float(st["slopes"][h]) * away
            w = torch.softmax(torch.where(some, x.masked_fill(~sees, -math.inf), 0.0), -1)
            out[row: row + n, h * hd: (h + 1) * hd] = torch.where(some, w @ v, 0.0)
        row += n
    return out


def _exact_page(part, dt, codes, scales, page, a):
    """Values part [n, KV, hd] into a page from slot a on (NaN: slots that nothing is written to)."""
    top = torch.nan_to_num(part).to(dt).double().abs().amax((0, 2))
    scale = 2.0 ** torch.ceil(torch.log2(top / 448)).clamp(-64, 64)
    if a:
        scale = torch.maximum(scale, scales[page])
        codes[page, :, :a] *= (scales[page] / scale)[:, None, None]
    now = codes[page, :, a: a + len(part)]
    new = (part / scale[:, None]).transpose(0, 1)
    codes[page, :, a: a + len(part)] = torch.where(torch.isnan(new), now, new)
    scales[page] = scale


def exact(c, seed):
    st = prepare(c, seed)
    if c["kind"] == "sample":
        return _exact_sample(st)
    if c["kind"] == "accept":
        return _exact_accept(c, st)
    if c["kind"] == "attention":
        return _exact_attention(c, st)
    H, KV, hd = HEADS[c["heads"]]
    P, row = c["page"], 0
    kc, vc, ks, vs = _value(st["k_pages"]), _value(st["v_pages"]), st["k_scales"].double(), st["v_scales"].double()
    if c["kind"] == "keep":
        for s, (p, ctx) in enumerate(_trees(c)):
            path = st["path"][s, : int(st["count"][s])].tolist()
            moved = [(ctx + to, ctx + x) for to, x in enumerate(path) if x > to]
            if not moved:
                continue
            table = st["table"][s].tolist()
            for codes, scales in ((kc, ks), (vc, vs)):
                new = torch.stack([codes[table[x // P], :, x % P] * scales[table[x // P]][:, None] for _, x in moved])
                for j in range(moved[0][0] // P, moved[-1][0] // P + 1):
                    here = [i for i, (to, _) in enumerate(moved) if to // P == j]
                    _exact_page(new[here[0]: here[-1] + 1], torch.float64, codes, scales, table[j], moved[here[0]][0] % P)
        return kc, vc, ks, vs
    rot, dt = c["rot"], DT[c["dtype"]]
    q_out = torch.zeros((st["rows"], H * hd), dtype=torch.float64, device="cuda")
    for s, (p, ctx) in enumerate(_trees(c)):
        n = len(p)
        if not n:
            continue
        depth = st["depth"][row: row + n].long()
        x = st["qkv"][row: row + n].double().reshape(n, H + 2 * KV, hd)
        qk, v = x[:, : H + KV], x[:, H + KV:]
        if st["wqk"] is not None:
            w = st["wqk"].double().reshape(2, 1, hd).repeat_interleave(torch.tensor([H, KV], device="cuda"), 0).reshape(H + KV, hd)
            qk = qk * (qk.pow(2).sum(-1, keepdim=True) / hd + EPS).rsqrt() * w
        z = st["cs"][ctx + depth.clamp(min=0)].double().reshape(n, 1, rot // 2, 2)
        pairs = qk[..., :rot].reshape(n, H + KV, rot // 2, 2) if c["inter"] else qk[..., :rot].reshape(n, H + KV, 2, rot // 2).transpose(2, 3)
        turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * torch.view_as_complex(z.contiguous()))
        turned = turned if c["inter"] else turned.transpose(2, 3)
        qk = torch.cat([turned.reshape(n, H + KV, rot), qk[..., rot:]], -1)
        real = (depth >= 0)[:, None]
        q_out[row: row + n] = torch.where(real, qk[:, :H].reshape(n, H * hd), 0.0)
        row += n
        for new, codes, scales in ((qk[:, H:], kc, ks), (v, vc, vs)):
            new = torch.where(real[..., None], new, math.nan)
            for j in range(ctx // P, -(-(ctx + n) // P)):
                a, b = max(0, ctx - j * P), min(P, ctx + n - j * P)  # the new slots of page j
                part = new[j * P + a - ctx: j * P + b - ctx]
                if not torch.isnan(part).all():
                    _exact_page(part, dt, codes, scales, int(st["table"][s, j]), a)
    return q_out, kc, vc, ks, vs
