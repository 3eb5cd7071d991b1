"""Plain evaluation in 64 bits of the paged 8-bit KV cache's operators (include/neko_hip.h), on the CPU, and batches to
try them on. Written from the formulas, one token and one head at a time where that is clearest."""
import numpy as np
import torch

F8 = torch.float8_e4m3fn


class Batch:
    """seqs: (new rows, length with them) of each sequence, in a cache of pages in random order; `free` more pages."""

    def __init__(self, seqs, page, seed, pad=0, free=2, slack=1):
        g = np.random.default_rng(seed)
        self.seqs, self.page = seqs, page
        used = [-(-length // page) for _, length in seqs]
        self.n_pages = sum(used) + free
        order = g.permutation(self.n_pages)
        width = max(max(used), 1) + slack
        self.table = np.full((len(seqs), width), -1, np.int32)
        at = 0
        for s, n in enumerate(used):
            self.table[s, :n] = order[at: at + n]
            at += n
        self.free = order[at:]
        self.row_start = np.cumsum([0] + [n for n, _ in seqs]).astype(np.int32)
        self.kv_len = np.array([length for _, length in seqs], np.int32)
        self.rows = int(self.row_start[-1]) + pad

    def tensors(self, dev):
        return tuple(torch.from_numpy(x).to(dev) for x in (self.table, self.row_start, self.kv_len))

    def places(self):
        """(row, sequence, position, page, slot) of each new row."""
        for s, (n, length) in enumerate(self.seqs):
            for i in range(n):
                pos = length - n + i
                yield int(self.row_start[s]) + i, s, pos, int(self.table[s, pos // self.page]), pos % self.page


def codes_of(x, scale):
    """Values -> E4M3 codes under a scale (torch's conversion: nearest, ties to even)."""
    return (x / scale).float().to(F8)


def need_scale(amax):
    """The smallest power of two with amax <= 448 * it, within 2^+-64."""
    e = -64
    while amax > 448 * 2.0 ** e and e < 64:
        e += 1
    return 2.0 ** e


def random_cache(n_pages, n_kv, page, hd, seed, spread=0.5):
    """(k_pages, v_pages, k_scales, v_scales) on the CPU, as the append would have left them."""
    g = torch.Generator().manual_seed(seed)
    pages, scales = [], []
    for _ in range(2):
        x = torch.randn((n_pages, n_kv, page, hd), generator=g) * torch.exp(torch.randn((n_pages, n_kv, 1, 1), generator=g) * spread)
        s = torch.tensor([[need_scale(float(v)) for v in row] for row in x.abs().amax((2, 3))], dtype=torch.float32)
        pages.append(codes_of(x, s[..., None, None]))
        scales.append(s)
    return pages[0], pages[1], scales[0], scales[1]


def turned(x, cs, pos, rot, inter):
    """x [heads, hd] of one token, float64, and what its roundings are relative to."""
    y, size = x.clone(), x.abs().clone()
    if rot:
        i = torch.arange(rot // 2)
        a, b = (2 * i, 2 * i + 1) if inter else (i, i + rot // 2)
        c, s = cs[pos, 0::2].double(), cs[pos, 1::2].double()
        y[:, a], y[:, b] = x[:, a] * c - x[:, b] * s, x[:, a] * s + x[:, b] * c
        size[:, a] = size[:, b] = x[:, a].abs() + x[:, b].abs()
    return y, size


def append(qkv, n_q, n_kv, hd, batch, cache, cs, eps, wqk, inter, dtype):
    """(q [rows, n_q, hd], its error scale, k values and v values of the new tokens by (page, slot), scales): the q
    rows in 64 bits (NaN: row not written); new (page, head) scales for k and v from values rounded to dtype."""
    rot = 0 if cs is None else cs.shape[1]
    q = torch.full((batch.rows, n_q, hd), float("nan"), dtype=torch.float64)
    size = torch.zeros_like(q)
    new = ({}, {})
    for row, s, pos, page, slot in batch.places():
        x = qkv[row].double()[: (n_q + 2 * n_kv) * hd].reshape(n_q + 2 * n_kv, hd)
        qk, v = x[: n_q + n_kv], x[n_q + n_kv:]
        if wqk is not None:
            w = wqk.double().reshape(2, hd)
            qk = qk / torch.sqrt(qk.square().mean(-1, keepdim=True) + eps) * torch.cat([w[:1].expand(n_q, hd), w[1:].expand(n_kv, hd)])
        y, z = turned(qk, cs, pos, rot, inter)
        q[row], size[row] = y[:n_q], z[:n_q]
        new[0][page, slot], new[1][page, slot] = y[n_q:], v
    scales = []
    for values, old in zip(new, (cache[2], cache[3])):
        scale = old.clone()
        for page in {p for p, _ in values}:
            slots = sorted(t for p, t in values if p == page)
            for h in range(n_kv):
                part = torch.stack([values[page, t][h] for t in slots]).to(dtype).double().abs()
                part = part[torch.isfinite(part)]
                need = need_scale(float(part.max()) if part.numel() else 0.0)
                scale[page, h] = max(need, float(old[page, h])) if slots[0] > 0 else need
        scales.append(scale)
    return q, size, new, scales


def attention(q, cache, batch, n_head, scale, softcap=0.0, window=0, slopes=None):
    """(out, a, s): rows in 64 bits; a = sum w |v| / sum w, the size that the weights' relative errors act on; s =
    the largest |scale| * sum |q_d k_d| of a row's keys, what the scores' roundings are relative to."""
    k_pages, v_pages, k_scales, v_scales = cache
    n_kv, hd = k_pages.shape[1], k_pages.shape[3]
    G = n_head // n_kv
    out = torch.zeros((batch.rows, n_head, hd), dtype=torch.float64)
    a, s_abs = torch.zeros_like(out), torch.zeros((batch.rows, n_head, 1), dtype=torch.float64)
    for s, (n, length) in enumerate(batch.seqs):
        if n == 0:
            continue
        reach = batch.table.shape[1] * batch.page
        keys = [j for j in range(min(length, reach)) if 0 <= batch.table[s, j // batch.page] < batch.n_pages]
        r0 = int(batch.row_start[s])
        if not keys:
            continue
        page = torch.tensor([int(batch.table[s, j // batch.page]) for j in keys])
        slot = torch.tensor([j % batch.page for j in keys])
        j = torch.tensor(keys)
        pos = length - n + torch.arange(n)
        sees = j[None, :] <= pos[:, None]
        if window:
            sees &= j[None, :] > pos[:, None] - window
        for h in range(n_head):
            g = h // G
            k = k_pages.float()[page, g, slot].double() * k_scales[page, g].double()[:, None]
            v = v_pages.float()[page, g, slot].double() * v_scales[page, g].double()[:, None]
            x = q[r0: r0 + n].double().reshape(n, n_head, hd)[:, h]
            t = (x @ k.T) * scale
            s_abs[r0: r0 + n, h, 0] = torch.where(sees, (x.abs() @ k.abs().T) * abs(scale), 0.0).amax(-1)
            if softcap:
                t = softcap * torch.tanh(t / softcap)
            if slopes is not None:
                t = t + float(slopes[h]) * (j[None, :] - pos[:, None])
                s_abs[r0: r0 + n, h, 0] += float(slopes[h]) * length
            t = torch.where(sees, t, -float("inf"))
            m = t.amax(-1, keepdim=True)
            w = torch.where(sees, torch.exp(t - torch.where(m == -float("inf"), 0.0, m)), 0.0)
            w = torch.where(sees.any(-1, keepdim=True), w / w.sum(-1, keepdim=True), 0.0)
            # (a weight of a key that is not seen is nothing, whatever its value)
            o = torch.stack([w[i][sees[i]] @ v[sees[i]] for i in range(n)])
            out[r0: r0 + n, h] = o
            a[r0: r0 + n, h] = torch.stack([w[i][sees[i]] @ v[sees[i]].abs() for i in range(n)])
    return out.reshape(batch.rows, -1), a.reshape(batch.rows, -1), s_abs.expand(-1, -1, hd).reshape(batch.rows, -1)
