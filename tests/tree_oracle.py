"""Plain evaluation in 64 bits, on the CPU, of drafted trees over the paged 8-bit KV cache and of sampling
(include/neko_hip.h). Written from the formulas, one row at a time."""
import numpy as np
import torch

import paged_oracle as P

U, H16 = 2.0 ** -24, 2.0 ** -11


def random_parents(n, reach, rng, padding=0):
    """A tree of n rows, parents at most `reach` rows before their children, and padding rows behind it."""
    return [-1] + [int(rng.integers(max(0, i - reach), i)) for i in range(1, n)] + [-2] * padding


def plan(parents):
    """(depth, the rows that each row sees) of one tree."""
    depth, sees = [], []
    for i, p in enumerate(parents):
        if p == -1:
            depth.append(0)
            sees.append({i})
        elif 0 <= p < i and depth[p] >= 0:
            depth.append(depth[p] + 1)
            sees.append(sees[p] | {i})
        else:
            depth.append(-1)
            sees.append(set())
    return depth, sees


class Trees:
    """Batches of trees: `trees` has (parents, tokens before the tree) of each sequence."""

    def __init__(self, trees, page, seed, pad=0, slack=1, words=None):
        self.trees = trees
        self.batch = P.Batch([(len(p), ctx + len(p)) for p, ctx in trees], page, seed, pad=pad, slack=slack)
        self.rows = self.batch.rows
        self.words = words or max(1, -(-max(len(p) for p, _ in trees) // 32))
        self.depth, self.sees = [], []
        for p, _ in trees:
            d, s = plan(p)
            self.depth += d
            self.sees += s
        self.depth += [-1] * pad
        self.sees += [set()] * pad
        self.parents = [x for p, _ in trees for x in p] + [-2] * pad

    def mask(self):
        m = np.zeros((self.rows, self.words), np.uint32)
        for r, s in enumerate(self.sees):
            for k in s:
                if k < 32 * self.words:
                    m[r, k // 32] |= np.uint32(1 << (k % 32))
        return torch.from_numpy(m.view(np.int32))

    def tensors(self, dev):
        """page_table, row_start, kv_len, depth."""
        return (*self.batch.tensors(dev), torch.tensor(self.depth, dtype=torch.int32, device=dev))


def attention(q, cache, t, n_head, scale, softcap=0.0, window=0, slopes=None):
    """(out, a, s) as paged_oracle.attention."""
    k_pages, v_pages, k_scales, v_scales = cache
    n_kv, hd, page = k_pages.shape[1], k_pages.shape[3], k_pages.shape[2]
    b, G = t.batch, n_head // k_pages.shape[1]
    out = torch.zeros((b.rows, n_head, hd), dtype=torch.float64)
    a, s_abs = torch.zeros_like(out), torch.zeros((b.rows, n_head, 1), dtype=torch.float64)
    for s, (n, length) in enumerate(b.seqs):
        base, r0 = length - n, int(b.row_start[s])
        if n == 0 or base < 0:
            continue
        keys = [j for j in range(min(length, b.table.shape[1] * page)) if 0 <= b.table[s, j // page] < b.n_pages]
        if not keys:
            continue
        ids = torch.tensor([int(b.table[s, j // page]) for j in keys])
        slot = torch.tensor([j % page for j in keys])
        depth = t.depth[r0: r0 + n]
        place = torch.tensor([j if j < base else base + depth[j - base] for j in keys])
        sees = torch.zeros((n, len(keys)), dtype=torch.bool)
        for i in range(n):
            if 0 <= depth[i] < n:
                sees[i] = torch.tensor([j < base or ((j - base) in t.sees[r0 + i] and j - base < 32 * t.words) for j in keys])
        pos = torch.tensor([base + d for d in depth])
        if window:
            sees &= place[None] > pos[:, None] - window
        k = k_pages.float()[ids, :, slot].double() * k_scales.double()[ids][..., None]
        v = v_pages.float()[ids, :, slot].double() * v_scales.double()[ids][..., None]
        for h in range(n_head):
            x = q[r0: r0 + n].double().reshape(n, n_head, hd)[:, h]
            kk, vv = k[:, h // G], v[:, h // G]
            y = (x @ kk.T) * scale
            s_abs[r0: r0 + n, h, 0] = torch.where(sees, (x.abs() @ kk.abs().T) * abs(scale), 0.0).amax(-1)
            if softcap:
                y = softcap * torch.tanh(y / softcap)
            if slopes is not None:
                y = y + float(slopes[h]) * (place[None] - pos[:, None])
                s_abs[r0: r0 + n, h, 0] += float(slopes[h]) * length
            for i in range(n):
                if sees[i].any():
                    w = torch.softmax(y[i][sees[i]], 0)
                    out[r0 + i, h] = w @ vv[sees[i]]
                    a[r0 + i, h] = w @ vv[sees[i]].abs()
    return out.reshape(b.rows, -1), a.reshape(b.rows, -1), s_abs.expand(-1, -1, hd).reshape(b.rows, -1)


def bar(out, a, s, n_keys, hd, dtype):
    """How far a result may be off (derived in test_gpu_tree.py)."""
    e = (hd + 4) * U * s + 8 * U + (n_keys / 32 + 64) * U
    x = 2 * e * a + 2 * U * out.abs()
    return x + H16 * out.abs() + 2.0 ** -25 + H16 * a if dtype == "f16" else x


def store(codes, scales, page, first, values):
    """Values {slot: [n_kv, hd]} into a page of a copy in 64 bits, whose slots before `first` stay: the page's codes (as
    E4M3 tensors) and scales after it. codes [n_kv, page, hd]; scales [n_kv]."""
    new = torch.stack([values[k] for k in sorted(values)])
    top = torch.where(torch.isfinite(new), new.abs(), 0.0).amax((0, 2))
    scale = torch.tensor([P.need_scale(float(x)) for x in top], dtype=torch.float64)
    if first:
        scale = torch.maximum(scale, scales.double())
    out = codes.clone()
    if first:
        ratio = (scales.double() / scale)[:, None, None]
        out[:, :first] = (codes[:, :first].float().double() * ratio).float().to(P.F8)
    for slot, x in values.items():
        out[:, slot] = (x / scale[:, None]).float().to(P.F8)
    return out, scale.float()


def keep(cache, t, path, count):
    """The cache after the paths' tokens are moved together."""
    k_pages, v_pages, k_scales, v_scales = (x.clone() for x in cache)
    b, page = t.batch, k_pages.shape[2]
    good = lambda s, j: j // page < b.table.shape[1] and 0 <= b.table[s, j // page] < b.n_pages  # noqa: E731
    for s, (n, length) in enumerate(b.seqs):
        base = length - n
        if base < 0:
            continue
        moved = [(k, int(path[s, k])) for k in range(max(0, min(int(count[s]), n, path.shape[1]))) if k < path[s, k] < n]
        for codes, scales in ((k_pages, k_scales), (v_pages, v_scales)):
            was = codes.float().double(), scales.double().clone()
            for j in sorted({(base + k) // page for k, _ in moved}):
                if not good(s, j * page):
                    continue
                here = [(k, x) for k, x in moved if (base + k) // page == j]
                begin = (base + moved[0][0]) % page if j == (base + moved[0][0]) // page else 0
                values = {}
                for k, x in here:
                    if good(s, base + x):
                        src = int(b.table[s, (base + x) // page])
                        values[(base + k) % page] = was[0][src, :, (base + x) % page] * was[1][src][:, None]
                if values:
                    id_ = int(b.table[s, j])
                    codes[id_], scales[id_] = store(codes[id_], scales[id_], id_, begin, values)
    return k_pages, v_pages, k_scales, v_scales


def walk(parents, tokens, sampled, most):
    """(path, next token) through one tree; none where its first row is padding."""
    if not parents or parents[0] != -1:
        return [], -1
    path = [0]
    while len(path) < most:
        below = [i for i in range(path[-1] + 1, len(parents)) if parents[i] == path[-1] and tokens[i] == sampled[path[-1]]]
        if not below or sampled[path[-1]] < 0:
            break
        path.append(below[0])
    return path, sampled[path[-1]]


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, shift=0.0, shift_p=0.0):
    """(token, how near to a border it was decided, how near to one top-p cut, relative to the weights' sums) of one row of
    float64 logits. shift, shift_p: what u and top_p are moved by."""
    x = np.where(np.isnan(logits), -np.inf, logits.astype(np.float64))
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf]
    if len(order) == 0:
        return -1, 1.0, 1.0
    top = x[order[0]]
    if not temperature > 0:
        return int(order[0]), 1.0, 1.0
    near = near_p = 1.0

    def weights(i):
        with np.errstate(invalid="ignore"):
            w = np.exp((x[i] - top) / temperature)
        return np.where(x[i] == top, 1.0, np.where(np.isnan(w), 0.0, w))

    if 0 < top_k < len(order):
        order = order[:top_k]
    w = weights(order)
    if top_p < 1:
        cum = np.cumsum(w)
        at = min(int(np.searchsorted(cum, (top_p + shift_p) * cum[-1], side="left")), len(cum) - 1) if top_p > 0 else 0
        if top_p > 0:
            near_p = float(np.abs(cum - top_p * cum[-1]).min() / cum[-1])
        order, w = order[: at + 1], w[: at + 1]
    if min_p > 0:
        order = order[w >= min(min_p, 1.0)]
    order = np.sort(order)
    cum = np.cumsum(weights(order))
    target = max(0.0, (min(max(u, 0.0), 1 - 2.0 ** -24) if u == u else 0.0) + shift) * cum[-1]
    if target > 0:
        near = min(near, float(np.abs(cum - target).min() / cum[-1]))
    return int(order[min(int(np.searchsorted(cum, target, side="right")), len(order) - 1)]), near, near_p
