"""Drafted trees' plans on the host (neko_tree_plan, ops.tree_plan), and what the tree and sampling entry points refuse
without a device."""
import ctypes

import numpy as np
import pytest

import tree_oracle as T
from nekochat_amd import NekoError, _lib, ops


@pytest.mark.parametrize("sizes", [[1], [5, 0, 33], [64, 32, 31], [0, 0, 2], [300, 7]])
def test_plan(sizes):
    rng = np.random.default_rng(sum(sizes))
    parents, start = [], [0]
    for n in sizes:
        p = [int(rng.integers(-3, i + 2)) for i in range(n)]  # parents, roots, padding and nonsense
        parents += p
        start.append(start[-1] + n)
    depth, mask = ops.tree_plan(np.array(parents + [0, -1], np.int32), np.array(start, np.int32))
    assert mask.shape == (len(parents) + 2, max(1, -(-max(sizes) // 32)))
    for s, n in enumerate(sizes):
        want_depth, sees = T.plan(parents[start[s]: start[s] + n])
        assert depth[start[s]: start[s] + n].tolist() == want_depth
        for i in range(n):
            bits = mask[start[s] + i].view(np.uint32)
            assert {k for k in range(32 * len(bits)) if bits[k // 32] >> (k % 32) & 1} == sees[i]
    assert depth[len(parents):].tolist() == [-1, -1] and not mask[len(parents):].any()


def test_plan_refuses():
    one = np.zeros(4, np.int32)
    for start in ([0], [-1, 2], [2, 1], [0, 5]):
        with pytest.raises(NekoError):
            ops.tree_plan(one, np.array(start, np.int32))
    with pytest.raises(NekoError):
        ops.tree_plan(np.full(1025, -1, np.int32), np.array([0, 1025], np.int32))
    with pytest.raises(NekoError):
        ops.tree_plan(one[None], np.array([0, 4], np.int32))
    L = _lib.lib
    start = (ctypes.c_int32 * 2)(0, 33)
    buf = (ctypes.c_int32 * 33)()
    ptr = lambda x: ctypes.cast(x, ctypes.c_void_p)  # noqa: E731
    assert L.neko_tree_plan(ptr(buf), ptr(start), 1, 1, ptr(buf), ptr(buf)) == _lib.NEKO_ERR_INVALID  # 33 rows, 32 bits
    assert L.neko_tree_plan(None, ptr(start), 1, 2, ptr(buf), ptr(buf)) == _lib.NEKO_ERR_INVALID
    assert L.neko_tree_plan(ptr(buf), ptr(start), 1, 0, ptr(buf), ptr(buf)) == _lib.NEKO_ERR_INVALID
    assert L.neko_tree_plan(None, None, 0, 1, None, None) == _lib.NEKO_OK


def test_no_context():
    L = _lib.lib
    assert L.neko_hip_sample(None, None, 8, 1, 8, None, None, None, None, None, None, 0) == _lib.NEKO_ERR_INVALID
    assert L.neko_hip_accept_tree(None, None, None, None, 0, None, None, 1, None, 1, None, None, None) == _lib.NEKO_ERR_INVALID
    assert L.neko_hip_keep_paged(None, None, None, None, 1, 1, None) == _lib.NEKO_ERR_INVALID
    assert L.neko_hip_attention_tree_paged(None, None, 1, 1, None, None, None, 1, 1.0, 0.0, 0, None, None, 1, 0) == _lib.NEKO_ERR_INVALID
    assert L.neko_hip_qk_norm_rope_tree_paged(None, None, 1, 1, 1, None, None, None, None, None, 0, 0, 0, 1e-6, None, 1, 0) == _lib.NEKO_ERR_INVALID
