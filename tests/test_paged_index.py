"""The paged KV cache's index arithmetic on the CPU (nekochat_amd/csrc/paged.h compiled for the host): what a batch's
arrays hold is known only on the device, so whatever stands in them -- page ids outside the cache, row ranges that run
backwards or past the rows, lengths short of the rows or past the table -- every index formed from it has to be inside
the cache and the call's rows, and for well-formed batches every new row is covered exactly once."""
import ctypes
import os
import re
import shutil
import subprocess

import numpy as np
import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


class Batch(ctypes.Structure):
    _fields_ = [("table", ctypes.c_void_p), ("row_start", ctypes.c_void_p), ("kv_len", ctypes.c_void_p),
                ("table_stride", ctypes.c_int64), ("n_pages", ctypes.c_int64), ("max_pages", ctypes.c_int32),
                ("n_seq", ctypes.c_int32), ("rows", ctypes.c_int32), ("page_log2", ctypes.c_int32),
                ("n_kv", ctypes.c_int32), ("hd", ctypes.c_int32)]


class Tiling(ctypes.Structure):
    _fields_ = [("group", ctypes.c_int32), ("tile_log2", ctypes.c_int32), ("unit_log2", ctypes.c_int32),
                ("target", ctypes.c_int32), ("least", ctypes.c_int32), ("window", ctypes.c_int32), ("span", ctypes.c_int32),
                ("min_rows", ctypes.c_int32), ("max_rows", ctypes.c_int32)]


@pytest.fixture(scope="module")
def lib():
    path = os.path.join(HERE, "cpp", "_build", "libpaged_index_check.so")
    if not os.path.exists(path):
        pytest.fail(f"{path} is not built (run __graft_entry__.build())")
    lib = ctypes.CDLL(path)
    lib.check_need_exp.argtypes = [ctypes.c_uint32]
    lib.check_scale_exp.argtypes = [ctypes.c_float]
    lib.check_segments.restype = ctypes.c_int64
    lib.check_segments.argtypes = [ctypes.c_void_p, ctypes.c_int32, ctypes.c_void_p, ctypes.c_int64]
    lib.check_page.argtypes = [ctypes.c_void_p, ctypes.c_int32, ctypes.c_int32]
    return lib


def _batch(rng, wild):
    """A random batch: well formed, or (wild) of any numbers."""
    n_seq = int(rng.integers(1, 12))
    log2 = int(rng.integers(4, 9))
    n_pages = int(rng.integers(1, 40))
    max_pages = int(rng.integers(1, 9))
    P = 1 << log2
    if wild:
        rows = int(rng.integers(1, 300))
        some = np.array([-2**31, -1, 0, 1, 5, rows, rows + 1, 2**30, 2**31 - 1])
        pick = lambda n, hi: np.where(rng.random(n) < 0.4, rng.choice(some, n), rng.integers(-3, hi, n)).astype(np.int32)
        start, length, table = pick(n_seq + 1, rows + 3), pick(n_seq, max_pages * P + 9), pick(n_seq * max_pages, n_pages + 3)
    else:
        length = rng.integers(0, max_pages * P + 1, n_seq).astype(np.int32)
        n = (length * rng.choice([0, 0.01, 0.5, 1], n_seq)).astype(np.int32)
        start = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
        rows = int(start[-1]) + int(rng.integers(0, 4))
        table = rng.integers(0, n_pages, n_seq * max_pages).astype(np.int32)
    b = Batch(table.ctypes.data, start.ctypes.data, length.ctypes.data, max_pages, n_pages, max_pages, n_seq, rows, log2, 2, 64)
    b.held = (table, start, length)
    return b


def _segments(lib, b, limit):
    room = b.rows + 2 * b.n_seq + 8
    out = np.zeros((room, 6), np.int32)
    n = lib.check_segments(ctypes.byref(b), limit, out.ctypes.data, room)
    assert n >= 0
    return out[:n]


@pytest.mark.parametrize("seed", range(200))
def test_segments_of_well_formed_batches_cover_each_row_once(lib, seed):
    rng = np.random.default_rng(seed)
    b = _batch(rng, wild=False)
    table, start, length = b.held
    P = 1 << b.page_log2
    limit = int(rng.choice([1 << 30, 100]))
    seen = np.zeros(b.rows, int)
    for s, page, a, e, row0, pos0 in _segments(lib, b, limit):
        n, first = start[s + 1] - start[s], length[s] - (start[s + 1] - start[s])
        assert 0 <= a < e <= P and pos0 % P == 0
        assert page == table[s * b.max_pages + pos0 // P]
        for slot in range(a, e):
            row, pos = row0 + slot, pos0 + slot
            assert start[s] <= row < start[s + 1] and pos == first + (row - start[s]) and pos < limit
            seen[row] += 1
        assert a == 0 or pos0 + a == first  # only a sequence's first page keeps earlier tokens
    want = np.zeros(b.rows, int)
    for s in range(b.n_seq):
        pos = length[s] - (start[s + 1] - start[s]) + np.arange(start[s + 1] - start[s])
        want[start[s]:start[s + 1]] = pos < limit
    assert np.array_equal(seen, want)


@pytest.mark.parametrize("seed", range(400))
def test_wild_batches_stay_inside_the_cache_and_the_rows(lib, seed):
    rng = np.random.default_rng(1000 + seed)
    b = _batch(rng, wild=True)
    P = 1 << b.page_log2
    for s, page, a, e, row0, pos0 in _segments(lib, b, int(rng.choice([1 << 30, 50]))):
        assert 0 <= page < b.n_pages and 0 <= a < e <= P and pos0 >= 0
        assert row0 + a >= 0 and row0 + e <= b.rows
    out = (ctypes.c_int32 * 3)()
    for s in range(b.n_seq):
        lib.check_seq(ctypes.byref(b), s, out)
        assert 0 <= out[0] <= b.rows and out[1] >= 0 and out[0] + out[1] <= b.rows and 0 <= out[2] <= 2**30
        for pos in (-2**31, -1, 0, P - 1, P, b.max_pages * P - 1, b.max_pages * P, 2**31 - 1):
            page = lib.check_page(ctypes.byref(b), s, pos)
            assert page == -1 or (0 <= page < b.n_pages and 0 <= pos < b.max_pages * P)


@pytest.mark.parametrize("seed", range(300))
def test_attention_blocks_stay_within_the_grid(lib, seed):
    rng = np.random.default_rng(5000 + seed)
    b = _batch(rng, wild=False)
    group = int(rng.choice([1, 2, 3, 4, 8, 16, 40]))
    few = int(rng.choice([0, 16, 32]))
    few = (few + 1, 2**31 - 1) if few and rng.random() < 0.5 else (1, few or 2**31 - 1)
    t = Tiling(group, int(rng.choice([4, 6, 7, 8])), int(rng.choice([6, 7, 9])), int(rng.choice([1, 7, 256, 1024])),
               int(rng.choice([1, 8])), int(rng.choice([0, 1, 40, 1000])), 0, *few)
    out = (ctypes.c_int64 * 7)()
    lib.check_blocks(ctypes.byref(b), ctypes.byref(t), out)
    tiles, blocks, tiles_bound, blocks_bound, uncovered, split, split_bound = out
    assert tiles <= tiles_bound and blocks <= blocks_bound and uncovered == 0 and split <= split_bound


def _plan(lib, rows, seqs, log2, max_pages, n_kv, tiling):
    start = np.cumsum([0] + [n for n, _ in seqs]).astype(np.int32)
    length = np.array([x for _, x in seqs], np.int32)
    b = Batch(0, start.ctypes.data, length.ctypes.data, max_pages, 1, max_pages, len(seqs), rows, log2, n_kv, 64)
    out = (ctypes.c_int64 * 7)()
    lib.check_plan(ctypes.byref(b), ctypes.byref(tiling), out)
    return list(out)


def _check_plan(lib, *args):
    tiles, blocks, split, uncovered, planned, blocks_bound, split_bound = _plan(lib, *args)
    assert uncovered == 0 and blocks <= blocks_bound
    assert split <= (split_bound if planned else 0), "splits that the launch has no place for"
    return split, planned


@pytest.mark.parametrize("seed", range(400))
def test_splits_are_those_that_the_launch_planned(lib, seed):
    """What the device splits has a place in the workspace and a merge, however few of the call's rows are a sequence's:
    a graph captured for many rows is replayed with few. One sequence alone is the case that the host plans by its rows."""
    rng = np.random.default_rng(9000 + seed)
    for _ in range(10):
        log2, n_kv = int(rng.integers(4, 9)), int(rng.choice([1, 2, 8, 12]))
        max_pages = int(np.exp(rng.uniform(0, 8)))
        reach = max_pages << log2
        n_seq = 1 if rng.random() < 0.6 else int(rng.integers(2, 40))
        seqs = []
        for _ in range(n_seq):
            length = int(rng.integers(0, reach + 1))
            seqs.append((min(length, int(np.exp(rng.uniform(0, 7))) - 1), length))
        rows = max(1, int(sum(n for n, _ in seqs) * np.exp(rng.uniform(0, 8)))) + int(rng.integers(0, 9))
        few = [(1, 2**31 - 1), (33, 2**31 - 1), (1, 32)][int(rng.integers(0, 3))]
        t = Tiling(int(rng.choice([1, 2, 4, 7, 16])), *[(4, 7), (4, 8), (7, 6)][int(rng.integers(0, 3))],
                   int(rng.choice([1, 256, 512, 768, 1024])), int(rng.choice([1, 4, 8])), int(rng.choice([0, 0, 40, 1000])), 0, *few)
        _check_plan(lib, rows, seqs, log2, max_pages, n_kv, t)


@pytest.mark.parametrize("tile_log2,unit_log2,target,least,rows,own,length,reach", [
    (7, 6, 512, 1, 2048, 500, 500, 8192), (7, 6, 512, 1, 2048, 500, 4096, 8192), (7, 6, 512, 1, 4096, 64, 8192, 8192),
    (7, 6, 512, 1, 8192, 1, 8192, 8192), (4, 7, 768, 4, 512, 1, 1100, 1104), (4, 7, 768, 4, 700, 1, 1040, 1040),
])
def test_one_sequence_with_rows_that_are_not_its_own(lib, tile_log2, unit_log2, target, least, rows, own, length, reach):
    """32 / 8 heads, both kernels' tilings: a chunk's last piece, or one token, in a buffer of many rows."""
    t = Tiling(4, tile_log2, unit_log2, target, least, 0, 0, 1, 2**31 - 1)
    split, planned = _check_plan(lib, rows, [(own, length)], 4, reach >> 4, 8, t)
    assert not planned and split == 0
    # With the sequence's own rows alone the same tiles are split, and planned for.
    split, planned = _check_plan(lib, own, [(own, length)], 4, reach >> 4, 8, t)
    assert planned and split > 0


@pytest.mark.parametrize("n_seq", [1, 2, 5, 6, 64, 300])
@pytest.mark.parametrize("wild", [False, True])
def test_the_sequence_of_a_row(lib, n_seq, wild):
    """The last sequence that begins at or before a row, from any that does, over idle places too; some sequence of the
    batch, from the given one on, whatever the starts are."""
    rng = np.random.default_rng(n_seq)
    for _ in range(40):
        n = rng.choice([0, 0, 0, 1, 4], n_seq)
        start = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
        rows = int(start[-1]) + int(rng.integers(1, 9))
        if wild:
            start = rng.integers(-5, rows + 5, n_seq + 1).astype(np.int32)
        length = np.ones(n_seq, np.int32)
        b = Batch(0, start.ctypes.data, length.ctypes.data, 1, 1, 1, n_seq, rows, 4, 1, 64)
        for row in range(rows):
            last = int(np.flatnonzero(start[:n_seq] <= row)[-1]) if (start[:n_seq] <= row).any() else 0
            for s in {0, int(rng.integers(0, last + 1)), last}:
                got = lib.check_seq_from(ctypes.byref(b), s, row)
                assert s <= got < n_seq
                if not wild:
                    assert got == last, (s, row)


def test_calls_without_a_context_are_refused():
    from nekochat_amd import _lib

    kv, batch = _lib.PagedKv(), _lib.PagedBatch()
    L = _lib.lib
    for pair in ((None, None), (ctypes.byref(kv), ctypes.byref(batch))):
        assert L.neko_hip_qk_norm_rope_paged(None, None, 0, 1, 1, *pair, None, None, 0, 0, 0, 1e-6, None, 0, 1) == _lib.NEKO_ERR_INVALID
        assert L.neko_hip_attention_paged(None, None, 0, 1, *pair, 1, 1.0, 0.0, 0, None, None, 0, 1) == _lib.NEKO_ERR_INVALID


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs gcc")
def test_the_documented_layer_compiles(tmp_path):
    root = os.path.dirname(HERE)
    with open(os.path.join(root, "INTEGRATION.md")) as f:
        block = next(b for b in re.findall(r"```c\n(.*?)```", f.read(), flags=re.S) if "neko_paged_kv" in b)
    src = tmp_path / "layer.c"
    src.write_text("#include <stddef.h>\n#include <stdint.h>\n#include \"neko_hip.h\"\n" + block)
    r = subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-fsyntax-only", "-I", os.path.join(root, "include"), str(src)],
                       capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr


def test_splits_are_the_ceiling(lib):
    rng = np.random.default_rng(2)
    for _ in range(20000):
        chunk = int(np.exp(rng.uniform(0, 14)))
        units = int(rng.integers(0, min(2**25, chunk * 4000)))
        if rng.random() < 0.5:
            units = units // chunk * chunk + int(rng.integers(-1, 2))
        units = max(units, 0)
        assert lib.check_splits(units, chunk) == max(1, -(-units // chunk)), (units, chunk)


def test_scale_exponents(lib):
    """The smallest power of two that brings amax to 448 or below, against the formula in 64 bits."""
    rng = np.random.default_rng(3)
    vals = np.concatenate([np.float32(448) * np.float32(2.0) ** np.arange(-60, 60, dtype=np.float32),
                           np.exp(rng.uniform(-40, 40, 4000)).astype(np.float32), np.float32([1, 3, 449, 447.9])])
    vals = np.concatenate([vals, np.nextafter(vals, np.float32(np.inf)), np.nextafter(vals, np.float32(0))]).astype(np.float32)
    for v in vals:
        e = lib.check_need_exp(int(v.view(np.uint32)))
        v = float(v)
        want = -64
        while v > 448 * 2.0 ** want and want < 64:
            want += 1
        assert e == want, v
    assert lib.check_need_exp(0) == -64
    assert lib.check_need_exp(int(np.float32(3e38).view(np.uint32))) == 64
    for e in (-64, -3, 0, 17, 64):
        assert lib.check_scale_exp(2.0 ** e) == e and lib.check_scale_exp(1.5 * 2.0 ** e) == e
    for s, e in ((0.0, -64), (float("inf"), 64), (float("nan"), 64), (-4.0, 2), (1e-30, -64), (1e30, 64)):
        assert lib.check_scale_exp(s) == e
