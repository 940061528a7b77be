"""Refusals of keep_tokens, fork_rows and rotaries of several axes, on the host (CPU only)."""
import ctypes

import numpy as np
import pytest
import torch

from kunserve_amd import KVPool, KVWeights, PageTable, Rotary, _lib, fork_rows, keep_tokens

CPU = torch.device("cpu")


def pool(pages=8, page=4):
    return KVPool.allocate(pages, 2, 1, page, 64, CPU)


def table(lists, lens, p):
    return PageTable.from_lists(lists, lens, p, upload=False)


@pytest.mark.parametrize("first,why", [(-1, "first place -1"), (9, "first place 9"), ([0, 0], "one per row"),
                                       (0.5, "whole number"), ([[0]], "one per row")])
def test_first_places(first, why):
    p = pool()
    with pytest.raises(ValueError, match=why):
        keep_tokens(p, table([[0, 1]], [8], p), first, [[1]])


@pytest.mark.parametrize("kept,why", [([[1, 1]], "must rise"), ([[2, 1]], "must rise"), ([[-1]], "must rise"),
                                      ([[8]], "must rise"), ([[1.0]], "whole numbers"), ([], "0 lists"),
                                      ([[[1]]], "whole numbers")])
def test_kept_places(kept, why):
    p = pool()
    with pytest.raises(ValueError, match=why):
        keep_tokens(p, table([[0, 1]], [8], p), 0, kept)


def test_pages_in_two_places():
    p = pool()
    with pytest.raises(ValueError, match="one place"):
        keep_tokens(p, table([[0, 1], [2, 1]], [8, 8], p), 0, [[1], [1]])
    with pytest.raises(ValueError, match="one place"):
        keep_tokens(p, table([[0, 1], [0, 2]], [8, 8], p), 0, [[1], [1]])
    # shared pages before the first places are no matter
    keep_tokens(p, table([[0, 1], [0, 2]], [8, 8], p), 4, [[], []])
    keep_tokens(p, table([], [], p), 0, [])


def test_tensors_and_weights_of_others():
    p = pool()
    t = table([[0, 1]], [8], p)
    for bad in (torch.zeros(1, 2), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32),
                torch.zeros(1, 4, dtype=torch.int32)[:, ::2]):
        with pytest.raises(ValueError, match="kept must be int32"):
            keep_tokens(p, t, 0, bad)
    with pytest.raises(ValueError, match="weights"):
        keep_tokens(p, t, 0, [[1]], weights=KVWeights(pool(9)))
    with pytest.raises(ValueError, match="weights"):
        fork_rows(p, [[0]], [1], [[1]], weights=KVWeights(pool(9)))


@pytest.mark.parametrize("lists,lens,out,why", [
    ([[0]], [1, 1], [[1]], "2 kv lengths"),
    ([[0]], [1], [[1], [2]], "and 2 page lists"),
    ([[0]], [-1], [[1]], "whole numbers, 0 at least"),
    ([[0]], [1.5], [[1]], "whole numbers"),
    ([[0, 1]], [8], [[0]], "needs 2"),
    ([[0]], [8], [[2, 3]], "needs 2"),
    ([[0, 1]], [8], [[0, 0]], "holds tokens of the rows"),
    ([[0, 1]], [8], [[1, 0]], "holds tokens of the rows"),
    ([[0, 1], [2]], [8, 4], [[0, 2], [3]], "holds tokens of the rows"),
    ([[0], [1]], [4, 4], [[3], [3]], "copied to twice"),
])
def test_fork_refusals(lists, lens, out, why):
    with pytest.raises(ValueError, match=why):
        fork_rows(pool(), lists, lens, out)


def fork_moves(lists, lens, page, num_pages, capacity=None):
    indptr = np.cumsum([0] + [len(x) for x in lists]).astype(np.int32)
    ids = np.array([i for x in lists for i in x] + [0], dtype=np.int32)
    lens = np.array(lens, dtype=np.int32)
    out = np.full((len(ids), 3), -7, dtype=np.int32)
    n = _lib.call("kunserve_fork_moves", indptr.ctypes.data, ids.ctypes.data, lens.ctypes.data,
                  len(lens), page, num_pages, out.ctypes.data,
                  len(out) if capacity is None else capacity)
    assert (out[n:] == -7).all()
    return out[:n].tolist()


@pytest.mark.parametrize("seed", range(20))
def test_fork_moves(seed):
    rng = np.random.default_rng(seed)
    page = int(rng.choice([4, 16]))
    lens = rng.integers(0, 5 * page, size=int(rng.integers(1, 7)))
    need = -(-lens // page)
    ids = iter(rng.permutation(80).tolist())
    rows = [[next(ids) for _ in range(n)] for n in need]
    out = [[i if rng.integers(2) else next(ids) for i in r] for r in rows]
    want = [[a, b, int(min(page, lens[r] - i * page))] for r in range(len(lens))
            for i, (a, b) in enumerate(zip(rows[r], out[r])) if a != b]
    # (pages behind the tokens in use are not looked at)
    assert fork_moves([x + [99] for x in rows] + [x + [rows[0][0] if rows[0] else 3] for x in out],
                      lens, page, 80) == want
    if want:
        with pytest.raises(_lib.KunserveError, match="moves"):
            fork_moves(rows + out, lens, page, 80, capacity=len(want) - 1)


@pytest.mark.parametrize("lists,lens,why", [
    ([[0], []], [4], "0 pages for 4"),
    ([[80], [1]], [4], "page id 80 outside"),
    ([[0], [-1]], [4], "page id -1 outside"),
    ([[0], [1]], [-4], "-4 tokens"),
])
def test_fork_moves_refusals(lists, lens, why):
    with pytest.raises(_lib.KunserveError, match=why):
        fork_moves(lists, lens, 4, 80)


def test_copy_pages_refusals():
    p, moves = pool(), np.zeros((300, 3), np.int32)
    for host, dev, n, why in ((None, None, 1, "either"), (moves, moves, 1, "either"),
                              (moves, None, 257, "256 at most"), (None, moves, -1, "-1 moves")):
        with pytest.raises(_lib.KunserveError, match=why):
            _lib.call("kunserve_copy_pages", p.desc(), None, None if host is None else host.ctypes.data,
                      None if dev is None else dev.ctypes.data, n, None)
    assert _lib.call("kunserve_copy_pages", p.desc(), None, None, None, 0, None) == 0


def test_keep_tokens_refuses_first_places():
    p = pool()
    zeros = np.zeros(300, np.int32)
    n = zeros.ctypes.data
    t = _lib.PageTable(indptr_dev=n, indices_dev=n, kv_len_dev=n, num_seqs=300)   # (refused unread)
    for host, dev, why in ((None, None, "either"), (n, n, "either"), (n, None, "256 at most")):
        with pytest.raises(_lib.KunserveError, match=why):
            _lib.call("kunserve_keep_tokens", p.desc(), None, ctypes.byref(t), host, dev, n, 1, 1, None)


def test_fork_pages_outside():
    with pytest.raises(IndexError, match="page id 8"):
        fork_rows(pool(), [[0]], [4], [[8]])


def test_fork_of_nothing():
    fork_rows(pool(), [], [], [])
    fork_rows(pool(), [[], [1]], [0, 4], [[], [1]])


@pytest.mark.parametrize("kw,why", [
    (dict(sections=[8, 8, 8]), "sections of 24 pairs"),
    (dict(sections=[16, 16], axes=[0] * 32), "sections or axes"),
    (dict(sections=[40, -8]), "0 at least"),
    (dict(sections=[16.0, 16.0]), "whole numbers"),
    (dict(sections=[]), "whole numbers"),
    (dict(axes=[0] * 31), "axes of 31 pairs"),
    (dict(axes=[-1] * 32), "0 at least"),
    (dict(axes=[[0] * 32]), "whole numbers"),
    (dict(axes=[5000] * 32), "1024 axes"),
])
def test_rotary_axes(kw, why):
    with pytest.raises(ValueError, match=why):
        Rotary(64, device=CPU, **kw)


def test_rotary_axes_of_pairs():
    r = Rotary(64, device=CPU, sections=[8, 0, 24])
    assert r.num_axes == 3 and r.pair_axis.tolist() == [0] * 8 + [2] * 24
    r = Rotary(64, device=CPU, axes=[i % 3 for i in range(32)])
    assert r.num_axes == 3 and r.pair_axis.dtype == torch.int32
    assert Rotary(64, device=CPU).num_axes == 1
    with pytest.raises(ValueError, match="positions on 2 axes"):
        r.check_positions(torch.zeros(2, 5, dtype=torch.int32))
    r.check_positions(torch.zeros(5, dtype=torch.int32))
    assert r.axes_desc(torch.zeros(3, 5, dtype=torch.int32)).position_stride == 5
    assert r.axes_desc(torch.zeros(5, dtype=torch.int32)).position_stride == 0
