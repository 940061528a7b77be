"""Cached tokens that change their place: keep_tokens, fork_rows, and a request that drafts,
verifies, keeps and goes on."""
import math

import numpy as np
import pytest
import torch

from helpers import random_pool, random_tensor
from kunserve_amd import (AttentionStep, KVPool, KVWeights, PageTable, Rotary, fork_rows,
                          keep_tokens)
from tree_ref import (check_out, random_pages, random_tree, tokens_of, tree_attention_ref)

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def moved(pool_t, lists, first, kept, page):
    """The tensor after keep_tokens, token by token."""
    want = pool_t.clone()
    for b, places in enumerate(kept):
        for j, e in enumerate(places):
            s, d = first[b] + e, first[b] + j
            want[lists[b][d // page], :, :, d % page] = pool_t[lists[b][s // page], :, :, s % page]
    return want


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page,dtype", [(4, F16), (16, BF16), (256, F16)])
def test_keep_tokens(device, dim, page, dtype):
    rng = np.random.default_rng(dim + page)
    lens = [1, 2, 40, 300, 700, 33, 1300]
    lists, pages = random_pages(rng, lens, page)
    pool = random_pool(pages, 3, 2, page, dim, device, 1, dtype=dtype)
    w = KVWeights(pool)
    w.w.uniform_()
    first = [0, 1, 17, 0, 100, 33, 5]
    kept = [sorted(rng.choice(n - f, size=max(0, (n - f) * s // 4), replace=False).tolist())
            for n, f, s in zip(lens, first, [4, 4, 1, 2, 3, 4, 3])]
    table = PageTable.from_lists(lists, lens, pool)
    want = [moved(t, lists, first, kept, page) for t in (pool.k, pool.v)]
    want_w = moved(w.w, lists, first, kept, page)
    keep_tokens(pool, table, first, kept, weights=w)
    assert torch.equal(pool.k, want[0]) and torch.equal(pool.v, want[1])
    assert torch.equal(w.w, want_w)


@pytest.mark.parametrize("rows", [255, 256, 257])
def test_keep_tokens_of_many_rows(device, rows):
    """First places of up to 256 rows go with the launch, of more by a copy of their own."""
    rng = np.random.default_rng(rows)
    lens = [4 + b % 9 for b in range(rows)]
    lists, pages = random_pages(rng, lens, 4)
    pool = random_pool(pages, 1, 1, 4, 64, device, 1)
    first = [b % 3 for b in range(rows)]
    kept = [sorted(rng.permutation(n - f)[:(n - f) // 2].tolist()) for n, f in zip(lens, first)]
    want = [moved(t, lists, first, kept, 4) for t in (pool.k, pool.v)]
    table = PageTable.from_lists(lists, lens, pool)
    if rows == 256:   # entries on the device too
        dev = torch.full((rows, max(map(len, kept))), -1, dtype=torch.int32)
        for b, x in enumerate(kept):
            dev[b, :len(x)] = torch.tensor(x, dtype=torch.int32)
        kept = dev.to(device)
    keep_tokens(pool, table, first, kept)
    assert torch.equal(pool.k, want[0]) and torch.equal(pool.v, want[1])


def test_keep_tokens_short_lists_and_device_entries(device):
    """Lists that one wave moves; entries that move nothing; a tensor's rows apart."""
    rng = np.random.default_rng(4)
    lens = [50, 64, 9, 100]
    lists, pages = random_pages(rng, lens, 16)
    pool = random_pool(pages, 2, 3, 16, 128, device, 1)
    table = PageTable.from_lists(lists, lens, pool)
    first = [40, 0, 9, 64]
    rows = torch.full((4, 12), -1, dtype=torch.int32, device=device)
    entries = [[0, 3, 9], [1, 0, 2, 63, 64, 1000, -7, 2**31 - 1], [0, 1], [5, 6, 30, 35]]
    for b, e in enumerate(entries):
        rows[b, :len(e)] = torch.tensor(e, dtype=torch.int32)
    want = []
    for t in (pool.k, pool.v):
        x = t.clone()
        for b, e in enumerate(entries):
            for j, s in enumerate(e):
                if j < s < lens[b] - first[b]:
                    a, d = first[b] + s, first[b] + j
                    x[lists[b][d // 16], :, :, d % 16] = t[lists[b][a // 16], :, :, a % 16]
        want.append(x)
    keep_tokens(pool, table, first, rows[:, :8])
    assert torch.equal(pool.k, want[0]) and torch.equal(pool.v, want[1])
    keep_tokens(pool, table, 0, [[], [], [], []])
    keep_tokens(pool, table, 0, rows[:, :0])
    assert torch.equal(pool.k, want[0])


def test_keep_tokens_bad_pages(device):
    """From C: a source page outside the pool gives zeros, a destination is not written."""
    pool = random_pool(4, 1, 1, 4, 64, device, 1)
    table = PageTable.from_lists([[0, 1, 2]], [12], pool)
    table.indices[1] = 77
    k = pool.k.clone()
    keep_tokens(pool, table, 0, [[4, 9]])
    assert not pool.k[0, :, :, 0].any() and torch.equal(pool.k[0, :, :, 1], k[2, :, :, 1])
    assert torch.equal(pool.k[1:], k[1:]) and torch.equal(pool.k[0, :, :, 2:], k[0, :, :, 2:])
    table.indices[:] = torch.tensor([-1, 1, 2], dtype=torch.int32)
    k = pool.k.clone()
    keep_tokens(pool, table, 0, [[4, 9]])
    assert torch.equal(pool.k, k)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page,dtype", [(4, BF16), (16, F16), (256, BF16)])
def test_fork_rows(device, dim, page, dtype):
    rng = np.random.default_rng(dim + page)
    lens = [0, 1, 2 * page, 3 * page + 1, 5 * page - 1, 5 * page - 1, 5 * page - 1]
    need = [-(-n // page) for n in lens]
    lists, pages = random_pages(rng, lens[:5], page)
    lists += [lists[4], lists[4]]                      # one row three times
    same = [0, 0, 1, 3, 4, 0, 3]                        # leading pages that stay shared
    ids = iter(range(pages, pages + sum(need)))
    out = [x[:s] + [next(ids) for _ in x[s:]] for x, s in zip(lists, same)]
    out[3] = out[3] + [0]                               # further pages are not looked at
    pool = random_pool(pages + sum(need), 3, 5, page, dim, device, 2, dtype=dtype)
    w = KVWeights(pool)
    w.w.uniform_()
    before = [t.clone() for t in (pool.k, pool.v, w.w)]
    fork_rows(pool, lists, lens, out, weights=w)
    for t, old in zip((pool.k, pool.v, w.w), before):
        want = old.clone()
        for b, n in enumerate(lens):
            for at in range(n):
                want[out[b][at // page], :, :, at % page] = old[lists[b][at // page], :, :, at % page]
        assert torch.equal(t, want)


@pytest.mark.parametrize("pages", [255, 256, 257])
def test_fork_rows_of_many_pages(device, pages):
    """Up to 256 moves go with the launch, more by a copy of their own."""
    n, rng = 2 * pages, np.random.default_rng(pages)
    pool = random_pool(n, 1, 1, 4, 64, device, 1)
    ids = rng.permutation(n).tolist()
    src, dst = ids[:pages], ids[pages:]
    old = [pool.k.clone(), pool.v.clone()]
    lens, rows, out = [], [], []
    for at in range(0, pages, 50):
        rows.append(src[at:at + 50])
        out.append(dst[at:at + 50])
        lens.append(4 * len(rows[-1]) - at % 4)
    fork_rows(pool, rows, lens, out)
    for t, was in zip((pool.k, pool.v), old):
        want = was.clone()
        for a, b, l in zip(rows, out, lens):
            for at in range(l):
                want[b[at // 4], :, :, at % 4] = was[a[at // 4], :, :, at % 4]
        assert torch.equal(t, want)


def test_fork_rows_of_more_pages_than_a_launch_takes(device):
    pages = 70001
    pool = random_pool(2 * pages, 1, 1, 4, 64, device, 1)
    ids = torch.randperm(2 * pages, generator=torch.Generator().manual_seed(1))
    src, dst = ids[:pages], ids[pages:]
    want = [t.clone() for t in (pool.k, pool.v)]
    for t in want:
        t[dst[:-1].to(device)] = t[src[:-1].to(device)]
        t[dst[-1], :, :, :3] = t[src[-1], :, :, :3]
    fork_rows(pool, [src.tolist()], [4 * pages - 1], [dst.tolist()])
    assert torch.equal(pool.k, want[0]) and torch.equal(pool.v, want[1])


def test_fork_rows_strides(device):
    big = torch.randn(12, 2, 2, 6, 16, 128, device=device).to(F16)
    pool = KVPool(big[:, :, 0, 1:4], big[:, :, 1, 1:4])
    old = big.clone()
    fork_rows(pool, [[0, 1, 2]], [41], [[0, 7, 9]])
    want = old.clone()
    want[7, :, :, 1:4] = old[1, :, :, 1:4]
    want[9, :, :, 1:4, :9] = old[2, :, :, 1:4, :9]
    assert torch.equal(big, want)


def test_step_keeps_its_weights_and_refuses_shared_pages(device):
    rng = np.random.default_rng(0)
    lists, pages = random_pages(rng, [60, 31], 16)
    pool = random_pool(pages, 2, 2, 16, 64, device, 1)
    w = KVWeights(pool)
    w.w.uniform_()
    trees = [random_tree(rng, 10, 3), random_tree(rng, 5, 3)]
    step = AttentionStep(pool, 4, [10, 5], [50, 26], [1, 1], lists, trees=trees, weights=w, learn=False)
    old = w.w.clone()
    kept = [[0, 4, 9], [2]]
    want = moved(pool.k, lists, [50, 26], kept, 16)
    step.keep_tokens(kept, weights=w)
    assert torch.equal(pool.k, want) and torch.equal(w.w, moved(old, lists, [50, 26], kept, 16))
    shared = AttentionStep(pool, 4, [10, 5], [50, 26], [1, 1], [lists[0], lists[0][:1] + lists[0][3:4]],
                           trees=trees)
    with pytest.raises(ValueError, match="in one place"):
        shared.keep_tokens(kept)
    with pytest.raises(ValueError, match="must rise"):
        step.keep_tokens([[0, 10], []])
    with pytest.raises(ValueError, match="kept must be int32"):
        step.keep_tokens(torch.zeros(2, 3, dtype=torch.int64, device=device))
    with pytest.raises(ValueError, match="kept must be int32"):
        step.keep_tokens(torch.zeros(3, 3, dtype=torch.int32, device=device))
    plain = AttentionStep(pool, 4, [10, 5], [50, 26], [1, 1], lists)
    want = moved(pool.k, lists, [50, 26], [[1], [0, 3]], 16)
    plain.keep_tokens([[1], [0, 3]])
    assert torch.equal(pool.k, want)


def test_captured(device):
    """A step's keep_tokens in a graph, with the accepted tokens of each replay."""
    rng = np.random.default_rng(6)
    lists, pages = random_pages(rng, [120, 90], 16)
    pool = random_pool(pages, 2, 2, 16, 128, device, 1)
    trees = [random_tree(rng, 20, 3), random_tree(rng, 10, 3)]
    step = AttentionStep(pool, 4, [20, 10], [100, 80], [1, 1], lists, trees=trees)
    kept = torch.full((2, 6), -1, dtype=torch.int32, device=device)
    table = step.table
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step.keep_tokens(kept)
        with pytest.raises(RuntimeError, match="capture"):
            step.keep_tokens([[1], [2]])
        with pytest.raises(RuntimeError, match="capture"):
            keep_tokens(pool, table, 0, kept)
        with pytest.raises(RuntimeError, match="capture"):
            fork_rows(pool, lists, [3, 3], lists)
    for places in ([[0, 3, 19], [9]], [[1, 2], [0, 4, 5, 6]], [[], [8, 9]]):
        kept.fill_(-1)
        for b, p in enumerate(places):
            kept[b, :len(p)] = torch.tensor(p, dtype=torch.int32, device=device)
        want = [moved(t, lists, [100, 80], places, 16) for t in (pool.k, pool.v)]
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(pool.k, want[0]) and torch.equal(pool.v, want[1])


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 64)])
def test_a_request_drafts_keeps_forks_and_goes_on(device, dtype, dim):
    """Prompt; two verified trees, whose accepted paths are kept; samples forked from it; a
    decoded token for each: the cache holds what decoding the accepted tokens one by one
    would have left, and each output is the formula's on that history."""
    hq, hkv, layers, page = 4, 2, 2, 16
    rng = np.random.default_rng(8)
    pool = random_pool(64, layers, hkv, page, dim, device, 3, dtype=dtype)
    rotary = Rotary(dim, device=device)
    ids = iter(rng.permutation(64).tolist())
    pages = [next(ids) for _ in range(5)]
    freq = torch.tensor(10000.0 ** (-np.arange(0, dim, 2) / dim), device=device)

    def turned(x, pos):   # [n, heads, dim] at positions [n], in 64 bits
        angle = torch.tensor(pos, device=device).double()[:, None] * freq
        a, b = x[..., :dim // 2].double(), x[..., dim // 2:].double()
        c, s = angle.cos()[:, None], angle.sin()[:, None]
        return torch.cat([a * c - b * s, b * c + a * s], dim=-1)

    def tensors(n, seed):
        return [random_tensor((layers, n, h, dim), device, seed + i, 1.0, dtype)
                for i, h in enumerate((hq, hkv, hkv))]

    history = [[torch.empty(0, hkv, dim, dtype=torch.float64, device=device)] * 2 for _ in range(layers)]
    tol = torch.finfo(dtype).eps

    def verify(step, n, trees, starts, pages_of, seed, layer_history):
        """Runs a step of one row and checks it; the row's rotated k and v by layer."""
        q, k, v = tensors(n, seed)
        new = []
        for layer in range(layers):
            out = step.run(layer, q[layer].clone(), k[layer], v[layer], rope=rotary)
            pos = [starts + int(d) for d in trees[1]]
            kk, qq = turned(k[layer], pos), turned(q[layer], pos)
            keys, vals = layer_history[layer]
            ref, mass = tree_attention_ref(
                qq, torch.cat([keys, kk]).transpose(0, 1), torch.cat([vals, v[layer].double()]).transpose(0, 1),
                trees[0], dim ** -0.5)
            # q and k enter rounded to 16 bits: 2 half steps of each product in a score of
            # sum |q k| / sqrt(dim) below 16, twice in a probability's quotient
            assert ((out.double() - ref).abs() <= ref.abs() * tol / 2 + mass * (32 * tol + 2 ** -12)).all()
            new.append((kk, v[layer].double()))
        return new

    n = 37
    step = AttentionStep(pool, hq, [n], [0], [1], [pages])
    new = verify(step, n, (list(range(-1, n - 1)), range(n)), 0, pages, 50, history)
    history = [[torch.cat([h[0], x]), torch.cat([h[1], y])] for h, (x, y) in zip(history, new)]
    for turn, (size, path) in enumerate([(12, None), (9, None)]):
        tree = random_tree(rng, size, 3)
        path, i = [], size - 1
        while i >= 0:
            path.insert(0, i)
            i = tree[i]
        step = AttentionStep(pool, hq, [size], [n], [1], [pages], trees=[tree])
        from kunserve_amd import tree_depths
        new = verify(step, size, (tree, tree_depths(tree)), n, pages, 60 + 10 * turn, history)
        step.keep_tokens(torch.tensor([path], dtype=torch.int32, device=device))
        history = [[torch.cat([h[0], x[path]]), torch.cat([h[1], y[path]])] for h, (x, y) in zip(history, new)]
        n += len(path)
        for layer in range(layers):
            for t, h in zip((pool.k, pool.v), history[layer]):
                got = tokens_of(t, layer, pages, n).double()
                assert ((got - h.transpose(0, 1)).abs() <= h.transpose(0, 1).abs() * tol / 2 + 2.0 ** -18).all()
    whole = n // page
    lists = [pages[:whole] + [next(ids)] for _ in range(3)]
    fork_rows(pool, [pages] * 3, [n] * 3, lists)
    for i, x in enumerate(lists):
        step = AttentionStep(pool, hq, [1], [n + 1], [0], [x])
        verify(step, 1, ([-1], [0]), n, x, 90 + 3 * i, history)
    for layer in range(layers):   # the request's own cache is as it was
        got = tokens_of(pool.k, layer, pages, n).double()
        h = history[layer][0].transpose(0, 1)
        assert ((got - h).abs() <= h.abs() * tol / 2 + 2.0 ** -18).all()


@pytest.mark.parametrize("rows,dim,page", [(1, 64, 4), (7, 128, 16), (9, 256, 16), (37, 64, 32)])
def test_fork_rows_of_one_prompt(device, rows, dim, page):
    """Samples of one prompt, some of them shorter than it, and a row of its own."""
    rng = np.random.default_rng(rows)
    prompt, lens = [3, 0, 5], [int(2 * page + rng.integers(1, page + 1)) for _ in range(rows)]
    other = [6, 7]
    ids = iter(range(8, 8 + 3 * rows + 2))
    out = [[3, next(ids), next(ids)] if b % 3 == 1 else [3, 0, next(ids)] for b in range(rows)]
    lists, lens = [prompt] * rows + [other], lens + [page + 1]
    out.append([next(ids), next(ids)])
    pool = random_pool(8 + 3 * rows + 2, 2, 3, page, dim, device, 1)
    w = KVWeights(pool)
    w.w.uniform_()
    before = [t.clone() for t in (pool.k, pool.v, w.w)]
    fork_rows(pool, lists, lens, out, weights=w)
    for t, old in zip((pool.k, pool.v, w.w), before):
        want = old.clone()
        for a, b, n in zip(lists, out, lens):
            for at in range(n):
                if a[at // page] != b[at // page]:
                    want[b[at // page], :, :, at % page] = old[a[at // page], :, :, at % page]
        assert torch.equal(t, want)
