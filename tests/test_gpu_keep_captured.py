"""keep_tokens of a step without trees in a graph: its rows' first places go with the launch,
up to as many rows as that takes."""
import numpy as np
import pytest
import torch

from helpers import random_pool, random_tensor
from kunserve_amd import AttentionStep, KVWeights
from tree_ref import random_pages

pytestmark = pytest.mark.gpu


def moved(t, lists, first, kept, page):
    want = t.clone()
    for b, places in enumerate(kept):
        for j, e in enumerate(places):
            s, d = first[b] + e, first[b] + j
            want[lists[b][d // page], :, :, d % page] = t[lists[b][s // page], :, :, s % page]
    return want


def entries(kept, width, device):
    rows = torch.full((len(kept), width), -1, dtype=torch.int32)
    for b, x in enumerate(kept):
        rows[b, :len(x)] = torch.tensor(x, dtype=torch.int32)
    return rows.to(device)


@pytest.mark.parametrize("rows", [2, 256])
@pytest.mark.parametrize("weighted", [False, True])
def test_replays_keep_what_the_tensor_says(device, rows, weighted):
    rng = np.random.default_rng(rows)
    sizes = [int(n) for n in rng.integers(1, 20, rows)]
    cached = [int(n) for n in rng.integers(0, 30, rows)]
    lists, pages = random_pages(rng, [a + b for a, b in zip(sizes, cached)], 4)
    pool = random_pool(pages, 2, 1, 4, 64, device, 1)
    w = KVWeights(pool) if weighted else None
    if weighted:
        w.w.uniform_()
    step = AttentionStep(pool, 2, sizes, cached, [1] * rows, lists)
    assert step.tree is None
    kept = entries([[]] * rows, 20, device)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step.keep_tokens(kept, weights=w)
    tensors = [pool.k, pool.v] + ([w.w] if weighted else [])
    for _ in range(4):
        places = [sorted(rng.choice(n, size=int(rng.integers(0, n + 1)), replace=False).tolist())
                  for n in sizes]
        kept.copy_(entries(places, 20, device))
        want = [moved(t, lists, cached, places, 4) for t in tensors]
        g.replay()
        random_tensor((64, 64), device, 1).sum()   # eager work between the replays
        torch.cuda.synchronize()
        assert all(torch.equal(t, x) for t, x in zip(tensors, want))


def test_two_graphs_and_eager_calls(device):
    """Steps of other rows captured one after the other: each keeps its own first places."""
    rng = np.random.default_rng(4)
    lists, pages = random_pages(rng, [40, 33], 16)
    pool = random_pool(pages, 1, 2, 16, 128, device, 1)
    steps = [AttentionStep(pool, 4, [10], [30], [1], lists[:1]),
             AttentionStep(pool, 4, [33], [0], [1], lists[1:])]
    kept = [entries([[0, 3, 9]], 3, device), entries([[1, 30, 32]], 3, device)]
    graphs = []
    for s, k in zip(steps, kept):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s.keep_tokens(k)
        graphs.append(g)
    for i in (1, 0, 0, 1):
        first, places = [(30, [0, 3, 9]), (0, [1, 30, 32])][i]
        want = moved(pool.k, lists[i:i + 1], [first], [places], 16)
        graphs[i].replay()
        torch.cuda.synchronize()
        assert torch.equal(pool.k, want)
        want = moved(pool.k, lists[i:i + 1], [first], [places], 16)
        steps[i].keep_tokens([places])
        assert torch.equal(pool.k, want)


def test_refusals(device):
    rng = np.random.default_rng(6)
    rows = 257
    lists, pages = random_pages(rng, [8] * rows, 4)
    pool = random_pool(pages, 1, 1, 4, 64, device, 1)
    many = AttentionStep(pool, 2, [4] * rows, [4] * rows, [1] * rows, lists)
    few = AttentionStep(pool, 2, [4], [4], [1], lists[:1])
    kept = entries([[1]] * rows, 1, device)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        few.keep_tokens(kept[:1])
        with pytest.raises(RuntimeError, match="257 rows .* capture"):
            many.keep_tokens(kept)
        with pytest.raises(RuntimeError, match="lists cannot be captured"):
            few.keep_tokens([[1]])
    want = moved(pool.k, lists[:1], [4], [[1]], 4)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(pool.k, want)
    want = moved(pool.k, lists, [4] * rows, [[1]] * rows, 4)
    many.keep_tokens(kept)   # not under a capture
    assert torch.equal(pool.k, want)
