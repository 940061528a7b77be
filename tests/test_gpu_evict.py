"""evict against a choice by full sorting, bit for bit."""
import numpy as np
import pytest
import torch

import operators_ref as ref
from helpers import random_pool
from kunserve_amd import KVWeights, evict

pytestmark = pytest.mark.gpu


def make(device, kvs, keeps, layers=2, heads=3, ps=16, d=64, dtype=torch.float16, seed=0,
         kind="skew"):
    need, out_need = [-(-n // ps) for n in kvs], [-(-min(b, n) // ps) for b, n in zip(keeps, kvs)]
    pages = sum(need) + sum(out_need) + 3
    perm = np.random.default_rng(seed).permutation(pages).tolist()
    take = lambda n: [perm.pop() for _ in range(n)]   # noqa: E731
    tables, outs = [take(n) for n in need], [take(n) for n in out_need]
    pool = random_pool(pages, layers, heads, ps, d, device, seed, dtype=dtype)
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    w = torch.randn((pages, layers, heads, ps), generator=g, device=device)
    if kind == "skew":
        w = torch.exp(2 * w)
    elif kind == "ties":
        w = torch.round(w)          # few values, zeros of both signs among them
    elif kind == "equal":
        w = torch.full_like(w, 0.25)
    elif kind == "odd":             # NaN, infinities, the lowest values, subnormals
        odd = torch.tensor([float("nan"), float("inf"), -float("inf"),
                            torch.finfo(torch.float32).min, 1e-40, -1e-40, 0.0], device=device)
        pick = torch.randint(0, 14, w.shape, generator=g, device=device)
        w = torch.where(pick < 7, odd[pick.clamp(max=6)], w)
    return pool, KVWeights(pool, w), tables, outs


def check(device, pool, weights, tables, kvs, outs, budget, sinks, recent):
    ps = pool.page_size
    old = [x.cpu().clone() for x in (pool.k, pool.v, weights.w)]
    kept = evict(pool, weights, tables, kvs, outs, budget, sinks, recent)
    torch.cuda.synchronize()
    keeps = np.minimum(np.broadcast_to(budget, len(kvs)), kvs)
    want = np.full((len(kvs), pool.num_layers, pool.num_kv_heads, int(keeps.max(initial=0))), -1,
                   dtype=np.int32)
    new = [x.clone() for x in old]
    for b, (n, m) in enumerate(zip(kvs, keeps)):
        if m == 0:
            continue
        t, o = np.array(tables[b]), np.array(outs[b])
        for layer in range(pool.num_layers):
            for h in range(pool.num_kv_heads):
                w = old[2][t, layer, h].numpy().reshape(-1)[:n]
                c = ref.choose(w, int(m), sinks, recent)
                want[b, layer, h, :m] = c
                j = np.arange(m)
                for x, y in zip(new, old):
                    x[o[j // ps], layer, h, j % ps] = y[t[c // ps], layer, h, c % ps]
    assert np.array_equal(kept.cpu().numpy(), want)
    for got, x in zip((pool.k, pool.v, weights.w), new):
        bits = torch.int32 if x.dtype == torch.float32 else torch.int16
        assert torch.equal(got.cpu().view(bits), x.view(bits))


@pytest.mark.parametrize("kind", ["skew", "ties", "equal", "odd"])
@pytest.mark.parametrize("sinks,recent", [(0, 0), (4, 0), (0, 9), (4, 100)])
def test_heaviest_tokens_stay(device, kind, sinks, recent):
    kvs = [1, 17, 300, 1025, 2000]
    keeps = [1, 5, 120, 1024, 333]
    args = make(device, kvs, keeps, seed=sinks + recent, kind=kind)
    check(device, *args[:3], kvs, args[3], keeps, sinks, recent)


@pytest.mark.parametrize("d,dtype,ps", [(64, torch.bfloat16, 4), (128, torch.float16, 256),
                                        (256, torch.bfloat16, 32)])
def test_types_head_sizes_and_pages(device, d, dtype, ps):
    kvs, keeps = [700, 255, 256, 257], [64, 128, 255, 1]
    args = make(device, kvs, keeps, layers=3, heads=2, ps=ps, d=d, dtype=dtype, seed=d)
    check(device, *args[:3], kvs, args[3], keeps, 3, 20)


def test_empty_and_short_requests(device):
    """Lengths of zero and one, budgets of zero, budgets over the length, and
    fewer than the first and last ones together."""
    kvs = [0, 1, 1, 40, 40, 40, 64]
    keeps = [10, 0, 5, 0, 100, 6, 64]
    args = make(device, kvs, keeps, seed=3)
    check(device, *args[:3], kvs, args[3], keeps, 4, 10)


def test_one_budget_for_all_and_none_at_all(device):
    kvs = [100, 50]
    args = make(device, kvs, [30, 30], seed=4)
    check(device, *args[:3], kvs, args[3], 30, 2, 2)
    assert evict(args[0], args[1], args[2], kvs, [[], []], 0).shape == (2, 2, 3, 0)
    assert evict(args[0], args[1], [], [], [], 5).shape == (0, 2, 3, 0)


def test_long_request(device):
    kvs, keeps = [70001], [4097]
    args = make(device, kvs, keeps, layers=1, heads=2, seed=5, kind="ties")
    check(device, *args[:3], kvs, args[3], keeps, 4, 64)


def test_strided_pools_and_weights(device):
    """Pools whose pages hold the heads apart, weights with gaps."""
    kvs, keeps = [130, 60], [50, 20]
    pool, weights, tables, outs = make(device, kvs, keeps, seed=6)
    from kunserve_amd import KVPool
    def apart(x):
        y = torch.zeros(x.shape[0] + 1, x.shape[2], x.shape[1], x.shape[3], x.shape[4] + 8,
                        dtype=x.dtype, device=device)
        z = y[1:].transpose(1, 2)[..., :x.shape[4]]
        z.copy_(x)
        return z
    p2 = KVPool(apart(pool.k), apart(pool.v))
    wide = torch.zeros(weights.w.shape[:3] + (40,), device=device)[..., 3:19]
    wide.copy_(weights.w)
    check(device, p2, KVWeights(p2, wide), tables, kvs, outs, keeps, 4, 4)


def test_shared_source_pages(device):
    """Two requests with the same pages each get their choice."""
    kvs, keeps = [200, 200], [40, 70]
    pool, weights, tables, outs = make(device, kvs, keeps, seed=7)
    tables[1] = tables[0]
    check(device, pool, weights, tables, kvs, outs, keeps, 2, 8)


def test_on_another_stream(device):
    kvs, keeps = [900], [200]
    pool, weights, tables, outs = make(device, kvs, keeps, seed=8)
    s = torch.cuda.Stream(device)
    s.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(s):
        check(device, pool, weights, tables, kvs, outs, keeps, 4, 4)


def test_refusals(device):
    kvs, keeps = [100, 60], [30, 20]
    pool, weights, tables, outs = make(device, kvs, keeps, seed=9)
    with pytest.raises(ValueError, match="holds"):
        evict(pool, weights, tables, kvs, [tables[0][:2], outs[1]], keeps)
    with pytest.raises(ValueError, match="twice"):
        evict(pool, weights, tables, kvs, [[outs[0][0]] * 2, outs[1]], keeps)
    with pytest.raises(ValueError, match="pages for"):
        evict(pool, weights, tables, kvs, [outs[0][:1], outs[1]], keeps)
    with pytest.raises(IndexError):
        evict(pool, weights, tables, kvs, [[pool.num_pages, 0], outs[1]], keeps)
    with pytest.raises(ValueError, match="negative"):
        evict(pool, weights, tables, kvs, outs, keeps, sinks=-1)
    with pytest.raises(ValueError, match="negative"):
        evict(pool, weights, tables, kvs, outs, [-1, 4])
    with pytest.raises(ValueError, match="one per request"):
        evict(pool, weights, tables, kvs, outs, [1, 2, 3])
    with pytest.raises(ValueError, match="page lists"):
        evict(pool, weights, tables[:1], kvs, outs, keeps)
    other = random_pool(pool.num_pages + 1, 2, 3, 16, 64, device, 1)
    with pytest.raises(ValueError, match="not those"):
        evict(other, weights, tables, kvs, outs, keeps)
    with pytest.raises(ValueError, match="weights must be"):
        KVWeights(pool, weights.w[:-1])
    with pytest.raises(ValueError, match="weights must be"):
        KVWeights(pool, weights.w.double())
