"""NaN keys in rows that learn weights: the weights of the row and KV head become NaN,
never infinite, also where every partition of a split row holds one; all others keep
their values, and an eviction after it keeps the tokens whose weights are numbers."""
import math

import numpy as np
import pytest
import torch

import operators_ref as ref
from helpers import random_pool, random_tensor
from kunserve_amd import AttentionStep, KVWeights, evict

pytestmark = pytest.mark.gpu
PS = 16


def rows(device, kvs, hkv, d, dtype, extra=0):
    need = [-(-n // PS) for n in kvs]
    pool = random_pool(sum(need) + extra, 1, hkv, PS, d, device, d, dtype=dtype)
    perm = np.random.default_rng(d).permutation(sum(need) + extra).tolist()
    tables = [[perm.pop() for _ in range(n)] for n in need]
    return pool, tables, perm


def learn(pool, tables, kvs, hq, w, part):
    device, hkv, d = pool.device, pool.num_kv_heads, pool.head_dim
    q = random_tensor((len(kvs), hq, d), device, 3, 2.0, pool.dtype)
    at = [(t[(n - 1) // PS], (n - 1) % PS) for t, n in zip(tables, kvs)]
    k, v = (torch.stack([x[p, 0, :, s] for p, s in at]) for x in (pool.k, pool.v))
    step = AttentionStep(pool, hq, [1] * len(kvs), kvs, [0] * len(kvs), tables, weights=w,
                         decode_part_tokens=part)
    return step, q, step.run(0, q, k, v)


@pytest.mark.parametrize("every", [False, True])
@pytest.mark.parametrize("part,long", [(0, 700), (256, 700), (256, 4200)])
@pytest.mark.parametrize("hq,hkv,d,dtype", [(4, 4, 64, torch.float16), (4, 2, 128, torch.bfloat16),
                                            (8, 2, 128, torch.float16), (8, 2, 256, torch.bfloat16),
                                            (34, 2, 64, torch.bfloat16)])
def test_weights(device, hq, hkv, d, dtype, part, long, every):
    """In one partition or in every one; combined by the launch, or (17 partitions) by a
    second one."""
    kvs = [long, 300, 20]
    pool, tables, _ = rows(device, kvs, hkv, d, dtype)
    host = pool.k.cpu()
    for t in (range(10, long, 128) if every else [300]):
        pool.k[tables[0][t // PS], 0, hkv - 1, t % PS, 1] = math.nan
    w = KVWeights(pool)
    w.w.uniform_(0, 1)
    before = w.w.cpu().double().numpy()
    step, q, _ = learn(pool, tables, kvs, hq, w, part)
    if part:
        assert (step._step.num_counters > 0) == (long == 700)
    got, qh = w.w.cpu().double().numpy(), q.cpu().double().numpy()
    for b, n in enumerate(kvs):
        c = np.arange(n)
        where = (np.array(tables[b])[c // PS], 0, slice(None), c % PS)
        k = ref.row_cache(host, 0, tables[b], n)
        _, _, p, dp = ref.attend(qh[b:b + 1], k, k, 1 / math.sqrt(d), dtype)
        want, tol = ref.add_weights(before[where].T, p, dp, 1, 16, hq // hkv)
        new = got[where].T
        if b == 0:
            assert np.isnan(new[-1]).all()
            new, want, tol = new[:-1], want[:-1], tol[:-1]
        assert np.all(np.abs(new - want) <= tol), b


def test_an_eviction_after_it(device):
    """Weights that are not numbers are the lightest: of a head with NaN keys in every
    partition stay, between the first and the last, the first tokens."""
    kvs = [700]
    pool, tables, free = rows(device, kvs, 2, 64, torch.float16, extra=3)
    for t in range(10, 700, 128):
        pool.k[tables[0][t // PS], 0, 1, t % PS, 1] = math.nan
    w = KVWeights(pool)
    learn(pool, tables, kvs, 8, w, 256)
    kept = evict(pool, w, tables, kvs, [free], 48, sinks=4, recent=8).cpu().numpy()
    assert kept[0, 0, 1].tolist() == list(range(40)) + list(range(692, 700))
    first = w.w[torch.tensor(tables[0], device=device), 0, 0].reshape(-1)[:700].cpu().numpy()
    np.testing.assert_array_equal(kept[0, 0, 0], ref.choose(first, 48, 4, 8))
