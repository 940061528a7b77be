"""A new token's weight comes from the observers that see it: a NaN query before it
leaves it a number."""
import math

import numpy as np
import pytest
import torch

import operators_ref as ref
from kunserve_amd import AttentionStep
from test_gpu_weights import build

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hq,hkv,d,dtype", [(4, 4, 64, torch.bfloat16), (8, 2, 128, torch.float16),
                                            (5, 1, 256, torch.float16)])
@pytest.mark.parametrize("long", [0, 64 * 256])
def test_nan_queries(device, hq, hkv, d, dtype, long):
    """The fourth-last query of a chunk is NaN in one head: of its KV head the last three
    tokens keep their weights, whether the last launch combines the statistics or
    (more than 64 partitions) another before it."""
    q_lens, kvs, window = [40, 20], [60 + long, 300], 8
    pool, tables, q, k, v, w = build(device, q_lens, kvs, hq, hkv, 256, d, dtype, seed=d)
    q[36, 0] = math.nan
    before = w.w.cpu().double().numpy()
    first = [n - t for t, n in zip(q_lens, kvs)]
    step = AttentionStep(pool, hq, q_lens, first, [1, 1], tables, weights=w, window=window)
    step.run(0, q, k, v)
    kh, got, at = pool.k.cpu(), w.w.cpu().double().numpy(), 0
    qh = torch.nan_to_num(q).cpu().double().numpy()
    for b, (t, n) in enumerate(zip(q_lens, kvs)):
        c = np.arange(n)
        where = (np.array(tables[b])[c // 256], 0, slice(None), c % 256)
        keys = ref.row_cache(kh, 0, tables[b], n)
        _, _, p, dp = ref.attend(qh[at:at + t], keys, keys, 1 / math.sqrt(d), dtype)
        want, tol = ref.add_weights(before[where].T, p, dp, t, window, hq // hkv)
        at += t
        new = got[where].T
        if b == 0:
            assert np.isnan(new[0, :n - 3]).all()
            new[0, :n - 3], want[0, :n - 3] = 0, 0
        assert np.all(np.abs(new - want) <= tol), b
