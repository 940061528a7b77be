"""A captured step with positions on several axes: every replay against the eager result and
the rotation in 64 bits."""
import numpy as np
import pytest
import torch

from helpers import random_pool, random_tensor
from kunserve_amd import AttentionStep, Rotary
from test_gpu_rotary_axes import close, turned
from tree_ref import random_pages, tokens_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("starts", [False, True])
def test_replays(device, dtype, starts):
    rng = np.random.default_rng(3)
    lists, pages = random_pages(rng, [40, 21], 16)
    pool = random_pool(pages, 1, 2, 16, 128, device, 1, dtype=dtype)
    r = Rotary(128, device=device, sections=[16, 24, 24])
    q, k, v = (random_tensor((31, h, 128), device, h, 1.0, dtype) for h in (4, 2, 2))
    pos = np.array([300, 7]) if starts else rng.integers(0, 500, (3, 31))
    step = AttentionStep(pool, 4, [30, 1], [10, 21], [1, 0], lists, rope_positions=pos)
    every = np.tile(np.concatenate([300 + np.arange(30), [7]]), (3, 1)) if starts else pos
    at = torch.tensor(every, device=device)
    want_q, want_k = (turned(x, at, r.pair_axis.long(), r.frequencies, 128, False) for x in (q, k))
    qq, out = q.clone(), torch.empty_like(q)
    want = step.run(0, qq, k, v, rope=r).clone()
    rotated, cache = qq.clone(), [t.clone() for t in (pool.k, pool.v)]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step.run(0, qq, k, v, out=out, rope=r)
    for i in range(4):
        qq.copy_(q)
        out.fill_(1.0)
        for t in (pool.k, pool.v):   # slots 10 to 15 of the first row's first page: it appends them
            t[lists[0][0], :, :, 10:] = 0
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(qq, rotated)
        assert torch.equal(pool.k, cache[0]) and torch.equal(pool.v, cache[1])
        random_tensor((64, 64), device, i).sum()
    assert close(qq, want_q, q)
    new = torch.cat([tokens_of(pool.k, 0, lists[0], 40)[:, 10:], tokens_of(pool.k, 0, lists[1], 21)[:, 20:]], 1)
    assert close(new.transpose(0, 1), want_k, k)
