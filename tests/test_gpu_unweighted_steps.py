"""Steps that learn nothing in a pool with weights (learn=False; KVWeights.clear for
tokens appended by an op): the new tokens' weights become 0 whatever their pages' last
user left, in every layer, and nothing else changes."""
import math

import numpy as np
import pytest
import torch

import operators_ref as ref
from helpers import random_pool, random_tensor
from kunserve_amd import (AttentionStep, KVPool, KVWeights, LlamaOp, PageTable, append_kv, evict)

pytestmark = pytest.mark.gpu
LEFT = [math.nan, math.inf, -math.inf, 7.0]     # what the last user left, by page


def stale(w):
    for page in range(w.shape[0]):
        w[page] = LEFT[page % 4]


def bits(w):
    return w.contiguous().view(torch.int32).cpu()


@pytest.mark.parametrize("ps", [4, 16, 256])
@pytest.mark.parametrize("strided", [False, True])
def test_the_new_tokens_and_no_others(device, ps, strided):
    """A prompt, a chunk and two decode rows; the decode rows share their first pages."""
    q_lens, kvs, flags = [1, 30, 1, 70], [600, 30, 700, 300], [0, 1, 0, 1]
    root = 512 // ps
    need = [-(-n // ps) for n in kvs]
    perm = np.random.default_rng(ps).permutation(sum(need) + 5).tolist()
    common = [perm.pop() for _ in range(root)]
    tables = [(common if f == 0 else []) + [perm.pop() for _ in range(n - (root if f == 0 else 0))]
              for n, f in zip(need, flags)]
    pool = random_pool(sum(need) + 5, 3, 2, ps, 128, device, 1)
    w = KVWeights(pool)
    if strided:
        wide = torch.zeros((pool.num_pages, 2, 5, ps + 8), device=device)
        w = KVWeights(pool, wide.transpose(1, 2)[:, 1:4, :, 4:4 + ps])
    stale(w.w)
    want = w.w.clone()
    for t, n, table in zip(q_lens, kvs, tables):
        for c in range(n - t, n):
            want[table[c // ps], :, :, c % ps] = 0
    q, k, v = (random_tensor((sum(q_lens), h, 128), device, h) for h in (8, 2, 2))
    first = [n if f == 0 else n - t for t, n, f in zip(q_lens, kvs, flags)]
    step = AttentionStep(pool, 8, q_lens, first, flags, tables, share_prefixes=True,
                         share_min_bytes=0, weights=w, learn=False)
    assert step.decode.plan.num_segments == 1
    twin = KVPool(pool.k.clone(), pool.v.clone())
    for layer in range(3):
        out = step.run(layer, q, k, v)
    assert torch.equal(bits(w.w), bits(want))
    plain = AttentionStep(twin, 8, q_lens, first, flags, tables, share_prefixes=True,
                          share_min_bytes=0)
    for layer in range(3):
        same = plain.run(layer, q, k, v)
    assert torch.equal(out.view(torch.int16), same.view(torch.int16))
    if strided:
        wide.transpose(1, 2)[:, 1:4, :, 4:4 + ps] = 0
        assert not wide.any()


def test_after_an_append(device):
    pool = random_pool(9, 40, 8, 16, 64, device, 1)    # more heads than a workgroup has threads
    w = KVWeights(pool)
    stale(w.w)
    want = w.w.clone()
    q_lens, kvs, tables = [0, 3, 0, 20], [20, 50, 0, 33], [[0, 1], [2, 3, 4, 5], [], [6, 7, 8]]
    for t, n, table in zip(q_lens, kvs, tables):
        for c in range(n - t, n):
            want[table[c // 16], :, :, c % 16] = 0
    table = PageTable.from_lists(tables, kvs, pool)
    qi = torch.tensor(np.r_[0, np.cumsum(q_lens)], dtype=torch.int32, device=device)
    k = random_tensor((25, 8, 64), device, 2)           # two tokens of no row
    append_kv(pool, 5, table, qi, k, k)
    w.clear(pool, table, qi, 25)
    assert torch.equal(bits(w.w), bits(want))


def test_requests_behind_a_learnt_prompt_are_shortened(device):
    """A prompt learns its weights; requests that share its pages append tokens in steps
    that learn nothing, on pages whose last user left NaN and infinities; an eviction
    then goes by the prompt's weights and takes the new tokens for weightless."""
    hq, hkv, d, ps, layers = 8, 2, 64, 16, 2
    op = LlamaOp(120, layers, hq, hkv, ps, d, 256, 1000, 8, 512, 4096, 1, device=device)
    free = np.random.default_rng(1).permutation(120).tolist()
    prompt = [free.pop() for _ in range(12)]
    weights = KVWeights(op.pool)
    stale(weights.w)

    def run(q_lens, first, flags, tables, **kw):
        total = sum(q_lens)
        s = op.pforward(len(tables), total, op.max_num_pages, 0, layers, [[1] * t for t in q_lens],
                        first, flags, tables, weights=weights, **kw)
        for layer in range(layers):
            s.run(layer, *(random_tensor((total, h, d), device, 10 + layer + h, 1.5)
                           for h in (hq, hkv, hkv)))

    run([192], [0], [1], [prompt], window=8)
    learnt = weights.w[prompt].clone()
    assert torch.isfinite(learnt).all()
    tables = [prompt + [free.pop() for _ in range(2)] for _ in range(3)]
    run([1] * 3, [193] * 3, [0] * 3, tables, share_prefixes=True, learn=False)
    run([1, 3, 1], [194, 193, 194], [0, 1, 0], tables, share_prefixes=True, learn=False)
    assert torch.equal(weights.w[prompt], learnt)
    kvs = [194, 196, 194]
    outs = [[free.pop() for _ in range(4)] for _ in range(3)]
    kept = evict(op.pool, weights, tables, kvs, outs, 64, sinks=4, recent=1).cpu().numpy()
    for b, n in enumerate(kvs):
        for layer in range(layers):
            for h in range(hkv):
                w = np.zeros(n, dtype=np.float32)
                w[:192] = learnt[:, layer, h].cpu().numpy().reshape(-1)
                np.testing.assert_array_equal(kept[b, layer, h], ref.choose(w, 64, 4, 1))
