"""Steps take q, k, v and out in pinned host memory, op by op: with shared prefixes,
weights and a Rotary as without."""
import math

import numpy as np
import pytest
import torch

import operators_ref as ref
from helpers import random_pool, random_tensor
from kunserve_amd import (AttentionStep, KVPool, KVWeights, PageTable, Rotary, SharedDecodePlan,
                          shared_decode)

pytestmark = pytest.mark.gpu
PS, D, HQ, HKV = 16, 128, 8, 2


def shared_rows(device, kvs, root=9):
    own = [-(-n // PS) - root for n in kvs]
    perm = np.random.default_rng(1).permutation(root + sum(own)).tolist()
    at, tables = root, []
    for n in own:
        tables.append(perm[:root] + perm[at:at + n])
        at += n
    return random_pool(root + sum(own), 1, HKV, PS, D, device, 2), tables


def tensors(device, tokens, pinned):
    q, k, v = (random_tensor((tokens, h, D), device, 3 + h, 1.5) for h in (HQ, HKV, HKV + 1))
    v = v[:, :HKV].contiguous()
    x = [q, k, v, torch.zeros_like(q)]
    return [t.cpu().pin_memory() for t in x] if pinned else x


def twin(pool):
    return KVPool(pool.k.clone(), pool.v.clone())


@pytest.mark.parametrize("rope", [False, True])
def test_shared_prefixes(device, rope):
    kvs = [160, 200, 171]
    pool, tables = shared_rows(device, kvs)
    got = []
    for pinned, p in ((False, pool), (True, twin(pool))):
        q, k, v, out = tensors(device, 3, pinned)
        step = AttentionStep(p, HQ, [1] * 3, kvs, [0] * 3, tables, share_prefixes=True,
                             share_min_bytes=0, rope_positions=[7, 100000, 0] if rope else None)
        assert step.decode.plan.num_segments == 1
        step.run(0, q, k, v, out=out, rope=Rotary(64, device=device) if rope else None)
        torch.cuda.synchronize()
        got.append([t.cpu().view(torch.int16) for t in (out, q, p.k, p.v)])
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_shared_decode_gives_a_device_tensor(device):
    kvs = [160, 200, 171]
    pool, tables = shared_rows(device, kvs)
    table = PageTable.from_lists(tables, kvs, pool)
    plan = SharedDecodePlan(table, HQ, HKV, PS, device, min_bytes=0)
    q = random_tensor((3, HQ, D), device, 5)
    want = shared_decode(pool, 0, table, q, plan)
    got = shared_decode(pool, 0, table, q.cpu().pin_memory(), plan)
    assert got.device == pool.device and torch.equal(got.view(torch.int16), want.view(torch.int16))


def test_weights(device):
    """A mixed step's rows through add_weights; a decode step's as well."""
    for q_lens, first, flags in (([5, 9], [40, 3], [1, 1]), ([1, 1], [45, 12], [0, 0])):
        kvs = [45, 12]
        pool = random_pool(4, 1, HKV, PS, D, device, 6)
        tables = [[2, 0, 3], [1]]
        q, k, v, out = tensors(device, sum(q_lens), True)
        w = KVWeights(pool)
        w.w.uniform_(0, 1)
        before = w.w.cpu().double().numpy()
        AttentionStep(pool, HQ, q_lens, first, flags, tables, weights=w, window=4).run(
            0, q, k, v, out=out)
        torch.cuda.synchronize()
        kh, got, at = pool.k.cpu(), w.w.cpu().double().numpy(), 0
        for t, n, table in zip(q_lens, kvs, tables):
            c = np.arange(n)
            where = (np.array(table)[c // PS], 0, slice(None), c % PS)
            keys = ref.row_cache(kh, 0, table, n)
            _, _, p, dp = ref.attend(q[at:at + t].double().numpy(), keys, keys, 1 / math.sqrt(D),
                                     torch.float16)
            want, tol = ref.add_weights(before[where].T, p, dp, t, 4, HQ // HKV)
            assert np.all(np.abs(got[where].T - want) <= tol)
            at += t


def test_pageable_memory_is_refused(device):
    kvs = [160, 200, 171]
    pool, tables = shared_rows(device, kvs)
    q, k, v, out = (t.cpu() for t in tensors(device, 3, False))
    step = AttentionStep(pool, HQ, [1] * 3, kvs, [0] * 3, tables, share_prefixes=True,
                         share_min_bytes=0)
    with pytest.raises(ValueError, match="on cpu"):
        step.run(0, q, k, v, out=out)
    with pytest.raises(ValueError, match="out is on cpu"):
        shared_decode(pool, 0, step.decode.table, q.to(device), step.decode.plan, out=out)
