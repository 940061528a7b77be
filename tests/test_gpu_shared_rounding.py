"""Rows behind shared pages have the paged decode's two-term probabilities, in narrow
workgroups and in wide ones. Tokens of two scores, their values of opposite signs and
such that the output nearly vanishes: what one 16-bit term of the second probability
loses (in bf16 0.9e-3 of 0.493) then stands far above every other bound of
operators_ref."""
import math

import numpy as np
import pytest
import torch

import operators_ref as ref
from helpers import random_tensor
from kunserve_amd import DecodePlan, KVPool, PageTable, SharedDecodePlan, paged_decode, shared_decode

pytestmark = pytest.mark.gpu
PS, D, HQ, HKV, ROOT = 16, 128, 8, 2, 40


def cancelling(device, dtype, rows=33):
    """exp(-8 / sqrt(128)) = 0.493 of every second token, of values 1 and -2."""
    kvs = [ROOT * PS + 5 + i for i in range(rows)]
    own = [-(-n // PS) - ROOT for n in kvs]
    perm = np.random.default_rng(0).permutation(ROOT + sum(own)).tolist()
    common, at, tables = perm[:ROOT], ROOT, []
    for n in own:
        tables.append(common + perm[at:at + n])
        at += n
    pool = KVPool.allocate(ROOT + sum(own), 1, HKV, PS, D, device, dtype)
    pool.k.zero_()
    pool.k[..., 1::2, 0] = -1.0
    pool.v.fill_(1.0)
    pool.v[..., 1::2, :] = -2.0
    q = torch.zeros((rows, HQ, D), dtype=dtype, device=device)
    q[:, :, 0] = 8.0
    return pool, tables, kvs, q


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("form", ["wide", "narrow", "alone"])
def test_two_terms(device, dtype, form):
    pool, tables, kvs, q = cancelling(device, dtype)
    table = PageTable.from_lists(tables, kvs, pool)
    if form == "alone":
        out = paged_decode(pool, 0, table, q, DecodePlan(kvs, HQ, HKV, device))
    else:
        plan = SharedDecodePlan(table, HQ, HKV, PS, device, min_bytes=0,
                                num_cus=1 if form == "wide" else 256)
        assert plan.num_segments == 1 and plan.shared_info.wide == (form == "wide")
        out = shared_decode(pool, 0, table, q, plan)
    got, qh = out.cpu().double().numpy(), q.cpu().double().numpy()
    kh, vh = pool.k.cpu(), pool.v.cpu()
    for b, n in enumerate(kvs):
        k, v = (ref.row_cache(x, 0, tables[b], n) for x in (kh, vh))
        want, tol, _, _ = ref.attend(qh[b:b + 1], k, v, 1 / math.sqrt(D), dtype)
        assert np.all(np.abs(got[b] - want[0]) <= tol[0]), (b, np.abs(got[b] - want[0]).max())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hkv", [(8, 2), (16, 1), (64, 8)])
def test_random_values(device, dtype, hq, hkv):
    rng = np.random.default_rng(hq)
    rows, root = 40, 30
    kvs = [root * PS + int(x) for x in rng.integers(1, 200, size=rows)]
    own = [-(-n // PS) - root for n in kvs]
    perm = rng.permutation(root + sum(own)).tolist()
    common, at, tables = perm[:root], root, []
    for n in own:
        tables.append(common + perm[at:at + n])
        at += n
    pool = KVPool.allocate(root + sum(own), 1, hkv, PS, D, device, dtype)
    pool.k.copy_(random_tensor(pool.k.shape, device, 1, dtype=dtype))
    pool.v.copy_(random_tensor(pool.v.shape, device, 2, dtype=dtype))
    q = random_tensor((rows, hq, D), device, 3, 2.0, dtype)
    table = PageTable.from_lists(tables, kvs, pool)
    plan = SharedDecodePlan(table, hq, hkv, PS, device, min_bytes=0, num_cus=1)
    assert plan.shared_info.wide == 1
    out = shared_decode(pool, 0, table, q, plan)
    got, qh = out.cpu().double().numpy(), q.cpu().double().numpy()
    kh, vh = pool.k.cpu(), pool.v.cpu()
    for b, n in enumerate(kvs):
        k, v = (ref.row_cache(x, 0, tables[b], n) for x in (kh, vh))
        want, tol, _, _ = ref.attend(qh[b:b + 1], k, v, 1 / math.sqrt(D), dtype)
        assert np.all(np.abs(got[b] - want[0]) <= tol[0]), b
