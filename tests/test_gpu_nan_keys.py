"""A NaN in a row's keys, or a score that is infinite, makes the outputs of its row and
KV head NaN, by the softmax's definition, whichever way the row is attended: whole or
split, by the vector or the matrix units, with its partials combined by the launch or
by a second one, behind shared pages, or while weights are learnt. Every other row and
head keeps its values (bounds of operators_ref)."""
import math

import numpy as np
import pytest
import torch

import operators_ref as ref
from helpers import random_pool, random_tensor
from kunserve_amd import (AttentionStep, DecodePlan, KVWeights, PageTable, SharedDecodePlan,
                          paged_decode, shared_decode)

pytestmark = pytest.mark.gpu

PS = 16
KVS = [257, 33, 700, 1030, 64, 900]
# row, KV head (-1: the last), places: one partition of a row, its only one, every one
# of 256, the first alone, the last token, and a row without any
BAD = [(0, 0, [256]), (1, -1, [7]), (2, 0, [1, 300, 699]), (3, -1, [5]), (4, 0, [63])]
HEADS = [(4, 4), (4, 2), (6, 2), (8, 2), (16, 1), (34, 2)]


def build(device, hq, hkv, d, dtype, root=0, value=math.nan):
    """Rows of KVS behind `root` shared pages, and the heads that stay clean."""
    rng = np.random.default_rng(hq + d)
    need = [-(-n // PS) for n in KVS]
    pages = root + sum(need)
    perm = rng.permutation(pages).tolist()
    common, at, tables = perm[:root], root, []
    for n in need:
        tables.append(common + perm[at:at + n])
        at += n
    kvs = [root * PS + n for n in KVS]
    pool = random_pool(pages, 1, hkv, PS, d, device, d + hq, dtype=dtype)
    clean = np.ones((len(kvs), hq), dtype=bool)
    ratio = hq // hkv
    marks = []
    for b, h, places in BAD:
        h %= hkv
        clean[b, h * ratio:(h + 1) * ratio] = False
        for t in places:
            t += root * PS
            marks.append((tables[b][t // PS], 0, h, t % PS, (5 * t) % d))
    q = random_tensor((len(kvs), hq, d), device, 3, 2.0, dtype)
    if value == math.inf:
        q = q.abs() + 2.0 ** -6     # every score of that token is +inf
    host = [x.cpu() for x in (pool.k, pool.v)]
    for m in marks:
        pool.k[m] = value
    return pool, tables, kvs, q, clean, host


def check(out, q, clean, tables, kvs, host, d, dtype):
    got, qh = out.cpu().double().numpy(), q.cpu().double().numpy()
    for b, n in enumerate(kvs):
        k, v = (ref.row_cache(x, 0, tables[b], n) for x in host)
        want, tol, _, _ = ref.attend(qh[b:b + 1], k, v, 1 / math.sqrt(d), dtype)
        assert np.isnan(got[b][~clean[b]]).all(), (b, got[b][~clean[b]])
        assert np.all((np.abs(got[b] - want[0]) <= tol[0])[clean[b]]), b


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("d,dtype", [(64, torch.float16), (128, torch.bfloat16),
                                     (128, torch.float16), (256, torch.bfloat16)])
@pytest.mark.parametrize("hq,hkv", HEADS)
def test_decode(device, hq, hkv, d, dtype, value):
    pool, tables, kvs, q, clean, host = build(device, hq, hkv, d, dtype, value=value)
    table = PageTable.from_lists(tables, kvs, pool)
    for part in (0, 256, 4096):
        out = paged_decode(pool, 0, table, q, DecodePlan(kvs, hq, hkv, device, part, head_dim=d))
        check(out, q, clean, tables, kvs, host, d, dtype)


def last_rows(pool, tables, kvs):
    at = [(t[(n - 1) // PS], (n - 1) % PS) for t, n in zip(tables, kvs)]
    return [torch.stack([x[p, 0, :, s] for p, s in at]) for x in (pool.k, pool.v)]


@pytest.mark.parametrize("learn", [False, True])
@pytest.mark.parametrize("d,dtype", [(64, torch.bfloat16), (128, torch.float16),
                                     (256, torch.float16)])
@pytest.mark.parametrize("hq,hkv", HEADS)
@pytest.mark.parametrize("part", [0, 256])
def test_steps(device, hq, hkv, d, dtype, learn, part):
    """Steps whose launch combines its split rows, and appends their last keys."""
    pool, tables, kvs, q, clean, host = build(device, hq, hkv, d, dtype)
    k, v = last_rows(pool, tables, kvs)
    weights = KVWeights(pool) if learn else None
    step = AttentionStep(pool, hq, [1] * len(kvs), kvs, [0] * len(kvs), tables, weights=weights,
                         decode_part_tokens=part)
    check(step.run(0, q, k, v), q, clean, tables, kvs, host, d, dtype)


def test_steps_with_a_second_launch(device):
    """A row of more partitions than its launch combines."""
    kvs = [4200, 300]
    pool = random_pool(300, 1, 2, PS, 128, device, 1)
    tables = [list(range(263)), list(range(263, 282))]
    host = [x.cpu() for x in (pool.k, pool.v)]
    for page in range(0, 262, 8):       # in every partition of 256
        pool.k[page, 0, 0, 3, 7] = math.nan
    q = random_tensor((2, 8, 128), device, 3, 2.0)
    clean = np.ones((2, 8), dtype=bool)
    clean[0, :4] = False
    for learn in (False, True):
        k, v = last_rows(pool, tables, kvs)
        step = AttentionStep(pool, 8, [1, 1], kvs, [0, 0], tables, decode_part_tokens=256,
                             weights=KVWeights(pool) if learn else None)
        assert step._step.num_counters == 0 and step.decode.plan.info.num_merge == 2
        check(step.run(0, q, k, v), q, clean, tables, kvs, host, 128, torch.float16)


@pytest.mark.parametrize("root", [5, 40])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hq,hkv", [(4, 4), (8, 2), (34, 2)])
def test_behind_shared_pages(device, hq, hkv, d, root):
    pool, tables, kvs, q, clean, host = build(device, hq, hkv, d, torch.bfloat16, root)
    table = PageTable.from_lists(tables, kvs, pool)
    plan = SharedDecodePlan(table, hq, hkv, PS, device, head_dim=d, min_bytes=0)
    assert plan.num_segments == 1
    out = shared_decode(pool, 0, table, q, plan)
    check(out, q, clean, tables, kvs, host, d, torch.bfloat16)
    plain = paged_decode(pool, 0, table, q, DecodePlan(kvs, hq, hkv, device, head_dim=d))
    check(plain, q, clean, tables, kvs, host, d, torch.bfloat16)
