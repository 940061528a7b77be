"""Attention weights of the cache (AttentionStep(weights=...), add_weights)
against the softmax in 64 bits."""
import math

import numpy as np
import pytest
import torch

import operators_ref as ref
from helpers import random_pool, random_tensor
from kunserve_amd import AttentionStep, KVWeights, PageTable, WeightsPlan, add_weights

pytestmark = pytest.mark.gpu


def build(device, q_lens, kvs, hq, hkv, ps, d, dtype, layers=1, seed=0, q_scale=2.0):
    need = [-(-n // ps) for n in kvs]
    pages = sum(need) + 3
    perm = np.random.default_rng(seed).permutation(pages).tolist()
    tables = [[perm.pop() for _ in range(n)] for n in need]
    pool = random_pool(pages, layers, hkv, ps, d, device, seed, dtype=dtype)
    t = int(sum(q_lens))
    q = random_tensor((t, hq, d), device, seed + 1, q_scale, dtype)
    k = random_tensor((t, hkv, d), device, seed + 2, dtype=dtype)
    v = random_tensor((t, hkv, d), device, seed + 3, dtype=dtype)
    w = torch.rand((pages, layers, hkv, ps), device=device,
                   generator=torch.Generator(device=device).manual_seed(seed))
    return pool, tables, q, k, v, KVWeights(pool, w)


def check(pool, tables, q, weights, before, out, q_lens, kvs, layer, window):
    """Weights and outputs after a layer ran, against 64 bits; what no row owns
    unchanged."""
    hkv, ps, d = pool.num_kv_heads, pool.page_size, pool.head_dim
    ratio = q.shape[1] // hkv
    kh, vh, qh = pool.k.cpu(), pool.v.cpu(), q.cpu().double().numpy()
    got = weights.w.cpu().double().numpy()
    want, tol = before.cpu().double().numpy().copy(), np.zeros(before.shape)
    at = 0
    for table, t, n in zip(tables, q_lens, kvs):
        rows = slice(at, at + t)
        at += t
        if t == 0:
            continue
        k, v = ref.row_cache(kh, layer, table, n), ref.row_cache(vh, layer, table, n)
        o, o_tol, p, dp = ref.attend(qh[rows], k, v, 1 / math.sqrt(d), pool.dtype,
                                     p_err=ref.half_step(pool.dtype) if t > 1 else None)
        if out is not None:
            assert np.all(np.abs(out[rows].cpu().double().numpy() - o) <= o_tol)
        c = np.arange(n)
        where = (np.array(table)[c // ps], layer, slice(None), c % ps)
        new, err = ref.add_weights(want[where].T, p, dp, t, window, ratio)
        want[where], tol[where] = new.T, err.T
    assert np.all(np.abs(got - want) <= tol), float(np.max(np.abs(got - want) - tol))


RATIOS = [(4, 4), (8, 4), (6, 2), (8, 2), (10, 2), (16, 2), (16, 1), (34, 2)]


@pytest.mark.parametrize("hq,hkv", RATIOS)
@pytest.mark.parametrize("d,dtype", [(64, torch.float16), (128, torch.bfloat16),
                                     (128, torch.float16), (256, torch.bfloat16)])
def test_decode_rows(device, hq, hkv, d, dtype):
    kvs = [1, 2, 17, 255, 256, 257, 700]
    q_lens = [1] * len(kvs)
    pool, tables, q, k, v, weights = build(device, q_lens, kvs, hq, hkv, 16, d, dtype, 2, hq + d)
    before = weights.w.clone()
    step = AttentionStep(pool, hq, q_lens, kvs, [0] * len(kvs), tables, weights=weights)
    out = step.run(1, q, k, v)
    check(pool, tables, q, weights, before, out, q_lens, kvs, 1, 16)


@pytest.mark.parametrize("window", [1, 3, 16, 40, 1000])
@pytest.mark.parametrize("hq,hkv,d,dtype", [(4, 4, 64, torch.bfloat16), (8, 2, 128, torch.float16),
                                            (5, 1, 256, torch.float16)])
def test_prompt_rows(device, window, hq, hkv, d, dtype):
    q_lens, kvs = [1, 2, 30, 64, 130], [1, 40, 30, 500, 333]
    pool, tables, q, k, v, weights = build(device, q_lens, kvs, hq, hkv, 16, d, dtype, seed=window)
    before = weights.w.clone()
    first = [n - t for t, n in zip(q_lens, kvs)]
    step = AttentionStep(pool, hq, q_lens, first, [1] * 5, tables, weights=weights, window=window)
    out = step.run(0, q, k, v)
    check(pool, tables, q, weights, before, out, q_lens, kvs, 0, window)


@pytest.mark.parametrize("ps", [4, 32, 256])
def test_mixed_steps_and_page_sizes(device, ps):
    q_lens, kvs = [1, 50, 1, 7], [300, 90, 33, 7]
    pool, tables, q, k, v, weights = build(device, q_lens, kvs, 8, 2, ps, 128, torch.bfloat16,
                                           seed=ps)
    before = weights.w.clone()
    step = AttentionStep(pool, 8, q_lens, [300, 40, 33, 0], [0, 1, 0, 1], tables, weights=weights,
                         window=8)
    out = step.run(0, q, k, v)
    check(pool, tables, q, weights, before, out, q_lens, kvs, 0, 8)


def test_long_rows_and_many(device):
    kvs = [9000, 4096, 1, 5000] + list(range(2, 40))
    q_lens = [1] * len(kvs)
    pool, tables, q, k, v, weights = build(device, q_lens, kvs, 8, 2, 16, 128, torch.float16)
    before = weights.w.clone()
    step = AttentionStep(pool, 8, q_lens, kvs, [0] * len(kvs), tables, weights=weights)
    out = step.run(0, q, k, v)
    check(pool, tables, q, weights, before, out, q_lens, kvs, 0, 16)


def test_weights_add_up_over_steps(device):
    """Prompt, then decode steps: what a cache has learnt is the sum, and pages
    need no clearing."""
    hq, hkv, d, ps = 8, 2, 64, 16
    pool, tables, q, k, v, weights = build(device, [40], [60], hq, hkv, ps, d, torch.float16,
                                           seed=3)
    weights.w.fill_(float("nan"))   # whatever the pages' last user left
    n = 0
    for t, flag in ((40, 1), (1, 0), (1, 0), (15, 1)):
        n += t
        x, y, z = (random_tensor((t, h, d), device, 50 + n + h) for h in (hq, hkv, hkv))
        step = AttentionStep(pool, hq, [t], [n if not flag else n - t], [flag], tables,
                             weights=weights, window=16)
        before = weights.w.clone()
        out = step.run(0, x, y, z)
        idx = np.arange(n)
        place = (torch.tensor(np.array(tables[0])[idx // ps], device=device), 0, slice(None),
                 torch.tensor(idx % ps, device=device))
        assert torch.isfinite(weights.w[place]).all()
        fixed = torch.nan_to_num(before)
        now = KVWeights(pool, torch.nan_to_num(weights.w))
        check(pool, [tables[0]], x, now, fixed, out, [t], [n], 0, 16)
    total = float(weights.w[place].sum())
    # every observer gave each KV head its query heads' ones, what later steps
    # overwrote aside: 16 + 1 + 1 + 15 observers of 8 heads
    assert abs(total - 33 * hq) < 1e-3 * 33 * hq


def test_padded_rows_of_add_weights(device):
    """A table with rows that bring no tokens in this step, and tokens behind
    the last row."""
    q_lens, kvs = [0, 3, 0, 1], [20, 50, 0, 33]
    pool, tables, q, k, v, weights = build(device, q_lens, kvs, 4, 2, 16, 64, torch.bfloat16)
    q = torch.cat([q, torch.full_like(q, float("nan"))])
    before = weights.w.clone()
    table = PageTable.from_lists(tables, kvs, pool)
    qi = np.r_[0, np.cumsum(q_lens)]
    plan = WeightsPlan(qi, kvs, 4, 2, device)
    add_weights(pool, weights, 0, table, torch.tensor(qi, dtype=torch.int32, device=device), q, plan)
    check(pool, tables, q[:4], weights, before, None, q_lens, kvs, 0, 2)


def test_values_that_are_not_finite(device):
    """NaN and infinity behind a row's end and in other rows' pages stay there;
    a NaN key makes its row's weights NaN and no other's."""
    q_lens, kvs = [1, 1, 1], [20, 40, 20]
    pool, tables, q, k, v, weights = build(device, q_lens, kvs, 8, 2, 16, 128, torch.bfloat16)
    pool.k[tables[0][1], :, :, 4:] = float("nan")     # behind row 0's end
    pool.v[tables[0][1], :, :, 4:] = float("inf")
    pool.k[tables[2][0], :, 0, 3, 0] = float("nan")
    before = weights.w.clone()
    step = AttentionStep(pool, 8, q_lens, kvs, [0, 0, 0], tables, weights=weights)
    out = step.run(0, q, k, v)
    bad = weights.w[tables[2][0], 0, 0]
    assert torch.isnan(bad).all()
    assert torch.isfinite(weights.w[tables[2][0], 0, 1]).all()
    check(pool, tables[:2], q[:2], weights, _with(before, weights, tables[2]), out[:2], q_lens[:2],
          kvs[:2], 0, 16)


def _with(before, weights, table):
    """`before`, with a row's new weights put in (it is not checked)."""
    w = before.clone()
    w[table] = torch.nan_to_num(weights.w[table])
    weights.w[table] = torch.nan_to_num(weights.w[table])
    return w


def test_strides_and_another_stream(device):
    """Weights with gaps, q as a slice, pools whose heads lie apart, on a stream of
    its own."""
    from kunserve_amd import KVPool
    q_lens, kvs = [1, 30, 1], [300, 90, 17]
    pool, tables, q, k, v, weights = build(device, q_lens, kvs, 8, 2, 16, 128, torch.float16)
    kk, vv = (torch.zeros((pool.num_pages, 2, 1, 16, 136), dtype=torch.float16,
                          device=device).transpose(1, 2)[..., :128] for _ in range(2))
    kk.copy_(pool.k)
    vv.copy_(pool.v)
    other = KVPool(kk, vv)
    wide = torch.full((pool.num_pages, 2, 2, 24), 5.0, device=device)
    w = KVWeights(other, wide[:, 1:, :, 4:20])
    w.w.copy_(weights.w)
    before = w.w.clone()
    big = random_tensor((32, 12, 128), device, 77, 2.0)
    big[:, 3:11] = q
    s = torch.cuda.Stream(device)
    s.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(s):
        step = AttentionStep(other, 8, q_lens, [300, 60, 17], [0, 1, 0], tables, weights=w,
                             window=7)
        out = step.run(0, big[:, 3:11], k, v)
    s.synchronize()
    check(other, tables, q, w, before, out, q_lens, kvs, 0, 7)
    wide[:, 1:, :, 4:20] = 5.0
    assert (wide == 5.0).all()


def test_rows_over_many_partitions(device):
    """A chunk on a prefix of more partitions than the last launch combines."""
    q_lens, kvs = [20, 40], [64 * 256 + 300, 50]
    pool, tables, q, k, v, weights = build(device, q_lens, kvs, 4, 2, 256, 64, torch.bfloat16)
    before = weights.w.clone()
    first = [n - t for t, n in zip(q_lens, kvs)]
    step = AttentionStep(pool, 4, q_lens, first, [1, 1], tables, weights=weights, window=5)
    assert step._weights_plan.info.num_combines > 0
    out = step.run(0, q, k, v)
    check(pool, tables, q, weights, before, out, q_lens, kvs, 0, 5)


def test_captured_step_replays(device):
    """A captured layer, replayed with eager work between, adds each time what
    the eager one adds."""
    q_lens, kvs = [1, 20, 1], [400, 60, 31]
    pool, tables, q, k, v, weights = build(device, q_lens, kvs, 8, 2, 16, 128, torch.float16)
    before = weights.w.clone()
    step = AttentionStep(pool, 8, q_lens, [400, 40, 31], [0, 1, 0], tables, weights=weights)
    out = torch.empty_like(q)
    want = []
    for _ in range(3):
        step.run(0, q, k, v, out=out)
        want.append(weights.w.clone())
    eager = out.clone()
    weights.w.copy_(before)
    out.zero_()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step.run(0, q, k, v, out=out)
    for i in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(weights.w, want[i])
        assert torch.equal(out.view(torch.int16), eager.view(torch.int16))
        torch.randn(1000, device=device).sum()


def test_refusals(device):
    q_lens, kvs = [1, 1], [40, 20]
    pool, tables, q, k, v, weights = build(device, q_lens, kvs, 4, 2, 16, 64, torch.float16)
    with pytest.raises(ValueError, match="in one place"):
        AttentionStep(pool, 4, q_lens, kvs, [0, 0], [tables[0], tables[0]], weights=weights)
    with pytest.raises(ValueError, match="window"):
        AttentionStep(pool, 4, q_lens, kvs, [0, 0], tables, weights=weights, window=0)
    other = random_pool(pool.num_pages, 2, 2, 16, 64, device, 1)
    with pytest.raises(ValueError, match="not those"):
        AttentionStep(other, 4, q_lens, kvs, [0, 0], tables, weights=weights)
    step = AttentionStep(pool, 4, q_lens, kvs, [0, 0], tables, weights=weights)
    with pytest.raises((RuntimeError, ValueError), match="overlaps q"):
        step.run(0, q, k, v, out=q)
    table = PageTable.from_lists(tables, kvs, pool)
    plan = WeightsPlan([0, 1, 2], kvs, 8, 4, device)
    qi = torch.tensor([0, 1, 2], dtype=torch.int32, device=device)
    with pytest.raises(RuntimeError, match="plan made for 8"):
        add_weights(pool, weights, 0, table, qi, q, plan)
    plan = WeightsPlan([0, 1, 2], [40, 21], 4, 4, device)
    with pytest.raises(ValueError, match="other rows"):
        add_weights(pool, weights, 0, table, qi, q, plan)
    plan = WeightsPlan([0, 1, 2], kvs, 4, 4, device)
    with pytest.raises(ValueError, match="on cpu"):
        add_weights(pool, weights, 0, table, qi, q.cpu(), plan)
    twice = PageTable.from_lists([tables[0], tables[0]], kvs, pool)
    with pytest.raises(ValueError, match="in one place"):
        add_weights(pool, weights, 0, twice, qi, q, plan)
    with pytest.raises(RuntimeError, match="sm_scale"):
        add_weights(pool, weights, 0, table, qi, q, plan, sm_scale=float("nan"))
