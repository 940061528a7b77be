"""Attention of drafted trees against the formula in 64 bits: head layouts, sizes, splits,
strides, masks, values that are not finite, graphs and mixed steps."""
import math

import numpy as np
import pytest
import torch

from helpers import random_pool, random_tensor
from kunserve_amd import (AttentionStep, KVPool, LlamaOp, PageTable, Rotary, TreePlan, _lib,
                          append_kv, rope_inv_freq, tree_attention, tree_depths)
from tree_ref import check_out, random_pages, random_tree, tokens_of, tree_attention_ref

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def make(device, sizes, prefixes, hq, hkv, dim, page, dtype, fan=4, roots=1, layers=1, seed=0):
    rng = np.random.default_rng(seed)
    lens = [p + n for p, n in zip(prefixes, sizes)]
    lists, pages = random_pages(rng, lens, page)
    pool = random_pool(pages, layers, hkv, page, dim, device, seed + 1, dtype=dtype)
    trees = [random_tree(rng, n, fan, min(n, roots)) for n in sizes]
    total = int(sum(sizes))
    q = random_tensor((total, hq, dim), device, seed + 2, 2.0, dtype)
    k = random_tensor((total, hkv, dim), device, seed + 3, 1.0, dtype)
    v = random_tensor((total, hkv, dim), device, seed + 4, 1.0, dtype)
    return pool, lists, lens, trees, q, k, v


def row_reference(pool, layer, pages, n_kv, tree, q, k, v, scale):
    keys, values = (tokens_of(t, layer, pages, n_kv).clone() for t in (pool.k, pool.v))
    if k is not None:
        keys[:, n_kv - len(tree):] = k.transpose(0, 1)
        values[:, n_kv - len(tree):] = v.transpose(0, 1)
    return tree_attention_ref(q, keys, values, tree, scale)


def check_step(pool, layer, lists, lens, trees, q, k, v, out, scale, what=""):
    at = 0
    for b, tree in enumerate(trees):
        new = slice(at, at + len(tree))
        at += len(tree)
        ref, mass = row_reference(pool, layer, lists[b], lens[b], tree, q[new], k[new], v[new], scale)
        check_out(out[new], ref, mass, f"{what} row {b}")
        # appended to their places
        for t, x in ((pool.k, k), (pool.v, v)):
            got = tokens_of(t, layer, lists[b], lens[b])[:, lens[b] - len(tree):]
            assert torch.equal(got, x[new].transpose(0, 1)), (what, b)


CASES = [
    # sizes, prefixes, hq, hkv, dim, page, dtype, fan, roots
    ([8], [100], 8, 2, 128, 16, BF16, 3, 1),
    ([1], [0], 4, 4, 64, 16, F16, 1, 1),
    ([1, 1, 1], [0, 1, 129], 32, 8, 128, 16, F16, 1, 1),
    ([5, 64, 1, 17], [0, 1500, 3, 257], 32, 8, 128, 16, BF16, 6, 1),
    ([33, 32, 31], [127, 128, 129], 8, 8, 128, 4, F16, 9, 2),
    ([7, 20], [1000, 40], 6, 2, 64, 4, BF16, 3, 1),
    ([40, 3, 70], [255, 256, 511], 16, 4, 64, 32, F16, 200, 1),
    ([12, 9], [900, 64], 8, 2, 256, 16, BF16, 4, 1),
    ([64, 2], [70, 1], 4, 4, 256, 4, F16, 5, 3),
    ([130, 200], [300, 0], 10, 2, 128, 256, F16, 20, 1),
    ([300], [50], 2, 2, 64, 16, BF16, 1, 1),
    ([70, 128], [65, 4], 3, 1, 256, 32, BF16, 70, 1),
    ([16], [2000], 64, 1, 128, 16, F16, 4, 1),
    ([3, 2], [333, 90], 71, 1, 64, 16, F16, 2, 1),
    ([9] * 24, list(range(0, 2400, 100)), 14, 2, 128, 16, BF16, 4, 1),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{len(c[0])}x{max(c[0])}-{c[2]}on{c[3]}-{c[4]}-{c[5]}")
@pytest.mark.parametrize("split", [None, 1, 2])
def test_against_64_bits(device, case, split):
    sizes, prefixes, hq, hkv, dim, page, dtype, fan, roots = case
    pool, lists, lens, trees, q, k, v = make(device, sizes, prefixes, hq, hkv, dim, page, dtype,
                                             fan, roots, layers=2, seed=dim + hq)
    table = PageTable.from_lists(lists, lens, pool)
    plan = TreePlan(table, trees, hq, hkv, page, device, head_dim=dim, part_rounds=split or 0)
    qi = torch.tensor(np.cumsum([0, *sizes]), dtype=torch.int32, device=device)
    append_kv(pool, 1, table, qi, k, v)
    out = tree_attention(pool, 1, table, q, plan)
    check_step(pool, 1, lists, lens, trees, q, k, v, out, dim ** -0.5, str(case))
    if split is None:   # a step appends within its launch
        for t in (pool.k, pool.v):
            t[:, 0] = t[:, 1].flip(0)
        step = AttentionStep(pool, hq, sizes, prefixes, [1] * len(sizes), lists, trees=trees)
        out = step.run(0, q, k, v)
        check_step(pool, 0, lists, lens, trees, q, k, v, out, dim ** -0.5, str(case))


def test_scale_strides_and_in_place(device):
    """Slices of a projection's rows, a pool in a larger one's heads, out over q."""
    pool, lists, lens, trees, q, k, v = make(device, [9, 30], [140, 700], 8, 2, 128, 16, BF16)
    big = torch.randn(pool.num_pages, 3, 2, 5, 16, 128, device=device).to(BF16)
    wide = KVPool(big[:, :, 0, 1:3], big[:, :, 1, 1:3])
    wide.k.copy_(pool.k.expand(-1, 3, -1, -1, -1))
    wide.v.copy_(pool.v.expand(-1, 3, -1, -1, -1))
    rows = torch.cat([q, k, v], dim=1)
    rest = big[:, :, :, 0].clone(), big[:, :, :, 3:].clone()
    step = AttentionStep(wide, 8, [9, 30], [140, 700], [1, 1], lists, sm_scale=0.2, trees=trees)
    out = step.run(2, rows[:, :8], rows[:, 8:10], rows[:, 10:], out=rows[:, :8])
    assert out.data_ptr() == rows.data_ptr()
    check_step(wide, 2, lists, lens, trees, q, k, v, out, 0.2)
    assert torch.equal(rows[:, 8:], torch.cat([k, v], dim=1))
    assert torch.equal(big[:, :, :, 0], rest[0]) and torch.equal(big[:, :, :, 3:], rest[1])


def test_out_in_ks_memory(device):
    """Such a layer's append is a launch of its own."""
    pool, lists, lens, trees, q, k, v = make(device, [9, 30], [140, 700], 2, 2, 128, 16, F16)
    kk = k.clone()
    step = AttentionStep(pool, 2, [9, 30], [140, 700], [1, 1], lists, trees=trees)
    out = step.run(0, q, kk, v, out=kk)
    check_step(pool, 0, lists, lens, trees, q, k, v, out, 128 ** -0.5)


@pytest.mark.parametrize("dim,dtype", [(64, F16), (128, BF16), (256, F16)])
@pytest.mark.parametrize("tokens", [6, 50])
def test_values_that_are_not_finite(device, dim, dtype, tokens):
    """NaN and infinite keys and values of a drafted token reach those that see it alone."""
    hq, hkv = 4, 2
    pool, lists, lens, trees, q, k, v = make(device, [tokens, 12], [300, 77], hq, hkv, dim, 16,
                                             dtype, fan=2, seed=5)
    bad = tokens - 3
    k[bad, 0, 1] = math.nan
    v[bad, 1, 2] = math.inf
    v[bad + 1, 0, 3] = math.nan
    step = AttentionStep(pool, hq, [tokens, 12], [300, 77], [1, 1], lists, trees=trees)
    out = step.run(0, q, k, v)
    from tree_ref import ancestors
    sees = torch.tensor(ancestors(trees[0]), device=device)
    new = slice(0, tokens)
    keys, values = (tokens_of(t, 0, lists[0], lens[0]).clone() for t in (pool.k, pool.v))
    clean = torch.nan_to_num(keys, nan=0.0)
    ref, mass = tree_attention_ref(q[new], clean, values, trees[0], dim ** -0.5)
    want_nan = torch.zeros_like(ref, dtype=torch.bool)
    want_nan[:, :2] |= sees[:, bad, None, None]                    # a NaN key: its head's rows
    want_nan[:, :2, 3] |= sees[:, bad + 1, None]                   # a NaN value: one dim
    assert torch.equal(torch.isnan(out[new]), want_nan)
    inf = torch.zeros_like(want_nan)
    inf[:, 2:, 2] = sees[:, bad, None]
    assert torch.equal(torch.isinf(out[new]), inf)
    fine = ~want_nan & ~inf
    check_out(torch.where(fine, out[new], 0), torch.where(fine, ref, 0), mass)
    ref, mass = row_reference(pool, 0, lists[1], lens[1], trees[1], q[tokens:], None, None, dim ** -0.5)
    check_out(out[tokens:], ref, mass)


@pytest.mark.parametrize("dim,dtype", [(64, BF16), (128, F16), (256, BF16)])
def test_prefix_values_that_are_not_finite(device, dim, dtype):
    """An infinite cached value gives an infinite output, no NaN; a NaN query row NaN, the
    rows beside it nothing."""
    pool, lists, lens, trees, q, k, v = make(device, [20], [500], 4, 2, dim, 16, dtype, seed=9)
    pool.v[lists[0][3], 0, 1, 5, 7] = math.inf
    q[4, 0, 0] = math.nan
    step = AttentionStep(pool, 4, [20], [500], [1], lists, trees=trees)
    out = step.run(0, q, k, v)
    assert torch.isinf(out[:, 2:, 7]).all() and torch.isnan(out[4, 0]).all()
    ref, mass = row_reference(pool, 0, lists[0], lens[0], trees[0], torch.nan_to_num(q), k, v,
                              dim ** -0.5)
    fine = torch.ones_like(ref, dtype=torch.bool)
    fine[4, 0] = False
    fine[:, 2:, 7] = False
    check_out(torch.where(fine, out, 0), torch.where(fine, ref, 0), mass)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("tokens", [1, 70])
def test_a_long_tail_far_below_the_maximum(device, dim, dtype, tokens):
    """One token with a score 17.5 above 20000 others, which together have 5e-4 of its
    probability, each 2^-25.2 (less than a step of fp16 at 0)."""
    n, page = 20000, 16
    rng = np.random.default_rng(dim + tokens)
    lists, pages = random_pages(rng, [n + tokens], page)
    pool = random_pool(pages, 1, 1, page, dim, device, 1, dtype=dtype)
    pool.k.zero_()
    pool.v.fill_(-3.0)
    at = 12345
    pool.k[lists[0][at // page], 0, 0, at % page] = 17.5 / math.sqrt(dim)
    pool.v[lists[0][at // page], 0, 0, at % page] = 1.0
    q = torch.ones(tokens, 2, dim, device=device, dtype=dtype)
    k = torch.zeros(tokens, 1, dim, device=device, dtype=dtype)
    v = torch.full((tokens, 1, dim), -3.0, device=device, dtype=dtype)
    tree = random_tree(rng, tokens, 4)
    step = AttentionStep(pool, 2, [tokens], [n], [1], lists, trees=[tree])
    out = step.run(0, q, k, v)
    check_step(pool, 0, lists, [n + tokens], [tree], q, k, v, out, 1 / math.sqrt(dim))


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_slots_behind_a_row_do_not_matter(device, dim):
    """Neither NaN behind the row's last token nor what its new slots held before."""
    pool, lists, lens, trees, q, k, v = make(device, [10, 3], [90, 6], 4, 2, dim, 16, F16)
    for b, (n, tree) in enumerate(zip(lens, trees)):
        for t in (pool.k, pool.v):
            for at in range(n - len(tree), 16 * len(lists[b])):
                t[lists[b][at // 16], :, :, at % 16] = math.nan
    step = AttentionStep(pool, 4, [10, 3], [90, 6], [1, 1], lists, trees=trees)
    out = step.run(0, q, k, v)
    check_step(pool, 0, lists, lens, trees, q, k, v, out, dim ** -0.5)


def test_bad_page_ids_are_dropped(device):
    """From C: tokens of page ids outside the pool leave the softmax and are not appended."""
    import ctypes
    for dim, page in [(64, 4), (64, 16), (128, 16), (256, 4)]:
        pool, lists, lens, trees, q, k, v = make(device, [9], [200], 4, 2, dim, page, F16)
        table = PageTable.from_lists(lists, lens, pool)
        plan = TreePlan(table, trees, 4, 2, page, device, head_dim=dim)
        qi = torch.tensor([0, 9], dtype=torch.int32, device=device)
        append_kv(pool, 0, table, qi, k, v)
        gone = [0, 5, len(lists[0]) - 1]
        table.indices[gone] = torch.tensor([-1, pool.num_pages, 2**31 - 1], dtype=torch.int32,
                                           device=device)
        out = tree_attention(pool, 0, table, q, plan)
        dropped = np.array([t // page in gone for t in range(lens[0])])
        keys, values = (tokens_of(t, 0, lists[0], lens[0]) for t in (pool.k, pool.v))
        ref, mass = tree_attention_ref(q, keys, values, trees[0], dim ** -0.5, dropped)
        check_out(out, ref, mass, str(dim))
        table.indices[:] = -1
        assert not tree_attention(pool, 0, table, q, plan).any()


def test_tokens_of_no_row_are_left(device):
    pool, lists, lens, trees, q, k, v = make(device, [4, 6], [50, 20], 4, 2, 128, 16, BF16)
    table = PageTable.from_lists(lists, lens, pool)
    plan = TreePlan(table, trees, 4, 2, 16, device, q_first=[3, 9])
    qq = torch.randn(20, 4, 128, device=device).to(BF16)
    out = torch.full_like(qq, 7.0)
    tree_attention(pool, 0, table, qq, plan, out=out)
    for b, first in enumerate([3, 9]):
        new = slice(first, first + len(trees[b]))
        ref, mass = row_reference(pool, 0, lists[b], lens[b], trees[b], qq[new], None, None, 128 ** -0.5)
        check_out(out[new], ref, mass)
    rest = torch.ones(20, dtype=torch.bool, device=device)
    rest[3:7] = False
    rest[9:15] = False
    assert (out[rest] == 7).all()


def test_mixed_step_equals_its_rows_apart(device):
    """Decode, prefill and tree rows in one step, with a Rotary: bit for bit what each gives in
    a step of its own."""
    rng = np.random.default_rng(11)
    sizes, firsts = [1, 9, 40, 1, 17], [301, 500, 64, 77, 1000]
    flags = [0, 1, 1, 0, 1]
    trees = [None, random_tree(rng, 9, 3), None, None, random_tree(rng, 17, 4, 2)]
    lens = [f if not p else f + n for n, f, p in zip(sizes, firsts, flags)]
    lists, pages = random_pages(rng, lens, 16)
    rotary = Rotary(128, device=device)
    total = sum(sizes)
    q, k, v = (random_tensor((total, h, 128), device, 20 + h, 1.0, BF16) for h in (8, 2, 3))
    v = v[:, :2].contiguous()
    pools = [random_pool(pages, 1, 2, 16, 128, device, 4, dtype=BF16) for _ in range(2)]
    step = AttentionStep(pools[0], 8, sizes, firsts, flags, lists, trees=trees)
    out = step.run(0, q.clone(), k, v, rope=rotary)
    at = 0
    for b, n in enumerate(sizes):
        one = AttentionStep(pools[1], 8, [n], [firsts[b]], [flags[b]], [lists[b]], trees=[trees[b]])
        new = slice(at, at + n)
        at += n
        got = one.run(0, q[new].clone(), k[new], v[new], rope=rotary)
        if trees[b] is not None:   # splits differ with the step: rounded to the last bit at most
            torch.testing.assert_close(out[new].float(), got.float(), rtol=2 ** -7, atol=2 ** -9)
        else:
            torch.testing.assert_close(out[new].float(), got.float(), rtol=2 ** -6, atol=2 ** -7)
    assert torch.equal(pools[0].k, pools[1].k) and torch.equal(pools[0].v, pools[1].v)


def test_positions_follow_the_tree(device):
    """Rotated keys of a tree's tokens are those of a chain's at the same depth."""
    rng = np.random.default_rng(2)
    tree = random_tree(rng, 12, 3)
    pool, lists, lens, _, q, k, v = make(device, [12], [100], 4, 2, 64, 16, F16)
    rotary = Rotary(64, device=device)
    for start in (None, [5000]):
        step = AttentionStep(pool, 4, [12], [100], [1], lists, trees=[tree], rope_positions=start)
        at = (100 if start is None else 5000) + tree_depths(tree)
        assert step.positions.tolist() == at.tolist()
        step.run(0, q.clone(), k, v, rope=rotary)
        f = torch.tensor(10000.0 ** (-np.arange(0, 64, 2) / 64), device=device)
        angle = torch.tensor(at, device=device).double()[:, None] * f
        a, b = k[:, :, :32].double(), k[:, :, 32:].double()
        c, s = angle.cos()[:, None], angle.sin()[:, None]
        want = torch.cat([a * c - b * s, b * c + a * s], dim=-1).transpose(0, 1)
        got = tokens_of(pool.k, 0, lists[0], 112)[:, 100:].double()
        # half a step of the output, and the fp32 rotation's 2^-22 of |a| + |b|
        assert ((got - want).abs() <= want.abs() * 2.0 ** -11 + 2.0 ** -20 * 8).all()
    with pytest.raises(ValueError, match="Rotary"):
        step.run(0, q, k, v, rope=(rope_inv_freq(64, device=device), False))


def test_chain_is_a_prefill_row(device):
    pool, lists, lens, _, q, k, v = make(device, [30], [400], 8, 2, 128, 16, BF16)
    chain = [list(range(-1, 29))]
    a = AttentionStep(pool, 8, [30], [400], [1], lists, trees=chain).run(0, q, k, v)
    b = AttentionStep(pool, 8, [30], [400], [1], lists).run(0, q, k, v)
    torch.testing.assert_close(a.float(), b.float(), rtol=2 ** -6, atol=2 ** -7)


def test_captured_steps_share_nothing(device):
    """Two captured steps, replayed in turn between eager work, against eager results."""
    sets = [make(device, s, p, 8, 2, 128, 16, BF16, seed=31 + i)
            for i, (s, p) in enumerate([([9, 30], [700, 90]), ([64], [2100])])]
    graphs, want = [], []
    for pool, lists, lens, trees, q, k, v in sets:
        sizes = [len(t) for t in trees]
        step = AttentionStep(pool, 8, sizes, [n - s for n, s in zip(lens, sizes)], [1] * len(sizes),
                             lists, trees=trees)
        out = torch.empty_like(q)
        want.append(step.run(0, q, k, v).clone())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step.run(0, q, k, v, out=out)
        graphs.append((g, out, step))
    for i in (0, 1, 0, 0, 1):
        g, out, step = graphs[i]
        out.fill_(3.0)
        g.replay()
        other = step.run(0, sets[i][4], sets[i][5], sets[i][6])
        torch.cuda.synchronize()
        assert torch.equal(out, want[i]) and torch.equal(other, want[i])


def test_another_stream(device):
    pool, lists, lens, trees, q, k, v = make(device, [40, 3], [800, 10], 8, 2, 128, 16, F16)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step = AttentionStep(pool, 8, [40, 3], [800, 10], [1, 1], lists, trees=trees)
        out = step.run(0, q, k, v)
    s.synchronize()
    check_step(pool, 0, lists, lens, trees, q, k, v, out, 128 ** -0.5)


def test_pinned_host_tensors(device):
    pool, lists, lens, trees, q, k, v = make(device, [10, 5], [300, 44], 4, 2, 128, 16, BF16)
    host = [t.cpu().pin_memory() for t in (q, k, v)]
    step = AttentionStep(pool, 4, [10, 5], [300, 44], [1, 1], lists, trees=trees)
    out = step.run(0, *host, out=torch.empty_like(q))
    check_step(pool, 0, lists, lens, trees, q, k, v, out, 128 ** -0.5)


def test_llama_op_and_fused_pages(device):
    """pforward takes trees, on the whole model and on a pipeline stage of fused pages."""
    op = LlamaOp(40, 4, 8, 2, 16, 128, 0, 0, 0, 0, 0, 1, device=device, dtype=BF16)
    for t in (op.pool.k, op.pool.v):
        t.normal_()
    rng = np.random.default_rng(1)
    tree = random_tree(rng, 14, 3)
    q, k, v = (random_tensor((14, h, 128), device, h, 1.0, BF16) for h in (8, 2, 2))
    pages = [3, 7, 1, 20]
    step = op.pforward(1, 14, 40, 0, 4, [[0] * 14], [50], [1], [pages], trees=[tree])
    out = step.run(3, q, k, v)
    ref, mass = row_reference(op.pool, 3, pages, 64, tree, q, k, v, 128 ** -0.5)
    check_out(out, ref, mass)
    stage = op.pforward(1, 14, 80, 2, 4, [[0] * 14], [50], [1], [[40 + p for p in pages]], trees=[tree])
    got = stage.run(3, q, k, v)
    assert torch.equal(got, out)


def test_refusals(device):
    pool, lists, lens, trees, q, k, v = make(device, [10], [300], 4, 2, 128, 16, F16)
    from kunserve_amd import KVWeights
    new = lambda **kw: AttentionStep(pool, 4, [10], [300], [1], lists, **{"trees": trees, **kw})   # noqa: E731
    with pytest.raises(ValueError, match="1 rows but 2 trees"):
        new(trees=trees * 2)
    with pytest.raises(ValueError, match="tree of 9"):
        new(trees=[trees[0][:9]])
    with pytest.raises(ValueError, match="prefill row"):
        AttentionStep(pool, 4, [1], [300], [0], lists, trees=[[-1]])
    with pytest.raises(ValueError, match="prefill row"):
        new(is_context_stage=[0])
    with pytest.raises(ValueError, match="learn=False"):
        new(weights=KVWeights(pool))
    with pytest.raises(ValueError, match="parent"):
        new(trees=[[0] * 10])
    new(weights=KVWeights(pool), learn=False).run(0, q, k, v)
    # one-token trees say what their rows are, also where every row is flagged
    step = AttentionStep(pool, 4, [1], [300], [1], lists, use_tensor_cores=True, trees=[[-1]])
    assert step.kv_len.tolist() == [301]
    table = PageTable.from_lists(lists, lens, pool)
    plan = TreePlan(table, trees, 4, 2, 16, device)
    with pytest.raises(ValueError, match="another table"):
        tree_attention(pool, 0, PageTable.from_lists(lists, lens, pool), q, plan)
    with pytest.raises(ValueError, match="end at 10"):
        tree_attention(pool, 0, table, q[:9], plan)
    with pytest.raises(ValueError, match="dtype"):
        tree_attention(pool, 0, table, q.to(BF16), plan)
    with pytest.raises(_lib.KunserveError, match="query heads"):
        tree_attention(pool, 0, table, torch.cat([q, q], dim=1), plan)
    with pytest.raises(_lib.KunserveError, match="layer"):
        tree_attention(pool, 1, table, q, plan)
    other = random_pool(pool.num_pages, 1, 2, 32, 128, device, 1)
    with pytest.raises(_lib.KunserveError, match="pages of"):
        tree_attention(other, 0, table, q, plan)
    with pytest.raises(_lib.KunserveError, match="16-byte"):
        tree_attention(pool, 0, table, q, plan, out=torch.empty(10, 4, 129, dtype=F16, device=device)[..., 1:])
    with pytest.raises(_lib.KunserveError, match="finite"):
        tree_attention(pool, 0, table, q, plan, sm_scale=math.nan)


def test_no_rows(device):
    pool = random_pool(4, 1, 2, 16, 128, device, 1)
    step = AttentionStep(pool, 4, [], [], [], [], trees=[])
    q = torch.empty(0, 4, 128, dtype=F16, device=device)
    assert step.run(0, q, q[:, :2], q[:, :2]).shape == q.shape
