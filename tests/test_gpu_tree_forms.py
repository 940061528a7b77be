"""Drafted trees in the forms that the kernel has apart: pages of 4, 8 and 16 tokens at every
head size, and workgroups of 32 to 256 columns, with values that are not finite and page ids
outside the pool in each."""
import math

import numpy as np
import pytest
import torch

from kunserve_amd import AttentionStep, PageTable, TreePlan, append_kv, tree_attention
from test_gpu_tree import check_step, make, row_reference
from tree_ref import ancestors, check_out, tokens_of, tree_attention_ref

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16

# (head_dim, query heads, KV heads, tokens of the widest row, columns of its workgroups)
FORMS = [(64, 4, 4, 20, 32), (64, 8, 4, 30, 64), (64, 8, 2, 64, 128),
         (128, 4, 4, 20, 32), (128, 8, 4, 30, 64), (128, 8, 4, 64, 128), (128, 16, 4, 64, 256),
         (256, 8, 4, 30, 64), (256, 8, 2, 64, 128)]
PAGES = [4, 8, 16]


def plan_of(pool, table, trees, hq, hkv, page, device, dim, columns, part_rounds=0):
    plan = TreePlan(table, trees, hq, hkv, page, device, head_dim=dim, part_rounds=part_rounds)
    assert plan.info.columns == columns
    return plan


@pytest.mark.parametrize("dim,hq,hkv,tokens,columns", FORMS)
@pytest.mark.parametrize("page", PAGES)
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_against_64_bits(device, dim, hq, hkv, tokens, columns, page, dtype):
    """Prefixes that end within a page, a load and a round, at one, and that are none."""
    sizes = [tokens, tokens - 1, tokens, 3, tokens]
    prefixes = [777, 256, 261, 5, 0]
    pool, lists, lens, trees, q, k, v = make(device, sizes, prefixes, hq, hkv, dim, page, dtype,
                                             seed=dim + page, layers=2)
    table = PageTable.from_lists(lists, lens, pool)
    qi = torch.tensor(np.cumsum([0, *sizes]), dtype=torch.int32, device=device)
    append_kv(pool, 1, table, qi, k, v)
    for split in (0, 1, 2):
        plan = plan_of(pool, table, trees, hq, hkv, page, device, dim, columns, split)
        out = tree_attention(pool, 1, table, q, plan)
        check_step(pool, 1, lists, lens, trees, q, k, v, out, dim ** -0.5, f"split {split}")
    step = AttentionStep(pool, hq, sizes, prefixes, [1] * len(sizes), lists, trees=trees)
    assert step.tree.plan.info.columns == columns
    before = [t[:, 1].clone() for t in (pool.k, pool.v)]
    out = step.run(0, q, k, v)   # appends within its launch
    check_step(pool, 0, lists, lens, trees, q, k, v, out, dim ** -0.5, "step")
    again = step.run(0, q, k, v)
    assert torch.equal(out, again)
    assert torch.equal(pool.k[:, 1], before[0]) and torch.equal(pool.v[:, 1], before[1])


@pytest.mark.parametrize("dim,hq,hkv,tokens,columns", FORMS)
@pytest.mark.parametrize("page", PAGES)
def test_bad_page_ids_are_dropped(device, dim, hq, hkv, tokens, columns, page):
    """From C: tokens of page ids outside the pool leave the softmax, cached and drafted ones."""
    pool, lists, lens, trees, q, k, v = make(device, [tokens], [300], hq, hkv, dim, page, F16)
    table = PageTable.from_lists(lists, lens, pool)
    plan = plan_of(pool, table, trees, hq, hkv, page, device, dim, columns)
    qi = torch.tensor([0, tokens], dtype=torch.int32, device=device)
    append_kv(pool, 0, table, qi, k, v)
    gone = [0, 5, 300 // page, len(lists[0]) - 1]
    table.indices[gone] = torch.tensor([-1, pool.num_pages, -2**31, 2**31 - 1], dtype=torch.int32,
                                       device=device)
    out = tree_attention(pool, 0, table, q, plan)
    dropped = np.array([t // page in gone for t in range(lens[0])])
    keys, values = (tokens_of(t, 0, lists[0], lens[0]) for t in (pool.k, pool.v))
    ref, mass = tree_attention_ref(q, keys, values, trees[0], dim ** -0.5, dropped)
    check_out(out, ref, mass)
    table.indices[:] = -1
    assert not tree_attention(pool, 0, table, q, plan).any()


@pytest.mark.parametrize("dim,hq,hkv,tokens,columns", FORMS)
@pytest.mark.parametrize("page", PAGES)
def test_drafted_values_that_are_not_finite(device, dim, hq, hkv, tokens, columns, page):
    """NaN and infinite keys and values of a drafted token reach those that see it alone; a
    score of +infinity makes its row and head NaN, one of -infinity has no weight."""
    dtype = BF16 if dim == 128 else F16
    pool, lists, lens, trees, q, k, v = make(device, [tokens, 12], [300, 77], hq, hkv, dim, page,
                                             dtype, fan=2, seed=5)
    ratio = hq // hkv
    last = hkv - 1
    nan, low, up, inf, nan_v = (tokens - n for n in (3, 5, 7, 9, 11))
    q[:tokens] = q[:tokens].abs() + 2.0 ** -6      # so that those scores' signs are their keys'
    k[nan, 0, 1] = math.nan
    k[low, last] = -math.inf
    if hkv > 2:
        k[up, 1, 3] = math.inf
    v[inf, last, 2] = math.inf
    v[nan_v, 0, 3] = math.nan
    step = AttentionStep(pool, hq, [tokens, 12], [300, 77], [1, 1], lists, trees=trees)
    assert step.tree.plan.info.columns == columns
    out = step.run(0, q, k, v)
    sees = torch.tensor(ancestors(trees[0]), device=device)
    keys, values = (tokens_of(t, 0, lists[0], lens[0]).clone() for t in (pool.k, pool.v))
    at = 300 + low                                 # a weight of 2^-big is none
    keys[last, at] = torch.where(torch.isinf(keys[last, at]), -2.0 ** 14, keys[last, at])
    keys = torch.nan_to_num(keys, nan=0.0, posinf=0.0)
    ref, mass = tree_attention_ref(q[:tokens], keys, values, trees[0], dim ** -0.5)
    want_nan = torch.zeros_like(ref, dtype=torch.bool)
    want_nan[:, :ratio] |= sees[:, nan, None, None]
    if hkv > 2:
        want_nan[:, ratio:2 * ratio] |= sees[:, up, None, None]
    want_nan[:, :ratio, 3] |= sees[:, nan_v, None]
    assert torch.equal(torch.isnan(out[:tokens]), want_nan)
    infinite = torch.zeros_like(want_nan)
    infinite[:, last * ratio:, 2] = sees[:, inf, None]
    assert torch.equal(torch.isinf(out[:tokens]), infinite)
    fine = ~want_nan & ~infinite
    check_out(torch.where(fine, out[:tokens], 0), torch.where(fine, ref, 0), mass)
    ref, mass = row_reference(pool, 0, lists[1], lens[1], trees[1], q[tokens:], None, None, dim ** -0.5)
    check_out(out[tokens:], ref, mass)


@pytest.mark.parametrize("dim,hq,hkv,tokens,columns", FORMS)
@pytest.mark.parametrize("page", PAGES)
@pytest.mark.parametrize("split", [0, 1])
def test_cached_values_that_are_not_finite(device, dim, hq, hkv, tokens, columns, page, split):
    """An infinite cached value gives an infinite output and no NaN, a NaN key its head's rows
    NaN, a NaN query row NaN and the rows beside it nothing."""
    dtype = F16 if dim == 128 else BF16
    pool, lists, lens, trees, q, k, v = make(device, [tokens], [500], hq, hkv, dim, page, dtype, seed=9)
    ratio = hq // hkv
    pool.v[lists[0][48 // page], 0, 1, 48 % page, 7] = math.inf
    pool.k[lists[0][333 // page], 0, 0, 333 % page, 5] = math.nan
    q[4, ratio] = math.nan
    table = PageTable.from_lists(lists, lens, pool)
    plan = plan_of(pool, table, trees, hq, hkv, page, device, dim, columns, split)
    qi = torch.tensor([0, tokens], dtype=torch.int32, device=device)
    append_kv(pool, 0, table, qi, k, v)
    out = tree_attention(pool, 0, table, q, plan)
    assert torch.isnan(out[:, :ratio]).all() and torch.isnan(out[4, ratio]).all()
    inf_rows = torch.ones(tokens, ratio, dtype=torch.bool, device=device)
    inf_rows[4, 0] = False
    assert torch.equal(torch.isinf(out[:, ratio:2 * ratio, 7]), inf_rows)
    keys, values = (tokens_of(t, 0, lists[0], lens[0]) for t in (pool.k, pool.v))
    ref, mass = tree_attention_ref(torch.nan_to_num(q), torch.nan_to_num(keys), values, trees[0],
                                   dim ** -0.5)
    fine = torch.ones_like(ref, dtype=torch.bool)
    fine[:, :ratio] = False
    fine[4, ratio] = False
    fine[:, ratio:2 * ratio, 7] = False
    check_out(torch.where(fine, out, 0), torch.where(fine, ref, 0), mass)
