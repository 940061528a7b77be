"""Plans of drafted trees and the host checks around them (CPU only)."""
import ctypes

import numpy as np
import pytest
import torch

from kunserve_amd import PageTable, TreePlan, _lib, tree_depths
from tree_ref import ancestors, random_pages, random_tree

CPU = torch.device("cpu")
ROUND = {64: 256, 128: 128, 256: 64}
REC = 16


def make(lens, trees, hq=8, hkv=2, dim=128, page=16, cus=256, part_rounds=0, q_first=None, seed=0):
    rng = np.random.default_rng(seed)
    lists, _ = random_pages(rng, lens, page)
    indptr = np.cumsum([0] + [len(x) for x in lists])
    table = PageTable(indptr, np.concatenate([np.array(x, np.int32) for x in lists] or [[]]), lens,
                      CPU, upload=False)
    return TreePlan(table, trees, hq, hkv, page, CPU, num_cus=cus, upload=False, head_dim=dim,
                    q_first=q_first, part_rounds=part_rounds)


def parts(plan):
    i = plan.info
    at = REC * i.num_work
    return (plan.plan_host[:at].reshape(-1, REC),
            plan.plan_host[at:at + 4 * i.num_merge].reshape(-1, 4),
            plan.plan_host[at + 4 * i.num_merge:].view(np.uint32))


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("part_rounds", [0, 1, 3, 1000])
@pytest.mark.parametrize("ratio,hkv", [(1, 2), (3, 2), (4, 1), (71, 1)])
def test_records_cover_every_column_and_round_once(dim, part_rounds, ratio, hkv):
    rng = np.random.default_rng(dim + part_rounds + ratio)
    sizes = [1, 7, 33, 0, 70, 64]
    lens = np.array([n + p for n, p in zip(sizes, [0, 1, 1400, 300, 777, ROUND[dim]])])
    plan = make(lens, [random_tree(rng, n, 5) for n in sizes], ratio * hkv, hkv, dim,
                part_rounds=part_rounds)
    rec, merges, _ = parts(plan)
    first = np.cumsum([0] + sizes)
    seen = {}
    for r in rec[rec[:, 0] > 0]:
        tokens, q0, prefix, _, c0, cols, head, np_, rb, re, slot, n, part = r[:13]
        b = int(np.searchsorted(first, q0, side="right") - 1)
        while sizes[b] == 0:
            b -= 1
        b = [i for i in range(len(sizes)) if first[i] == q0 and sizes[i] == tokens][0]
        assert prefix == lens[b] - sizes[b] and np_ == -(-prefix // ROUND[dim])
        assert 0 <= rb < re <= np_ + -(-tokens // ROUND[dim])
        assert 0 < cols <= plan.info.columns <= (256 if dim == 128 else 128) and c0 + cols <= tokens * ratio
        assert (slot < 0) == (n == 1) and 0 <= part < n
        for c in range(c0, c0 + cols):
            for i in range(rb, re):
                key = (b, int(head), c, i)
                assert key not in seen
                seen[key] = (int(slot), int(n), int(part))
    want = sum(n * ratio * hkv * (-(-(int(l) - n) // ROUND[dim]) + -(-n // ROUND[dim]))
               for n, l in zip(sizes, lens))
    assert len(seen) == want
    # every token of a split row has slots of its own, merged in order
    used = set()
    for token, s0, n, _ in merges:
        assert n > 1 and not used & set(range(s0, s0 + n))
        used |= set(range(s0, s0 + n))
        b = [i for i in range(len(sizes)) if first[i] <= token < first[i + 1]][0]
        assert {v[0] + (token - first[b]) * v[1] for k, v in seen.items() if k[0] == b} == {s0}
    assert used == set(range(plan.info.num_slots))


@pytest.mark.parametrize("lens,tokens,hkv,dim,split,workgroups", [
    ([1508], 8, 8, 128, True, 104),             # one row: a round to a workgroup
    ([4104] * 64, 8, 8, 128, False, 512),       # two whole rows and heads to a CU
    ([4104] * 16, 8, 8, 128, True, 512),        # a quarter of a row
    ([1000] * 21, 16, 32, 64, False, 672),      # whole rows end before halves would
    ([4160] * 4, 64, 4, 256, True, 256),        # one workgroup to a CU
], ids=["one", "filled", "quarters", "nearly", "dim256"])
def test_runs_fill_the_device(lens, tokens, hkv, dim, split, workgroups):
    trees = [list(range(-1, tokens - 1))] * len(lens)
    plan = make(np.array(lens), trees, hkv * (1 if dim == 64 else 4), hkv, dim, cus=256)
    rec, _, _ = parts(plan)
    rec = rec[rec[:, 0] > 0]
    assert (plan.info.num_slots > 0) == split
    assert abs(len(rec) - workgroups) <= workgroups // 8, len(rec)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_masks_are_the_ancestors(dim):
    """The bit of drafted token u is where the score tiles' lanes look for it: element x of
    lane half h of a tile is element x % 8 of lane group 2 (x / 8) + h."""
    rng = np.random.default_rng(dim)
    tpl, step = 64 // (dim // 8), 8 * (64 // (dim // 8))
    for n, fan, roots in [(1, 1, 1), (40, 3, 1), (300, 300, 4), (70, 1, 1)]:
        tree = random_tree(rng, n, fan, roots)
        plan = make([n + 5], [tree], dim=dim)
        _, _, masks = parts(plan)
        words = -(-n // ROUND[dim]) * ROUND[dim] // 32
        masks = masks.reshape(n, words)
        got = np.zeros((n, n), dtype=bool)
        for u in range(n):
            r, v = divmod(u, ROUND[dim])
            wave, e, row = v // step, v % step // tpl, v % tpl
            group = {64: row & 3, 128: row, 256: 2 * (wave & 1) + row}[dim]
            tile = {64: 2 * wave + (row >> 2), 128: wave, 256: wave >> 1}[dim]
            word = masks[:, r * (ROUND[dim] // 32) + tile]
            got[:, u] = word >> np.uint32(16 * (group & 1) + 8 * (group >> 1) + e) & 1
        assert np.array_equal(got, ancestors(tree))
        assert sum(bin(int(w)).count("1") for w in masks.ravel()) == ancestors(tree).sum()


def test_depths():
    rng = np.random.default_rng(3)
    for n, fan, roots in [(1, 1, 1), (50, 4, 2), (200, 1, 1), (128, 200, 1)]:
        tree = random_tree(rng, n, fan, roots)
        assert np.array_equal(tree_depths(tree), ancestors(tree).sum(1) - 1)
    assert tree_depths([]).size == 0


@pytest.mark.parametrize("tree,why", [([0], "parent 0"), ([-1, 2, 0], "parent 2"), ([-2], "parent -2"),
                                      ([-1, 1], "parent 1"), ([0.0], "whole numbers"),
                                      ([[-1]], "whole numbers")])
def test_trees_that_are_none(tree, why):
    with pytest.raises(ValueError, match=why):
        make([10], [tree])
    with pytest.raises(ValueError, match=why):
        tree_depths(tree)


def test_plan_refusals():
    with pytest.raises(ValueError, match="2 trees"):
        make([10], [[-1], [-1]])
    with pytest.raises(_lib.KunserveError, match="new tokens of"):
        make([1], [[-1, 0]])
    with pytest.raises(ValueError, match="first tokens"):
        make([10], [[-1]], q_first=[-1])
    with pytest.raises(_lib.KunserveError, match="multiple"):
        make([10], [[-1]], hq=3, hkv=2)
    with pytest.raises(_lib.KunserveError, match="power of two"):
        make([12], [[-1]], page=12)
    with pytest.raises(_lib.KunserveError, match="negative"):
        make([10], [[-1]], part_rounds=-1)
    assert make([], []).info.plan_ints == 0
    assert _lib.lib().kunserve_tree_plan_bound(None, None, 1, 8, 2, 128) == -1
    assert _lib.lib().kunserve_tree_plan_bound(None, None, 0, 8, 2, 96) == -1


def test_plan_buffer_too_small():
    q, kv, ip = (np.array(x, np.int32) for x in ([0, 2], [9], [0, 1]))
    up = np.array([-1, 0], np.int32)
    buf, info = np.zeros(4, np.int32), _lib.TreePlanInfo()
    with pytest.raises(_lib.KunserveError) as e:
        _lib.call("kunserve_tree_plan", ip.ctypes.data, q.ctypes.data, None, kv.ctypes.data,
                  up.ctypes.data, 1, 8, 2, 16, 128, 256, 0, buf.ctypes.data, 4, ctypes.byref(info))
    assert e.value.code == _lib.ENOSPC


def test_bound_holds():
    rng = np.random.default_rng(7)
    for _ in range(60):
        dim = int(rng.choice([64, 128, 256]))
        hkv = int(rng.choice([1, 2, 8]))
        hq = hkv * int(rng.integers(1, 9))
        sizes = rng.integers(0, 150, int(rng.integers(1, 9)))
        lens = sizes + rng.integers(0, 3000, sizes.size)
        plan = make(lens, [random_tree(rng, int(n), 9) for n in sizes], hq, hkv, dim,
                    part_rounds=int(rng.integers(0, 3)), cus=int(rng.choice([1, 256])))
        qi = np.cumsum([0, *sizes]).astype(np.int32)
        kv = lens.astype(np.int32)
        assert plan.info.plan_ints <= _lib.lib().kunserve_tree_plan_bound(
            qi.ctypes.data, kv.ctypes.data, len(kv), hq, hkv, dim)


def test_info_is_that_of_the_header():
    assert ctypes.sizeof(_lib.TreePlanInfo) == 40 and ctypes.sizeof(_lib.RotaryAxes) == 24
