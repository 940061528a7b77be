"""Steps of tokens that each have a position of their own on one axis: rope_positions
[1, num_tokens], with a Rotary whose sections name one axis and with a plain one."""
import numpy as np
import pytest
import torch

from helpers import random_pool, random_tensor
from kunserve_amd import AttentionStep, PageTable, Rotary, rotary_append_kv
from tree_ref import random_pages, random_tree, tokens_of

pytestmark = pytest.mark.gpu

F16 = torch.float16
SIZES, FIRSTS, FLAGS = [12, 1, 30], [28, 9, 3], [1, 0, 1]
LENS = [40, 9, 33]


def turned(x, pos, freq):
    """x [n, heads, D] rotated at pos [n] in 64 bits, pairs (j, j + D / 2)."""
    angle = pos.double()[:, None] * freq
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    a, b = x.double().chunk(2, dim=-1)
    return torch.cat([a * c - b * s, b * c + a * s], dim=-1)


def close(got, want):
    """Half a step of the value, and the fp32 rotation's 2^-20 of |a| + |b| (below 8)."""
    return bool(((got.double() - want).abs() <= want.abs() * 2.0 ** -11 + 2.0 ** -17).all())


def make(device, seed=3):
    rng = np.random.default_rng(seed)
    lists, pages = random_pages(rng, LENS, 16)
    q, k, v = (random_tensor((sum(SIZES), h, 128), device, h, 1.0, F16) for h in (4, 2, 2))
    return rng, lists, pages, q, k, v


@pytest.mark.parametrize("sections", [None, [64]])
@pytest.mark.parametrize("pinned", [False, True])
def test_against_64_bits(device, sections, pinned):
    rng, lists, pages, q, k, v = make(device)
    rotary = Rotary(128, device=device, sections=sections)
    pos = rng.integers(0, 2**20, (1, len(q)))
    at = torch.tensor(pos[0], device=device)
    want_q, want_k = turned(q, at, rotary.frequencies), turned(k, at, rotary.frequencies)
    pool = random_pool(pages, 1, 2, 16, 128, device, 1)
    # (pinned host tensors go op by op, which a mixed step's prefill rows do not)
    rows = [0, 2] if pinned else [0, 1, 2]
    tokens = torch.cat([torch.arange(a, a + n) for b, (a, n) in enumerate(zip([0, 12, 13], SIZES))
                        if b in rows])
    step = AttentionStep(pool, 4, *([x[b] for b in rows] for x in (SIZES, FIRSTS, FLAGS, lists)),
                         rope_positions=pos[:, tokens.numpy()])
    tensors = [t.cpu()[tokens].pin_memory() if pinned else t.clone() for t in (q, k, v)]
    out = torch.empty(len(tokens), 4, 128, dtype=F16, device=device)
    step.run(0, *tensors, out=out, rope=rotary)
    torch.cuda.synchronize()
    assert close(tensors[0].to(device), want_q[tokens.to(device)])
    for b in rows:
        a = [0, 12, 13][b]
        got = tokens_of(pool.k, 0, lists[b], LENS[b])[:, LENS[b] - SIZES[b]:].transpose(0, 1)
        assert close(got, want_k[a:a + SIZES[b]])


def test_one_row_of_many_tokens_and_many_rows_of_one(device):
    """As many tokens as rows, and one row: the array still names tokens."""
    for sizes, firsts, flags in (([1, 1, 1], [30, 9, 3], [0, 0, 0]), ([5], [20], [1])):
        lens = [f + n if p else f for n, f, p in zip(sizes, firsts, flags)]
        lists, pages = random_pages(np.random.default_rng(1), lens, 16)
        q, k, v = (random_tensor((sum(sizes), h, 128), device, h, 1.0, F16) for h in (4, 2, 2))
        pos = np.arange(sum(sizes))[None] * 977 + 5
        rotary = Rotary(128, device=device)
        pool = random_pool(pages, 1, 2, 16, 128, device, 1)
        qq = q.clone()
        AttentionStep(pool, 4, sizes, firsts, flags, lists, rope_positions=pos).run(0, qq, k, v, rope=rotary)
        assert close(qq, turned(q, torch.tensor(pos[0], device=device), rotary.frequencies))


def test_as_the_prologue_alone(device):
    """A step's rotation is rotary_append_kv's, bit for bit, and a tree's own places give way."""
    rng = np.random.default_rng(5)
    tree = random_tree(rng, 20, 3)
    lists, pages = random_pages(rng, [90], 16)
    q, k, v = (random_tensor((20, h, 128), device, h, 1.0, F16) for h in (4, 2, 2))
    pos = rng.integers(0, 5000, (1, 20))
    dev = torch.tensor(pos, dtype=torch.int32, device=device)
    for sections in (None, [64]):
        rotary = Rotary(128, device=device, sections=sections)
        pools = [random_pool(pages, 1, 2, 16, 128, device, 1) for _ in range(2)]
        qs = [q.clone(), q.clone()]
        AttentionStep(pools[0], 4, [20], [70], [1], lists, trees=[tree],
                      rope_positions=pos).run(0, qs[0], k, v, rope=rotary)
        table = PageTable.from_lists(lists, [90], pools[1])
        rotary_append_kv(pools[1], 0, table, torch.tensor([0, 20], dtype=torch.int32, device=device),
                         qs[1], k, v, rotary, positions=dev)
        assert torch.equal(qs[0], qs[1]) and torch.equal(pools[0].k, pools[1].k)


def test_refusals(device):
    rng, lists, pages, q, k, v = make(device)
    pool = random_pool(pages, 1, 2, 16, 128, device, 1)
    new = lambda pos: AttentionStep(pool, 4, SIZES, FIRSTS, FLAGS, lists, rope_positions=pos)   # noqa: E731
    pos = rng.integers(0, 500, (1, len(q)))
    for bad, why in ((pos[:, 1:], "rope_positions"), (pos[:0], "rope_positions"), (pos.astype(float), "whole"),
                     (pos - 1000, "lie in"), (pos + 2**31, "lie in")):
        with pytest.raises(ValueError, match=why):
            new(bad)
    for nested in (pos.tolist(), (pos[0],), [[7, 100, 3]]):   # one list in a list: no array of an axis
        with pytest.raises(ValueError, match="3 rows but"):
            new(nested)
    step = new(pos)
    with pytest.raises(ValueError, match="positions on 1 axes"):
        step.run(0, q.clone(), k, v, rope=Rotary(128, device=device, sections=[16, 24, 24]))
    with pytest.raises(ValueError, match="Rotary"):
        step.run(0, q.clone(), k, v, rope=(torch.ones(64, device=device), False))


def test_captured(device):
    """Each replay against the eager result and the formula."""
    rng, lists, pages, q, k, v = make(device)
    pool = random_pool(pages, 1, 2, 16, 128, device, 1)
    rotary = Rotary(128, device=device, sections=[64])
    pos = rng.integers(0, 500, (1, len(q)))
    step = AttentionStep(pool, 4, SIZES, FIRSTS, FLAGS, lists, rope_positions=pos)
    first = q.clone()
    want = step.run(0, first, k, v, rope=rotary).clone()
    qq, out = q.clone(), torch.empty_like(q)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step.run(0, qq, k, v, out=out, rope=rotary)
    for _ in range(3):
        qq.copy_(q)
        out.fill_(1.0)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(qq, first)
    assert close(qq, turned(q, torch.tensor(pos[0], device=device), rotary.frequencies))
