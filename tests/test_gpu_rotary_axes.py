"""Rotary positions on several axes against the formula in 64 bits."""
import numpy as np
import pytest
import torch

from helpers import random_pool, random_tensor
from kunserve_amd import AttentionStep, PageTable, Rotary, rotary_append_kv
from tree_ref import random_pages, tokens_of

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def turned(x, pos, axis, freq, rotary_dim, interleave, scale=1.0):
    """x [n, heads, D], pos [axes, n]: rotated in 64 bits."""
    angle = pos.double()[axis].t() * freq           # [n, pairs]
    c, s = (angle.cos() * scale)[:, None], (angle.sin() * scale)[:, None]
    y = x.double().clone()
    a, b = ((slice(0, rotary_dim, 2), slice(1, rotary_dim, 2)) if interleave else
            (slice(0, rotary_dim // 2), slice(rotary_dim // 2, rotary_dim)))
    u, w = y[..., a].clone(), y[..., b].clone()
    y[..., a] = u * c - w * s
    y[..., b] = w * c + u * s
    return y


def close(got, want, x, scale=1.0):
    """Half a step of the value; the fp32 rotation's sines, products and sum and the angle's
    2^-24 of half a turn: below 2^-20 of |a| + |b|, which are below 8 here."""
    err = (got.double() - want).abs()
    return bool((err <= want.abs() * torch.finfo(got.dtype).eps / 2 + 8 * 2.0 ** -20 * scale).all())


@pytest.mark.parametrize("dim,rotary_dim,interleave,dtype,kw", [
    (128, 128, False, BF16, dict(sections=[16, 24, 24])),
    (128, 128, True, F16, dict(sections=[1, 0, 63])),
    (128, 64, False, F16, dict(axes=[i % 3 for i in range(32)])),
    (64, 64, False, F16, dict(sections=[32])),
    (64, 16, True, BF16, dict(axes=[7] * 8)),
    (256, 256, False, BF16, dict(sections=[32, 32, 32, 32])),
])
@pytest.mark.parametrize("separate", [False, True])
def test_against_64_bits(device, dim, rotary_dim, interleave, dtype, kw, separate):
    hq, hkv = 6, 2
    rng = np.random.default_rng(dim + rotary_dim)
    ql, lens = [1, 5, 40], [1, 77, 40]
    lists, pages = random_pages(rng, lens, 16)
    pool = random_pool(pages, 2, hkv, 16, dim, device, 1, dtype=dtype)
    n = sum(ql)
    q, k, v = (random_tensor((n, h, dim), device, 5 + i, 1.0, dtype) for i, h in enumerate((hq, hkv, hkv)))
    scale = 1.25
    rotary = Rotary(rotary_dim, 1e6, interleave=interleave, device=device, scale=scale, **kw)
    pos = torch.tensor(rng.integers(0, 2**20, (rotary.num_axes, n)), dtype=torch.int32, device=device)
    pos[:, 0] = 0
    pos[-1, 1] = 2**31 - 1
    table = PageTable.from_lists(lists, lens, pool)
    qi = torch.tensor(np.cumsum([0, *ql]), dtype=torch.int32, device=device)
    axis = rotary.pair_axis.long()
    want_q = turned(q, pos, axis, rotary.frequencies, rotary_dim, interleave, scale)
    want_k = turned(k, pos, axis, rotary.frequencies, rotary_dim, interleave, scale)
    old = pool.k[:, 0].clone()
    src = q.clone()
    out = torch.empty_like(q) if separate else None
    got = rotary_append_kv(pool, 1, table, qi, src, k, v, rotary, positions=pos, out=out)
    assert close(got, want_q, q) and (not separate or torch.equal(src, q))
    at = 0
    for b, m in enumerate(ql):
        new = slice(at, at + m)
        at += m
        assert close(tokens_of(pool.k, 1, lists[b], lens[b])[:, lens[b] - m:].transpose(0, 1), want_k[new], k)
        assert torch.equal(tokens_of(pool.v, 1, lists[b], lens[b])[:, lens[b] - m:], v[new].transpose(0, 1))
    assert torch.equal(pool.k[:, 0], old)


def test_one_position_is_every_axis_s(device):
    """Text: positions [tokens], or none, are those of a rotary of one axis, bit for bit."""
    rng = np.random.default_rng(3)
    lists, pages = random_pages(rng, [50, 9], 16)
    q, k, v = (random_tensor((30, h, 128), device, h, 1.0, BF16) for h in (4, 2, 2))
    qi = torch.tensor([0, 21, 30], dtype=torch.int32, device=device)
    pos = torch.arange(1000, 1030, dtype=torch.int32, device=device)
    for positions in (None, pos, pos[None].expand(3, -1).contiguous()):
        got = []
        for kw in (dict(), dict(sections=[16, 24, 24])):
            pool = random_pool(pages, 1, 2, 16, 128, device, 1, dtype=BF16)
            table = PageTable.from_lists(lists, [50, 9], pool)
            p = pos if not kw and positions is not None else positions
            got.append((rotary_append_kv(pool, 0, table, qi, q.clone(), k, v,
                                         Rotary(128, device=device, **kw), positions=p), pool.k))
        assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])


def test_steps(device):
    """A step's rope_positions on axes; text rows' single starts; refusals."""
    rng = np.random.default_rng(3)
    lens = [40, 9, 33]
    lists, pages = random_pages(rng, lens, 16)
    rotary = Rotary(128, device=device, sections=[16, 24, 24])
    plain = Rotary(128, device=device)
    ql, first, flags = [12, 1, 30], [28, 9, 3], [1, 0, 1]
    n = sum(ql)
    q, k, v = (random_tensor((n, h, 128), device, h, 1.0, F16) for h in (4, 2, 2))
    pos = rng.integers(0, 500, (3, n))
    pool = random_pool(pages, 1, 2, 16, 128, device, 1)
    step = AttentionStep(pool, 4, ql, first, flags, lists, rope_positions=pos)
    qq = q.clone()
    step.run(0, qq, k, v, rope=rotary)
    want = turned(q, torch.tensor(pos, device=device), rotary.pair_axis.long(), rotary.frequencies, 128, False)
    assert close(qq, want, q)
    at = 0
    wk = turned(k, torch.tensor(pos, device=device), rotary.pair_axis.long(), rotary.frequencies, 128, False)
    for b, m in enumerate(ql):
        assert close(tokens_of(pool.k, 0, lists[b], lens[b])[:, lens[b] - m:].transpose(0, 1), wk[at:at + m], k)
        at += m
    with pytest.raises(ValueError, match="positions on 3 axes"):
        step.run(0, q.clone(), k, v, rope=plain)
    with pytest.raises(ValueError, match="Rotary"):
        step.run(0, q.clone(), k, v, rope=(plain.frequencies.float(), False))
    # pinned host tensors go op by op, to the same bits (not in a mixed step)
    rows = torch.cat([torch.arange(12), torch.arange(13, 43)])
    other = random_pool(pages, 1, 2, 16, 128, device, 1)
    host = [t.cpu()[rows].pin_memory() for t in (q, k, v)]
    part = AttentionStep(other, 4, [12, 30], [28, 3], [1, 1], [lists[0], lists[2]],
                         rope_positions=pos[:, rows.numpy()])
    part.run(0, *host, out=torch.empty(42, 4, 128, dtype=F16, device=device), rope=rotary)
    torch.cuda.synchronize()
    assert torch.equal(host[0], qq.cpu()[rows])
    for b in (0, 2):
        assert torch.equal(tokens_of(other.k, 0, lists[b], lens[b]), tokens_of(pool.k, 0, lists[b], lens[b]))
    # starts, and no positions at all
    for starts in ([7, 100, 3], None):
        got = []
        for r in (rotary, plain):
            p = random_pool(pages, 1, 2, 16, 128, device, 1)
            s = AttentionStep(p, 4, ql, first, flags, lists, rope_positions=starts)
            got.append((s.run(0, q.clone(), k, v, rope=r), p.k))
        assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    for bad, why in ((pos[:, 1:], "rope_positions"), (pos.astype(float), "whole numbers"),
                     (pos - 1000, "lie in"), (pos + 2**31, "lie in"), (pos[:0], "rope_positions")):
        with pytest.raises(ValueError, match=why):
            AttentionStep(pool, 4, ql, first, flags, lists, rope_positions=bad)


def test_refusals(device):
    pool = random_pool(4, 1, 2, 16, 128, device, 1)
    table = PageTable.from_lists([[0]], [10], pool)
    qi = torch.tensor([0, 10], dtype=torch.int32, device=device)
    q, k = (torch.zeros(10, h, 128, dtype=F16, device=device) for h in (4, 2))
    r = Rotary(128, device=device, sections=[32, 32])
    for bad, why in ((torch.zeros(3, 10), "3 axes"), (torch.zeros(2, 9), "positions"),
                     (torch.zeros(2, 10), "int32"), (torch.zeros(10, 2, dtype=torch.int32).t(), "contiguous")):
        bad = bad.to(device) if bad.dtype == torch.int32 or "int32" in why else bad.int().to(device)
        with pytest.raises(ValueError, match=why):
            rotary_append_kv(pool, 0, table, qi, q, k, k, r, positions=bad)


def test_captured(device):
    rng = np.random.default_rng(3)
    lists, pages = random_pages(rng, [40], 16)
    pool = random_pool(pages, 1, 2, 16, 128, device, 1)
    r = Rotary(128, device=device, sections=[16, 24, 24])
    q, k, v = (random_tensor((30, h, 128), device, h, 1.0, F16) for h in (4, 2, 2))
    pos = rng.integers(0, 500, (3, 30))
    step = AttentionStep(pool, 4, [30], [10], [1], lists, rope_positions=pos)
    want = step.run(0, q.clone(), k, v, rope=r).clone()
    qq, out = q.clone(), torch.empty_like(q)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step.run(0, qq, k, v, out=out, rope=r)
    for _ in range(3):
        qq.copy_(q)
        out.fill_(1.0)
        pool.k[:, :, :, 10:] = 0
        g.replay()
        torch.cuda.synchronize()
        # (slots that the row does not append to were zeroed: prefix tokens 10..15)
        again = AttentionStep(pool, 4, [30], [10], [1], lists, rope_positions=pos).run(0, q.clone(), k, v, rope=r)
        assert torch.equal(out, again)
    assert want.shape == out.shape
