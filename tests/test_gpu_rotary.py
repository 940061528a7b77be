"""rotary_append_kv and steps with a Rotary against the rotation in 64 bits."""
import numpy as np
import pytest
import torch

import operators_ref as ref
from helpers import random_pool, random_tensor
from kunserve_amd import AttentionStep, KVPool, PageTable, Rotary, append_kv, rotary_append_kv

pytestmark = pytest.mark.gpu

# sine and cosine of an angle in turns that fp32 rounds (2^-25 of a turn at
# most half a turn away: 2^-24 pi rad), their own rounding (2 ulp) and that of
# the scale, two products and a sum: 16 roundings cover them.
TRIG = 16 * ref.W


def tolerance(want, mag, dtype):
    sub = 2.0 ** -25 if dtype == torch.float16 else 0.0
    return ref.half_step(dtype) * np.abs(want) + TRIG * mag * (1 + ref.half_step(dtype)) + sub


def setup(device, q_lens, pre, hq, hkv, ps, d, dtype, seed=0):
    q_lens = np.asarray(q_lens)
    kv = q_lens + np.asarray(pre)
    need = -(-kv // ps)
    pages = int(need.sum()) + 3
    perm = np.random.default_rng(seed).permutation(pages)
    tables, at = [], 0
    for n in need:
        tables.append(perm[at:at + n].tolist())
        at += n
    pool = random_pool(pages, 2, hkv, ps, d, device, seed, dtype=dtype)
    t = int(q_lens.sum())
    q = random_tensor((t, hq, d), device, seed + 1, dtype=dtype)
    k = random_tensor((t, hkv, d), device, seed + 2, dtype=dtype)
    v = random_tensor((t, hkv, d), device, seed + 3, dtype=dtype)
    indptr = torch.tensor(np.r_[0, np.cumsum(q_lens)], dtype=torch.int32, device=device)
    slots = [(tables[b][c // ps], c % ps) for b in range(len(q_lens))
             for c in range(int(kv[b] - q_lens[b]), int(kv[b]))]
    return pool, tables, kv, q, k, v, indptr, slots


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d,r", [(64, 64), (64, 16), (128, 128), (128, 64), (128, 32), (256, 256),
                                 (256, 48)])
@pytest.mark.parametrize("interleave", [False, True])
def test_rotates_part_of_the_head_at_its_positions(device, dtype, d, r, interleave):
    q_lens, pre = [1, 1, 5, 1, 33], [0, 40, 11, 300, 64]
    pool, tables, kv, q, k, v, indptr, slots = setup(device, q_lens, pre, 6, 2, 16, d, dtype, d + r)
    rot = Rotary(r, 10000.0, interleave, dict(rope_type="yarn", factor=8.0,
                                              original_max_position_embeddings=512), device)
    pos = np.random.default_rng(1).integers(0, 2**20, size=q.shape[0])
    pos[:3] = [0, 1, 2**31 - 1]
    positions = torch.tensor(pos, dtype=torch.int32, device=device)
    before = [pool.k.clone(), pool.v.clone()]
    table = PageTable.from_lists(tables, kv, pool)
    out = torch.full_like(q, 7.0)
    got = rotary_append_kv(pool, 1, table, indptr, q.clone(), k, v, rot, positions, out)
    torch.cuda.synchronize()
    assert got is out
    f = rot.frequencies.cpu().numpy()
    want, mag = ref.rotate(q.cpu().double().numpy(), pos, f, rot.scale, interleave)
    assert np.all(np.abs(out.cpu().double().numpy() - want) <= tolerance(want, mag, dtype))
    # what is not rotated passes bit for bit, in place and apart
    assert torch.equal(out[..., r:].view(torch.int16), q[..., r:].view(torch.int16))
    in_place = q.clone()
    rotary_append_kv(pool, 1, table, indptr, in_place, k, v, rot, positions)
    assert torch.equal(in_place.view(torch.int16), out.view(torch.int16))
    wk, mk = ref.rotate(k.cpu().double().numpy(), pos, f, rot.scale, interleave)
    page, slot = (torch.tensor(x, device=device) for x in zip(*slots))
    gk = pool.k[page, 1, :, slot].cpu().double().numpy()
    assert np.all(np.abs(gk - wk) <= tolerance(wk, mk, dtype))
    assert torch.equal(pool.v[page, 1, :, slot].view(torch.int16), v.view(torch.int16))
    # no other element of the pool changed
    for now, old, new in ((pool.k, before[0], gk), (pool.v, before[1], None)):
        old[page, 1, :, slot] = now[page, 1, :, slot]
        assert torch.equal(now.view(torch.int16), old.view(torch.int16))


def test_without_positions_tokens_rotate_at_their_places(device):
    pool, tables, kv, q, k, v, indptr, _ = setup(device, [3, 1, 20], [5, 77, 0], 4, 4, 16, 128,
                                                 torch.bfloat16)
    rot = Rotary(128, 500000.0, device=device)
    table = PageTable.from_lists(tables, kv, pool)
    own = np.concatenate([np.arange(n - t, n) for t, n in zip([3, 1, 20], kv)])
    a, b = torch.empty_like(q), torch.empty_like(q)
    rotary_append_kv(pool, 0, table, indptr, q, k, v, rot, out=a)
    rotary_append_kv(pool, 0, table, indptr, q, k, v, rot, out=b,
                     positions=torch.tensor(own, dtype=torch.int32, device=device))
    assert torch.equal(a.view(torch.int16), b.view(torch.int16))


def test_strided_tensors_and_tokens_of_no_row(device):
    """q, k and v as slices of one projection, and more tokens than the rows
    own: those behind the last row are left as they were."""
    pool, tables, kv, _, _, _, indptr, slots = setup(device, [1, 4], [30, 2], 4, 2, 16, 64,
                                                     torch.float16)
    qkv = random_tensor((8, 8 * 64), device, 5)
    q, k, v = (x.unflatten(1, (-1, 64)) for x in qkv.split([256, 128, 128], dim=1))
    rot = Rotary(32, device=device, interleave=True)
    table = PageTable.from_lists(tables, kv, pool)
    want, mag = ref.rotate(q[:5].cpu().double().numpy(), [30, 2, 3, 4, 5],
                           rot.frequencies.cpu().numpy(), 1.0, True)
    rest = qkv.clone()
    rotary_append_kv(pool, 0, table, indptr, q, k, v, rot)
    torch.cuda.synchronize()
    assert np.all(np.abs(q[:5].cpu().double().numpy() - want) <= tolerance(want, mag, torch.float16))
    rest[:5, :256] = qkv[:5, :256]
    assert torch.equal(rest.view(torch.int16), qkv.view(torch.int16))
    page, slot = (torch.tensor(x, device=device) for x in zip(*slots))
    assert torch.equal(pool.v[page, 0, :, slot].view(torch.int16), v[:5].view(torch.int16))


def test_a_step_rotates_its_rows_where_they_are(device):
    """AttentionStep.run(rope=Rotary) with rope_positions: the prologue's q and
    cache, then attention on them, as the pieces give."""
    q_lens, pre = [1, 7, 1], [99, 20, 5]
    pool, tables, kv, q, k, v, indptr, _ = setup(device, q_lens, pre, 8, 2, 16, 128,
                                                 torch.bfloat16)
    rot = Rotary(64, device=device, scaling=dict(rope_type="linear", factor=2.0))
    starts = [100000, 20, 777]
    twin = KVPool(pool.k.clone(), pool.v.clone())
    first = [100, 20, 6]
    step = AttentionStep(pool, 8, q_lens, first, [0, 1, 0], tables, rope_positions=starts)
    q1 = q.clone()
    out = step.run(1, q1, k, v, rope=rot)
    pos = np.concatenate([s + np.arange(t) for s, t in zip(starts, q_lens)])
    table = PageTable.from_lists(tables, kv, twin)
    q2 = torch.empty_like(q)
    rotary_append_kv(twin, 1, table, indptr, q, k, v, rot, out=q2,
                     positions=torch.tensor(pos, dtype=torch.int32, device=device))
    assert torch.equal(q1.view(torch.int16), q2.view(torch.int16))
    assert torch.equal(pool.k.view(torch.int16), twin.k.view(torch.int16))
    assert torch.equal(pool.v.view(torch.int16), twin.v.view(torch.int16))
    turned = twin.k[:, 1].clone()
    plain = AttentionStep(twin, 8, q_lens, first, [0, 1, 0], tables)
    page = torch.tensor([tables[b][c // 16] for b in range(3)
                         for c in range(kv[b] - q_lens[b], kv[b])], device=device)
    slot = torch.tensor([c % 16 for b in range(3) for c in range(kv[b] - q_lens[b], kv[b])],
                        device=device)
    want = plain.run(1, q2, turned[page, :, slot].contiguous(), v)
    assert torch.equal(out.view(torch.int16), want.view(torch.int16))
    with pytest.raises(ValueError, match="need a Rotary"):
        step.run(1, q1, k, v, rope=(torch.ones(64, device=device), False))


def test_refusals(device):
    pool, tables, kv, q, k, v, indptr, _ = setup(device, [1, 2], [3, 4], 4, 2, 16, 64,
                                                 torch.float16)
    table = PageTable.from_lists(tables, kv, pool)
    with pytest.raises(ValueError, match="exceeds head_dim"):
        rotary_append_kv(pool, 0, table, indptr, q, k, v, Rotary(128, device=device))
    rot = Rotary(64, device=device)
    with pytest.raises(ValueError, match="positions"):
        rotary_append_kv(pool, 0, table, indptr, q, k, v, rot,
                         torch.zeros(3, dtype=torch.int64, device=device))
    with pytest.raises(RuntimeError, match="overlaps q"):
        both = torch.zeros((4, 4, 64), dtype=torch.float16, device=device)
        rotary_append_kv(pool, 0, table, indptr, both[:3], k, v, rot, out=both[1:])
    with pytest.raises(RuntimeError, match="overlaps k_new"):
        kv4 = torch.zeros((3, 4, 64), dtype=torch.float16, device=device)
        rotary_append_kv(pool, 0, table, indptr, q, kv4[:, :2], v, rot, out=kv4)
    with pytest.raises(RuntimeError, match="share memory"):
        rotary_append_kv(pool, 0, table, indptr, q, k, v, rot,
                         out=torch.zeros((1, 4, 64), dtype=torch.float16,
                                         device=device).expand(3, 4, 64))
    with pytest.raises(ValueError, match="does not match the pool"):
        rotary_append_kv(pool, 0, table, indptr, q.bfloat16(), k, v, rot)
    with pytest.raises(ValueError, match="on cpu"):
        rotary_append_kv(pool, 0, table, indptr, q.cpu(), k, v, rot)
    with pytest.raises(ValueError, match="frequencies are on"):
        rotary_append_kv(pool, 0, table, indptr, q, k, v, Rotary(64, device="cpu"))
    with pytest.raises(RuntimeError, match="layer"):
        rotary_append_kv(pool, 2, table, indptr, q, k, v, rot)
