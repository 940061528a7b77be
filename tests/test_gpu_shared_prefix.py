"""Decode rows that share pages (AttentionStep(share_prefixes=True),
shared_decode) against attention in 64 bits."""
import math

import numpy as np
import pytest
import torch

import operators_ref as ref
from helpers import random_pool, random_tensor
from kunserve_amd import AttentionStep, PageTable, SharedDecodePlan, paged_kv, shared_decode

pytestmark = pytest.mark.gpu


def tree(rng, ps, specs):
    """Page lists of rows from (path, tokens): the path names the shared pieces
    [(name, pages)], then private pages up to the row's tokens."""
    made, tables, at = {}, [], 0
    for path, n in specs:
        t = []
        for name, pages in path:
            if name not in made:
                made[name] = list(range(at, at + pages))
                at += pages
            t += made[name]
        more = -(-n // ps) - len(t)
        assert more >= 0
        t += range(at, at + more)
        at += more
        tables.append(t)
    perm = rng.permutation(at + 2)
    return [[int(perm[p]) for p in t] for t in tables], at + 2


def run(device, specs, hq, hkv, ps, d, dtype, seed=0, layers=2, layer=1, poke=None, **kw):
    rng = np.random.default_rng(seed)
    tables, pages = tree(rng, ps, specs)
    kvs = [n for _, n in specs]
    pool = random_pool(pages, layers, hkv, ps, d, device, seed, dtype=dtype)
    n = len(kvs)
    q = random_tensor((n, hq, d), device, seed + 1, 2.0, dtype)
    k = random_tensor((n, hkv, d), device, seed + 2, dtype=dtype)
    v = random_tensor((n, hkv, d), device, seed + 3, dtype=dtype)
    if poke:
        poke(pool, tables)
    before = [pool.k.clone(), pool.v.clone()]
    step = AttentionStep(pool, hq, [1] * n, kvs, [0] * n, tables, share_prefixes=True,
                         share_min_bytes=0, **kw)
    out = step.run(layer, q, k, v)
    torch.cuda.synchronize()
    # the new tokens are appended, nothing else changes
    page = torch.tensor([t[(m - 1) // ps] for t, m in zip(tables, kvs)], device=device)
    slot = torch.tensor([(m - 1) % ps for m in kvs], device=device)
    for now, old, new in zip((pool.k, pool.v), before, (k, v)):
        old[page, layer, :, slot] = new
        assert torch.equal(now.view(torch.int16), old.view(torch.int16))
    return step, pool, tables, kvs, q, out


def check(pool, tables, kvs, q, out, layer=1, step=None, plan=None):
    """A workgroup of many columns rounds its probabilities once to the element type
    for the matrix units, u of each, so of sum p |v| (others: in two terms, u^2)."""
    plan = step.decode.plan if step is not None else plan
    wide = isinstance(plan, SharedDecodePlan) and plan.shared_info.wide
    p_err = ref.half_step(pool.dtype) if wide else None
    kh, vh = pool.k.cpu(), pool.v.cpu()
    got, qh = out.cpu().double().numpy(), q.cpu().double().numpy()
    for b in range(len(kvs)):
        k, v = (ref.row_cache(x, layer, tables[b], kvs[b]) for x in (kh, vh))
        want, tol, _, _ = ref.attend(qh[b:b + 1], k, v, 1 / math.sqrt(pool.head_dim), pool.dtype,
                                   p_err)
        assert np.all(np.abs(got[b] - want[0]) <= tol[0]), (
            b, float(np.max(np.abs(got[b] - want[0]) - tol[0])))


@pytest.mark.parametrize("hq,hkv", [(4, 4), (8, 4), (6, 2), (8, 2), (10, 2), (16, 2), (16, 1),
                                    (34, 2)])
@pytest.mark.parametrize("d,dtype", [(64, torch.float16), (128, torch.bfloat16),
                                     (128, torch.float16), (256, torch.bfloat16)])
def test_one_prefix(device, hq, hkv, d, dtype):
    root = [("r", 9)]
    specs = [(root, 144 + m) for m in (1, 2, 15, 16, 17, 100, 300)]
    step, *rest = run(device, specs, hq, hkv, 16, d, dtype, seed=hq + d)
    assert step.decode.plan.num_segments == 1
    check(*rest, step=step)


@pytest.mark.parametrize("rows", [2, 5, 16, 17, 33, 70, 150])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_numbers_of_rows(device, rows, d):
    root = [("r", 20)]
    specs = [(root, 320 + 1 + (7 * i) % 40) for i in range(rows)]
    step, *rest = run(device, specs, 8, 2, 16, d, torch.bfloat16, seed=rows)
    assert step.decode.plan.num_segments == 1
    check(*rest, step=step)


@pytest.mark.parametrize("rows", [16, 17, 33, 70, 150])
@pytest.mark.parametrize("ps,pages", [(4, 80), (8, 37), (16, 20), (64, 5), (256, 2)])
def test_wide_workgroups(device, monkeypatch, rows, ps, pages):
    """Planned for one CU, so that segments of 64 columns and more are work enough for
    workgroups of 128."""
    monkeypatch.setattr(paged_kv, "_num_cus", lambda device: 1)
    root = [("r", pages)]
    specs = [(root, pages * ps + 1 + (7 * i) % 40) for i in range(rows)]
    step, *rest = run(device, specs, 8, 2, ps, 128, [torch.float16, torch.bfloat16][rows % 2],
                      seed=rows + ps)
    assert step.decode.plan.num_segments == 1 and step.decode.plan.shared_info.wide == 1
    check(*rest, step=step)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("ps", [4, 8, 32])
def test_other_pages(device, ps, d):
    """Pages smaller than what a wave loads at a time, tails that end inside one, at
    one, one token behind it, and longer than the waves' first steps."""
    root = [("r", 96 // ps)]
    specs = [(root, 96 + m) for m in (1, ps - 1, ps, ps + 1, 31, 64, 65, 255, 257, 600)]
    step, *rest = run(device, specs, 4, 2, ps, d, torch.float16, seed=ps + d)
    assert step.decode.plan.num_segments == 1
    check(*rest, step=step)


def test_prefixes_of_prefixes_and_strangers(device):
    """A tree of three levels, two roots, rows that share nothing, rows with
    identical page lists but their new tokens', and a row of one token."""
    a, ab, abc, ad, e = ("a", 12), ("ab", 6), ("abc", 5), ("ad", 7), ("e", 5)
    specs = [([a, ab, abc], 400), ([e], 90), ([a, ab, abc], 369), ([], 1), ([a, ab], 300),
             ([a, ad], 305), ([], 500), ([a, ad], 420), ([e], 81), ([a], 193), ([a, ab], 290),
             ([], 17), ([a, ab, abc], 700)]
    step, *rest = run(device, specs, 8, 2, 16, 128, torch.float16, seed=5)
    assert step.decode.plan.num_segments == 5
    check(*rest, step=step)


def test_large_pages_and_short_shares(device):
    """256-token pages; a shared page that the row's new token is in is not
    shared, nor are runs shorter than a segment."""
    specs = [([("r", 2)], n) for n in (513, 600, 769)] + [([("x", 3)], 49), ([("x", 3)], 64)]
    step, *rest = run(device, specs[:3], 8, 2, 256, 128, torch.bfloat16, seed=6)
    assert step.decode.plan.num_segments == 1
    check(*rest, step=step)
    step, *rest = run(device, [([("x", 2)], 33), ([("x", 2)], 40)], 8, 2, 16, 64, torch.float16)
    assert not isinstance(step.decode.plan, SharedDecodePlan)
    check(*rest, step=step)


def test_long_prefix_is_split(device):
    specs = [([("r", 600)], 9600 + m) for m in (5, 900)]
    step, *rest = run(device, specs, 8, 1, 16, 128, torch.bfloat16, seed=7, layers=1, layer=0)
    assert step.decode.plan.shared_info.num_shared > 8
    check(*rest, layer=0, step=step)


def test_within_a_mixed_step(device):
    """Decode rows among prompt chunks: only they share, in place."""
    from kunserve_amd import KVPool
    rng = np.random.default_rng(8)
    tables, pages = tree(rng, 16, [([("r", 10)], 161), ([("r", 10)], 200), ([], 50),
                                   ([("r", 10)], 170)])
    pool = random_pool(pages, 1, 2, 16, 128, device, 8)
    q_lens, first, flag = [1, 1, 30, 1], [161, 200, 20, 170], [0, 0, 1, 0]
    q, k, v = (random_tensor((33, h, 128), device, 9 + h) for h in (8, 2, 2))
    twin = KVPool(pool.k.clone(), pool.v.clone())
    out = AttentionStep(pool, 8, q_lens, first, flag, tables, share_prefixes=True,
                        share_min_bytes=0).run(0, q, k, v)
    want = AttentionStep(twin, 8, q_lens, first, flag, tables).run(0, q, k, v)
    assert torch.equal(pool.k.view(torch.int16), twin.k.view(torch.int16))
    assert torch.equal(out[2:32].view(torch.int16), want[2:32].view(torch.int16))
    rows = torch.tensor([0, 1, 32], device=device)
    check(pool, [tables[i] for i in (0, 1, 3)], [161, 200, 170], q[rows], out[rows], layer=0)


def test_values_that_are_not_finite(device):
    """An infinite value in a shared page stays in its dim, a NaN key makes its
    rows NaN, and what lies behind the rows' ends shows nowhere."""
    def poke(pool, tables):
        pool.v[tables[0][2], 1, 0, 5, 7] = float("inf")
        pool.k[tables[2][1], 1, 1, 3, 0] = float("nan")
        for t, n in zip(tables, kvs):
            pool.k[t[-1], :, :, n % 16 or 16:] = float("nan")
            pool.v[t[-1], :, :, n % 16 or 16:] = float("nan")
    kvs = [150, 170, 130, 131]
    specs = [([("r", 8)], 150), ([("r", 8)], 170), ([("s", 8)], 130), ([("s", 8)], 131)]
    step, pool, tables, kvs, q, out = run(device, specs, 8, 2, 16, 128, torch.bfloat16, poke=poke)
    assert torch.isinf(out[:2, :4, 7]).all()
    ok = torch.ones((4, 8, 128), dtype=torch.bool, device=device)
    ok[:2, :4, 7] = False
    ok[2:, 4:] = False
    assert torch.isnan(out[2:, 4:]).all() and torch.isfinite(out[ok]).all()
    pool.v[tables[0][2], 1, 0, 5, 7] = 0
    pool.k[tables[2][1], 1, 1, 3, 0] = 0
    clean = [pool.k.cpu(), pool.v.cpu()]
    got, qh = out.cpu().double().numpy(), q.cpu().double().numpy()
    for b in range(4):
        k, v = (ref.row_cache(x, 1, tables[b], kvs[b]) for x in clean)
        want, tol, _, _ = ref.attend(qh[b:b + 1], k, v, 1 / math.sqrt(128), pool.dtype)
        good = ok[b].cpu().numpy()
        assert np.all((np.abs(got[b] - want[0]) <= tol[0])[good])


@pytest.mark.parametrize("d", [64, 256])
def test_infinite_values_at_other_head_sizes(device, d):
    def poke(pool, tables):
        pool.v[tables[0][2], 1, 0, 5, d - 3] = -float("inf")
    specs = [([("r", 8)], 150 + i) for i in range(5)]
    _, _, _, _, _, out = run(device, specs, 8, 2, 16, d, torch.float16, poke=poke)
    bad = torch.zeros((5, 8, d), dtype=torch.bool, device=device)
    bad[:, :4, d - 3] = True
    assert (out[bad] == -float("inf")).all() and torch.isfinite(out[~bad]).all()


def test_infinite_values_in_wide_workgroups(device, monkeypatch):
    monkeypatch.setattr(paged_kv, "_num_cus", lambda device: 1)

    def poke(pool, tables):
        pool.v[tables[0][2], 1, 0, 5, 40] = float("inf")
    specs = [([("r", 20)], 330 + i) for i in range(21)]
    step, _, _, _, _, out = run(device, specs, 8, 2, 16, 128, torch.bfloat16, poke=poke)
    assert step.decode.plan.shared_info.wide == 1
    bad = torch.zeros((21, 8, 128), dtype=torch.bool, device=device)
    bad[:, :4, 40] = True
    assert (out[bad] == float("inf")).all() and torch.isfinite(out[~bad]).all()


def test_page_ids_outside_the_pool_drop_out(device):
    """Through the op itself, with a table the shim did not check: a shared id
    outside the pool drops its tokens for every row."""
    rng = np.random.default_rng(11)
    tables, pages = tree(rng, 16, [([("r", 9)], 160), ([("r", 9)], 200)])
    pool = random_pool(pages, 1, 2, 16, 128, device, 11)
    bad = [list(t) for t in tables]
    for t in bad:
        t[3] = pages + 5
    kvs = [160, 200]
    indptr = np.r_[0, np.cumsum([len(t) for t in bad])]
    table = PageTable(indptr, np.concatenate(bad), kvs, device)
    plan = SharedDecodePlan(table, 8, 2, 16, device, min_bytes=0)
    assert plan.num_segments == 1
    q = random_tensor((2, 8, 128), device, 12, 2.0)
    out = shared_decode(pool, 0, table, q, plan)
    kh, vh, qh = pool.k.cpu(), pool.v.cpu(), q.cpu().double().numpy()
    for b in range(2):
        k, v = (ref.row_cache(x, 0, tables[b], kvs[b]) for x in (kh, vh))
        valid = np.ones(kvs[b], dtype=bool)
        valid[48:64] = False
        want, tol, _, _ = ref.attend(qh[b:b + 1], k, v, 1 / math.sqrt(128), pool.dtype, valid=valid)
        assert np.all(np.abs(out[b].cpu().double().numpy() - want[0]) <= tol[0])


@pytest.mark.parametrize("d,ps,cus", [(64, 4, 256), (64, 8, 256), (128, 4, 256), (128, 16, 1),
                                      (128, 8, 1), (256, 16, 256), (256, 4, 256)])
def test_page_ids_outside_the_pool_in_segments_and_tails(device, d, ps, cus):
    """Bad ids in the shared pages and in each row's own, in first and later steps, NaN
    in page 0, which is read in their place: 18 rows, narrow workgroups and wide ones."""
    rng = np.random.default_rng(13)
    kvs = [480 + 37 * i for i in range(18)]
    tables, pages = tree(rng, ps, [([("r", 400 // ps)], n) for n in kvs])
    pool = random_pool(pages + 1, 1, 2, ps, d, device, 13)
    tables = [[p + 1 for p in t] for t in tables]
    pool.k[0] = float("nan")
    pool.v[0] = float("nan")
    bad = [list(t) for t in tables]
    drops = [[] for _ in kvs]
    for b, t in enumerate(bad):
        for at in (16 // ps, 200 // ps, 400 // ps + b % 3, (kvs[b] - 1) // ps - 1):
            t[at] = [pages + 7, -1][at < 400 // ps and at > 20]
            drops[b].append(at)
    shared = bad[0][:400 // ps]
    assert all(t[:400 // ps] == shared for t in bad)
    indptr = np.r_[0, np.cumsum([len(t) for t in bad])]
    table = PageTable(indptr, np.concatenate(bad), kvs, device)
    plan = SharedDecodePlan(table, 8, 2, ps, device, head_dim=d, min_bytes=0, num_cus=cus)
    assert plan.num_segments == 1 and plan.shared_info.wide == (cus == 1)
    q = random_tensor((len(kvs), 8, d), device, 14, 2.0)
    out = shared_decode(pool, 0, table, q, plan)
    p_err = ref.half_step(pool.dtype) if cus == 1 else None
    kh, vh, qh = pool.k.cpu(), pool.v.cpu(), q.cpu().double().numpy()
    for b in range(len(kvs)):
        k, v = (ref.row_cache(x, 0, tables[b], kvs[b]) for x in (kh, vh))
        valid = np.ones(kvs[b], dtype=bool)
        for at in drops[b]:
            valid[at * ps:(at + 1) * ps] = False
        want, tol, _, _ = ref.attend(qh[b:b + 1], k, v, 1 / math.sqrt(d), pool.dtype, p_err,
                                     valid=valid)
        assert np.all(np.abs(out[b].cpu().double().numpy() - want[0]) <= tol[0]), b


def test_rows_of_no_and_of_one_token(device):
    """Through the op: a row with an empty cache gives zeros beside rows that
    share, a row of one token its value."""
    rng = np.random.default_rng(17)
    kvs = [0, 160, 1, 200]
    tables, pages = tree(rng, 16, [([], 0), ([("r", 9)], 160), ([], 1), ([("r", 9)], 200)])
    pool = random_pool(pages, 1, 2, 16, 128, device, 17, dtype=torch.bfloat16)
    table = PageTable.from_lists(tables, kvs, pool)
    plan = SharedDecodePlan(table, 8, 2, 16, device, min_bytes=0)
    assert plan.num_segments == 1
    q = random_tensor((4, 8, 128), device, 18, 2.0, torch.bfloat16)
    out = shared_decode(pool, 0, table, q, plan)
    assert not out[0].any()
    one = pool.v[tables[2][0], 0, :, 0].repeat_interleave(4, dim=0)
    assert torch.equal(out[2].view(torch.int16), one.view(torch.int16))
    rows = [1, 3]
    check(pool, [tables[b] for b in rows], [kvs[b] for b in rows], q[rows], out[rows], layer=0)
    none = PageTable.from_lists([], [], pool)
    empty = SharedDecodePlan(none, 8, 2, 16, device)
    assert shared_decode(pool, 0, none, q[:0], empty).shape == (0, 8, 128)


def test_strided_tensors_and_a_row_map(device):
    """q and out as slices of wider tensors, rows anywhere among the tokens, what
    is of no row left as it was; pools with gaps."""
    from kunserve_amd import KVPool
    rng = np.random.default_rng(19)
    kvs = [150 + 11 * i for i in range(20)]
    tables, pages = tree(rng, 16, [([("r", 9)], n) for n in kvs])
    dense = random_pool(pages, 2, 2, 16, 128, device, 19, dtype=torch.bfloat16)
    k, v = (torch.zeros((pages, 2, 3, 16, 136), dtype=torch.bfloat16,
                        device=device)[:, :, :2, :, :128] for _ in range(2))
    k.copy_(dense.k)
    v.copy_(dense.v)
    pool = KVPool(k, v)
    table = PageTable.from_lists(tables, kvs, pool)
    plan = SharedDecodePlan(table, 8, 2, 16, device, min_bytes=0)
    wide = random_tensor((40, 12, 128), device, 20, 2.0, torch.bfloat16)
    q = wide[:, 2:10]
    where = torch.tensor(rng.permutation(40)[:20], dtype=torch.int32, device=device)
    outs = torch.full((40, 10, 128), 7.0, dtype=torch.bfloat16, device=device)
    out = shared_decode(pool, 1, table, q, plan, out=outs[:, 1:9], q_token=where)
    check(dense, tables, kvs, q[where.long()], out[where.long()], plan=plan)
    rest = torch.ones(40, dtype=torch.bool, device=device)
    rest[where.long()] = False
    assert (outs[rest] == 7).all() and (outs[:, 0] == 7).all() and (outs[:, 9] == 7).all()


def test_captured_layer_replays(device):
    rng = np.random.default_rng(13)
    kvs = [330, 400, 321]
    tables, pages = tree(rng, 16, [([("r", 20)], n) for n in kvs])
    pool = random_pool(pages, 1, 2, 16, 128, device, 13)
    q, k, v = (random_tensor((3, h, 128), device, 14 + h) for h in (8, 2, 2))
    step = AttentionStep(pool, 8, [1] * 3, kvs, [0] * 3, tables, share_prefixes=True,
                         share_min_bytes=0)
    out = torch.empty_like(q)
    eager = step.run(0, q, k, v).clone()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step.run(0, q, k, v, out=out)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.view(torch.int16), eager.view(torch.int16))
        torch.randn(1000, device=device).sum()


def test_two_steps_on_two_streams(device):
    """Steps have their own workspaces: two of them at once give what each gives
    alone."""
    sets = []
    for seed in (20, 21):
        specs = [([("r", 40)], 640 + 9 * i) for i in range(1, 20)]
        step, pool, tables, kvs, q, out = run(device, specs, 8, 2, 16, 128, torch.bfloat16,
                                              seed=seed)
        k = random_tensor((19, 2, 128), device, seed + 2, dtype=torch.bfloat16)
        v = random_tensor((19, 2, 128), device, seed + 3, dtype=torch.bfloat16)
        sets.append((step, q, k, v, out, torch.cuda.Stream(device)))
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for step, q, k, v, out, s in sets:
            with torch.cuda.stream(s):
                got.append((step.run(1, q, k, v), out))
    torch.cuda.synchronize()
    assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in got)


def test_refusals(device):
    rng = np.random.default_rng(15)
    tables, pages = tree(rng, 16, [([("r", 9)], 160), ([("r", 9)], 200)])
    pool = random_pool(pages, 1, 2, 16, 128, device, 15)
    table = PageTable.from_lists(tables, [160, 200], pool)
    q = random_tensor((2, 8, 128), device, 16)
    plan = SharedDecodePlan(table, 16, 2, 16, device, min_bytes=0)
    with pytest.raises(RuntimeError, match="group size"):
        shared_decode(pool, 0, table, q, plan)
    plan = SharedDecodePlan(table, 8, 2, 16, device, head_dim=64, min_bytes=0)
    with pytest.raises(RuntimeError, match="head_dim"):
        shared_decode(pool, 0, table, q, plan)
    plan = SharedDecodePlan(table, 8, 2, 16, device, min_bytes=0)
    with pytest.raises(ValueError, match="rows"):
        shared_decode(pool, 0, table, q[:1], plan)
    with pytest.raises(ValueError, match="another table"):
        shared_decode(pool, 0, PageTable.from_lists(tables, [160, 200], pool), q, plan)
    with pytest.raises(ValueError, match="on cpu"):
        shared_decode(pool, 0, table, q.cpu(), plan)
    with pytest.raises(RuntimeError, match="sm_scale"):
        shared_decode(pool, 0, table, q, plan, sm_scale=0.0)
    with pytest.raises(RuntimeError):
        SharedDecodePlan(table, 8, 2, 16, device, head_dim=96)
