"""kunserve_shared_plan on the host: every row's tokens are covered exactly once
by the segments on its path and its tail, by workgroups whose rows do hold the
same pages there."""
import ctypes

import numpy as np
import pytest
from hypothesis import HealthCheck, given, settings, strategies as st

from kunserve_amd import _lib


def plan_of(tables, kv, hq, hkv, ps, d, cus=256, min_bytes=0):
    kv = np.asarray(kv, dtype=np.int32)
    indptr = np.r_[0, np.cumsum([len(t) for t in tables])].astype(np.int32)
    indices = (np.concatenate(tables) if indptr[-1] else np.zeros(0)).astype(np.int32)
    n = len(kv)
    cap = _lib.lib().kunserve_shared_plan_bound(kv.ctypes.data if n else None, n, hq)
    buf = np.full(max(cap, 4), -9, dtype=np.int32)
    info = _lib.SharedPlanInfo()
    _lib.call("kunserve_shared_plan", indptr.ctypes.data, indices.ctypes.data,
              kv.ctypes.data if n else None, n, hq, hkv, ps, d, cus, min_bytes, buf.ctypes.data,
              cap, ctypes.byref(info))
    assert info.plan_ints <= cap
    return info, buf[:info.plan_ints]


def check(tables, kv, hq, hkv, ps, d, cus=256):
    info, plan = plan_of(tables, kv, hq, hkv, ps, d, cus)
    dec = info.decode
    group = dec.group_size
    heads = hq // group
    work = plan[:4 * dec.num_work].reshape(-1, 4)
    merges = plan[4 * dec.num_work:dec.plan_ints].reshape(-1, 4)
    shared = plan[dec.plan_ints:dec.plan_ints + 8 * info.num_shared].reshape(-1, 8)
    at = dec.plan_ints + 8 * info.num_shared
    pairs = plan[at:at + 2 * info.num_pairs].reshape(-1, 2)
    starts = np.r_[0, np.cumsum([len(t) for t in tables])]
    at += 2 * info.num_pairs
    np.testing.assert_array_equal(plan[at:at + dec.num_work],
                                  np.where(work[:, 0] < 0, 0, starts[work[:, 0]]))
    # the pages of four waves' first steps (4096 elements each), a granule at a time
    step, load = 4096 // d, 512 // d
    granule = 16 if ps >= 16 else load
    ids = plan[at + dec.num_work:].reshape(dec.num_work, 0 if ps < load else 4 * step // granule)
    for (b, lo, hi, _), got_ids in zip(work.tolist(), ids.tolist()):
        if b >= 0 and kv[b]:
            assert got_ids == [tables[b][min(lo + i * granule, hi - 1) // ps]
                               for i in range(len(got_ids))]
    assert dec.num_work % 8 == 0 and info.num_shared % 8 == 0
    first = {int(b): (int(s0), int(m)) for b, s0, m, _ in merges}
    # (row, head group) -> [(begin, end, slot)]
    got = {(b, h): [] for b in range(len(kv)) for h in range(heads)}
    for b, lo, hi, slot in work[work[:, 0] >= 0].tolist():
        assert hi - lo <= dec.part_tokens
        for h in range(heads):
            got[b, h].append((lo, hi, slot))
    for nrows, at, lo, hi, place, rep, h, pages_at in shared[shared[:, 0] > 0].tolist():
        cols = nrows * group
        wide = info.wide and d == 128
        assert 0 < cols <= (128 if wide else 16) and 0 <= h < heads and lo < hi
        assert lo % 4 == 0 and hi - lo <= 4096
        rows = pairs[at:at + nrows]
        assert rep in pairs[:, 0] and pages_at == starts[rep]
        want = tables[rep][lo // ps:-(-hi // ps)]
        for b, s0 in rows.tolist():
            assert tables[b][lo // ps:-(-hi // ps)] == want
            assert hi <= (kv[b] - 1) // ps * ps     # before its new token's page
            assert s0 == first[b][0]
            got[b, h].append((lo, hi, s0 + place))
    slots = []
    for (b, h), parts in got.items():
        parts.sort()
        if kv[b] == 0:
            assert parts == [(0, 0, -1)]
            continue
        assert parts[0][0] == 0 and parts[-1][1] == kv[b]
        assert all(x[1] == y[0] for x, y in zip(parts, parts[1:]))
        mine = [p[2] for p in parts]
        if len(parts) == 1:
            assert mine == [-1] and b not in first
        else:
            s0, m = first[b]
            assert m == len(parts) and sorted(mine) == list(range(s0, s0 + m))
            if h == 0:
                slots += mine
    assert sorted(slots) == list(range(dec.num_slots))
    return info


@st.composite
def trees(draw):
    ps = draw(st.sampled_from([4, 16, 256]))
    made, at, tables, kv = [[]], 0, [], []
    for _ in range(draw(st.integers(0, 6))):     # prefixes of prefixes
        base = draw(st.sampled_from(made))
        n = draw(st.integers(1, max(1, 2000 // ps)))
        made.append(base + list(range(at, at + n)))
        at += n
    for _ in range(draw(st.integers(0, 20))):
        base = draw(st.sampled_from(made))
        n = draw(st.integers(0, max(1, 700 // ps)))
        t = base + list(range(at, at + n))
        at += n
        tables.append(t)
        kv.append(draw(st.integers(max(0, len(t) * ps - 3 * ps), len(t) * ps)))
    return ps, tables, kv


@settings(max_examples=80, deadline=None, suppress_health_check=[HealthCheck.too_slow])
@given(tree=trees(), heads=st.sampled_from([(1, 1), (4, 4), (8, 2), (6, 2), (34, 2), (16, 1)]),
       d=st.sampled_from([64, 128, 256]), cus=st.sampled_from([0, 1, 64, 256]))
def test_every_token_once(tree, heads, d, cus):
    ps, tables, kv = tree
    check(tables, kv, *heads, ps, d, cus)


def rows(root, branches, ps=16):
    """Rows behind one root of pages, each with so many pages of its own."""
    at, out = root, []
    for n in branches:
        out.append(list(range(root)) + list(range(at, at + n)))
        at += n
    return out


def test_segments_follow_the_tree():
    a, b, c = list(range(10)), list(range(10, 16)), list(range(16, 30))
    tables = [a + b + [30], a + c + [31], a + b + [32], a + c + [33], a + [34], [35] * 3]
    kv = [len(t) * 16 - 3 for t in tables]
    info = check(tables, kv, 8, 2, 16, 128)
    assert info.num_segments == 3      # a; a b; a c
    info = check([a, a], [160, 160], 8, 2, 16, 128)
    assert info.num_segments == 1      # whole lists alike: but for the last page
    info = check([a[:4] + [30], a[:4] + [31]], [70, 80], 8, 2, 16, 128)
    assert info.num_segments == 1      # 64 tokens
    info = check([a[:3] + [30], a[:3] + [31]], [60, 64], 8, 2, 16, 128)
    assert info.num_segments == 0      # 48
    info = check([a + [30], a + [31]], [161, 64], 8, 2, 16, 128)
    assert info.num_segments == 0      # the second row's new token is in page 3


def test_wide_workgroups_take_many_columns():
    t = rows(20, [1] * 40)
    kv = [len(x) * 16 - 5 for x in t]
    assert check(t, kv, 8, 2, 16, 128, cus=1).wide == 1
    assert check(t, kv, 8, 2, 16, 64, cus=1).wide == 0
    assert check(t[:15], kv[:15], 8, 2, 16, 128, cus=1).wide == 0    # 60 columns
    # narrow ones would have 0.0115 us a token, 320 tokens, 10 tiles of columns and 2 KV
    # heads of work: 73.6 us, 20 for each CU up to 3
    assert check(t, kv, 8, 2, 16, 128, cus=3).wide == 1
    assert check(t, kv, 8, 2, 16, 128, cus=4).wide == 0


def test_sharing_has_to_pay():
    t = rows(64, [2] * 8)
    kv = [len(x) * 16 - 5 for x in t]
    saved = 7 * 1024 * 2 * 128 * 4
    assert plan_of(t, kv, 8, 2, 16, 128, min_bytes=saved)[0].num_segments == 1
    assert plan_of(t, kv, 8, 2, 16, 128, min_bytes=saved + 1)[0].num_segments == 0
    assert plan_of(t, kv, 8, 2, 16, 128, min_bytes=-1)[0].num_segments == 0    # 7 MB
    assert plan_of(t, kv, 32, 8, 16, 128, min_bytes=-1)[0].num_segments == 1   # 29 MB


def test_plans_beyond_the_first_buffer(monkeypatch):
    """SharedDecodePlan tries a small buffer before the bound's; a plan that does
    not fit is made again."""
    import torch
    from kunserve_amd import PageTable, SharedDecodePlan, paged_kv

    t = rows(20, [1] * 40)
    kv = [len(x) * 16 - 5 for x in t]
    indptr = np.r_[0, np.cumsum([len(x) for x in t])]
    table = PageTable(indptr, np.concatenate(t), kv, torch.device("cpu"), upload=False)
    make = lambda: SharedDecodePlan(table, 8, 2, 16, torch.device("cpu"), num_cus=256,   # noqa: E731
                                    upload=False, min_bytes=0)
    want = make().plan_host
    monkeypatch.setattr(paged_kv, "_SHARED_PLAN_INTS", 16)
    assert len(want) > 16
    np.testing.assert_array_equal(make().plan_host, want)
    with pytest.raises(_lib.KunserveError, match="power of two"):
        SharedDecodePlan(table, 8, 2, 12, torch.device("cpu"), num_cus=256, upload=False)


def test_refusals():
    with pytest.raises(_lib.KunserveError, match="multiple"):
        plan_of([[0]], [3], 5, 2, 16, 128)
    with pytest.raises(_lib.KunserveError, match="power of two"):
        plan_of([[0]], [3], 4, 2, 12, 128)
    with pytest.raises(_lib.KunserveError, match="pages for"):
        plan_of([[0]], [17], 4, 2, 16, 128)
    with pytest.raises(_lib.KunserveError, match="pages for"):
        plan_of([[0]], [-1], 4, 2, 16, 128)
    with pytest.raises(_lib.KunserveError) as e:
        plan_of([[0]], [3], 4, 2, 16, 96)
    assert e.value.code == _lib.EUNSUPPORTED
    info, buf = _lib.SharedPlanInfo(), np.zeros(4, np.int32)
    arr = np.array([0, 1], np.int32)
    with pytest.raises(_lib.KunserveError) as e:
        _lib.call("kunserve_shared_plan", arr.ctypes.data, arr.ctypes.data,
                  np.array([7], np.int32).ctypes.data, 1, 4, 2, 16, 128, 256, 0, buf.ctypes.data,
                  4, ctypes.byref(info))
    assert e.value.code == _lib.ENOSPC


def test_a_plan_and_its_pool():
    """Checks of the launch that come before it: the pool's page size is the plan's,
    and a token's stride fits the kernel's 32-bit offsets."""
    info, _ = plan_of(rows(4, [1] * 3), [70, 70, 70], 4, 2, 16, 128)
    buf = np.zeros(64, np.uint8)
    at = -(-buf.ctypes.data // 16) * 16
    three = _lib.Tensor3(at, 512, 128)

    def decode(page_size=16, token_stride=128, **kw):
        pool = _lib.KVPool(k=at, v=at, num_pages=1, page_stride=1 << 40, layer_stride=1 << 39,
                           head_stride=1 << 38, token_stride=token_stride, num_layers=1,
                           num_kv_heads=2, page_size=page_size, head_dim=128, dtype=0)
        table = _lib.PageTable(at, at, at, 3)
        _lib.call("kunserve_shared_decode", ctypes.byref(pool), 0, ctypes.byref(table), None,
                  ctypes.byref(three), ctypes.byref(three), 4, 1.0, at, ctypes.byref(info), None,
                  0, None)

    assert info.num_segments == 1
    with pytest.raises(_lib.KunserveError, match="pages of 16"):
        decode(page_size=32)
    with pytest.raises(_lib.KunserveError, match="2\\^28"):
        decode(token_stride=1 << 28)
