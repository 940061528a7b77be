"""kunserve_weights_plan on the host, and what the weights and the eviction refuse
before they reach a device."""
import ctypes

import numpy as np
import pytest
import torch
from hypothesis import given, settings, strategies as st

from kunserve_amd import KVPool, KVWeights, WeightsPlan, _lib, evict

CPU = torch.device("cpu")


def plan_of(q_lens, kv, hq, window, decodes=None):
    return WeightsPlan(np.r_[0, np.cumsum(q_lens)], kv, hq, window, CPU, upload=False,
                       decodes=decodes)


@settings(max_examples=60, deadline=None)
@given(rows=st.lists(st.tuples(st.integers(0, 600), st.integers(0, 40000), st.booleans()),
                     max_size=12),
       hq=st.sampled_from([1, 8, 34]), window=st.sampled_from([1, 16, 700]))
def test_rows_are_covered_once(rows, hq, window):
    q = [1 if dec else a for a, _, dec in rows]
    kv = [n + k for n, (_, k, _) in zip(q, rows)]
    dec = [int(x) for _, _, x in rows]
    p = plan_of(q, kv, hq, window, dec)
    info, ints = p.info, p.plan_host
    items, rest = ints[:4 * info.num_items].reshape(-1, 4), ints[4 * info.num_items:]
    comb, rest = rest[:4 * info.num_combines].reshape(-1, 4), rest[4 * info.num_combines:]
    score, at = rest[:4 * info.num_score_items].reshape(-1, 4), rest[4 * info.num_score_items:]
    assert len(at) == info.num_score_rows == sum(dec) and info.num_seqs == len(rows)
    columns = tokens = 0
    many = any(-(-n // 256) > 64 for n, t, x in zip(kv, q, dec) if t and not x)
    row = 0
    for b, (t, n, x) in enumerate(zip(q, kv, dec)):
        if x:
            mine = score[score[:, 0] == row]
            assert mine[:, 1].tolist() == list(range(0, n, 256)) and set(mine[:, 2]) <= {tokens}
            assert at[row] == tokens
            tokens += n
            row += 1
            assert not (items[:, 0] == b).any()
            continue
        mine = items[items[:, 0] == b]
        if t == 0:
            assert not len(mine)
            continue
        parts, cols = -(-n // 256), min(t, window) * hq
        assert mine[:, 1].tolist() == list(range(0, n, 256))
        assert set(mine[:, 2]) == {columns} and set(mine[:, 3]) == {parts}
        if many:
            c = comb[comb[:, 0] == b]
            assert c[:, 1].tolist() == list(range(0, cols, 256)) and set(c[:, 3]) == {parts}
        columns += (parts + 1) * cols
    assert bool(info.num_combines) == many
    assert info.num_columns == columns and info.score_tokens == tokens
    need = p.workspace_bytes()
    assert need >= 8 * columns + 4 * hq * (tokens + sum(dec))


def test_plan_refusals():
    with pytest.raises(_lib.KunserveError, match="window"):
        plan_of([1], [3], 4, 0)
    with pytest.raises(_lib.KunserveError, match="new tokens"):
        plan_of([4], [3], 4, 8)
    with pytest.raises(_lib.KunserveError, match="decodes 2 tokens"):
        plan_of([2], [3], 4, 8, [1])
    with pytest.raises(ValueError, match="decode marks"):
        plan_of([1], [3], 4, 8, [1, 0])
    with pytest.raises(ValueError, match="num_seqs"):
        WeightsPlan([0, 1], [3, 4], 4, 8, CPU, upload=False)
    with pytest.raises(_lib.KunserveError, match="too many"):
        plan_of([2**20], [2**30], 64, 2**20)


@pytest.fixture
def pool():
    return KVPool.allocate(12, 2, 2, 16, 64, CPU)


def test_weights_refusals(pool):
    w = KVWeights(pool)
    assert w.w.shape == (12, 2, 2, 16) and not w.w.any()
    for bad in (torch.zeros(12, 2, 2, 8), torch.zeros(12, 2, 2, 16, dtype=torch.float64),
                torch.zeros(12, 2, 2, 32)[..., ::2]):
        with pytest.raises(ValueError, match="weights must be"):
            KVWeights(pool, bad)
    with pytest.raises(ValueError, match="share memory"):
        KVWeights(pool, torch.zeros(1, 2, 2, 16).expand(12, 2, 2, 16))
    with pytest.raises(ValueError, match="not those"):
        w.check(KVPool.allocate(13, 2, 2, 16, 64, CPU))


def test_evict_refusals(pool, monkeypatch):
    def no_call(name, *args):
        raise AssertionError(f"{name} was called")

    w = KVWeights(pool)
    monkeypatch.setattr(_lib, "call", no_call)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    tables, kv, out = [[0, 1, 2], [3, 4]], [40, 20], [[5, 6], [7]]
    ok = dict(budget=[20, 10])
    assert evict(pool, w, tables, kv, out, 0).shape == (2, 2, 2, 0)
    assert evict(pool, w, [], [], [], 9).shape == (0, 2, 2, 0)
    for kw, what in ((dict(budget=[20, 10, 3]), "one per request"), (dict(budget=-1), "negative"),
                     (dict(budget=[[20, 10]]), "one per request"),
                     (dict(budget=0.2), "whole numbers"), (dict(budget=[1.0, 2.0]), "whole"),
                     (dict(ok, sinks=-1), "negative"), (dict(ok, recent=-2), "negative")):
        with pytest.raises(ValueError, match=what):
            evict(pool, w, tables, kv, out, **kw)
    for args, what in (((tables[:1], kv, out), "page lists"), ((tables, kv, out[:1]), "page lists"),
                       ((tables, [40, -20], out), "negative"),
                       ((tables, kv, [[5], [7]]), "pages for"),
                       ((tables, kv, [[5, 2], [7]]), "holds tokens"),
                       ((tables, kv, [[5, 7], [7]]), "twice"),
                       ((tables, [2**31, 20], out), "over")):
        with pytest.raises(ValueError, match=what):
            evict(pool, w, *args, **ok)
    with pytest.raises(IndexError):
        evict(pool, w, tables, kv, [[5, 12], [7]], **ok)
    with pytest.raises(IndexError):
        evict(pool, w, [[0, 1, -2], [3, 4]], kv, out, **ok)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="captured"):
        evict(pool, w, tables, kv, out, **ok)
