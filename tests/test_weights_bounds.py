"""add_weights runs its plan's rows alone: the workspace is laid out by the plan's
q_indptr, so the launches get the plan's copy, and what reaches past q or is no index
array on the device is refused before a launch."""
import numpy as np
import pytest
import torch

from kunserve_amd import KVPool, KVWeights, PageTable, WeightsPlan, _lib, add_weights

CPU = torch.device("cpu")


@pytest.fixture
def calls(monkeypatch):
    """Launches are recorded, not made; the plans are the library's."""
    made, call = [], _lib.call

    def record(name, *args):
        if name != "kunserve_cache_weights":
            return call(name, *args)
        made.append(args)
        return 0
    monkeypatch.setattr(_lib, "call", record)
    monkeypatch.setattr("kunserve_amd.cache_weights._stream_ptr", lambda device: 0)
    return made


def setup(q_lens, kvs):
    pool = KVPool.allocate(24, 1, 2, 16, 64, CPU)
    at, tables = 0, []
    for n in kvs:
        need = -(-n // 16)
        tables.append(list(range(at, at + need)))
        at += need
    table = PageTable.from_lists(tables, kvs, pool, upload=False)
    table.bind([torch.from_numpy(a) for a in table.host_arrays()])
    qi = np.r_[0, np.cumsum(q_lens)].astype(np.int32)
    plan = WeightsPlan(qi, kvs, 4, 16, CPU, upload=False)
    plan.bind([torch.from_numpy(a) for a in plan.host_arrays()])
    q = torch.zeros((int(qi[-1]), 4, 64), dtype=torch.float16)
    return pool, KVWeights(pool), table, torch.from_numpy(qi), q, plan


def test_the_launch_reads_the_plans_rows(calls):
    """30 observers a row where the plan has one: statistics of 2 x 16 x 4 columns
    in a workspace of 2 x 4."""
    pool, w, table, qi, q, plan = setup([1, 1], [40, 70])
    other = torch.tensor([0, 30, 60], dtype=torch.int32)
    add_weights(pool, w, 0, table, other, torch.zeros((60, 4, 64), dtype=torch.float16), plan)
    add_weights(pool, w, 0, table, qi, q, plan)
    for args in calls:
        given = np.ctypeslib.as_array((np.ctypeslib.ctypes.c_int32 * 3).from_address(args[4]))
        np.testing.assert_array_equal(given, [0, 1, 2])


def test_q_holds_the_plans_tokens(calls):
    pool, w, table, qi, q, plan = setup([3, 5], [40, 70])
    with pytest.raises(ValueError, match="7 tokens, the plan's rows end at 8"):
        add_weights(pool, w, 0, table, qi, q[:7], plan)
    assert not calls
    add_weights(pool, w, 0, table, qi, torch.cat([q, q]), plan)   # tokens of no row
    assert len(calls) == 1


@pytest.mark.parametrize("bad", [
    lambda qi: qi.long(), lambda qi: qi[:2], lambda qi: torch.stack([qi, qi], 1)[:, 0],
    lambda qi: qi.to("meta")])
def test_q_indptr_is_an_index_array_of_the_device(calls, bad):
    pool, w, table, qi, q, plan = setup([1, 1], [40, 70])
    with pytest.raises(ValueError, match="q_indptr"):
        add_weights(pool, w, 0, table, bad(qi), q, plan)
    assert not calls


def test_plans_that_are_not_on_the_device_or_begin_before_q(calls):
    pool, w, table, qi, q, plan = setup([1, 1], [40, 70])
    bare = WeightsPlan([0, 1, 2], [40, 70], 4, 16, CPU, upload=False)
    with pytest.raises(RuntimeError, match="bound"):
        add_weights(pool, w, 0, table, qi, q, bare)
    assert not calls
    with pytest.raises(_lib.KunserveError, match="begins at -1"):
        WeightsPlan([-1, 0, 1], [40, 70], 4, 16, CPU, upload=False)
