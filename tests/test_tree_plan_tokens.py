"""Which tokens of q and out, and which of a table's pages, a tree plan's rows may have (CPU
only)."""
import ctypes

import numpy as np
import pytest
import torch

from kunserve_amd import PageTable, TreePlan, _lib

CPU = torch.device("cpu")
TREES = [[-1, 0, 0], [-1], [], [-1, -1]]


def plan(q_first):
    lens = [20, 9, 4, 7]
    indptr = np.cumsum([0, 2, 1, 1, 1])
    table = PageTable(indptr, np.arange(5), lens, CPU, upload=False)
    return TreePlan(table, TREES, 4, 2, 16, CPU, num_cus=256, head_dim=64, q_first=q_first, upload=False)


@pytest.mark.parametrize("q_first", [None, [0, 3, 4, 4], [5, 0, 0, 1], [10, 13, 11, 2], [2, 1, 2**31 - 1, 30]])
def test_rows_apart(q_first):
    assert plan(q_first).info.num_work > 0


@pytest.mark.parametrize("q_first", [[0, 0, 9, 5], [0, 2, 9, 5], [4, 6, 0, 9], [3, 0, 9, 2], [8, 0, 9, 7]])
def test_rows_with_tokens_in_common(q_first):
    """Their outputs would be written by one another."""
    with pytest.raises(_lib.KunserveError, match="rows .* have token") as e:
        plan(q_first)
    assert e.value.code == _lib.EINVAL


def test_tokens_past_32_bits():
    """From C: a row's last token is counted in 32 bits on the device."""
    q, kv, ip = (np.array(x, np.int32) for x in ([0, 2], [9], [0, 1]))
    up, first = np.array([-1, 0], np.int32), np.zeros(1, np.int32)
    buf, info = np.zeros(4096, np.int32), _lib.TreePlanInfo()

    def make():
        _lib.call("kunserve_tree_plan", ip.ctypes.data, q.ctypes.data, first.ctypes.data,
                  kv.ctypes.data, up.ctypes.data, 1, 4, 2, 16, 64, 256, 0, buf.ctypes.data,
                  len(buf), ctypes.byref(info))
    first[0] = 2**31 - 2
    make()
    first[0] = 2**31 - 1
    with pytest.raises(_lib.KunserveError, match="first token is 2147483647"):
        make()


def test_pages_before_the_table():
    """A row's page ids are read from where the plan says."""
    table = PageTable(np.array([-2, 2]), np.arange(2), [20], CPU, upload=False)
    with pytest.raises(_lib.KunserveError, match="pages start at -2"):
        TreePlan(table, [[-1, 0]], 4, 2, 16, CPU, num_cus=256, head_dim=64, upload=False)
