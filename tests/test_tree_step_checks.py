"""What a step refuses of its tree rows it refuses before its first launch, so that neither q,
rotated in place, nor a page is changed by a call that fails (CPU only: nothing is launched)."""
import ctypes

import numpy as np
import pytest
import torch

from kunserve_amd import KVPool, PageTable, Rotary, TreePlan, _lib

CPU = torch.device("cpu")
HQ, HKV, DIM, PAGE = 4, 2, 64, 16


class Call:
    """A layer of a step of two tree rows, as the C entry takes it; its rotary would be the
    first launch."""

    def __init__(self):
        lists, lens, trees = [[0, 1], [2]], [20, 9], [[-1, 0, 0], [-1]]
        self.pool = KVPool.allocate(4, 1, HKV, PAGE, DIM, CPU)
        self.table = PageTable.from_lists(lists, lens, self.pool, upload=False)
        self.plan = TreePlan(self.table, trees, HQ, HKV, PAGE, CPU, num_cus=256, head_dim=DIM,
                             part_rounds=1, upload=False)
        self.table.bind([torch.from_numpy(x) for x in self.table.host_arrays()])
        self.plan.bind([torch.from_numpy(x) for x in self.plan.host_arrays()])
        assert self.plan.info.num_slots > 0
        self.q, self.k, self.v, self.out = (torch.zeros(4, h, DIM + 8, dtype=torch.float16)
                                            for h in (HQ, HKV, HKV, HQ))
        self.qi = torch.tensor([0, 3, 4], dtype=torch.int32)
        self.workspace = torch.zeros(self.plan.workspace_bytes() + 16, dtype=torch.uint8)
        at = self.workspace.data_ptr()
        self.more = _lib.StepMore(self.table._desc, self.plan.plan.data_ptr(), self.plan.info)
        self.step = _lib.Step(pool=self.pool._desc, table=self.table._desc,
                              q_indptr_dev=self.qi.data_ptr(), num_tokens=4, num_qo_heads=HQ,
                              sm_scale=0.125, workspace_dev=at + -at % 16,
                              workspace_bytes=self.plan.workspace_bytes())
        self.out_at = self.out.data_ptr()
        self.out_strides = [(DIM + 8) * HQ, DIM + 8]
        self.rotary = Rotary(DIM, device=CPU)

    def run(self):
        def three(t):
            return t.data_ptr(), t.stride(0), t.stride(1)
        io = _lib.STEP_IO.pack(*three(self.q), *three(self.k), *three(self.v), self.out_at,
                               *self.out_strides, 0, 0)
        _lib.call("kunserve_attention_step_more", ctypes.byref(self.step), None,
                  ctypes.byref(self.more), 0, io, self.rotary.desc, None)


@pytest.mark.parametrize("at,strides", [(2, None), (4, None), (0, [(DIM + 8) * HQ + 2, DIM + 8]),
                                        (0, [(DIM + 8) * HQ, DIM + 7])])
def test_out(at, strides):
    c = Call()
    c.out_at += at
    c.out_strides = strides or c.out_strides
    with pytest.raises(_lib.KunserveError, match="out 8-byte aligned") as e:
        c.run()
    assert e.value.code == _lib.EINVAL


def test_workspace():
    c = Call()
    c.step.workspace_bytes -= 1
    with pytest.raises(_lib.KunserveError, match="bytes") as e:
        c.run()
    assert e.value.code == _lib.ENOSPC
    c.step.workspace_bytes += 1
    c.step.workspace_dev += 8
    with pytest.raises(_lib.KunserveError, match="workspace must be 16-byte aligned") as e:
        c.run()
    assert e.value.code == _lib.EINVAL


@pytest.mark.parametrize("field,value,why", [
    ("head_dim", 128, "head_dim 128"), ("page_size", 32, "pages of 32"), ("num_qo_heads", 8, "8 query heads"),
    ("num_kv_heads", 4, "on 4"), ("num_seqs", 3, "3 rows"), ("columns", 48, "48 columns")])
def test_plan(field, value, why):
    c = Call()
    setattr(c.more.tree_info, field, value)
    with pytest.raises(_lib.KunserveError, match=why) as e:
        c.run()
    assert e.value.code == _lib.EINVAL


def test_null_plan():
    c = Call()
    c.more.tree_plan_dev = None
    with pytest.raises(_lib.KunserveError, match="null plan") as e:
        c.run()
    assert e.value.code == _lib.EINVAL
