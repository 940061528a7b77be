"""rotary_append_kv refuses what its launch would read as an index array without its
being one."""
import numpy as np
import pytest
import torch

from kunserve_amd import KVPool, PageTable, Rotary, _lib, rotary_append_kv

CPU = torch.device("cpu")


@pytest.mark.parametrize("bad", [
    lambda qi: qi.long(), lambda qi: qi[:2], lambda qi: qi.float(),
    lambda qi: torch.stack([qi, qi], 1)[:, 0], lambda qi: qi.to("meta"),
    lambda qi: qi.reshape(1, 3)])
def test_q_indptr(monkeypatch, bad):
    def no_call(name, *args):
        raise AssertionError(f"{name} was called")

    pool = KVPool.allocate(8, 1, 2, 16, 64, CPU)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: None)   # as the pool's index here
    table = PageTable(np.array([0, 1, 2]), np.array([3, 4]), np.array([5, 6]), CPU, upload=False)
    q, k = (torch.zeros((2, h, 64), dtype=torch.float16) for h in (4, 2))
    qi = torch.tensor([0, 1, 2], dtype=torch.int32)
    monkeypatch.setattr(_lib, "call", no_call)
    with pytest.raises(ValueError, match="q_indptr"):
        rotary_append_kv(pool, 0, table, bad(qi), q, k, k, Rotary(32, device="cpu"))
