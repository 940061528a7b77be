"""What KVWeights.clear and steps that learn nothing refuse before they reach a
device."""
import numpy as np
import pytest
import torch

from kunserve_amd import AttentionStep, KVPool, KVWeights, PageTable, _lib

CPU = torch.device("cpu")


def test_refusals(monkeypatch):
    pool = KVPool.allocate(12, 2, 2, 16, 64, CPU)
    w = KVWeights(pool)
    with pytest.raises(ValueError, match="with weights"):
        AttentionStep(pool, 4, [1], [5], [0], [[0]], learn=False)
    with pytest.raises(ValueError, match="not those"):
        AttentionStep(KVPool.allocate(13, 2, 2, 16, 64, CPU), 4, [1], [5], [0], [[0]], weights=w,
                      learn=False)
    table = PageTable(np.array([0, 1]), np.array([3]), np.array([5]), CPU, upload=False)
    for bad in (torch.tensor([0, 1]), torch.tensor([0, 1, 2], dtype=torch.int32)):
        with pytest.raises(ValueError, match="q_indptr"):
            w.clear(pool, table, bad, 1)
    table.bind([torch.from_numpy(a) for a in table.host_arrays()])
    monkeypatch.setattr("kunserve_amd.cache_weights._stream_ptr", lambda device: 0)
    qi = torch.tensor([0, 1], dtype=torch.int32)
    with pytest.raises(_lib.KunserveError, match="num_tokens"):
        w.clear(pool, table, qi, -1)
    w.clear(pool, table, qi, 0)      # nothing to launch
