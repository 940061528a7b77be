"""Rotary positions are whole numbers: others are refused, not cut."""
import numpy as np
import pytest
import torch

from kunserve_amd import AttentionStep, KVPool


@pytest.mark.parametrize("bad,what", [([1.5], "whole"), (np.array([3.0]), "whole"), (["3"], "whole"),
                                      ([1, 2], "1 rows"), ([[1]], "1 rows"), ([-1], "2\\^31"),
                                      ([2**31], "2\\^31"), (np.array([2**40]), "2\\^31")])
def test_refusals(bad, what):
    pool = KVPool.allocate(2, 1, 2, 16, 64, torch.device("cpu"))
    with pytest.raises(ValueError, match=what):
        AttentionStep(pool, 4, [1], [5], [0], [[0]], rope_positions=bad)
