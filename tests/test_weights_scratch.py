"""A step's scratch for scores is bounded: decode rows beyond score_bytes take
add_weights' passes over K."""
import numpy as np
import pytest
import torch

from kunserve_amd import KVPool, KVWeights, WeightsPlan

CPU = torch.device("cpu")


def plan(kv, hq, score_bytes=None, decodes=None):
    pool = KVPool.allocate(1, 1, 1, 16, 64, CPU)
    w = KVWeights(pool) if score_bytes is None else KVWeights(pool, score_bytes=score_bytes)
    n = len(kv)
    return w.plan(np.arange(n + 1), kv, hq, 16, [True] * n if decodes is None else decodes)


def test_the_default_is_bounded():
    """512 rows of 32768 tokens at 64 heads: 4.3 GB in scores."""
    p = plan([32768] * 512, 64)
    assert p.info.score_tokens * 64 * 4 <= 256 << 20
    # the other rows: 129 statistics of 64 columns each
    assert p.workspace_bytes() <= (256 << 20) + 512 * (129 * 64 * 8 + 64 * 4) + 16
    assert plan([8192] * 128, 64).info.num_items == 0      # 256 MiB: all in scores


@pytest.mark.parametrize("limit,rows", [(0, 0), (4 * 8 * 300, 1), (4 * 8 * 300 - 1, 0),
                                        (4 * 8 * 1000, 2), (4 * 8 * 1301, 3), (1 << 40, 3)])
def test_rows_within_the_limit(limit, rows):
    kv = [300, 700, 301]
    p = plan(kv, 8, limit)
    info = p.info
    assert info.num_score_rows == 3
    at = p.plan_host[info.plan_ints - 3:]
    np.testing.assert_array_equal(at, [0, 300, 1000][:rows] + [-1] * (3 - rows))
    items = p.plan_host[:4 * info.num_items].reshape(-1, 4)
    assert sorted(set(items[:, 0].tolist())) == list(range(rows, 3))
    assert info.score_tokens == sum(kv[:rows])


def test_prompt_rows_do_not_count():
    p = plan([300, 700, 301], 8, 4 * 8 * 700, [False, True, True])
    info = p.info
    np.testing.assert_array_equal(p.plan_host[info.plan_ints - 2:], [0, -1])
    items = p.plan_host[:4 * info.num_items].reshape(-1, 4)
    assert set(items[:, 0].tolist()) == {0, 2}


def test_marks():
    with pytest.raises(RuntimeError, match="decodes 2 tokens"):
        WeightsPlan([0, 2], [40], 4, 8, CPU, upload=False, decodes=[2])


def test_marks_of_other_rows():
    with pytest.raises(ValueError, match="3 rows but"):
        plan([300, 700, 301], 8, 0, [True])
    assert plan([], 8, 0).workspace_bytes() == 0
