"""Weights of steps whose decode rows do not all leave scores, against 64 bits."""
import pytest
import torch

from kunserve_amd import AttentionStep, KVWeights
from test_gpu_weights import build, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [0, 1, 3])
@pytest.mark.parametrize("hq,hkv,d,dtype", [(4, 4, 64, torch.float16), (8, 2, 64, torch.bfloat16),
                                            (4, 2, 128, torch.bfloat16), (8, 2, 128, torch.float16),
                                            (34, 2, 128, torch.bfloat16),
                                            (8, 2, 256, torch.float16), (4, 4, 256, torch.bfloat16)])
def test_rows_with_and_without_scores(device, hq, hkv, d, dtype, rows):
    """Decode rows in one and in several partitions, beside a prompt's chunk."""
    q_lens, kvs, flags = [1, 1, 20, 1, 1], [300, 1, 90, 700, 1500], [0, 0, 1, 0, 0]
    pool, tables, q, k, v, w = build(device, q_lens, kvs, hq, hkv, 16, d, dtype, 1, hq + d)
    limit = 4 * hq * [0, 300, 1001][min(rows, 2)]
    w = KVWeights(pool, w.w, score_bytes=limit)
    before = w.w.clone()
    step = AttentionStep(pool, hq, q_lens, [300, 1, 70, 700, 1500], flags, tables, weights=w,
                         window=8)
    assert step._weights_plan.info.score_tokens == [0, 300, 1001][min(rows, 2)]
    plain = AttentionStep(pool, hq, q_lens, [300, 1, 70, 700, 1500], flags, tables)
    want = plain.run(0, q, k, v)
    out = step.run(0, q, k, v)
    assert torch.equal(out.view(torch.int16), want.view(torch.int16))
    check(pool, tables, q, w, before, out, q_lens, kvs, 0, 8)
