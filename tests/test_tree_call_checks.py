"""What tree_attention refuses of its caller's tensors before it launches (CPU only)."""
import pytest
import torch

from kunserve_amd import KVPool, PageTable, TreePlan, tree_attention

CPU = torch.device("cpu")


@pytest.fixture
def call():
    pool = KVPool.allocate(4, 1, 2, 16, 64, CPU)
    table = PageTable.from_lists([[0, 1]], [20], pool, upload=False)
    plan = TreePlan(table, [[-1, 0, 0]], 4, 2, 16, CPU, num_cus=256, head_dim=64, part_rounds=1,
                    upload=False)
    assert plan.workspace_bytes() > 0
    table.bind([torch.from_numpy(x) for x in table.host_arrays()])
    plan.bind([torch.from_numpy(x) for x in plan.host_arrays()])
    return pool, table, torch.zeros(3, 4, 64, dtype=torch.float16), plan


def test_workspace_elsewhere(call):
    pool, table, q, plan = call
    with pytest.raises(ValueError, match="workspace is on meta"):
        tree_attention(pool, 0, table, q, plan,
                       workspace=torch.empty(plan.workspace_bytes(), dtype=torch.uint8, device="meta"))


@pytest.mark.parametrize("ws", ["expanded", "every other", "transposed"])
def test_workspace_with_gaps(call, ws):
    """Bytes that it has but not in one piece: the kernel would write past it."""
    pool, table, q, plan = call
    n = plan.workspace_bytes() // 4
    t = {"expanded": torch.empty(1).expand(n), "every other": torch.empty(2 * n)[::2],
         "transposed": torch.empty(4, n).t()}[ws]
    assert t.numel() * 4 >= plan.workspace_bytes()
    with pytest.raises(ValueError, match="workspace .* contiguous"):
        tree_attention(pool, 0, table, q, plan, workspace=t)


def test_plan_and_table_elsewhere(call):
    pool, table, q, plan = call
    at, plan.plan = plan.plan, plan.plan.to("meta")
    with pytest.raises(ValueError, match="plan is on meta"):
        tree_attention(pool, 0, table, q, plan)
    plan.plan = at
    table.bind([torch.from_numpy(x).to("meta") for x in table.host_arrays()])
    with pytest.raises(ValueError, match="table is on meta"):
        tree_attention(pool, 0, table, q, plan)


def test_table_and_plan_that_are_not_bound():
    pool = KVPool.allocate(4, 1, 2, 16, 64, CPU)
    table = PageTable.from_lists([[0, 1]], [20], pool, upload=False)
    plan = TreePlan(table, [[-1, 0, 0]], 4, 2, 16, CPU, num_cus=256, head_dim=64, upload=False)
    q = torch.zeros(3, 4, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="page table used before"):
        tree_attention(pool, 0, table, q, plan)
    table.bind([torch.from_numpy(x) for x in table.host_arrays()])
    with pytest.raises(RuntimeError, match="tree plan used before"):
        tree_attention(pool, 0, table, q, plan)
