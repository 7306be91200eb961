"""Calls with nothing to do: no tokens, no requests, groups without members, requests without new tokens."""
import pytest
import torch

from cache8_cases import Step, check
from test_cache8_gpu import ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("form,act", [("int8", "bf16"), ("e4m3", "f32")])
def test_no_tokens(form, act):
    from swifttransformer_b200 import ops
    step = Step([(40, 1), (20, 1)], 4, 2, 64, form, act, 16, seed=1)
    none, q = ints([]), step.q[:0]
    pool = step.pool.view(torch.int8).clone()
    ops.qkv_to_cache8(q.new_empty((0, 512)), None, q.new_empty((0, 256)), step.pool, step.scales, 1, none, none, step.slots, step.table, 4, 2, 64)
    assert ops.cache8_rows(step.pool, step.scales, 1, q.new_empty((0, 256)), none, none, step.slots, step.table).shape == (0, 256)
    args = (none, none, step.slots, step.table, 4, 0.1)
    assert ops.attention_cache8_single(q, step.pool, step.scales, 1, q.new_empty((0, 256)), None, 0, *args).shape == (0, 256)
    for plan in (ops.portion_plan([], [], 4, 2), ops.portion_plan([0, 0], [5, 0], 4, 2)):
        got = ops.attention_cache8_tiles(q, step.pool, step.scales, 1, q.new_empty((0, 256)), plan, none, step.slots, step.table, 4, 0.1)
        assert got.shape == (0, 256)
    for plan in (ops.shared_prefix_plan([], [], 4, 2), ops.shared_prefix_plan([[], []], [64, 0], 4, 2)):
        got = ops.attention_shared_prefix(q, step.pool, 1, q.new_empty((0, 256)), plan, *args, scales=step.scales)
        assert got.shape == (0, 256)
    torch.cuda.synchronize()
    assert torch.equal(step.pool.view(torch.int8), pool) and ops.kernel_status("cuda") == 0


@pytest.mark.parametrize("form,act", [("int8", "bf16"), ("e4m3", "f32")])
def test_nothing_among_something(form, act):
    """Requests without new tokens between others, an empty group, and tokens that no plan names."""
    from swifttransformer_b200 import ops
    step = Step([(10, 3), (4, 0), (0, 130), (7, 0)], 4, 2, 64, form, act, 16, seed=1)
    plan = ops.portion_plan([3, 0, 130, 0], [10, 4, 0, 7], 4, 2)
    check(step, ops.attention_cache8_tiles(step.q, step.pool, step.scales, step.layer, step.out(), plan, step.positions, step.slots, step.table, 4,
                                           step.scale, status=step.status))
    plan = ops.shared_prefix_plan([[], [0, 1, 2], []], [500, 8, 0], 4, 2)
    got = ops.attention_shared_prefix(step.q, step.pool, step.layer, step.out(), plan, step.positions, step.seq, step.slots, step.table, 4, step.scale,
                                      scales=step.scales, status=step.status)
    check(step, got, rows=[0, 1, 2])
    assert float(got[3:].min()) == 77.0 == float(got[3:].max()) and int(step.status) == 0
