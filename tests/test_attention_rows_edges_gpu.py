"""Tiles of query rows at the edges of what a call may hold."""
import math

import pytest
import torch

from cache8_cases import Step, check
from test_shared_prefix_gpu import FORMS, shared

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("form,act", FORMS)
@pytest.mark.parametrize("dim", [64, 128, 40])
@pytest.mark.parametrize("far", [2 ** 31 - 1, 2 ** 31 - 2])
def test_the_last_position_there_is(form, act, dim, far):
    """A member far past the block table sees the shared keys like the others."""
    step = Step([(40, 1), (47, 1), (44, 1)], 4, 2, dim, form, act, 16, seed=dim, shared=[([0, 1, 2], 32)])
    step.positions[1] = far
    check(step, shared(step, [[0, 1, 2]], [32]))
    assert int(step.status) == 1


@pytest.mark.parametrize("form,act,dim", [("int8", "bf16", 64), ("e4m3", "bf16", 128), ("int8", "f32", 64), ("e4m3", "f32", 40)])
@pytest.mark.parametrize("window", [0, 30])
def test_portions_that_end_in_padding(form, act, dim, window):
    """Tokens of a portion that are padding need no page, wherever they would stand."""
    from swifttransformer_b200 import ops
    step = Step([(20, 90), (0, 70)], 2, 2, dim, form, act, 16, seed=dim)
    for t in [*range(50, 90), *range(90 + 64, 160)]:
        step.pos_list[t], step.positions[t] = -1, -1
    s = step.slots.tolist()
    step.table[s[0], 70 // 16 + 1:] = -1                           # keys 0 .. 69 are there
    step.table[s[1], 4:] = -1
    plan = ops.portion_plan([90, 70], [20, 0], 2, 2, window, "cuda")
    got = ops.attention_cache8_tiles(step.q, step.pool, step.scales, step.layer, step.out(), plan, step.positions, step.slots, step.table, 2,
                                     step.scale, window, step.status)
    check(step, got, window=window)
    assert int(step.status) == 0


@pytest.mark.parametrize("form,act,dim", [("int8", "bf16", 64), ("int8", "f32", 64), ("e4m3", "f32", 40), ("int8", "bf16", 13)])
def test_a_row_that_is_not_finite_and_weighs_next_to_nothing(form, act, dim):
    """A key that a query sees reaches it, however small its weight: a product of NaN is NaN."""
    from swifttransformer_b200 import ops
    step = Step([(0, 40)], 2, 2, dim, form, act, 16, seed=2)
    pages = step.table[int(step.slots[0])].long()
    step.q[:] = 0.0
    step.q[:, 0] = step.q[:, dim] = 1.0
    raw = step.pool.view(torch.int8)
    one = int(torch.ones(1).to(step.pool.dtype).view(torch.int8))
    raw[pages, step.layer, 0] = one                                 # scores: scale times the key's row scale
    step.scales[pages, step.layer, 0] = 1.0
    step.scales[pages[0], step.layer, 0, :, 3] = 4000.0             # from key 3 on a score 300 and more above the others
    step.scales[pages[1], step.layer, 1, 0, 4] = math.nan           # key 20, head 0: its values
    plan = ops.portion_plan([40], [0], 2, 2, 0, "cuda")
    got = ops.attention_cache8_tiles(step.q, step.pool, step.scales, step.layer, step.out(), plan, step.positions, step.slots, step.table, 2,
                                     step.scale, 0, step.status)
    assert torch.isnan(got[20:, :dim]).all() and torch.isfinite(got[:20, :dim]).all() and torch.isfinite(got[:, dim:]).all()
