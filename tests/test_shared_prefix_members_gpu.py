"""Shared prefixes whose members have not the same keys of them: which table a key is found by, and which keys are not asked for."""
import math

import pytest
import torch

from cache8_cases import Step, check
from test_shared_prefix_gpu import FORMS, shared

pytestmark = pytest.mark.gpu


def release(step, window, page_size=16):
    """Every request gives back the pages that lie before its own token's window."""
    for (before, _), slot in zip(step.requests, step.slots.tolist()):
        step.table[slot, :max(0, before - window + 1) // page_size] = -1


def same_keys(step, whole, others, prefix, page_size=16):
    """The first `prefix` keys and values of request `whole`, as far as they reach, are those of the others, in their pages too."""
    pool = step.pool.view(torch.int8) if step.scales is not None else step.pool
    src = step.table[int(step.slots[whole])].long()
    for r in others:
        n = min(sum(step.requests[r]), prefix)
        step.k[r][:, :n], step.v[r][:, :n] = step.k[whole][:, :n], step.v[whole][:, :n]
        dst = step.table[int(step.slots[r])].long()
        for j in range(-(-n // page_size)):
            live = min(page_size, n - page_size * j)
            pool[dst[j], :, :, :, :live] = pool[src[j], :, :, :, :live]
            if step.scales is not None:
                step.scales[dst[j], :, :, :, :live] = step.scales[src[j], :, :, :, :live]


@pytest.mark.parametrize("form,act", FORMS)
@pytest.mark.parametrize("dim", [64, 128, 24])
@pytest.mark.parametrize("order", [[0, 1, 2, 3, 4, 5, 6, 7], [7, 6, 1, 0, 5, 4, 3, 2], [1, 5, 0, 2, 3, 4, 6, 7]])
def test_members_in_any_order(form, act, dim, order):
    """Members that stand inside the shared keys, whose tables end there, before those that have them all."""
    step = Step([(100, 1), (3, 1), (126, 4), (0, 1)], 4, 2, dim, form, act, 16, seed=dim, pad=1)
    same_keys(step, 2, (0, 1, 3), 128)
    check(step, shared(step, [order], [128]))
    assert int(step.status) == 0


@pytest.mark.parametrize("form,act", FORMS)
@pytest.mark.parametrize("window", [1, 20, 100, 400])
@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 64), (2, 2, 128), (3, 1, 40)])
def test_pages_before_the_windows_are_released(form, act, window, heads, kv, dim):
    """Every member has given back what lies before its own window; one that is further ahead, and stands first, has not what others need."""
    prefix = 640
    at = [900, 650, 640, 700, 641, 660, 655, 800]
    step = Step([(p, 1) for p in at], heads, kv, dim, form, act, 16, seed=window, shared=[(list(range(8)), prefix)])
    release(step, window)
    check(step, shared(step, [list(range(8))], [prefix], window=window), window=window)
    assert int(step.status) == 0


@pytest.mark.parametrize("form,act", FORMS)
@pytest.mark.parametrize("dim", [64, 128, 40])
@pytest.mark.parametrize("members", [3, 70])
def test_many_members_far_apart(form, act, dim, members):
    """Members all over the shared keys, in no order, each with the pages of its own window: several tiles, several lengths of them."""
    prefix, window = 1500, 90
    at = [(389 * i + 700) % 1600 for i in range(members)]
    step = Step([(p, 1) for p in at], 2, 1, dim, form, act, 16, seed=members, layers=1, layer=0)
    whole = max(range(members), key=lambda r: at[r])
    same_keys(step, whole, [r for r in range(members) if r != whole], prefix)
    check(step, shared(step, [list(range(members))], [prefix]))
    assert int(step.status) == 0
    release(step, window)
    check(step, shared(step, [list(range(members))], [prefix], window=window), window=window)
    assert int(step.status) == 0


@pytest.mark.parametrize("form,act", FORMS)
@pytest.mark.parametrize("dim", [64, 128, 40])
@pytest.mark.parametrize("what", [math.inf, math.nan])
def test_numbers_behind_every_window(form, act, dim, what):
    """Values and keys that are not finite, in rows that no member's window reaches, at its edge and in whole chunks before it."""
    step = Step([(300, 1), (340, 1)], 2, 2, dim, form, act, 16, seed=3, shared=[([0, 1], 290)])
    for r in (0, 1):
        pages = step.table[int(step.slots[r])].long()
        for key in (5, 64, 200, 249, 250):                         # windows of 50: keys 251 and 291 on
            if step.scales is not None:
                step.scales[pages[key // 16], step.layer, :, :, key % 16] = math.nan
            else:
                step.pool[pages[key // 16], step.layer, :, :, key % 16] = what
    check(step, shared(step, [[0, 1]], [290], window=50), window=50)
    assert int(step.status) == 0


@pytest.mark.parametrize("form,act", FORMS)
@pytest.mark.parametrize("dim", [64, 128, 40])
def test_a_prefix_that_nobody_has_reached(form, act, dim):
    """Shared keys behind every member's position belong to no query: they need no page."""
    step = Step([(40, 1), (60, 1), (7, 1)], 4, 2, dim, form, act, 16, seed=4, shared=[([1, 0], 41), ([1, 2], 8)])
    check(step, shared(step, [[0, 1, 2]], [500]))
    assert int(step.status) == 0


def windowed(step, groups, lens, window, starts):
    from swifttransformer_b200 import ops
    plan = ops.shared_prefix_plan(groups, lens, step.heads, step.kv, "cuda", 300, window, starts)

    def call():
        return ops.attention_shared_prefix(step.q, step.pool, step.layer, step.out(), plan, step.positions, step.seq, step.slots, step.table,
                                           step.heads, step.scale, window, scales=step.scales, status=step.status)
    return call


@pytest.mark.parametrize("form,act", FORMS)
@pytest.mark.parametrize("window", [1, 20, 100, 400])
@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 64), (2, 2, 128), (3, 1, 40)])
def test_plans_for_a_window(form, act, window, heads, kv, dim):
    """Plans that leave out what their window hides: the same plan again when the tokens have moved on, groups of which nothing shared is
    seen, and one that shares nothing."""
    at = [700, 650, 640, 690, 900, 910, 12]
    step = Step([(p, 1) for p in at], heads, kv, dim, form, act, 16, seed=window, shared=[([0, 1, 2, 3], 640), ([4, 5], 500)])
    call = windowed(step, [[0, 1, 2, 3], [4, 5], [6]], [640, 500, 0], window, [640, 900, 0])
    for positions in ([680, 645, 640, 690, 900, 901, 12], at):
        step.pos_list = list(positions)
        step.positions.copy_(torch.tensor(positions, dtype=torch.int32))
        if positions is at:
            release(step, window)
        check(step, call(), window=window)
        assert int(step.status) == 0


@pytest.mark.parametrize("form,act", [("bf16", "bf16"), ("int8", "f32"), ("f32", "f32")])
@pytest.mark.parametrize("dim", [64, 40])
def test_a_token_before_the_plans_start(form, act, dim):
    step = Step([(700, 1), (640, 1)], 2, 2, dim, form, act, 16, seed=1, shared=[([0, 1], 640)])
    call = windowed(step, [[0, 1]], [640], 100, [640])
    check(step, call(), window=100)
    assert int(step.status) == 0
    step.positions[1] = 500
    got = call()
    check(step, got, window=100, rows=[0])
    assert int(step.status) == 1
