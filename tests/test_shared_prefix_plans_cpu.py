"""Plans of shared prefixes with a window, and what they refuse (no GPU)."""
import pytest
import torch

from swifttransformer_b200 import ops
from swifttransformer_b200.ops import KernelError
from test_cache8_cpu import Fake, base, chunks, fake  # noqa: F401


def test_a_plan_for_a_window():
    plan = ops.shared_prefix_plan([[5, 2], [0], [7, 8], [1]], [300, 10, 128, 64], 4, 4, "cpu", 17, 100, [310, 0, 500, 164])
    assert plan.tiles.view(-1, 6).tolist() == [[0, 2, -1, 211, 300, 0], [2, 1, -1, 0, 10, 20], [3, 2, -1, 128, 128, 36], [5, 1, -1, 64, 64, 36]]
    assert plan.info.view(-1, 3).tolist() == [[300, 0, 0], [300, 0, 1], [10, 1, 0], [128, 2, 0], [128, 2, 1], [64, 3, 0]]
    assert plan.window == 100 and plan.total == 36 == 4 * sum(chunks(t) + 3 for t in plan.tiles.view(-1, 6).tolist() if chunks(t))
    long = ops.shared_prefix_plan([list(range(64))], [8000], 32, 32, "cpu", 100, 512, [8000])
    assert long.total * 10 < ops.shared_prefix_plan([list(range(64))], [8000], 32, 32, "cpu", 100).total


@pytest.mark.parametrize("more", [dict(window=-1, starts=[4]), dict(window=5), dict(starts=[4]), dict(window=5, starts=[4, 4]),
                                  dict(window=5, starts=[-1])])
def test_plans_refuse(more):
    with pytest.raises(KernelError):
        ops.shared_prefix_plan([[1]], [4], 4, 4, "cpu", **more)


@pytest.mark.parametrize("window", [0, 4, 6])
def test_calls_refuse_a_plan_for_another_window(fake, window):  # noqa: F811
    a = base(fake, window=window)
    a.pop("items"), a.pop("n_items")
    plan = ops.shared_prefix_plan([[0, 1, 2, 3]], [4], 4, 2, "cpu", 0, 5, [10])
    plan.tiles = fake(plan.tiles)
    with pytest.raises(KernelError, match="window"):
        ops.attention_shared_prefix(**a, plan=plan)


@pytest.mark.parametrize("make", [
    lambda: ops.shared_prefix_plan([[0]], [2 ** 33], 1, 1, "cpu"), lambda: ops.shared_prefix_plan([[0]], [2 ** 31 - 1], 1, 1, "cpu"),
    lambda: ops.shared_prefix_plan([[0]], [2 ** 31], 1, 1, "cpu", 0, 10, [2 ** 31]),
    lambda: ops.shared_prefix_plan([[2 ** 31]], [4], 1, 1, "cpu"), lambda: ops.portion_plan([4], [2 ** 31 - 8], 1, 1, 8, "cpu"),
    lambda: ops.portion_plan([4], [2 ** 32], 1, 1, 8, "cpu"), lambda: ops.portion_plan([1], [2 ** 31 - 2], 1, 1, device="cpu")])
def test_plans_refuse_what_passes_an_int(make):
    with pytest.raises(KernelError):
        make()


def test_the_longest_plans():
    plan = ops.portion_plan([4], [0x7fff0000 - 4], 1, 1, 8, "cpu")
    assert plan.tiles.tolist() == [0, 4, 0, 0x7fff0000 - 11, 0x7fff0000, 0] and plan.total == 4
    assert ops.shared_prefix_plan([[0]], [0x7fff0000], 1, 1, "cpu").total == 0x7fff0000 // 64 + 3
