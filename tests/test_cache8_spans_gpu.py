"""Single tokens whose windows lie past the block table, near the last position there is."""
import pytest

from cache8_cases import Step, check
from test_cache8_gpu import single
from test_shared_prefix_gpu import shared

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("form,act,dim", [("int8", "bf16", 64), ("e4m3", "f32", 128), ("int8", "f32", 24), ("e4m3", "bf16", 13)])
@pytest.mark.parametrize("window", [1, 70, 100, 700])
@pytest.mark.parametrize("far", [2 ** 31 - 1, 2 ** 31 - 200, 2 ** 30])
def test_windows_past_the_table(form, act, dim, window, far):
    """Such a token has no key and gets zeros, whatever the number of warps that look for one."""
    step = Step([(31, 1), (1500, 1), (20, 1)], 4, 2, dim, form, act, 16, seed=dim)
    step.positions[1] = far
    got = single(step, window=window)
    check(step, got, window=window, rows=[0, 2])
    assert float(got[1].abs().max()) == 0.0 and int(step.status) == 1


@pytest.mark.parametrize("form,act,dim", [("bf16", "bf16", 64), ("f32", "f32", 64), ("int8", "bf16", 128), ("e4m3", "f32", 24)])
@pytest.mark.parametrize("window", [0, 70])
def test_own_keys_past_the_table(form, act, dim, window):
    """Tokens behind shared keys, one of them with a window that lies past the table."""
    step = Step([(60, 1), (63, 1), (50, 1)], 4, 2, dim, form, act, 16, seed=dim, shared=[([0, 1, 2], 48)])
    if window:
        step.positions[1] = 2 ** 31 - 1
        got = shared(step, [[0, 1, 2]], [48], window=window)
        check(step, got, window=window, rows=[0, 2])
        assert float(got[1].abs().max()) == 0.0 and int(step.status) == 1
    else:
        check(step, shared(step, [[0], [1, 2]], [0, 48]))
        assert int(step.status) == 0
