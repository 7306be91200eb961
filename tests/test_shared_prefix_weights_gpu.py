"""Shared prefixes over bfloat16 caches: the weights are not rounded to eight bits."""
import pytest

from cache8_cases import Step
from test_shared_prefix_gpu import shared

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kv,dim", [(4, 4, 64), (8, 2, 64), (4, 4, 128), (8, 2, 128), (6, 2, 80), (2, 1, 96), (3, 3, 48)])
@pytest.mark.parametrize("prefix", [500, 2500])
def test_weights_in_two_numbers(heads, kv, dim, prefix):
    """`Step.expected` allows a weight 2^-8 of itself over bfloat16 caches.  In two bfloat16 numbers it is off by half a step of the second,
    2^-9 of what the first leaves, at most 2^-9 of the weight: 2^-18; 2^-17 is allowed.  With A = sum w |v|, the bounds for the
    two forms differ by 2^-8 A."""
    step = Step([(prefix + 7 * i % 60, 1) for i in range(20)], heads, kv, dim, "bf16", "bf16", 16, seed=dim, shared=[(list(range(20)), prefix)],
                layers=1, layer=0)
    got = shared(step, [list(range(20))], [prefix], max_own=60).double()
    want, wide = step.expected()
    step.form = "f32"
    same, narrow = step.expected()
    assert bool((same == want).all())
    tol = narrow + (wide - narrow) * 2.0 ** (8 - 17)
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), float(((got - want).abs() / tol).max()))
