"""Which keys a single token reads, at the ends of what an int holds (no GPU)."""
import pytest

from swifttransformer_b200 import ops

LAST = 2 ** 31 - 1
REACH = 0x7fff0000                  # the most keys that a block table stands for


def span(pos, window, shared, reach):
    both = ops.lib().st_attention_single8_span(pos, window, shared, reach)
    return both & 0xffffffff, both >> 32


@pytest.mark.parametrize("reach", [1, 8, 160, 80000, REACH])
@pytest.mark.parametrize("window", [0, 1, 3, 70, 4096, 2 ** 30, LAST])
@pytest.mark.parametrize("shared", [0, 33, 100000, 2 ** 31 - 2 ** 17])
def test_the_keys_of_a_token(reach, window, shared):
    for pos in (-1, 0, 1, 7, 95, 159, 160, 200, 79999, 100500, 2 ** 30, REACH - 1, REACH, LAST - 1, LAST):
        lo, hi = span(pos, window, shared, reach)
        first = max(pos - window + 1 if window else 0, shared, 0)
        end = min(pos + 1, reach)
        if first < end:
            assert (lo, hi) == (first, end)
        else:
            assert lo == hi == end                      # none
        # keys that warps form ahead of the last run: 8 blocks of 16 warps, five turns, 32 keys
        assert 0 <= lo <= hi <= reach and lo + 5 * 8 * 16 * 32 <= LAST
