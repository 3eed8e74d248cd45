"""That tests with exact scores tell in how many bits softmax weights are held: weights of other roundings, made in numpy."""
import numpy as np
import pytest

from paged_levels import FP16, TWO_FP16, Levels, cancelling, far_below, odd_weights


def one(x):
    return x.astype(np.float16).astype(np.float64)


def two(x):
    return one(x) + one(x - one(x))


@pytest.mark.parametrize("n", [64, 700, 5000])
def test_weights_in_one_fp16_number_are_told_from_two(n):
    q0 = odd_weights(6)
    w = Levels(*cancelling(n, q0))
    q = w.levels(np.tile(q0, 2))
    right, within_two, _, _ = w.attention_within(q, TWO_FP16)
    _, within_one, _, _ = w.attention_within(q, FP16)
    off_one, off_two = (np.abs(w.attention_within(q, FP16, f)[0] - right) for f in (one, two))
    if n < 5000:  # (there the sums' own rounding is as large)
        assert np.all((off_one > 2 * within_two).any(-1))  # of every head
    assert np.all(off_one <= within_one) and np.all(off_two <= within_two / 4)


@pytest.mark.parametrize("depth", [15.87, 18.4, 20.6, 25.2])
def test_weights_beside_a_largest_one_of_1_are_told_from_those_with_room(depth):
    w = Levels(*far_below(1000, depth))
    q = w.levels(16)
    for rounded, weight in ((one, FP16), (two, TWO_FP16)):
        right, within, _, _ = w.attention_within(q, weight)
        assert np.all(np.abs(w.attention_within(q, weight, rounded)[0] - right) <= within / 2)
        low = w.attention_within(q, weight, lambda x: 128 * rounded(x / 128))[0]
        assert np.any(np.abs(low - right) > within)
