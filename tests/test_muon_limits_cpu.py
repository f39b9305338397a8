"""The range in which the header lets coefficients move singular values: what a kernel keeps between products is finite inside it, and the
limit on s^2 + b / 2c is one that s and a + b s^2 + c s^4 do not imply."""
import os
import re

import numpy as np
import pytest

from oracle import heads_and_updates as R

# coefficients of the steps, all numbers of the header's list below 15, the largest of them near it
EDGES = [[(3.85, 0, 0), (0.2, 0, 0.01)], [(3.0, 0, 0), (0.2, 0.236, 0.02)], [(14.9, 0, 0)], [(14.0, -16.0, 1.0)], [(1.0, 13.9, 0)],
         [(1.2, 0, 0), (9.5, -8.0, 0.5), (1.0, -1.0, 0.5)]]


def kept_numbers(s, steps):
    for a, b, c in steps:
        yield abs(s)
        if c:
            yield abs(s * s + b / (2 * c))
        yield abs(a + b * s * s + c * s ** 4)
        s = s * (a + b * s * s + c * s ** 4)
    yield abs(s)


@pytest.mark.parametrize("bits", [22, 11])
@pytest.mark.parametrize("steps", EDGES, ids=lambda s: str(len(s)))
def test_inside_the_range_all_is_finite(steps, bits):
    most = max(kept_numbers(1.0, steps))
    assert most < 15
    ref, error = R.factor_error(np.float64([[0.5]]), steps, len(steps), 1e-7, bits)
    assert np.isfinite(error) and error <= 0.1 * np.abs(ref).max() + 0.1


def test_the_square_has_a_limit_of_its_own():
    steps = [(4.05, 0, 0), (0.2, 0, 0.01)]
    with np.errstate(over="ignore", invalid="ignore"):
        ref, error = R.factor_error(np.float64([[0.5]]), steps, 2, 1e-7, 22)
    assert abs(ref[0, 0]) < 15 and np.isnan(error)
    over = [x for x in kept_numbers(1.0, steps) if x >= 15]
    assert over == [4.05 ** 2]
    header = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "autograd_b200.h")).read()
    assert re.search(r"\|s\^2 \+ b / 2c\|", header), "the limit is not in the header"
