"""Orthogonal factors of matrices with numbers that are none: a matrix with a NaN or an infinity becomes NaN altogether, whatever the steps,
and those beside it come out as without it; and coefficients at the limits of what is kept between products."""
import numpy as np
import pytest

from gpu_util import check_clean_status, env
from test_gpu_muon import BITS, PRECISIONS, Matrices, close, gradient
from test_muon_limits_cpu import EDGES

pytestmark = pytest.mark.gpu

# one launch on one CTA and on a cluster; single CTAs, contractions shared by a cluster, pairs whose tiles reach into the matrix behind (384 rows)
SHAPES = [(5, 70, 90), (5, 30, 700), (5, 150, 140), (5, 140, 1500), (24, 270, 300)]


@PRECISIONS
@pytest.mark.parametrize("steps", [0, 1, 5])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_nan_and_infinity_fill_their_matrix_and_no_other(shape, steps, precision):
    ctx, alloc, be = env()
    rng = np.random.default_rng(sum(shape) + steps)
    g = gradient(rng, *shape)
    b = Matrices(np.ones_like(g))
    a = Matrices(g)
    be.orthogonalise(a.argument, b.argument, steps=steps, precision=precision)
    clean = b.read()
    a.free()
    bad = g.copy()
    bad[1, shape[1] - 1, 3] = np.nan
    bad[2, 0, shape[2] - 1] = np.inf
    bad[4, 5, 0], bad[4, 6, 0] = -np.inf, np.inf
    a = Matrices(bad)
    be.orthogonalise(a.argument, b.argument, steps=steps, precision=precision)
    got = b.read()
    for i in range(shape[0]):
        if i in (1, 2, 4):
            assert np.isnan(got[i]).all(), i
        else:
            assert np.array_equal(got[i], clean[i]), i
    check_clean_status()
    a.free(), b.free()


@pytest.mark.parametrize("shape", [(3, 70, 90), (3, 150, 140)], ids=lambda s: "x".join(map(str, s)))
def test_a_step_with_an_infinite_gradient(shape):
    """The parameters of that matrix become NaN, its momentum is infinite where the gradient is; the others move as without it."""
    ctx, alloc, be = env()
    rng = np.random.default_rng(3)
    g, m, p = gradient(rng, *shape), gradient(rng, *shape), (0.02 * rng.standard_normal(shape)).astype(np.float32)
    results = []
    for value in (g[1, 2, 3], np.float32(np.inf)):
        g[1, 2, 3] = value
        tp, tg, tm = Matrices(p), Matrices(g), Matrices(m)
        be.muon_step(tp.argument, tg.argument, tm.argument, 0.02)
        results.append((tp.read(), tm.read()))
        for t in (tp, tg, tm):
            t.free()
    (p0, m0), (p1, m1) = results
    assert np.isnan(p1[1]).all() and m1[1, 2, 3] == np.inf
    m1[1, 2, 3] = m0[1, 2, 3]
    assert np.array_equal(m0, m1) and np.array_equal(p0[[0, 2]], p1[[0, 2]])
    check_clean_status()


def one_direction_error(steps, bits):
    """How far the singular value 1 may be off after the steps.

    A product errs by e of itself: two operands by half a step each (2^-23 or 2^-12), and the kernel's factor for what truncation loses on
    average, 3.2e-7 for 128 elements, stays whole where a sum has one term and loses nothing: 2^-20 or 2^-10 in all.  What is stored is rounded by
    half a step.  A = s^2 + h is off by d = e s^2 + r |A|, Q = (a - h^2 c) + c A^2 by 2 |c A| d + e |c| A^2 + r |Q| (of the whole square: where
    h^2 c is large, most of it cancels), s Q by |s| times that, by e |s Q| and by what s was off, times the step's derivative."""
    e, r = (2.0 ** -20, 2.0 ** -23) if bits == 22 else (2.0 ** -10, 2.0 ** -12)
    s, off = 1.0, r
    for a, b, c in steps:
        h = b / (2 * c) if c else 0.0
        if c:
            d = e * s * s + r * abs(s * s + h)
            dq = 2 * abs(c * (s * s + h)) * d + e * abs(c) * (s * s + h) ** 2
        else:
            dq = e * abs(b) * s * s
        q = a + b * s * s + c * s ** 4
        off = abs(a + 3 * b * s * s + 5 * c * s ** 4) * off + abs(s) * (dq + r * abs(q)) + (e + r) * abs(s * q)
        s *= q
    return off


@PRECISIONS
@pytest.mark.parametrize("steps", EDGES, ids=lambda s: str(len(s)))
@pytest.mark.parametrize("shape", [(1, 1, 1), (2, 70, 90), (1, 40, 700), (2, 150, 140), (1, 140, 1500), (24, 270, 300)],
                         ids=lambda s: "x".join(map(str, s)))
def test_singular_values_up_to_the_limits(shape, steps, precision):
    """Matrices of one direction, the singular value of which is 1: one element that has it all (in a corner, beside the padding), and rows
    and columns that share it."""
    ctx, alloc, be = env()
    rng = np.random.default_rng(sum(shape))
    g = np.zeros(shape, np.float32)
    g[:, -1, -1] = 3.0
    if shape[0] > 1:
        g[1] = np.outer(rng.standard_normal(shape[1]), rng.standard_normal(shape[2]))
    a = Matrices(g)
    b = Matrices(np.ones_like(g))
    be.orthogonalise(a.argument, b.argument, steps=len(steps), coefficients=steps, precision=precision)
    got = b.read()
    for i in sorted({0, min(1, shape[0] - 1), shape[0] - 1}):
        close(got[i], g[i], precision, len(steps), steps, more=one_direction_error(steps, BITS[precision]))
    check_clean_status()
    a.free(), b.free()
