"""Orthogonal factors of matrices with numbers that are none: a matrix with a NaN or an infinity becomes NaN altogether, whatever the steps,
and those beside it come out as without it."""
import numpy as np
import pytest

from autograd_b200 import _native as N
from gpu_util import check_clean_status, env
from oracle import heads_and_updates as R
from test_gpu_muon import PRECISIONS, Matrices, gradient

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
