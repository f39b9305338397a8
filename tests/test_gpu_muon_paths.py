"""Orthogonal factors on every kind of launch that the sizes lead to, the kind being asserted: products on pairs of CTAs with one tile and
several to a pair, ragged last blocks, blocks below the diagonal read as transposes of three and more blocks to a side; lists of
more matrices than a launch takes, or than the workspace holds; the same bits every time; products as exact as those of fp32 numbers.

Bounds: of some matrices of a list, `close` of test_gpu_muon.py.  The others have numbers of the same distribution, so that the form with
rounded operands errs by about as much: eight times the first one's error and 2^-17 (twice those of `close`) of the norm."""
import numpy as np
import pytest

from autograd_b200 import _native as N
from gpu_util import check_clean_status, env
from oracle import heads_and_updates as R
from test_gpu_muon import BITS, PRECISIONS, Matrices, close, gradient

pytestmark = pytest.mark.gpu

ONE, SINGLE, PAIRS, CLUSTERS = N.AG_NS_ONE_LAUNCH, N.AG_NS_SINGLE, N.AG_NS_PAIRS, N.AG_NS_CLUSTERS


def forms(count, rows, cols):
    ctx = env()[0]
    return tuple(ctx.orthogonalise_form(count, rows, cols, k)[0] for k in range(3))


def all_close(got, g, precision, looked_at, **kw):
    first = None
    if min(g.shape[1:]) > 1000:   # the form with rounded operands takes minutes: three times what the header says of the norm
        looked_at, first = (), (2.0 ** -17 if precision == N.AG_CE_3XTF32 else 2.0 ** -5) + (2.0 ** -8 if kw.get("out") == "bf16" else 0)
    for i in range(len(g)):
        if i in looked_at:
            close(got[i], g[i], precision, **kw)
        if first is None:
            ref, error = R.factor_error(g[i], kw.get("coefficients", R.NEWTON_SCHULZ), kw.get("steps", 5), 1e-7, BITS[precision])
            first = 8 * error / np.linalg.norm(ref) + 2.0 ** -17 + (2.0 ** -7 if kw.get("out") == "bf16" else 0)
        else:
            ref = R.factor(g[i], steps=kw.get("steps", 5))
        assert np.linalg.norm(got[i] - ref) <= first * np.linalg.norm(ref), i


# matrices and what computes X X^T, its square and the next X on a GPU of 148 SMs
PATHS = [((6, 384, 1536), (CLUSTERS, SINGLE, PAIRS)), ((9, 384, 2048), (CLUSTERS, SINGLE, PAIRS)), ((16, 384, 1536), (SINGLE, SINGLE, PAIRS)),
         ((20, 600, 700), (PAIRS, PAIRS, PAIRS)), ((24, 270, 300), (PAIRS, PAIRS, SINGLE)), ((10, 1400, 300), (CLUSTERS, SINGLE, PAIRS)),
         ((1, 200, 3000), (CLUSTERS, SINGLE, SINGLE)), ((3, 1300, 1400), (PAIRS, PAIRS, PAIRS)), ((8, 1100, 1030), (PAIRS, PAIRS, PAIRS)),
         ((5, 1100, 1030), (SINGLE, SINGLE, PAIRS)), ((2, 130, 140), (SINGLE, SINGLE, SINGLE)), ((2, 64, 256), (ONE, ONE, ONE))]


@PRECISIONS
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape,path", PATHS, ids=lambda v: "x".join(map(str, v)))
def test_every_kind_of_launch(shape, path, dtype, precision):
    ctx, alloc, be = env()
    assert forms(*shape) == path
    g = gradient(np.random.default_rng(sum(shape)), *shape, dtype)
    a, b = Matrices(g, dtype), Matrices(np.full(shape, 2.0, np.float32), dtype)
    be.orthogonalise(a.argument, b.argument, precision=precision)
    all_close(b.read(), g, precision, (0, shape[0] - 1), out=dtype)
    assert np.array_equal(a.read(), g)
    check_clean_status()
    a.free(), b.free()


@PRECISIONS
def test_a_matrix_twice_and_more_matrices_than_a_launch_takes(precision):
    """97 on the general path are 49 and 48 of them; the last one is the fourth again."""
    ctx, alloc, be = env()
    form, batch = ctx.orthogonalise_form(97, 130, 140, 2)
    assert form != ONE and batch == 49
    g = gradient(np.random.default_rng(1), 97, 130, 140)
    g[96] = g[3]
    a, b = Matrices(g, apart=True), Matrices(np.zeros_like(g), apart=True)
    be.orthogonalise(a.tensors[:96] + [a.tensors[3]], b.tensors, precision=precision)
    got = b.read()
    all_close(got, g, precision, (0, 48, 49, 96))
    assert np.array_equal(got[96], got[3])
    check_clean_status()
    a.free(), b.free()


@PRECISIONS
def test_steps_on_more_matrices_than_a_launch_takes(precision):
    ctx, alloc, be = env()
    shape, lr = (97, 130, 140), 0.02
    rng = np.random.default_rng(2)
    g, m, p = gradient(rng, *shape, "bf16"), gradient(rng, *shape), (0.02 * rng.standard_normal(shape)).astype(np.float32)
    tp, tg, tm = Matrices(p, apart=True), Matrices(g, "bf16", apart=True), Matrices(m, apart=True)
    be.muon_step(tp.tensors, tg.tensors, tm.tensors, lr, weight_decay=0.1, precision=precision)
    got_p, got_m = tp.read(), tm.read()
    scale, u = 0.2 * np.sqrt(140), 2.0 ** -24
    moved = (p * (1 - lr * 0.1) - got_p) / (lr * scale)   # the factors, and the roundings of p over lr scale (0.047): 2^-18.6 of |p|
    for i in range(97):
        _, ref_m, of = R.muon(p[i], g[i], m[i], lr, weight_decay=0.1, scale=scale)
        assert (np.abs(got_m[i] - ref_m) <= 4 * u * (np.abs(m[i]) + np.abs(g[i]))).all()
        more = 2 * u * np.linalg.norm(p[i]) / (lr * scale) + 4 * u * np.linalg.norm(moved[i])
        of = g[i] + 0.95 * (got_m[i] - g[i])
        if i in (0, 48, 49, 96):
            close(moved[i], of, precision, more=more)
        else:
            ref = R.factor(of)
            assert np.linalg.norm(moved[i] - ref) <= (2.0 ** -16 if precision == N.AG_CE_3XTF32 else 2.0 ** -6) * np.linalg.norm(ref) + more, i
    check_clean_status()
    for t in (tp, tg, tm):
        t.free()


@PRECISIONS
def test_more_matrices_than_the_workspace_holds(precision):
    """Five of 2000 x 6000 are three and two: the second batch finds the first one's numbers in the workspace."""
    ctx, alloc, be = env()
    assert ctx.orthogonalise_form(5, 2000, 6000, 2) == (PAIRS, 3)
    g = gradient(np.random.default_rng(3), 5, 2000, 6000)
    a = Matrices(g, apart=True)
    be.orthogonalise(a.tensors, a.tensors, steps=1, precision=precision)   # in their places
    got = a.read()
    # one step, on 64 bits: no form with rounded operands of this size; 22 bits through three products, or 11 (each within 2^-10 of the norm)
    for i in range(5):
        ref = R.factor(g[i], steps=1)
        assert np.linalg.norm(got[i] - ref) <= (2.0 ** -18 if precision == N.AG_CE_3XTF32 else 2.0 ** -8) * np.linalg.norm(ref), i
    check_clean_status()
    a.free()


@PRECISIONS
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(4, 1500, 3000), (20, 600, 700), (3, 1001, 340), (1, 200, 3000), (2, 64, 256), (1, 128, 4000)],
                         ids=lambda s: "x".join(map(str, s)))
def test_the_same_bits_every_time(shape, dtype, precision):
    """Five calls, with other work between them and other numbers in the workspace."""
    ctx, alloc, be = env()
    rng = np.random.default_rng(sum(shape))
    a, b = Matrices(gradient(rng, *shape, dtype), dtype), Matrices(np.zeros(shape, np.float32), dtype)
    other = Matrices(rng.standard_normal((3, 300, 900)).astype(np.float32))
    first = None
    for _ in range(5):
        be.orthogonalise(a.argument, b.argument, precision=precision)
        got = b.read()
        assert first is None or np.array_equal(got, first)
        first = got
        be.orthogonalise(other.argument, other.argument)
    check_clean_status()
    a.free(), b.free(), other.free()


def fp32_factor(u):
    x = np.asarray(u, np.float32)
    x = x / np.float32(max(np.sqrt(np.sum(x.astype(np.float64) ** 2)), 1e-7))
    x = np.ascontiguousarray(x.T) if x.shape[0] > x.shape[1] else x
    a, b, c = (np.float32(v) for v in R.NEWTON_SCHULZ)
    for _ in range(5):
        g = x @ x.T
        x = a * x + (b * g + c * (g @ g)) @ x
    return x if x.shape == u.shape else x.T


KINDS = {"normal": lambda r, s: r.standard_normal(s), "positive": lambda r, s: r.random(s) + 0.1, "sparse": lambda r, s: r.standard_normal(s) * (r.random(s) < 0.02),
         "wide": lambda r, s: r.standard_normal(s) * np.exp(2 * r.standard_normal(s)), "ones": lambda r, s: np.where(r.random(s) < 0.5, -1.0, 1.0)}


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape", [(1, 40, 64), (1, 96, 200), (1, 128, 3000), (1, 201, 333), (1, 640, 700), (1, 150, 5000), (20, 600, 700)],
                         ids=lambda s: "x".join(map(str, s)))
def test_products_as_exact_as_fp32_ones(shape, kind):
    """Numbers of one sign, of two values, mostly zeros, of very different sizes: what truncation takes of a sum depends on them.  Operands have two bits
    fewer than fp32 ones, so that the factor may be off by four times what it is with fp32 products; 2^-20 stands for
    what is put back of truncated sums."""
    ctx, alloc, be = env()
    g = KINDS[kind](np.random.default_rng(sum(shape)), shape).astype(np.float32)
    a, b = Matrices(g), Matrices(np.zeros(shape, np.float32))
    be.orthogonalise(a.argument, b.argument)
    got = b.read()[0]
    ref = R.factor(g[0])
    norm = np.linalg.norm(ref)
    off, plain = np.linalg.norm(got - ref) / norm, np.linalg.norm(fp32_factor(g[0]) - ref) / norm
    print(shape, kind, f"{off:.2e} {plain:.2e}")
    assert off <= 4 * plain + 2.0 ** -20
    check_clean_status()
    a.free(), b.free()


def test_forms_that_do_not_exist_are_refused():
    ctx, alloc, be = env()
    for bad in ((0, 3, 3, 0), (1, 0, 3, 0), (1, 3, 3, 3), (1, 3, 3, -1), (1, 1 << 16, 1 << 16, 0)):
        with pytest.raises(N.AgError):
            ctx.orthogonalise_form(*bad)
