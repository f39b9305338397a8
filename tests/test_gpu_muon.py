"""Orthogonal factors and the step along them against the 64-bit forms.

A factor may be off by four times what the form with rounded operands and truncated sums is (oracle.heads_and_updates.factor_error:
operands of 22 significant bits, or 11 of products of 16-bit operands), by 2^-18 of its norm (the error of a form with one
number or a few may be small by chance), and by half a step of its type.  An update adds the roundings of its own arithmetic: p by 2^-24 of each of |p| (twice) and of its change (four times); m by 4 u (|m| + |g|)."""
import numpy as np
import pytest

from autograd_b200 import _native as N
from autograd_b200 import hostgraph as hg
from autograd_b200.backend import bf16_bits_to_f32, f32_to_bf16_bits
from gpu_util import check_clean_status, env, free, up
from oracle import heads_and_updates as R

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
SENTINEL = 777.0
BITS = {N.AG_CE_3XTF32: 22, N.AG_CE_BF16: 11}
PRECISIONS = pytest.mark.parametrize("precision", [N.AG_CE_3XTF32, N.AG_CE_BF16], ids=["pairs", "half"])


def rounded(x, dtype):
    return bf16_bits_to_f32(f32_to_bf16_bits(x)) if dtype == "bf16" else np.ascontiguousarray(x, np.float32)


def gradient(rng, count, rows, cols, dtype="f32"):
    r = min(4, rows, cols)
    g = rng.standard_normal((count, rows, r)) @ rng.standard_normal((count, r, cols)) / np.sqrt(r)
    return rounded((0.5 * g + rng.standard_normal((count, rows, cols))) * 1e-3, dtype)


class Matrices:
    """Matrices of their own, or one stack of them, `shift` elements behind an aligned address, with elements around them that stay."""

    def __init__(self, x, dtype="f32", apart=False, shift=0):
        ctx, alloc, be = env()
        self.shape, self.dtype, self.kind = x.shape, dtype, np.uint16 if dtype == "bf16" else np.float32
        self.each, self.shift, self.buffers = (1 if apart else len(x)), shift, []
        n = int(np.prod(x.shape[1:])) * self.each
        self.tensors = []
        for i in range(0, len(x), self.each):
            host = np.full(n + shift + 9, SENTINEL, np.float32)
            host[shift:shift + n] = x[i:i + self.each].reshape(-1)
            whole = up(f32_to_bf16_bits(host) if dtype == "bf16" else host)
            self.buffers.append(whole)
            shape = x.shape[1:] if apart else x.shape
            t = hg.HostTensor(shape, self.kind, requires_grad=False)
            t.storage = alloc.view(whole.storage, shift * (2 if dtype == "bf16" else 4), shape, self.kind)
            self.tensors.append(t)
        self.argument = self.tensors if apart else self.tensors[0]

    def read(self):
        ctx, alloc, be = env()
        out = []
        for whole in self.buffers:
            got = np.asarray(be.copy_to_host(whole), np.float32)
            n = got.size - self.shift - 9
            assert (np.delete(got, np.s_[self.shift:self.shift + n]) == rounded(np.float32([SENTINEL]), self.dtype)).all(), "written outside"
            out.append(got[self.shift:self.shift + n])
        return np.concatenate(out).reshape(self.shape).astype(np.float64)

    def free(self):
        free(*self.buffers)


def close(got, u, precision, steps=5, coefficients=R.NEWTON_SCHULZ, eps=1e-7, out="f32", more=0.0, by=1.0):
    ref, error = R.factor_error(u, coefficients, steps, eps, BITS[precision])
    ref = by * ref
    bound = 4 * abs(by) * error + (2.0 ** -18 + (2.0 ** -8 if out == "bf16" else 0)) * np.linalg.norm(ref) + more
    off = np.linalg.norm(got - ref)
    assert np.isfinite(got).all() and off <= bound, (off, bound, np.linalg.norm(ref))
    return off / max(np.linalg.norm(ref), 1e-300)


SHAPES = [(1, 1, 1), (1, 1, 9), (2, 7, 1), (2, 2, 2), (3, 16, 16), (2, 64, 256), (1, 100, 33), (2, 129, 65), (1, 127, 257), (3, 333, 201),
          (1, 384, 384), (2, 200, 64), (1, 64, 1000), (1, 1000, 3), (2, 128, 128), (1, 256, 640), (1, 257, 255), (1, 513, 520), (35, 20, 30),
          # clusters of several CTAs, slices of one to five groups, the last of them in part or not at all; more rounds than one
          (1, 20, 500), (1, 128, 1030), (1, 33, 2100), (1, 2900, 77), (1, 70, 4000), (2, 5100, 128), (160, 40, 65), (20, 17, 700), (1, 100, 5200),
          # contractions shared by clusters of 2, 4 and 8, the last parts of them short or empty; tiles of both sizes, an odd number of them
          (1, 200, 3000), (1, 130, 2113), (2, 300, 1300), (1, 1100, 390), (3, 260, 640), (1, 700, 650), (9, 300, 420), (24, 270, 300)]


@PRECISIONS
@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("bf16", "bf16"), ("f32", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_factor(shape, dtype, out, precision):
    ctx, alloc, be = env()
    rng = np.random.default_rng(sum(shape))
    g = gradient(rng, *shape, dtype)
    shift = 3 if shape[1] % 2 else 0
    a, b = Matrices(g, dtype, shift=shift), Matrices(np.full(shape, 2.0, np.float32), out, shift=shift)
    be.orthogonalise(a.argument, b.argument, precision=precision)
    got = b.read()
    for i in range(shape[0]):
        if i in (0, shape[0] // 2, shape[0] - 1):
            close(got[i], g[i], precision, out=out)
        else:   # the form with rounded operands takes long: of the other matrices, that they are theirs
            ref = R.factor(g[i])
            assert np.linalg.norm(got[i] - ref) <= 0.1 * np.linalg.norm(ref)
    assert np.array_equal(a.read(), g)
    check_clean_status()
    a.free(), b.free()


@PRECISIONS
@pytest.mark.parametrize("steps", [0, 1, 5])
@pytest.mark.parametrize("shape", [(2, 64, 256), (1, 300, 20), (2, 5, 9), (2, 130, 140)], ids=lambda s: "x".join(map(str, s)))
def test_narrower_words_in_the_matrix_place(shape, steps, precision):
    """bf16 factors begin where their fp32 matrices do: what a CTA writes is what others read."""
    ctx, alloc, be = env()
    rng = np.random.default_rng(sum(shape) + steps)
    g = gradient(rng, *shape)
    n = shape[1] * shape[2]
    for _ in range(10):
        a = Matrices(g, apart=True)
        outs = []
        for t in a.tensors:
            o = hg.HostTensor(shape[1:], np.uint16, requires_grad=False)
            o.storage = alloc.view(t.storage, 0, shape[1:], np.uint16)
            outs.append(o)
        be.orthogonalise(a.argument, outs, steps=steps, precision=precision)
        for i, whole in enumerate(a.buffers):
            words = np.asarray(be.copy_to_host(whole)).view(np.uint16)
            close(bf16_bits_to_f32(words[:n].copy()).reshape(shape[1:]).astype(np.float64), g[i], precision, steps, out="bf16")
            assert np.array_equal(words[n:2 * n], np.ascontiguousarray(g[i]).reshape(-1).view(np.uint16)[n:]), "more than the factor was written"
        a.free()
    check_clean_status()


@PRECISIONS
@pytest.mark.parametrize("steps,coefficients", [(0, R.NEWTON_SCHULZ), (1, R.NEWTON_SCHULZ), (2, (1.5, -0.5, 0.0)), (3, (2.0, -1.5, 0.5)),
                                                (3, [(8.2, -23.0, 16.5), (4.0, -2.9, 0.55), (1.9, -1.25, 0.4)])])
def test_steps_and_coefficients(steps, coefficients, precision):
    ctx, alloc, be = env()
    for rows, cols in ((48, 70), (200, 130)):
        g = gradient(np.random.default_rng(3), 2, rows, cols)
        a = Matrices(g)
        be.orthogonalise(a.argument, a.argument, steps=steps, coefficients=coefficients, precision=precision)   # in its place
        got = a.read()
        for i in range(2):
            close(got[i], g[i], precision, steps, coefficients)
        a.free()
    check_clean_status()


@PRECISIONS
def test_sizes_of_numbers_and_matrices_of_nothing(precision):
    """Scales of 1e30 and 1e-30, a matrix of zeros, one element, a single direction, rows that differ by 1e4; NaN and infinity stay in
    their matrix."""
    ctx, alloc, be = env()
    rng = np.random.default_rng(5)
    g = gradient(rng, 9, 70, 90) * 1e3
    g[0] *= 1e30
    g[1] *= 1e-30
    g[2] = 0
    g[3] = 0
    g[3, 5, 7] = -2.0
    g[4] = rng.standard_normal((70, 1)).astype(np.float32) * rng.standard_normal((1, 90)).astype(np.float32)
    g[5, ::2] *= 1e-4
    g[6, 3, 4] = np.nan
    g[7, 3, 4] = np.inf
    g = np.ascontiguousarray(g, np.float32)
    a, b = Matrices(g), Matrices(np.ones_like(g))
    be.orthogonalise(a.argument, b.argument, eps=1e-35, precision=precision)
    got = b.read()
    assert not got[2].any()
    for i in (0, 1, 3, 4, 5, 8):
        close(got[i], g[i], precision, eps=1e-35)
    assert np.isnan(got[6]).all() and np.isnan(got[7]).any()
    # a norm below eps is not blown up
    be.orthogonalise(a.argument, b.argument, eps=1e-3, precision=precision)
    close(b.read()[1], g[1], precision, eps=1e-3)
    check_clean_status()
    a.free(), b.free()


@PRECISIONS
@pytest.mark.parametrize("apart", [False, True])
@pytest.mark.parametrize("grad", ["f32", "bf16"])
@pytest.mark.parametrize("nesterov", [False, True])
@pytest.mark.parametrize("shape", [(3, 70, 90), (2, 150, 64), (40, 9, 5), (1, 128, 192)], ids=lambda s: "x".join(map(str, s)))
def test_step(shape, nesterov, grad, apart, precision):
    ctx, alloc, be = env()
    rng = np.random.default_rng(sum(shape) + nesterov)
    count, rows, cols = shape
    g, m, p = gradient(rng, *shape, grad), gradient(rng, *shape), (0.02 * rng.standard_normal(shape)).astype(np.float32)
    shift = 1 if rows % 2 else 0
    tp, tg, tm = Matrices(p, apart=apart, shift=shift), Matrices(g, grad, apart, shift), Matrices(m, apart=apart, shift=shift)
    kw = dict(momentum=0.9, nesterov=nesterov, weight_decay=0.1, grad_scale=0.25)
    lr, scale = 0.02, 0.2 * np.sqrt(max(rows, cols))
    for _ in range(2):
        before_p, before_m = tp.read(), tm.read()
        be.muon_step(tp.argument, tg.argument, tm.argument, lr, precision=precision, **kw)
        got_p, got_m = tp.read(), tm.read()
        for i in range(count):
            ref, ref_m, _ = R.muon(before_p[i], g[i], before_m[i], lr, scale=scale, **kw)
            assert (np.abs(got_m[i] - ref_m) <= 4 * U * (np.abs(before_m[i]) + np.abs(g[i]))).all()
            # what the factor is taken of: the stored momentum
            u = g[i] * 0.25 + 0.9 * (got_m[i] - g[i] * 0.25) if nesterov else got_m[i]
            moved = got_p[i] - before_p[i] * (1 - lr * 0.1)
            more = 2 * U * np.linalg.norm(before_p[i]) + 4 * U * np.linalg.norm(moved)
            close(moved, u, precision, more=more, by=-lr * scale)
    assert np.array_equal(tg.read(), g)
    check_clean_status()
    for t in (tp, tg, tm):
        t.free()


def test_other_batches_stay_apart():
    """More matrices than a launch takes, of which the workspace holds a part, and a matrix in two places of the list that are no
    outputs."""
    ctx, alloc, be = env()
    rng = np.random.default_rng(9)
    g = gradient(rng, 70, 33, 12)
    a, b = Matrices(g, apart=True), Matrices(np.zeros_like(g), apart=True)
    order = list(range(69)) + [3]
    be.orthogonalise([a.tensors[i] for i in order], b.tensors)
    got = b.read()
    for k, i in enumerate(order):
        close(got[k], g[i], N.AG_CE_3XTF32)
    assert np.array_equal(got[69], got[3])
    check_clean_status()
    a.free(), b.free()


def test_same_result_every_time_on_streams_and_in_recordings():
    import autograd_b200 as ag
    ctx, alloc, be = env()
    rng = np.random.default_rng(10)
    g = gradient(rng, 3, 300, 200)
    a = Matrices(g)
    other = ag.create(0)
    ctx.synchronize()
    results = []
    for backend, graph in ((be, False), (be, False), (other[2], False), (be, True)):
        b = Matrices(np.zeros_like(g))
        ctx.synchronize()
        if graph:   # the arrays of addresses are read while the launches are recorded
            at, n, shape, kind = be._matrices("g", a.argument)
            to = be._matrices("out", b.argument)[0]
            co = be._coefficients(be.NEWTON_SCHULZ, 5)
            need = ctx.orthogonalise_scratch_bytes(n, *shape)
            ws = up(np.zeros(need, np.uint8))
            rec = ctx.record(lambda r: r.orthogonalise(_at(at), _at(to), n, *shape, _at(co), 5, 1e-7, N.AG_CE_3XTF32, 0, 0, ws, need))
            for t in (at, to, co):
                for i in range(len(t)):
                    t[i] = 0
            ctx.replay(rec)
            ctx.replay(rec)
            ctx.synchronize()
            ctx.drop_recording(rec)
            free(ws)
        else:
            backend.orthogonalise(a.argument, b.argument)
            backend.synchronize()
        results.append(b.read())
        b.free()
    assert all(np.array_equal(results[0], r) for r in results[1:])
    close(results[0][1], g[1], N.AG_CE_3XTF32)
    check_clean_status()
    other[0].check_status()
    a.free()


def _at(array):
    import ctypes
    return ctypes.addressof(array)


def test_workspace_is_not_exceeded_and_no_matrices_are_no_work():
    ctx, alloc, be = env()
    g = gradient(np.random.default_rng(1), 2, 130, 70)
    a, b = Matrices(g), Matrices(np.zeros_like(g))
    need = ctx.orthogonalise_scratch_bytes(2, 130, 70)
    ws = up(np.full(need + 4096, 171, np.uint8))
    at, n, shape, _ = be._matrices("g", a.argument)
    to, co = be._matrices("out", b.argument)[0], be._coefficients(be.NEWTON_SCHULZ, 5)
    with pytest.raises(N.AgError) as e:
        ctx.orthogonalise(_at(at), _at(to), n, *shape, _at(co), 5, 1e-7, N.AG_CE_3XTF32, 0, 0, ws, need - 1)
    assert e.value.code == N.AG_ERR_SCRATCH
    ctx.orthogonalise(_at(at), _at(to), n, *shape, _at(co), 5, 1e-7, N.AG_CE_3XTF32, 0, 0, ws, need)
    assert (be.copy_to_host(ws)[need:] == 171).all()
    close(b.read()[0], g[0], N.AG_CE_3XTF32)
    be.orthogonalise([], [])
    be.muon_step([], [], [], 0.1)
    check_clean_status()
    a.free(), b.free(), free(ws)
