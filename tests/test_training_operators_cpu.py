"""Normalised heads and orthogonal updates, what needs no GPU: the 64-bit forms against differences and singular values, what the
calls refuse, what the backend hands to the C interface."""
import ctypes

import numpy as np
import pytest

from autograd_b200 import _native as N
from autograd_b200 import hostgraph as hg
from autograd_b200.backend import CudaBackend
from autograd_b200.storage import CudaAllocator, CudaMemPointer, Storage
from oracle import heads_and_updates as R


@pytest.mark.parametrize("rot", [0, 6, 8])
def test_gradient_of_heads_is_their_derivative(rot):
    rng = np.random.default_rng(rot)
    x, dy, gamma = rng.standard_normal((2, 3, 8)), rng.standard_normal((2, 3, 8)), rng.standard_normal(8)
    a = rng.standard_normal((2, rot // 2))
    c, s = np.cos(a), np.sin(a)

    def loss(x, gamma):
        return (R.heads(x, gamma, c, s, 1e-6) * dy).sum()
    dx, dgamma = R.heads_backward(dy, x, gamma, c, s, 1e-6)
    for got, at, f in ((dx, x, lambda v: loss(v, gamma)), (dgamma, gamma, lambda v: loss(x, v))):
        for i in np.ndindex(at.shape):
            up, down = at.copy(), at.copy()
            up[i] += 1e-6
            down[i] -= 1e-6
            # third derivative times step^2 / 6 < 1e-9, rounding 1e-15 / step = 1e-9
            assert abs((f(up) - f(down)) / 2e-6 - got[i]) < 1e-7


@pytest.mark.parametrize("shape", [(5, 9), (9, 5), (6, 6), (1, 4)])
def test_factor_is_the_polynomial_of_the_singular_values(shape):
    g = np.random.default_rng(1).standard_normal(shape)
    u, s, vt = np.linalg.svd(g, full_matrices=False)
    s = s / np.sqrt((s ** 2).sum())
    for a, b, c in R.triples(R.NEWTON_SCHULZ, 5):
        s = a * s + b * s ** 3 + c * s ** 5
    assert np.abs(R.factor(g) - (u * s) @ vt).max() < 1e-12
    assert R.factor_error(g, R.NEWTON_SCHULZ, 5, 1e-7, 22)[1] < 1e-4 < R.factor_error(g, R.NEWTON_SCHULZ, 5, 1e-7, 11)[1]


# ---------------------------------------------------------------------------- refusals of the C interface
# A context of zeros is enough for calls that are refused before they reach a device
SPACE = ctypes.create_string_buffer(1 << 16)
CTX = ctypes.addressof(SPACE)
BASE = 1 << 40
FAR = 1 << 32
ORDER = {
    "ag_qk_norm_rope_forward": "ctx q k q_gamma k_gamma cos sin positions q_out k_out tokens seq rows H HKV D rot q_stride k_stride "
                               "q_out_stride k_out_stride eps sign dtype",
    "ag_qk_norm_rope_backward": "ctx dq_out dk_out q k q_gamma k_gamma cos sin positions dq dk dq_gamma dk_gamma partials bytes tokens "
                                "seq rows H HKV D rot dq_out_stride dk_out_stride q_stride k_stride dq_stride dk_stride eps sign "
                                "accumulate dtype",
    "ag_orthogonalise": "ctx g out count rows cols coefficients steps eps precision dtype out_dtype scratch bytes",
    "ag_muon_step": "ctx p g m count rows cols lr momentum nesterov decay scale grad_scale coefficients steps eps precision dtype "
                    "scratch bytes"}
HEADS = dict(ctx=CTX, q=BASE, k=BASE + FAR, q_gamma=0, k_gamma=0, cos=BASE + 2 * FAR, sin=BASE + 2 * FAR, positions=0, q_out=BASE + 3 * FAR,
             k_out=BASE + 4 * FAR, tokens=6, seq=3, rows=3, H=4, HKV=2, D=16, rot=16, q_stride=64, k_stride=32, q_out_stride=64,
             k_out_stride=32, eps=1e-6, sign=1, dtype=0, dq_out=BASE + 5 * FAR, dk_out=BASE + 6 * FAR, dq=BASE + 3 * FAR,
             dk=BASE + 4 * FAR, dq_gamma=0, dk_gamma=0, partials=0, bytes=0, dq_out_stride=64, dk_out_stride=32, dq_stride=64,
             dk_stride=32, accumulate=0)


def _array(kind, values):
    return (kind * len(values))(*values)


def _addresses(first):
    return _array(ctypes.c_void_p, [first + i * (1 << 20) for i in range(3)])


MATS = dict(ctx=CTX, p=_addresses(BASE), out=_addresses(BASE), g=_addresses(BASE + FAR), m=_addresses(BASE + 2 * FAR), count=3, rows=20,
            cols=30, lr=0.1, momentum=0.9, nesterov=1, decay=0.0, scale=1.0, grad_scale=1.0,
            coefficients=_array(ctypes.c_float, [3.4, -4.7, 2.0] * 5), steps=5, eps=1e-7, precision=N.AG_CE_3XTF32, dtype=0, out_dtype=0,
            scratch=BASE + 3 * FAR, bytes=1 << 30)


def _call(name, **change):
    a = dict(MATS if "qk" not in name else HEADS)
    a.update(change)
    return getattr(N.load_library(), name)(*(a[k] for k in ORDER[name].split()))


QK = ["ag_qk_norm_rope_forward", "ag_qk_norm_rope_backward"]
NS = ["ag_orthogonalise", "ag_muon_step"]
NAN, INF = float("nan"), float("inf")
REFUSED = (
    [(n, c) for n in QK for c in (
        dict(ctx=0), dict(tokens=-1), dict(tokens=1 << 31), dict(D=0), dict(D=15, rot=0), dict(D=-16), dict(D=N.AG_QK_MAX_D + 2, rot=0),
        dict(rot=-2), dict(rot=18), dict(rot=7), dict(dtype=2), dict(dtype=-1), dict(eps=-1.0), dict(eps=NAN), dict(eps=INF), dict(cos=0),
        dict(sin=0), dict(rows=0), dict(rows=2), dict(seq=0), dict(seq=-3), dict(rows=0, positions=BASE + 7 * FAR), dict(H=0), dict(H=-4),
        dict(HKV=0), dict(H=70000, q_stride=1 << 22, q_out_stride=1 << 22, dq_stride=1 << 22, dq_out_stride=1 << 22),
        dict(q_stride=63), dict(k_stride=31), dict(q_stride=-64), dict(q_stride=1 << 31), dict(q=0, k=0), dict(q=BASE + 2),
        dict(q=BASE + 1, dtype=1), dict(q_gamma=BASE + 2), dict(cos=BASE + 2 * FAR + 1), dict(positions=BASE + 7 * FAR + 2))] +
    [("ag_qk_norm_rope_forward", c) for c in (
        dict(q_out=0), dict(k_out=0), dict(q_out_stride=63), dict(k_out_stride=-1), dict(q_out=BASE + 4), dict(q_out=BASE, q_out_stride=65),
        dict(q_out=BASE + FAR), dict(k_out=BASE + 3 * FAR), dict(q_out=BASE - 4 * 300), dict(k_out=BASE + 64 * 4),
        # slices of packed rows that reach into one another
        dict(q_stride=96, q_out=BASE + 4 * 48, q_out_stride=96))] +
    [("ag_qk_norm_rope_backward", c) for c in (
        dict(dq=0), dict(dk=0), dict(dq_out=0), dict(dk_out=0), dict(dq_stride=63), dict(dq_out_stride=63), dict(dq=BASE + 4),
        dict(dq=BASE + 6 * FAR), dict(dk=BASE + 3 * FAR), dict(dq=BASE + 5 * FAR, dq_stride=70), dict(dq_gamma=BASE + 8 * FAR),
        dict(dq_gamma=BASE + 8 * FAR + 2, partials=BASE + 9 * FAR, bytes=1 << 20), dict(dk_gamma=BASE + 8 * FAR, partials=BASE + 9 * FAR + 2, bytes=1 << 20),
        dict(dq_gamma=BASE + 8 * FAR, dk_gamma=BASE + 8 * FAR + 60, partials=BASE + 9 * FAR, bytes=1 << 24),
        dict(dq_gamma=BASE + 8 * FAR + 60, dk_gamma=BASE + 8 * FAR, partials=BASE + 9 * FAR, bytes=1 << 24))] +
    [(n, c) for n in NS for c in (
        dict(ctx=0), dict(count=-1), dict(rows=0), dict(cols=-3), dict(rows=16385, cols=16385), dict(rows=2, cols=(1 << 20) + 1),
        dict(rows=16384, cols=1 << 17), dict(steps=-1), dict(steps=33), dict(coefficients=None), dict(eps=0.0), dict(eps=-1.0), dict(eps=NAN),
        dict(eps=INF), dict(precision=N.AG_CE_FP32), dict(precision=N.AG_CE_BF16X3), dict(precision=9), dict(dtype=2), dict(g=None),
        dict(coefficients=_array(ctypes.c_float, [3.4, -4.7, 2.0] * 4 + [NAN, 1, 1])),
        dict(coefficients=_array(ctypes.c_float, [3.4, -4.7, 2.0] * 4 + [3.4, -4.7, 0.2])),
        dict(coefficients=_array(ctypes.c_float, [3.4, 1e3, 100.0] * 5)), dict(scratch=0), dict(scratch=BASE + 3 * FAR + 128),
        dict(g=_array(ctypes.c_void_p, [BASE + FAR, 0, BASE + 2 * FAR])), dict(g=_addresses(BASE + FAR + 2)), dict(g=_addresses(BASE + 4)),
        dict(scratch=BASE + FAR), dict(scratch=BASE - 256))] +
    [("ag_orthogonalise", c) for c in (
        dict(out=None), dict(out_dtype=5), dict(out=_addresses(BASE + 1)), dict(out=_array(ctypes.c_void_p, [BASE, BASE + 2396, BASE + FAR // 2])),
        dict(out=_array(ctypes.c_void_p, [BASE, BASE, BASE + FAR // 2])), dict(out=_addresses(BASE + FAR), dtype=1),
        dict(g=_addresses(BASE + 4)), dict(g=_array(ctypes.c_void_p, [BASE + (1 << 20), BASE, BASE + FAR])),
        # a factor of 16-bit words in its matrix's place, and another one in what is left of it
        dict(g=_array(ctypes.c_void_p, [BASE, BASE + 2400, BASE + FAR]), out=_array(ctypes.c_void_p, [BASE, BASE + 1200, BASE + FAR]), out_dtype=1))] +
    [("ag_muon_step", c) for c in (
        dict(p=None), dict(m=None), dict(lr=NAN), dict(lr=INF), dict(momentum=-0.1), dict(momentum=1.1), dict(momentum=NAN), dict(decay=INF),
        dict(scale=NAN), dict(grad_scale=INF), dict(m=_addresses(BASE)), dict(m=_addresses(BASE + FAR)), dict(g=_addresses(BASE)),
        dict(p=_array(ctypes.c_void_p, [BASE, BASE + 8, BASE + FAR // 2])), dict(p=_addresses(BASE + 2)))])


@pytest.mark.parametrize("name,change", REFUSED, ids=lambda v: v[3:] if isinstance(v, str) else ",".join(v))
def test_calls_that_are_refused(name, change):
    assert _call(name, **change) == N.AG_ERR_INVALID
    if change.get("ctx", 1):
        assert ctypes.string_at(N.load_library().ag_last_error(CTX)).startswith(name.encode())


def test_short_workspaces_are_refused():
    need = N.load_library().ag_orthogonalise_scratch_bytes(3, 20, 30, N.AG_CE_3XTF32)
    assert need > 0
    for name in NS:
        assert _call(name, bytes=need - 1) == N.AG_ERR_SCRATCH
    for bad in ((0, 20, 30, 1), (3, 0, 30, 1), (3, 20, -1, 1), (3, 16385, 16385, 1), (3, 20, 30, 0), (3, 2, (1 << 20) + 1, 1),
                (1, 16384, 1 << 17, 1)):
        assert N.load_library().ag_orthogonalise_scratch_bytes(*bad) == 0


def test_no_tokens_and_no_matrices_are_no_work():
    for name in QK:
        assert _call(name, tokens=0, q=0, k=0) == N.AG_OK
    for name in NS:
        assert _call(name, count=0, scratch=0, bytes=0, g=None, p=None, m=None, out=None) == N.AG_OK


# ---------------------------------------------------------------------------- the backend's methods
class _Recorder:
    def __init__(self):
        self.calls = []

    def alloc(self, nbytes):
        return BASE

    def qk_norm_partials_bytes(self, *a):
        return 1000

    def orthogonalise_scratch_bytes(self, *a):
        return 4096

    def __getattr__(self, name):
        return lambda *a: self.calls.append((name,) + a)


def _tensor(shape, dtype=np.float32, at=BASE):
    t = hg.HostTensor(shape, dtype)
    t.storage = Storage(CudaMemPointer(at), shape, dtype, "cuda", int(np.prod(shape)) * 4)
    return t


def _backend():
    ctx = _Recorder()
    return ctx, CudaBackend(ctx, CudaAllocator(ctx))


def test_heads_that_the_backend_hands_over():
    ctx, be = _backend()
    q, k, cos, g = _tensor((2, 3, 4, 16), np.uint16), _tensor((2, 3, 2, 16), np.uint16), _tensor((5, 6)), _tensor((16,))
    y, z, at = _tensor((2, 3, 4, 16), np.uint16), _tensor((2, 3, 2, 16), np.uint16), _tensor((2, 3), np.int32)
    be.qk_norm_rope_forward(q, k, cos, cos, y, z, 1e-6, q_gamma=g, q_stride=128, k_stride=128)
    assert ctx.calls[-1] == ("qk_norm_rope_forward", q, k, g, None, cos, cos, None, y, z, 6, 3, 5, 4, 2, 16, 12, 128, 128, 64, 32, 1e-6, 1,
                             N.AG_BF16)
    be.qk_norm_rope_forward(q, k, None, None, q, k, 1e-6, q_stride=128, k_stride=128, positions=at, sin_sign=-1)
    assert ctx.calls[-1] == ("qk_norm_rope_forward", q, k, None, None, None, None, None, q, k, 6, 3, 0, 4, 2, 16, 0, 128, 128, 128, 128, 1e-6,
                             -1, N.AG_BF16)
    be.qk_norm_rope_forward(None, k, cos, cos, None, z, 1e-6, positions=at)
    assert ctx.calls[-1] == ("qk_norm_rope_forward", None, k, None, None, cos, cos, at, None, z, 6, 3, 5, 0, 2, 16, 12, 0, 32, 0, 32, 1e-6, 1,
                             N.AG_BF16)
    be.qk_norm_rope_backward(y, z, q, k, cos, cos, y, k, 1e-6, k_gamma=g, dk_gamma=g, q_stride=128, k_stride=96, accumulate=True)
    name, *a = ctx.calls[-1]
    assert name == "qk_norm_rope_backward" and a[:13] == [y, z, q, k, None, g, cos, cos, None, y, k, None, g]
    assert a[14] >= 1000 and a[15:] == [6, 3, 5, 4, 2, 16, 12, 64, 32, 128, 96, 64, 96, 1e-6, 1, True, N.AG_BF16]
    be.qk_norm_rope_backward(y, None, q, None, cos, cos, z if False else y, None, 1e-6, positions=at)
    assert ctx.calls[-1][14:16] == (0, 0)


def test_heads_that_do_not_fit_are_refused():
    ctx, be = _backend()
    q, k, cos = _tensor((2, 3, 4, 16)), _tensor((2, 3, 2, 16)), _tensor((5, 8))
    at, f = _tensor((6,), np.int32), be.qk_norm_rope_forward
    for bad in (lambda: f(None, None, cos, cos, None, None, 1e-6), lambda: f(q, k, cos, cos, q, None, 1e-6), lambda: f(q, None, cos, cos, q, k, 1e-6),
                lambda: f(q, k, cos, None, q, k, 1e-6), lambda: f(q, k, _tensor((5, 9)), _tensor((5, 9)), q, k, 1e-6),
                lambda: f(q, k, _tensor((2, 8)), _tensor((2, 8)), q, k, 1e-6), lambda: f(q, k, cos, _tensor((5, 7)), q, k, 1e-6),
                lambda: f(q, k, cos, cos, k, k, 1e-6), lambda: f(q, _tensor((2, 3, 2, 8)), cos, cos, q, k, 1e-6),
                lambda: f(q, _tensor((2, 3, 2, 16), np.uint16), cos, cos, q, k, 1e-6), lambda: f(q, _tensor((1, 6, 2, 16)), cos, cos, q, k, 1e-6),
                lambda: f(q, k, cos, cos, q, k, 1e-6, q_gamma=_tensor((15,))), lambda: f(q, k, cos, cos, q, k, 1e-6, positions=_tensor((5,), np.int32)),
                lambda: be.qk_norm_rope_backward(q, k, q, k, cos, cos, q, None, 1e-6),
                lambda: be.qk_norm_rope_backward(q, k, q, k, cos, cos, q, k, 1e-6, dk_gamma=_tensor((4,)))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: f(q, k, cos, cos, q, k, 1e-6, positions=_tensor((6,), np.int64)), lambda: f(q, k, cos, cos, q, k, 1e-6, positions=_tensor((6,))),
                lambda: f(_tensor((2, 3, 4, 16), np.float64), None, cos, cos, q, None, 1e-6)):
        with pytest.raises(TypeError):
            bad()
    assert not ctx.calls
    f(q, k, cos, cos, q, k, 1e-6, positions=at)


def test_matrices_that_the_backend_hands_over():
    ctx, be = _backend()
    stack, one, bits = _tensor((3, 20, 30)), [_tensor((20, 30), at=BASE + i * 8192) for i in range(3)], _tensor((3, 20, 30), np.uint16, BASE + FAR)
    seen = []

    def grab(*a):   # the arrays live as long as the call
        seen.append([a[0], [list((ctypes.c_void_p * n).from_address(x)) for x, n in a[1]], list((ctypes.c_float * a[2][1]).from_address(a[2][0])), a[3]])
    ctx.orthogonalise = lambda g, o, n, r, c, co, s, e, p, d, od, sc, sb: grab("f", [(g, n), (o, n)], (co, 3 * s), (n, r, c, s, e, p, d, od, sb))
    ctx.muon_step = lambda p, g, m, n, r, c, lr, mo, ne, wd, sc, gs, co, s, e, pr, gd, ws, wb: grab(
        "m", [(p, n), (g, n), (m, n)], (co, 3 * s), (n, r, c, lr, mo, ne, wd, sc, gs, s, e, pr, gd))
    be.orthogonalise(stack, bits, steps=2, coefficients=[(1, 2, 3), (4, 5, 6)], precision=N.AG_CE_BF16)
    assert seen[-1] == ["f", [[BASE, BASE + 2400, BASE + 4800], [BASE + FAR, BASE + FAR + 1200, BASE + FAR + 2400]], [1, 2, 3, 4, 5, 6],
                        (3, 20, 30, 2, 1e-7, N.AG_CE_BF16, N.AG_F32, N.AG_BF16, 4096)]
    be.muon_step([t.storage for t in one], bits, one, 0.5, momentum=0.8, weight_decay=0.1, grad_scale=2.0, steps=1, coefficients=(1, 2, 3))
    assert seen[-1] == ["m", [[t.storage.ptr.address for t in one], [BASE + FAR + 1200 * i for i in range(3)],
                              [t.storage.ptr.address for t in one]], [1, 2, 3],
                        (3, 20, 30, 0.5, 0.8, True, 0.1, 0.2 * 30 ** 0.5, 2.0, 1, 1e-7, N.AG_CE_3XTF32, N.AG_BF16)]
    be.orthogonalise([], [])
    be.muon_step([], [], [], 1.0)
    assert len(seen) == 2


def test_matrices_that_do_not_fit_are_refused():
    ctx, be = _backend()
    a, b = _tensor((3, 20, 30)), _tensor((3, 30, 20))
    for bad in (lambda: be.orthogonalise(a, b), lambda: be.orthogonalise(_tensor((30,)), a), lambda: be.orthogonalise([a, b], [a, b]),
                lambda: be.orthogonalise(a, _tensor((2, 20, 30))), lambda: be.orthogonalise(a, a, coefficients=(1, 2)),
                lambda: be.orthogonalise(a, a, coefficients=[(1, 2, 3)] * 4), lambda: be.orthogonalise([a, _tensor((20, 30), np.uint16)], a),
                lambda: be.muon_step(a, a, b, 0.1), lambda: be.muon_step(a, [], a, 0.1)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: be.muon_step(_tensor((3, 20, 30), np.uint16), a, a, 0.1), lambda: be.muon_step(a, a, _tensor((3, 20, 30), np.uint16), 0.1),
                lambda: be.orthogonalise(_tensor((3, 4), np.float64), a)):
        with pytest.raises(TypeError):
            bad()
    assert not ctx.calls


@pytest.mark.parametrize("compiled", [True, False])
@pytest.mark.parametrize("name", QK + NS)
def test_both_bindings_take_the_arguments(name, compiled):
    """Tensors, integers, None and numbers in their places; a context that is null fails every call after that."""
    calls = N.calls if compiled else N._CheckedCalls(N.lib)
    values = {N._ptr: [_tensor((4, 64)), BASE, None, np.int64(BASE)], N._i64: [64], N._int: [4, np.int32(4)], N._f32: [1, 0.5], N._f64: [1, 0.5],
              N._sz: [100]}
    args = [values[t][i % len(values[t])] for i, t in enumerate(N.SIGNATURES[name][1][1:])]
    with pytest.raises(N.AgError):
        getattr(calls, name)(0, *args)
    with pytest.raises((TypeError, ValueError)):
        getattr(calls, name)(0, *args[:-1])
