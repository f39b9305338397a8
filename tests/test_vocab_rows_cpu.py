"""Operators on rows of logits, what needs no GPU: the 64-bit forms against differences, what the calls refuse, what they
hand to the C interface."""
import ctypes

import numpy as np
import pytest

from autograd_b200 import _native as N
from autograd_b200 import hostgraph as hg
from autograd_b200.backend import CudaBackend
from autograd_b200.storage import CudaAllocator, CudaMemPointer, Storage
from oracle import vocab_rows as R

RNG = np.random.default_rng


def _differences(f, x, step=1e-6):
    g = np.zeros_like(x)
    for i in np.ndindex(x.shape):
        up, down = x.copy(), x.copy()
        up[i] += step
        down[i] -= step
        g[i] = (f(up) - f(down)) / (2 * step)
    return g


@pytest.mark.parametrize("temperature", [1.0, 0.6, 2.5])
def test_gradient_of_log_probabilities_is_their_derivative(temperature):
    rng = RNG(3)
    x, ids = rng.standard_normal((4, 9)) * 2, np.array([3, -1, 8, 9])
    a, b = rng.standard_normal(4), rng.standard_normal(4)

    def f(z):
        lp, h, _, _, _ = R.token_logprobs(z, ids, temperature)
        return np.sum(a * lp + b * h)
    g, _, _ = R.token_logprobs_backward(x, ids, a, b, temperature)
    # central differences: step^2 f''' / 6 < 1e-11, rounding 1e-15 / step = 1e-9
    assert np.max(np.abs(g - _differences(f, x))) < 1e-8


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("temperature", [1.0, 0.6, 2.5])
def test_gradient_of_distillation_is_its_derivative(temperature, rest):
    rng = RNG(4)
    x = rng.standard_normal((4, 11)) * 2
    ids = np.array([[1, 4, 10], [2, -1, 3], [5, 5, 0], [-1, -1, 12]])
    t = np.log(rng.random((4, 3)) * 0.3) if rest else rng.standard_normal((4, 3))
    w = np.array([0.5, 0.2, 1.0, 0.3])
    got = R.distill(x, ids, t, w, 0.7, temperature, rest)
    diff = _differences(lambda z: 0.7 * R.distill(z, ids, t, w, 0.7, temperature, rest)["loss"], x)
    assert np.max(np.abs(got["dlogits"] - diff)) < 1e-8
    assert got["row_loss"][3] == 0 and not got["dlogits"][3].any()


@pytest.mark.parametrize("gap", [10.0, 100.0, 1000.0])
def test_gradient_of_a_small_rest_is_its_derivative(gap):
    """The unlisted tokens have e^-gap of the student's mass: no number of 64 bits in the last case."""
    rng = RNG(5)
    x = rng.standard_normal((3, 11))
    ids = np.array([[1, 4, 10], [2, 0, 3], [5, 5, 0]])
    t = np.log(rng.random((3, 3)) * 0.3)
    listed = np.zeros(x.shape, bool)
    np.put_along_axis(listed, ids, True, 1)
    x = np.where(listed, x, x - gap)
    got = R.distill(x, ids, t, rest=True)
    diff = _differences(lambda z: R.distill(z, ids, t, rest=True)["loss"], x, 1e-4)
    # rounding 1e-16 gap / step = 1e-9, third derivative times step^2 / 6 = 2e-9
    assert np.max(np.abs(got["dlogits"] - diff)) < 1e-8
    left = 1 - np.exp(t).sum(1)
    # what flows into them is p_rest (Q + r) - r, a third of which is the mean's
    assert np.allclose(np.where(listed, 0.0, got["dlogits"]).sum(1) * 3, np.exp(got["log_rest"]) - left, rtol=1e-9, atol=0)


def test_what_roundings_leave_of_a_list_is_no_rest():
    """Lists of all tokens that can occur, as log-probabilities in 32 bits: the others have p_rest = 0, or e^-1e9."""
    rng = RNG(6)
    z = rng.standard_normal((400, 20)) * 2
    t = (z - np.log(np.exp(z).sum(1, keepdims=True))).astype(np.float32)
    assert np.any(np.exp(t.astype(np.float64)).sum(1) < 1)
    ids = np.tile(np.arange(20), (400, 1))
    for mask in (-np.inf, -1e9):
        x = np.full((400, 30), mask)
        x[:, :20] = rng.standard_normal((400, 20))
        got = R.distill(x, ids, t, rest=True)
        lp = x[:, :20] - np.log(np.exp(x[:, :20]).sum(1, keepdims=True))
        q = np.exp(t.astype(np.float64))
        assert np.allclose(got["row_loss"], (q * (t - lp)).sum(1), rtol=1e-12)
        assert not got["dlogits"][:, 20:].any()
    # eight times that is one
    got = R.distill(x, ids, np.log(np.exp(t.astype(np.float64)) * (1 - 2.0 ** -15)), rest=True)
    assert np.all(got["row_loss"] > 1e4)


# ---------------------------------------------------------------------------- refusals of the C interface
# A context of zeros is enough for calls that are refused before they reach a device; one that is not refused fails to launch
# with another code.
SPACE = ctypes.create_string_buffer(1 << 16)
CTX = ctypes.addressof(SPACE)
BASE = 1 << 40


def _call(name, **change):
    a = dict(ctx=CTX, logits=BASE, ld=100, ids=BASE, logprob=BASE, entropy=0, stats=BASE, top_ids=BASE, top_logprobs=BASE,
             dlogprob=BASE, dentropy=BASE, dres=0, dlogits=BASE + (1 << 30), ld_grad=100, row_scale=0, dloss=BASE, loss=BASE,
             row_loss=BASE, N=4, V=100, top=5, temperature=1.0, mode=0, dtype=0)
    a.update(change)
    order = {
        "ag_token_logprobs_forward": "ctx logits ld ids logprob entropy stats top_ids top_logprobs N V top temperature dtype",
        "ag_token_logprobs_backward": "ctx logits ld ids stats dlogprob dentropy dres dlogits ld_grad N V temperature dtype",
        "ag_distill_forward": "ctx logits ld ids top_logprobs row_scale loss row_loss stats N V top temperature mode dtype",
        "ag_distill_backward": "ctx logits ld ids top_logprobs row_scale stats dloss dres dlogits ld_grad N V top temperature "
                               "mode dtype",
        "ag_distill_forward_backward": "ctx logits ld ids top_logprobs row_scale dloss loss row_loss stats dlogits ld_grad N V "
                                       "top temperature mode dtype"}
    return getattr(N.load_library(), name)(*(a[k] for k in order[name].split()))


ALL = ["ag_token_logprobs_forward", "ag_token_logprobs_backward", "ag_distill_forward", "ag_distill_backward",
       "ag_distill_forward_backward"]
GRAD = [n for n in ALL if "backward" in n]
DISTILL = [n for n in ALL if "distill" in n]
REFUSED = (
    [(n, c) for n in ALL for c in (
        dict(ctx=0), dict(N=-1), dict(N=1 << 31), dict(V=0), dict(V=-5), dict(ld=99), dict(ld=-100), dict(dtype=2), dict(dtype=-1),
        dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=float("nan")), dict(temperature=float("inf")),
        dict(temperature=1e-5), dict(logits=0), dict(logits=BASE + 2), dict(logits=BASE + 1, dtype=1), dict(stats=BASE + 4),
        dict(ld=1 << 31))] +
    [(n, dict(V=N.AG_VOCAB_MAX + 1, ld=N.AG_VOCAB_MAX + 1, ld_grad=N.AG_VOCAB_MAX + 1)) for n in ALL if n != "ag_token_logprobs_backward"] +
    [("ag_token_logprobs_forward", c) for c in (
        dict(top=-1), dict(top=N.AG_TOP_MAX + 1, V=1000, ld=1000), dict(top=6, V=5), dict(ids=0), dict(top_ids=0), dict(top_logprobs=0))] +
    [("ag_token_logprobs_backward", c) for c in (dict(ids=0), dict(stats=0))] +
    [(n, c) for n in GRAD for c in (
        dict(ld_grad=99), dict(ld_grad=-1), dict(ld_grad=-100), dict(dlogits=0), dict(dlogits=BASE + 2), dict(dlogits=BASE + 400),
        dict(dlogits=BASE, ld_grad=101), dict(dlogits=BASE - 4 * 399))] +
    [(n, c) for n in GRAD if "forward" not in n for c in (
        dict(dres=BASE + (1 << 30) + 4), dict(dres=BASE + 2))] +
    [(n, c) for n in DISTILL for c in (
        dict(top=0), dict(top=-1), dict(top=N.AG_DISTILL_MAX + 1, V=1000, ld=1000, ld_grad=1000), dict(mode=2), dict(mode=-1),
        dict(ids=0), dict(top_logprobs=0))] +
    [("ag_token_logprobs_forward", {k: BASE + 2}) for k in ("ids", "logprob", "entropy", "top_ids", "top_logprobs")] +
    [("ag_token_logprobs_backward", {k: BASE + 1}) for k in ("ids", "dlogprob", "dentropy")] +
    [(n, {k: BASE + 2}) for n in DISTILL for k in ("ids", "top_logprobs", "row_scale")] +
    [(n, {k: BASE + 2}) for n in DISTILL if "forward" in n for k in ("loss", "row_loss")] +
    [(n, dict(row_loss=0)) for n in DISTILL if "forward" in n] + [(n, dict(dloss=0)) for n in DISTILL if "backward" in n] +
    [("ag_distill_backward", dict(stats=0))])


@pytest.mark.parametrize("name,change", REFUSED, ids=lambda v: v[3:] if isinstance(v, str) else ",".join(f"{k}={x}" for k, x in v.items()))
def test_calls_that_are_refused(name, change):
    assert _call(name, **change) == N.AG_ERR_INVALID
    if change.get("ctx", 1):
        assert ctypes.string_at(N.load_library().ag_last_error(CTX)).startswith(name.encode())


@pytest.mark.parametrize("name", ALL)
def test_no_rows_are_no_work(name):
    assert _call(name, N=0, loss=0, logits=0, ids=0, logprob=0, dlogprob=0, dlogits=0, stats=0, top_ids=0) == N.AG_OK


# ---------------------------------------------------------------------------- the backend's methods
class _Recorder:
    def __init__(self):
        self.calls = []

    def alloc(self, nbytes):
        return BASE

    def __getattr__(self, name):
        return lambda *a: self.calls.append((name,) + a)


def _tensor(shape, dtype=np.float32):
    t = hg.HostTensor(shape, dtype)
    t.storage = Storage(CudaMemPointer(BASE), shape, dtype, "cuda", int(np.prod(shape)) * 4)
    return t


def _backend():
    ctx = _Recorder()
    return ctx, CudaBackend(ctx, CudaAllocator(ctx))


def test_what_the_methods_hand_over():
    ctx, be = _backend()
    x, ids, row, st = _tensor((2, 3, 64), np.uint16), _tensor((2, 3), np.int32), _tensor((2, 3)), _tensor((6, 4))
    k_ids, k = _tensor((2, 3, 5), np.int32), _tensor((2, 3, 5))
    one, g, weight = _tensor((1,)), _tensor((6, 80), np.uint16), _tensor((6,))
    be.token_logprobs_forward(x, ids, row, entropy=weight, stats=st, top_ids=k_ids, top_logprobs=k, temperature=0.5, vocab=60)
    assert ctx.calls[-1] == ("token_logprobs_forward", x, 64, ids, row, weight, st, k_ids, k, 6, 60, 5, 0.5, N.AG_BF16)
    be.token_logprobs_forward(x, None, None, entropy=weight)
    assert ctx.calls[-1] == ("token_logprobs_forward", x, 64, None, None, weight, None, None, None, 6, 64, 0, 1.0, N.AG_BF16)
    be.token_logprobs_backward(x, ids, st, row, None, g, dres=g)
    assert ctx.calls[-1] == ("token_logprobs_backward", x, 64, ids, st, row, None, g, g, 80, 6, 64, 1.0, N.AG_BF16)
    be.distill_forward(x, k_ids, k, row, loss=one, rest=True)
    assert ctx.calls[-1] == ("distill_forward", x, 64, k_ids, k, None, one, row, None, 6, 64, 5, 1.0, N.AG_DISTILL_REST, N.AG_BF16)
    be.distill_backward(x, k_ids, k, st, one, g, row_scale=weight, temperature=2.0)
    assert ctx.calls[-1] == ("distill_backward", x, 64, k_ids, k, weight, st, one, None, g, 80, 6, 64, 5, 2.0, N.AG_DISTILL_RENORM,
                             N.AG_BF16)
    be.distill_forward_backward(x, k_ids, k, one, row, x, loss=one, vocab=50)
    assert ctx.calls[-1] == ("distill_forward_backward", x, 64, k_ids, k, None, one, one, row, None, x, 64, 6, 50, 5, 1.0,
                             N.AG_DISTILL_RENORM, N.AG_BF16)


def test_tensors_that_do_not_fit_are_refused():
    ctx, be = _backend()
    x, ids, row, st = _tensor((6, 64)), _tensor((6,), np.int32), _tensor((6,)), _tensor((6, 4))
    k_ids, k, one, g = _tensor((6, 5), np.int32), _tensor((6, 5)), _tensor((1,)), _tensor((6, 64))
    short, wide = _tensor((5,)), _tensor((6,), np.int64)
    for bad in (lambda: be.token_logprobs_forward(x, ids, row, vocab=65), lambda: be.token_logprobs_forward(x, ids, row, vocab=0),
                lambda: be.token_logprobs_forward(x, ids, short), lambda: be.token_logprobs_forward(x, ids, row, top_ids=k_ids),
                lambda: be.token_logprobs_forward(x, ids, row, stats=row),
                lambda: be.token_logprobs_forward(x, ids, row, top_ids=k_ids, top_logprobs=st),
                lambda: be.token_logprobs_backward(x, ids, st, row, short, g),
                lambda: be.token_logprobs_backward(x, ids, st, row, row, _tensor((5, 64))),
                lambda: be.token_logprobs_backward(x, ids, st, row, row, _tensor((6, 64), np.uint16)),
                lambda: be.token_logprobs_backward(x, ids, st, row, row, g, dres=_tensor((6, 65))),
                lambda: be.distill_forward(x, k_ids, st, row), lambda: be.distill_forward(x, k_ids, k, row, loss=row),
                lambda: be.distill_forward(x, k_ids, k, row, row_scale=short),
                lambda: be.distill_backward(x, k_ids, k, row, one, g), lambda: be.distill_backward(x, k_ids, k, st, row, g),
                lambda: be.distill_forward_backward(x, k_ids, k, one, row, _tensor((7, 64)))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: be.token_logprobs_forward(x, wide, row), lambda: be.token_logprobs_forward(x, row, row),
                lambda: be.distill_forward(x, k, k, row), lambda: be.token_logprobs_forward(_tensor((6, 64), np.float64), ids, row)):
        with pytest.raises(TypeError):
            bad()
    assert not ctx.calls


@pytest.mark.parametrize("compiled", [True, False])
@pytest.mark.parametrize("name", ALL)
def test_both_bindings_take_the_arguments(name, compiled):
    """Tensors, integers, None and numbers in their places; a context that is null fails every call after that."""
    calls = N.calls if compiled else N._CheckedCalls(N.lib)
    values = {N._ptr: [_tensor((4, 64)), BASE, None, np.int64(BASE)], N._i64: [64], N._int: [4, np.int32(4)], N._f32: [1, 0.5]}
    args = [values[t][i % len(values[t])] for i, t in enumerate(N.SIGNATURES[name][1][1:])]
    with pytest.raises(N.AgError):
        getattr(calls, name)(0, *args)
    with pytest.raises((TypeError, ValueError)):
        getattr(calls, name)(0, *args[:-1])


def test_alternatives_are_asked_for_with_both_outputs():
    """One of the two by itself would be left as it was."""
    ctx, be = _backend()
    x, k_ids, k = _tensor((6, 64)), _tensor((6, 5), np.int32), _tensor((6, 5))
    for half in (dict(top_ids=k_ids), dict(top_logprobs=k)):
        with pytest.raises(ValueError):
            be.token_logprobs_forward(x, None, None, **half)
    assert not ctx.calls
