"""Heads normalised and rotated, and their gradients, against the 64-bit forms.

Bounds, in units u = 2^-24 (half a step of fp32).  The sum of squares of a head: a lane adds up to 32 terms, then five lanes'
sums, so at most 37 u of itself; inv is off by half of that and by 3 u of its own: 22 u.  A normalised element adds two products:
24 u; the rotation two products and a sum of it and its partner: y is off by 27 u (|yn| + |yn partner|), 32 u here.
w is off by 2 u (|dy| + |dy partner|); mean(v x) by 40 u of mean |v x| and by what v is; dx = inv (v - x inv^2 mean(v x)) by 22 u
for inv, three times in the second term: 80 u in all of inv (|v| + |v partner| + |x| inv^2 mean (|v| + |v partner|) |x|).
dgamma adds at most `terms` numbers in a chain, each off by 26 u: (terms + 32) u of the sum of their sizes.  bf16 outputs add 2^-8 of
their value."""
import zlib

import numpy as np
import pytest

from autograd_b200 import _native as N
from autograd_b200.backend import bf16_bits_to_f32, f32_to_bf16_bits
from gpu_util import check_clean_status, empty, env, free, up
from oracle import heads_and_updates as R

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
SENTINEL = 777.0
EPS = 1e-6


def rounded(x, dtype):
    return bf16_bits_to_f32(f32_to_bf16_bits(x)) if dtype == "bf16" else np.ascontiguousarray(x, np.float32)


def size(dtype):
    return 2 if dtype == "bf16" else 4


class Rows:
    """tokens x width elements on the device, `stride` apart, the first `shift` elements behind an aligned address; everything
    else in the buffer is SENTINEL and has to stay."""

    def __init__(self, x, dtype, stride=None, shift=0, behind=5):
        ctx, alloc, be = env()
        self.dtype, self.shape = dtype, x.shape
        n, w = x.shape[0], int(np.prod(x.shape[1:]))
        self.stride = w if stride is None else stride
        host = np.full(shift + max(n, 1) * self.stride + behind, SENTINEL, np.float32)
        self.at = shift + np.arange(n)[:, None] * self.stride + np.arange(w)
        host[self.at] = x.reshape(n, w)
        self.whole = up(f32_to_bf16_bits(host) if dtype == "bf16" else host)
        self.address = self.whole.storage.ptr.address + shift * size(dtype)
        self.mine = np.zeros(host.size, bool)
        self.mine[self.at] = True

    def read(self):
        got = env()[0].copy_to_host(self.whole.storage.ptr.address, self.mine.shape, np.uint16 if self.dtype == "bf16" else np.float32)
        got = bf16_bits_to_f32(got) if self.dtype == "bf16" else got
        assert (got[~self.mine] == rounded(np.float32([SENTINEL]), self.dtype)).all(), "written outside the rows"
        return got[self.at].reshape(self.shape).astype(np.float64)


def tables(rows, rot, theta=1e4):
    a = np.arange(rows)[:, None] * theta ** (-np.arange(0, rot, 2) / max(rot, 1))
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


def inputs(rng, n, heads, d, dtype):
    x = rng.standard_normal((n, heads, d)) * np.exp(2 * rng.standard_normal((n, heads, 1)))
    x[..., ::7] *= 30
    if n * heads > 2:
        x[n // 2, heads // 2] = 0.0
    return rounded(x.astype(np.float32), dtype)


def place(rng, n, seq, rows, given):
    return rng.integers(0, rows, n).astype(np.int32) if given else (np.arange(n) % seq).astype(np.int32)


def partner(y, rot):
    h, z = rot // 2, np.array(np.abs(y))
    z[..., :h], z[..., h:rot] = np.abs(y[..., h:rot]), np.abs(y[..., :h])
    z[..., rot:] = 0
    return z + np.abs(y)


def near(got, ref, bound, dtype, what):
    bound = bound + (2.0 ** -8 * np.abs(ref) if dtype == "bf16" else 0) + 1e-40
    off = np.abs(got - ref) - bound
    assert np.isfinite(got).all(), what
    if off.size and off.max() > 0:
        i = np.unravel_index(off.argmax(), off.shape)
        raise AssertionError(f"{what} at {i}: {got[i]!r} instead of {ref[i]!r}, bound {np.broadcast_to(bound, ref.shape)[i]:.3e}")


# tokens, seq, heads, kv, D, rot
SHAPES = [(1, 1, 10, 10, 128, 128), (64, 1, 12, 2, 128, 128), (333, 111, 7, 3, 80, 40), (130, 65, 4, 4, 64, 64), (77, 77, 3, 1, 256, 256),
          (9, 3, 5, 2, 50, 50), (41, 41, 2, 1, 74, 36), (5, 5, 1, 1, 2, 2), (6, 3, 3, 2, 6, 0), (12, 4, 2, 2, 1024, 1024), (11, 11, 1, 3, 1022, 510),
          (3, 3, 2, 1, 514, 514), (4, 2, 33, 8, 96, 24), (1000, 250, 1, 1, 16, 16), (19, 19, 2, 2, 512, 128), (7, 7, 3, 1, 768, 768),
          (2, 2, 1, 1, 1000, 600), (1, 1, 1, 1, 4, 2), (29, 29, 2, 1, 308, 104), (8, 8, 3, 2, 160, 80)]
LAYOUTS = ["dense", "packed", "shifted"]


def operands(rng, shape, dtype, layout):
    n, seq, h, kv, d, rot = shape
    q, k = inputs(rng, n, h, d, dtype), inputs(rng, n, kv, d, dtype)
    pitch = {"dense": (None, None), "packed": ((h + 2 * kv) * d, (h + 2 * kv) * d), "shifted": (h * d + 3, kv * d + 1)}[layout]
    return q, k, pitch, 1 if layout == "shifted" else 0


def addresses(*arrays):
    return [0 if a is None else up(a) for a in arrays]


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_forward(shape, dtype, layout):
    ctx, alloc, be = env()
    rng = np.random.default_rng(zlib.crc32(repr((shape, dtype, layout)).encode()))
    n, seq, h, kv, d, rot = shape
    q, k, pitch, shift = operands(rng, shape, dtype, layout)
    rows = seq + 3
    cos, sin = tables(rows, rot)
    given = layout == "packed"
    at = place(rng, n, seq, rows, given)
    gamma = (1 + 0.3 * rng.standard_normal((2, d))).astype(np.float32) if layout != "shifted" else (None, None)
    x = [Rows(t, dtype, p, shift) for t, p in zip((q, k), pitch)]
    y = [Rows(np.full(t.shape, 5.0, np.float32), dtype, None if layout != "shifted" else p, shift) for t, p in zip((q, k), pitch)]
    c, s, p, gq, gk = addresses(cos if rot else None, sin if rot else None, at if given else None, *gamma)
    sign = -1 if layout == "dense" else 1
    ctx.qk_norm_rope_forward(x[0].address, x[1].address, gq, gk, c, s, p, y[0].address, y[1].address, n, seq, rows, h, kv, d, rot,
                             x[0].stride, x[1].stride, y[0].stride, y[1].stride, EPS, sign, N.AG_BF16 if dtype == "bf16" else N.AG_F32)
    for t, out, g in ((q, y[0], gamma[0]), (k, y[1], gamma[1])):
        plain = R.heads(t, g, cos[at], np.zeros_like(sin[at]), EPS) if not rot else R.heads(t, g, np.ones_like(cos[at]), 0 * sin[at], EPS)
        ref = R.heads(t, g, cos[at], sign * sin[at], EPS)
        near(out.read(), ref, 32 * U * partner(plain, rot), dtype, "y")
    for r in x:
        r.read()
    check_clean_status()
    free(*(r.whole for r in x + y), *(t for t in (c, s, p, gq, gk) if t))


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES + [(5000, 1250, 3, 2, 64, 32)], ids=lambda s: "x".join(map(str, s)))
def test_backward(shape, dtype, layout):
    ctx, alloc, be = env()
    rng = np.random.default_rng(zlib.crc32(repr((layout, dtype, shape)).encode()))
    n, seq, h, kv, d, rot = shape
    q, k, pitch, shift = operands(rng, shape, dtype, layout)
    dy = [rounded(rng.standard_normal(t.shape).astype(np.float32), dtype) for t in (q, k)]
    rows = seq + 3
    cos, sin = tables(rows, rot)
    given = layout == "packed"
    at = place(rng, n, seq, rows, given)
    weighted = layout != "shifted"
    gamma = (1 + 0.3 * rng.standard_normal((2, d))).astype(np.float32) if weighted else (None, None)
    x = [Rows(t, dtype, p, shift) for t, p in zip((q, k), pitch)]
    g = [Rows(t, dtype, None, shift) for t in dy]
    old = [rounded(rng.standard_normal(t.shape).astype(np.float32), dtype) for t in (q, k)]
    dx = [Rows(t, dtype, p, shift) for t, p in zip(old, pitch)]
    accumulate = layout == "dense"
    start = rng.standard_normal((2, d)).astype(np.float32)
    c, s, p, gq, gk, dgq, dgk = addresses(cos if rot else None, sin if rot else None, at if given else None, *gamma, *(start if weighted else (None, None)))
    need = ctx.qk_norm_partials_bytes(h, kv, d)
    part = up(np.full(need // 4 + 8, SENTINEL, np.float32))
    ctx.qk_norm_rope_backward(g[0].address, g[1].address, x[0].address, x[1].address, gq, gk, c, s, p, dx[0].address, dx[1].address, dgq, dgk,
                              part, need, n, seq, rows, h, kv, d, rot, g[0].stride, g[1].stride, x[0].stride, x[1].stride,
                              dx[0].stride, dx[1].stride, EPS, 1, accumulate, N.AG_BF16 if dtype == "bf16" else N.AG_F32)
    for i, (t, dyt, gam, out, dg) in enumerate(((q, dy[0], gamma[0], dx[0], dgq), (k, dy[1], gamma[1], dx[1], dgk))):
        ref, dgamma = R.heads_backward(dyt, t, gam, cos[at], sin[at], EPS)
        t = t.astype(np.float64)
        inv = 1 / np.sqrt(np.mean(t * t, -1, keepdims=True) + EPS)
        w = partner(dyt.astype(np.float64), rot)
        v = w * (1 if gam is None else np.abs(gam))
        bound = 80 * U * inv * (v + np.abs(t) * inv ** 2 * np.mean(v * np.abs(t), -1, keepdims=True))
        if accumulate:
            ref, bound = ref + old[i], bound + U * np.abs(ref + old[i])
        near(out.read(), ref, bound, dtype, "dx")
        if weighted:
            terms = n * t.shape[1]
            sizes = (w * np.abs(t) * inv).reshape(-1, d).sum(0)
            near(be.copy_to_host(dg).astype(np.float64), dgamma + start[i], (terms + 32) * U * sizes + U * np.abs(dgamma + start[i]), "f32", "dgamma")
    assert (be.copy_to_host(part)[need // 4:] == SENTINEL).all()
    for r in x + g:
        r.read()
    check_clean_status()
    free(part, *(r.whole for r in x + g + dx), *(t for t in (c, s, p, gq, gk, dgq, dgk) if t))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_in_place_and_by_the_backend(dtype):
    """Outputs in their inputs' place, inside packed rows; the backward's in the place of the incoming gradients."""
    ctx, alloc, be = env()
    rng = np.random.default_rng(2)
    b, t, h, kv, d = 2, 13, 6, 2, 64
    n, width = b * t, (h + 2 * kv) * d
    cos, sin = tables(t, d)
    at = np.arange(n) % t
    gamma = (1 + 0.3 * rng.standard_normal((2, d))).astype(np.float32)
    x = inputs(rng, n, h + 2 * kv, d, dtype)
    packed = up(f32_to_bf16_bits(x) if dtype == "bf16" else x)
    saved = up(f32_to_bf16_bits(x) if dtype == "bf16" else x)
    kind = np.uint16 if dtype == "bf16" else np.float32

    def part(whole, first, count):
        v = empty((0,))
        free(v)
        v.shape, v.dtype = (b, t, count, d), kind
        v.storage = alloc.view(whole.storage, first * d * size(dtype), (b, t, count, d), kind)
        return v
    q, k = part(packed, 0, h), part(packed, h, kv)
    q0, k0 = part(saved, 0, h), part(saved, h, kv)
    c, s, gq, gk = addresses(cos, sin, *gamma)
    be.qk_norm_rope_forward(q, k, c, s, q, k, EPS, q_gamma=gq, k_gamma=gk, q_stride=width, k_stride=width)
    got = np.asarray(be.copy_to_host(packed), np.float64)
    for lo, hi, g in ((0, h, gamma[0]), (h, h + kv, gamma[1])):
        near(got[:, lo:hi], R.heads(x[:, lo:hi], g, cos[at], sin[at], EPS), 32 * U * partner(R.heads(x[:, lo:hi], g, cos[at] * 0 + 1, sin[at] * 0, EPS), d),
             dtype, "in place")
    assert np.array_equal(got[:, h + kv:], x[:, h + kv:]), "values were touched"
    dgamma = up(np.zeros((2, d), np.float32))

    def row(i):
        v = empty((0,))
        free(v)
        v.shape, v.dtype, v.storage = (d,), np.float32, alloc.view(dgamma.storage, i * d * 4, (d,), np.float32)
        return v
    be.qk_norm_rope_backward(q, k, q0, k0, c, s, q, k, EPS, q_gamma=gq, k_gamma=gk, dq_gamma=row(0), dk_gamma=row(1), q_stride=width,
                             k_stride=width, dq_out_stride=width, dk_out_stride=width)
    back = np.asarray(be.copy_to_host(packed), np.float64)
    for i, (lo, hi) in enumerate(((0, h), (h, h + kv))):
        ref, dg = R.heads_backward(got[:, lo:hi], x[:, lo:hi], gamma[i], cos[at], sin[at], EPS)
        y = x[:, lo:hi].astype(np.float64)
        inv = 1 / np.sqrt(np.mean(y * y, -1, keepdims=True) + EPS)
        v = partner(got[:, lo:hi], d) * np.abs(gamma[i])
        near(back[:, lo:hi], ref, 80 * U * inv * (v + np.abs(y) * inv ** 2 * np.mean(v * np.abs(y), -1, keepdims=True)), dtype, "gradient in place")
        near(be.copy_to_host(dgamma)[i].astype(np.float64), dg, (n * h + 32) * U * (partner(got[:, lo:hi], d) * np.abs(y) * inv).reshape(-1, d).sum(0), "f32", "dgamma")
    check_clean_status()
    free(packed, saved, dgamma, c, s, gq, gk)


@pytest.mark.parametrize("n,h,kv,d", [(1, 1, 1, 8), (600, 6, 2, 128), (37, 3, 3, 74)])
def test_one_weight_for_queries_and_keys(n, h, kv, d):
    """Its gradient is the sum of both sides', many times over the same."""
    ctx, alloc, be = env()
    rng = np.random.default_rng(n)
    x = [inputs(rng, n, heads, d, "f32").reshape(1, n, heads, d) for heads in (h, kv)]
    dy = [rng.standard_normal(t.shape).astype(np.float32) for t in x]
    cos, sin = tables(n, d)
    gamma = (1 + 0.3 * rng.standard_normal(d)).astype(np.float32)
    c, s, g, q, k, dq, dk, ox, ok = (up(t) for t in (cos, sin, gamma, *x, *dy, *(np.zeros_like(t) for t in x)))
    ref, bound = np.ones(d), U * np.ones(d)
    for t, dyt in zip(x, dy):
        dgamma = R.heads_backward(dyt[0], t[0], gamma, cos, sin, EPS)[1]
        y = t[0].astype(np.float64)
        inv = 1 / np.sqrt(np.mean(y * y, -1, keepdims=True) + EPS)
        ref = ref + dgamma
        bound = bound + (n * (h + kv) + 32) * U * (partner(dyt[0].astype(np.float64), d) * np.abs(y) * inv).reshape(-1, d).sum(0)
    first = None
    for _ in range(20):
        dg = up(np.ones(d, np.float32))
        be.qk_norm_rope_backward(dq, dk, q, k, c, s, ox, ok, EPS, q_gamma=g, k_gamma=g, dq_gamma=dg, dk_gamma=dg)
        got = be.copy_to_host(dg)
        near(got.astype(np.float64), ref, bound + U * np.abs(ref), "f32", "dgamma")
        first = got if first is None else first
        assert np.array_equal(got, first)
        free(dg)
    check_clean_status()
    free(c, s, g, q, k, dq, dk, ox, ok)


@pytest.mark.parametrize("only", ["q", "k"])
def test_one_side_alone(only):
    ctx, alloc, be = env()
    rng = np.random.default_rng(4)
    x = inputs(rng, 10, 3, 32, "f32").reshape(2, 5, 3, 32)
    cos, sin = tables(5, 32)
    t, c, s, y, dx = up(x), up(cos), up(sin), up(np.zeros_like(x)), up(np.zeros_like(x))
    dg = up(np.zeros(32, np.float32))
    a = {"q": (t, None), "k": (None, t)}[only]
    be.qk_norm_rope_forward(*a, c, s, *((y, None) if only == "q" else (None, y)), EPS)
    ref = R.heads(x, None, cos[None], sin[None], EPS)
    near(be.copy_to_host(y).astype(np.float64), ref, 64 * U * partner(ref, 32) * 2, "f32", only)
    be.qk_norm_rope_backward(*((y, None) if only == "q" else (None, y)), *a, c, s, *((dx, None) if only == "q" else (None, dx)), EPS,
                             **{f"d{only}_gamma": dg})
    ref, dgamma = R.heads_backward(be.copy_to_host(y), x, None, cos[None], sin[None], EPS)
    got = be.copy_to_host(dx).astype(np.float64)
    # dy = y of unit weights: v x sums to D / inv, so that next to nothing is left of the difference of the two terms
    inv = 1 / np.sqrt(np.mean(x.astype(np.float64) ** 2, -1, keepdims=True) + EPS)
    v = partner(be.copy_to_host(y).astype(np.float64), 32)
    near(got, ref, 80 * U * inv * (v + np.abs(x) * inv ** 2 * np.mean(v * np.abs(x), -1, keepdims=True)), "f32", "dx")
    near(be.copy_to_host(dg).astype(np.float64), dgamma, (30 + 32) * U * (v * np.abs(x) * inv).reshape(-1, 32).sum(0), "f32", "dgamma")
    check_clean_status()
    free(t, c, s, y, dx, dg)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_nan_and_infinity_stay_in_their_head_and_positions_in_their_tables(dtype):
    ctx, alloc, be = env()
    rng = np.random.default_rng(8)
    n, h, d = 6, 4, 64
    x = inputs(rng, n, h, d, dtype)
    x[1, 2, 5], x[3, 0, 60] = np.nan, np.inf
    x[0, 1] = 1e-30                      # its squares are no numbers of 32 bits: y = x / sqrt(eps)
    cos, sin = tables(7, d)
    at = np.array([0, 6, -1, 3, 7, 2 ** 30], np.int32)
    kind = np.uint16 if dtype == "bf16" else np.float32
    word = f32_to_bf16_bits if dtype == "bf16" else np.ascontiguousarray
    gamma = np.ones(d, np.float32)
    t, c, s, p, y, g = up(word(x)), up(cos), up(sin), up(at), up(np.full(x.shape, 3, kind)), up(gamma)
    be.qk_norm_rope_forward(t, None, c, s, y, None, EPS, q_gamma=g, positions=p)
    assert ctx.status() == N.AG_STATUS_BAD_INDEX
    got = be.copy_to_host(y)
    assert not got[[2, 4, 5]].any()
    bad = np.zeros((n, h), bool)
    bad[1, 2] = bad[3, 0] = True
    assert np.isnan(got[1, 2]).all() and np.isnan(got[3, 0]).any() and np.isfinite(got[~bad]).all()
    ref = R.heads(x[0], gamma, cos[0][None], sin[0][None], EPS)
    near(got[0].astype(np.float64), ref, 64 * U * partner(ref, d) * 2, dtype, "others")
    dy, dx, dg = up(word(rounded(rng.standard_normal(x.shape).astype(np.float32), dtype))), up(np.full(x.shape, 3, kind)), up(np.zeros(d, np.float32))
    be.qk_norm_rope_backward(dy, None, t, None, c, s, dx, None, EPS, q_gamma=g, dq_gamma=dg, positions=p)
    assert ctx.status() == N.AG_STATUS_BAD_INDEX
    back = be.copy_to_host(dx)
    assert not back[[2, 4, 5]].any() and np.isnan(back[1, 2]).all() and np.isfinite(back[~bad]).all()
    free(t, c, s, p, y, g, dy, dx, dg)


def test_same_result_every_time_and_on_another_stream():
    """The weights' gradients are added in a fixed order, on any stream, in a recorded graph too."""
    import autograd_b200 as ag
    ctx, alloc, be = env()
    rng = np.random.default_rng(11)
    n, h, kv, d = 4096, 5, 2, 128
    q, k = inputs(rng, n, h, d, "f32"), inputs(rng, n, kv, d, "f32")
    cos, sin = tables(n, d)
    dy = rng.standard_normal(q.shape).astype(np.float32), rng.standard_normal(k.shape).astype(np.float32)
    tq, tk, c, s, dq, dk, gq, gk = (up(a) for a in (q, k, cos, sin, *dy, np.zeros_like(q), np.zeros_like(k)))
    results = []
    other = ag.create(0)
    ctx.synchronize()
    for backend, times, graph in ((be, 2, False), (other[2], 1, False), (be, 1, True)):
        for _ in range(times):
            w = [up(np.zeros(d, np.float32)) for _ in range(2)]
            ctx.synchronize()

            def call(b):
                b.qk_norm_rope_backward(dq, dk, tq, tk, c, s, gq, gk, EPS, dq_gamma=w[0], dk_gamma=w[1])
            if graph:
                need = ctx.qk_norm_partials_bytes(h, kv, d)
                part = up(np.zeros(need, np.uint8))

                def launches(rec):
                    rec.qk_norm_rope_backward(dq, dk, tq, tk, 0, 0, c, s, 0, gq, gk, w[0], w[1], part, need, n, n, n, h, kv, d, d,
                                              h * d, kv * d, h * d, kv * d, h * d, kv * d, EPS)
                rec = ctx.record(launches)
                ctx.replay(rec)
                ctx.synchronize()
                ctx.drop_recording(rec)
                free(part)
            else:
                call(backend)
                backend.synchronize()
            results.append([be.copy_to_host(t) for t in (gq, gk, *w)])
            free(*w)
    for r in results[1:]:
        assert all(np.array_equal(a, b) for a, b in zip(results[0], r))
    check_clean_status()
    other[0].check_status()
    free(tq, tk, c, s, dq, dk, gq, gk)


def test_no_tokens():
    ctx, alloc, be = env()
    t, c = up(np.zeros((0, 4, 64), np.float32)), up(np.zeros((4, 32), np.float32))
    be.qk_norm_rope_forward(t, None, c, c, t, None, EPS)
    be.qk_norm_rope_backward(t, None, t, None, c, c, t, None, EPS)
    check_clean_status()
    free(c)


def test_beyond_32_bits_of_elements():
    """Rows that far apart that the last token lies behind 2^32 elements."""
    ctx, alloc, be = env()
    n, d, stride = 5, 64, 1_100_000_000
    whole = alloc.alloc((4 * stride + d,), np.uint16)
    rng = np.random.default_rng(1)
    x = rounded(rng.standard_normal((n, 1, d)).astype(np.float32), "bf16")
    base = whole.ptr.address
    for i in range(n):
        ctx.copy_from_host(base + i * stride * 2, f32_to_bf16_bits(x[i, 0]))
    cos, sin = tables(n, d)
    c, s, y = up(cos), up(sin), up(np.zeros((n, 1, d), np.uint16))
    ctx.qk_norm_rope_forward(base, 0, 0, 0, c, s, 0, y, 0, n, n, n, 1, 0, d, d, stride, 0, d, 0, EPS, 1, N.AG_BF16)
    ref = R.heads(x, None, cos, sin, EPS)
    near(be.copy_to_host(y).astype(np.float64), ref, 64 * U * partner(ref, d) * 2, "bf16", "y")
    check_clean_status()
    free(c, s, y)
    alloc.free(whole)
