"""Log-probabilities of given tokens, entropies and likeliest tokens, and their gradient, against the 64-bit forms.

Bounds, in units u = 2^-24 (half a step of fp32): (x - m) / temperature is off by 4 u of itself (three roundings and the one of
1 / temperature); the sum of exponentials by 2^-22 = 4 u for each exponential, what its argument is off by (weighted by p:
4 u (L - H) <= 50 u), and a rounding per addition of a chain, at most 200 of them (a thread's terms, the threads, the blocks):
L by less than 300 u.  So a log-probability is off by (300 + 8 |lp|) u, and an entropy, the difference of L and a sum that is off
by 300 u of itself, by 300 (2 + L + H) u.  A gradient term p (...) is off by what p is: (300 + 16 |lp|) u of itself.  Gradients
stored in bf16 add 2^-8 of their value."""
import numpy as np
import pytest

from autograd_b200.backend import bf16_bits_to_f32, f32_to_bf16_bits
from gpu_util import check_clean_status, empty, env, free, up
from oracle import vocab_rows as R

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
LOWEST = {"f32": np.float32(-3.4028235e38), "bf16": np.float32(-3.3895314e38)}
SENTINEL = 777.0


def rounded(x, dtype):
    return bf16_bits_to_f32(f32_to_bf16_bits(x)) if dtype == "bf16" else np.ascontiguousarray(x, np.float32)


def rows_of(rng, n, v, dtype):
    """Rows where such a kernel goes wrong, as far as n reaches; the last ones are ordinary."""
    x = (rng.standard_normal((n, v)) * 2).astype(np.float32)
    low = LOWEST[dtype]
    kinds = [
        lambda r: np.where(rng.random(v) < 0.9, -np.inf, r),
        lambda r: np.full(v, -np.inf),
        lambda r: np.where(np.arange(v) == v // 2, 1.5, -np.inf),
        lambda r: np.where(rng.random(v) < 0.5, low, r),
        lambda r: np.full(v, low),
        lambda r: np.zeros(v),
        lambda r: np.where(rng.random(v) < 0.5, 0.0, -0.0),
        lambda r: np.where(np.arange(v) == v - 1, np.nan, r),
        lambda r: np.where(np.arange(v) == 0, np.inf, r),
        lambda r: r + 3e4,
        lambda r: np.sort(r),
        lambda r: np.sort(r)[::-1],
        lambda r: np.round(r),
        lambda r: np.where(np.arange(v) == v // 3, 60.0, r),
        lambda r: np.where(rng.random(v) < 0.01, r, -1e4),
        lambda r: np.full(v, np.nan),
        lambda r: np.where(np.arange(v) % 2 == 0, -np.inf, low),
    ]
    for i, f in enumerate(kinds[:n]):
        x[i] = f(x[i])
    return rounded(x, dtype)


def words(x, dtype):
    return f32_to_bf16_bits(x) if dtype == "bf16" else np.ascontiguousarray(x, np.float32)


def store(x, dtype, ld=None, shift=0):
    """Rows on the device, ld elements apart, the first one `shift` elements behind an aligned address; what is between is NaN."""
    ctx, alloc, be = env()
    n, v = x.shape
    ld = v if ld is None else ld
    host = np.full(shift + n * ld, np.nan, np.float32)
    host[shift:].reshape(n, ld)[:, :v] = x
    whole = up(words(host, dtype))
    size = 2 if dtype == "bf16" else 4
    t = empty((0,))
    free(t)
    t.shape, t.dtype = (n, ld), whole.storage.dtype
    t.storage = alloc.view(whole.storage, shift * size, (n, ld), whole.storage.dtype)
    return t, whole


def fetch(t, whole_count, dtype):
    ctx, alloc, be = env()
    raw = ctx.copy_to_host(t.storage.ptr.buffer_id, (whole_count,), np.uint16 if dtype == "bf16" else np.float32)
    return bf16_bits_to_f32(raw) if dtype == "bf16" else raw


def near(got, ref, bound, what):
    """Equal where ref is infinite or NaN, within bound elsewhere."""
    got, ref = np.asarray(got, np.float64), np.asarray(ref, np.float64)
    # the outputs are 32-bit numbers: what lies half a step beyond the largest of them, (2 - 2^-24) 2^127, rounds to infinity
    # (a logit of -3.4e38 at temperature 0.7 has the log-probability -4.9e38)
    ref = np.where(np.abs(ref) >= (2 - 2.0 ** -24) * 2.0 ** 127, np.copysign(np.inf, ref), ref)
    finite = np.isfinite(ref)
    assert np.array_equal(np.isnan(got), np.isnan(ref)), (what, "NaN", np.argwhere(np.isnan(got) != np.isnan(ref))[:5])
    same = ~finite & ~np.isnan(ref)
    assert np.array_equal(got[same], ref[same]), (what, "infinities")
    off = np.abs(got[finite] - ref[finite]) - np.broadcast_to(bound, ref.shape)[finite]
    if off.size and off.max() > 0:
        i = np.argwhere(finite)[off.argmax()]
        raise AssertionError(f"{what}: at {tuple(i)}: {got[tuple(i)]!r} instead of {ref[tuple(i)]!r}, {off.max():.3e} beyond the bound")


def forward(x, ids, dtype, top=0, temperature=1.0, ld=None, shift=0, stats=True):
    ctx, alloc, be = env()
    n, v = x.shape
    t, whole = store(x, dtype, ld, shift)
    keep = [whole]
    row = up(np.full(n + 3, SENTINEL, np.float32))   # three elements behind the last row, which stay
    ent = up(np.full(n + 3, SENTINEL, np.float32))
    st = up(np.full((n + 1, 4), SENTINEL, np.float32)) if stats else None
    ti = up(np.full((n + 1) * max(top, 1), 77, np.int32)) if top else None
    tl = up(np.full((n + 1) * max(top, 1), SENTINEL, np.float32)) if top else None
    tid = up(ids.astype(np.int32)) if ids is not None else None
    keep += [row, ent, st, ti, tl, tid]
    ctx.token_logprobs_forward(t, t.shape[1], tid, row if ids is not None else None, ent, st, ti, tl, n, v, top, temperature,
                               1 if dtype == "bf16" else 0)
    out = {"logprob": be.copy_to_host(row), "entropy": be.copy_to_host(ent)}
    if stats:
        out["stats"] = be.copy_to_host(st)
        assert (out["stats"][n:] == SENTINEL).all()
        out["stats"] = out["stats"][:n]
    if top:
        out["top_ids"], out["top_logprobs"] = be.copy_to_host(ti), be.copy_to_host(tl)
        assert (out["top_ids"][n * top:] == 77).all() and (out["top_logprobs"][n * top:] == SENTINEL).all()
        out["top_ids"], out["top_logprobs"] = (out[k][:n * top].reshape(n, top) for k in ("top_ids", "top_logprobs"))
    for k in ("logprob", "entropy"):
        assert (out[k][n:] == SENTINEL).all(), k
        out[k] = out[k][:n]
    free(*keep)
    return out


def check_forward(x, ids, out, top, temperature):
    lp_id, h, lp, m, total = R.token_logprobs(x, ids, temperature)
    with np.errstate(all="ignore"):
        near(out["logprob"], lp_id, (300 + 8 * np.abs(lp_id)) * U, "log-probability")
        near(out["entropy"], h, 300 * (2 + np.abs(total) + h) * U, "entropy")
        if "stats" in out:
            assert np.array_equal(out["stats"][:, 0][~np.isnan(total)], m[~np.isnan(total)].astype(np.float32))
            near(out["stats"][:, 1], total, 300 * U + np.abs(total) * U, "log of the sum")
            near(out["stats"][:, 2], h, 300 * (2 + np.abs(total) + h) * U, "entropy in the statistics")
            assert not out["stats"][:, 3].any()
        if top:
            at = R.top(x, top)
            assert np.array_equal(out["top_ids"], at), np.argwhere(out["top_ids"] != at)[:5]
            ref = np.take_along_axis(lp, at.astype(np.int64), 1)
            near(out["top_logprobs"], ref, (300 + 8 * np.abs(ref)) * U, "alternatives")


VOCABS = [1, 2, 3, 7, 31, 33, 127, 128, 129, 640, 1000, 1026, 4099, 5003, 16384, 32768, 50257]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("v", VOCABS)
def test_forward(v, dtype):
    rng = np.random.default_rng(v)
    n = 20
    x = rows_of(rng, n, v, dtype)
    ids = rng.integers(0, v, n)
    ids[18], ids[19] = -1, v
    top = min(v, 20)
    for temperature in (1.0, 0.7):
        check_forward(x, ids, forward(x, ids, dtype, top, temperature), top, temperature)
    check_clean_status()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("v,n", [(151936, 3), (151936, 19), (393216, 18), (262145, 2), (100003, 1)])
def test_forward_wide(v, n, dtype):
    rng = np.random.default_rng(v + n)
    x = rows_of(rng, n, v, dtype)[::-1]     # the ordinary rows first, so that few rows have them
    ids = rng.integers(0, v, n)
    for top in (0, 128):
        check_forward(x, ids, forward(x, ids, dtype, top, 1.3), top, 1.3)
    check_clean_status()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("top", [1, 2, 5, 31, 32, 33, 64, 100, 127, 128])
def test_alternatives(top, dtype):
    rng = np.random.default_rng(top)
    for n, v in ((1, 128), (17, 129), (300, 1000), (40, 5003), (20, 32768), (5, 65537)):
        x = rows_of(rng, n, v, dtype)
        check_forward(x, np.zeros(n, np.int64), forward(x, np.zeros(n), dtype, top), top, 1.0)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_alternatives_of_rows_with_many_equal_logits(dtype):
    """A threshold that many logits equal, or that nearly all of a row pass."""
    rng = np.random.default_rng(5)
    for v in (1000, 32768, 50257):
        x = np.zeros((12, v), np.float32)
        x[0, rng.permutation(v)[:40]] = 1.0
        x[1, rng.permutation(v)[:200]] = 1.0
        x[2, v // 2:] = 1.0
        x[3] = np.arange(v) / v
        x[4] = -np.arange(v) / v
        x[5] = rng.integers(0, 3, v)
        x[6, -130:] = 2.0
        x[7, :130] = 2.0
        x[8] = np.where(np.arange(v) % 4 == 0, 5.0 + np.arange(v) / v, 0.0)
        x[9] = np.where(np.arange(v) // 4 % 512 == 3, 5.0 + np.arange(v) / v, -1.0)
        x[10] = np.where(np.arange(v) < v // 8, 3.0 + rng.random(v), 0.0)
        x[11] = np.where(np.arange(v) >= v - v // 8, 3.0 + np.arange(v) / v, 0.0)
        x = rounded(x, dtype)
        for top in (1, 20, 128):
            check_forward(x, np.zeros(12, np.int64), forward(x, np.zeros(12), dtype, top), top, 1.0)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("mask", [-np.inf, -1e9, None])
def test_alternatives_where_few_tokens_are_allowed(mask, dtype):
    """Fewer than are asked for, or hardly more; the others masked with -inf, a large number, the lowest one."""
    rng = np.random.default_rng(6)
    mask = LOWEST[dtype] if mask is None else mask
    for n, v in ((600, 5003), (40, 32768), (3, 50257)):
        x = np.full((n, v), mask, np.float32)
        for r in range(n):
            x[r, rng.permutation(v)[:(0, 1, 5, 19, 20, 21, 60)[r % 7]]] = rng.standard_normal((0, 1, 5, 19, 20, 21, 60)[r % 7])
        x = rounded(x, dtype)
        for top in (20, 128):
            check_forward(x, np.zeros(n, np.int64), forward(x, np.zeros(n), dtype, top), top, 1.0)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 2, 9, 64, 147, 148, 149, 300, 1200, 5000])
def test_forward_row_counts(rows, dtype):
    rng = np.random.default_rng(rows)
    for v in (333, 4000, 40000 if rows < 2000 else 640):
        x = rounded(rng.standard_normal((rows, v)).astype(np.float32) * 3, dtype)
        ids = rng.integers(-1, v, rows)
        check_forward(x, ids, forward(x, ids, dtype, 7, 0.9), 7, 0.9)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shift", [0, 1, 2, 3, 5, 7])
@pytest.mark.parametrize("pad", [0, 1, 2, 3, 8, 47])
def test_strides_and_shifts(shift, pad, dtype):
    rng = np.random.default_rng(shift * 50 + pad)
    for v in (5, 640, 1001, 20001):
        x = rounded(rng.standard_normal((6, v)).astype(np.float32) * 3, dtype)
        ids = rng.integers(0, v, 6)
        out = forward(x, ids, dtype, min(v, 9), 1.0, v + pad, shift)
        check_forward(x, ids, out, min(v, 9), 1.0)
        a, b = rng.standard_normal(6), rng.standard_normal(6)
        check_backward(x, ids, a, b, dtype, 1.0, ld=v + pad, shift=shift, ld_grad=v + pad, shift_grad=shift)
        check_backward(x, ids, a, b, dtype, 1.0, ld=v + pad, shift=shift, ld_grad=v + 5, shift_grad=0)


def check_backward(x, ids, a, b, dtype, temperature, ld=None, shift=0, ld_grad=None, shift_grad=0, dres=None, place=None):
    """place: None, "logits" (the gradient takes their place) or "dres" (it is added to what is there)."""
    ctx, alloc, be = env()
    n, v = x.shape
    a = None if a is None else a.astype(np.float32)
    b = None if b is None else b.astype(np.float32)
    ld = v if ld is None else ld
    t, whole = store(x, dtype, ld, shift)
    _, h, lp, m, total = R.token_logprobs(x, ids, temperature)
    st = up(np.stack([m, total, h, np.zeros(n)], 1).astype(np.float32))
    tid, ta, tb = up(ids.astype(np.int32)), None if a is None else up(a), None if b is None else up(b)
    if place == "logits":
        out, whole_out, ld_grad, shift_grad = t, whole, ld, shift
    else:
        ld_grad = v if ld_grad is None else ld_grad
        out, whole_out = store(np.full((n, v), SENTINEL) if place != "dres" else dres, dtype, ld_grad, shift_grad)
    tr = whole_r = None
    if place == "dres":
        tr = out
    elif dres is not None:
        tr, whole_r = store(dres, dtype, ld_grad, shift_grad)
    ctx.token_logprobs_backward(t, ld, tid, st, ta, tb, tr, out, ld_grad, n, v, temperature, 1 if dtype == "bf16" else 0)
    got = fetch(out, shift_grad + n * ld_grad, dtype)
    rows = got[shift_grad:].reshape(n, ld_grad)
    assert np.isnan(got[:shift_grad]).all() and np.isnan(rows[:, v:]).all(), "written beside the rows"
    ref, size, _ = R.token_logprobs_backward(x, ids, a, b, temperature)
    if dres is not None:
        ref = ref + dres
        size = size + np.abs(dres)
    with np.errstate(all="ignore"):
        bound = size * (300 + 16 * np.where(np.isfinite(lp), np.abs(lp), 0.0)) * U
        if dtype == "bf16":
            bound = bound + np.abs(ref) * 2.0 ** -8 + 2.0 ** -133  # half a step, of the smallest numbers too
        # exponentials below 2^-126 are zero
        bound = bound + 2.0 ** -126 * (2 + (0 if a is None else np.abs(a).max()) + (0 if b is None else 200 * np.abs(b).max())) / temperature
    near(rows[:, :v], ref, bound, "gradient")
    free(*{id(w): w for w in (whole, whole_out, whole_r, st, tid, ta, tb) if w is not None}.values())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("v", VOCABS)
def test_backward(v, dtype):
    rng = np.random.default_rng(v + 1)
    n = 20
    x = rows_of(rng, n, v, dtype)
    ids = rng.integers(0, v, n)
    ids[18], ids[19] = -1, v
    a, b = rng.standard_normal(n), rng.standard_normal(n)
    a[17], b[17] = 0.0, 0.0
    check_backward(x, ids, a, b, dtype, 1.0)
    check_backward(x, ids, a, None, dtype, 0.7)
    check_backward(x, ids, None, b, dtype, 2.0)
    dres = rounded(rng.standard_normal((n, v)).astype(np.float32), dtype)
    check_backward(x, ids, a, b, dtype, 1.0, dres=dres)
    check_backward(x, ids, a, b, dtype, 1.0, dres=dres, place="dres")
    check_backward(x, ids, a, b, dtype, 1.0, place="logits")
    check_clean_status()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,v", [(1, 151936), (3, 500001), (149, 4000), (3000, 129), (700, 8191)])
def test_backward_sizes(rows, v, dtype):
    rng = np.random.default_rng(rows)
    x = rounded(rng.standard_normal((rows, v)).astype(np.float32) * 3, dtype)
    ids = rng.integers(-1, v, rows)
    check_backward(x, ids, rng.standard_normal(rows), rng.standard_normal(rows) * 0.1, dtype, 1.0)


def test_rows_without_gradient_do_not_read_their_logits():
    """A row of weight 0 (padding) may hold anything, NaN too."""
    x = np.full((3, 100), np.nan, np.float32)
    x[1] = np.arange(100) / 50
    ctx, alloc, be = env()
    t, whole = store(x, "f32")
    _, h, _, m, total = R.token_logprobs(x, np.zeros(3, np.int64))
    st = up(np.stack([m, total, h, np.zeros(3)], 1).astype(np.float32))
    a, ids, out = up(np.array([0, 1, 0], np.float32)), up(np.array([5, 5, -1], np.int32)), up(np.full((3, 100), 9.0, np.float32))
    ctx.token_logprobs_backward(t, 100, ids, st, a, None, None, out, 100, 3, 100)
    got = be.copy_to_host(out)
    assert not got[0].any() and not got[2].any() and np.isfinite(got[1]).all() and got[1, 5] > 0
    free(whole, st, a, ids, out)


def test_outputs_may_be_left_out_and_agree():
    ctx, alloc, be = env()
    rng = np.random.default_rng(8)
    x = rng.standard_normal((30, 777)).astype(np.float32)
    ids = rng.integers(0, 777, 30)
    full = forward(x, ids, "f32", 11)
    assert np.array_equal(forward(x, ids, "f32", 11, stats=False)["top_ids"], full["top_ids"])
    t, e, h = up(x), up(np.zeros(30, np.float32)), up(ids.astype(np.int32))
    be.token_logprobs_forward(t, None, None, entropy=e)
    assert np.array_equal(be.copy_to_host(e), forward(x, None, "f32")["entropy"])
    be.token_logprobs_forward(t, h, e)
    assert np.array_equal(be.copy_to_host(e), forward(x, ids, "f32")["logprob"])
    be.token_logprobs_forward(t, None, None)  # nothing asked for
    free(t, e, h)


def test_the_same_call_gives_the_same_bits():
    rng = np.random.default_rng(9)
    for n, v, dtype in ((3, 151936, "bf16"), (500, 5003, "f32"), (700, 32768, "f32")):
        x = rounded(rng.standard_normal((n, v)).astype(np.float32) * 2, dtype)
        ids = rng.integers(0, v, n)
        first = forward(x, ids, dtype, 33)
        for _ in range(3):
            again = forward(x, ids, dtype, 33)
            assert all(np.array_equal(first[k], again[k]) for k in first)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_beyond_31_bits_of_elements(dtype):
    """Three rows 2^30 elements apart and more: the last one starts beyond 2^31."""
    ctx, alloc, be = env()
    v, ld = 2001, (1 << 30) + 24
    size = 2 if dtype == "bf16" else 4
    rng = np.random.default_rng(3)
    x = rounded(rng.standard_normal((3, v)).astype(np.float32), dtype)
    ids = np.array([0, 5, 2000])
    big = alloc.alloc((2 * ld + v,), np.uint16 if dtype == "bf16" else np.float32)
    base = big.ptr.address
    for r in range(3):
        ctx.copy_from_host(base + r * ld * size, words(x[r], dtype))
    lp, ent, st = up(np.zeros(3, np.float32)), up(np.zeros(3, np.float32)), up(np.zeros((3, 4), np.float32))
    ti, tl, tid, a = up(np.zeros((3, 6), np.int32)), up(np.zeros((3, 6), np.float32)), up(ids.astype(np.int32)), up(np.ones(3, np.float32))
    ctx.token_logprobs_forward(base, ld, tid, lp, ent, st, ti, tl, 3, v, 6, 1.0, 1 if dtype == "bf16" else 0)
    check_forward(x, ids, {"logprob": be.copy_to_host(lp), "entropy": be.copy_to_host(ent), "top_ids": be.copy_to_host(ti),
                           "top_logprobs": be.copy_to_host(tl), "stats": be.copy_to_host(st)}, 6, 1.0)
    ctx.token_logprobs_backward(base, ld, tid, st, a, None, None, base, ld, 3, v, 1.0, 1 if dtype == "bf16" else 0)
    ref, size_, l = R.token_logprobs_backward(x, ids, np.ones(3), None)
    for r in range(3):
        raw = ctx.copy_to_host(base + r * ld * size, (v,), np.uint16 if dtype == "bf16" else np.float32)
        got = bf16_bits_to_f32(raw) if dtype == "bf16" else raw
        near(got, ref[r], size_[r] * (700 + 16 * np.abs(l[r])) * U + (np.abs(ref[r]) * 2.0 ** -8 if dtype == "bf16" else 0), "gradient")
    ctx.synchronize()
    alloc.free(big)
    free(lp, ent, st, ti, tl, tid, a)


def test_recorded_calls_follow_their_inputs():
    """Two recordings that are replayed in turn, with other logits each time, beside eager calls."""
    ctx, alloc, be = env()
    rng = np.random.default_rng(12)
    n, v, top = 37, 5003, 9
    t = [up(np.zeros((n, v), np.float32)) for _ in range(2)]
    out = [{"logprob": up(np.zeros(n, np.float32)), "entropy": up(np.zeros(n, np.float32)), "stats": up(np.zeros((n, 4), np.float32)),
            "top_ids": up(np.zeros((n, top), np.int32)), "top_logprobs": up(np.zeros((n, top), np.float32))} for _ in range(2)]
    grad = [up(np.zeros((n, v), np.float32)) for _ in range(2)]
    ids = rng.integers(0, v, n)
    tid, a = up(ids.astype(np.int32)), up(np.ones(n, np.float32))

    def calls(c, i):
        o = out[i]
        c.token_logprobs_forward(t[i], v, tid, o["logprob"], o["entropy"], o["stats"], o["top_ids"], o["top_logprobs"], n, v, top)
        c.token_logprobs_backward(t[i], v, tid, o["stats"], a, a, None, grad[i], v, n, v)
    for i in range(2):
        calls(ctx, i)
    ctx.synchronize()
    graphs = [ctx.record(lambda c, i=i: calls(c, i)) for i in range(2)]
    for _ in range(3):
        x = [rng.standard_normal((n, v)).astype(np.float32) for _ in range(2)]
        for i in range(2):
            be.copy_from_host(t[i], x[i])
        for i in range(2):
            ctx.replay(graphs[i])
        for i in range(2):
            check_forward(x[i], ids, {k: be.copy_to_host(w) for k, w in out[i].items()}, top, 1.0)
            ref, size, lp = R.token_logprobs_backward(x[i], ids, np.ones(n), np.ones(n))
            near(be.copy_to_host(grad[i]), ref, size * (700 + 16 * np.abs(lp)) * U + 2.0 ** -118, "gradient")
    for g in graphs:
        ctx.drop_recording(g)
    free(*t, *grad, tid, a, *(w for o in out for w in o.values()))
    check_clean_status()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,v", [(700, 1003), (700, 9003), (700, 20003), (300, 33003), (24, 33003), (3, 50257)])
def test_edges_of_rows_whose_logits_all_reach_the_bound(n, v, dtype):
    """Rows that start and end between two 16-byte boundaries, where far more logits pass than there is room for: what lies beside
    the packets finds the list full, whichever warp comes first.  With 64, 128, 256 threads per row and with blocks that share one."""
    rng = np.random.default_rng(v)
    x = np.zeros((n, v), np.float32)
    x[1::3] = 2.5
    x[2::3] = rng.integers(0, 2, (len(x[2::3]), v))
    x = rounded(x, dtype)
    for top in (1, 2, 20, 128):
        for shift, pad in ((1, 0), (3, 1), (0, 2)):
            check_forward(x, np.zeros(n, np.int64), forward(x, np.zeros(n), dtype, top, 1.0, v + pad, shift), top, 1.0)
    check_clean_status()
