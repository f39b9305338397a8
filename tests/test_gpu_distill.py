"""Distillation from a teacher's top logits, against the 64-bit forms.

Bounds in units u = 2^-24, as in the tests of log-probabilities: ln p is off by (300 + 8 |ln p|) u; q by 8 u and 4 u |t / temperature|
of itself, ln q by as much; r = 1 - sum q by 8 u (1 + sum q |t|) <= 40 u of 1 and ln r by that over r; ln p_rest like ln p.  So a
row's loss is off by 400 u of the sizes of its terms, where r's are taken whole (|ln r| + |ln p_rest| + 1 instead of r times
them).  A gradient's terms are off by (400 + 16 |ln p|) u of themselves, r p / p_rest also by 40 u of p / p_rest (the oracle's
`size` has a tenth of that ratio in it).  Gradients stored in bf16 add 2^-8 of their value.  The loss adds a rounding of its sum's
size."""
import numpy as np
import pytest

import autograd_b200 as ag
from autograd_b200.backend import bf16_bits_to_f32, f32_to_bf16_bits
from gpu_util import check_clean_status, down, empty, env, free, up
from oracle import vocab_rows as R
from test_gpu_logprobs import LOWEST, SENTINEL, U, fetch, near, rounded, rows_of, store, words

pytestmark = pytest.mark.gpu


def teacher_of(rng, n, v, top, rest):
    """Lists with unused slots, repeated tokens, tokens of probability 0, rows without any."""
    ids = np.stack([rng.permutation(v)[:top] if v >= top else rng.integers(0, v, top) for _ in range(n)]).astype(np.int32)
    t = rng.standard_normal((n, top)).astype(np.float32) * 2
    if rest:
        with np.errstate(all="ignore"):
            t = t - np.log(np.sum(np.exp(t.astype(np.float64)), 1, keepdims=True)) + np.log(rng.uniform(0.3, 0.98, (n, 1)))
        t = t.astype(np.float32)
    ids[2::7, top // 2:] = -1
    if n > 3:
        ids[3] = -5
    if n > 5 and top > 2:
        ids[5, 1] = ids[5, 0]
        t[5, 2] = -np.inf
    if n > 6:
        t[6] = -np.inf
    return ids, t


def run(x, ids, t, dtype, what, row_scale=None, dloss=1.0, temperature=1.0, rest=False, ld=None, shift=0, ld_grad=None,
        shift_grad=0, place=None, dres=None):
    """what: "both" (forward_backward) or "apart" (forward, then backward from its statistics)."""
    ctx, alloc, be = env()
    n, v = x.shape
    top = ids.shape[1]
    d, mode = (1 if dtype == "bf16" else 0), (ag.AG_DISTILL_REST if rest else ag.AG_DISTILL_RENORM)
    ld = v if ld is None else ld
    tx, whole = store(x, dtype, ld, shift)
    if place == "logits":
        out, whole_out, ld_grad, shift_grad = tx, whole, ld, shift
    else:
        ld_grad = v if ld_grad is None else ld_grad
        out, whole_out = store(np.full((n, v), SENTINEL) if place != "dres" else dres, dtype, ld_grad, shift_grad)
    tr = whole_r = None
    if place == "dres":
        tr = out
    elif dres is not None:
        tr, whole_r = store(dres, dtype, ld_grad, shift_grad)
    ti, tt = up(ids), up(t)
    w = None if row_scale is None else up(np.asarray(row_scale, np.float32))
    dl, loss = up(np.array([dloss], np.float32)), up(np.array([SENTINEL] * 2, np.float32))
    row, st = up(np.full(n + 3, SENTINEL, np.float32)), up(np.full((n + 1, 4), SENTINEL, np.float32))
    if what == "both":
        ctx.distill_forward_backward(tx, ld, ti, tt, w, dl, loss, row, st, out, ld_grad, n, v, top, temperature, mode, d)
    else:
        ctx.distill_forward(tx, ld, ti, tt, w, loss, row, st, n, v, top, temperature, mode, d)
        ctx.distill_backward(tx, ld, ti, tt, w, st, dl, tr, out, ld_grad, n, v, top, temperature, mode, d)
    got = fetch(out, shift_grad + n * ld_grad, dtype)
    rows = got[shift_grad:].reshape(n, ld_grad)
    assert np.isnan(got[:shift_grad]).all() and np.isnan(rows[:, v:]).all(), "written beside the rows"
    r, s, l = down(row), down(st), down(loss)
    assert (r[n:] == SENTINEL).all() and (s[n:] == SENTINEL).all() and l[1] == SENTINEL
    free(*{id(q): q for q in (whole, whole_out, whole_r, ti, tt, w, dl, loss, row, st) if q is not None}.values())
    return {"row_loss": r[:n], "loss": l[0], "dlogits": rows[:, :v].copy(), "stats": s[:n]}


def check(x, ids, t, dtype, what, dres=None, **kw):
    got = run(x, ids, t, dtype, what, dres=dres, **kw)
    scale = kw.get("row_scale")
    ref = R.distill(x, ids, t, None if scale is None else np.asarray(scale, np.float32), np.float32(kw.get("dloss", 1.0)),
                    kw.get("temperature", 1.0), kw.get("rest", False))
    with np.errstate(all="ignore"):
        near(got["row_loss"], ref["row_loss"], 400 * U * ref["loss_size"], "loss of a row")
        take = ref["weight"] != 0
        near(got["loss"], ref["loss"], U * np.sum(np.abs(ref["weight"][take]) * (400 * ref["loss_size"][take])) + U * abs(ref["loss"])
             + 2 * U * np.sum(np.abs(ref["weight"][take] * ref["row_loss"][take])), "loss")
        g, size = ref["dlogits"], ref["size"]
        if dres is not None:
            g, size = g + dres, size + np.abs(dres)
        bound = size * (400 + 16 * np.where(np.isfinite(ref["lp"]), np.abs(ref["lp"]), 0.0)) * U + 2.0 ** -120
        if dtype == "bf16":
            bound = bound + np.abs(g) * 2.0 ** -8 + 2.0 ** -133
    near(got["dlogits"], g, bound, "gradient")
    return got


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("v", [1, 2, 5, 33, 128, 640, 1001, 4099, 16384, 32768, 50257])
def test_distill(v, rest, dtype):
    rng = np.random.default_rng(v)
    n, top = 24, min(v, 19)
    x = rows_of(rng, n, v, dtype)
    ids, t = teacher_of(rng, n, v, top, rest)
    w = rng.random(n)
    w[20] = 0.0
    for what in ("both", "apart"):
        check(x, ids, t, dtype, what, rest=rest)
        check(x, ids, t, dtype, what, rest=rest, row_scale=w, dloss=0.37, temperature=1.7)
        check(x, ids, t, dtype, what, rest=rest, place="logits")
    dres = rounded(rng.standard_normal((n, v)).astype(np.float32), dtype)
    check(x, ids, t, dtype, "apart", rest=rest, dres=dres)
    check(x, ids, t, dtype, "apart", rest=rest, dres=dres, place="dres")
    check_clean_status()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("top", [1, 2, 31, 32, 33, 100, 255, 256])
def test_lengths_of_the_list(top, dtype):
    rng = np.random.default_rng(top)
    for n, v in ((9, 256), (40, 1000), (12, 50257)):
        x = rounded(rng.standard_normal((n, v)).astype(np.float32) * 2, dtype)
        for rest in (False, True):
            ids, t = teacher_of(rng, n, v, top, rest)
            for what in ("both", "apart"):
                check(x, ids, t, dtype, what, rest=rest)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,v", [(1, 151936), (19, 151936), (2, 393216), (5000, 640), (700, 5000), (149, 32768), (300, 100)])
def test_sizes(n, v, dtype):
    rng = np.random.default_rng(n)
    x = rounded(rng.standard_normal((n, v)).astype(np.float32) * 2, dtype)
    for rest in (False, True):
        ids, t = teacher_of(rng, n, v, 40, rest)
        for what in ("both", "apart"):
            check(x, ids, t, dtype, what, rest=rest)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shift", [0, 1, 3, 6])
@pytest.mark.parametrize("pad", [0, 1, 2, 8, 47])
def test_strides_and_shifts(shift, pad, dtype):
    rng = np.random.default_rng(shift * 50 + pad)
    for v in (9, 641, 20001):
        x = rounded(rng.standard_normal((6, v)).astype(np.float32) * 2, dtype)
        ids, t = teacher_of(rng, 6, v, 7, True)
        for what in ("both", "apart"):
            check(x, ids, t, dtype, what, rest=True, ld=v + pad, shift=shift, ld_grad=v + pad, shift_grad=shift)
            check(x, ids, t, dtype, what, rest=True, ld=v + pad, shift=shift, ld_grad=v + 3, shift_grad=2)
            check(x, ids, t, dtype, what, rest=False, ld=v + pad, shift=shift, place="logits")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_small_rest_keeps_its_digits(dtype):
    """The student gives everything but 1e-7 to the listed tokens: 1 - sum would have one digit of that left."""
    n, v = 4, 3000
    x = np.zeros((n, v), np.float32)
    x[:, :4] = 24.0
    x = rounded(x + np.linspace(-0.5, 0.5, v)[None, :], dtype)
    ids = np.tile(np.arange(4, dtype=np.int32), (n, 1))
    t = np.log(np.full((n, 4), 0.2475, np.float32))
    got = check(x, ids, t, dtype, "both", rest=True)
    ref = R.distill(x, ids, t, rest=True)
    assert np.max(np.abs(got["stats"][:, 2] - ref["log_rest"])) < 400 * U * 20
    check(x, ids, t, dtype, "apart", rest=True)


def test_a_listed_token_outside_the_vocabulary_is_reported():
    ctx, _, _ = env()
    rng = np.random.default_rng(1)
    x = rng.standard_normal((5, 50)).astype(np.float32)
    ids, t = teacher_of(rng, 5, 50, 6, False)
    ids[1, 3], ids[4, 0] = 50, 2 ** 31 - 1
    check(x, ids, t, "f32", "both")
    assert ctx.status() == ag.AG_STATUS_BAD_INDEX
    check(x, ids, t, "f32", "apart")
    assert ctx.status() == ag.AG_STATUS_BAD_INDEX
    assert ctx.status() == 0


def test_rows_of_weight_zero_may_hold_anything():
    rng = np.random.default_rng(2)
    x = rng.standard_normal((4, 64)).astype(np.float32)
    x[1], x[2, 3] = np.nan, np.inf
    ids, t = np.tile(np.arange(5, dtype=np.int32), (4, 1)), rng.standard_normal((4, 5)).astype(np.float32)
    for what in ("both", "apart"):
        got = run(x, ids, t, "f32", what, row_scale=[0.5, 0.0, 0.0, 0.5])
        assert np.isfinite(got["loss"]) and not got["dlogits"][1:3].any() and np.isfinite(got["dlogits"]).all()


def test_no_rows_have_loss_zero():
    ctx, alloc, be = env()
    loss = up(np.array([5.0], np.float32))
    ctx.distill_forward(0, 10, 0, 0, None, loss, 0, 0, 0, 10, 3)
    assert down(loss)[0] == 0.0
    free(loss)


def test_teacher_that_is_not_a_number_spoils_its_row_only():
    rng = np.random.default_rng(3)
    x = rng.standard_normal((4, 200)).astype(np.float32)
    for rest in (False, True):
        ids, t = np.tile(np.arange(5, dtype=np.int32), (4, 1)), np.log(rng.random((4, 5)).astype(np.float32) / 6)
        t[2, 1] = np.nan
        for what in ("both", "apart"):
            got = run(x, ids, t, "f32", what, rest=rest)
            assert np.isnan(got["row_loss"][2]) and np.isnan(got["dlogits"][2]).all() and np.isnan(got["loss"])
            keep = [0, 1, 3]
            ref = R.distill(x[keep], ids[keep], t[keep], row_scale=np.full(3, 0.25), rest=rest)
            near(got["row_loss"][keep], ref["row_loss"], 400 * U * ref["loss_size"], "loss of a row")
            near(got["dlogits"][keep], ref["dlogits"], ref["size"] * 600 * U + 2.0 ** -120, "gradient")


def test_the_same_call_gives_the_same_bits():
    rng = np.random.default_rng(9)
    for n, v, dtype in ((3, 151936, "bf16"), (500, 5003, "f32"), (300, 32768, "f32")):
        x = rounded(rng.standard_normal((n, v)).astype(np.float32) * 2, dtype)
        ids, t = teacher_of(rng, n, v, 50, True)
        for what in ("both", "apart"):
            first = run(x, ids, t, dtype, what, rest=True)
            for _ in range(2):
                again = run(x, ids, t, dtype, what, rest=True)
                assert all(np.array_equal(first[k], again[k]) for k in first)


def test_recorded_calls_follow_their_inputs():
    ctx, alloc, be = env()
    rng = np.random.default_rng(12)
    n, v, top = 37, 5003, 9
    tx, g, row, loss, dl = (up(np.zeros(s, np.float32)) for s in ((n, v), (n, v), (n,), (1,), (1,)))
    ti, tt, st = up(np.zeros((n, top), np.int32)), up(np.zeros((n, top), np.float32)), up(np.zeros((n, 4), np.float32))

    def apart(c):
        c.distill_forward(tx, v, ti, tt, None, loss, row, st, n, v, top, 1.0, ag.AG_DISTILL_REST)
        c.distill_backward(tx, v, ti, tt, None, st, dl, None, g, v, n, v, top, 1.0, ag.AG_DISTILL_REST)

    def both(c):
        c.distill_forward_backward(tx, v, ti, tt, None, dl, loss, row, None, g, v, n, v, top, 1.0, ag.AG_DISTILL_REST)
    for f in (apart, both):
        f(ctx)
        ctx.synchronize()
        graph = ctx.record(f)
        for _ in range(2):
            x = rng.standard_normal((n, v)).astype(np.float32)
            ids, t = teacher_of(rng, n, v, top, True)
            scale = float(rng.random())
            for a, b in ((tx, x), (ti, ids), (tt, t), (dl, np.array([scale], np.float32))):
                be.copy_from_host(a, b)
            ctx.replay(graph)
            ref = R.distill(x, ids, t, dloss=np.float32(scale), rest=True)
            near(down(row), ref["row_loss"], 400 * U * ref["loss_size"], "loss of a row")
            near(down(g), ref["dlogits"], ref["size"] * (400 + 16 * np.abs(ref["lp"])) * U + 2.0 ** -120, "gradient")
        ctx.drop_recording(graph)
    free(tx, g, row, loss, dl, ti, tt, st)


def test_a_student_learns_from_its_teachers_list():
    """The operators as a training program strings them together: the teacher's head, its likeliest tokens with their
    log-probabilities, the student's head (a padded vocabulary), loss and gradient in the logits' place, back through the head."""
    ctx, alloc, be = env()
    rng = np.random.default_rng(31)
    n, c, v, width, top = 200, 128, 1001, 1008, 24
    f32 = np.float32
    hidden = (rng.standard_normal((n, c)) / np.sqrt(c)).astype(f32)
    teacher_w = rng.standard_normal((c, width)).astype(f32) * 2
    student_w = rng.standard_normal((c, width)).astype(f32) * 2
    student_w[:, v:] = 0   # a padded column
    th, tw, sw = up(hidden), up(teacher_w), up(student_w)
    tz, sz = up(np.zeros((n, width), f32)), up(np.zeros((n, width), f32))
    ids, lp = up(np.zeros((n, top), np.int32)), up(np.zeros((n, top), f32))
    row, loss, one = up(np.zeros(n, f32)), up(np.zeros(1, f32)), up(np.ones(1, f32))
    dh, dw = up(np.zeros((n, c), f32)), up(np.zeros((c, width), f32))
    nbytes = ctx.linear_add_scratch_bytes(n, c, width)
    ws = alloc.alloc((nbytes,), np.uint8)
    for w, z in ((tw, tz), (sw, sz)):
        ctx.linear_add_forward(None, th, w, None, z, n, c, width, ag.AG_CE_3XTF32, ws, nbytes)
    be.token_logprobs_forward(tz, None, None, top_ids=ids, top_logprobs=lp, temperature=2.0, vocab=v)
    be.distill_forward_backward(sz, ids, lp, one, row, sz, loss=loss, temperature=2.0, rest=True, vocab=v)
    z = down(tz)[:, :v]
    got_ids = down(ids)
    assert np.array_equal(got_ids, R.top(z, top))
    x = hidden.astype(np.float64) @ student_w.astype(np.float64)
    grad = down(sz)
    # what the padded columns hold is the head's output for them, 0: no gradient goes into them
    assert not grad[:, v:].any()
    ctx.linear_add_backward(sz, th, sw, None, dh, dw, None, n, c, width, ag.AG_CE_3XTF32, ws, nbytes)
    ref = R.distill(x[:, :v], got_ids, down(lp), temperature=2.0, rest=True)
    # the projection is fp32-grade: 2^-22 of the sizes of its terms per product, here 2e-6 of logits of size 2, which moves a
    # gradient by 1e-5 of itself; 1e-4 is what the framework holds fp32 gradients to
    assert abs(down(loss)[0] - ref["loss"]) < 1e-5 * abs(ref["loss"])
    for got, want in ((grad[:, :v], ref["dlogits"]), (down(dh), ref["dlogits"] @ student_w[:, :v].astype(np.float64).T),
                      (down(dw)[:, :v], hidden.astype(np.float64).T @ ref["dlogits"])):
        assert np.max(np.abs(got - want)) < 1e-4 * np.sqrt(np.mean(want ** 2)) + 1e-4 * np.max(np.abs(want))
    ctx.synchronize()
    alloc.free(ws)
    free(th, tw, sw, tz, sz, ids, lp, row, loss, one, dh, dw)
    check_clean_status()


def test_a_policy_step_after_a_head():
    """Head, log-probabilities and entropy of the rollouts' tokens, their gradient onto a loss's that is there already."""
    ctx, alloc, be = env()
    rng = np.random.default_rng(32)
    n, c, v = 96, 64, 640
    hidden, w = rng.standard_normal((n, c)).astype(np.float32) / 8, rng.standard_normal((c, v)).astype(np.float32)
    th, tw, z = up(hidden), up(w), up(np.zeros((n, v), np.float32))
    nbytes = ctx.linear_add_scratch_bytes(n, c, v)
    ws = alloc.alloc((nbytes,), np.uint8)
    ctx.linear_add_forward(None, th, tw, None, z, n, c, v, ag.AG_CE_3XTF32, ws, nbytes)
    ids = rng.integers(-1, v, n)
    tid, lp, ent, st = up(ids.astype(np.int32)), up(np.zeros(n, np.float32)), up(np.zeros(n, np.float32)), up(np.zeros((n, 4), np.float32))
    be.token_logprobs_forward(z, tid, lp, entropy=ent, stats=st)
    x = down(z).astype(np.float64)
    want, h, lps, _, _ = R.token_logprobs(x, ids)
    near(down(lp), want, (300 + 8 * np.abs(want)) * U, "log-probability")
    a, b, there = (rng.standard_normal(s).astype(np.float32) for s in (n, n, (n, v)))
    ta, tb, g = up(a), up(b), up(there)
    be.token_logprobs_backward(z, tid, st, ta, tb, g, dres=g)
    ref, size, _ = R.token_logprobs_backward(x, ids, a, b)
    near(down(g), ref + there, (size * 1000 + np.abs(there)) * U, "gradient")
    ctx.synchronize()
    alloc.free(ws)
    free(th, tw, z, tid, lp, ent, st, ta, tb, g)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,v", [(1, 4097), (2, 32768), (3, 151937), (40, 50257), (100, 20001), (200, 32768)])
def test_gradients_in_the_place_of_few_wide_logits(n, v, dtype):
    """Rows that several blocks share: one reads the listed logits of all others before those are written over."""
    rng = np.random.default_rng(v)
    x = rounded(rng.standard_normal((n, v)).astype(np.float32) * 2, dtype)
    for rest in (False, True):
        ids, t = teacher_of(rng, n, v, 200, rest)
        for what in ("both", "apart"):
            check(x, ids, t, dtype, what, rest=rest, place="logits", temperature=0.8)
            check(x, ids, t, dtype, what, rest=rest, place="logits", ld=v + 3, shift=1)


def test_tokens_that_are_listed_many_times():
    rng = np.random.default_rng(7)
    for n, v, top in ((5, 40, 64), (600, 700, 60), (3, 33000, 256)):
        x = rng.standard_normal((n, v)).astype(np.float32)
        x[:, 5] = -np.inf
        ids = rng.choice([0, 5, 7, v - 1, -1], (n, top)).astype(np.int32)
        for rest in (False, True):
            t = np.log(rng.random((n, top)) / top).astype(np.float32)
            t[ids == 5] = -np.inf
            for what in ("both", "apart"):
                check(x, ids, t, "f32", what, rest=rest)


def test_two_streams_at_once():
    """The same calls from two threads, each with a device context of its own, on logits of its own."""
    import threading

    ctx, alloc, be = env()
    rng = np.random.default_rng(17)
    n, v, top = 24, 40000, 30
    work = []
    for _ in range(2):
        x = rng.standard_normal((n, v)).astype(np.float32)
        ids, t = teacher_of(rng, n, v, top, True)
        c = ag.CudaContext(0)
        dev = [up(a) for a in (x, ids, t, np.ones(1, np.float32), np.zeros(1, np.float32), np.zeros(n, np.float32),
                               np.zeros((n, v), np.float32), np.zeros((n, top), np.int32), np.zeros((n, top), np.float32))]
        work.append((x, ids, t, c, dev))
    ctx.synchronize()

    def run_on(c, dev):
        tx, ti, tt, dl, loss, row, g, oi, ol = dev
        for _ in range(50):
            c.token_logprobs_forward(tx, v, None, None, None, None, oi, ol, n, v, top)
            c.distill_forward_backward(tx, v, ti, tt, None, dl, loss, row, None, g, v, n, v, top, 1.0, ag.AG_DISTILL_REST)
    threads = [threading.Thread(target=run_on, args=(w[3], w[4])) for w in work]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    for x, ids, t, c, dev in work:
        c.synchronize()
        assert c.status() == 0
        ref = R.distill(x, ids, t, rest=True)
        assert np.array_equal(down(dev[7]), R.top(x, top))
        near(down(dev[5]), ref["row_loss"], 400 * U * ref["loss_size"], "loss of a row")
        near(down(dev[6]), ref["dlogits"], ref["size"] * (400 + 16 * np.abs(ref["lp"])) * U + 2.0 ** -120, "gradient")
        c.close()
        free(*dev)


def test_logits_of_weights_stored_by_token():
    """Weights (V, C), as the CE head has them: the logits are the projection's backward product, dact += dout . w^T."""
    ctx, alloc, be = env()
    rng = np.random.default_rng(33)
    n, c, v = 70, 64, 500
    hidden, w = (rng.standard_normal((n, c)) / 8).astype(np.float32), rng.standard_normal((v, c)).astype(np.float32)
    th, tw, z = up(hidden), up(w), up(np.zeros((n, v), np.float32))
    nbytes = ctx.linear_add_scratch_bytes(n, v, c)
    ws = alloc.alloc((nbytes,), np.uint8)
    ctx.linear_add_backward(th, None, tw, None, z, None, None, n, v, c, ag.AG_CE_3XTF32, ws, nbytes)
    lp, ids = up(np.zeros(n, np.float32)), rng.integers(0, v, n)
    tid = up(ids.astype(np.int32))
    be.token_logprobs_forward(z, tid, lp)
    want = R.token_logprobs(hidden.astype(np.float64) @ w.astype(np.float64).T, ids)[0]
    # fp32-grade logits of size 1: 64 terms of at most 1/2, each product off by 2^-22 of its terms; twice that in a difference
    near(down(lp), want, 2 * 64 * 2.0 ** -23 + (300 + 8 * np.abs(want)) * U, "log-probability")
    ctx.synchronize()
    alloc.free(ws)
    free(th, tw, z, lp, tid)


GAPS = [5.0, 20.0, 30.0, 34.0, 60.0, 80.0, 90.0, 95.0, 110.0, 200.0, 1e3, 3e4]


def far_rests(rng, n, v, top, dtype, temperature):
    """Rows whose unlisted tokens together have e^-5 to e^-30000 of the student's mass, the last four of every sixteen with those
    masked by a finite number; lists of `top` tokens (at most half) that leave 0.01 to 0.5 of the teacher's mass."""
    ids = np.stack([rng.permutation(v)[:top] for _ in range(n)]).astype(np.int32)
    x = rng.standard_normal((n, v))
    masks = [-1e4, -1e9, -1e30 if temperature < 1 else LOWEST[dtype], -65504.0]
    for i in range(n):
        k = i % 16
        listed = x[i, ids[i]].copy()
        x[i] = x[i] * temperature - (GAPS[k] + np.log(v)) * temperature if k < 12 else masks[k - 12]
        x[i, ids[i]] = listed * temperature
    t = rng.standard_normal((n, top))
    t = t - np.log(np.exp(t).sum(1, keepdims=True)) + np.log(rng.uniform(0.5, 0.99, (n, 1)))
    return rounded(x.astype(np.float32), dtype), ids, t.astype(np.float32)


def check_far(x, ids, t, dtype, temperature, got, dres=None, made=False, row_scale=None, dloss=1.0):
    """An unlisted token's p is off by (400 + 16 |ln p|) u of itself, its part of p_rest by that with its own logarithm for ln p: it is
    one power, from the unlisted tokens' statistics.  Down to ln p_rest = -32 it comes from p and p_rest instead, where ln p_rest
    adds to the logarithm and what is flushed below 2^-126 is multiplied by r / p_rest; with statistics made from ln p_rest at any."""
    ref = R.distill(x, ids, t, row_scale, np.float32(dloss), temperature, True)
    near(got["row_loss"], ref["row_loss"], 400 * U * ref["loss_size"], "loss of a row")
    _, q, _, left, _ = R.teacher(ids, t, x.shape[1], temperature, True)
    with np.errstate(all="ignore"):
        p, part = np.exp(ref["lp"]), np.exp(ref["share"])
        rest = np.abs(ref["log_rest"])[:, None]
        s = np.abs(dloss * ref["weight"] / temperature)[:, None]
        mass = np.zeros(x.shape)
        np.add.at(mass, (np.arange(len(x))[:, None], ids), q)
        full = (q.sum(1) + left)[:, None]
        by = np.where(np.isfinite(ref["share"]), np.abs(ref["share"]), 0.0) + np.where(made | (rest < 33), rest, 0.0)
        bound = s * U * ((p * full + mass) * (400 + 16 * np.where(p > 0, np.abs(ref["lp"]), 0.0)) + (left[:, None] + 0.1) * part * (400 + 16 * by))
        bound = bound + s * 2.0 ** -125 * np.where(rest < 33, 1 + np.exp(np.minimum(rest, 33)), 1.0) + 2.0 ** -120
    g = ref["dlogits"]
    if dres is not None:
        g, bound = g + dres, bound + 2 * U * (np.abs(dres) + np.abs(g))
    if dtype == "bf16":
        bound = bound + np.abs(g) * 2.0 ** -8 + 2.0 ** -133
    near(got["dlogits"], g, bound, "gradient")
    return ref


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("temperature", [1.0, 0.1, 3.0])
@pytest.mark.parametrize("n,v,top", [(16, 61, 9), (32, 1003, 40), (700, 641, 19), (300, 20003, 64), (16, 50257, 256), (1, 32768, 20)])
def test_a_rest_that_the_student_gives_almost_nothing(n, v, top, temperature, dtype):
    """The gradient into the unlisted tokens sums to r whatever p_rest is: neither p nor 1 / p_rest has to be a number for that."""
    rng = np.random.default_rng(n + v)
    x, ids, t = far_rests(rng, n, v, top, dtype, temperature)
    if n == 1:
        x[0, np.setdiff1d(np.arange(v), ids[0])] = -1e3 * temperature
        x = rounded(x, dtype)
    kw = dict(temperature=temperature, rest=True)
    for what in ("both", "apart"):
        got = run(x, ids, t, dtype, what, **kw)
        ref = check_far(x, ids, t, dtype, temperature, got)
        check_far(x, ids, t, dtype, temperature, run(x, ids, t, dtype, what, place="logits", ld=v + 3, shift=1, **kw))
        far = ref["log_rest"] < -32
        assert far.any() and np.isfinite(got["dlogits"]).all()
    w = rng.random(n)
    dres = rounded(rng.standard_normal((n, v)).astype(np.float32), dtype)
    got = run(x, ids, t, dtype, "apart", dres=dres, row_scale=w, dloss=0.6, **kw)
    check_far(x, ids, t, dtype, temperature, got, dres, row_scale=w.astype(np.float32), dloss=0.6)
    check_clean_status()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_gradient_from_the_logarithm_of_a_small_rest(dtype):
    """Statistics (m, L, ln p_rest, 0) that a program has worked out itself, also where the loss leaves others."""
    ctx, alloc, be = env()
    rng = np.random.default_rng(21)
    n, v, top = 32, 1003, 40
    x, ids, t = far_rests(rng, n, v, top, dtype, 1.0)
    keep = np.arange(n) % 16 < 11  # down to e^-1000
    x, ids, t = x[keep], ids[keep], t[keep]
    n = len(x)
    ref = R.distill(x, ids, t, rest=True)
    _, m, total = R.log_softmax(x)
    st = np.stack([m, total, ref["log_rest"], np.zeros(n)], 1).astype(np.float32)
    tx, ti, tt, ts, one, g = up(words(x, dtype)), up(ids), up(t), up(st), up(np.ones(1, np.float32)), up(words(np.zeros((n, v), np.float32), dtype))
    ctx.distill_backward(tx, v, ti, tt, None, ts, one, None, g, v, n, v, top, 1.0, ag.AG_DISTILL_REST, 1 if dtype == "bf16" else 0)
    got = fetch(g, n * v, dtype).reshape(n, v)
    check_far(x, ids, t, dtype, 1.0, {"row_loss": ref["row_loss"], "dlogits": got}, made=True)
    free(tx, ti, tt, ts, one, g)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("mask", [-np.inf, -1e9])
@pytest.mark.parametrize("n,v,temperature", [(40, 1003, 1.0), (700, 5003, 0.7), (300, 20003, 2.0), (9, 50257, 1.0)])
def test_lists_of_all_the_tokens_that_are_allowed(n, v, temperature, mask, dtype):
    """A teacher's likeliest tokens under a grammar that allows fewer than are asked for, its student under the same: what the list
    leaves is rounding, and no rest that the forbidden tokens, of which the student thinks nothing, could have."""
    ctx, alloc, be = env()
    rng = np.random.default_rng(n)
    d = 1 if dtype == "bf16" else 0
    for top in (20, 128):
        teacher, student = np.full((n, v), mask, np.float32), np.full((n, v), mask, np.float32)
        for r in range(n):
            at = rng.permutation(v)[:(1, 2, 5, 13, 19, 20)[r % 6] * (1 if top == 20 else 6)]
            teacher[r, at], student[r, at] = rng.standard_normal(len(at)) * 3, rng.standard_normal(len(at)) * 2
        teacher, student = rounded(teacher, dtype), rounded(student, dtype)
        tz, ti, tl = up(words(teacher, dtype)), up(np.zeros((n, top), np.int32)), up(np.zeros((n, top), np.float32))
        ctx.token_logprobs_forward(tz, v, None, None, None, None, ti, tl, n, v, top, temperature, d)
        ids, t = down(ti), down(tl)
        free(tz, ti, tl)
        # 25 u and 7 u for each |t|, of at most ln 120 on average: what counts as no rest is 64 u
        assert np.all(np.abs(1 - np.exp(t.astype(np.float64)).sum(1)) < 60 * U)
        for what in ("both", "apart"):
            got = check(student, ids, t, dtype, what, rest=True, temperature=temperature)
            assert np.isfinite(got["row_loss"]).all() and np.isfinite(got["loss"])
            assert not got["dlogits"][student < -1e8].any()
    check_clean_status()


@pytest.mark.parametrize("rest", [2.0 ** -16, 2.0 ** -12])
def test_a_rest_above_what_roundings_leave_counts(rest):
    """64 tokens of (1 - rest) / 64 each: t = -4.2 is off by 2^-22 at most, the sum as much of itself."""
    rng = np.random.default_rng(4)
    x = rng.standard_normal((20, 500)).astype(np.float32)
    ids = np.stack([rng.permutation(500)[:64] for _ in range(20)]).astype(np.int32)
    t = np.full((20, 64), np.log((1 - rest) / 64), np.float32)
    ref = R.distill(x, ids, t, rest=True)
    size = np.abs(np.log(rest)) + np.abs(ref["log_rest"])
    for what in ("both", "apart"):
        got = check(x, ids, t, "f32", what, rest=True)
        without = R.distill(x, ids, t + np.float32(2 * rest), rest=True)   # nothing left
        # the rest is worth rest * (ln rest - ln p_rest), which 32 bits of the sum show
        assert np.all(np.abs(got["row_loss"] - without["row_loss"]) > rest * (size.min() / 4))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,v", [(250, 40001), (209, 100003)])
def test_gradients_in_the_place_of_many_wide_logits(n, v, dtype):
    """Blocks share a row for what L2 holds, with a list that lies in the parts of all of them and is long enough for all warps."""
    rng = np.random.default_rng(v)
    x = rounded(rng.standard_normal((n, v)).astype(np.float32) * 2, dtype)
    ids, t = teacher_of(rng, n, v, 256, True)
    for rest in (False, True):
        check(x, ids, t, dtype, "both", rest=rest, place="logits")
