"""Normalised heads and orthogonal updates as a training step uses them: a packed projection onto queries and keys, the heads
normalised and rotated, a loss of them, the gradients back through all of it, and a step on the projection."""
import numpy as np
import pytest

from autograd_b200 import _native as N
from gpu_util import check_clean_status, down, empty, env, free, node, run_backward, run_forward, up
from oracle import heads_and_updates as R

pytestmark = pytest.mark.gpu


def test_projection_heads_loss_gradient_and_step():
    ctx, alloc, be = env()
    rng = np.random.default_rng(0)
    b, t, h, kv, d, c = 2, 24, 4, 2, 32, 96
    n, width, eps, lr = b * t, (h + 2 * kv) * d, 1e-6, 0.02
    x = rng.standard_normal((b, t, c)).astype(np.float32)
    w = (0.1 * rng.standard_normal((c, width))).astype(np.float32)
    gamma = (1 + 0.2 * rng.standard_normal((2, d))).astype(np.float32)
    a = np.arange(t)[:, None] * 1e4 ** (-np.arange(0, d, 2) / d)
    cos, sin = np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)
    dq, dk = rng.standard_normal((b, t, h, d)).astype(np.float32), rng.standard_normal((b, t, kv, d)).astype(np.float32)

    act, weight = up(x, requires_grad=False), up(w, grad=0)
    bias, rest = up(np.zeros(width, np.float32), requires_grad=False), up(np.zeros((b, t, width), np.float32), requires_grad=False)
    qkv = empty((b, t, width), grad=0)
    linear = node("FusedLinearAddOp", (rest, act, weight, bias), (qkv,))
    run_forward(linear)

    def part(storage, first, count):
        v = empty((0,))
        free(v)
        v.shape = (b, t, count, d)
        v.storage = alloc.view(storage, first * d * 4, v.shape, np.float32)
        return v
    q, k = part(qkv.storage, 0, h), part(qkv.storage, h, kv)
    gq, gk = part(qkv.grad.storage, 0, h), part(qkv.grad.storage, h, kv)
    tc, ts, wq, wk = up(cos), up(sin), up(gamma[0], grad=0), up(gamma[1], grad=0)
    yq, yk, tdq, tdk = empty((b, t, h, d)), empty((b, t, kv, d)), up(dq), up(dk)
    m = up(np.zeros_like(w))
    kw = dict(q_gamma=wq, k_gamma=wk, q_stride=width, k_stride=width)
    be.qk_norm_rope_forward(q, k, tc, ts, yq, yk, eps, **kw)
    be.qk_norm_rope_backward(tdq, tdk, q, k, tc, ts, gq, gk, eps, dq_gamma=wq.grad, dk_gamma=wk.grad, dq_stride=width, dk_stride=width, **kw)
    run_backward(linear)
    be.muon_step(weight, weight.grad, m, lr, weight_decay=0.1)

    # the same in 64 bits
    z = (x.reshape(n, c).astype(np.float64) @ w).reshape(n, h + 2 * kv, d)
    at = np.arange(n) % t
    dz = np.zeros_like(z)
    for lo, hi, g, out, dy, dg in ((0, h, gamma[0], yq, dq, wq.grad), (h, h + kv, gamma[1], yk, dk, wk.grad)):
        dy = dy.reshape(n, hi - lo, d)
        ref = R.heads(z[:, lo:hi], g, cos[at], sin[at], eps)
        got = down(out).reshape(ref.shape)
        assert np.abs(got - ref).max() <= 1e-5 * (np.abs(ref).max() + 1)
        dz[:, lo:hi], dgamma = R.heads_backward(dy, z[:, lo:hi], g, cos[at], sin[at], eps)
        assert np.abs(down(dg) - dgamma).max() <= 1e-4 * np.sqrt(np.mean(dgamma ** 2))
    dw = x.reshape(n, c).astype(np.float64).T @ dz.reshape(n, width)
    got = down(weight.grad).astype(np.float64)
    assert np.abs(got - dw).max() <= 1e-4 * np.sqrt(np.mean(dw ** 2)) + 1e-4 * np.abs(dw).max()
    # a step on the gradient that the kernels made
    ref, ref_m, u = R.muon(w, got, np.zeros_like(w), lr, weight_decay=0.1, scale=0.2 * np.sqrt(max(c, width)))
    new = down(weight).astype(np.float64)
    factor, error = R.factor_error(u, R.NEWTON_SCHULZ, 5, 1e-7, 22)
    bound = (4 * error + 2.0 ** -18 * np.linalg.norm(factor)) * lr * 0.2 * np.sqrt(max(c, width))
    assert np.linalg.norm(new - ref) <= bound + 2.0 ** -22 * np.linalg.norm(ref)
    assert np.abs(down(m) - ref_m).max() <= 2.0 ** -20 * np.abs(ref_m).max()
    # and the derivative of the loss along the step's direction, by differences
    def loss(v):
        y = (x.reshape(n, c).astype(np.float64) @ v).reshape(n, h + 2 * kv, d)
        return (sum((R.heads(y[:, lo:hi], g, cos[at], sin[at], eps) * dy.reshape(n, hi - lo, d)).sum()
                    for lo, hi, g, dy in ((0, h, gamma[0], dq), (h, h + kv, gamma[1], dk))))
    step = new - w
    slope = (loss(w + 1e-5 * step) - loss(w - 1e-5 * step)) / 2e-5
    assert abs((got * step).sum() - slope) <= 1e-4 * np.linalg.norm(got) * np.linalg.norm(step)
    check_clean_status()


def test_step_with_normalised_heads():
    """The step's heads against the 64-bit form: outputs, input gradients, the weights' gradients in the bucket that is reduced, the loss
    behind them; the same result from a recorded step."""
    from autograd_b200.step import FusedLayerStep, StepConfig
    ctx, alloc, be = env()
    cfg = StepConfig(n_layer=2, n_embd=64, n_head=2, head_dim=32, seq_len=24, vocab=128, batch=2, qk_norm=True)
    plain = FusedLayerStep(ctx, alloc, be, StepConfig(**{**cfg.__dict__, "qk_norm": False}))
    step = FusedLayerStep(ctx, alloc, be, cfg)
    n, h, d, c = cfg.tokens, cfg.n_head, cfg.head_dim, cfg.n_embd
    rng = np.random.default_rng(0)
    ids = rng.integers(0, cfg.vocab, (2, n)).astype(np.int32)
    gamma = (1 + 0.3 * rng.standard_normal((2, 2, d))).astype(np.float32)
    ctx.copy_from_host(step.head_gamma, gamma)
    for s in (plain, step):
        ctx.copy_from_host(s.ids, ids[0])
        ctx.copy_from_host(s.targets, ids[1])

    def read(address, *shape):
        return ctx.copy_to_host(address, shape, np.float32)
    cos, sin = read(step.cos, cfg.seq_len, d // 2), read(step.sin, cfg.seq_len, d // 2)
    at = np.arange(n) % cfg.seq_len
    results = []
    for _ in range(3):
        step.step()
        results.append([read(a, n, h, d) for a in (*step.qk_out, *step.dqk)] + [read(step.small_bucket, step.n_small + 1)])
    assert all(np.array_equal(a, b) for r in results[1:] for a, b in zip(results[0], r))
    plain.step()
    *heads, small = results[0]
    assert step.n_small == plain.n_small + 2 * 2 * d and small[-1] == plain.read_loss()
    assert np.array_equal(small[:plain.n_small], read(plain.small_bucket, plain.n_small))
    for layer in range(2):
        for side, x in enumerate((step.q, step.k)):
            x, dy = read(x, n, h, d), read(step.dqk_out[side], n, h, d)
            dx, dgamma = R.heads_backward(dy, x, gamma[layer, side], cos[at], -sin[at], cfg.eps)
            got = small[plain.n_small + (2 * layer + side) * d:][:d]
            assert np.abs(got - dgamma).max() <= 1e-5 * np.abs(dgamma).max() + 1e-5
            if layer == 1:   # the last forward pass
                ref = R.heads(x, gamma[layer, side], cos[at], -sin[at], cfg.eps)
                assert np.abs(heads[side] - ref).max() <= 1e-5 * np.abs(ref).max()
            else:            # the last backward pass
                assert np.abs(heads[2 + side] - dx).max() <= 1e-5 * np.abs(dx).max()
    check_clean_status()
    plain.close()
    step.close()
