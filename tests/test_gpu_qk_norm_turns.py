"""Normalised heads of so many tokens that a group of lanes goes from token to token several times, the last time with a part of the
groups: every output of the forward pass, and gradients of weights in which each token counts."""
import zlib

import numpy as np
import pytest

from autograd_b200 import _native as N
from gpu_util import check_clean_status, env, free, up
from oracle import heads_and_updates as R
from test_gpu_qk_norm import EPS, LAYOUTS, U, Rows, addresses, near, operands, partner, place, tables

pytestmark = pytest.mark.gpu

# tokens, sequence (longer and shorter than what a group moves on by, no divisor of it), heads, key heads, D, columns that rotate.  148 SMs of at most eight
# blocks of 8 to 128 tokens and two heads: two turns and more, none of the numbers of tokens fills the last
SHAPES = [(20011, 2858, 7, 3, 64, 32), (20011, 20011, 7, 3, 64, 64), (20011, 7, 7, 3, 64, 64), (9001, 77, 5, 3, 74, 74), (6007, 1001, 5, 5, 128, 128),
          (3001, 100, 2, 1, 1024, 512), (50021, 5000, 4, 4, 16, 8)]


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_forward_of_several_turns(shape, dtype, layout):
    ctx, alloc, be = env()
    rng = np.random.default_rng(zlib.crc32(repr((shape, dtype, layout)).encode()))
    n, seq, h, kv, d, rot = shape
    q, k, pitch, shift = operands(rng, shape, dtype, layout)
    rows = seq + 3
    cos, sin = tables(rows, rot)
    given = layout == "packed"
    at = place(rng, n, seq, rows, given)
    gamma = (1 + 0.3 * rng.standard_normal((2, d))).astype(np.float32)
    x = [Rows(t, dtype, p, shift) for t, p in zip((q, k), pitch)]
    y = [Rows(np.full(t.shape, 5.0, np.float32), dtype, None if layout != "shifted" else p, shift) for t, p in zip((q, k), pitch)]
    c, s, p, gq, gk = addresses(cos, sin, at if given else None, *gamma)
    ctx.qk_norm_rope_forward(x[0].address, x[1].address, gq, gk, c, s, p, y[0].address, y[1].address, n, seq, rows, h, kv, d, rot,
                             x[0].stride, x[1].stride, y[0].stride, y[1].stride, EPS, 1, N.AG_BF16 if dtype == "bf16" else N.AG_F32)
    for t, out, g in ((q, y[0], gamma[0]), (k, y[1], gamma[1])):
        plain = R.heads(t, g, np.ones_like(cos[at]), 0 * sin[at], EPS)
        near(out.read(), R.heads(t, g, cos[at], sin[at], EPS), 32 * U * partner(plain, rot), dtype, "y")
    check_clean_status()
    free(*(r.whole for r in x + y), *(t for t in (c, s, p, gq, gk) if t))


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_gradients_of_weights_count_every_token_once(shape, dtype, layout):
    """Elements 1 and -1, gradients of 1 and 3, quarter turns: what a token adds is an odd number (times inv, which is 1 up to 3 u), so that a token
    that is left out or taken twice changes a sum by 1 at least.  Sums err by 3 u of n heads numbers of up to 3, at most 0.09 here, and by u of partial
    sums below 2^15 at each of at most 400 additions in a chain, 0.8 if all fell to one side; 0.25 stands for both, as partial sums
    stay near the root of n heads, 2^10.  dx is looked over too."""
    ctx, alloc, be = env()
    rng = np.random.default_rng(zlib.crc32(repr((layout, dtype, shape)).encode()))
    n, seq, h, kv, d, rot = shape
    _, _, pitch, shift = operands(rng, (1, 1, h, kv, d, rot), dtype, layout)
    q, k = (rng.choice([-1.0, 1.0], (n, m, d)).astype(np.float32) for m in (h, kv))
    dy = [rng.choice([-3.0, -1.0, 1.0, 3.0], t.shape).astype(np.float32) for t in (q, k)]
    rows = seq + 3
    quarter = (np.arange(rows)[:, None] * np.arange(1, rot // 2 + 1)) % 4
    cos, sin = (np.float32(v)[quarter] for v in ([1, 0, -1, 0], [0, 1, 0, -1]))
    given = layout == "packed"
    at = place(rng, n, seq, rows, given)
    x = [Rows(t, dtype, p, shift) for t, p in zip((q, k), pitch)]
    g = [Rows(t, dtype, None, shift) for t in dy]
    dx = [Rows(np.full(t.shape, 5.0, np.float32), dtype, p, shift) for t, p in zip((q, k), pitch)]
    start = np.float32(rng.integers(-50, 50, (2, d)))
    c, s, p, dgq, dgk = addresses(cos, sin, at if given else None, *start)
    need = ctx.qk_norm_partials_bytes(h, kv, d)
    part = up(np.zeros(need, np.uint8))
    ctx.qk_norm_rope_backward(g[0].address, g[1].address, x[0].address, x[1].address, 0, 0, c, s, p, dx[0].address, dx[1].address, dgq, dgk, part, need,
                              n, seq, rows, h, kv, d, rot, g[0].stride, g[1].stride, x[0].stride, x[1].stride, dx[0].stride, dx[1].stride, 0.0, 1,
                              False, N.AG_BF16 if dtype == "bf16" else N.AG_F32)
    for i, (t, dyt, out, dg) in enumerate(((q, dy[0], dx[0], dgq), (k, dy[1], dx[1], dgk))):
        ref, dgamma = R.heads_backward(dyt, t, None, cos[at], sin[at], 0.0)
        assert np.array_equal(dgamma, np.round(dgamma))
        off = be.copy_to_host(dg).astype(np.float64) - dgamma - start[i]
        assert np.abs(off).max() <= 0.25, np.abs(off).max()
        # |x| = inv = 1: the bound of test_gpu_qk_norm.py
        v = partner(dyt.astype(np.float64), rot)
        near(out.read(), ref, 80 * U * (v + np.mean(v, -1, keepdims=True)), dtype, "dx")
    check_clean_status()
    free(part, *(r.whole for r in x + g + dx), *(t for t in (c, s, p, dgq, dgk) if t))
