"""Products of projections and heads whose waits run out: the kernel says so and returns by itself, and the next calls give the same bits as
the one before.  The hook makes the issuer of one launch give up at once, while its operands are under way."""
import numpy as np
import pytest

from autograd_b200 import _native as N
from gpu_util import check_clean_status, down, empty, env, free, node, run_backward, run_forward, up

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def usual_precision():
    be = env()[2]
    kept = be.ce_precision
    yield
    be.ce_precision = kept


def gives_up_and_goes_on(call, read):
    ctx = env()[0]
    call()
    right = read()
    check_clean_status()
    ctx.debug_expire_products()
    call()
    ctx.synchronize()
    assert ctx.status() == N.AG_STATUS_WAIT_EXPIRED
    for _ in range(2):   # the hook is spent, the status was read
        call()
        assert all(np.array_equal(a, b) for a, b in zip(read(), right))
        check_clean_status()


@pytest.mark.parametrize("precision", [N.AG_CE_3XTF32, N.AG_CE_BF16], ids=["pairs", "half"])
@pytest.mark.parametrize("n,k,c", [(40, 64, 96), (500, 384, 384), (4096, 1536, 1536), (300, 2048, 264)])
def test_projection(n, k, c, precision):
    ctx, alloc, be = env()
    be.ce_precision = precision
    rng = np.random.default_rng(n)
    x, act, w = (rng.standard_normal(s).astype(np.float32) for s in ((n, c), (n, k), (k, c)))
    x, act, w, b = up(x, grad=0), up(act, grad=0), up(w, grad=0), up(np.zeros(c, np.float32), grad=0)
    out = empty((n, c), grad=rng.standard_normal((n, c)).astype(np.float32))
    linear = node("FusedLinearAddOp", (x, act, w, b), (out,))
    gives_up_and_goes_on(lambda: run_forward(linear), lambda: [down(out)])

    def backward():
        for t in (x, act, w, b):
            be.fill_storage2(t.grad.storage, 0)
        run_backward(linear)
    gives_up_and_goes_on(backward, lambda: [down(t.grad) for t in (x, act, w, b)])
    free(x, act, w, b, out)


@pytest.mark.parametrize("precision", [N.AG_CE_3XTF32, N.AG_CE_BF16], ids=["pairs", "half"])
@pytest.mark.parametrize("n,c,v", [(40, 64, 300), (1000, 768, 8000), (4096, 640, 9000), (300, 1280, 20001)])
def test_head(n, c, v, precision):
    ctx, alloc, be = env()
    be.ce_precision = precision
    rng = np.random.default_rng(n)
    x, w = up(rng.standard_normal((n, c)).astype(np.float32), grad=0), up((0.1 * rng.standard_normal((v, c))).astype(np.float32), grad=0)
    targets = up(rng.integers(0, v, n).astype(np.int32), requires_grad=False)
    loss = empty((1,), grad=np.ones(1, np.float32))
    head = node("FusedLinearCrossEntropyOp", (x, w, targets), (loss,))
    gives_up_and_goes_on(lambda: run_forward(head), lambda: [down(loss)])

    def backward():
        for t in (x, w):
            be.fill_storage2(t.grad.storage, 0)
        run_backward(head)
    gives_up_and_goes_on(backward, lambda: [down(t.grad) for t in (x, w)])
    free(x, w, targets, loss)
