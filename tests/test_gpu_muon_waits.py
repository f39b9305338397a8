"""Products of an orthogonal factor whose waits run out: the kernel says so and returns by itself, and the next call is as if nothing had
been.  The hook makes the issuer of one product's launch give up at once, while its operands (or a small matrix's products) are under way."""
import numpy as np
import pytest

from autograd_b200 import _native as N
from gpu_util import check_clean_status, env
from test_gpu_muon import PRECISIONS, Matrices, gradient

pytestmark = pytest.mark.gpu

# matrices, products that run before the one that gives up: small ones on one CTA and on clusters, contractions shared by a cluster, single CTAs,
# pairs (X X^T, A A, Q X)
CASES = [((1, 64, 64), 0), ((2, 64, 256), 0), ((1, 128, 4000), 0), ((1, 200, 3000), 0), ((2, 130, 140), 0), ((2, 130, 140), 2),
         ((24, 270, 300), 0), ((24, 270, 300), 1), ((6, 384, 1536), 2), ((6, 384, 1536), 14)]


@PRECISIONS
@pytest.mark.parametrize("shape,after", CASES, ids=lambda v: "x".join(map(str, v)) if isinstance(v, tuple) else f"after{v}")
def test_a_wait_that_runs_out_leaves_the_context_usable(shape, after, precision):
    ctx, alloc, be = env()
    a = Matrices(gradient(np.random.default_rng(sum(shape)), *shape))
    b = Matrices(np.zeros(shape, np.float32))
    be.orthogonalise(a.argument, b.argument, precision=precision)
    right = b.read()
    check_clean_status()
    launches = ctx.launch_count
    ctx.debug_expire_products(after)
    be.orthogonalise(a.argument, b.argument, precision=precision)
    ctx.synchronize()
    assert ctx.status() == N.AG_STATUS_WAIT_EXPIRED
    launches = ctx.launch_count - launches
    for _ in range(2):   # the hook is spent, the status was read
        before = ctx.launch_count
        be.orthogonalise(a.argument, b.argument, precision=precision)
        assert np.array_equal(b.read(), right) and ctx.launch_count - before == launches
        check_clean_status()
    a.free(), b.free()


def test_products_that_cannot_be_counted_are_refused():
    ctx, alloc, be = env()
    with pytest.raises(N.AgError):
        ctx.debug_expire_products(-1)
