"""GPU: what a refused call over pages leaves behind: nothing."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _works(orn, ctx):
    x, t, out = ctx.to_device(np.zeros((1, 8), np.float32)), ctx.to_device(np.array([7], np.uint32)), ctx.alloc(4)
    ctx.token_logprobs(x, orn.F32, 1, 8, t, 1, 0, out)
    ok = abs(out.download(np.float32, (1,))[0] + np.log(8)) < 1e-6
    for d in (x, t, out): d.free()
    return ok


def test_a_pool_that_does_not_fit(orn, ctx):
    """Pages for a terabyte are refused, and neither the call after that nor a pool that fits hears of it."""
    assert _works(orn, ctx)
    for _ in range(2):
        with pytest.raises(orn.OrnithError, match="out of memory"): orn.KvPool(ctx, 4, 1 << 20, 256, 8, 256, 2, 4)
        assert _works(orn, ctx)
    with pytest.raises(orn.OrnithError, match="out of memory"): ctx.alloc(1 << 42)
    pool = orn.KvPool(ctx, 1, 8, 16, 1, 64, 2, 4)
    s = pool.open()
    pool.extend([s], 40)
    assert pool.seq(s)[0] == 40 and pool.batch([s]).s.max_rows == 40
    pool.close()
    assert _works(orn, ctx)
