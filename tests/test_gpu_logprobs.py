"""GPU: log probabilities of given tokens, logsumexp, entropy and the most probable alternatives against 64 bits.

Tolerances. With d_i = x_i - m (exact or rounded once: u = 2^-24 relative), an exponential carries a relative error of at most
(2 |d_i| + 4) u: the rounding of d_i and of its product with log2 e, and two units of the instruction. A sum of V terms in chains of at
most V / 64 and a tree above them adds (V / 64 + 32) u. So L is off by eps = (2 D + V / 64 + 40) u relative, D = sum p_i |d_i|;
ln L by eps and 4 u |ln L|; a log probability by that, u |d_t| and a rounding of the result; S / L by 2 eps of sum p_i |d_i|."""
import numpy as np
import pytest

import util

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _run(orn, ctx, x, dtype, tokens, k, stride=None, offset=0, want_entropy=True, want_lse=True):
    """x: fp32 or bf16 bits [rows, V]; the device rows start `offset` elements in and lie `stride` apart, NaN between them."""
    rows, V = x.shape
    stride = stride or V
    host = np.full(offset + rows * stride, np.nan, np.float32) if dtype == orn.F32 else np.full(offset + rows * stride, 0x7fc0, np.uint16)
    for r in range(rows):
        host[offset + r * stride:offset + r * stride + V] = x[r]
    n = tokens.shape[1] if tokens is not None else 0
    buf = ctx.to_device(host)

    class At:
        def __init__(self): self.ptr = type(buf.ptr)(buf.ptr.value + offset * host.itemsize)
    dt = ctx.to_device(tokens.astype(np.uint32)) if n else None
    outs = [np.full((rows, n), 7.0, np.float32), np.full(rows, 7.0, np.float32), np.full(rows, 7.0, np.float32), np.full((rows, k), 7, np.uint32),
            np.full((rows, k), 7.0, np.float32)]
    bufs = [ctx.to_device(o) if o.size else None for o in outs]
    ctx.token_logprobs(At(), dtype, rows, V, dt, n, k, bufs[0], bufs[1] if want_entropy else None, bufs[2] if want_lse else None, bufs[3], bufs[4],
                       row_stride=stride)
    got = [b.download(o.dtype, o.shape) if b else o for b, o in zip(bufs, outs)]
    for b in bufs + [buf, dt]:
        if b: b.free()
    return got


def _want(x, tokens, k):
    """x: float64 [V] without NaN or +inf -> (logprobs, entropy, lse, ids, top logprobs, tolerances of the first three)"""
    V = x.size
    ids = np.lexsort((np.arange(V), -x))[:k]
    if not np.isfinite(x).any():
        return np.full(len(tokens), -np.inf), 0.0, -np.inf, ids, np.full(k, -np.inf), 0.0, 0.0, 0.0
    m = x.max()
    d = x - m
    with np.errstate(invalid="ignore"):
        e = np.exp(d)
        L = e.sum()
        p = e / L
        mag = np.where(p > 0, p * np.abs(np.where(p > 0, d, 0.0)), 0.0).sum()
    lp = np.array([d[t] - np.log(L) if t < V else -np.inf for t in tokens])
    eps = (2 * mag + V / 64 + 40) * U
    tol_log = eps + 4 * U * np.log(L)
    ok = np.isfinite(lp)
    tol_lp = tol_log + 2 * U * np.abs(lp[ok]).max(initial=0.0)
    return lp, np.log(L) + mag, m + np.log(L), ids, d[ids] - np.log(L), tol_lp, tol_log + 3 * eps * mag + 2 * U * (np.log(L) + mag), tol_log + 2 * U * abs(m + np.log(L))


def _check(x, tokens, k, got):
    lp, ent, lse, ids, tlp = got
    for r in range(x.shape[0]):
        w = _want(x[r].astype(np.float64), tokens[r] if tokens is not None else [], k)
        assert np.array_equal(ids[r], w[3]), (r, ids[r], w[3])
        for g, v, tol in ((lp[r], w[0], w[5]), (ent[r], w[1], w[6]), (lse[r], w[2], w[7]), (tlp[r], w[4], None)):
            g, v = np.atleast_1d(g).astype(np.float64), np.atleast_1d(v)
            fin = np.isfinite(v)
            if tol is None:
                tol = w[5] + 4 * U * np.abs(v[fin]).max(initial=0.0)
            assert np.array_equal(g[~fin], v[~fin]), (r, g, v)
            assert np.all(np.abs(g[fin] - v[fin]) <= tol), (r, np.abs(g[fin] - v[fin]).max(), tol)


SIZES = [(1, 1), (1, 2), (3, 63), (2, 64), (5, 511), (2, 512), (3, 513), (1, 1000), (4, 4095), (4, 4096), (2, 4097), (3, 8191), (2, 12345), (1, 32768), (7, 32769),
         (2, 65536), (3, 100003), (2, 248320), (70, 3001), (300, 515), (1030, 40)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,V", SIZES)
def test_values(orn, ctx, rows, V, dtype):
    rng = np.random.default_rng(rows * 1000003 + V)
    x = (rng.standard_normal((rows, V)) * 3).astype(np.float32)
    x[::2, V // 2] += 15
    tokens = rng.integers(0, V, (rows, 3))
    tokens[:, 0], tokens[:, 2] = V - 1, x.argmax(1)
    if dtype == "bf16":
        b = util.f32_to_bf16(x)
        for k in sorted({0, 1, min(V, 8), min(V, 32)}):
            _check(util.bf16_to_f32(b), tokens, k, _run(orn, ctx, b, orn.BF16, tokens, k))
    else:
        for k in sorted({0, min(V, 20), min(V, 32)}):
            _check(x, tokens, k, _run(orn, ctx, x, orn.F32, tokens, k))


@pytest.mark.parametrize("offset,pad", [(0, 1), (1, 0), (3, 5), (7, 8), (5, 3), (8, 16), (2, 6)])
@pytest.mark.parametrize("V", [7, 1000, 20011])
def test_rows_at_any_address(orn, ctx, V, offset, pad):
    rng = np.random.default_rng(V + offset)
    x = rng.standard_normal((4, V)).astype(np.float32)
    tokens = rng.integers(0, V, (4, 1))
    k = min(V, 6)
    _check(x, tokens, k, _run(orn, ctx, x, orn.F32, tokens, k, V + pad, offset))
    b = util.f32_to_bf16(x)
    _check(util.bf16_to_f32(b), tokens, k, _run(orn, ctx, b, orn.BF16, tokens, k, V + pad, offset))


@pytest.mark.parametrize("V", [40, 700, 5000, 33000, 248320])
def test_ties_and_masks(orn, ctx, V):
    """Constant rows, a few levels only, all but a few tokens masked (by -inf, by the type's lowest value), nothing left, one token left:
    the alternatives in their order, equal ones by the lower id."""
    rng = np.random.default_rng(V)
    low = np.float32(-3.3895313892515355e38)             # bf16's lowest
    rows = [np.zeros(V), np.full(V, -5.5), rng.integers(0, 3, V) * 0.5, np.where(rng.random(V) < 0.999, -np.inf, rng.standard_normal(V)),
            np.where(np.arange(V) == V - 1, 1.0, -np.inf), np.full(V, -np.inf), np.where(rng.random(V) < 0.9, low, rng.standard_normal(V)), np.full(V, low),
            np.arange(V) * 2.0 ** -10, -np.arange(V) * 2.0 ** -10, np.where(np.arange(V) % 7 == 0, 0.0, -0.0)]
    x = np.stack(rows).astype(np.float32)
    b = util.f32_to_bf16(x)
    tokens = np.stack([np.zeros(len(rows)), np.full(len(rows), V - 1), rng.integers(0, V, len(rows))], 1).astype(np.int64)
    for k in (1, 5, 32):
        _check(util.bf16_to_f32(b), tokens, k, _run(orn, ctx, b, orn.BF16, tokens, k))
        _check(x, tokens, k, _run(orn, ctx, x, orn.F32, tokens, k))


def test_large_magnitudes(orn, ctx):
    """Logits of 3e38 and differences that overflow: the distribution is the largest one's."""
    x = np.zeros((3, 3000), np.float32)
    x[0, 5], x[0, 6] = 3e38, -3e38
    x[1] = -3e38
    x[1, 1234] = 3e38
    x[2] = 3e38
    tokens = np.array([[5, 0], [1234, 0], [2, 2999]])
    lp, ent, lse, ids, tlp = _run(orn, ctx, x, orn.F32, tokens, 4)
    assert np.array_equal(ids, [[5, 0, 1, 2], [1234, 0, 1, 2], [0, 1, 2, 3]])
    assert lp[0, 0] == 0 and lp[0, 1] == np.float32(-3e38) and lp[1, 0] == 0 and ent[0] == 0 and ent[1] == 0
    assert np.allclose(lp[2], -np.log(3000), rtol=1e-6) and np.allclose(ent[2], np.log(3000), rtol=1e-6)
    assert lse[0] == np.float32(3e38) and lse[2] == np.float32(3e38)


@pytest.mark.parametrize("V", [33, 5000, 70000])
def test_no_distribution(orn, ctx, V):
    """NaN or +inf among the logits: lse and entropy are no finite numbers, ids go by value with NaN last; the rows beside are as ever."""
    rng = np.random.default_rng(3)
    x = rng.standard_normal((5, V)).astype(np.float32)
    x[0, V // 3], x[1, V - 1], x[2, 0], x[2, 1] = np.nan, np.inf, np.nan, np.inf
    x[3, :] = np.nan
    tokens = rng.integers(2, V - 1, (5, 1))
    lp, ent, lse, ids, tlp = _run(orn, ctx, x, orn.F32, tokens, 8)
    assert np.isnan(ent[:4]).all() and not np.isfinite(lse[:4]).any() and not np.isfinite(lp[:4]).any()
    for r in range(4):
        key = np.where(np.isnan(x[r]), -np.inf, x[r])
        order = np.lexsort((np.arange(V), np.isnan(x[r]), -key))
        assert np.array_equal(ids[r], order[:8]), r
    _check(x[4:], tokens[4:], 8, [g[4:] for g in (lp, ent, lse, ids, tlp)])


def test_ids_past_the_end_and_optional_outputs(orn, ctx):
    rng = np.random.default_rng(5)
    x = rng.standard_normal((2, 900)).astype(np.float32)
    tokens = np.array([[900, 0xffffffff, 899], [5, 2 ** 31, 1000]])
    got = _run(orn, ctx, x, orn.F32, tokens, 0)
    _check(x, tokens, 0, got)
    assert np.isneginf(got[0][0, :2]).all() and np.isneginf(got[0][1, 1:]).all()
    none = _run(orn, ctx, x, orn.F32, None, 3, want_entropy=False, want_lse=False)
    assert (none[1] == 7).all() and (none[2] == 7).all() and np.array_equal(none[3], _run(orn, ctx, x, orn.F32, tokens, 3)[3])


def test_calls_in_a_row_and_two_contexts(orn, ctx):
    """A call's workspace says nothing to the next one, on one context or on two."""
    rng = np.random.default_rng(9)
    other = orn.Ctx(0)
    for rows, V, k in ((6, 40000, 20), (1, 100, 3), (2, 40000, 20), (9, 248320, 5), (3, 513, 32)):
        x = rng.standard_normal((rows, V)).astype(np.float32)
        tokens = rng.integers(0, V, (rows, 2))
        a = _run(orn, ctx, x, orn.F32, tokens, k)
        b = _run(orn, other, x, orn.F32, tokens, k)
        _check(x, tokens, k, a)
        assert all(np.array_equal(p, q) for p, q in zip(a, b))
    other.close()


def test_sure_tokens_keep_their_digits(orn, ctx):
    """log p = -ln(1 + rest) with a small rest: off by 200 u of it, u = 2^-24 (an exponential 20 u with its argument's rounding, up to 140
    additions one after another, the logarithm and the end 10), not by u of the 1 beside it."""
    rng = np.random.default_rng(37)
    for V in (600, 5000, 248320):
        x = rng.standard_normal((3, V)).astype(np.float32) - np.float32(16.0 + np.log(V / 600))
        at = rng.integers(0, V, (3, 1))
        np.put_along_axis(x, at, np.float32(0.25), 1)
        d = x.astype(np.float64) - 0.25
        np.put_along_axis(d, at, -np.inf, 1)
        rest = np.exp(d).sum(1)
        got = _run(orn, ctx, x, orn.F32, at, 0)[0][:, 0].astype(np.float64)
        assert (np.abs(got + np.log1p(rest)) <= 200 * 2.0 ** -24 * rest).all(), (V, got, rest)
