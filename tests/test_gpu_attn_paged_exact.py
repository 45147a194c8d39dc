"""GPU: the attention over a paged KV cache held to tolerances of single keys and of fp32 probabilities.

Counted keys. A key is c u or -c u with u of ones and minus ones, a query u or -u, so that a score is +S or -S with S = c hd a power of two
(its product with any fp32 constant is exact) and 2 S scale log2(e) over 160: a key of the larger score has probability weight
exactly 1, one of the other exactly 0. Values are whole numbers up to 8: every sum is a whole number below 2^24, exact in fp32 in any
order. What is left is one reciprocal and one product (4 u, u = 2^-24, is more than both) and the rounding to bf16, 2^-8 of the result: a
key that is lost, taken twice or taken from another row shows.

Probabilities. Queries and keys are whole numbers up to 3: scores are exact, too, and a probability is off by delta = 4 u |score scale
log2(e)| from its exponent (the constant, the reference point's product, the fused product, the difference of two of them) and 4 u from its exponential. It goes to the
value product as bf16 and what that leaves, rounded to bf16 in turn: 2^-8 of 2^-8. It enters the sum of probabilities, too (each
twice), and a sum of n terms is off by (n + 8) u of A = sum p |v| / sum p; 2^-8 of the result at the end."""
import numpy as np
import pytest

import util
from test_gpu_attn_paged import Case, _attend, _bits, _f

pytestmark = pytest.mark.gpu
U, HALF = 2.0 ** -24, 2.0 ** -8


def _counted(orn, ctx, rng, lens, T, shared, R, Hq, Hkv, hd, alias=False):
    """One call over counted keys against their sums, and the same call again. alias: all sequences have the same pages throughout."""
    B, G, ns = len(lens), Hq // Hkv, shared // R
    c = Case(ctx, rng, lens[:1] if alias else lens, T, shared, R, Hq, Hkv, hd)
    if alias: c.B, c.lens, c.table, c.max_rows = B, lens, np.repeat(c.table, B, 0), max(lens)
    cmul, scale = 4.0 if hd == 256 else 8.0, hd ** -0.5
    assert 2 * cmul * hd * scale * 1.44 > 160
    unit = rng.choice([-1.0, 1.0], hd).astype(np.float32)
    at = {}                                                                     # sequence: its keys' signs and its values

    def fill(ids, n):
        sign, val = rng.choice([-1, 1], (Hkv, n)), rng.integers(1, 9, (Hkv, n, hd)) * rng.choice([-1, 1], (Hkv, n, hd))
        kb, vb = util.f32_to_bf16((sign[..., None] * cmul * unit).astype(np.float32)), util.f32_to_bf16(val.astype(np.float32))
        for i in range(-(-n // R)):
            m = min(R, n - i * R)
            c.k[0, ids[i], :, :m], c.v[0, ids[i], :, :m] = kb[:, i * R:i * R + m], vb[:, i * R:i * R + m]
        return sign, val

    if shared: at["shared"] = fill(c.table[0, :ns], shared)
    for b in range(1 if alias else B):
        n = max(lens[b] - shared, 0)
        if n: at[b] = fill(c.table[b, ns:], n)
    c.upload(orn)
    qs = rng.choice([-1, 1], (B, T, Hq))
    q = util.f32_to_bf16((qs[..., None] * unit).astype(np.float32))
    got = _attend(orn, ctx, c, q, None, scale)
    assert np.array_equal(_attend(orn, ctx, c, q, None, scale), got)
    g, of_shared = _f(got), {}
    for b in range(B):
        for t in range(T):
            keys = lens[b] - T + t + 1
            for hk in range(Hkv):
                for s in (-1, 1):
                    heads = [h for h in range(hk * G, hk * G + G) if qs[b, t, h] == s]
                    if not heads: continue
                    total, count = np.zeros(hd), 0
                    parts = ((at.get("shared"), min(keys, shared)), (at.get(0 if alias else b), keys - shared))
                    for which, (part, n) in enumerate(parts):
                        if part is None or n <= 0: continue
                        if (which, hk, s, n) in of_shared and (which == 0 or alias): a = of_shared[which, hk, s, n]
                        else:
                            a = of_shared[which, hk, s, n] = (part[1][hk, :n][part[0][hk, :n] == s].sum(0), int((part[0][hk, :n] == s).sum()))
                        total, count = total + a[0], count + a[1]
                    assert count and np.abs(total).max() < 2 ** 24
                    want = total / count
                    off = np.abs(g[b, t, heads] - want)
                    assert (off <= (HALF + 4 * U) * np.abs(want)).all(), (b, t, hk, s, off.max())
    c.free()


# 256 compute units: (a) chunks of thousands of keys for tiles of 64 rows, (b) more slots than a turn of the join takes
# (32 at a width of 256, 64 at 128, 128 at 64), (c) chunks as long as a workgroup's page ids allow
@pytest.mark.parametrize("Hq,Hkv,hd,B,T,shared,own,R", [
    (16, 2, 256, 64, 4, 32768, 512, 64), (16, 2, 256, 64, 4, 32768, 100, 16), (16, 2, 256, 16, 4, 16256, 77, 64), (24, 2, 128, 64, 4, 16384, 300, 32),
    (8, 1, 64, 64, 4, 16384, 200, 256),
    (16, 2, 256, 8, 1, 6592, 200, 64), (8, 1, 256, 2, 1, 7040, 90, 64), (32, 8, 128, 4, 2, 1984, 333, 16), (4, 1, 128, 1, 1, 14000, 5, 16), (4, 1, 64, 1, 1, 26000, 30, 16)])
def test_counted_keys(orn, ctx, Hq, Hkv, hd, B, T, shared, own, R):
    rng = np.random.default_rng(hd + B + own)
    _counted(orn, ctx, rng, [shared // R * R + own - (b * own // 2) // B for b in range(B)], T, shared // R * R, R, Hq, Hkv, hd)


@pytest.mark.parametrize("Hq,Hkv,hd,B,T,n,R", [
    (8, 1, 256, 1, 1, 7000, 64), (4, 1, 128, 1, 2, 13501, 16), (4, 1, 64, 1, 1, 25111, 256), (16, 2, 256, 3, 16, 9001, 64), (8, 2, 64, 1, 64, 30001, 128)])
def test_counted_keys_of_one_sequence(orn, ctx, Hq, Hkv, hd, B, T, n, R):
    """Nothing shared: the same, cut into the sequences' own chunks."""
    rng = np.random.default_rng(hd + n)
    _counted(orn, ctx, rng, [n - 1001 * b for b in range(B)], T, 0, R, Hq, Hkv, hd)


def test_counted_keys_on_small_pages(orn, ctx):
    """Enough sequences for one chunk each, longer than the 4032 rows that a workgroup can name in pages of 16."""
    rng = np.random.default_rng(41)
    _counted(orn, ctx, rng, [9000 - 7 * b for b in range(512)], 1, 0, 16, 4, 1, 64, alias=True)
    _counted(orn, ctx, rng, [9000 - 7 * b for b in range(128)], 40, 0, 16, 4, 1, 64, alias=True)


@pytest.mark.parametrize("lens,T,shared", [([40, 33], 1, 0), ([700, 690, 650], 2, 640), ([2100, 2049], 1, 0), ([300, 280, 10], 20, 256), ([400 + 7 * i for i in range(20)], 1, 384)])
@pytest.mark.parametrize("Hq,Hkv,hd", [(16, 2, 256), (24, 2, 128), (8, 1, 64), (3, 1, 64)])
def test_probabilities(orn, ctx, Hq, Hkv, hd, lens, T, shared):
    rng = np.random.default_rng(hd + T)
    c = Case(ctx, rng, lens, T, shared, 64, Hq, Hkv, hd)
    for b in range(c.B):
        for i in range(-(-max(lens[b], shared) // 64)):
            if b == 0 or i >= shared // 64: c.k[0, c.table[b, i]] = util.f32_to_bf16(rng.integers(-3, 4, (Hkv, 64, hd)).astype(np.float32))
    c.upload(orn)
    q = util.f32_to_bf16(rng.integers(-3, 4, (c.B, T, Hq, hd)).astype(np.float32))
    scale = hd ** -0.5
    g = _f(_attend(orn, ctx, c, q, None, scale))
    qf = _f(q)
    for b in range(c.B):
        k, v = c.rows(c.k, b, lens[b]), c.rows(c.v, b, lens[b])
        for t in range(T):
            n = lens[b] - T + t + 1
            if n <= 0: continue
            for h in range(Hq):
                kk, vv = k[h // (Hq // Hkv), :n], v[h // (Hq // Hkv), :n]
                s = kk @ qf[b, t, h]
                delta = 4 * U * (np.abs(s).max() * scale * 1.4427) + 4 * U
                p = np.exp((s - s.max()) * scale)
                o, A = p @ vv / p.sum(), p @ np.abs(vv) / p.sum()
                tol = HALF * np.abs(o) + 2 * (HALF * HALF + 2 * delta + (n + 8) * U) * A
                off = np.abs(g[b, t, h] - o) - tol
                assert (off <= 0).all(), (b, t, h, off.max(), A.max())
    c.free()
