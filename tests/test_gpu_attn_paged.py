"""GPU: the append and the attention over a paged KV cache, for a batch of sequences that share a prefix, against 64 bits.

Tolerances, u = 2^-24. Append: a normed and rotated value is a c - b s (or with +) of fp32 numbers, each product within 16 u of its own
(the norm's sum of up to 256 squares adds (4 + 6 + 4) / 2 u), then half a bf16 step, 2^-8 of the result.
Attention: with A = sum p_j |v_j| / sum p_j, a probability handed on as bf16 is off by 2^-8 of itself, one whose score is off by delta =
(hd + 4) u scale max_j sum_i |q_i k_ji| by 2 delta, and sums over n keys by (n + 8) u; the gate's sigmoid by 16 u; the result is rounded
to bf16, 2^-8 of it. (A probability that is off enters the sum of probabilities too: each term counts twice.)"""
import numpy as np
import pytest

import util

pytestmark = pytest.mark.gpu
U, HALF = 2.0 ** -24, 2.0 ** -8


def _bits(rng, shape, std=1.0):
    return util.f32_to_bf16((rng.standard_normal(shape) * std).astype(np.float32))


def _f(b):
    return util.bf16_to_f32(b).astype(np.float64)


class Case:
    """Sequences of given lengths whose first `shared` rows lie on the same pages, the others on pages of their own in no order; page
    rows that belong to nobody, and whole pages, hold NaN. lens is what the device is told; held the rows there are pages for."""

    def __init__(self, ctx, rng, lens, T, shared, R, Hq, Hkv, hd, layers=1, layer=0, spare=2, stride_more=1):
        self.ctx, self.lens, self.T, self.shared, self.R, self.Hq, self.Hkv, self.hd, self.layers, self.layer = ctx, lens, T, shared, R, Hq, Hkv, hd, layers, layer
        B, ns = len(lens), shared // R
        self.B = B
        held = [max(n, shared) for n in lens]
        need = [-(-n // R) - ns for n in held]
        self.n_pages = ns + sum(need) + spare
        ids = rng.permutation(self.n_pages).astype(np.uint32)
        self.stride = max(1, max(-(-n // R) for n in held)) + stride_more
        self.table = np.full((B, self.stride), 0xfffffff0, np.uint32)   # entries behind a sequence's pages name no page
        at = ns
        for b in range(B):
            self.table[b, :ns] = ids[:ns]
            self.table[b, ns:ns + need[b]] = ids[at:at + need[b]]
            at += need[b]
        self.k, self.v = (np.full((layers, self.n_pages, Hkv, R, hd), 0x7fc0, np.uint16) for _ in range(2))
        for x in (self.k, self.v):
            for b in range(B):
                for i in range(-(-held[b] // R)):
                    n = min(R, held[b] - i * R)
                    if b == 0 or i >= ns: x[layer, self.table[b, i], :, :n] = _bits(rng, (Hkv, n, hd))
        self.max_rows = max(max(lens), shared)

    def rows(self, x, b, n):
        """[Hkv, n, hd] of a sequence's first n rows (float64)"""
        ids = self.table[b, :-(-n // self.R)]
        return _f(x[self.layer][ids].transpose(1, 0, 2, 3).reshape(self.Hkv, -1, self.hd)[:, :n])

    def upload(self, orn):
        c = self.ctx
        self.dk, self.dv = ([c.to_device(x[i]) for i in range(self.layers)] for x in (self.k, self.v))
        self.dt, self.dl = c.to_device(self.table), c.to_device(np.array(self.lens, np.int32))
        self.pages = orn.KvPages(self.dk, self.dv, self.n_pages, self.R, self.Hkv, self.hd)
        self.batch = orn.KvBatch(self.B, self.dt, self.stride, self.dl, self.shared, self.max_rows)
        return self

    def free(self, *more):
        for b in self.dk + self.dv + [self.dt, self.dl] + list(more):
            if b: b.free()


def _want(c, q, qg, scale):
    """(result, tolerance) [B, T, Hq, hd]"""
    B, T, Hq, hd = q.shape
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    qf = _f(q)
    g = 1 / (1 + np.exp(-_f(qg[..., hd:]))) if qg is not None else np.ones(q.shape)
    for b in range(B):
        n = c.lens[b]
        if n <= 0: continue
        k, v = c.rows(c.k, b, n), c.rows(c.v, b, n)
        for t in range(T):
            keys = n - T + t + 1
            if keys <= 0: continue
            for h in range(Hq):
                kk, vv = k[h // (Hq // c.Hkv), :keys], v[h // (Hq // c.Hkv), :keys]
                s = kk @ qf[b, t, h] * scale
                p = np.exp(s - s.max())
                L = p.sum()
                o, A = p @ vv / L, p @ np.abs(vv) / L
                delta = (hd + 4) * U * scale * (np.abs(kk) @ np.abs(qf[b, t, h])).max()
                y = o * g[b, t, h]
                out[b, t, h] = y
                tol[b, t, h] = 2 * (HALF + 2 * delta + (keys + 8) * U) * A * g[b, t, h] + (HALF + 16 * U) * np.abs(y)
    return out, tol


def _attend(orn, ctx, c, q, qg, scale, poison=True):
    dq, dg = ctx.to_device(q), ctx.to_device(qg) if qg is not None else None
    out = ctx.to_device(np.full(q.size + 64, 0x7fc1, np.uint16))
    ctx.sdpa_paged_gated(c.pages, c.layer, c.batch, dq, dg, c.T, c.Hq, scale, out)
    got = out.download(np.uint16, (q.size + 64,))
    assert (got[q.size:] == 0x7fc1).all()               # what lies behind the last row is left as it was
    for x in (dq, dg, out):
        if x: x.free()
    return got[:q.size].reshape(q.shape)


def _check(orn, ctx, rng, c, gate=True, std=1.0):
    q = _bits(rng, (c.B, c.T, c.Hq, c.hd), std)
    qg = _bits(rng, (c.B, c.T, c.Hq, 2 * c.hd)) if gate else None
    if qg is not None: qg[..., :c.hd] = 0x7fc0           # the query half is not read
    scale = c.hd ** -0.5
    got = _attend(orn, ctx, c, q, qg, scale)
    want, tol = _want(c, q, qg, scale)
    g = _f(got)
    assert np.isfinite(g).all()
    over = np.abs(g - want) - tol
    assert (over <= 0).all(), (np.unravel_index(over.argmax(), over.shape), over.max(), np.abs(g - want).max())
    assert np.array_equal(_attend(orn, ctx, c, q, qg, scale), got)      # and the same bits again
    return got


SHAPES = [(16, 2, 256), (8, 8, 64), (12, 4, 128), (4, 1, 256), (3, 1, 64), (24, 2, 128), (6, 2, 256), (40, 2, 64), (5, 5, 128)]


@pytest.mark.parametrize("Hq,Hkv,hd", SHAPES)
@pytest.mark.parametrize("R", [16, 64, 256])
def test_heads_and_page_sizes(orn, ctx, Hq, Hkv, hd, R):
    rng = np.random.default_rng(Hq * 100 + R)
    for lens, T, shared in (([1, 2, 3], 1, 0), ([300, 257, 260], 2, 256), ([700, 1100, 513, 600], 1, 512)):
        c = Case(ctx, rng, lens, T, shared, R, Hq, Hkv, hd, layers=2, layer=1).upload(orn)
        _check(orn, ctx, rng, c)
        c.free()


@pytest.mark.parametrize("lens,T,shared,R", [
    ([1], 1, 0, 16), ([15], 1, 0, 16), ([16], 1, 0, 16), ([17], 1, 0, 16), ([63, 64, 65, 66], 1, 0, 64), ([127, 128, 129, 255, 256, 257], 3, 0, 32), ([5, 900], 4, 0, 64),
    ([64], 1, 64, 64), ([65], 1, 64, 64), ([64, 64], 1, 64, 64), ([66, 64, 70, 1000], 2, 64, 64), ([512 + i for i in range(1, 18)], 1, 512, 16), ([2049], 8, 2048, 256),
    ([3000, 2900], 16, 2816, 64), ([200, 130], 64, 0, 64), ([128 + 30] * 33, 1, 128, 128), ([4000], 1, 0, 16), ([4096 + 7, 4096 + 1], 1, 4096, 64), ([40] * 70, 2, 32, 32),
    # a shared part that ends inside a key block, and one as long as everything
    ([176, 200, 180], 1, 176, 16), ([336, 340], 2, 336, 16), ([1040] * 3, 1, 1040, 16)])
def test_lengths(orn, ctx, lens, T, shared, R):
    rng = np.random.default_rng(sum(lens) + T)
    c = Case(ctx, rng, lens, T, shared, R, 16, 2, 256).upload(orn)
    _check(orn, ctx, rng, c, gate=bool(sum(lens) % 2), std=2.0)
    c.free()


@pytest.mark.parametrize("lens,T,shared", [([0, 5, 0], 1, 0), ([3, 40, 1, 0], 4, 0), ([0, 0], 2, 0), ([0, 200, 64, 1, 127, 128, 129], 1, 128), ([130, 2, 128, 64, 0], 5, 128),
                                           ([0, 1500, 600], 2, 1024)])
def test_short_and_empty_sequences(orn, ctx, lens, T, shared):
    """Padded batches: rows of negative position are zeros, sequences that end inside (or before) the shared rows see what they hold."""
    rng = np.random.default_rng(7 + len(lens))
    for Hq, Hkv, hd in ((16, 2, 256), (6, 3, 64)):
        c = Case(ctx, rng, lens, T, shared, 64, Hq, Hkv, hd).upload(orn)
        got = _check(orn, ctx, rng, c)
        for b, n in enumerate(lens):
            for t in range(T):
                if n - T + t < 0: assert not (got[b, t] & 0x7fff).any()
        c.free()


def test_device_lengths_and_ids_out_of_range(orn, ctx):
    """What cannot be checked on the host: lengths below 0 and above max_rows, page ids past the end."""
    rng = np.random.default_rng(11)
    c = Case(ctx, rng, [200, 200, 200], 1, 64, 64, 16, 2, 256).upload(orn)
    q, qg = _bits(rng, (3, 1, 16, 256)), _bits(rng, (3, 1, 16, 512))
    want = _attend(orn, ctx, c, q, qg, 0.0625)
    c.dl.upload(np.array([2 ** 31 - 1, -5, 201], np.int32))
    got = _attend(orn, ctx, c, q, qg, 0.0625)
    assert np.array_equal(got[[0, 2]], want[[0, 2]]) and not (got[1] & 0x7fff).any()
    c.dl.upload(np.array([200, 200, 200], np.int32))
    # a wrong id reads the last page: give that page the rows and the result must be the same
    last = c.n_pages - 1
    own = c.table[1, 2]
    for x, d in ((c.k, c.dk), (c.v, c.dv)):
        x[0, [own, last]] = x[0, [last, own]]
        d[0].upload(x[0])
    t = c.table.copy()
    swap = {int(own): last, last: int(own)}
    for i in np.ndindex(t.shape): t[i] = swap.get(int(t[i]), int(t[i]))
    t[1, 2] = 0xffffffff
    c.dt.upload(t)
    assert np.array_equal(_attend(orn, ctx, c, q, qg, 0.0625), want)
    c.free()


@pytest.mark.parametrize("Hq,Hkv,hd", [(16, 2, 256), (4, 2, 128), (2, 2, 64)])
@pytest.mark.parametrize("lens,T,shared", [([70, 90], 4, 0), ([520, 700], 8, 512), ([200, 131], 3, 128), ([1030] * 9, 4, 1024)])
def test_values_of_later_rows_stay_out(orn, ctx, Hq, Hkv, hd, lens, T, shared):
    """Infinite and NaN keys and values in a row that only later queries see: the earlier rows are what they are without them."""
    rng = np.random.default_rng(T)
    c = Case(ctx, rng, lens, T, shared, 64, Hq, Hkv, hd).upload(orn)
    q, qg = _bits(rng, (len(lens), T, Hq, hd)), _bits(rng, (len(lens), T, Hq, 2 * hd))
    clean = _attend(orn, ctx, c, q, qg, hd ** -0.5)
    for b, t, x, bits in ((0, T - 1, c.k, 0x7fc0), (0, T - 1, c.v, 0x7f80), (1, 1, c.v, 0x7fc0), (1, T - 1, c.k, 0xff80)):
        pos = lens[b] - T + t
        x[0, c.table[b, pos // 64], :, pos % 64, ::7] = bits
    c.dk[0].upload(c.k[0])
    c.dv[0].upload(c.v[0])
    got = _attend(orn, ctx, c, q, qg, hd ** -0.5)
    assert np.array_equal(got[0, :T - 1], clean[0, :T - 1]) and np.array_equal(got[1, :1], clean[1, :1])
    assert np.array_equal(got[2:], clean[2:])
    g = util.bf16_to_f32(got)
    assert np.isnan(g[0, T - 1]).all() and np.isnan(g[1, 1:][..., ::7]).all()
    # a value row holds the NaN in every seventh channel only: the others go on (rows before the infinite key)
    assert np.isfinite(np.delete(g[1, 1:T - 1], np.arange(0, hd, 7), -1)).all()
    c.free()


def test_rows_that_see_only_minus_infinity_scores(orn, ctx):
    """Keys of the type's lowest value and of minus infinity among ordinary ones have no weight."""
    rng = np.random.default_rng(13)
    c = Case(ctx, rng, [100, 300], 1, 64, 64, 4, 2, 64).upload(orn)
    q = np.abs(_bits(rng, (2, 1, 4, 64)) & 0x7fff).astype(np.uint16)       # positive queries
    clean_k = c.k.copy()
    drop = [3, 10, 63]
    c.k[0, c.table[0, 0], :, drop] = 0xff80
    c.k[0, c.table[1, 2], :, 7] = 0xff7f
    c.dk[0].upload(c.k[0])
    got = _f(_attend(orn, ctx, c, q, None, 0.125))
    qf = _f(q)
    for b, n in enumerate(c.lens):
        k, v = c.rows(c.k, b, n), c.rows(c.v, b, n)
        for h in range(4):
            with np.errstate(invalid="ignore", over="ignore"):
                s = k[h // 2] @ qf[b, 0, h] * 0.125
            s = np.where(s < -1e30, -np.inf, s)
            p = np.exp(s - s.max())
            o, A = p @ v[h // 2] / p.sum(), p @ np.abs(v[h // 2]) / p.sum()
            assert (np.abs(got[b, 0, h] - o) <= 2 * HALF * 1.1 * A + HALF * np.abs(o) + 1e-4).all()
    assert not np.array_equal(c.k, clean_k)
    c.free()


def test_peaked_scores(orn, ctx):
    """Scores hundreds apart, the largest in the last rows or in the first: the running maximum moves late or never."""
    rng = np.random.default_rng(17)
    for order in (1, -1):
        c = Case(ctx, rng, [1500, 1400, 1301], 1, 1280, 64, 16, 2, 256)
        q = _bits(rng, (3, 1, 16, 256))
        q[:, :, :] = q[0, 0, 0]
        for b in range(3):
            for j in range(c.lens[b]):
                f = 0.001 * (j if order > 0 else c.lens[b] - j)
                c.k[0, c.table[b, j // 64], :, j % 64] = util.f32_to_bf16((util.bf16_to_f32(q[0, 0, 0]) * f).astype(np.float32))
        c.upload(orn)
        got, (want, tol) = _f(_attend(orn, ctx, c, q, None, 0.0625)), _want(c, q, None, 0.0625)
        assert (np.abs(got - want) <= tol).all(), order
        c.free()


def test_agrees_with_the_contiguous_decode(orn, ctx):
    """One sequence over pages and the same rows in a contiguous cache through sdpa_decode_gated: both within their roundings."""
    rng = np.random.default_rng(19)
    n, T, Hq, Hkv, hd = 777, 3, 16, 2, 256
    c = Case(ctx, rng, [n], T, 0, 64, Hq, Hkv, hd).upload(orn)
    q, qg = _bits(rng, (1, T, Hq, hd)), _bits(rng, (1, T, Hq, 2 * hd))
    got = _f(_attend(orn, ctx, c, q, qg, 0.0625))
    cap = 1024
    dk, dv, dq, dg, out = ctx.alloc(Hkv * cap * hd * 2), ctx.alloc(Hkv * cap * hd * 2), ctx.to_device(q), ctx.to_device(qg), ctx.alloc(q.nbytes)
    ctx.kv_pages_store(c.pages, 0, dk, dv, cap, 0, n, c.table[0, :-(-n // 64)], 0)
    ctx.sdpa_decode_gated(dq, dk, dv, dg, T, Hq, Hkv, hd, n - T, cap, 0.0625, out)
    ref = _f(out.download(np.uint16, q.shape))
    want, tol = _want(c, q, qg, 0.0625)
    # (the contiguous form rounds the attention, and four steps of the gate, to bf16)
    assert (np.abs(got - ref) <= tol + 6 * HALF * np.abs(want)).all()
    c.free(dk, dv, dq, dg, out)


def _append(orn, ctx, c, rng, rope, eps=1e-6, npos=None):
    B, T, Hq, Hkv, hd = c.B, c.T, c.Hq, c.Hkv, c.hd
    qg, kx, vx = _bits(rng, (B, T, Hq, 2 * hd)), _bits(rng, (B, T, Hkv, hd)), _bits(rng, (B, T, Hkv, hd))
    qw, kw = (util.f32_to_bf16((1 + 0.1 * rng.standard_normal(hd)).astype(np.float32)) for _ in range(2))
    npos = npos or max(c.max_rows, 1)
    cos, sin = ctx.rope_table(npos, rope, 1e4) if rope else (ctx.alloc(16), ctx.alloc(16))
    table = [x.download(np.float32, (npos, rope // 2)).astype(np.float64) for x in (cos, sin)] if rope else None
    dq = ctx.to_device(np.full(B * T * Hq * hd + 64, 0x7fc1, np.uint16))
    d = [ctx.to_device(x) for x in (qg, kx, vx, qw, kw)]
    ctx.attn_prep_paged(c.pages, c.layer, c.batch, *d, T, Hq, rope, eps, cos, sin, npos, dq)
    q = dq.download(np.uint16, (B * T * Hq * hd + 64,))
    assert (q[-64:] == 0x7fc1).all()
    for x in d + [dq, cos, sin]: x.free()

    def head(x, w, pos):
        y = _f(x)
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * _f(w)
        z, mag, h = y.copy(), np.abs(y), rope // 2
        if rope:
            co, si = table[0][pos], table[1][pos]
            z[..., :h], z[..., h:rope] = y[..., :h] * co - y[..., h:rope] * si, y[..., h:rope] * co + y[..., :h] * si
            mag[..., :h], mag[..., h:rope] = np.abs(y[..., :h] * co) + np.abs(y[..., h:rope] * si), np.abs(y[..., h:rope] * co) + np.abs(y[..., :h] * si)
        return z, HALF * np.abs(z) + 32 * U * mag

    q = q[:-64].reshape(B, T, Hq, hd)
    k, v = (x[c.layer].download(np.uint16, c.k.shape[1:]) for x in (c.dk, c.dv))
    wk, wv = c.k[c.layer].copy(), c.v[c.layer].copy()
    for b in range(B):
        for t in range(T):
            pos = c.lens[b] - T + t
            if pos < 0:
                assert (q[b, t] == 0x7fc1).all()
                continue
            page, row = c.table[b, pos // c.R], pos % c.R
            for got, x, w in ((q[b, t], qg[b, t, :, :hd], qw), (k[page, :, row], kx[b, t], kw)):
                z, tol = head(x, w, pos)
                assert (np.abs(_f(got) - z) <= tol).all(), (b, t)
            wk[page, :, row], wv[page, :, row] = k[page, :, row], vx[b, t]
    assert np.array_equal(k, wk) and np.array_equal(v, wv)              # every other row as it was
    return q


@pytest.mark.parametrize("Hq,Hkv,hd,rope", [(16, 2, 256, 64), (16, 2, 256, 256), (16, 2, 256, 8), (8, 8, 64, 16), (5, 5, 64, 64), (12, 4, 128, 32), (6, 1, 128, 128), (4, 1, 256, 0)])
@pytest.mark.parametrize("lens,T,R", [([1], 1, 16), ([16, 17, 200], 1, 16), ([70, 64, 3, 300], 5, 64), ([0, 2, 40], 4, 32), ([256, 257], 64, 256)])
def test_append(orn, ctx, Hq, Hkv, hd, rope, lens, T, R):
    rng = np.random.default_rng(hd + rope + T)
    c = Case(ctx, rng, lens, T, 0, R, Hq, Hkv, hd, layers=2, layer=1).upload(orn)
    _append(orn, ctx, c, rng, rope)
    c.free()


def test_append_through_a_wrong_page_id(orn, ctx):
    """A row whose table entry names no page goes nowhere; the others are written."""
    rng = np.random.default_rng(23)
    c = Case(ctx, rng, [65, 66], 2, 0, 64, 4, 2, 64).upload(orn)
    t = c.table.copy()
    t[0, 1] = c.n_pages
    c.dt.upload(t)
    bufs = [ctx.to_device(_bits(rng, s)) for s in ((2, 2, 4, 128), (2, 2, 2, 64), (2, 2, 2, 64), (64,), (64,))]
    cos, sin = ctx.rope_table(66, 64, 1e4)
    dq = ctx.alloc(2 * 2 * 4 * 64 * 2)
    ctx.attn_prep_paged(c.pages, 0, c.batch, *bufs, 2, 4, 64, 1e-6, cos, sin, 66, dq)
    v = c.dv[0].download(np.uint16, c.v.shape[1:])
    vx = bufs[2].download(np.uint16, (2, 2, 2, 64))
    w = c.v[0].copy()
    w[t[0, 0], :, 63], w[t[1, 1], :, 0], w[t[1, 1], :, 1] = vx[0, 0], vx[1, 0], vx[1, 1]
    assert np.array_equal(v, w)
    c.free(cos, sin, dq, *bufs)


def test_continuations_of_one_prompt(orn, ctx):
    """A prompt's contiguous cache goes into a pool, is forked, and every continuation takes its own tokens, three steps of one row and
    one of two with a row taken back: append, attention, and the scores of what was chosen. Each step against 64 bits over the rows that
    each sequence should hold by then."""
    rng = np.random.default_rng(29)
    Hq, Hkv, hd, R, n, B, V, rope = 16, 2, 256, 64, 203, 5, 5003, 64
    pool = orn.KvPool(ctx, 2, 24, R, Hkv, hd, 8, 8)
    cap = 256
    kc, vc = _bits(rng, (Hkv, cap, hd)), _bits(rng, (Hkv, cap, hd))
    dk, dv = ctx.to_device(kc), ctx.to_device(vc)
    first = pool.open()
    pool.extend([first], n)
    pool.load(first, 1, dk, dv, cap, 0, n, 0)
    seqs = [first] + pool.fork(first, B - 1)
    rows = [[(kc[:, j], vc[:, j]) for j in range(n)] for _ in range(B)]
    cos, sin = ctx.rope_table(512, rope, 1e7)
    qw, kw = (ctx.to_device(util.f32_to_bf16(np.ones(hd, np.float32))) for _ in range(2))
    for step, T in enumerate((1, 1, 2, 1)):
        pool.extend(seqs, T)
        batch = pool.batch(seqs)
        assert batch.s.shared_rows == 192
        qg, kx, vx = _bits(rng, (B, T, Hq, 2 * hd)), _bits(rng, (B, T, Hkv, hd)), _bits(rng, (B, T, Hkv, hd))
        dg, dkx, dvx = (ctx.to_device(x) for x in (qg, kx, vx))
        dq, out = ctx.alloc(B * T * Hq * hd * 2), ctx.alloc(B * T * Hq * hd * 2)
        ctx.attn_prep_paged(pool.pages, 1, batch, dg, dkx, dvx, qw, kw, T, Hq, rope, 1e-6, cos, sin, 512, dq)
        ctx.sdpa_paged_gated(pool.pages, 1, batch, dq, dg, T, Hq, hd ** -0.5, out)
        q, got = dq.download(np.uint16, (B, T, Hq, hd)), _f(out.download(np.uint16, (B, T, Hq, hd)))
        tk, tv = ctx.alloc(Hkv * 512 * hd * 2), ctx.alloc(Hkv * 512 * hd * 2)
        for b, s in enumerate(seqs):
            m, _ = pool.seq(s)
            pool.store(s, 1, tk, tv, 512, 0, m, 0)
            k, v = (x.download(np.uint16, (Hkv, 512, hd))[:, :m] for x in (tk, tv))
            old = m - T
            assert old == len(rows[b])
            for j in range(old): assert np.array_equal(k[:, j], rows[b][j][0]) and np.array_equal(v[:, j], rows[b][j][1]), (step, b, j)
            assert np.array_equal(v[:, old:], vx[b].transpose(1, 0, 2))
            rows[b] += [(k[:, old + t], v[:, old + t]) for t in range(T)]

            class One:
                lens, Hkv, k_, v_ = [m], 2, k, v
                def rows(self, x, _, n): return _f(x[:, :n])
            one = One()
            one.k, one.v = k, v
            want, tol = _want(one, q[b:b + 1], qg[b:b + 1], hd ** -0.5)
            assert (np.abs(got[b] - want[0]) <= tol[0]).all(), (step, b)
        if T == 2:                                        # the second row is a draft that was not accepted
            for b, s in enumerate(seqs):
                pool.truncate(s, len(rows[b]) - 1)
                rows[b].pop()
        logits = (rng.standard_normal((B, V)) * 3).astype(np.float32)
        token = logits.argmax(1).astype(np.uint32)
        dx, dt, dl = ctx.to_device(logits), ctx.to_device(token), ctx.alloc(B * 4)
        ctx.token_logprobs(dx, orn.F32, B, V, dt, 1, 0, dl)
        lp = dl.download(np.float32, (B,))
        x = logits.astype(np.float64)
        assert np.allclose(lp, x.max(1) - np.log(np.exp(x - x.max(1, keepdims=True)).sum(1)) - x.max(1), rtol=0, atol=1e-5)
        for d in (dg, dkx, dvx, dq, out, tk, tv, dx, dt, dl): d.free()
    for s in seqs[1:]: pool.close_seq(s)
    assert pool.stats()[0] == 4                           # 207 rows of the one that was kept
    for d in (dk, dv, cos, sin, qw, kw): d.free()
    pool.close()


def test_two_contexts(orn, ctx):
    """Calls of two contexts, issued in turn and in flight together, each with partial sums of its own."""
    other, rng = orn.Ctx(0), np.random.default_rng(29)
    got = []
    for x in (ctx, other):
        cases = []
        rng = np.random.default_rng(29)
        for lens, T, shared in (([3000, 2500], 2, 2432), ([900] * 12, 4, 832), ([5000], 1, 0)):
            c = Case(x, rng, lens, T, shared, 64, 16, 2, 256).upload(orn)
            q = _bits(rng, (c.B, T, 16, 256))
            cases.append((c, q, x.to_device(q), x.alloc(q.nbytes)))
        got.append(cases)
    for i in range(3):
        for cases in got:
            c, q, dq, out = cases[i]
            c.ctx.sdpa_paged_gated(c.pages, 0, c.batch, dq, None, c.T, 16, 0.0625, out)
    for i in range(3):
        a, b = (cases[i][3].download(np.uint16, cases[i][1].shape) for cases in got)
        c, q = got[0][i][:2]
        want, tol = _want(c, q, None, 0.0625)
        assert np.array_equal(a, b) and (np.abs(_f(a) - want) <= tol).all(), i
    for cases in got:
        for c, _, dq, out in cases: c.free(dq, out)
    other.close()


def test_pages_past_four_gigabytes(orn, ctx):
    """Page ids whose bytes lie behind 2^32, in every call over pages: the same bits as at low ids."""
    rng = np.random.default_rng(31)
    lens, T, R, Hq, Hkv, hd, rope, big = [300, 257], 2, 64, 16, 2, 256, 64, 70000
    low = Case(ctx, rng, lens, T, 128, R, Hq, Hkv, hd).upload(orn)
    up = big - low.n_pages
    k, v = (ctx.alloc(big * Hkv * R * hd * 2) for _ in range(2))
    pages = orn.KvPages([k], [v], big, R, Hkv, hd)
    one = [ctx.alloc(Hkv * R * hd * 2) for _ in range(2)]
    named = sorted({int(i) for b in range(2) for i in low.table[b, :-(-lens[b] // R)]})
    for i in named:
        for x, a in zip(one, (low.k, low.v)): x.upload(a[0, i])
        ctx.kv_pages_load(pages, 0, *one, R, 0, R, [i + up], 0)
    table = low.table.copy()
    table[table < low.n_pages] += np.uint32(up)
    dt = ctx.to_device(table)
    batch = orn.KvBatch(2, dt, low.stride, low.dl, 128, low.max_rows)
    new = [ctx.to_device(_bits(rng, s)) for s in ((2, T, Hq, 2 * hd), (2, T, Hkv, hd), (2, T, Hkv, hd), (hd,), (hd,))]
    cos, sin = ctx.rope_table(low.max_rows, rope, 1e4)
    res = []
    for p, b in ((low.pages, low.batch), (pages, batch)):
        q, out = ctx.alloc(2 * T * Hq * hd * 2), ctx.alloc(2 * T * Hq * hd * 2)
        ctx.attn_prep_paged(p, 0, b, *new, T, Hq, rope, 1e-6, cos, sin, low.max_rows, q)
        ctx.sdpa_paged_gated(p, 0, b, q, new[0], T, Hq, 0.0625, out)
        res.append([x.download(np.uint16, (2, T, Hq, hd)) for x in (q, out)])
        for x in (q, out): x.free()
    assert all(np.array_equal(a, b) for a, b in zip(*res)) and np.isfinite(_f(res[0][1])).all()
    ctx.kv_pages_copy(pages, [i + up for i in named], [i + 7 for i in range(len(named))], R)
    kv = [x.download(np.uint16, low.k.shape[1:]) for x in (low.dk[0], low.dv[0])]
    for n, i in enumerate(named):
        for page in (i + up, n + 7):
            ctx.kv_pages_store(pages, 0, *one, R, 0, R, [page], 0)
            for x, a in zip(one, kv): assert np.array_equal(x.download(np.uint16, (Hkv, R, hd)), a[i]), (i, page)
    low.free(k, v, dt, cos, sin, *one, *new)


# more than 128 query rows a KV head: tiles of 64 rows, in the shared part alone or in the sequences' own too
MANY = [(16, 2, 256), (24, 2, 128), (8, 1, 64)]


@pytest.mark.parametrize("Hq,Hkv,hd", MANY)
@pytest.mark.parametrize("lens,T,shared,R", [([300, 280, 10], 20, 256, 64), ([400 + 7 * i for i in range(20)], 1, 384, 64), ([90] * 9 + [0, 3, 128], 3, 64, 16), ([65], 33, 0, 16),
                                             ([1100, 1025], 24, 1024, 256), ([130, 128, 129], 20, 128, 128)])
def test_many_rows(orn, ctx, Hq, Hkv, hd, lens, T, shared, R):
    rng = np.random.default_rng(hd + T)
    c = Case(ctx, rng, lens, T, shared, R, Hq, Hkv, hd).upload(orn)
    _check(orn, ctx, rng, c, std=2.0)
    c.free()


@pytest.mark.parametrize("Hq,Hkv,hd", MANY)
@pytest.mark.parametrize("lens,T,shared", [([520, 700], 20, 512), ([300, 290], 25, 0), ([260] * 30, 2, 256)])
def test_values_of_later_rows_stay_out_of_many(orn, ctx, Hq, Hkv, hd, lens, T, shared):
    test_values_of_later_rows_stay_out(orn, ctx, Hq, Hkv, hd, lens, T, shared)
