"""GPU: scores and values that are not finite in the attention over a paged KV cache, wherever its cuts fall.

Keys are u, -u or -inf in one channel, queries u (u: ones and minus ones, u of that channel 1), so that a score is S, -S or -inf and a
weight exactly 1 or, 2 S scale log2(e) > 160 binary orders below, 0."""
import numpy as np
import pytest

import util
from test_gpu_attn_paged import Case, _attend, _f

pytestmark = pytest.mark.gpu

# (query heads, KV heads, head width), lengths, new rows, shared rows: one launch; shared and own chunks; many chunks; tiles of 64 rows
FORMS = [((4, 2, 64), [60], 1, 0), ((16, 2, 256), [100, 150], 2, 0), ((16, 2, 256), [600, 700, 650], 1, 576), ((8, 1, 128), [2500, 2000], 2, 0),
         ((16, 2, 256), [1100, 1190, 1080], 20, 1024), ((16, 1, 64), [900, 800], 20, 0), ((16, 2, 256), [40, 33], 24, 0)]


def _case(rng, ctx, heads, lens, T, shared, key):
    """key(b, j): +1 or -1 for a key of sequence b (its row j) that scores S or -S, 0 for one that scores minus infinity"""
    Hq, Hkv, hd = heads
    c = Case(ctx, rng, lens, T, shared, 64, Hq, Hkv, hd)
    unit = rng.choice([-1.0, 1.0], hd).astype(np.float32)
    unit[5] = 1
    row = {s: util.f32_to_bf16(s * (4 if hd == 256 else 8) * unit) for s in (1, -1)}
    row[0] = np.zeros(hd, np.uint16)
    row[0][5] = 0xff80
    for b in range(c.B):
        for j in range(shared if b else 0, max(lens[b], shared)): c.k[0, c.table[b, j // 64], :, j % 64] = row[key(b, j)]
    return c, np.broadcast_to(util.f32_to_bf16(unit), (c.B, T, Hq, hd)).copy()


def _run(orn, ctx, c, q):
    c.upload(orn)
    got = _f(_attend(orn, ctx, c, q, None, c.hd ** -0.5))
    c.free()
    return got


@pytest.mark.parametrize("heads,lens,T,shared", FORMS)
def test_every_score_is_minus_infinity(orn, ctx, heads, lens, T, shared):
    rng = np.random.default_rng(1)
    c, q = _case(rng, ctx, heads, lens, T, shared, lambda b, j: 0)
    got = _run(orn, ctx, c, q)
    for b, n in enumerate(lens):
        for t in range(T):
            if n - T + t < 0: assert (got[b, t] == 0).all()
            else: assert np.isnan(got[b, t]).all(), (b, t)


@pytest.mark.parametrize("heads,lens,T,shared", FORMS)
def test_parts_of_minus_infinity_scores(orn, ctx, heads, lens, T, shared):
    """Everything but the last rows of the last sequence and one early row of the first: whole chunks and wavefronts have no finite score."""
    rng = np.random.default_rng(2)
    last, one = len(lens) - 1, min(lens[0], max(shared, lens[0])) // 3
    alive = lambda b, j: 1 if (b == last and j >= lens[b] - T - 2 and j >= shared) or (b == 0 and j == one) else 0
    c, q = _case(rng, ctx, heads, lens, T, shared, alive)
    got = _run(orn, ctx, c, q)
    for b, n in enumerate(lens):
        v = c.rows(c.v, b, n)
        for t in range(T):
            seen = [j for j in range(max(n - T + t + 1, 0)) if alive(0 if j < shared else b, j)]
            for h in range(heads[0]):
                if not seen and n - T + t >= 0: assert np.isnan(got[b, t, h]).all(), (b, t, h)
                elif seen:
                    vv = v[h // (heads[0] // heads[1])][seen]
                    want = vv.mean(0)
                    # one reciprocal, sums of len(seen) terms, the rounding to bf16
                    assert (np.abs(got[b, t, h] - want) <= 2.0 ** -8 * np.abs(want) + (len(seen) + 4) * 2.0 ** -24 * np.abs(vv).mean(0)).all(), (b, t, h)


@pytest.mark.parametrize("weight", [1, -1])
@pytest.mark.parametrize("heads,lens,T,shared", FORMS)
def test_infinite_values(orn, ctx, heads, lens, T, shared, weight):
    """An infinite value with the weight of the row's largest score leaves its channel infinite, one whose weight underflows not
    finite, wherever it lies; the other channels, and the rows that do not see it, are as without it."""
    for place in sorted({0, 17, lens[-1] // 2, max(lens[-1] - T - 1, 0), lens[-1] - 1, max(shared - 1, 0)}):
        rng = np.random.default_rng(3)
        c, q = _case(rng, ctx, heads, lens, T, shared, lambda b, j: weight if j == place else 1)
        last = len(lens) - 1
        clean = _run(orn, ctx, c, q)
        c.v[0, c.table[last, place // 64], :, place % 64, 3] = 0xff80
        got = _run(orn, ctx, c, q)
        for b, n in enumerate(lens):
            for t in range(T):
                if n - T + t >= place and (b == last or place < shared):
                    x = got[b, t, :, 3]
                    assert not np.isfinite(x).any(), (place, b, t)
                    if weight == 1 or n - T + t + 1 == 1: assert (x == -np.inf).all(), (place, b, t, x)
                    assert np.array_equal(np.delete(got[b, t], 3, -1), np.delete(clean[b, t], 3, -1)), (place, b, t)
                else: assert np.array_equal(got[b, t], clean[b, t]), (place, b, t)


@pytest.mark.parametrize("heads,lens,T,shared", FORMS)
def test_infinite_values_in_parts_of_no_weight(orn, ctx, heads, lens, T, shared):
    """The last row of every sequence alone has weight; an infinite value lies among rows of which whole chunks have none."""
    last = len(lens) - 1
    for place in sorted({0, 17, lens[-1] // 2, max(shared - 1, 0)}):
        rng = np.random.default_rng(5)
        c, q = _case(rng, ctx, heads, lens, T, shared, lambda b, j: 1 if j >= lens[b] - T else -1)
        clean = _run(orn, ctx, c, q)
        c.v[0, c.table[last, place // 64], :, place % 64, 3] = 0x7f80
        got = _run(orn, ctx, c, q)
        for b, n in enumerate(lens):
            for t in range(T):
                if n - T + t >= place and (b == last or place < shared):
                    assert not np.isfinite(got[b, t, :, 3]).any(), (place, b, t)
                    assert np.array_equal(np.delete(got[b, t], 3, -1), np.delete(clean[b, t], 3, -1)), (place, b, t)
                else: assert np.array_equal(got[b, t], clean[b, t]), (place, b, t)


@pytest.mark.parametrize("heads,lens,T,shared", [((16, 2, 256), [0, 5, 2, 0], 4, 0), ((6, 3, 64), [0, 200, 64, 1], 2, 128), ((16, 2, 256), [0, 900, 3], 24, 64), ((8, 1, 128), [0, 0], 1, 0)])
def test_gates_of_rows_that_see_nothing(orn, ctx, heads, lens, T, shared):
    """Padded rows are zeros whatever their queries and gates hold; the others do not notice."""
    rng = np.random.default_rng(7)
    Hq, Hkv, hd = heads
    c = Case(ctx, rng, lens, T, shared, 64, Hq, Hkv, hd).upload(orn)
    q, qg = util.bf16_normal(rng, (c.B, T, Hq, hd)), util.bf16_normal(rng, (c.B, T, Hq, 2 * hd))
    clean = _attend(orn, ctx, c, q, qg, hd ** -0.5)
    for b, n in enumerate(lens):
        for t in range(T):
            if n - T + t < 0:
                assert not (clean[b, t] & 0x7fff).any()
                q[b, t, :, ::3], qg[b, t, :, ::2], qg[b, t, :, 1::2] = 0x7f80, 0x7fc0, 0xff80
    got = _attend(orn, ctx, c, q, qg, hd ** -0.5)
    assert np.array_equal(got & 0x7fff, clean & 0x7fff) and np.array_equal(got[clean != 0], clean[clean != 0])
    c.free()
