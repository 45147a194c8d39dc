"""GPU: a prompt that a model has run goes from its caches into pages, and several continuations of it attend there."""
import ctypes as C

import numpy as np
import pytest

import synth
import util
from test_gpu_attn_paged import _want


def test_arguments(orn):
    k, v = C.c_void_p(), C.c_void_p()
    assert orn.lib().ornith_caches_layer_kv(None, 0, C.byref(k), C.byref(v)) == 1
    assert b"null argument" in orn.lib().ornith_last_error()


@pytest.mark.gpu
def test_a_models_prompt_in_pages(orn, ctx):
    s = synth.SynthModel(synth.TINY, seed=11)
    ws = s.upload(orn, ctx)
    model = orn.TextModel(ctx, ws, s.text_config(orn))
    Hkv, hd, Hq = s.cfg["num_key_value_heads"], s.cfg["head_dim"], s.cfg["num_attention_heads"]
    full = [i for i in range(s.cfg["num_hidden_layers"]) if (i + 1) % s.cfg["full_attention_interval"] == 0]
    rng = np.random.default_rng(3)
    toks = rng.integers(0, s.cfg["vocab_size"], 37).astype(np.uint32)
    caches = model.make_cache(24, 4)
    for i in range(0, 37, 12): model.forward(caches, toks[i:i + 12])            # past the 24 rows that they begin with
    n = caches.offset
    assert n == 37 and caches.capacity > 24
    with pytest.raises(orn.OrnithError, match="gated-delta layer"): caches.layer_kv(0)
    for bad in (-1, s.cfg["num_hidden_layers"]):
        with pytest.raises(orn.OrnithError, match="layer"): caches.layer_kv(bad)
    pool = orn.KvPool(ctx, len(full), 12, 16, Hkv, hd, 4, 4)
    first = pool.open()
    pool.extend([first], n)
    rows = {}
    for i, layer in enumerate(full):
        k, v = caches.layer_kv(layer)
        pool.load(first, i, k, v, caches.capacity, 0, n, 0)
        rows[i] = []
        for d in (k, v):
            a = np.empty((Hkv, caches.capacity, hd), np.uint16)
            orn._check(orn.lib().ornith_download(ctx.h, a.ctypes.data_as(C.c_void_p), d.ptr, C.c_size_t(a.nbytes)), "download")
            rows[i].append(a[:, :n])
        assert all(x.any(-1).all() for x in rows[i])                            # (a row of zeros would be one that nobody wrote)
    seqs = [first] + pool.fork(first, 2)
    batch = pool.batch(seqs)
    back = [ctx.alloc(Hkv * 64 * hd * 2) for _ in range(2)]
    q = util.bf16_normal(rng, (3, 1, Hq, hd))
    dq, out = ctx.to_device(q), ctx.alloc(q.nbytes)
    for i in range(len(full)):
        for seq in seqs:
            pool.store(seq, i, *back, 64, 0, n, 0)
            for d, want in zip(back, rows[i]): assert np.array_equal(d.download(np.uint16, (Hkv, 64, hd))[:, :n], want)
        ctx.sdpa_paged_gated(pool.pages, i, batch, dq, None, 1, Hq, hd ** -0.5, out)
        got = util.bf16_to_f32(out.download(np.uint16, q.shape)).astype(np.float64)

        class Rows:
            def rows(self, x, b, n): return util.bf16_to_f32(x[:, :n]).astype(np.float64)
        c = Rows()
        c.lens, c.Hkv, c.k, c.v = [n] * 3, Hkv, *rows[i]
        want, tol = _want(c, q, None, hd ** -0.5)
        assert (np.abs(got - want) <= tol).all(), i
    for d in back + [dq, out]: d.free()
    pool.close()
    caches.close()
    model.close()
    ws.close()
