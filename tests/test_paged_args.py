"""CPU: what the calls over paged KV caches and the token scores refuse. Arguments are checked before anything of the context is
touched, so a call that is right in everything but its context says just that."""
import ctypes as C

import numpy as np
import pytest


def _refused(orn, rc, text):
    assert rc == 1
    assert text in orn.lib().ornith_last_error().decode(), orn.lib().ornith_last_error().decode()


class _At:
    def __init__(self, a): self.ptr = C.c_void_p(a)


def _pages(orn, n_layers=2, n_pages=8, page_rows=64, Hkv=2, hd=256, at=0x1000):
    return orn.KvPages([_At(at)] * n_layers, [_At(at)] * n_layers, n_pages, page_rows, Hkv, hd)


def _batch(orn, B=2, stride=4, shared=64, most=200, at=0x1000):
    return orn.KvBatch(B, _At(at), stride, _At(at), shared, most)


BAD_PAGES = [(dict(page_rows=48), "power of two"), (dict(page_rows=8), "power of two"), (dict(page_rows=512), "power of two"),
             (dict(hd=96), "head width"), (dict(n_pages=0), "0 pages"), (dict(Hkv=0), "0 KV heads"), (dict(at=0x1008), "misaligned"),
             (dict(at=0), "null or misaligned")]


def _copy(orn, pages, src, dst, rows=64):
    src, dst = np.array(src, np.uint32), np.array(dst, np.uint32)
    return orn.lib().ornith_kv_pages_copy(None, C.byref(pages.s), src.ctypes.data_as(C.c_void_p), dst.ctypes.data_as(C.c_void_p), src.size, rows)


def _sdpa(orn, pages, batch, layer=0, T=2, Hq=16, scale=1.0, q=0x1000, qg=0x1000, out=0x1000):
    return orn.lib().ornith_sdpa_paged_gated(None, C.byref(pages.s), layer, C.byref(batch.s) if batch else None, C.c_void_p(q), C.c_void_p(qg), T, Hq,
                                             C.c_float(scale), C.c_void_p(out))


def _prep(orn, pages, batch, layer=0, T=2, Hq=16, rope=64, npos=1000, p=0x1000):
    return orn.lib().ornith_attn_prep_paged(None, C.byref(pages.s), layer, C.byref(batch.s), *[C.c_void_p(p)] * 5, T, Hq, rope, C.c_float(1e-6),
                                            C.c_void_p(p), C.c_void_p(p), npos, C.c_void_p(p))


@pytest.mark.parametrize("change,text", BAD_PAGES)
def test_pages_descriptor(orn, change, text):
    for call in (lambda p: _copy(orn, p, [0], [1], 1), lambda p: _sdpa(orn, p, _batch(orn, shared=0, most=10)), lambda p: _prep(orn, p, _batch(orn, shared=0, most=10))):
        _refused(orn, call(_pages(orn, **change)), text)


def test_copy(orn):
    pages = _pages(orn)
    _refused(orn, _copy(orn, pages, [0, 1], [2, 2]), "written twice")
    _refused(orn, _copy(orn, pages, [0, 2], [2, 3]), "read and written")
    _refused(orn, _copy(orn, pages, [3], [3]), "read and written")
    _refused(orn, _copy(orn, pages, [8], [3]), "page 8 to 3 of 8")
    _refused(orn, _copy(orn, pages, [0], [0xffffffff]), "of 8")
    _refused(orn, _copy(orn, pages, [0], [1], 65), "65 rows")
    _refused(orn, _copy(orn, pages, [0], [1], -1), "-1 rows")
    _refused(orn, _copy(orn, pages, [0, 0], [1, 2]), "null context")


@pytest.mark.parametrize("change,text", [
    (dict(row0=-1), "rows [-1"), (dict(row0=90), "of a cache of 100"), (dict(cap=10), "of a cache of 10"), (dict(rows=-1), "rows"), (dict(at=-1), "rows [-1"),
    (dict(at=120), "of 2 pages"), (dict(ids=[1, 1]), "twice"), (dict(ids=[1, 8]), "page 8 of 8"), (dict(layer=2), "layer 2"), (dict(k=0), "null or misaligned cache"),
    (dict(k=0x1004), "misaligned"), (dict(ids=[]), "of 0 pages"), (dict(), "null context")])
def test_load_and_store(orn, change, text):
    a = dict(layer=0, k=0x1000, cap=100, row0=0, rows=70, ids=[1, 2], at=10)
    a.update(change)
    ids = np.array(a["ids"], np.uint32)
    for name in ("load", "store"):
        if name == "store" and a["ids"] == [1, 1]:
            text = "null context"                       # reading a page twice is harmless
        rc = getattr(orn.lib(), "ornith_kv_pages_" + name)(None, C.byref(_pages(orn).s), a["layer"], C.c_void_p(a["k"]), C.c_void_p(a["k"]), a["cap"],
                                                           a["row0"], a["rows"], ids.ctypes.data_as(C.c_void_p), ids.size, a["at"])
        _refused(orn, rc, text)


@pytest.mark.parametrize("change,text", [
    (dict(B=0), "0 sequences"), (dict(B=4097), "4097 sequences"), (dict(at=0), "no page tables"), (dict(stride=0), "no page tables"), (dict(most=257), "257 rows in 4 pages"),
    (dict(most=-1), "-1 rows"), (dict(shared=32), "32 shared rows"), (dict(shared=-64), "shared rows"), (dict(shared=256, most=200), "256 shared rows")])
def test_batch_descriptor(orn, change, text):
    for call in (_sdpa, _prep):
        _refused(orn, call(orn, _pages(orn), _batch(orn, **change)), text)


@pytest.mark.parametrize("change,text", [
    (dict(T=0), "0 new rows"), (dict(T=65), "65 new rows"), (dict(Hq=15), "15 query heads"), (dict(Hq=0), "0 query heads"), (dict(layer=2), "layer 2"), (dict(layer=-1), "layer -1"),
    (dict(), "null context")])
def test_both_calls(orn, change, text):
    for call in (_sdpa, _prep):
        _refused(orn, call(orn, _pages(orn), _batch(orn), **change), text)
    _refused(orn, _sdpa(orn, _pages(orn), _batch(orn, B=4096, most=10, shared=0), T=16), "65535 in all")


@pytest.mark.parametrize("scale", [0.0, -1.0, float("nan"), float("inf")])
def test_attention_scale(orn, scale):
    _refused(orn, _sdpa(orn, _pages(orn), _batch(orn), scale=scale), "scale")


def test_attention_pointers(orn):
    _refused(orn, _sdpa(orn, _pages(orn), None), "null batch")
    _refused(orn, _sdpa(orn, _pages(orn), _batch(orn), q=0), "null argument")
    _refused(orn, _sdpa(orn, _pages(orn), _batch(orn), q=0x1002), "16-byte")
    _refused(orn, _sdpa(orn, _pages(orn), _batch(orn), qg=0), "null context")     # without a gate


@pytest.mark.parametrize("change,text", [(dict(rope=4), "4 rotary"), (dict(rope=260), "260 rotary"), (dict(npos=199), "199 positions"), (dict(p=0), "null argument")])
def test_prep(orn, change, text):
    _refused(orn, _prep(orn, _pages(orn), _batch(orn), **change), text)


def _score(orn, x=0x1000, dtype=1, rows=2, V=10, stride=10, tokens=0x1000, n=1, k=3, lp=0x1000, ids=0x1000, tlp=0x1000):
    return orn.lib().ornith_token_logprobs(None, C.c_void_p(x), dtype, rows, V, C.c_int64(stride), C.c_void_p(tokens), n, k, C.c_void_p(lp), None, None,
                                           C.c_void_p(ids), C.c_void_p(tlp))


@pytest.mark.parametrize("change,text", [
    (dict(x=0), "null logits"), (dict(x=0x1001), "misaligned"), (dict(x=0x1002, dtype=0), "misaligned"), (dict(dtype=2), "dtype"), (dict(rows=0), "rows=0"), (dict(V=0), "V=0"),
    (dict(stride=9), "row_stride=9"), (dict(n=-1), "-1 tokens"), (dict(tokens=0), "without their arrays"), (dict(lp=0), "without their arrays"), (dict(k=33, V=100, stride=100), "33 alternatives"),
    (dict(k=11), "11 alternatives of 10"), (dict(k=-1), "-1 alternatives"), (dict(ids=0), "alternatives without"), (dict(tlp=0), "alternatives without"), (dict(), "null context"),
    (dict(n=0, tokens=0, lp=0, k=0, ids=0, tlp=0), "null context")])
def test_token_logprobs(orn, change, text):
    _refused(orn, _score(orn, **change), text)


@pytest.mark.parametrize("args,text", [((0, 8, 64, 2, 256, 2, 4), "0 layers"), ((1, 8, 64, 2, 256, 0, 4), "0 sequences"), ((1, 8, 64, 2, 256, 2, 9), "9 pages"),
                                       ((1, 8, 60, 2, 256, 2, 4), "power of two"), ((1, 8, 64, 2, 100, 2, 4), "head width"), ((1, 8, 64, 2, 256, 2, 4), "null context")])
def test_pool_create(orn, args, text):
    h = C.c_void_p()
    _refused(orn, orn.lib().ornith_kv_pool_create(None, *args, C.byref(h)), text)
    assert not h.value


def test_positions_past_thirty_bits(orn):
    """Positions stay small enough for what is added to them."""
    for call in (_sdpa, _prep):
        _refused(orn, call(orn, _pages(orn), _batch(orn, stride=1 << 25, most=(1 << 30) + 1)), "at most 2^30")
    ids = np.zeros((1 << 22) + 1, np.uint32)
    for name in ("load", "store"):
        _refused(orn, getattr(orn.lib(), "ornith_kv_pages_" + name)(None, C.byref(_pages(orn, page_rows=256).s), 0, C.c_void_p(0x1000), C.c_void_p(0x1000), 100, 0, 10,
                                                                    ids.ctypes.data_as(C.c_void_p), ids.size, (1 << 30) - 9), "rows [1073741815, +10)")
    h = C.c_void_p()
    _refused(orn, orn.lib().ornith_kv_pool_create(None, 1, (1 << 22) + 1, 256, 1, 64, 1, (1 << 22) + 1, C.byref(h)), "4194305 pages of 256 rows")
