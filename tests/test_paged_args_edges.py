"""CPU: the ends of the ranges of what the calls over paged KV caches and the token scores take."""
import ctypes as C

import numpy as np
import pytest

from test_paged_args import _batch, _copy, _pages, _refused, _score, _sdpa


@pytest.mark.parametrize("ids", [[1 << 32], [-1], [1.0], [True], ["1"], np.array([(1 << 32) + 1]), np.array([-1]), np.array([1 << 32], np.uint64), np.array([2.5])])
def test_page_ids_of_other_types(orn, ids):
    """A number that is no 32-bit page id is refused; it is not wrapped or cut to one."""
    ctx = orn.Ctx.__new__(orn.Ctx)
    ctx.h = None
    for call in (lambda: ctx.kv_pages_copy(_pages(orn), ids, [3], 1), lambda: ctx.kv_pages_copy(_pages(orn), [3], ids, 1),
                 lambda: ctx.kv_pages_load(_pages(orn), 0, _pages(orn).keep[0][0], _pages(orn).keep[0][0], 64, 0, 1, ids, 0),
                 lambda: ctx.kv_pages_store(_pages(orn), 0, _pages(orn).keep[0][0], _pages(orn).keep[0][0], 64, 0, 1, ids, 0)):
        with pytest.raises((TypeError, OverflowError), match="page ids"): call()


@pytest.mark.parametrize("dtype", [np.int8, np.uint8, np.int32, np.uint32, np.int64, np.uint64])
def test_page_ids_of_whole_types(orn, dtype):
    n, ids = orn._ids(np.array([[0, 7], [100, 3]], dtype)[:, ::-1])
    assert n == 4 and list(ids) == [7, 0, 3, 100]
    assert list(orn._ids(range(3))[1]) == [0, 1, 2] and orn._ids([]) == (0, None) and orn._ids(np.zeros(0)) == (0, None)
    assert list(orn._ids([np.uint32(5), np.int64(2 ** 32 - 1)])[1]) == [5, 2 ** 32 - 1]


def test_more_tokens_a_row_than_can_be_counted(orn):
    """The finishing threads step through a row's tokens by 1024: the number of the next one stays below 2^31."""
    _refused(orn, _score(orn, n=(1 << 30) + 1), "1073741825 tokens a row (at most 2^30)")
    _refused(orn, _score(orn, n=2 ** 31 - 1), "2147483647 tokens a row")
    _refused(orn, _score(orn, n=1 << 30), "null context")


@pytest.mark.parametrize("scale", [3.4e38, 2.4e38])
def test_attention_scale_past_its_binary_logarithm(orn, scale):
    """Scores are counted in binary orders, scale log2(e) of them a unit: a scale whose product is infinite would make 0 infinity of a row's best score."""
    _refused(orn, _sdpa(orn, _pages(orn), _batch(orn), scale=scale), "scale")
    _refused(orn, _sdpa(orn, _pages(orn), _batch(orn), scale=2.3e38), "null context")


def test_as_many_pages_as_an_int_counts(orn):
    """The set of pages that a copy or a load looks through is sized in 64 bits: no exception leaves a call."""
    most = 2 ** 31 - 1
    pages = _pages(orn, n_pages=most)
    _refused(orn, _copy(orn, pages, [0, most - 1], [most - 2, 5]), "null context")
    _refused(orn, _copy(orn, pages, [0, most - 1], [7, most - 1]), "read and written")
    _refused(orn, _copy(orn, pages, [0], [most]), "of 2147483647")
    ids = np.array([most - 1, most - 1], np.uint32)
    _refused(orn, orn.lib().ornith_kv_pages_load(None, C.byref(pages.s), 0, C.c_void_p(0x1000), C.c_void_p(0x1000), 100, 0, 70, ids.ctypes.data_as(C.c_void_p), 2, 10), "twice")
