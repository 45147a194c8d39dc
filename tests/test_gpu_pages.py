"""GPU: pages of a KV cache copied, loaded from and stored to contiguous caches, and the pool that keeps them, against the same moves
in numpy: every byte, those that nothing may touch among them."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _pool(orn, ctx, rng, layers, n, R, Hkv, hd):
    host = [[rng.integers(0, 65536, (n, Hkv, R, hd), dtype=np.uint16) for _ in range(layers)] for _ in range(2)]
    bufs = [[ctx.to_device(a) for a in h] for h in host]
    return host, bufs, orn.KvPages(bufs[0], bufs[1], n, R, Hkv, hd)


def _same(host, bufs):
    return all(np.array_equal(b.download(np.uint16, a.shape), a) for h, d in zip(host, bufs) for a, b in zip(h, d))


def _free(bufs):
    for b in [b for d in bufs for b in d]: b.free()


@pytest.mark.parametrize("layers,R,Hkv,hd", [(1, 16, 1, 64), (2, 64, 2, 256), (3, 32, 8, 128), (1, 256, 3, 64), (70, 16, 1, 64), (10, 128, 2, 128)])
def test_copy(orn, ctx, layers, R, Hkv, hd):
    rng = np.random.default_rng(R + Hkv)
    n = 12
    host, bufs, pages = _pool(orn, ctx, rng, layers, n, R, Hkv, hd)
    for rows in sorted({0, 1, R // 2 - 1, R - 1, R}):
        ids = rng.permutation(n)
        for src, dst in (([ids[0]], [ids[1]]), ([ids[0]] * 3 + [ids[1]], ids[2:6]), ([], []), (ids[:6], ids[6:])):
            ctx.kv_pages_copy(pages, np.array(src, np.uint32), np.array(dst, np.uint32), rows)
            for h in host:
                for a in h:
                    for s, d in zip(src, dst): a[d, :, :rows] = a[s, :, :rows]
            assert _same(host, bufs), (rows, src, dst)
    _free(bufs)


def test_copy_of_many_pages(orn, ctx):
    """More pairs than one launch's arguments hold."""
    rng = np.random.default_rng(2)
    host, bufs, pages = _pool(orn, ctx, rng, 2, 1100, 16, 1, 64)
    ids = rng.permutation(1100).astype(np.uint32)
    ctx.kv_pages_copy(pages, ids[:550], ids[550:], 16)
    for h in host:
        for a in h: a[ids[550:]] = a[ids[:550]]
    assert _same(host, bufs)
    _free(bufs)


@pytest.mark.parametrize("R,Hkv,hd,n_ids,row0,rows,at", [
    (16, 1, 64, 3, 0, 48, 0), (16, 2, 128, 4, 5, 1, 15), (16, 2, 128, 4, 5, 2, 15), (64, 2, 256, 3, 7, 100, 33), (64, 2, 256, 3, 0, 0, 10), (32, 8, 64, 600, 3, 18000, 1111),
    (256, 3, 128, 2, 11, 300, 200)])
def test_load_and_store(orn, ctx, R, Hkv, hd, n_ids, row0, rows, at):
    rng = np.random.default_rng(at + rows)
    n, cap = n_ids + 3, row0 + rows + 9
    host, bufs, pages = _pool(orn, ctx, rng, 2, n, R, Hkv, hd)
    cache = [rng.integers(0, 65536, (Hkv, cap, hd), dtype=np.uint16) for _ in range(2)]
    dev = [ctx.to_device(c) for c in cache]
    ids = rng.permutation(n)[:n_ids]
    ctx.kv_pages_load(pages, 1, dev[0], dev[1], cap, row0, rows, ids, at)
    for h, c in zip(host, cache):
        for j in range(rows): h[1][ids[(at + j) // R], :, (at + j) % R] = c[:, row0 + j]
    assert _same(host, bufs)
    back = [rng.integers(0, 65536, (Hkv, cap, hd), dtype=np.uint16) for _ in range(2)]
    dback = [ctx.to_device(b) for b in back]
    ctx.kv_pages_store(pages, 1, dback[0], dback[1], cap, row0, rows, ids, at)
    for b, c in zip(back, cache): b[:, row0:row0 + rows] = c[:, row0:row0 + rows]
    assert all(np.array_equal(d.download(np.uint16, b.shape), b) for d, b in zip(dback, back)) and _same(host, bufs)
    _free([dev, dback] + bufs)


    def __init__(self): self.rows = {}


def test_pool_against_a_model_of_it(orn, ctx):
    """Some hundred random calls: every sequence reads back the rows that were written to it or to what it was forked from, the pages
    in use are as few as sharing allows, and a call that fails changes nothing."""
    R, Hkv, hd, n_pages, max_seqs, max_pages, layers = 16, 2, 64, 60, 9, 8, 2
    pool = orn.KvPool(ctx, layers, n_pages, R, Hkv, hd, max_seqs, max_pages)
    rng = np.random.default_rng(4)
    held, serial = {}, 0
    cap = R * max_pages
    dev = [ctx.alloc(Hkv * cap * hd * 2) for _ in range(2)]

    def content(rows, which):
        a = np.zeros((Hkv, cap, hd), np.uint16)
        for j, s in enumerate(rows): a[:, j] = (np.arange(Hkv * hd).reshape(Hkv, hd) * 7 + s * 13 + which * 5) % 65521
        return a

    def check(seq):
        rows, ids = pool.seq(seq)
        assert rows == len(held[seq]) and len(ids) == -(-rows // R) and len(set(ids)) == len(ids)
        for layer in range(layers):
            for d in dev: d.zero()
            pool.store(seq, layer, dev[0], dev[1], cap, 0, rows, 0)
            for which in range(2): assert np.array_equal(dev[which].download(np.uint16, (Hkv, cap, hd)), content(held[seq], which + 2 * layer)), seq
        return ids

    def write(seq, at):
        new = held[seq][at:]
        for layer in range(layers):
            for which in range(2): dev[which].upload(content(new, which + 2 * layer))
            pool.load(seq, layer, dev[0], dev[1], cap, 0, len(new), at)

    failed = 0
    for step in range(260):
        what = rng.choice(["open", "fork", "extend", "extend", "extend", "truncate", "close", "compact", "batch"])
        seqs = sorted(held)
        if what == "open":
            if len(held) < max_seqs:
                s = pool.open()
                assert s == min(set(range(max_seqs)) - set(held))
                held[s] = []
            else:
                with pytest.raises(orn.OrnithError, match="in use"): pool.open()
        elif what == "fork" and seqs:
            s, n = int(rng.choice(seqs)), int(rng.integers(1, 4))
            if len(held) + n <= max_seqs:
                for c in pool.fork(s, n): held[c] = list(held[s])
            else:
                with pytest.raises(orn.OrnithError, match="are free"): pool.fork(s, n)
        elif what == "extend" and seqs:
            some, n = [int(s) for s in rng.permutation(seqs)[:rng.integers(1, len(seqs) + 1)]], int(rng.integers(1, 40))
            before = pool.stats()
            try:
                pool.extend(some, n)
            except orn.OrnithError as e:
                assert "needed" in str(e) or "at most" in str(e)
                assert pool.stats() == before
                failed += 1
            else:
                for s in some:
                    at = len(held[s])
                    held[s] = held[s] + list(range(serial, serial + n))
                    serial += n
                    write(s, at)
        elif what == "truncate" and seqs:
            s = int(rng.choice(seqs))
            held[s] = held[s][:int(rng.integers(0, len(held[s]) + 1))]
            pool.truncate(s, len(held[s]))
        elif what == "close" and len(seqs) > 4:
            s = int(rng.choice(seqs))
            pool.close_seq(s)
            del held[s]
        elif what == "compact":
            pool.compact()
            used = {int(i) for s in held for i in pool.seq(s)[1]}
            assert used == set(range(len(used)))
        elif what == "batch" and seqs:
            some = [int(s) for s in rng.permutation(seqs)[:rng.integers(1, len(seqs) + 1)]]
            b = pool.batch(some).s
            table = orn.DeviceBuffer.__new__(orn.DeviceBuffer)
            table.ctx, table.ptr, table.nbytes = ctx, C.c_void_p(b.d_table), len(some) * b.table_stride * 4
            lens = orn.DeviceBuffer.__new__(orn.DeviceBuffer)
            lens.ctx, lens.ptr, lens.nbytes = ctx, C.c_void_p(b.d_lens), len(some) * 4
            t, n = table.download(np.uint32, (len(some), b.table_stride)), lens.download(np.int32, (len(some),))
            for i, s in enumerate(some):
                ids = pool.seq(s)[1]
                assert n[i] == len(held[s]) and np.array_equal(t[i, :len(ids)], ids)
            common = 0
            while all(len(held[s]) >= (common + 1) * R for s in some) and len({t[i, common] for i in range(len(some))}) == 1: common += 1
            assert (b.B, b.shared_rows, b.max_rows) == (len(some), common * R, max(len(held[s]) for s in some))
        ids = [i for s in sorted(held) for i in check(s)]
        used, shared, n_open = pool.stats()
        assert used == len(set(ids)) and shared == sum(ids.count(i) > 1 for i in set(ids)) and n_open == len(held)
    assert failed > 3 and serial > 500
    for d in dev: d.free()
    pool.close()


def test_pool_refusals(orn, ctx):
    pool = orn.KvPool(ctx, 1, 8, 16, 1, 64, 4, 4)
    a = pool.open()
    pool.extend([a], 40)
    b, = pool.fork(a, 1)
    cache = ctx.alloc(64 * 64 * 2)
    for call, text in ((lambda: pool.extend([a, a], 1), "twice"), (lambda: pool.extend([3], 1), "no sequence 3"), (lambda: pool.extend([a], 25), "at most 4"),
                       (lambda: pool.extend([a], -1), "-1 rows"), (lambda: pool.truncate(a, 41), "41 rows of 40"), (lambda: pool.close_seq(-1), "no sequence -1"),
                       (lambda: pool.fork(a, 0), "0 forks"), (lambda: pool.batch([a, a]), "twice"), (lambda: pool.batch([]), "0 sequences"),
                       (lambda: pool.load(a, 0, cache, cache, 64, 0, 8, 0), "is shared"), (lambda: pool.store(a, 0, cache, cache, 64, 0, 41, 0), "of 40"),
                       (lambda: pool.load(a, 1, cache, cache, 64, 0, 0, 41), "of 40")):
        with pytest.raises(orn.OrnithError, match=text): call()
    assert pool.stats() == (3, 3, 2)
    pool.extend([a, b], 8)                               # the first copies the shared page, the last holder keeps it
    assert pool.stats() == (4, 2, 2)
    pool.close_seq(a)
    pool.close_seq(b)
    assert pool.stats() == (0, 0, 0)
    cache.free()
    pool.close()


def test_pool_takes_the_lowest_pages(orn, ctx):
    pool = orn.KvPool(ctx, 1, 40, 16, 1, 64, 6, 12)
    a, b = pool.open(), pool.open()
    pool.extend([a, b], 16 * 5)
    assert list(pool.seq(a)[1]) == list(range(5)) and list(pool.seq(b)[1]) == list(range(5, 10))
    pool.truncate(a, 16 * 2)                             # 2, 3, 4 are free
    with pytest.raises(orn.OrnithError, match="at most 12"): pool.extend([a, b], 16 * 10)
    pool.extend([b], 16 * 4)
    assert list(pool.seq(b)[1]) == [5, 6, 7, 8, 9, 2, 3, 4, 10]
    c, d = pool.fork(a, 2)
    pool.extend([c, d], 17)
    assert [list(pool.seq(s)[1]) for s in (c, d)] == [[0, 1, 11, 12], [0, 1, 13, 14]]
    e, f = pool.fork(c, 2)                               # 12 holds one row and has three holders
    with pytest.raises(orn.OrnithError, match="30 pages needed, 25 of 40 free"): pool.extend([c, e, f, d], 16 * 8 - 15)   # 7 each, 2 copies
    assert pool.stats() == (15, 4, 6)
    pool.extend([c, e, f], 1)                            # two of the three copy it
    assert [int(pool.seq(s)[1][3]) for s in (c, e, f)] == [15, 16, 12] and pool.stats() == (17, 3, 6)
    pool.close_seq(b)
    assert pool.compact() == 6 and pool.stats()[0] == 8
    pool.extend([a], 1)
    assert list(pool.seq(a)[1]) == [0, 1, 8]
    pool.close()


def test_pages_of_a_closed_pool(orn, ctx):
    pool = orn.KvPool(ctx, 1, 4, 16, 1, 64, 2, 4)
    pages = pool.pages
    pool.close()
    with pytest.raises(orn.OrnithError, match="0 layers"): ctx.kv_pages_copy(pages, [0], [1], 16)
    with pytest.raises(orn.OrnithError, match="no sequence 0"): pool.seq(0)
