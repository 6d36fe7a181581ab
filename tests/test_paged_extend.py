"""CPU: PagedKV.extend and tb_cuda_kv_pool_extend_all are all or nothing, and no copy that is due gets lost."""
import random

import numpy as np
import pytest

from trailblaze_b200._lib import lib
from trailblaze_b200.paged import PagedKV, PagePool


class Host(PagedKV):
    """The sequences' side of a PagedKV over host marks in the place of device pages."""

    def __init__(self, n_pages, page_size):
        self._pool = PagePool(n_pages, page_size)
        self.marks = np.full((n_pages, page_size), -1, np.int64)

    def copy_pages(self, src, dst):
        self.marks[np.asarray(dst, int)] = self.marks[np.asarray(src, int)]

    def write(self, seq, first, values):
        pages, size = self.pool.pages(seq), self.pool.page_size
        for i, v in enumerate(values, first):
            self.marks[pages[i // size], i % size] = v

    def read(self, seq):
        pages, size = self.pool.pages(seq), self.pool.page_size
        return [int(self.marks[pages[i // size], i % size]) for i in range(self.pool.length(seq))]

    def state(self, seqs):
        return [(self.pool.length(s), self.pool.pages(s).tolist()) for s in seqs], self.pool.free_pages


def test_a_refused_extension_changes_nothing():
    c = Host(3, 16)
    a = c.pool.new()
    c.extend({a: 20})
    c.write(a, 0, range(20))
    b = c.fork(a)
    before = c.state([a, b])
    with pytest.raises(RuntimeError):
        c.extend({b: 1, a: 40})
    assert c.state([a, b]) == before
    c.extend({b: 1})   # the copy is due now
    c.write(b, 20, [99])
    assert c.read(b) == list(range(20)) + [99] and c.read(a) == list(range(20))


@pytest.mark.parametrize("seed", range(8))
def test_extend_all_against_one_by_one(seed):
    """Random forests of forks: where every extension fits one after the other, the call does the same; where one
    does not, lengths, tables, holders and free pages are what they were."""
    rng = random.Random(seed)
    c, model, mark, refused = Host(rng.choice([9, 20]), 16), {}, 0, 0
    for _ in range(300):
        op = rng.random()
        if op < 0.15 or not model:
            model[c.pool.new()] = []
        elif op < 0.3:
            s = rng.choice(list(model))
            model[c.fork(s)] = list(model[s])
        elif op < 0.42:
            s = rng.choice(list(model))
            c.free(s)
            del model[s]
        else:
            new = {s: rng.randrange(0, 30) for s in rng.sample(list(model), rng.randint(1, len(model)))}
            before = c.state(model)
            try:
                c.extend(new)
            except RuntimeError:
                refused += 1
                assert c.state(model) == before
                # a page for each copy and each page that a length reaches: without that many it can be refused
                need = sum(-(-(len(model[s]) + n) // 16) - -(-len(model[s]) // 16) + 1 for s, n in new.items())
                assert need > c.pool.free_pages
            else:
                for s, n in new.items():
                    c.write(s, len(model[s]), range(mark, mark + n))
                    model[s] += range(mark, mark + n)
                    mark += n
        for s, want in model.items():
            assert c.read(s) == want
    assert refused > 0
    for s in model:
        c.free(s)
    assert c.pool.free_pages == c.pool.n_pages   # no holder was lost or counted twice


def test_extend_all_of_the_c_entry():
    L = lib()
    arr = lambda *x: np.asarray(x, np.int32)  # noqa: E731
    p = L.tb_cuda_kv_pool_create(4, 16)
    s, out = L.tb_cuda_kv_pool_new(p), np.full((2, 4), -7, np.int32)

    def call(seqs, n, count=None):
        seqs, n = arr(*seqs), arr(*n)
        return L.tb_cuda_kv_pool_extend_all(p, seqs.ctypes.data, n.ctypes.data, len(seqs) if count is None else count,
                                            out[0].ctypes.data, out[1].ctypes.data)
    assert call([s, 5], [1, 1]) == -1 and call([s], [1], -1) == -1 and call([s, s], [1, -1]) == -1
    assert L.tb_cuda_kv_pool_extend_all(None, None, None, 0, None, None) == -1
    assert L.tb_cuda_kv_pool_extend_all(p, None, None, 1, None, None) == -1
    assert L.tb_cuda_kv_pool_len(p, s) == 0 and L.tb_cuda_kv_pool_free_pages(p) == 4
    assert call([], []) == 0 and call([s, s], [10, 10]) == 0 and L.tb_cuda_kv_pool_len(p, s) == 20
    f, g = L.tb_cuda_kv_pool_fork(p, s), L.tb_cuda_kv_pool_fork(p, s)
    assert call([f, g], [1, 13]) == -1                      # two copies and a page: three, and two are free
    assert L.tb_cuda_kv_pool_free_pages(p) == 2 and L.tb_cuda_kv_pool_len(p, f) == 20
    assert call([f, s, g], [1, 1, 1]) == 2                  # the last holder of the shared page keeps it
    assert out[0, :2].tolist() == [1, 1] and out[1, :2].tolist() == [2, 3]
    L.tb_cuda_kv_pool_destroy(p)


def test_the_width_of_a_table_is_checked():
    import ctypes
    from trailblaze_b200._lib import KvBatch, KvCache, KvRows
    L = lib()
    c = KvCache(0x10000, 0x20000, 30, 2, 8, 16, 4, 128, 65536, 8192, 2048, 128)
    r = KvRows(0x40000, 4096, 128)

    def attend(*tail):
        b = KvBatch(0x1000, 0x2000, *tail)
        return L.tb_cuda_kv_attend_dev(ctypes.byref(c), 0, ctypes.byref(b), 30, 16, ctypes.byref(r), ctypes.byref(r), 0.1, 0, 0,
                                       0x50000, 1 << 30, None)
    assert attend(0x3000, 2, 0, 1, 16, 4) == 1 and attend(0x3000, 2, 0, 1, 16, 4, 3) == 1
    assert attend(0x3000, 2, 0, 1, 16, 0, 3) == 1 and attend(None, 2, 0, 1, 16, 0, 0) == 1
    assert attend(0x3000, 2, 0, 1, 16, 4, -1) == 0 and attend(None, 2, 0, 1, 16, 0, 3) == 0


def test_numbers_that_do_not_fit_are_refused():
    """ctypes and numpy drop the upper bits of a number that is too large for a C int."""
    c = Host(4, 16)
    s = c.pool.new()
    c.extend({s: 20})
    far = 2 ** 32
    for call in (lambda: c.pool.extend(s, far + 1), lambda: c.pool.extend(s + far, 1), lambda: c.extend({s: far + 1}),
                 lambda: c.extend({s + far: 1}), lambda: c.extend({s: np.int64(far + 1)}), lambda: c.pool.truncate(s, far + 5),
                 lambda: c.pool.free(s + far), lambda: c.pool.fork(s + far), lambda: c.pool.length(s + far),
                 lambda: c.pool.pages(s + far), lambda: PagePool(far + 4, 16), lambda: PagePool(4, far + 16),
                 lambda: PagedKV.copy_pages(c, [far], [1]), lambda: PagedKV.copy_pages(c, np.asarray([0]), np.asarray([far + 1])),
                 lambda: PagedKV.copy_pages(c, [0.5], [1])):
        with pytest.raises(ValueError):
            call()
    assert c.pool.length(s) == 20 and c.pool.free_pages == 2
