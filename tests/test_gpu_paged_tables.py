"""What attention over the paged cache reads of a page table: entries that count, as far as the table goes."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from test_gpu_paged import BF16, F16, F32, Case, paged  # noqa: E402,F401

from oracle import paged_ref as R  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("io,cache", [(BF16, BF16), (F32, F32), (F16, BF16)])
@pytest.mark.parametrize("page", [16, 48])
@pytest.mark.parametrize("window,sinks", [(1, 0), (50, 0), (100, 20), (333, 5), (64, 200)])
def test_pages_behind_the_window_are_not_looked_at(paged, kq, io, cache, page, window, sinks):  # noqa: F811
    """Pages between the first tokens and the window of a sequence's first new token may be gone: the call is what
    it is with them, bit for bit, without an error.  The last page behind the window is seen again by one more."""
    new, lens = [1, 150, 40, 3], [900, 1000, 777, 130]
    c = Case(paged, new, lens, 8, 2, 64, io, cache, page, seed=60)
    want = c.cache.attend(1, c.batch, c.q, window=window, sinks=sinks)
    c.check(want, window, sinks)
    table, gone = c.batch.pages.clone(), 0
    for s, (n, length) in enumerate(zip(new, lens)):
        low = max(0, length - n - window + 1)   # the first position in the window of the first new token
        for i in range(-(-sinks // page), low // page):
            table[s, i] = -1
            gone += 1
    assert gone > 10
    b = paged.Batch(c.batch.start, c.batch.lens, table, c.q.shape[0], max(new), max(lens))
    assert torch.equal(c.cache.attend(1, b, c.q, window=window, sinks=sinks), want)
    assert kq.tb_cuda_last_error() == 0
    low = max(0, 1000 - 150 - window + 1)
    if low % page and low // page >= -(-sinks // page):   # the page that the window begins in does count
        table[1, low // page] = -1
        c.cache.attend(1, b, c.q, window=window, sinks=sinks)
        torch.cuda.synchronize()
        assert kq.tb_cuda_last_error() == 2


@pytest.mark.parametrize("io,cache,new", [(BF16, BF16, 1), (BF16, BF16, 60), (F32, F32, 60)])
def test_a_table_is_as_wide_as_it_says(paged, kq, io, cache, new):  # noqa: F811
    """A table that is a slice of a wider one: a sequence with more positions than the slice has pages for is an
    error, whatever stands beside the slice; the others are right (not the same bits: the work is cut between
    CTAs by the sequences that there are)."""
    c = Case(paged, [new] * 3, [200, 160, 100], 8, 2, 64, io, cache, 16, seed=61)
    want = c.cache.attend(1, c.batch, c.q)
    wide = torch.zeros(3, 40, dtype=torch.int32, device="cuda")
    wide[:, 4:4 + c.batch.pages.shape[1]] = c.batch.pages
    b = paged.Batch(c.batch.start, c.batch.lens, wide[:, 4:4 + c.batch.pages.shape[1]], c.q.shape[0], new, 200)
    assert torch.equal(c.cache.attend(1, b, c.q), want)
    assert kq.tb_cuda_last_error() == 0
    b = paged.Batch(c.batch.start, c.batch.lens, wide[:, 4:14], c.q.shape[0], new, 200)   # 160 positions
    got = c.cache.attend(1, b, c.q)
    torch.cuda.synchronize()
    assert kq.tb_cuda_last_error() == 2
    assert not bool(got[:new].any())
    ref, bound = R.attend(c.q, c.k[1], c.v[1], c.start, c.lens, c.table, 1 / 8)
    assert bool(((got[new:].double() - ref[new:]).abs() <= bound[new:]).all())
    k0 = c.k.clone()
    c.cache.append(1, b, c.q, c.nk, c.nv)
    torch.cuda.synchronize()
    assert kq.tb_cuda_last_error() == 2
    own = [int(p) for p in c.table[0, :13]]
    assert torch.equal(c.k[:, own].nan_to_num(nan=5.0), k0[:, own].nan_to_num(nan=5.0))


def test_one_table_for_all_sequences(paged, kq):  # noqa: F811
    """Rows of a table may be one row: forks of one sequence that have nothing of their own yet."""
    c = Case(paged, [1] * 3, [300, 300, 300], 8, 2, 64, BF16, BF16, 16, seed=62)
    one = paged.Batch(c.batch.start, c.batch.lens, c.batch.pages[:1].expand(3, -1), 3, 1, 300)
    c.table = c.table[:1].expand(3, -1)
    c.check(c.cache.attend(1, one, c.q))
    assert kq.tb_cuda_last_error() == 0


def test_a_table_of_no_pages(paged, kq):  # noqa: F811
    c = Case(paged, [1] * 2, [20, 30], 4, 2, 64, F32, F32, 16, seed=63)
    none = paged.Batch(c.batch.start, c.batch.lens, c.batch.pages[:, :0], 2, 1, 30)
    assert not bool(c.cache.attend(1, none, c.q).any())
    assert kq.tb_cuda_last_error() == 2
