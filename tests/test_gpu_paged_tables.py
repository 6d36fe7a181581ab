"""What attention over the paged cache reads of a page table: entries that count, as far as the table goes."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from test_gpu_paged import BF16, F16, F32, Case, paged  # noqa: E402,F401

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
