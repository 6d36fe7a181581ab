"""Which kernel a call of attention takes is no part of its result: hints of any value, any number of query heads
per kv head, and rows of sequences with pages outside the pool; append in every order of the pool."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from test_gpu_paged import BF16, F16, F32, Case, paged, ulp_half  # noqa: E402,F401

from oracle import paged_ref as R  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("io,cache", [(F32, F32), (BF16, BF16), (F16, F32), (F32, BF16)])
@pytest.mark.parametrize("max_new,max_len", [(0, 0), (1, 1), (1, 2 ** 31 - 1), (7, 50), (2 ** 31 - 1, 1), (2 ** 31 - 1, 2 ** 31 - 1)])
@pytest.mark.parametrize("new,lens", [([1] * 5, [300, 7, 64, 1025, 16]), ([200], [333]), ([60, 1, 0, 130, 1], [90, 500, 30, 130, 1])])
def test_hints_of_any_value(paged, kq, io, cache, max_new, max_len, new, lens):  # noqa: F811
    """max_new and max_len choose between kernels and change no result, understated or overstated."""
    c = Case(paged, new, lens, 8, 2, 64, io, cache, 16, seed=70)
    b = paged.Batch(c.batch.start, c.batch.lens, c.batch.pages, c.q.shape[0], max_new, max_len)
    c.check(c.cache.attend(1, b, c.q))
    c.check(c.cache.attend(1, b, c.q, window=50, sinks=3), 50, 3)
    assert kq.tb_cuda_last_error() == 0


@pytest.mark.parametrize("io,cache", [(F32, F32), (BF16, BF16), (F16, BF16)])
@pytest.mark.parametrize("heads,kv_heads", [(129, 1), (160, 1), (258, 2), (128, 1), (96, 1)])
def test_many_query_heads_per_kv_head(paged, kq, io, cache, heads, kv_heads):  # noqa: F811
    """A token's rows of one kv head fill a row tile, or do not fit one."""
    c = Case(paged, [1, 9, 3], [40, 33, 200], heads, kv_heads, 64, io, cache, 16, seed=71)
    c.check(c.cache.attend(1, c.batch, c.q))
    assert kq.tb_cuda_last_error() == 0


@pytest.mark.parametrize("io", [F32, BF16])
@pytest.mark.parametrize("entry", [-1, 2 ** 31 - 1])
def test_rows_of_a_bad_page(paged, kq, io, entry):  # noqa: F811
    """New tokens at positions 14 to 19 of a sequence whose second page is none: attention sees the first 16 only,
    append stores what has a page and gives zeros for the rest, and the word is set by both."""
    c = Case(paged, [2, 6, 1], [20, 20, 40], 4, 2, 64, io, io, 16, seed=72)
    table = c.batch.pages.clone()
    table[1, 1] = entry
    b = paged.Batch(c.batch.start, c.batch.lens, table, 9, 6, 40)
    out = c.cache.attend(1, b, c.q)
    torch.cuda.synchronize()
    assert kq.tb_cuda_last_error() == 2
    rows = list(range(2, 8))
    ref, bound = R.attend(c.q[rows], c.k[1], c.v[1], list(range(7)), [min(15 + i, 16) for i in range(6)], [c.table[1]] * 6, 1 / 8)
    assert bool(((out[rows].double() - ref).abs() <= bound).all())
    other = [0, 1, 8]
    ref, bound = R.attend(c.q, c.k[1], c.v[1], c.start, c.lens, c.table, 1 / 8)
    assert bool(((out[other].double() - ref[other]).abs() <= bound[other]).all())
    k0, v0 = c.k.clone(), c.v.clone()
    qo = c.cache.append(1, b, c.q, c.nk, c.nv)
    torch.cuda.synchronize()
    assert kq.tb_cuda_last_error() == 2
    assert torch.equal(qo[[0, 1, 2, 3, 8]], c.q[[0, 1, 2, 3, 8]]) and not bool(qo[4:8].any())
    for now, then, rows in ((c.k, k0, c.nk), (c.v, v0, c.nv)):
        for s, t, p in ((0, 0, 18), (0, 1, 19), (1, 2, 14), (1, 3, 15), (2, 8, 39)):
            then[1, c.table[s, p // 16], :, p % 16] = rows[t]
        assert torch.equal(now.nan_to_num(nan=5.0), then.nan_to_num(nan=5.0))


@pytest.mark.parametrize("order", ["lphsd", "lpshd", "plhsd", "gap"])
@pytest.mark.parametrize("io,cache", [(F32, BF16), (F16, F16)])
def test_append_in_every_order(paged, kq, order, io, cache):  # noqa: F811
    """The pool's memory order changes where a position lies and nothing else."""
    c = Case(paged, [3, 40, 1], [20, 55, 300], 6, 2, 64, io, cache, 48, seed=73, order=order)
    rope = paged.Rope.make(300, 32, interleaved=True)
    k0, v0 = c.k.clone(), c.v.clone()
    c.cache.append(1, c.batch, c.q, c.nk, c.nv, rope=rope)
    assert kq.tb_cuda_last_error() == 0
    for s, n in enumerate(c.lens):
        lo, hi = c.start[s], c.start[s + 1]
        pos = torch.arange(n - (hi - lo), n, device="cuda")
        pg = c.table[s][pos // 48]
        got, want = c.k[1][pg, :, pos % 48], R.turn(c.nk[lo:hi], rope.table, pos, True)
        rel = 4 * R.U32 * want.abs().amax(-1, keepdim=True) * 2
        assert bool(((got.double() - want).abs() <= rel * (1 + R.U[cache]) + ulp_half(want, cache)).all())
        assert torch.equal(c.v[1][pg, :, pos % 48], c.nv[lo:hi].float().to(cache))
        k0[1][pg, :, pos % 48], v0[1][pg, :, pos % 48] = c.k[1][pg, :, pos % 48], c.v[1][pg, :, pos % 48]
    for now, then in ((c.k, k0), (c.v, v0)):
        assert torch.equal(now.nan_to_num(nan=5.0), then.nan_to_num(nan=5.0))
