"""NaN and infinities in the cache of long chunks: what the rows are that see them, that the others do not change,
and that such a call stays a call of the same order, with no error, however many rows it touches."""
import math
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from test_gpu_paged import BF16, F16, F32, Case, paged  # noqa: E402,F401

from oracle import paged_ref as R  # noqa: E402

pytestmark = pytest.mark.gpu


def device_us(call):
    a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    call()
    torch.cuda.synchronize()
    a.record()
    call()
    b.record()
    torch.cuda.synchronize()
    return 1e3 * a.elapsed_time(b)


@pytest.mark.parametrize("io,cache", [(BF16, BF16), (F16, F16), (F32, F32), (F32, BF16)])
@pytest.mark.parametrize("which,bad", [("k", math.nan), ("v", math.nan), ("v", math.inf)])
def test_a_long_prompt_with_a_value_that_is_not_finite(paged, kq, io, cache, which, bad):  # noqa: F811
    """Position 0 is seen by all rows of a prompt of 3000 tokens, position 2000 by a third.  Rows that see a NaN
    in K are NaN, rows that see one dimension of V are NaN or infinite there and right elsewhere; nothing that waits
    meanwhile gives up, and the call takes no more than 100 times its usual time (a row at a time and a position at
    a time it was some thousand)."""
    n, dim, heads, kv = 3000, 128, 8, 2
    g = torch.Generator(device="cuda")
    g.manual_seed(50)
    c = paged.PagedKV.alloc(1, -(-n // 32), 32, kv, dim, cache)
    s = c.pool.new()
    c.extend({s: n})
    c.k.copy_(torch.randn(c.k.shape, generator=g, device="cuda"))
    c.v.copy_(torch.randn(c.v.shape, generator=g, device="cuda"))
    q = torch.randn(n, heads, dim, generator=g, device="cuda").to(io)
    batch, table = c.batch([s], [n]), torch.from_numpy(c.pool.pages(s)).cuda().long()
    want = c.attend(0, batch, q)
    usual = device_us(lambda: c.attend(0, batch, q))
    for where in (0, 2000):
        t = getattr(c, which)
        row = t[0, table[where // 32], :, where % 32]
        kept = row.clone()
        row[:, 5] = bad
        got = c.attend(0, batch, q)
        took = device_us(lambda: c.attend(0, batch, q))
        row.copy_(kept)
        assert kq.tb_cuda_last_error() == 0
        assert torch.equal(got[:where], want[:where]) or bool((got[:where] - want[:where]).abs().max() <= 0.05)
        if which == "k":
            assert bool(got[where:].isnan().all())
        else:
            assert not bool(got[where:, :, 5].isfinite().any()) and bool(got[:, :, :5].isfinite().all())
            rows = [where, where + 1, 2500, n - 1]
            ref, bound = R.attend(q[rows], c.k[0], c.v[0], [0, 1, 2, 3, 4], [r + 1 for r in rows], [table] * 4,
                                  1 / math.sqrt(dim))
            ok = (got[rows].double() - ref).abs() <= bound
            assert bool(ok[..., :5].all()) and bool(ok[..., 6:].all())
        assert took <= 100 * usual, (where, took, usual)


@pytest.mark.parametrize("io", [F32, BF16])
def test_a_bad_page_is_its_items_alone(paged, kq, io):  # noqa: F811
    """Many short sequences on a CTA, one with a page outside the pool: the others' rows are bit for bit what they
    are without it."""
    new = [20] * 300
    lens = [20 + 7 * (i % 40) for i in range(300)]
    c = Case(paged, new, lens, 8, 2, 64, io, io, 16, seed=51)
    want = c.cache.attend(1, c.batch, c.q)
    assert kq.tb_cuda_last_error() == 0
    table = c.batch.pages.clone()
    for s in (39, 150, 299):
        table[s, 0] = -1
    b = paged.Batch(c.batch.start, c.batch.lens, table, c.q.shape[0], 20, max(lens))
    got = c.cache.attend(1, b, c.q)
    torch.cuda.synchronize()
    assert kq.tb_cuda_last_error() == 2
    good = [r for s in range(300) if s not in (39, 150, 299) for r in range(20 * s, 20 * s + 20)]
    assert torch.equal(got[good], want[good])
    s = 39   # without its first 16 positions
    rows, n = list(range(20 * s, 20 * s + 20)), lens[s]
    ref, bound = R.attend(c.q[rows], c.k[1], c.v[1], list(range(21)), [n - 20 + r + 1 - 16 for r in range(20)],
                          [c.table[s, 1:]] * 20, 1 / 8)
    assert bool(((got[rows].double() - ref).abs() <= bound).all())


@pytest.mark.parametrize("io,cache", [(F32, F32), (BF16, BF16), (F16, F16), (F16, BF16)])
@pytest.mark.parametrize("every", [1, 3, 40])
def test_many_items_with_hidden_values(paged, kq, io, cache, every):  # noqa: F811
    """A NaN in V that only a sequence's last token sees, in all of many short sequences on a CTA or in some: the
    other rows are right, the last ones NaN, and sequences without one are bit for bit what they were."""
    new = [20] * 300
    lens = [20 + 7 * (i % 40) for i in range(300)]
    c = Case(paged, new, lens, 8, 2, 64, io, cache, 16, seed=52)
    want = c.cache.attend(1, c.batch, c.q)
    hit = list(range(0, 300, every))
    for s in hit:
        c.v[1, c.table[s, (lens[s] - 1) // 16], :, (lens[s] - 1) % 16] = math.nan
    got = c.cache.attend(1, c.batch, c.q)
    assert kq.tb_cuda_last_error() == 0
    ends = torch.tensor([20 * s + 19 for s in hit], device="cuda")
    assert bool(got[ends].isnan().all())
    rest = torch.ones(6000, dtype=torch.bool, device="cuda")
    rest[ends] = False
    assert bool(got[rest].isfinite().all())
    clean = torch.tensor([s not in hit for s in range(300)], device="cuda").repeat_interleave(20)
    if every == 40:
        assert torch.equal(got[clean], want[clean])
    c.v.nan_to_num_(nan=0.0)
    rows = [r for s in (0, 1, 80, 299) for r in range(20 * s, 20 * s + 19)]
    at = [lens[r // 20] - 20 + r % 20 + 1 for r in rows]
    ref, bound = R.attend(c.q[rows], c.k[1], c.v[1], list(range(len(rows) + 1)), at, [c.table[r // 20] for r in rows], 1 / 8)
    assert bool(((got[rows].double() - ref).abs() <= bound).all())


@pytest.mark.parametrize("cache", [F32, F16, BF16])
@pytest.mark.parametrize("new,length", [(1, 40), (40, 64)])
def test_products_beyond_fp32(paged, kq, cache, new, length):  # noqa: F811
    """Queries so large that q . k leaves fp32 while scale * q . k does not: rows like any other."""
    c = Case(paged, [new], [length], 4, 2, 64, F32, cache, 16, seed=53)
    q, scale = c.q * 2.0 ** 125, 2.0 ** -125 / 8
    c.k.mul_(2.0)
    got = c.cache.attend(1, c.batch, q, scale=scale)
    ref, bound = R.attend(q, c.k[1], c.v[1], c.start, c.lens, c.table, scale)
    assert bool(((got.double() - ref).abs() <= bound).all())
