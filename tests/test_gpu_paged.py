"""The paged cache's operators on the GPU against their definitions in 64 bits (oracle/paged_ref.py).

Attention is held to the oracle's element-wise bound; append to half an ulp of the stored type plus the
roundings of its few fp32 operations; copies bit for bit.  Cache slots that no position uses hold NaN
throughout, page tables are shuffled, unused table entries are out of range."""
import itertools
import math

import numpy as np
import pytest
import torch

from oracle import paged_ref as R

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def paged(kq):
    from trailblaze_b200 import paged as P
    return P


def layout(shape, dtype, order):
    """A [layers, pages, heads, page size, dim] tensor of NaN whose memory order is `order`; "gap" leaves
    16 bytes and more between rows."""
    full = dict(zip("lphsd", shape))
    names = "lpshd" if order == "lpshd" else "plhsd" if order == "plhsd" else "lphsd"
    sizes = [full[n] for n in names]
    if order == "gap":
        sizes[-1] += 16
    t = torch.full(sizes, math.nan, dtype=dtype, device="cuda")[..., :shape[-1]]
    return t.permute(*[names.index(n) for n in "lphsd"])


class Case:
    def __init__(self, P, new, lens, heads, kv_heads, dim, io, cache, page, seed=0, order="lphsd", layers=2, pad=0):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
        need = [-(-n // page) for n in lens]
        total = sum(need) + 2
        perm = torch.randperm(total, generator=g, device="cuda").tolist()
        width = max(1, max(need, default=0)) + 1
        table, it = np.full((len(lens), width), 2 ** 31 - 1, np.int64), iter(perm)
        for s, n in enumerate(need):
            for i in range(n):
                table[s, i] = next(it)
        self.k, self.v = (layout((layers, total, kv_heads, page, dim), cache, order) for _ in range(2))
        for s, n in enumerate(lens):
            for p in range(n):
                for t in (self.k, self.v):
                    t[1, table[s, p // page], :, p % page] = rnd(kv_heads, dim).to(cache)
        self.start = np.cumsum([0] + list(new)).tolist()
        self.lens, T = list(lens), int(sum(new)) + pad
        self.table = torch.from_numpy(table).cuda()
        qkv = (2.0 * rnd(T, heads + 2 * kv_heads, dim)).to(io)   # the fused projection's rows: strided heads
        self.q, self.nk, self.nv = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
        self.cache = P.PagedKV(self.k, self.v)
        self.batch = P.Batch(torch.tensor(self.start, dtype=torch.int32, device="cuda"),
                             torch.tensor(lens, dtype=torch.int32, device="cuda"), self.table.to(torch.int32), T,
                             max(new, default=0), max(lens, default=0))

    def check(self, out, window=0, sinks=0, scale=None, q=None):
        scale = 1 / math.sqrt(self.q.shape[2]) if scale is None else scale
        ref, bound = R.attend(self.q if q is None else q, self.k[1], self.v[1], self.start, self.lens, self.table, scale,
                              window, sinks)
        rows = slice(0, self.start[-1])
        off = ((out[rows].double() - ref[rows]).abs() - bound[rows]).nan_to_num(nan=math.inf)
        assert float(off.max()) <= 0.0 if off.numel() else True, (float(off.max()), int(off.argmax()))


HEADS = [(8, 2, 128), (4, 4, 64), (7, 1, 128), (6, 2, 64), (40, 2, 64), (8, 1, 128)]
TYPES = [(a, b) for a in (F32, F16, BF16) for b in (F32, F16, BF16)]


@pytest.mark.parametrize("io,cache", TYPES)
@pytest.mark.parametrize("heads,kv_heads,dim", [HEADS[0], HEADS[3]])
def test_single_tokens(paged, kq, io, cache, heads, kv_heads, dim):
    """One new token a sequence: lengths from 1 over page, tile and split ends to a long one; an empty one."""
    lens = [1, 2, 15, 16, 17, 31, 32, 33, 127, 128, 129, 255, 300, 0, 1025]
    c = Case(paged, [1 if n else 0 for n in lens], lens, heads, kv_heads, dim, io, cache, 16, seed=1)
    c.check(c.cache.attend(1, c.batch, c.q))
    assert kq.tb_cuda_last_error() == 0


@pytest.mark.parametrize("io,cache", [(F32, F32), (F16, F16), (BF16, BF16), (F32, BF16), (BF16, F32)])
@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
@pytest.mark.parametrize("page", [16, 48, 128])
def test_chunks(paged, kq, io, cache, heads, kv_heads, dim, page):
    """Chunks of several lengths in one batch, empty ones among them, after contexts of several lengths."""
    new = [3, 0, 1, 40, 17, 2]
    lens = [3, 5, 70, 40, 190, 2]
    c = Case(paged, new, lens, heads, kv_heads, dim, io, cache, page, seed=2, pad=3)
    out = torch.full_like(c.q, 7.0)
    c.check(c.cache.attend(1, c.batch, c.q, out=out))
    assert bool((out[c.start[-1]:] == 7.0).all())   # rows of no sequence are left alone
    assert kq.tb_cuda_last_error() == 0


@pytest.mark.parametrize("io,cache,dim", [(BF16, BF16, 128), (F16, F16, 64), (F32, F32, 128)])
def test_long_chunk(paged, kq, io, cache, dim):
    """Enough rows for several row tiles, ends inside tiles on both axes."""
    c = Case(paged, [301, 1, 133], [333, 200, 700], 4, 2, dim, io, cache, 32, seed=3)
    c.check(c.cache.attend(1, c.batch, c.q))


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 0), (16, 4), (64, 5), (100, 16), (128, 200), (33, 0),
                                          (2 ** 31 - 1, 3)])
@pytest.mark.parametrize("io,cache", [(F32, F32), (BF16, BF16), (F32, F16)])
def test_windows(paged, kq, io, cache, window, sinks):
    new, lens = [1, 1, 70, 150, 1], [300, 5, 333, 150, 129]
    c = Case(paged, new, lens, 4, 2, 128, io, cache, 16, seed=4)
    c.check(c.cache.attend(1, c.batch, c.q, window=window, sinks=sinks), window, sinks)


@pytest.mark.parametrize("order", ["lphsd", "lpshd", "plhsd", "gap"])
@pytest.mark.parametrize("cache", [F32, BF16])
def test_layouts(paged, kq, order, cache):
    """Other memory orders of the pool, rows with gaps, heads apart; results equal the plain order's bit for bit."""
    outs = []
    for o in ("lphsd", order):
        c = Case(paged, [1, 20, 5], [50, 60, 5], 4, 2, 128, cache, cache, 32, seed=5, order=o)
        outs.append(c.cache.attend(1, c.batch, c.q))
        c.check(outs[-1])
    assert torch.equal(outs[0], outs[1])


@pytest.mark.parametrize("io", [F32, BF16])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_hidden_values_have_no_influence(paged, kq, io, bad):
    """NaN and infinities in positions that some rows of a tile see and others do not: rows that do not see
    them are what they are without them."""
    new, lens = [40, 1], [60, 90]
    c = Case(paged, new, lens, 4, 2, 128, io, io, 16, seed=6)
    want = c.cache.attend(1, c.batch, c.q, window=30, sinks=2)
    c.check(want, 30, 2)
    where = 45   # a position of the first chunk (20 .. 59): rows at 20 .. 44 do not see it, nor 75 and later
    page = int(c.table[0, where // 16])
    for t in (c.k, c.v):
        t[1, page, :, where % 16] = bad
    page = int(c.table[1, 50 // 16])   # hidden from the single token at 89 by its window
    for t in (c.k, c.v):
        t[1, page, :, 50 % 16] = bad
    got = c.cache.attend(1, c.batch, c.q, window=30, sinks=2)
    blind = list(range(0, where - 20)) + [40]
    assert torch.equal(got[blind].isnan(), want[blind].isnan()) and not bool(got[blind].isnan().any())
    ref, bound = R.attend(c.q, torch.where(c.k[1].isfinite(), c.k[1], 0), torch.where(c.v[1].isfinite(), c.v[1], 0),
                          c.start, c.lens, c.table, 1 / math.sqrt(128), 30, 2)
    assert bool(((got[blind].double() - ref[blind]).abs() <= bound[blind]).all())
    if math.isnan(bad):
        assert bool(got[where - 20:40].isnan().all())   # rows that see it


@pytest.mark.parametrize("io", [F32, F16, BF16])
@pytest.mark.parametrize("which", ["k", "v"])
def test_nan_in_k_or_v_alone(paged, kq, io, which):
    """A NaN that a row sees makes its output NaN, wherever in a tile it lies; rows before it stay finite."""
    for where in (0, 1, 37, 100, 255):
        c = Case(paged, [300, 1], [300, 270], 4, 2, 64, io, io, 16, seed=18)
        for s in range(2):
            page = int(c.table[s, where // 16])
            (c.k if which == "k" else c.v)[1, page, :, where % 16] = math.nan
        got = c.cache.attend(1, c.batch, c.q).isnan()
        assert bool(got[where:].all()) and not bool(got[:where].any()), where


@pytest.mark.parametrize("io,cache", TYPES)
def test_long_chunks_of_all_types(paged, kq, io, cache):
    """Several row tiles and splits for every pair of types, negative scales among them."""
    c = Case(paged, [150, 1, 37], [190, 100, 400], 6, 2, 64, io, cache, 48, seed=19)
    c.check(c.cache.attend(1, c.batch, c.q, window=90, sinks=3), 90, 3)
    c.check(c.cache.attend(1, c.batch, c.q, scale=-0.1), scale=-0.1)
    c = Case(paged, [200], [700], 4, 1, 128, io, cache, 16, seed=20)
    c.check(c.cache.attend(1, c.batch, c.q))
    assert kq.tb_cuda_last_error() == 0


def test_large_scores(paged, kq):
    """Scores up to some thousands: the running maximum keeps every exponent at or below zero."""
    c = Case(paged, [1, 33], [500, 100], 4, 2, 128, F32, F32, 16, seed=7)
    c.check(c.cache.attend(1, c.batch, c.q, scale=30.0), scale=30.0)
    c.check(c.cache.attend(1, c.batch, c.q, scale=-2.0), scale=-2.0)
    c.check(c.cache.attend(1, c.batch, c.q, scale=0.0), scale=0.0)


def test_wide_activations_on_narrow_cache(paged, kq):
    """fp32 queries far outside the 16-bit types' ranges, each row of its own size."""
    for cache in (F16, BF16):
        c = Case(paged, [1, 20], [200, 64], 4, 2, 128, F32, cache, 16, seed=8)
        size = torch.exp2(torch.randint(-60, 60, (c.q.shape[0], 4, 1), device="cuda").float())
        q = c.q * size
        for sc in (2.0 ** -40, 1.0 / 2 ** 60):
            got = c.cache.attend(1, c.batch, q, scale=sc)
            ref, bound = R.attend(q, c.k[1], c.v[1], c.start, c.lens, c.table, sc)
            assert bool(((got.double() - ref).abs() <= bound).all())


def test_repeatable_and_streams(paged, kq):
    """The same call gives the same bits, on another stream too, and calls on two streams do not disturb
    each other."""
    c = Case(paged, [1] * 5, [2000, 17, 900, 1, 333], 8, 2, 128, BF16, BF16, 16, seed=9)
    want = c.cache.attend(1, c.batch, c.q)
    torch.cuda.synchronize()
    outs, streams = [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(8):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(c.cache.attend(1, c.batch, c.q))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


@pytest.mark.parametrize("heads,kv_heads", [(12, 4), (25, 5), (28, 4), (5, 1), (33, 3)])
def test_repeatable_chunks_of_odd_groups(paged, kq, heads, kv_heads):
    """Groups of heads that do not divide a row tile leave rows unused; what lies there must not show."""
    c = Case(paged, [300, 33, 1, 70], [900, 33, 500, 1234], heads, kv_heads, 64, BF16, BF16, 16, seed=22)
    want = c.cache.attend(1, c.batch, c.q)
    c.check(want)
    other = Case(paged, [128], [512], 8, 1, 64, BF16, BF16, 16, seed=23)
    for i in range(12):
        other.cache.attend(1, other.batch, other.q * (10.0 ** (i - 6)))   # other leftovers in shared memory
        assert torch.equal(c.cache.attend(1, c.batch, c.q), want)


@pytest.mark.parametrize("cache", [F32, BF16])
@pytest.mark.parametrize("heads,kv_heads,dim", [(12, 4, 64), (25, 5, 128), (28, 4, 128)])
def test_repeatable_fp32_chunks(paged, kq, cache, heads, kv_heads, dim):
    c = Case(paged, [300, 33, 1, 70], [900, 33, 500, 1234], heads, kv_heads, dim, F32, cache, 16, seed=24)
    want = c.cache.attend(1, c.batch, c.q)
    c.check(want)
    other = Case(paged, [128], [512], 8, 1, 64, F32, cache, 16, seed=25)
    for i in range(12):
        other.cache.attend(1, other.batch, other.q * (10.0 ** (i - 6)))
        assert torch.equal(c.cache.attend(1, c.batch, c.q), want)


def test_bad_tables_are_errors_not_faults(paged, kq):
    """Ranges, lengths and pages that cannot be: the error word is set, the sequence's rows are zero (a page
    outside the pool only hides its positions), the other sequences are right."""
    P = paged
    base = dict(new=[2, 3, 1], lens=[20, 30, 40], heads=4, kv_heads=2, dim=64, io=F32, cache=F32, page=16, seed=10)
    assert kq.tb_cuda_last_error() == 0
    for what in ("len", "short", "page", "negative page", "range"):
        c = Case(P, **base)
        start, lens, table = list(c.start), list(c.lens), c.table.to(torch.int32).clone()
        if what == "len":
            lens[1] = 16 * table.shape[1] + 1
        elif what == "short":
            lens[1] = 2
        elif what == "page":
            table[1, 1] = c.k.shape[1]
        elif what == "negative page":
            table[1, 1] = -1
        else:
            start[2] = 1   # runs backwards; the last sequence then begins at row 1
        b = P.Batch(torch.tensor(start, dtype=torch.int32, device="cuda"),
                    torch.tensor(lens, dtype=torch.int32, device="cuda"), table, c.q.shape[0], 3, 40)
        out = c.cache.attend(1, b, c.q, out=torch.full_like(c.q, 7.0))
        torch.cuda.synchronize()
        assert kq.tb_cuda_last_error() == 2, what
        ref, bound = R.attend(c.q, c.k[1], c.v[1], c.start, c.lens, c.table, 1 / 8)
        good = [0, 1, 5] if what != "range" else [0]
        assert bool(((out[good].double() - ref[good]).abs() <= bound[good]).all()), what
        if what in ("len", "short"):
            assert bool((out[2:5] == 0).all())
        elif "page" in what:   # 16 positions are left
            ref, bound = R.attend(c.q[2:5], c.k[1], c.v[1], [0, 3], [16], c.table[1:2], 1 / 8)
            q = c.q[4:5]
            ref, bound = R.attend(q, c.k[1], c.v[1], [0, 1], [16], c.table[1:2], 1 / 8)
            assert bool(((out[4:5].double() - ref).abs() <= bound).all())
        # the same tables never make append write outside its pages
        k0, v0 = c.k.clone(), c.v.clone()
        qo = c.cache.append(1, b, c.q, c.nk, c.nv)
        torch.cuda.synchronize()
        assert kq.tb_cuda_last_error() == 2, what
        changed = ((c.k != k0) & ~(c.k.isnan() & k0.isnan())).any(-1).any(2)
        assert int(changed.sum()) <= 6
        if what in ("len", "short", "page", "negative page"):
            assert bool((qo[2:5] == 0).all()) or "page" in what


@pytest.mark.parametrize("io", [F32, BF16])
def test_bad_page_of_a_split_chunk(paged, kq, io):
    """A page outside the pool in a chunk whose positions are shared out over several CTAs: its positions are
    hidden from every row, whichever CTA joins the parts."""
    c = Case(paged, [256], [1500], 4, 1, 64, io, io, 16, seed=21)
    for bad in (3, 40, 70):   # seen by all rows
        table = c.table.to(torch.int32).clone()
        table[0, bad] = -5
        b = paged.Batch(torch.tensor(c.start, dtype=torch.int32, device="cuda"),
                        torch.tensor(c.lens, dtype=torch.int32, device="cuda"), table, 256, 256, 1500)
        out = c.cache.attend(1, b, c.q)
        torch.cuda.synchronize()
        assert kq.tb_cuda_last_error() == 2
        rows = [0, 1, 100, 255]   # without the page the other positions close up: same scores, 16 fewer
        keep = torch.cat([c.table[0, :bad], c.table[0, bad + 1:94]])
        ref, bound = R.attend(c.q[rows], c.k[1], c.v[1], [0, 1, 2, 3, 4], [1500 - 256 + r + 1 - 16 for r in rows],
                              [keep] * 4, 1 / 8)
        assert bool(((out[rows].double() - ref).abs() <= bound).all()), bad


@pytest.mark.parametrize("n", [0, 1])
def test_empty_batches(paged, kq, n):
    c = Case(paged, [0] * n, [7] * n, 4, 2, 64, BF16, BF16, 16, seed=11)
    out = c.cache.attend(1, c.batch, c.q)
    assert out.shape == (0, 4, 64)
    assert c.cache.append(1, c.batch, c.q, c.nk, c.nv).shape == (0, 4, 64)
    assert kq.tb_cuda_last_error() == 0


def test_many_sequences(paged, kq):
    """More sequences than a CTA has threads, most of them empty or single."""
    rng = np.random.default_rng(12)
    lens = [int(x) for x in rng.integers(0, 40, 700)]
    new = [min(n, int(x)) for n, x in zip(lens, rng.integers(0, 3, 700))]
    c = Case(paged, new, lens, 4, 2, 64, F32, F32, 16, seed=12)
    c.check(c.cache.attend(1, c.batch, c.q))
    assert kq.tb_cuda_last_error() == 0


# ---- append -------------------------------------------------------------------------------------

def ulp_half(x, dtype):
    """Half an ulp at x: relative to the next power of two at most, absolute among the subnormals."""
    return x.abs() * R.U[dtype] + torch.finfo(dtype).tiny * R.U[dtype]


@pytest.mark.parametrize("io,cache", TYPES)
@pytest.mark.parametrize("dim,rot,inter,norm", [(128, 128, True, True), (128, 64, False, False), (64, 64, False, True),
                                                (64, 18, False, False), (128, 34, True, False), (128, 0, False, True),
                                                (64, 0, False, False)])
def test_append(paged, kq, io, cache, dim, rot, inter, norm):
    new, lens = [1, 0, 5, 33, 2], [1, 4, 70, 33, 18]
    c = Case(paged, new, lens, 6, 2, dim, io, cache, 16, seed=13, pad=2, order="lpshd" if norm else "lphsd")
    rope = paged.Rope.make(max(lens), rot, base=1e4, interleaved=inter) if rot else None
    qn = 1 + 0.1 * torch.randn(dim, device="cuda") if norm else None
    kn = 1 + 0.1 * torch.randn(dim, device="cuda") if norm else None
    k0, v0 = c.k.clone(), c.v.clone()
    out = torch.full_like(c.q, 7.0)
    assert c.cache.append(1, c.batch, c.q, c.nk, c.nv, q_out=out, rope=rope, q_norm=qn, k_norm=kn, eps=1e-5) is out
    assert kq.tb_cuda_last_error() == 0
    assert bool((out[c.start[-1]:] == 7.0).all())
    for s, n in enumerate(lens):
        lo, hi = c.start[s], c.start[s + 1]
        pos = torch.arange(n - (hi - lo), n, device="cuda")
        table = rope.table if rope else None

        def close(got, x, w, dtype):
            ref = R.turn(x, table, pos, inter, w, 1e-5)
            # the norm: dim + 4 roundings of the sum and the factor; the rotation: 3 of at most |a| + |b|
            rel = ((dim + 8) if w is not None else 0) * R.U32 + (4 * R.U32 if rot else 0)
            size = ref.abs().amax(-1, keepdim=True) * 2
            tol = rel * size + ulp_half(ref, dtype) + R.U[dtype] * rel * size
            assert bool(((got.double() - ref).abs() <= tol).all())
            if not rot and w is None:
                assert torch.equal(got, x.to(dtype))

        close(out[lo:hi], c.q[lo:hi], qn, io)
        pg = c.table[s][pos // 16]
        close(c.k[1][pg, :, pos % 16], c.nk[lo:hi], kn, cache)
        assert torch.equal(c.v[1][pg, :, pos % 16], c.nv[lo:hi].float().to(cache))
        k0[1][pg, :, pos % 16] = c.k[1][pg, :, pos % 16]
        v0[1][pg, :, pos % 16] = c.v[1][pg, :, pos % 16]
    for now, then in ((c.k, k0), (c.v, v0)):   # nothing else was written
        assert torch.equal(now.nan_to_num(nan=5.0), then.nan_to_num(nan=5.0))


def test_append_in_place_and_past_the_table(paged, kq):
    c = Case(paged, [4, 3], [10, 30], 4, 2, 64, F32, F32, 16, seed=14)
    rope = paged.Rope.make(28, 64)
    q = c.q.contiguous()
    want = c.cache.append(1, c.batch, q, c.nk, c.nv, rope=rope)
    torch.cuda.synchronize()
    assert kq.tb_cuda_last_error() == 2   # positions 28 and 29 have no angles
    assert bool((want[5:7] == 0).all()) and bool((want[:5] != 0).any())
    c.cache.append(1, c.batch, q, c.nk, c.nv, q_out=q, rope=rope)
    assert kq.tb_cuda_last_error() == 2 and torch.equal(q, want)


@pytest.mark.parametrize("kw", [dict(), dict(scaling="linear", factor=8.0), dict(scaling="ntk", factor=4.0),
                                dict(scaling="yarn", factor=16.0, orig_len=4096),
                                dict(scaling="yarn", factor=4.0, orig_len=2048, beta_fast=16.0, beta_slow=2.0,
                                     attn_factor=1.5)])
def test_rope_table(paged, kq, kw):
    t = paged.Rope.make(70000, 96, base=1e6, **kw).table.cpu().double()
    ref = {"beta_fast": 32.0, "beta_slow": 1.0, **kw}
    want = R.rope_table(70000, 96, 1e6, **ref)
    # rounded once; the angle (up to 7e4) and pow in 64 bits are off by a few 2^-53 of themselves
    assert float((t - want).abs().max()) <= 1.5 * R.U32 + 7e4 * 16 * 2.0 ** -53


# ---- copies -------------------------------------------------------------------------------------

@pytest.mark.parametrize("order", ["lphsd", "lpshd", "plhsd", "gap"])
@pytest.mark.parametrize("dtype,heads,page,dim", [(F32, 3, 16, 64), (BF16, 2, 48, 128), (F16, 1, 16, 64)])
def test_copy_pages(paged, kq, order, dtype, heads, page, dim):
    shape = (3, 600, heads, page, dim)
    k, v = layout(shape, dtype, order), layout(shape, dtype, order)
    k.copy_(torch.randn(shape, device="cuda"))
    v.copy_(torch.randn(shape, device="cuda"))
    cache = paged.PagedKV(k, v)
    ids = np.random.default_rng(15).permutation(600).astype(np.int32)
    for src, dst in (([], []), ([ids[0]], [ids[1]]), ([ids[0]] * 3, ids[1:4]), (ids[:290], ids[300:590])):
        wk, wv = k.clone(), v.clone()
        for a, b in zip(src, dst):
            wk[:, int(b)] = k[:, int(a)]
            wv[:, int(b)] = v[:, int(a)]
        cache.copy_pages(src, dst)
        assert torch.equal(k, wk) and torch.equal(v, wv)
    many = np.full(599, ids[7], np.int32)   # one source for every other page: more pairs than one launch takes
    cache.copy_pages(many, np.asarray([i for i in ids if i != ids[7]], np.int32))
    assert bool((k == k[:, int(ids[7])][:, None]).all()) and bool((v == v[:, int(ids[7])][:, None]).all())


def test_copy_refusals(paged, kq):
    k = torch.zeros(1, 4, 1, 16, 64, device="cuda")
    cache = paged.PagedKV(k, torch.zeros_like(k))
    for src, dst in (([0], [4]), ([4], [0]), ([-1], [0]), ([0], [-1]), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([0], [0])):
        with pytest.raises(ValueError):
            cache.copy_pages(src, dst)
    with pytest.raises(ValueError):
        cache.copy_pages([0, 1], [2])


# ---- together -----------------------------------------------------------------------------------

def test_wrapper_refusals(paged, kq):
    c = Case(paged, [2], [20], 4, 2, 64, F32, F32, 16, seed=16)
    q = c.q
    for bad in (q[:1], q.double(), q[:, :3], q[:, :, :32], q.transpose(1, 2).contiguous().transpose(1, 2)):
        with pytest.raises(ValueError):
            c.cache.attend(1, c.batch, bad)
    with pytest.raises(ValueError):
        c.cache.attend(2, c.batch, q)
    with pytest.raises(ValueError):
        c.cache.attend(1, c.batch, q, window=-1)
    with pytest.raises(ValueError):
        c.cache.append(1, c.batch, q, c.nk.half(), c.nv)
    with pytest.raises(ValueError):
        c.cache.append(1, c.batch, q, c.nk, c.nv, q_norm=torch.ones(32, device="cuda"))
    with pytest.raises(ValueError):
        paged.PagedKV(torch.zeros(1, 2, 1, 24, 64, device="cuda"), torch.zeros(1, 2, 1, 24, 64, device="cuda"))
    with pytest.raises(ValueError):
        paged.Rope.make(8, 64, scaling="other")


def test_fork_append_attend_compact(paged, kq):
    """A prompt, two forks that go their own ways, an end and a compaction: every sequence attends as one that
    was built alone."""
    g = torch.Generator(device="cuda")
    g.manual_seed(17)
    cache = paged.PagedKV.alloc(2, 24, 16, 2, 64, torch.bfloat16)
    cache.k.fill_(math.nan)
    cache.v.fill_(math.nan)
    rope = paged.Rope.make(200, 64)
    hist = {}

    def feed(seqs, new):
        cache.extend(dict(zip(seqs, new)))
        b = cache.batch(seqs, new)
        T = b.n_tokens
        rows = [torch.randn(T, h, 64, generator=g, device="cuda").to(torch.bfloat16) for h in (4, 2, 2)]
        at = 0
        for s, n in zip(seqs, new):
            hist.setdefault(s, []).append((rows[1][at:at + n], rows[2][at:at + n]))
            at += n
        outs = []
        for layer in range(2):
            q = cache.append(layer, b, *rows, rope=rope)
            outs.append(cache.attend(layer, b, q))
        assert torch.equal(outs[0], outs[1])
        at = 0
        for s, n in zip(seqs, new):
            # what the pages hold for the sequence is its own history, rotated and rounded once
            kk, vv = (torch.cat([h[i] for h in hist[s]]) for i in (0, 1))
            L = kk.shape[0]
            pos = torch.arange(L, device="cuda")
            table = torch.from_numpy(cache.pool.pages(s)).cuda().long()
            got = [t[1][table[pos // 16], :, pos % 16] for t in (cache.k, cache.v)]
            want = R.turn(kk, rope.table, pos, False)
            size = want.abs().amax(-1, keepdim=True) * 2
            assert bool(((got[0].double() - want).abs() <= ulp_half(want, BF16) + 5 * R.U32 * size).all())
            assert torch.equal(got[1], vv)
            ref, bound = R.attend(q[at:at + n], cache.k[1], cache.v[1], [0, n], [L], [table], 1 / 8)
            assert bool(((outs[1][at:at + n].double() - ref).abs() <= bound).all())
            at += n

    a = cache.pool.new()
    feed([a], [37])
    b = cache.fork(a)
    c = cache.fork(a)
    hist[b], hist[c] = list(hist[a]), list(hist[a])
    feed([b, a, c], [1, 5, 20])
    feed([c, b], [1, 1])
    cache.free(a)
    del hist[a]
    cache.compact()
    used = set(cache.pool.pages(b)) | set(cache.pool.pages(c))
    assert used == set(range(len(used)))
    feed([b, c], [30, 1])
    assert kq.tb_cuda_last_error() == 0
