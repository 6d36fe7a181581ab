"""How exact attention over the paged cache is: small numerators beside a large one, and fp32 results as such.

Tolerances are derived where they stand; oracle/paged_ref.py is the definition in 64 bits."""
import math
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from test_gpu_paged import BF16, F16, F32, Case, paged  # noqa: E402,F401

from oracle import paged_ref as R  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("io,cache", [(F32, F16), (BF16, F16), (F16, F16), (F32, BF16), (F32, F32), (BF16, BF16)])
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("gap", [12.0, 20.0, 25.5, 28.0])
def test_one_position_outweighs_the_rest(paged, kq, io, cache, new, gap):  # noqa: F811
    """A first position whose score stands 2^gap above the others' and whose V is zero, as a first token's often
    is: the output is what the others' numerators leave, some 2^-gap of V each.

    Each numerator is off by a relative 2 ds + 8 u (ds: the score's error as in the oracle), the sums over n
    positions by n u each, so the output by that of sum p |v|; numerators rounded to 16 bits (a chunk of 16-bit
    activations over a cache of their type) add half an ulp, for fp16 2^-32 of the largest numerator at least."""
    n, dim, heads = 6000, 128, 4
    g = torch.Generator(device="cuda")
    g.manual_seed(40)
    c = paged.PagedKV.alloc(1, n // 16, 16, 1, dim, cache)
    s = c.pool.new()
    c.extend({s: n})
    table = torch.from_numpy(c.pool.pages(s)).cuda().long()
    k = torch.randn(n, dim, generator=g, device="cuda")
    k[:, 0] = -gap * math.log(2) / 16 + 0.02 * torch.randn(n, generator=g, device="cuda")
    k[0, 0] = gap * math.log(2) / 16
    v = 64.0 * (0.5 + torch.rand(n, dim, generator=g, device="cuda"))
    v[0] = 0
    pos = torch.arange(n, device="cuda")
    c.k[0, table[pos // 16], 0, pos % 16] = k.to(cache)
    c.v[0, table[pos // 16], 0, pos % 16] = v.to(cache)
    q = torch.zeros(new, heads, dim, dtype=io, device="cuda")
    q[:, :, 0] = 8.0
    got = c.attend(0, c.batch([s], [new]), q, scale=1.0)
    assert kq.tb_cuda_last_error() == 0
    ks, vs = (t[0, table[pos // 16], 0, pos % 16].double() for t in (c.k, c.v))
    for t in range(new):
        m = n - new + t + 1
        sc = ks[:m, 0] * 8.0
        p = torch.exp(sc - sc.max())
        total = p.sum()
        pv = (p[:, None] * vs[:m]).sum(0) / total   # V is not negative
        rel = 2 * 4 * (dim + 4) * R.U32 * float(sc.abs().max()) + (8 + 2 * m) * R.U32
        bound = rel * pv + R.U[io] * pv + torch.finfo(io).tiny * R.U[io]
        if new > 1 and io == cache and io != F32:
            least = 2.0 ** -32 if io == F16 else 0.0
            bound += ((R.U[io] * p + least)[:, None] * vs[:m]).sum(0) / total
        off = (got[t].double() - pv).abs() - bound
        assert float(off.max()) <= 0.0, (t, float(off.max()), float(pv.max()))


def exact(c, q, scale, window=0, sinks=0):
    """The definition in 64 bits, a kv head's rows of a sequence together."""
    T, H, D = q.shape
    nk, ps = c.k.shape[2], c.k.shape[3]
    out = torch.zeros(T, H, D, dtype=torch.float64, device="cuda")
    for s, n in enumerate(c.lens):
        lo, hi = c.start[s], c.start[s + 1]
        if lo == hi:
            continue
        j = torch.arange(n, device="cuda")
        pos = torch.arange(n - (hi - lo), n, device="cuda")[:, None]
        see = (j <= pos) & ((pos - j < window) | (j < sinks) if window else True)
        for h in range(nk):
            k, v = (t[1, c.table[s][j // ps], h, j % ps].double() for t in (c.k, c.v))
            x = q[lo:hi, h * (H // nk):(h + 1) * (H // nk)].double()
            p = torch.softmax(torch.einsum("thd,jd->thj", x, k).mul(scale).masked_fill(~see[:, None], -math.inf), -1)
            out[lo:hi, h * (H // nk):(h + 1) * (H // nk)] = p @ v
    return out


def rel2(a, b):
    return float((a.double() - b).norm() / b.norm())


KINDS = {"single": ([1] * 6, [1, 33, 300, 1025, 2000, 129]), "few": ([5, 3, 2], [333, 70, 1500]),
         "chunk": ([150, 70, 1], [400, 700, 90])}


@pytest.mark.parametrize("io,cache", [(a, b) for a in (F32, F16, BF16) for b in (F32, F16, BF16)])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 128), (12, 4, 64)])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 4)])
def test_relative_error(paged, kq, io, cache, heads, kv_heads, dim, kind, window, sinks):  # noqa: F811
    """The relative 2-norm of the error, which a worst-case bound cannot tell: operands in parts lose some 2^-21 of
    a product, with no preferred sign, so do the sums; eight such are allowed.  A kernel that lost its low
    parts would be off by 2^-12 and more.  What is rounded to 16 bits at the end is off by that rounding besides; in
    chunks of 16-bit activations over a cache of their type the numerators are, too, independently: root 2 of it,
    and a tenth for chance."""
    new, lens = KINDS[kind]
    c = Case(paged, new, lens, heads, kv_heads, dim, io, cache, 16, seed=42)
    got = c.cache.attend(1, c.batch, c.q, window=window, sinks=sinks)
    want = exact(c, c.q, 1 / math.sqrt(dim), window, sinks)
    off, once = rel2(got, want), rel2(want.to(io), want)
    chunk = kind == "chunk" and io == cache and io != F32
    assert off <= 8 * 2.0 ** -21 + (0.0 if io == F32 else (math.sqrt(2) if chunk else 1.0) * 1.1 * once), (off, once)


@pytest.mark.parametrize("io,cache", [(F32, F32), (F32, F16), (F32, BF16), (BF16, F16)])
@pytest.mark.parametrize("new", [1, 16])
def test_relative_error_of_long_contexts(paged, kq, io, cache, new):  # noqa: F811
    """The same at 20000 positions: one sequence (cut between many CTAs) and, for each of its kv heads, long sums."""
    c = Case(paged, [new], [20000], 4, 1, 128, io, cache, 128, seed=43)
    want = exact(c, c.q, 1 / math.sqrt(128))
    off, once = rel2(c.cache.attend(1, c.batch, c.q), want), rel2(want.to(io), want)
    assert off <= 8 * 2.0 ** -21 + (0.0 if io == F32 else 1.1 * once), (off, once)
