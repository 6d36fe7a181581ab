"""How exact attention over the paged cache is: small numerators beside a large one, and fp32 results as such.

Tolerances are derived where they stand; oracle/paged_ref.py is the definition in 64 bits."""
import math
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from test_gpu_paged import BF16, F16, F32, paged  # noqa: E402,F401

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
