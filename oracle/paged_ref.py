"""The paged cache's operators by their definitions, in 64 bits, one sequence and head at a time.

Pages are looked up position by position, every sum runs over the visible positions only, and nothing
here shares code with the library.  Tensors are torch's, on any device.  `attend` also returns a bound
on what an evaluation in 32 bits may be off by, element by element.
"""
import math

import torch

U32 = 2.0 ** -24                                                   # half an ulp of 1 in each type
U = {torch.float32: U32, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def gather(cache, table, length, head):
    """Positions [0, length) of one head: cache [pages, heads, page size, dim], table: page numbers."""
    ps = cache.shape[2]
    pos = torch.arange(length, device=cache.device)
    return cache[table.long()[pos // ps], head, pos % ps].double()


def visible(pos, length, window, sinks, device):
    j = torch.arange(length, device=device)
    see = j <= pos
    if window:
        see = see & ((pos - j < window) | (j < sinks))
    return see


def attend(q, kc, vc, start, lens, pages, scale, window=0, sinks=0):
    """q [T, heads, dim]; kc, vc [pages, kv heads, page size, dim]; lists start, lens; pages: tables.

    Returns (out, bound), both float64 [T, heads, dim]; rows of no sequence are NaN in both.  The bound:
    a score is a sum of dim products, each product and partial sum off by at most one rounding (counted
    as four, since operands may be split into parts of fewer bits whose dropped products stay below
    2^-22): ds = 4 (dim + 4) u sum |q k| scale, relative errors of exp below 2 ds + 8 u, of the sums over
    n positions n u each; all of it times max |v|.  An output that is rounded to 16 bits adds half an ulp
    of its own; 16-bit probabilities (allowed for 16-bit activations) add half an ulp of theirs times
    sum p |v|, and the same again in the normaliser."""
    T, H, D = q.shape
    nk = kc.shape[1]
    out = torch.full((T, H, D), math.nan, dtype=torch.float64, device=q.device)
    bound = out.clone()
    u = U[q.dtype]
    for b, length in enumerate(lens):
        lo, hi = start[b], start[b + 1]
        for h in range(H):
            if lo == hi:
                continue
            k = gather(kc, pages[b], length, h // (H // nk))
            v = gather(vc, pages[b], length, h // (H // nk))
            for t in range(lo, hi):
                pos = length - (hi - t)
                see = visible(pos, length, window, sinks, q.device)
                x = q[t, h].double()
                ks, vs = k[see], v[see]
                s = (ks * x).sum(-1) * scale
                p = torch.exp(s - s.max())
                p = p / p.sum()
                o = (p[:, None] * vs).sum(0)
                out[t, h] = o
                ds = 4 * (D + 4) * U32 * float((ks * x).abs().sum(-1).max()) * abs(scale)
                rel = 2 * ds + (8 + 2 * len(p)) * U32
                pv = (p[:, None] * vs.abs()).sum(0)
                bound[t, h] = vs.abs().max() * rel + (u * o.abs() + 2 * u * pv if u > U32 else U32 * o.abs())
    return out, bound


def turn(x, table, pos, interleaved, norm=None, eps=0.0):
    """Per-head RMS norm, then rotation at positions pos [T]: x [T, heads, dim] -> float64."""
    x = x.double()
    if norm is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * norm.double()
    if table is None:
        return x
    half = table.shape[1]
    y = x.clone()
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        c, s = table[pos, i, 0].double()[:, None], table[pos, i, 1].double()[:, None]
        y[..., a] = x[..., a] * c - x[..., b] * s
        y[..., b] = x[..., a] * s + x[..., b] * c
    return y


def rope_table(n_pos, rot, base, scaling=None, factor=1.0, orig_len=0, beta_fast=32.0, beta_slow=1.0, attn_factor=0.0):
    """[n_pos][rot / 2][2] float64 by the formulas of tb_rope_scale."""
    i = torch.arange(rot // 2, dtype=torch.float64)
    if scaling == "ntk":
        base = base * factor ** (rot / (rot - 2))
    f = base ** (-2 * i / rot)
    if scaling == "linear":
        f = f / factor
    if scaling == "yarn":
        r = orig_len * f / (2 * math.pi)
        g = ((r - beta_slow) / (beta_fast - beta_slow)).clamp(0, 1)
        f = f * (g + (1 - g) / factor)
    m = attn_factor or (0.1 * math.log(factor) + 1.0 if scaling == "yarn" else 1.0)
    a = torch.arange(n_pos, dtype=torch.float64)[:, None] * f
    return torch.stack([a.cos() * m, a.sin() * m], -1)
