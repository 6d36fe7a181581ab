"""The paged cache's operators at the sizes that count: rotary append, attention, page copies.

A case says which operator it is (`op`) and its sizes.  `prepare` makes the tensors that a serving
program has in hand; `run` passes them once through the operator, in plain torch or, where `own` is
true, through trailblaze_b200.paged.  `exact` is the definition in 64 bits.

The operators:
  append   per-head RMS norm (optional) and rotary positions of a ragged batch's new q and k rows;
           k and v go into the pages of each sequence, q is returned
  attend   each new token's q over its sequence's cached positions j <= i (its own position i), with
           a window: only i - j < window, or j < sinks
  copy     pages dst[n] = pages src[n] of K and V in every layer (forked tails, compaction)
"""
import math
import random

import numpy as np
import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}


# ---- cases --------------------------------------------------------------------------------------

def _attend(name, seqs, new, length, heads, kv_heads, dim, io, cache, page, window=0, sinks=0, ragged=0):
    """ragged 0: every sequence has `new` new tokens and `length` positions; else these are the most,
    and the sequences' own are spread below them by a generator seeded with `ragged`."""
    return {"op": "attend", "name": name, "seqs": seqs, "new": new, "length": length, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "io": io, "cache": cache, "page": page, "window": window,
            "sinks": sinks, "ragged": ragged}


def _append(name, seqs, new, length, heads, kv_heads, dim, io, cache, page, rot, interleaved, norm, ragged=0):
    return {"op": "append", "name": name, "seqs": seqs, "new": new, "length": length, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "io": io, "cache": cache, "page": page, "rot": rot,
            "interleaved": interleaved, "norm": norm, "ragged": ragged}


def _copy(name, layers, pages, moves, kv_heads, dim, cache, page, fan):
    """moves page pairs in a pool of `pages`; fan destinations share one source."""
    return {"op": "copy", "name": name, "layers": layers, "pages": pages, "moves": moves, "kv_heads": kv_heads,
            "dim": dim, "cache": cache, "page": page, "fan": fan}


def listed():
    return [
        # one token of one sequence at the decode benchmark's context, everything fp32: latency
        _attend("decode 1 x 4096 f32", 1, 1, 4096, 32, 8, 128, "f32", "f32", 16),
        # a serving batch's decode step, contexts of very different lengths
        _attend("decode 64 ragged bf16", 64, 1, 16384, 32, 8, 128, "bf16", "bf16", 32, ragged=11),
        # the fp32 decode path's activations over a half-size cache, 8 query heads per kv head
        _attend("decode 16 x 2048 f32 on bf16", 16, 1, 2048, 32, 4, 128, "f32", "bf16", 64),
        # one chunk of a long prompt (512 tokens at a time) late in its context
        _attend("chunk 512 at 4096 bf16", 1, 512, 4096, 32, 8, 128, "bf16", "bf16", 64),
        # a long prompt in one go
        _attend("prompt 8192 bf16", 1, 8192, 8192, 32, 8, 128, "bf16", "bf16", 128),
        # a chunk deep in a long context, sliding window and first tokens kept
        _attend("window 4096+4 at 16384 bf16", 1, 2048, 16384, 32, 8, 128, "bf16", "bf16", 64, 4096, 4),
        # prompts and single tokens in one batch, empty sequences, one kv head per head, odd pages
        _attend("mixed 24 ragged f16", 24, 611, 1733, 16, 16, 64, "f16", "f16", 48, ragged=23),
        # the fp32 prefill chunk
        _attend("chunk 512 at 1024 f32", 1, 512, 1024, 32, 8, 128, "f32", "f32", 16),
        # one token's q, k and v with the per-head norms, pairs interleaved: latency
        _append("append 1 f32 norm", 1, 1, 4096, 32, 8, 128, "f32", "f32", 16, 128, True, True),
        # a prompt's rows, half of each head rotated, halves paired
        _append("append 8192 bf16", 1, 8192, 8192, 32, 8, 128, "bf16", "bf16", 64, 64, False, False),
        # three forks of one sequence: its last page copied for each, in all 36 layers
        _copy("fork 3 x 36 layers bf16", 36, 64, 3, 8, 128, "bf16", 32, 3),
        # compaction of a cache after its sequences ended
        _copy("compact 384 x 36 layers bf16", 36, 1024, 384, 8, 128, "bf16", 32, 1),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


_HEADS = [(32, 8, 128), (32, 4, 128), (16, 16, 64), (8, 1, 128), (12, 4, 64), (28, 4, 128), (8, 8, 128), (25, 5, 64)]
_PAIRS = [("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"), ("bf16", "bf16"), ("f16", "f16")]
_PAGES = [16, 32, 48, 64, 128]


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "append", "copy"])
    if op == "copy":
        page, fan = rng.choice(_PAGES), rng.choice([1, 1, 2, 4])
        kv_heads, dim, cache = rng.choice([1, 4, 8]), rng.choice([64, 128]), rng.choice(["f32", "f16", "bf16"])
        layers = _log(rng, 1, 48)
        one = page * kv_heads * dim * _BYTES[cache] * layers
        moves = _log(rng, 1, max(1, min(384, 100663296 // one * 2)))
        c = _copy("", layers, moves * 2 + rng.randrange(1, 64), moves, kv_heads, dim, cache, page, fan)
    else:
        heads, kv_heads, dim = rng.choice(_HEADS)
        io, cache = rng.choice(_PAIRS)
        page = rng.choice(_PAGES)
        if op == "append":
            length = _log(rng, 1, 8192)
            new = length if rng.random() < 0.5 else 1
            seqs = _log(rng, 1, max(1, min(64, 8192 // new)))
            c = _append("", seqs, new, length, heads, kv_heads, dim, io, cache, page,
                        rng.choice([dim, dim, dim // 2, dim // 4 + 2]), rng.random() < 0.5, rng.random() < 0.5,
                        rng.randrange(0, 1 << 20))
        else:
            kind = rng.choice(["decode", "chunk", "prompt"])
            if kind == "decode":
                seqs, new, length = _log(rng, 1, 64), rng.choice([1, 1, 1, 2, 4]), _log(rng, 4, 16384)
            elif kind == "chunk":
                seqs, new = _log(rng, 1, 8), _log(rng, 2, 1024)
                length = _log(rng, new, 16384)
            else:
                seqs, new = _log(rng, 1, 8), _log(rng, 2, 4096)
                length = new
            # the scores' size, so that every case stays below the largest listed one
            seqs = max(1, min(seqs, 500_000_000 // (heads * new * length)))
            most = 400_000_000 if io == "f32" else 2_000_000_000
            length = max(new, min(length, most // (heads * new * seqs)))
            window, sinks = rng.choice([(0, 0), (0, 0), (_log(rng, 1, 4096), 0), (_log(rng, 16, 4096), rng.choice([1, 4, 16]))])
            c = _attend("", seqs, new, length, heads, kv_heads, dim, io, cache, page, window, sinks,
                        rng.randrange(0, 1 << 20) if seqs > 1 else 0)
    del c["name"]
    return c


def _lengths(case):
    """(new tokens, positions after them) of each sequence."""
    s, new, length = case["seqs"], case["new"], case["length"]
    if not case["ragged"]:
        return [new] * s, [length] * s
    r = random.Random(case["ragged"])
    news, lens = [], []
    for i in range(s):
        n = new if i == 0 or new == 1 else r.choice([0, 1, 1, _log(r, 1, new), _log(r, 1, new)])
        lens.append(length if i == 0 else r.randint(n, length) if n else r.randint(0, length))
        news.append(min(n, lens[-1]))
    return news, lens


# ---- inputs -------------------------------------------------------------------------------------

def _pages_of(case, lens, g):
    """(pages in the pool, the sequences' page table): pages are handed out in random order; unused
    entries are -1."""
    ps = case["page"]
    need = [-(-n // ps) for n in lens]
    total = sum(need) + 3
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    width = max(1, max(need))
    at = np.full((len(lens), width), -1, dtype=np.int64)
    done = 0
    for i, n in enumerate(need):
        at[i, :n] = np.arange(done, done + n)
        done += n
    at = torch.from_numpy(at).cuda()
    return total, torch.where(at >= 0, order[at.clamp(min=0)], -1).to(torch.int32).contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {"case": case}
    if case["op"] == "copy":
        shape = (case["layers"], case["pages"], case["kv_heads"], case["page"], case["dim"])
        s["k"] = torch.empty(shape, dtype=_TYPES[case["cache"]], device="cuda").normal_(generator=g)
        s["v"] = torch.empty(shape, dtype=_TYPES[case["cache"]], device="cuda").normal_(generator=g)
        ids = torch.randperm(case["pages"], generator=g, device="cuda").cpu().numpy().astype(np.int32)
        m = case["moves"]
        s["src"] = np.ascontiguousarray(np.repeat(ids[m:m + -(-m // case["fan"])], case["fan"])[:m])
        s["dst"] = np.ascontiguousarray(ids[:m])
        if own:
            from trailblaze_b200 import paged
            s["cache"] = paged.PagedKV(s["k"], s["v"])
        return s
    news, lens = _lengths(case)
    t, nh, nk, d = sum(news), case["heads"], case["kv_heads"], case["dim"]
    total, s["pages"] = _pages_of(case, lens, g)
    shape = (1, total, nk, case["page"], d)
    s["k"] = torch.empty(shape, dtype=_TYPES[case["cache"]], device="cuda").normal_(generator=g)
    s["v"] = torch.empty(shape, dtype=_TYPES[case["cache"]], device="cuda").normal_(generator=g)
    s["start"] = torch.tensor(np.cumsum([0] + news), dtype=torch.int32, device="cuda")
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s["max_new"], s["max_len"] = max(news), max(lens)
    # the rows of the fused projection: q, k and v of a token side by side
    qkv = torch.empty(t, nh + 2 * nk, d, dtype=torch.float32, device="cuda").normal_(generator=g)
    if case["op"] == "attend":   # normed heads: scores with a standard deviation of about 2
        qkv.mul_(2.0)
    qkv = qkv.to(_TYPES[case["io"]])
    s["q"], s["new_k"], s["new_v"] = qkv[:, :nh], qkv[:, nh:nh + nk], qkv[:, nh + nk:]
    if case["op"] == "append":
        half = case["rot"] // 2
        angle = torch.outer(torch.arange(s["max_len"], dtype=torch.float64, device="cuda"),
                            1e6 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half))
        s["rope"] = torch.stack([angle.cos(), angle.sin()], dim=-1).float()   # [position][pair][cos, sin]
        s["q_norm"] = s["k_norm"] = None
        if case["norm"]:
            s["q_norm"] = 1.0 + 0.1 * torch.randn(d, generator=g, device="cuda")
            s["k_norm"] = 1.0 + 0.1 * torch.randn(d, generator=g, device="cuda")
    if own:
        from trailblaze_b200 import paged
        s["cache"] = paged.PagedKV(s["k"], s["v"])
        s["batch"] = paged.Batch(s["start"], s["lens"], s["pages"], t, s["max_new"], s["max_len"])
        if case["op"] == "append":
            s["table"] = paged.Rope(s["rope"], interleaved=case["interleaved"])
    return s


# ---- one pass -----------------------------------------------------------------------------------

def run(s):
    c = s["case"]
    if own:
        if c["op"] == "copy":
            s["cache"].copy_pages(s["src"], s["dst"])
            return {"k": s["k"], "v": s["v"]}
        if c["op"] == "append":
            q = s["cache"].append(0, s["batch"], s["q"], s["new_k"], s["new_v"], rope=s["table"],
                                  q_norm=s["q_norm"], k_norm=s["k_norm"], eps=1e-6)
            return {"q": q, "k": s["k"], "v": s["v"]}
        return s["cache"].attend(0, s["batch"], s["q"], window=c["window"], sinks=c["sinks"])
    return {"copy": _plain_copy, "append": _plain_append, "attend": _plain_attend}[c["op"]](s, c)


def _plain_copy(s, c):
    src = torch.from_numpy(s["src"]).to("cuda", torch.int64, non_blocking=True)
    dst = torch.from_numpy(s["dst"]).to("cuda", torch.int64, non_blocking=True)
    s["k"][:, dst] = s["k"][:, src]
    s["v"][:, dst] = s["v"][:, src]
    return {"k": s["k"], "v": s["v"]}


def _rows(s):
    """(sequence, position) of every new token."""
    t = s["q"].shape[0]
    row = torch.arange(t, device="cuda")
    seq = torch.searchsorted(s["start"][1:].contiguous(), row.to(torch.int32), right=True)
    return seq, s["lens"][seq].long() - s["start"][seq + 1].long() + row


def _plain_append(s, c):
    seq, pos = _rows(s)
    cos, sin = s["rope"][pos].unsqueeze(1).unbind(-1)   # [token][1][pair]

    def turn(x, norm):
        x = x.float()
        if norm is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * norm
        r, rest = x[..., :c["rot"]], x[..., c["rot"]:]
        a, b = (r[..., 0::2], r[..., 1::2]) if c["interleaved"] else r.chunk(2, dim=-1)
        a, b = a * cos - b * sin, a * sin + b * cos
        r = torch.stack([a, b], dim=-1).flatten(-2) if c["interleaved"] else torch.cat([a, b], dim=-1)
        return torch.cat([r, rest], dim=-1)

    q = turn(s["q"], s["q_norm"]).to(s["q"].dtype)
    page = s["pages"][seq, pos // c["page"]].long()
    s["k"][0, page, :, pos % c["page"]] = turn(s["new_k"], s["k_norm"]).to(s["k"].dtype)
    s["v"][0, page, :, pos % c["page"]] = s["new_v"].float().to(s["v"].dtype)
    return {"q": q, "k": s["k"], "v": s["v"]}


def _plain_attend(s, c):
    n, m = s["max_new"], s["max_len"]
    nh, nk, d = c["heads"], c["kv_heads"], c["dim"]
    S = s["lens"].shape[0]
    # the batch padded to its longest sequence and chunk: K and V [S][kv head][position][dim]
    at = s["pages"][:, :max(1, -(-m // c["page"]))].clamp(min=0).long()
    k = s["k"][0][at].transpose(1, 2).reshape(S, nk, -1, d)[:, :, :m].float()
    v = s["v"][0][at].transpose(1, 2).reshape(S, nk, -1, d)[:, :, :m].float()
    seq, pos = _rows(s)
    row = pos - (s["lens"][seq].long() - (s["start"][seq + 1] - s["start"][seq]).long())
    q = torch.zeros(S, n, nh, d, device="cuda")
    q[seq, row] = s["q"].float()
    q = q.view(S, n, nk, nh // nk, d).permute(0, 2, 3, 1, 4).reshape(S, nk, -1, d)   # rows: head, then token
    w = (q @ k.transpose(-1, -2)).mul_(1.0 / math.sqrt(d))
    i = (s["lens"].long() - (s["start"][1:] - s["start"][:-1]).long()).view(S, 1, 1) + torch.arange(n, device="cuda").view(1, n, 1)
    j = torch.arange(m, device="cuda").view(1, 1, m)
    seen = j <= i
    if c["window"]:
        seen = seen & ((i - j < c["window"]) | (j < c["sinks"]))
    w = w.view(S, nk, nh // nk, n, m).masked_fill_(~seen.view(S, 1, 1, n, m), -1e30)
    w = w.sub_(w.amax(-1, keepdim=True)).exp_()
    w = w.div_(w.sum(-1, keepdim=True)).view(S, nk, -1, m)
    o = (w @ v).view(S, nh, n, d).transpose(1, 2)
    return o[seq, row].to(s["q"].dtype)


# ---- what cannot be done without ----------------------------------------------------------------

def _visible(n, length, window, sinks):
    """(query-key pairs, keys that any query sees) of one sequence's n new tokens."""
    if n == 0:
        return 0, 0
    i = np.arange(length - n, length, dtype=np.int64)
    if not window:
        return int((i + 1).sum()), length
    near = np.minimum(i + 1, window)
    first = np.minimum(np.maximum(i + 1 - window, 0), sinks)
    lo = max(0, length - n - window + 1)
    return int((near + first).sum()), length - lo + min(lo, sinks)


def work(case):
    c = case
    if c["op"] == "copy":
        one = c["layers"] * c["page"] * c["kv_heads"] * c["dim"] * _BYTES[c["cache"]] * 2
        return {"bytes": one * (-(-c["moves"] // c["fan"]) + c["moves"]), "flops": 0}
    news, lens = _lengths(c)
    t, io, cb = sum(news), _BYTES[c["io"]], _BYTES[c["cache"]]
    row_q, row_kv = c["heads"] * c["dim"], 2 * c["kv_heads"] * c["dim"]
    if c["op"] == "append":
        table = t * c["rot"] * 4
        flops = t * (c["heads"] + c["kv_heads"]) * (3 * c["rot"] + (4 * c["dim"] if c["norm"] else 0))
        return {"bytes": t * (2 * row_q * io + row_kv * (io + cb)) + table, "flops": flops}
    seen = [_visible(n, m, c["window"], c["sinks"]) for n, m in zip(news, lens)]
    return {"bytes": 2 * t * row_q * io + sum(keys for _, keys in seen) * row_kv * cb,
            "flops": 4 * sum(pairs for pairs, _ in seen) * row_q}


# ---- the definition in 64 bits ------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "copy":
        out = {}
        for name in ("k", "v"):
            t = s[name].clone()
            for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
                t[:, b].copy_(s[name][:, a])
            out[name] = t
        return out
    c, ps = case, case["page"]
    start, lens = s["start"].tolist(), s["lens"].tolist()
    if c["op"] == "append":
        half = c["rot"] // 2
        first = list(range(0, c["rot"], 2)) if c["interleaved"] else list(range(half))
        second = list(range(1, c["rot"], 2)) if c["interleaved"] else list(range(half, c["rot"]))
        q = s["q"].double()
        k, v = s["k"].double(), s["v"].double()
        for b, length in enumerate(lens):
            lo, hi = start[b], start[b + 1]
            if lo == hi:
                continue
            pos = torch.arange(length - (hi - lo), length, device="cuda")
            cs = s["rope"][pos].double()
            new = []
            for x, norm in ((s["q"][lo:hi].double(), s["q_norm"]), (s["new_k"][lo:hi].double(), s["k_norm"])):
                if norm is not None:
                    x = x / (x.pow(2).sum(-1, keepdim=True) / c["dim"] + 1e-6).sqrt() * norm.double()
                y = x.clone()
                y[..., first] = x[..., first] * cs[:, None, :, 0] - x[..., second] * cs[:, None, :, 1]
                y[..., second] = x[..., second] * cs[:, None, :, 0] + x[..., first] * cs[:, None, :, 1]
                new.append(y)
            q[lo:hi] = new[0]
            where = s["pages"][b].long()[pos // ps]
            k[0].permute(0, 2, 1, 3)[where, pos % ps] = new[1]
            v[0].permute(0, 2, 1, 3)[where, pos % ps] = s["new_v"][lo:hi].double()
        return {"q": q, "k": k, "v": v}
    group = c["heads"] // c["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, length in enumerate(lens):
        lo, hi = start[b], start[b + 1]
        if lo == hi:
            continue
        where = s["pages"][b, :-(-length // ps)].long()
        for h in range(c["kv_heads"]):
            k = s["k"][0, where, h].reshape(-1, c["dim"])[:length].double()
            v = s["v"][0, where, h].reshape(-1, c["dim"])[:length].double()
            for r in range(lo, hi, 1024):
                e = min(hi, r + 1024)
                q = s["q"][r:e, h * group:(h + 1) * group].double()
                w = torch.einsum("tgd,jd->tgj", q, k) / math.sqrt(c["dim"])
                i = torch.arange(length - (hi - r), length - (hi - e), device="cuda")[:, None]
                j = torch.arange(length, device="cuda")[None, :]
                hide = j > i
                if c["window"]:
                    hide |= (j <= i - c["window"]) & (j >= c["sinks"])
                w = torch.softmax(w.masked_fill(hide[:, None], -math.inf), dim=-1)
                out[r:e, h * group:(h + 1) * group] = torch.einsum("tgj,jd->tgd", w, v)
    return out
