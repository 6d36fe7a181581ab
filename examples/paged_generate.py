"""Several continuations of one prompt over the paged cache, with a small random-init model.

    python examples/paged_generate.py [--samples 4] [--prompt 40] [--new 24] [--cache bf16] [--window 0 --sinks 0]

The prompt runs once as a chunk; each sample is a fork of it that shares the prompt's pages (its
part-filled last page is copied when the fork first grows), all samples step together as one ragged
batch, each ends by itself, and its pages return to the pool, which is compacted at the end.  The
projections are the library's quantized matvecs (norms, SwiGLU and residuals fused), positions are
rotary with by-parts scaling, tokens are drawn by the library's top-k sampler.
"""
from __future__ import annotations

import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from trailblaze_b200 import load, qtypes as Q  # noqa: E402
from trailblaze_b200.decoder import ModelShape, device_weights  # noqa: E402
from trailblaze_b200.paged import PagedKV, Rope  # noqa: E402

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


class PagedModel:
    """A dense model's layers over a PagedKV: weights as trailblaze_b200.decoder.Decoder takes them."""

    def __init__(self, shape: ModelShape, cache: PagedKV, rope: Rope, window: int = 0, sinks: int = 0):
        self.kq = load()
        self.s, self.cache, self.rope, self.window, self.sinks = shape, cache, rope, window, sinks
        self.layers, self.head = [], None

    def set_layer(self, wqkv, wo, wgu, wd, attn_norm, ffn_norm, q_norm, k_norm):
        self.layers.append((wqkv, wo, wgu, wd, attn_norm, ffn_norm, q_norm, k_norm))

    def set_head(self, emb, out_norm, w_out):
        self.head = (emb, out_norm, w_out)

    def _rows(self, w, qt, m, x, y, norm=None, res=None, ymode=0):
        """y[t] = W x[t] (+ res[t]) for every row, x RMS-normed first where norm is given."""
        st = torch.cuda.current_stream().cuda_stream
        for t in range(x.shape[0]):
            if not self.kq.tb_cuda_matvec_fused_dev(
                    w.data_ptr(), qt, m, x.shape[1], x[t].data_ptr(), y[t].data_ptr(), xmode=1 if norm is not None else 0,
                    d_norm_w=norm.data_ptr() if norm is not None else 0, eps=self.s.norm_eps,
                    d_res=res[t].data_ptr() if res is not None else 0, ymode=ymode, stream=st):
                raise RuntimeError("matvec refused")
        return y

    def forward(self, tokens: list[int], seqs: list[int], new: list[int]) -> torch.Tensor:
        """Feeds new[i] tokens to seqs[i] (tokens: all rows in order); the logits of each sequence's last."""
        s, c = self.s, self.cache
        H, NH, NK, D, F = s.hidden, s.n_heads, s.n_kv_heads, s.head_dim, s.ffn_dim
        c.extend(dict(zip(seqs, new)))
        batch = c.batch(seqs, new)
        T, st = len(tokens), torch.cuda.current_stream().cuda_stream
        buf = lambda n: torch.empty(T, n, device="cuda")  # noqa: E731
        x, emb = buf(H), self.head[0]
        rb = Q.row_bytes(s.w_qt, H)
        for t, tok in enumerate(tokens):
            if not self.kq.tb_cuda_dequant_dev(emb.data_ptr() + tok * rb, s.w_qt, 1, H, x[t].data_ptr(), stream=st):
                raise RuntimeError("embedding refused")
        for li, (wqkv, wo, wgu, wd, an, fn, qn, kn) in enumerate(self.layers):
            qkv = self._rows(wqkv, s.a_qt, (NH + 2 * NK) * D, x, buf((NH + 2 * NK) * D), norm=an).view(T, -1, D)
            q = c.append(li, batch, qkv[:, :NH], qkv[:, NH:NH + NK], qkv[:, NH + NK:], rope=self.rope, q_norm=qn,
                         k_norm=kn, eps=s.norm_eps)
            o = c.attend(li, batch, q, window=self.window, sinks=self.sinks).view(T, NH * D)
            x = self._rows(wo, s.a_qt, H, o, buf(H), res=x)
            act = self._rows(wgu, s.w_qt, 2 * F, x, buf(F), norm=fn, ymode=1)
            x = self._rows(wd, s.down_qt, H, act, buf(H), res=x)
        last = x[(np.cumsum(new) - 1).tolist()]
        return self._rows(self.head[2], s.out_qt, s.vocab, last, torch.empty(len(seqs), s.vocab, device="cuda"),
                          norm=self.head[1])

    def sample(self, logits: torch.Tensor, u, top_k: int = 40, temperature: float = 0.8) -> list[int]:
        out = torch.zeros(logits.shape[0], dtype=torch.int32, device="cuda")
        st = torch.cuda.current_stream().cuda_stream
        for i in range(logits.shape[0]):
            if not self.kq.tb_cuda_sample_dev(logits[i].data_ptr(), logits.shape[1], top_k, 0.95, temperature,
                                              float(u[i]), out[i:].data_ptr(), st):
                raise RuntimeError("sampler refused")
        return out.tolist()


def random_model(shape: ModelShape, cache: PagedKV, rope: Rope, seed: int = 1, **kw) -> PagedModel:
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s, m = shape, PagedModel(shape, cache, rope, **kw)
    H, NH, NK, D, F = s.hidden, s.n_heads, s.n_kv_heads, s.head_dim, s.ffn_dim
    norm = lambda n: 1.0 + 0.1 * torch.randn(n, device="cuda", generator=g)  # noqa: E731
    for _ in range(s.n_layers):
        m.set_layer(device_weights(s.a_qt, (NH + 2 * NK) * D, H, g), device_weights(s.a_qt, H, NH * D, g),
                    device_weights(s.w_qt, 2 * F, H, g), device_weights(s.down_qt, H, F, g), norm(H), norm(H), norm(D),
                    norm(D))
    m.set_head(device_weights(s.w_qt, s.vocab, H, g), norm(H), device_weights(s.out_qt, s.vocab, H, g))
    return m


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--samples", type=int, default=4)
    ap.add_argument("--prompt", type=int, default=40)
    ap.add_argument("--new", type=int, default=24)
    ap.add_argument("--cache", choices=TYPES, default="bf16")
    ap.add_argument("--window", type=int, default=0)
    ap.add_argument("--sinks", type=int, default=0)
    ap.add_argument("--seed", type=int, default=1)
    a = ap.parse_args()
    torch.cuda.init()
    if load().tb_cuda_init() != 1:
        raise SystemExit("no device")
    shape = ModelShape(4, 1024, 8, 2, 128, 2048, 4096, down_qt=Q.Q4_K)
    page = 16
    pages = -(-a.prompt // page) + a.samples * (-(-a.new // page) + 2)
    cache = PagedKV.alloc(shape.n_layers, pages, page, shape.n_kv_heads, shape.head_dim, TYPES[a.cache])
    rope = Rope.make(a.prompt + a.new, shape.head_dim, base=shape.rope_base, interleaved=True, scaling="yarn", factor=4.0,
                     orig_len=max(1, (a.prompt + a.new) // 4))
    model = random_model(shape, cache, rope, a.seed, window=a.window, sinks=a.sinks)
    rng = np.random.default_rng(a.seed)
    prompt = rng.integers(0, shape.vocab, a.prompt).tolist()
    root = cache.pool.new()
    logits = model.forward(prompt, [root], [a.prompt])
    live = {cache.fork(root): [] for _ in range(a.samples)}
    cache.free(root)
    done, logits = {}, logits.expand(a.samples, -1).contiguous()
    stop = {s: int(rng.integers(a.new // 2, a.new + 1)) for s in live}   # a random end for each sample
    while live:
        seqs = list(live)
        toks = model.sample(logits, rng.random(len(seqs)))
        for s, t in zip(seqs, toks):
            live[s].append(t)
        for s in [s for s in seqs if len(live[s]) >= stop[s]]:
            done[s] = live.pop(s)
            cache.free(s)
        if live:
            logits = model.forward([v[-1] for v in live.values()], list(live), [1] * len(live))
    for s, v in sorted(done.items()):
        print(f"sample {s}: {len(v)} tokens {v}")
    print(f"{cache.compact()} pages moved, {cache.pool.free_pages} of {pages} free; device error "
          f"{load().tb_cuda_last_error()}")


if __name__ == "__main__":
    main()
