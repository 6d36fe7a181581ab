"""The paged cache's operators together, as examples/paged_generate.py uses them: the same model through the
library's own decoder (its order with the per-head norm before one rotation, fp32 cache) and over the paged
cache, as a prompt chunk, as single tokens and in a batch of forks."""
import ctypes
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(REPO, "examples"))

TOL = 1e-3   # relative L2 of logits: the decoder's own bound against its oracle


def rel(a, b):
    a, b = np.asarray(a, np.float64), np.asarray(b, np.float64)
    return float(np.linalg.norm(a - b) / np.linalg.norm(b))


def test_same_logits_as_the_decoder(kq):
    from paged_generate import random_model
    from trailblaze_b200 import qtypes as Q
    from trailblaze_b200.decoder import Decoder, ModelShape
    from trailblaze_b200.paged import PagedKV, Rope
    s = ModelShape(2, 512, 8, 2, 128, 1024, 1000, down_qt=Q.Q4_K)
    cache = PagedKV.alloc(2, 32, 16, 2, 128, torch.float32)
    m = random_model(s, cache, Rope.make(64, 128, base=s.rope_base, interleaved=True), seed=3)
    dec = Decoder(s, 64, quirks=False)
    try:
        for li, (wqkv, wo, wgu, wd, an, fn, qn, kn) in enumerate(m.layers):
            dec.set_layer(li, wqkv, s.a_qt, wo, s.a_qt, wgu, s.w_qt, wd, s.down_qt, an, fn, qn, kn)
        dec.set_head(m.head[0], s.w_qt, m.head[1], m.head[2], s.out_qt)
        torch.cuda.synchronize()
        toks = np.random.default_rng(3).integers(0, 1000, 37).tolist()
        want = []
        for p, t in enumerate(toks):
            lg = np.zeros(1000, np.float32)
            assert dec.L.tb_cuda_dec_step(dec.d, t, p, ctypes.byref(ctypes.c_int()),
                                          lg.ctypes.data_as(ctypes.POINTER(ctypes.c_float))) == 1
            want.append(lg)
        one, two = cache.pool.new(), cache.pool.new()
        got = m.forward(toks[:30], [one], [30]).cpu().numpy()           # a chunk
        assert rel(got[0], want[29]) <= TOL
        fork = cache.fork(one)
        got = m.forward(toks[30:33] + toks[:20] + [7], [one, two, fork], [3, 20, 1]).cpu().numpy()   # a ragged batch
        assert rel(got[0], want[32]) <= TOL and rel(got[1], want[19]) <= TOL
        for p in range(33, 37):                                          # single tokens, two sequences apart
            got = m.forward([toks[p], toks[p - 13]], [one, two], [1, 1]).cpu().numpy()
            assert rel(got[0], want[p]) <= TOL and rel(got[1], want[p - 13]) <= TOL
        assert kq.tb_cuda_last_error() == 0
    finally:
        dec.close()


@pytest.mark.parametrize("args", [[], ["--cache", "f16", "--window", "24", "--sinks", "4", "--samples", "3"]])
def test_example_runs(kq, args):
    r = subprocess.run([sys.executable, os.path.join(REPO, "examples", "paged_generate.py"), *args], capture_output=True,
                       text=True, timeout=120, cwd=REPO)
    assert r.returncode == 0, r.stderr[-2000:]
    assert "device error 0" in r.stdout and r.stdout.count("sample ") == (3 if args else 4)
