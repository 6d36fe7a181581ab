"""How the paged cache is called from Python: what is refused, whose workspace a call uses, what a table's
shape lets the kernels read.  The numbers are held to oracle/paged_ref.py as in test_gpu_paged.py."""
import math
import os
import sys

import numpy as np
import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from test_gpu_paged import BF16, F16, F32, Case, paged  # noqa: E402,F401

from oracle import paged_ref as R  # noqa: E402

pytestmark = pytest.mark.gpu


def test_tables_on_another_device_are_refused(paged, kq):  # noqa: F811
    """A batch's or a rotary table's pointers go to a kernel on the cache's device."""
    c = Case(paged, [2], [20], 4, 2, 64, F32, F32, 16, seed=30)
    rope = paged.Rope.make(32, 64)
    c.cache.append(1, c.batch, c.q, c.nk, c.nv, rope=rope)
    rope.device = torch.device("cuda", 1)   # as one made there has it
    with pytest.raises(ValueError, match="rotary"):
        c.cache.append(1, c.batch, c.q, c.nk, c.nv, rope=rope)
    c.batch.device = torch.device("cuda", 1)
    with pytest.raises(ValueError, match="batch"):
        c.cache.append(1, c.batch, c.q, c.nk, c.nv)
    with pytest.raises(ValueError, match="batch"):
        c.cache.attend(1, c.batch, c.q)


CHILD = r"""
import sys
sys.path[:0] = [{repo!r}, {tests!r}]
import torch
from trailblaze_b200 import load, paged as P
from test_gpu_paged import BF16, F32, Case
kq = load()
assert kq.tb_cuda_init() == 1
"""


def child(body, **env):
    """A process of its own: the wait limit is read once, when the library starts."""
    import subprocess
    here = os.path.dirname(os.path.abspath(__file__))
    code = CHILD.format(repo=os.path.dirname(here), tests=here) + body
    r = subprocess.run([sys.executable, "-c", code], env=dict(os.environ, **env), capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-3000:]
    return [ln.split()[1:] for ln in r.stdout.splitlines() if ln.startswith("RESULT")]


def test_a_failed_wait_drains_what_is_in_flight():
    """A one-poll limit makes waits of the three attention kernels run out while copies and products are under
    way: each call ends with the error word 1 (or 0, where every poll found its work done), what was in flight has
    landed, and the process and its device memory are as they should be."""
    res = child(r"""
for io, new, lens in ((BF16, [1] * 9, [3000] * 9), (F32, [1, 1], [5000, 33]), (BF16, [300, 40], [4000, 900]),
                      (F32, [200, 40], [3000, 900])):
    c = Case(P, new, lens, 8, 2, 128, io, io, 16, seed=31)
    guard = torch.full((1 << 20,), 7, dtype=torch.int32, device="cuda")
    k, v, q = c.k.clone(), c.v.clone(), c.q.clone()
    for _ in range(5):
        c.cache.attend(1, c.batch, c.q)
    torch.cuda.synchronize()
    same = all(torch.equal(a.view(torch.uint8), b.contiguous().view(torch.uint8)) for a, b in ((k, c.k), (v, c.v), (q, c.q)))
    print("RESULT", kq.tb_cuda_last_error(), int(same), int((guard == 7).all()))
""", TB_WAIT_LIMIT="1")
    assert len(res) == 4
    for err, same, guard in res:
        assert err in ("0", "1") and same == "1" and guard == "1", res


def test_counters_balance_after_a_wait_that_ran_out():
    """Arrival counters that start far below zero make every join's wait run out.  The call reports it (error word
    1) and takes from the counters what arrives there, no more and no less: zeroed, they serve the next call."""
    res = child(r"""
for io, cache, new, lens in ((BF16, BF16, [1] * 9, [3000] * 9), (F32, F32, [1, 1], [5000, 33]),
                             (BF16, BF16, [300, 40, 1], [4000, 900, 700]), (F32, F32, [200, 40, 2], [3000, 900, 700]),
                             (F32, BF16, [200], [3000])):
    c = Case(P, new, lens, 8, 2, 128, io, cache, 16, seed=32)
    want = c.cache.attend(1, c.batch, c.q)
    torch.cuda.synchronize()
    first = kq.tb_cuda_last_error()
    (ws, *_), = c.cache._ws.values()
    n = ws[:2048].view(torch.int32)
    zero = bool((n == 0).all())
    n.fill_(-1000)
    c.cache.attend(1, c.batch, c.q)
    torch.cuda.synchronize()
    err, kept = kq.tb_cuda_last_error(), bool((n == -1000).all())
    n.zero_()
    again = c.cache.attend(1, c.batch, c.q)
    torch.cuda.synchronize()
    print("RESULT", first, int(zero), err, int(kept), kq.tb_cuda_last_error(), int(torch.equal(again, want)))
""", TB_WAIT_LIMIT="200000")
    assert res == [["0", "1", "1", "1", "0", "1"]] * 5, res


def captured(c, stream, **kw):
    """The append and attention of c's batch as a graph, and its output."""
    graph = torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        out = c.cache.attend(1, c.batch, c.cache.append(1, c.batch, c.q, c.nk, c.nv), **kw)
    return graph, out


@pytest.mark.parametrize("io,cache,new,lens", [(BF16, BF16, [1] * 5, [2000, 17, 900, 64, 333]),
                                               (BF16, BF16, [200, 1], [1500, 700]), (F32, F32, [100, 3], [900, 2000])])
def test_captured_calls_have_workspaces_of_their_own(paged, kq, io, cache, new, lens):  # noqa: F811
    """Two graphs captured on one stream, the second replayed first, both replayed on streams of their own beside
    eager calls on the capture stream: no call has another's counters or parts."""
    cases = [Case(paged, new, lens, 8, 2, 128, io, cache, 16, seed=33 + i) for i in range(2)]
    for c in cases:
        c.want = c.cache.attend(1, c.batch, c.cache.append(1, c.batch, c.q, c.nk, c.nv)).clone()
    torch.cuda.synchronize()
    stream, side = torch.cuda.Stream(), [torch.cuda.Stream(), torch.cuda.Stream()]
    one = cases[0]
    made = [(one, *captured(one, stream)), (one, *captured(one, stream)), (cases[1], *captured(cases[1], stream))]
    assert stream.cuda_stream not in one.cache._ws and stream.cuda_stream not in cases[1].cache._ws
    for c, graph, out in reversed(made):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, c.want)
        out.zero_()
    with torch.cuda.stream(stream):
        one.cache.attend(1, one.batch, one.q)   # the capture stream's own, from here on
    torch.cuda.synchronize()
    for _ in range(20):
        for (c, graph, out), s in zip(made, side):
            with torch.cuda.stream(s):
                graph.replay()
        with torch.cuda.stream(stream):
            eager = one.cache.attend(1, one.batch, one.q)
    torch.cuda.synchronize()
    assert torch.equal(eager, one.want) and all(torch.equal(out, c.want) for c, _, out in made[:2])
    assert kq.tb_cuda_last_error() == 0


def test_a_workspace_of_the_callers(paged, kq):  # noqa: F811
    c = Case(paged, [1, 40], [700, 333], 8, 2, 128, BF16, BF16, 16, seed=36)
    c.cache.append(1, c.batch, c.q, c.nk, c.nv)   # as the captured step does
    want = c.cache.attend(1, c.batch, c.q)
    ws = c.cache.workspace()
    before = dict(c.cache._ws)
    for _ in range(3):
        assert torch.equal(c.cache.attend(1, c.batch, c.q, workspace=ws), want)
    torch.cuda.synchronize()
    graph, out = captured(c, torch.cuda.Stream(), workspace=ws)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    assert c.cache._ws == before
    for bad in (ws[:-16], ws[8:], ws.view(torch.int32), ws[::2], ws.cpu()):
        with pytest.raises(ValueError):
            c.cache.attend(1, c.batch, c.q, workspace=bad)


def test_a_captured_step_follows_its_tables(paged, kq):  # noqa: F811
    """The kernels find their work from the tables on the device: a replay after they changed is a call of the
    changed batch."""
    c = Case(paged, [1, 1, 1], [400, 90, 33], 8, 2, 128, BF16, BF16, 16, seed=37)
    ws, out = c.cache.workspace(), torch.empty_like(c.q)
    c.cache.attend(1, c.batch, c.q, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.cache.attend(1, c.batch, c.q, out=out, workspace=ws)
    for lens in ([400, 90, 33], [1, 64, 17], [399, 16, 32]):
        c.batch.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        c.lens = lens
        graph.replay()
        torch.cuda.synchronize()
        c.check(out)
    assert kq.tb_cuda_last_error() == 0


def test_a_rotary_table_of_no_positions(paged, kq):  # noqa: F811
    """Every position is past it: the error word, and nothing is stored."""
    c = Case(paged, [1, 3], [1, 20], 4, 2, 64, F32, F32, 16, seed=38)
    k0 = c.k.clone()
    out = c.cache.append(1, c.batch, c.q, c.nk, c.nv, rope=paged.Rope.make(0, 64))
    torch.cuda.synchronize()
    assert kq.tb_cuda_last_error() == 2
    assert not bool(out.any()) and torch.equal(c.k.nan_to_num(nan=5.0), k0.nan_to_num(nan=5.0))
    with pytest.raises(ValueError):   # pairs there must be
        c.cache.append(1, c.batch, c.q, c.nk, c.nv, rope=paged.Rope(torch.empty(4, 0, 2, device="cuda")))


def test_rows_that_want_a_gradient_are_refused(paged, kq):  # noqa: F811
    """There is no backward pass, and outputs without a graph would lose the gradient without a word."""
    c = Case(paged, [2], [20], 4, 2, 64, F32, F32, 16, seed=39)
    q, w = c.q.clone().requires_grad_(), torch.ones(64, device="cuda", requires_grad=True)
    for call in (lambda: c.cache.attend(1, c.batch, q), lambda: c.cache.append(1, c.batch, q, c.nk, c.nv),
                 lambda: c.cache.append(1, c.batch, c.q, c.nk, c.nv.clone().requires_grad_()),
                 lambda: c.cache.append(1, c.batch, c.q, c.nk, c.nv, k_norm=w)):
        with pytest.raises(ValueError, match="backward"):
            call()
        with torch.no_grad():
            call()
    assert torch.equal(c.cache.attend(1, c.batch, q.detach()), c.cache.attend(1, c.batch, c.q))


def test_numbers_that_do_not_fit_are_refused(paged, kq):  # noqa: F811
    """ctypes drops the upper bits of a number that is too large for a C int."""
    c = Case(paged, [2], [20], 4, 2, 64, F32, F32, 16, seed=41)
    far = 2 ** 32
    for kw in (dict(window=far + 3), dict(window=-far + 3), dict(window=4, sinks=far + 1), dict(window=4, sinks=-1)):
        with pytest.raises(ValueError):
            c.cache.attend(1, c.batch, c.q, **kw)
    for layer in (far + 1, far, -1, 2):
        with pytest.raises(ValueError):
            c.cache.attend(layer, c.batch, c.q)
        with pytest.raises(ValueError):
            c.cache.append(layer, c.batch, c.q, c.nk, c.nv)
    for tail in ((far + 2, 2, 20), (2, far + 2, 20), (2, 2, far + 20)):
        with pytest.raises(ValueError):
            paged.Batch(c.batch.start, c.batch.lens, c.batch.pages, *tail)
    for args in ((far + 8, 64), (8, far + 64)):
        with pytest.raises(ValueError):
            paged.Rope.make(*args)
    assert torch.equal(c.cache.attend(1, c.batch, c.q, window=2 ** 31 - 1), c.cache.attend(1, c.batch, c.q))
