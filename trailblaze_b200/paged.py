"""Python handle on the paged cache (include/tb_gguf_dequant.h part 4).

    cache = PagedKV.alloc(n_layers, n_pages, page_size, n_kv_heads, head_dim)
    rope = Rope.make(max_positions, head_dim, base=1e6)
    seq = cache.pool.new()
    cache.extend({seq: n_prompt})                 # pages for the new positions
    batch = cache.batch([seq], [n_prompt])        # the step's tables, for every layer
    for layer in ...:
        q = cache.append(layer, batch, q, k, v, rope=rope)   # norm, rotate, store K and V
        o = cache.attend(layer, batch, q)

Everything on the device goes through the C entry points, on torch's current
stream; a refused call raises.  Tensors are kept alive by their own holders:
what a call reads must live until its work on the stream is done, which torch's
allocator sees to for the current stream.
"""
from __future__ import annotations

import ctypes
import math
import operator

import numpy as np
import torch

from . import qtypes as Q
from ._lib import KvBatch, KvCache, KvRope, KvRows, RopeScale, lib

# the current stream's handle on a device, without a torch.cuda.Stream around it (some microseconds of a
# call that a decode step makes for every layer)
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else \
    lambda index: torch.cuda.current_stream(index).cuda_stream
# likewise without the checks that torch is initialised, which a cache's tensors answer
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_capturing = getattr(torch._C, "_cuda_isCurrentStreamCapturing", torch.cuda.is_current_stream_capturing)

_WS_ZEROED = 2048   # TB_KV_WS_ZEROED

_TYPES = {torch.float32: Q.F32, torch.float16: Q.F16, torch.bfloat16: Q.BF16}


def _type(t: torch.Tensor) -> int:
    if t.dtype not in _TYPES:
        raise ValueError(f"{t.dtype}: float32, float16 or bfloat16 expected")
    return _TYPES[t.dtype]


def _rows(t: torch.Tensor, heads: int, dim: int, device) -> KvRows:
    shape, stride = t.shape, t.stride()
    if len(shape) != 3 or shape[1] != heads or shape[2] != dim or stride[2] != 1:
        raise ValueError(f"rows of shape {tuple(shape)}, strides {stride}: [tokens, {heads}, {dim}] with "
                         "contiguous dimensions expected")
    if t.device != device:
        raise ValueError(f"rows on {t.device}: the cache is on {device}")
    # a dimension of one element has no stride of its own
    return KvRows(t.data_ptr(), stride[0] if shape[0] > 1 else 0, stride[1] if heads > 1 else 0)


def _int(n, what: str) -> int:
    """A C int: ctypes and numpy would drop the upper bits of a larger one."""
    n = operator.index(n)
    if not -2 ** 31 <= n < 2 ** 31:
        raise ValueError(f"{what}: {n} does not fit 32 bits")
    return n


def _ints(a, what: str) -> np.ndarray:
    a = np.asarray(a)
    if a.dtype != np.int32:
        b = a.astype(np.int32)
        if a.size and (a.dtype.kind not in "iu" or a.tobytes() != b.astype(a.dtype).tobytes()):
            raise ValueError(f"{what}: whole numbers of 32 bits expected")
        a = b
    return np.ascontiguousarray(a)


def _no_grad(t: torch.Tensor) -> None:
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError("the paged cache has no backward pass: detached rows and weights, or torch.no_grad(), expected")


def _vector(t: torch.Tensor | None, n: int, what: str, device) -> int | None:
    if t is None:
        return None
    _no_grad(t)
    if t.dtype != torch.float32 or t.shape != (n,) or not t.is_contiguous() or t.device != device:
        raise ValueError(f"{what}: a contiguous float32 vector of {n} on {device} expected")
    return t.data_ptr()


class Rope:
    """A rotary table [positions][rot_dim / 2][2] (cos, sin), fp32, and how its pairs lie in a head:
    interleaved (2 i, 2 i + 1) or halves (i, i + rot_dim / 2)."""

    def __init__(self, table: torch.Tensor, interleaved: bool = False):
        if table.dim() != 3 or table.shape[2] != 2 or table.dtype != torch.float32 or not table.is_contiguous() \
                or not table.is_cuda:
            raise ValueError("a contiguous float32 CUDA table [positions, pairs, 2] expected")
        self.table, self.interleaved, self.device = table, bool(interleaved), table.device
        # a table of no positions has no memory, and no table means no rotation: one row that no position is in
        self._memory = table if table.numel() else torch.empty(1, max(1, table.shape[1]), 2, device=table.device)
        self._plain = self.struct(None, None, 0.0)

    def struct(self, q_norm, k_norm, eps) -> KvRope:
        return KvRope(self._memory.data_ptr(), q_norm, k_norm, self.table.shape[0], 2 * self.table.shape[1],
                      self.interleaved, eps)

    @classmethod
    def make(cls, n_pos: int, rot_dim: int, base: float = 1e4, interleaved: bool = False, scaling: str | None = None,
             factor: float = 1.0, orig_len: int = 0, beta_fast: float = 0.0, beta_slow: float = 0.0,
             attn_factor: float = 0.0, device="cuda") -> "Rope":
        """scaling: None, "linear", "ntk" or "yarn" (tb_rope_scale in the header has the formulas)."""
        mode = {None: 0, "linear": 1, "ntk": 2, "yarn": 3}.get(scaling, -1)
        if _int(n_pos, "n_pos") < 0 or _int(rot_dim, "rot_dim") <= 0 or rot_dim % 2:
            raise ValueError(f"a table of {n_pos} positions and {rot_dim} rotary dimensions")
        t = torch.empty(n_pos, rot_dim // 2, 2, dtype=torch.float32, device=device)
        s = RopeScale(base, factor, beta_fast, beta_slow, attn_factor, mode, _int(orig_len, "orig_len"))
        with torch.cuda.device(t.device):
            if t.numel() and lib().tb_cuda_rope_table_dev(t.data_ptr(), n_pos, rot_dim, ctypes.byref(s),
                                                          torch.cuda.current_stream().cuda_stream) != 1:
                raise ValueError("tb_cuda_rope_table_dev refused the scaling")
        return cls(t, interleaved)


class Batch:
    """One step's ragged batch: device int32 tensors start [S + 1], lens [S], pages [S, width], and the
    host's numbers (rows in the step's buffers, the most new tokens and positions of a sequence)."""

    def __init__(self, start: torch.Tensor, lens: torch.Tensor, pages: torch.Tensor, n_tokens: int, max_new: int,
                 max_len: int):
        n = lens.shape[0]
        for t, shape in ((start, (n + 1,)), (lens, (n,)), (pages, (n, pages.shape[-1]))):
            if t.dtype != torch.int32 or not t.is_cuda or tuple(t.shape) != shape or t.device != start.device:
                raise ValueError(f"int32 CUDA tensors [S + 1], [S], [S, width] expected, got {t.dtype} {tuple(t.shape)}")
        if n and (not start.is_contiguous() or not lens.is_contiguous() or (pages.shape[1] > 1 and pages.stride(1) != 1)):
            raise ValueError("start and lens contiguous, rows of pages contiguous")
        self.start, self.lens, self.pages, self.device = start, lens, pages, start.device
        self.n_tokens = n_tokens
        width = pages.shape[1]
        stride = pages.stride(0) if n > 1 and width else width   # a dimension of one element has no stride of its own
        if stride >= 2 ** 31:
            raise ValueError(f"rows of pages {stride} entries apart")
        self.struct = KvBatch(start.data_ptr(), lens.data_ptr(), pages.data_ptr(), n, _int(n_tokens, "n_tokens"),
                              _int(max_new, "max_new"), _int(max_len, "max_len"), stride, width)
        self._ref = ctypes.byref(self.struct)


class PagePool:
    """Host bookkeeping of n_pages pages (tb_cuda_kv_pool_*)."""

    def __init__(self, n_pages: int, page_size: int):
        self.L = lib()
        self.n_pages, self.page_size = n_pages, page_size
        self.p = self.L.tb_cuda_kv_pool_create(_int(n_pages, "n_pages"), _int(page_size, "page_size"))
        if not self.p:
            raise ValueError(f"a pool of {n_pages} pages of {page_size} positions")

    def __del__(self):
        if getattr(self, "p", None):
            self.L.tb_cuda_kv_pool_destroy(self.p)
            self.p = None

    def _id(self, r: int, what: str) -> int:
        if r < 0:
            raise RuntimeError(f"{what} failed ({self.free_pages} of {self.n_pages} pages free)")
        return r

    def new(self) -> int:
        return self._id(self.L.tb_cuda_kv_pool_new(self.p), "new")

    def fork(self, seq: int) -> int:
        return self._id(self.L.tb_cuda_kv_pool_fork(self.p, _int(seq, "seq")), f"fork({seq})")

    def extend(self, seq: int, n: int) -> tuple[int, int] | None:
        """Room for n more positions; the (source, destination) of a page to copy first, if any."""
        a, b = ctypes.c_int(-1), ctypes.c_int(-1)
        r = self._id(self.L.tb_cuda_kv_pool_extend(self.p, _int(seq, "seq"), _int(n, "n"), ctypes.byref(a), ctypes.byref(b)),
                     f"extend({seq}, {n})")
        return (a.value, b.value) if r else None

    def extend_all(self, new: dict[int, int]) -> tuple[np.ndarray, np.ndarray]:
        """Room for new[seq] more positions of each sequence, or of none where one cannot have it; the (sources,
        destinations) of the pages to copy first."""
        seqs, n = _ints(list(new), "sequences"), _ints(list(new.values()), "positions")
        src, dst = np.empty(len(new), np.int32), np.empty(len(new), np.int32)
        m = self._id(self.L.tb_cuda_kv_pool_extend_all(self.p, seqs.ctypes.data, n.ctypes.data, len(new), src.ctypes.data,
                                                       dst.ctypes.data), f"extend({new})")
        return src[:m], dst[:m]

    def truncate(self, seq: int, length: int) -> None:
        if self.L.tb_cuda_kv_pool_truncate(self.p, _int(seq, "seq"), _int(length, "length")) != 1:
            raise RuntimeError(f"truncate({seq}, {length}) failed")

    def free(self, seq: int) -> None:
        if self.L.tb_cuda_kv_pool_free(self.p, _int(seq, "seq")) != 1:
            raise RuntimeError(f"free({seq}) failed")

    def compact(self) -> tuple[np.ndarray, np.ndarray]:
        """Moves the pages in use to the lowest numbers; the (sources, destinations) to copy."""
        src, dst = np.empty(self.n_pages, np.int32), np.empty(self.n_pages, np.int32)
        n = self._id(self.L.tb_cuda_kv_pool_compact(self.p, src.ctypes.data, dst.ctypes.data, self.n_pages), "compact")
        return src[:n], dst[:n]

    def length(self, seq: int) -> int:
        return self._id(self.L.tb_cuda_kv_pool_len(self.p, _int(seq, "seq")), f"length({seq})")

    def pages(self, seq: int) -> np.ndarray:
        n = self._id(self.L.tb_cuda_kv_pool_pages(self.p, _int(seq, "seq"), None, 0), f"pages({seq})")
        a = np.empty(n, np.int32)
        self.L.tb_cuda_kv_pool_pages(self.p, seq, a.ctypes.data, n)
        return a

    @property
    def free_pages(self) -> int:
        return self.L.tb_cuda_kv_pool_free_pages(self.p)


class PagedKV:
    """K and V of every layer in pages: tensors [layers, pages, kv heads, page size, head dim], any
    strides that the header allows (other orders are views with the dimensions permuted)."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor):
        if k.dim() != 5 or k.shape != v.shape or k.stride() != v.stride() or k.dtype != v.dtype or \
                k.device != v.device or not k.is_cuda or k.stride(4) != 1:
            raise ValueError("k and v: CUDA tensors [layers, pages, kv heads, page size, head dim] of one shape, type "
                             "and strides, dimensions contiguous")
        self.L = lib()
        self.k, self.v, self.device = k, v, k.device
        n_layers, n_pages, heads, page, dim = k.shape
        if 0 in k.shape or page % 16 or page > 65536 or dim not in (64, 128):
            raise ValueError(f"a cache of shape {tuple(k.shape)}: pages of a multiple of 16 positions up to 65536, heads "
                             "of 64 or 128 dimensions expected")
        # a dimension of one element has no stride of its own
        st = [s if n > 1 else dim for s, n in zip(k.stride(), k.shape)]
        self.struct = KvCache(k.data_ptr(), v.data_ptr(), _type(k), n_layers, n_pages, page, heads, dim, st[0], st[1],
                              st[2], st[3])
        self._ref = ctypes.byref(self.struct)
        self.n_layers, self.n_pages, self.n_kv_heads, self.page_size, self.head_dim = k.shape
        self._pool: PagePool | None = None
        self._ws: dict[int, tuple] = {}   # by stream: calls that may overlap have one each

    @classmethod
    def alloc(cls, n_layers: int, n_pages: int, page_size: int, n_kv_heads: int, head_dim: int,
              dtype: torch.dtype = torch.bfloat16, device="cuda") -> "PagedKV":
        shape = (n_layers, n_pages, n_kv_heads, page_size, head_dim)
        return cls(torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device))

    # ---- the sequences ----
    @property
    def pool(self) -> PagePool:
        """The bookkeeping of this cache's pages, made at its first use (a caller with page tables of its
        own has none)."""
        if self._pool is None:
            self._pool = PagePool(self.n_pages, self.page_size)
        return self._pool

    def extend(self, new: dict[int, int]) -> None:
        """Room for new[seq] more positions of each sequence; part-filled pages that are shared are copied.  Where
        one of them cannot have it, none gets any (and the call raises)."""
        self.copy_pages(*self.pool.extend_all(new))

    def fork(self, seq: int) -> int:
        return self.pool.fork(seq)

    def free(self, seq: int) -> None:
        self.pool.free(seq)

    def compact(self) -> int:
        """Moves the pages in use to the front of the pool; returns how many moved."""
        src, dst = self.pool.compact()
        self.copy_pages(src, dst)
        return len(src)

    def batch(self, seqs: list[int], new: list[int], n_tokens: int | None = None) -> Batch:
        """The tables of a step that appends (or has appended) new[i] tokens to seqs[i], rows in this order."""
        lens = [self.pool.length(s) for s in seqs]
        tables = [self.pool.pages(s) for s in seqs]
        width = max([len(t) for t in tables], default=0) or 1
        start = _ints(np.concatenate([[0], np.cumsum(np.asarray(new, np.int64))]), "new")
        at = np.full((len(seqs), width), -1, np.int32)
        for i, t in enumerate(tables):
            at[i, :len(t)] = t
        up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(self.device)  # noqa: E731
        return Batch(up(start), up(np.asarray(lens, np.int32)), up(at), int(start[-1]) if n_tokens is None else n_tokens,
                     max(new, default=0), max(lens, default=0))

    # ---- the operators ----
    def append(self, layer: int, batch: Batch, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
               q_out: torch.Tensor | None = None, rope: Rope | None = None, q_norm: torch.Tensor | None = None,
               k_norm: torch.Tensor | None = None, eps: float = 1e-6) -> torch.Tensor:
        """Norms and rotates q (returned, or in q_out) and k, and stores k and v at the batch's positions."""
        heads, dim, dev = q.shape[1] if q.dim() == 3 else 0, self.head_dim, self.device
        self._tokens(batch, q, k, v)
        if not 0 <= layer < self.n_layers:
            raise ValueError(f"layer {layer} of {self.n_layers}")
        if rope is not None and rope.device != dev:
            raise ValueError(f"rotary table on {rope.device}: the cache is on {dev}")
        rq, rk, rv = _rows(q, heads, dim, dev), _rows(k, self.n_kv_heads, dim, dev), _rows(v, self.n_kv_heads, dim, dev)
        if q_out is None:
            q_out = torch.empty_like(q)
        elif q_out.shape != q.shape or q_out.dtype != q.dtype:
            raise ValueError("q_out: the shape and type of q expected")
        ro = _rows(q_out, heads, dim, dev)
        if q_norm is None and k_norm is None:
            r = rope._plain if rope else None
        else:
            qn, kn = _vector(q_norm, dim, "q_norm", dev), _vector(k_norm, dim, "k_norm", dev)
            r = rope.struct(qn, kn, eps) if rope else KvRope(None, qn, kn, 0, 0, 0, eps)
        if self._on_device(self.L.tb_cuda_kv_append_dev, self._ref, layer, batch._ref, _type(q), heads,
                           ctypes.byref(rq), ctypes.byref(rk), ctypes.byref(rv), ctypes.byref(ro),
                           ctypes.byref(r) if r is not None else None, _raw_stream(dev.index)) != 1:
            raise ValueError("tb_cuda_kv_append_dev refused the call")
        return q_out

    def workspace(self) -> torch.Tensor:
        """A workspace for attend(), zeroed.  Calls that may overlap on the GPU need one each.  Without one, calls on
        a stream share that stream's, and a call that is captured into a graph gets its own, filled with zeros
        in the graph: a graph that takes one from outside has a launch less for every call."""
        return torch.zeros(self.L.tb_cuda_kv_attend_ws(), dtype=torch.uint8, device=self.device)

    def _own_workspace(self, stream: int) -> tuple:
        if _capturing():
            # from the graph's memory and not kept: what ran on the stream before, another graph captured on
            # it and this graph's replays on any stream have nothing of it in common
            ws = torch.empty(self.L.tb_cuda_kv_attend_ws(), dtype=torch.uint8, device=self.device)
            ws[:_WS_ZEROED].zero_()
            return ws, ws.data_ptr(), ws.numel()
        ws = self._ws.get(stream)
        if ws is None:
            ws = self.workspace()
            ws = self._ws[stream] = (ws, ws.data_ptr(), ws.numel())
        return ws

    def attend(self, layer: int, batch: Batch, q: torch.Tensor, out: torch.Tensor | None = None,
               scale: float | None = None, window: int = 0, sinks: int = 0,
               workspace: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of the batch's new tokens over their sequences' positions (tb_cuda_kv_attend_dev); out must not
        overlap q."""
        heads, dim, dev = q.shape[1] if q.dim() == 3 else 0, self.head_dim, self.device
        self._tokens(batch, q)
        if not (0 <= window < 2 ** 31 and 0 <= sinks < 2 ** 31 and 0 <= layer < self.n_layers):
            raise ValueError(f"layer {layer} of {self.n_layers}, window {window}, {sinks} first tokens")
        rq = _rows(q, heads, dim, dev)
        if out is None:
            out = torch.empty_like(q)
        elif out.shape != q.shape or out.dtype != q.dtype:
            raise ValueError("out: the shape and type of q expected")
        ro = _rows(out, heads, dim, dev)
        stream = _raw_stream(dev.index)
        if workspace is None:
            ws = self._own_workspace(stream)
        elif workspace.dtype != torch.uint8 or workspace.device != dev or not workspace.is_contiguous():
            raise ValueError(f"workspace: a contiguous uint8 tensor on {dev} expected")
        else:
            ws = workspace, workspace.data_ptr(), workspace.numel()
        if self._on_device(self.L.tb_cuda_kv_attend_dev, self._ref, layer, batch._ref, _type(q), heads,
                           ctypes.byref(rq), ctypes.byref(ro), 1.0 / math.sqrt(dim) if scale is None else scale, window,
                           sinks, ws[1], ws[2], stream) != 1:
            raise ValueError("tb_cuda_kv_attend_dev refused the call")
        return out

    def copy_pages(self, src, dst) -> None:
        """Pages dst[i] = pages src[i], K and V of every layer; host sequences of page numbers."""
        src, dst = _ints(src, "src"), _ints(dst, "dst")
        if src.ndim != 1 or src.shape != dst.shape:
            raise ValueError("src and dst: page numbers, one for one")
        if self._on_device(self.L.tb_cuda_kv_copy_dev, self._ref, src.ctypes.data, dst.ctypes.data, src.size,
                           _raw_stream(self.device.index)) != 1:
            raise ValueError("tb_cuda_kv_copy_dev refused the pages")

    def _on_device(self, call, *args) -> int:
        """The entry points launch on the current device: the cache's, for the length of the call."""
        if _current_device() == self.device.index:
            return call(*args)
        with torch.cuda.device(self.device):
            return call(*args)

    def _tokens(self, batch: Batch, *rows: torch.Tensor) -> None:
        n, dtype = batch.n_tokens, rows[0].dtype
        if batch.device != self.device:
            raise ValueError(f"batch on {batch.device}: the cache is on {self.device}")
        for t in rows:
            if t.dim() != 3 or t.shape[0] != n:
                raise ValueError(f"rows of shape {tuple(t.shape)}: the batch has {n} rows")
            if t.dtype != dtype:
                raise ValueError("q, k and v of one type expected")
            if t.requires_grad:
                _no_grad(t)
