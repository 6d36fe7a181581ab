"""CPU: the paged cache's host bookkeeping (tb_cuda_kv_pool_*) against a model of who holds what, and the
refusals of the operators' entry points, which come before any launch."""
import ctypes
import random

import numpy as np
import pytest

from trailblaze_b200._lib import KvBatch, KvCache, KvRope, KvRows, RopeScale, lib
from trailblaze_b200.paged import PagePool


def check(pool, model, contents):
    """Every sequence's positions still hold what the model says; free pages are exactly the unheld ones."""
    held = set()
    for s, want in model.items():
        pg = pool.pages(s)
        assert pool.length(s) == len(want)
        assert len(pg) == -(-len(want) // pool.page_size)
        held |= set(pg.tolist())
        for i, w in enumerate(want):
            assert contents[pg[i // pool.page_size], i % pool.page_size] == w, (s, i)
    assert pool.free_pages == pool.n_pages - len(held)
    return held


@pytest.mark.parametrize("seed", range(6))
def test_random_histories(seed):
    """new, extend, fork, truncate, free and compact in random order; pages hold unique marks, copies are made
    exactly where the pool asks for them."""
    rng = random.Random(seed)
    pool = PagePool(rng.choice([7, 24, 61]), rng.choice([16, 32]))
    contents = np.full((pool.n_pages, pool.page_size), -1, np.int64)
    model, mark = {}, 0
    for _ in range(400):
        op = rng.random()
        if op < 0.15:
            s = pool.new()
            assert s not in model
            model[s] = []
        elif op < 0.55 and model:
            s, n = rng.choice(list(model)), rng.randrange(0, 40)
            before = pool.free_pages
            try:
                move = pool.extend(s, n)
            except RuntimeError:
                assert pool.free_pages == before and pool.length(s) == len(model[s])
                need = -(-(len(model[s]) + n) // pool.page_size) - len(pool.pages(s))
                assert need + 1 > before   # the copy may take one more
                continue
            if move:
                contents[move[1]] = contents[move[0]]
            pg = pool.pages(s)
            for i in range(len(model[s]), len(model[s]) + n):
                mark += 1
                contents[pg[i // pool.page_size], i % pool.page_size] = mark
                model[s].append(mark)
        elif op < 0.7 and model:
            s = rng.choice(list(model))
            f = pool.fork(s)
            assert f not in model
            model[f] = list(model[s])
        elif op < 0.8 and model:
            s = rng.choice(list(model))
            n = rng.randrange(0, len(model[s]) + 1)
            pool.truncate(s, n)
            del model[s][n:]
        elif op < 0.92 and model:
            s = rng.choice(list(model))
            pool.free(s)
            del model[s]
        else:
            src, dst = pool.compact()
            assert not set(src.tolist()) & set(dst.tolist()) and len(set(dst.tolist())) == len(dst)
            contents[dst] = contents[src]
            held = check(pool, model, contents)
            assert held == set(range(len(held)))   # dense
        check(pool, model, contents)


def test_pool_refusals():
    L = lib()
    assert not L.tb_cuda_kv_pool_create(0, 16) and not L.tb_cuda_kv_pool_create(4, 0)
    assert not L.tb_cuda_kv_pool_create(4, 20) and not L.tb_cuda_kv_pool_create(4, 65552)
    p = L.tb_cuda_kv_pool_create(4, 16)
    assert L.tb_cuda_kv_pool_extend(p, 0, 1, None, None) == -1     # no such sequence
    s = L.tb_cuda_kv_pool_new(p)
    assert L.tb_cuda_kv_pool_extend(p, s, -1, None, None) == -1
    assert L.tb_cuda_kv_pool_extend(p, s, 65, None, None) == -1 and L.tb_cuda_kv_pool_free_pages(p) == 4
    assert L.tb_cuda_kv_pool_extend(p, s, 2 ** 31 - 1, None, None) == -1
    assert L.tb_cuda_kv_pool_extend(p, s, 20, None, None) == 0
    assert L.tb_cuda_kv_pool_extend(p, s, 2 ** 31 - 1, None, None) == -1   # more than INT_MAX positions
    f = L.tb_cuda_kv_pool_fork(p, s)
    assert L.tb_cuda_kv_pool_extend(p, f, 1, None, None) == -1     # a copy is due and nowhere to name it
    assert L.tb_cuda_kv_pool_extend(p, f, 0, None, None) == 0      # nothing to append, nothing to copy
    assert L.tb_cuda_kv_pool_truncate(p, s, 21) == 0 and L.tb_cuda_kv_pool_truncate(p, s, -1) == 0
    assert L.tb_cuda_kv_pool_free(p, 9) == 0 and L.tb_cuda_kv_pool_free(None, 0) == 0
    assert L.tb_cuda_kv_pool_compact(p, None, None, 4) == -1 and L.tb_cuda_kv_pool_compact(p, None, None, 0) == 0
    assert L.tb_cuda_kv_pool_len(p, 9) == -1 and L.tb_cuda_kv_pool_pages(p, 9, None, 0) == -1
    L.tb_cuda_kv_pool_destroy(p)
    L.tb_cuda_kv_pool_destroy(None)


def arguments():
    """Arguments that the entry points accept as far as the host can tell (nothing is launched: no rows)."""
    c = KvCache(0x10000, 0x20000, 30, 2, 8, 16, 4, 128, 65536, 8192, 2048, 128)
    b = KvBatch(0x1000, 0x2000, 0x3000, 2, 0, 1, 16, 4)
    r = KvRows(0x40000, 4096, 128)
    return c, b, r


def attend(L, c, b, r, layer=0, io=30, heads=16, scale=0.1, window=0, sinks=0, ws=0x50000, n=1 << 30):
    return L.tb_cuda_kv_attend_dev(ctypes.byref(c), layer, ctypes.byref(b), io, heads, ctypes.byref(r), ctypes.byref(r),
                                   scale, window, sinks, ws, n, None)


def append(L, c, b, r, rope=None, layer=0, io=30, heads=16):
    x = ctypes.byref(r)
    return L.tb_cuda_kv_append_dev(ctypes.byref(c), layer, ctypes.byref(b), io, heads, x, x, x, x,
                                   ctypes.byref(rope) if rope else None, None)


BAD_CACHE = [("type", 12), ("n_layers", 0), ("n_pages", 0), ("page_size", 24), ("page_size", 0), ("n_kv_heads", 0),
             ("head_dim", 96), ("pos_stride", 64), ("pos_stride", 132), ("head_stride", 1024), ("page_stride", 4096),
             ("layer_stride", 8192), ("k", 0x10008), ("v", 0), ("page_stride", -8192)]


@pytest.mark.parametrize("field,value", BAD_CACHE)
def test_cache_refusals(field, value):
    L = lib()
    c, b, r = arguments()
    assert attend(L, c, b, r) == 1 and append(L, c, b, r) == 1   # no rows: accepted, nothing to launch
    setattr(c, field, value)
    assert attend(L, c, b, r) == 0 and append(L, c, b, r) == 0
    one = (ctypes.c_int * 1)(0)
    assert L.tb_cuda_kv_copy_dev(ctypes.byref(c), one, one, 0, None) == 0


def test_argument_refusals():
    L = lib()
    c, b, r = arguments()
    assert attend(L, c, b, r, layer=2) == 0 and attend(L, c, b, r, layer=-1) == 0
    assert attend(L, c, b, r, heads=6) == 0 and attend(L, c, b, r, heads=0) == 0 and attend(L, c, b, r, io=12) == 0
    assert attend(L, c, b, r, window=-1) == 0 and attend(L, c, b, r, sinks=-1) == 0
    assert attend(L, c, b, r, scale=float("nan")) == 0 and attend(L, c, b, r, scale=float("inf")) == 0
    assert attend(L, c, b, r, ws=0) == 0 and attend(L, c, b, r, ws=0x50008) == 0 and attend(L, c, b, r, n=8) == 0
    for field, value in (("n_seqs", -1), ("n_tokens", -1), ("pages_stride", -1), ("max_new", -1), ("max_len", -1),
                         ("d_start", 0), ("d_len", 0), ("d_pages", 0)):
        c, b, r = arguments()
        setattr(b, field, value)
        assert attend(L, c, b, r) == 0 and append(L, c, b, r) == 0, field
    for field, value in (("p", 0), ("p", 0x40008), ("row", 4100), ("head", 132), ("row", -4096), ("head", 64)):
        c, b, r = arguments()
        b.n_tokens, b.n_seqs = 3, 0
        assert attend(L, c, b, r) == 1 and append(L, c, b, r) == 1   # rows of no sequence
        setattr(r, field, value)
        assert attend(L, c, b, r) == 0 and append(L, c, b, r) == 0, field
    c, b, r = arguments()
    for rope in (KvRope(0x1004, None, None, 4, 64, 0, 0.0), KvRope(0x1000, None, None, 4, 63, 0, 0.0),
                 KvRope(0x1000, None, None, 4, 130, 0, 0.0), KvRope(0x1000, None, None, -1, 64, 0, 0.0),
                 KvRope(None, 0x1004, None, 0, 0, 0, 1e-6), KvRope(None, 0x1000, None, 0, 0, 0, float("nan"))):
        assert append(L, c, b, r, rope) == 0
    assert append(L, c, b, r, KvRope(0x1000, 0x1000, None, 4, 64, 1, 1e-6)) == 1


def test_rope_table_refusals():
    L = lib()
    ok = dict(base=1e4, factor=4.0, beta_fast=0.0, beta_slow=0.0, attn_factor=0.0, mode=3, orig_len=4096)

    def call(n=0, rot=64, p=0x1000, **kw):
        return L.tb_cuda_rope_table_dev(p, n, rot, ctypes.byref(RopeScale(**{**ok, **kw})), None)
    assert call() == 1
    for kw in (dict(base=0.0), dict(base=float("nan")), dict(factor=0.5), dict(mode=4), dict(mode=-1), dict(orig_len=0),
               dict(beta_fast=1.0, beta_slow=2.0), dict(attn_factor=-1.0), dict(rot=63), dict(rot=0), dict(n=-1), dict(p=0),
               dict(mode=2, rot=2)):
        assert call(**kw) == 0, kw
