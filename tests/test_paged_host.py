"""Host side of the paged KV cache: its book-keeping, and the refusals that come before any launch (fake addresses are never dereferenced)."""
import ctypes

import numpy as np
import pytest
import torch

from tscale_b200 import abi, ops

NULL = abi.Ptr2D(None, 0, 0, 0)
FAKE = 4096


def _kv(**kw):
    f = dict(k=FAKE, v=FAKE, k_scale=FAKE, v_scale=FAKE, pos=FAKE, weight=FAKE, page_count=10, page_size=64, kv_heads=2)
    f.update(kw)
    return abi.PagedKv(*(f[n] for n, _ in abi.PagedKv._fields_))


def _cfg(**kw):
    f = dict(head_dim=64, kv_dtype=abi.TSA_I8, scale_dtype=abi.TSA_F16, out_dtype=abi.TSA_F32, qk_vec_scale=1.0)
    f.update(kw)
    return abi.PagedCfg(*(f[n] for n, _ in abi.PagedCfg._fields_))


def _plane(cols, rows, stride=None, data=FAKE):
    return abi.Ptr2D(data, cols * 4 if stride is None else stride, cols, rows)


def _append(cfg=None, kv=None, table=None, ctx=FAKE, starts=FAKE, n=3, rows=5, k=None, ks=None):
    k = k or abi.Ptr2D(FAKE, 128, 128, 5)
    ks = ks or _plane(5, 2)
    return abi.lib().tsa_paged_append(ctypes.byref(cfg or _cfg()), ctypes.byref(kv or _kv()), table or _plane(4, 3), ctx, FAKE, starts, n, rows, k, ks, k, ks,
                                      None, None)


def _decode(cfg=None, kv=None, table=None, ctx=FAKE, tokens=FAKE, n=3, max_ctx=200, q=None, qs=NULL, window=9, out=None, heads=4, ws=FAKE, ws_bytes=1 << 30):
    return abi.lib().tsa_paged_decode(ctypes.byref(cfg or _cfg()), ctypes.byref(kv or _kv()), table or _plane(4, 3), ctx, tokens, n, max_ctx,
                                      q or abi.Ptr2D(FAKE, 256, 256, 3), qs, window, 0.0, out or abi.Ptr2D(FAKE, 1024, 256, 3), heads, ws, ws_bytes, None, None)


def _select(kv=None, tokens=FAKE, n=3, max_ctx=200, keep=50, recent=4, moves=FAKE, cap=50, counts=FAKE, new=FAKE):
    return abi.lib().tsa_paged_evict_select(ctypes.byref(kv or _kv()), _plane(4, 3), FAKE, tokens, n, max_ctx, keep, recent, moves, cap, counts, new, None, None)


def _move(cfg=None, kv=None, moves=FAKE, cap=5, counts=FAKE, n=3):
    return abi.lib().tsa_paged_evict_move(ctypes.byref(cfg or _cfg()), ctypes.byref(kv or _kv()), _plane(4, 3), moves, cap, counts, n, None, None)


POOLS = [(dict(page_size=48), b"page size"), (dict(page_size=8), b"page size"), (dict(page_size=512), b"page size"), (dict(page_count=0), b"pages"),
         (dict(kv_heads=0), b"pages"), (dict(page_count=1 << 20, kv_heads=1 << 12), b"pages"), (dict(kv_heads=65536), b"key heads"), (dict(k=None), b"null"), (dict(v_scale=None), b"null"),
         (dict(k=FAKE + 8), b"aligned"), (dict(pos=FAKE + 4), b"aligned")]


@pytest.mark.parametrize("kw,text", POOLS)
def test_pools_that_are_refused(kw, text):
    for call in (_append, _decode, _move):
        assert call(kv=_kv(**kw)) == abi.TSA_BAD_ARG and text in abi.lib().tsa_last_error()


@pytest.mark.parametrize("kw", [dict(head_dim=96), dict(head_dim=256), dict(kv_dtype=abi.TSA_F16), dict(scale_dtype=abi.TSA_BF16)])
def test_types_that_are_refused(kw):
    for call in (_append, _decode, _move):
        assert call(cfg=_cfg(**kw)) == abi.TSA_BAD_ARG


@pytest.mark.parametrize("call,kw,text", [
    (_append, dict(n=-1), b"sequences"), (_append, dict(n=70000), b"sequences"), (_append, dict(table=NULL), b"page table"), (_append, dict(ctx=None), b"page table"),
    (_append, dict(table=_plane(4, 2)), b"page table"), (_append, dict(table=_plane((1 << 24) + 1, 3)), b"2^30"), (_append, dict(table=_plane(4, 3, stride=18)), b"page table"), (_append, dict(rows=-1), b"row count"),
    (_append, dict(starts=None), b"rowStarts"), (_append, dict(k=abi.Ptr2D(FAKE, 128, 100, 5)), b"extents"), (_append, dict(k=abi.Ptr2D(FAKE, 128, 128, 4)), b"extents"),
    (_append, dict(k=abi.Ptr2D(FAKE + 8, 128, 128, 5)), b"aligned"), (_append, dict(k=abi.Ptr2D(FAKE, 136, 128, 5)), b"aligned"),
    (_append, dict(ks=_plane(4, 2)), b"kvHeads"), (_append, dict(ks=_plane(5, 1)), b"kvHeads"), (_append, dict(ks=_plane(5, 2, stride=22)), b"aligned"),
    (_append, dict(k=NULL), b"null"),
    (_decode, dict(cfg=_cfg(out_dtype=abi.TSA_I8)), b"out dtype"), (_decode, dict(heads=3), b"evenly"), (_decode, dict(heads=0), b"evenly"),
    (_decode, dict(window=-1), b"window"), (_decode, dict(max_ctx=-1), b"window"), (_decode, dict(tokens=None), b"go together"),
    (_decode, dict(kv=_kv(pos=None)), b"go together"), (_decode, dict(q=NULL), b"null"), (_decode, dict(q=abi.Ptr2D(FAKE, 256, 255, 3)), b"extents"),
    (_decode, dict(q=abi.Ptr2D(FAKE, 264, 256, 3)), b"aligned"), (_decode, dict(out=abi.Ptr2D(FAKE, 1024, 256, 2)), b"extents"),
    (_decode, dict(out=abi.Ptr2D(FAKE + 4, 1024, 256, 3)), b"aligned"), (_decode, dict(qs=_plane(3, 3)), b"qScale"), (_decode, dict(qs=_plane(4, 3, stride=18)), b"qScale"),
    (_decode, dict(ws=None, max_ctx=20000, window=5000), b"workspace"), (_decode, dict(ws=None, max_ctx=20000, window=5000, kv=_kv(weight=None)), b"workspace"),
    (_decode, dict(ws_bytes=100, max_ctx=20000, window=5000), b"workspace"), (_decode, dict(ws=FAKE + 8), b"workspace"),
    (_decode, dict(n=60000, table=_plane(1 << 24, 60000), max_ctx=1 << 29, q=abi.Ptr2D(FAKE, 256, 256, 60000), out=abi.Ptr2D(FAKE, 1024, 256, 60000)), b"too much"),
    (_select, dict(kv=_kv(weight=None)), b"weights"), (_select, dict(keep=0), b"keep"), (_select, dict(recent=51), b"keep"), (_select, dict(recent=-1), b"keep"),
    (_select, dict(tokens=None), b"go together"), (_select, dict(cap=49), b"room for 50"), (_select, dict(cap=0, max_ctx=40), b"room for 1"),
    (_select, dict(moves=None), b"null"), (_select, dict(moves=FAKE + 4), b"aligned"), (_select, dict(new=None), b"null"),
    (_move, dict(cap=-1), b"moveCap"), (_move, dict(moves=None), b"moves"), (_move, dict(moves=FAKE + 4), b"moves"), (_move, dict(counts=None), b"null"),
])
def test_arguments_that_are_refused(call, kw, text):
    assert call(**kw) == abi.TSA_BAD_ARG and text in abi.lib().tsa_last_error(), abi.lib().tsa_last_error()


def test_calls_without_work_launch_nothing():
    assert _append(n=0, rows=0) == abi.TSA_OK and _append(rows=0) == abi.TSA_OK and _decode(n=0) == abi.TSA_OK
    assert _select(n=0) == abi.TSA_OK and _move(n=0) == abi.TSA_OK and _move(cap=0) == abi.TSA_OK


def test_workspace_sizes():
    need = lambda n, heads, ctx, window=1 << 30, **kw: abi.lib().tsa_paged_decode_workspace_bytes(  # noqa: E731
        ctypes.byref(_cfg()), ctypes.byref(_kv(**kw)), n, heads, ctx, window)
    assert need(3, 4, 200) == need(3, 4, 200, weight=None) == 0  # a cluster per key head
    assert need(3, 4, 20000) - need(3, 4, 20000, weight=None) == 256 + 3 * 4 * 20000 * 4 and need(3, 4, 20000, weight=None) > 0
    assert need(3, 4, 20000, 64) == 0 and need(3, 4, 20000, 1500) > 0  # a short window: its keys are listed in shared memory
    assert need(3, 4, 20000, 64, pos=None, weight=None) == 0 and need(300, 4, 20000, 64, pos=None, weight=None) == 0
    assert need(0, 4, 200) == 0 and need(3, 1, 200) == 0 and need(3, 4, -1) == 0 and need(3, 4, 200, -1) == 0


def _tensors(**kw):
    plane = (10, 2, 64)
    t = dict(k=torch.zeros(plane + (64,), dtype=torch.int8), v=torch.zeros(plane + (64,), dtype=torch.int8), k_scale=torch.ones(plane, dtype=torch.float16),
             v_scale=torch.ones(plane, dtype=torch.float16), pos=torch.zeros(plane, dtype=torch.int32), weight=torch.zeros(plane))
    t.update(kw)
    return ops.PagedKV(**t)


TABLE, CTX = torch.zeros((3, 4), dtype=torch.int32), torch.ones(3, dtype=torch.int32)


@pytest.mark.parametrize("kw", [
    dict(v=torch.zeros((10, 2, 64, 128), dtype=torch.int8)), dict(v=torch.zeros((10, 2, 64, 64), dtype=torch.uint8)), dict(k=None), dict(v_scale=None),
    dict(k_scale=torch.ones((10, 2, 64))), dict(k_scale=torch.ones((10, 64, 2), dtype=torch.float16).transpose(1, 2)), dict(pos=torch.zeros((10, 2, 64))),
    dict(weight=torch.zeros((10, 2, 64), dtype=torch.float64)), dict(weight=torch.zeros((10, 2, 32))),
    dict(k=torch.zeros((10, 2, 64, 128), dtype=torch.int8)[..., :64], v=torch.zeros((10, 2, 64, 128), dtype=torch.int8)[..., :64])])
def test_tensors_that_are_refused(kw):
    q = torch.zeros((3, 256), dtype=torch.int8)
    with pytest.raises(AssertionError):
        ops.paged_decode(_tensors(**kw), TABLE, CTX, q, None, 5, 0.0, tokens=CTX)


def test_other_arguments_that_are_refused():
    q, kv = torch.zeros((3, 256), dtype=torch.int8), _tensors()
    row, scale = torch.zeros((3, 128), dtype=torch.int8), torch.ones((2, 3))
    for args, kw in (((TABLE, CTX, q.to(torch.uint8), None, 5, 0.0), {}), ((TABLE.long(), CTX, q, None, 5, 0.0), {}), ((TABLE, CTX.long(), q, None, 5, 0.0), {}),
                     ((TABLE, CTX, q, torch.ones((3, 4), dtype=torch.float16), 5, 0.0), {}), ((TABLE, CTX, q, None, 5, 0.0), dict(tokens=CTX[:2])),
                     ((TABLE, CTX, torch.zeros((3, 100), dtype=torch.int8), None, 5, 0.0), {}), ((TABLE, CTX, q, None, 5, 0.0), {})):  # the last: not on a GPU
        with pytest.raises(AssertionError):
            ops.paged_decode(kv, *args, **kw)
    for kw in (dict(max_ctx=1 << 32), dict(max_ctx=-1 << 40)):  # would be another number in 32 bits
        with pytest.raises(AssertionError, match="32 bits"):
            ops.paged_decode(kv, TABLE, CTX, q, None, 5, 0.0, tokens=CTX, **kw)
        with pytest.raises(AssertionError, match="32 bits"):
            ops.paged_evict_select(kv, TABLE, CTX, 5, 1, tokens=CTX, **kw)
    with pytest.raises(TypeError):
        ops.paged_decode(kv[:5], TABLE, CTX, q, None, 5, 0.0)
    for args in ((row, scale.half(), row, scale), (row.to(torch.uint8), scale, row, scale), (row, scale, row, scale)):
        with pytest.raises(AssertionError):
            ops.paged_append(kv, TABLE, CTX, *args, tokens=CTX)
    with pytest.raises(AssertionError):
        ops.paged_append(kv, TABLE, CTX, row, scale, row, scale, row_starts=torch.zeros(3, dtype=torch.int32))
    moves, counts = torch.zeros((3, 2, 5, 2), dtype=torch.int32), torch.zeros((3, 2), dtype=torch.int32)
    for m, c in ((moves[..., :1], counts), (moves, counts[:, :1]), (moves.long(), counts), (moves[:2], counts), (moves, counts)):
        with pytest.raises(AssertionError):
            ops.paged_evict_move(kv, TABLE, m, c)
    with pytest.raises(AssertionError):
        ops.paged_evict_select(kv._replace(weight=None), TABLE, CTX, 5, 1)


def _taken(cache):
    used = cache.page_table[cache.page_table >= 0].tolist()
    assert sorted(used + cache.free) == list(range(cache.page_count))
    for s, n in enumerate(cache.lens):
        pages = -(-int(n) // cache.page_size)
        assert (cache.page_table[s, :pages] >= 0).all() and (cache.page_table[s, pages:] == -1).all()
    assert cache.ctx_lens.tolist() == cache.lens.tolist()
    return len(used)


def test_book_keeping():
    cache = ops.PagedKVCache(3, 12, 2, 64, "cpu", page_size=16, max_pages=8, evict=True)
    table = cache.page_table
    assert cache.extend([17, 0, 16]).tolist() == [0, 17, 17, 33] and _taken(cache) == 3
    assert cache.extend() is None and _taken(cache) == 5 and cache.lens.tolist() == [18, 1, 17] and cache.tokens.tolist() == [18, 1, 17]
    before = cache._host.copy()
    for counts in ([200, 0, 0], [50, 50, 50], -1, [128 - 17, 0, 0]):  # beyond a sequence's pages, beyond the pool, negative
        with pytest.raises(abi.TsaError):
            cache.extend(counts)
        assert np.array_equal(cache._host, before) and _taken(cache) == 5
    cache.release(0)
    assert _taken(cache) == 3 and cache.lens.tolist() == [0, 1, 17] and cache.tokens.tolist() == [0, 1, 17]
    cache.extend([100, 15, 0])
    assert _taken(cache) == 10 and cache.page_table is table
    with pytest.raises(ValueError):
        ops.PagedKVCache(0, 12, 2, 64, "cpu")


def test_struct_layouts():
    assert ctypes.sizeof(abi.PagedKv) == 64 and ctypes.sizeof(abi.PagedCfg) == 20
