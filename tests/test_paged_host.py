"""Host side of the paged-cache operators: the chunk attention's plans cover
every row and key once, and every entry refuses what it cannot do.  CPU."""
import ctypes as C

import numpy as np
import pytest
import torch

import d2sd
from d2sd import _lib
from d2sd.paged import _spans


def _pages(kv, P):
    return np.concatenate([[0], np.cumsum([-(-n // P) for n in kv])]).astype(np.int32)


def _plan(qo, kv, hq=32, hkv=8, d=128, fmt="bf16", P=16, window=-1, cus=256, max_splits=0, spare=0):
    pi = _pages(np.asarray(kv) + spare, P)
    batch = d2sd.PagedBatch(np.concatenate([[0], np.cumsum(qo)]), kv, pi, np.zeros(pi[-1], np.int32), P, device="cpu")
    attn = d2sd.PagedChunkAttention("cpu").plan(batch, hq, hkv, d, kv_format=fmt, window_left=window, num_cus=cus,
                                                max_splits=max_splits)
    n, host = attn.info.num_items, attn.plan_host
    items = host[:n * _lib.CHUNK_ITEM_INTS].reshape(n, _lib.CHUNK_ITEM_INTS)
    merges = host[n * _lib.CHUNK_ITEM_INTS:].reshape(-1, _lib.CHUNK_MERGE_INTS)
    assert merges.shape[0] == attn.info.num_merges
    return attn, items, merges


@pytest.mark.parametrize("qo,kv,hq,hkv,d", [
    ([1], [1], 32, 8, 128), ([1], [1000], 32, 8, 128), ([1] * 32, list(range(8192, 32768, 768)), 64, 8, 128),
    ([1000] + [1] * 23, [4000] + [1300] * 23, 32, 8, 128), ([0, 5, 0], [3, 5, 0], 28, 4, 128),
    ([2048, 2048], [15000, 16384], 32, 8, 128), ([1024] * 4, [8000, 3000, 2500, 7777], 64, 8, 64),
    ([8, 9, 33], [9000, 9000, 9000], 16, 16, 64), ([7], [3], 8, 2, 64), ([], [], 8, 2, 64)])
@pytest.mark.parametrize("cus,max_splits,window", [(256, 0, -1), (1024, 0, -1), (256, 1, -1), (4, 3, 100)])
def test_plan_covers_every_row_and_chunk_once(qo, kv, hq, hkv, d, cus, max_splits, window):
    # (a request may have more new tokens than cached keys now: rows without a key are planned all the same)
    attn, items, merges = _plan(qo, kv, hq, hkv, d, window=window, cus=cus, max_splits=max_splits)
    g = hq // hkv
    starts = np.concatenate([[0], np.cumsum(qo)])
    seen, slots = {}, set()
    for req, kvh, q0, nq, row0, nrows, pb, pe, chunk, nchunks, slot, kind in items[:, :12].tolist():
        assert q0 == starts[req] and nq == qo[req] and 0 <= chunk < nchunks
        assert (pe - pb) * 16 >= kv[req]
        assert kind == (1 if qo[req] * g <= 32 else 0) and nrows <= (32 if kind else 256 if attn.info.form == 0 else 128)
        assert (req, kvh, row0, chunk) not in seen
        seen[(req, kvh, row0, chunk)] = (nrows, nchunks, slot)
        if nchunks > 1:
            rows = set(range(slot + chunk * nrows, slot + (chunk + 1) * nrows))
            assert not rows & slots
            slots |= rows
    for r, n in enumerate(qo):
        for h in range(hkv):
            mine = sorted((k[2], k[3], *v) for k, v in seen.items() if k[:2] == (r, h))
            covered = 0
            for row0, chunk, nrows, nchunks, _ in mine:
                if chunk == 0:
                    assert row0 == covered
                    covered += nrows
                assert nchunks == sum(1 for m in mine if m[0] == row0)
            assert covered == n * g
    if max_splits == 1:
        assert not slots and not len(merges)
    assert attn.info.workspace_bytes == len(slots) * (d + 1) * 4 and slots == set(range(len(slots)))
    # merges: every row of a split group once, with the group's slots
    merged = set()
    for q0, kvh, row0, nrows, slot, stride, nchunks, _ in merges.tolist():
        assert nrows <= 1024 // d
        group = next(v for k, v in seen.items()
                     if starts[k[0]] == q0 and qo[k[0]] and k[1] == kvh and k[2] <= row0 < k[2] + v[0])
        base = next(k[2] for k, v in seen.items() if v is group)
        assert (stride, nchunks, slot) == (group[0], group[1], group[2] + row0 - base)
        for i in range(nrows):
            assert (q0, kvh, row0 + i) not in merged
            merged.add((q0, kvh, row0 + i))
    split_rows = sum(v[0] for k, v in seen.items() if v[1] > 1 and k[3] == 0)
    assert len(merged) == split_rows


def test_plan_splits_a_lone_long_request_and_not_a_full_batch():
    _, items, merges = _plan([1], [32768])
    assert len(items) > 64 and len(merges)
    _, items, merges = _plan([1] * 512, [500] * 512)
    assert len(items) == 512 * 8 and not len(merges)


def test_plan_picks_the_workgroup_for_the_rows():
    """Tokens alone, eight waves where rows fill the device, four where only shorter items do, four for heads of 64."""
    form = lambda *a, **kw: _plan(*a, **kw)[0].info.form  # noqa: E731
    assert form([1] * 4, [5000] * 4) == 2 and form([4], [900]) == 2
    assert form([1] * 32, [20000] * 32) == 3 and form([1] * 32, [20000] * 32, window=127) == 2
    assert form([2048, 2048], [16384, 16384]) == 0
    assert form([1000], [2100]) == 1
    assert form([2048, 2048], [16384, 16384], 64, 8, 64) == 1


def test_plan_deals_kv_heads_to_xcds_in_turn():
    _, items, _ = _plan([2048], [16384])
    assert all(int(items[i, 1]) == i % 8 for i in range(len(items)))


def test_spans_cover_each_token_once():
    n = np.array([0, 1, 16, 17, 100])
    row = np.concatenate([[0], np.cumsum(n)])
    pi = np.arange(6) * 10
    s = _spans(np.zeros(5, int), n, row[:-1], np.arange(5), False, pi)
    got = [(r, f + i, w + i) for r, c, f, e, w, *_ in s.tolist() for i in range(c)]
    assert sorted(got) == [(r, i, row[r] + i) for r in range(5) for i in range(n[r])] and (s[:, 1] <= 16).all()
    s = _spans(n, n, row[:-1], np.arange(5), True, pi)
    got = [(r, n[r] - f + i, w + i) for r, c, f, e, w, *_ in s.tolist() for i in range(c)]  # cache of n tokens
    assert sorted(got) == [(r, i, row[r] + i) for r in range(5) for i in range(n[r])]


@pytest.mark.parametrize("kw", [dict(qo=[0, 2], kv=[3], pi=[0, 0]), dict(qo=[1, 2], kv=[3], pi=[0, 1]),
                                dict(qo=[0, 2, 1], kv=[3, 3], pi=[0, 1, 2]), dict(qo=[0, 2], kv=[-1], pi=[0, 1]),
                                dict(qo=[0, 2], kv=[3], pi=[0, 9]), dict(qo=[0, 2], kv=[3], pi=[0, 1], P=12),
                                dict(qo=[0], kv=[3], pi=[0, 1]), dict(qo=[0, 2], kv=[2 ** 31], pi=[0, 1]),
                                dict(qo=[0, 2], kv=[17], pi=[0, 1]), dict(qo=[0, 2], kv=[3], pi=[-1, 1])])
def test_batch_refuses(kw):
    with pytest.raises(ValueError):
        d2sd.PagedBatch(kw["qo"], kw["kv"], kw["pi"], [0, 1], kw.get("P", 16), device="cpu")


def test_set_kv_len_stays_within_the_pages():
    b = d2sd.PagedBatch([0, 1], [3], [0, 1], [0], 16, device="cpu")
    b.set_kv_len([16])
    assert b.kv_len.tolist() == [16]
    for bad in ([17], [-1], [1, 2]):
        with pytest.raises(ValueError):
            b.set_kv_len(bad)


@pytest.mark.parametrize("kw", [dict(head_dim=96), dict(num_qo_heads=30), dict(num_kv_heads=0), dict(window_left=-2),
                                dict(max_splits=-1)])
def test_plan_refuses(kw):
    b = d2sd.PagedBatch([0, 1], [3], [0, 1], [0], 16, device="cpu")
    args = dict(num_qo_heads=32, num_kv_heads=8, head_dim=128)
    args.update({k: v for k, v in kw.items() if k in args})
    with pytest.raises(RuntimeError, match="chunk_plan"):
        d2sd.PagedChunkAttention("cpu").plan(b, **args, **{k: v for k, v in kw.items() if k not in args})


def test_plan_and_run_refuse_on_the_host():
    b = d2sd.PagedBatch([0, 1], [3], [0, 1], [0], 16, device="cpu")
    for kw in (dict(kv_format="int8"), dict(sm_scale=0.0), dict(sm_scale=-1.0), dict(sm_scale=float("nan")),
               dict(sinks=torch.zeros(3))):
        with pytest.raises(ValueError):
            d2sd.PagedChunkAttention("cpu").plan(b, 32, 8, 128, **kw)
    with pytest.raises(RuntimeError):
        d2sd.PagedChunkAttention("cpu").run(torch.zeros(1, 32, 128), None)
    with pytest.raises(ValueError):  # CPU pools
        d2sd.PagedKVCache(torch.zeros(2, 8, 16, 128, dtype=torch.bfloat16), torch.zeros(2, 8, 16, 128, dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        d2sd.PagedKVCache.allocate(2, 16, 8, 128, "int8", device="cpu")


def _cache(buf, fmt=0, **kw):
    c = _lib.PagedCache()
    c.k = c.v = buf
    c.k_scale = c.v_scale = buf if fmt else None
    c.stride_page, c.stride_head, c.stride_tok = 8 * 16 * 128, 16 * 128, 128
    c.format, c.num_pages, c.page_size, c.num_kv_heads, c.head_dim = fmt, 4, 16, 8, 128
    for k, v in kw.items():
        setattr(c, k, v)
    return c


BUF = C.create_string_buffer(1 << 16)
AT = (C.addressof(BUF) + 15) & ~15


@pytest.mark.parametrize("fmt,bad", [(0, dict(format=4)), (0, dict(format=-1)), (0, dict(num_pages=0)), (0, dict(page_size=24)),
                                     (0, dict(page_size=0)), (0, dict(num_kv_heads=0)), (0, dict(head_dim=48)),
                                     (0, dict(head_dim=288)), (0, dict(k=None)), (1, dict(k_scale=None)),
                                     (2, dict(v_scale=None)), (0, dict(stride_tok=4)), (2, dict(stride_head=8)),
                                     (0, dict(stride_page=-8)), (3, dict(scale_stride_tok=-1)), (0, dict(k=AT + 8))])
@pytest.mark.parametrize("fn", ["d2sd_cache_write", "d2sd_cache_read"])
def test_cache_entries_refuse_bad_caches(fn, fmt, bad):
    a = _lib.CacheIoArgs()
    a.cache = _cache(AT, fmt, **bad)
    a.items = a.kv_len = a.page_table = a.k = a.v = AT
    a.stride_n, a.stride_h, a.num_items = 1024, 128, 1
    assert getattr(_lib.lib, fn)(C.byref(a), None) != 0
    assert fn[5:].encode() in _lib.lib.d2sd_last_error()


@pytest.mark.parametrize("bad", [dict(num_items=-1), dict(items=None), dict(kv_len=None), dict(page_table=None), dict(k=None),
                                 dict(v=None), dict(k=AT + 2), dict(stride_n=4), dict(stride_h=-8), dict(items=AT + 4)])
def test_cache_entries_refuse_bad_arguments(bad):
    a = _lib.CacheIoArgs()
    a.cache = _cache(AT)
    a.items = a.kv_len = a.page_table = a.k = a.v = AT
    a.stride_n, a.stride_h, a.num_items = 1024, 128, 1
    for k, v in bad.items():
        setattr(a, k, v)
    for fn in ("d2sd_cache_write", "d2sd_cache_read"):
        assert getattr(_lib.lib, fn)(C.byref(a), None) != 0
        assert getattr(_lib.lib, fn)(None, None) != 0


@pytest.mark.parametrize("bad", [dict(q=None), dict(out=None), dict(lse=None), dict(plan=None), dict(kv_len=None),
                                 dict(page_table=None), dict(q=AT + 2), dict(q_stride_n=4), dict(o_stride_h=2),
                                 dict(sm_scale=0.0), dict(sm_scale=float("inf")), dict(workspace=None),
                                 dict(workspace_bytes=8), dict(workspace=AT + 4), "format", "page_size", "heads", "dim", "form", "wide"])
def test_chunk_run_refuses(bad):
    info = _plan([1], [32768])[0].info
    assert info.workspace_bytes > 0
    a = _lib.ChunkRunArgs()
    a.cache = _cache(AT)
    a.plan = a.kv_len = a.page_table = a.q = a.out = a.lse = a.workspace = AT
    a.q_stride_n = a.o_stride_n = 4096
    a.q_stride_h = a.o_stride_h = 128
    a.lse_stride_n, a.sm_scale, a.workspace_bytes = 32, 0.1, info.workspace_bytes
    if isinstance(bad, dict):
        for k, v in bad.items():
            setattr(a, k, v)
    elif bad == "form":
        info.form = 4
    elif bad == "wide":
        a.cache.stride_page = 1 << 32
    else:
        a.cache = _cache(AT, **{"format": dict(fmt=2), "page_size": dict(page_size=32), "heads": dict(num_kv_heads=4),
                                "dim": dict(head_dim=64)}[bad])
    assert _lib.lib.d2sd_chunk_run(C.byref(info), C.byref(a), None) != 0
    assert b"chunk_run" in _lib.lib.d2sd_last_error()
    assert _lib.lib.d2sd_chunk_run(None, C.byref(a), None) != 0


def test_structs_match_the_header():
    """The new structs' sizes and offsets, as a C compiler lays them out."""
    import test_abi_layout as abi
    structs = {"RotaryArgs": "d2sd_rotary_args", "PagedCache": "d2sd_paged_cache", "CacheIoArgs": "d2sd_cache_io_args",
               "ChunkPlanDesc": "d2sd_chunk_plan_desc", "ChunkPlanInfo": "d2sd_chunk_plan_info",
               "ChunkRunArgs": "d2sd_chunk_run_args"}
    old, abi.STRUCTS = abi.STRUCTS, structs
    try:
        abi.test_ctypes_structs_name_every_c_field_in_order()
        abi.test_ctypes_structs_match_the_c_header()
    finally:
        abi.STRUCTS = old
