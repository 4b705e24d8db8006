"""Host side of the paged-cache operators at the limits of their arguments.  CPU."""
import ctypes as C

import numpy as np
import pytest

import d2sd
from d2sd import _lib


def _plan(qo, kv, pages, P=16, **kw):
    pi = np.concatenate([[0], np.cumsum(pages)])
    b = d2sd.PagedBatch(np.concatenate([[0], np.cumsum(qo)]), kv, pi, np.zeros(int(pi[-1]), np.int32), P, device="cpu")
    return d2sd.PagedChunkAttention("cpu").plan(b, 8, 2, 128, num_cus=kw.pop("num_cus", 256), **kw)


def test_a_window_as_wide_as_the_pages_is_none():
    """Positions below 0 (a cache cut back under its new tokens) less a width near 2^31 leave 32 bits."""
    args = [40, 3], [60, 300], [4, 19]
    none = _plan(*args)
    for window, planned in ((2 ** 31 - 1, -1), (2 ** 31 - 41, -1), (304, -1), (303, 303), (0, 0)):
        got = _plan(*args, window_left=window)
        assert got.info.window_left == planned
        if planned == -1:
            assert np.array_equal(got.plan_host, none.plan_host)
    # and a narrower one that leaves them all the same is refused
    with pytest.raises(RuntimeError, match="window_left"):
        _plan([2 ** 21], [0], [2047], P=2 ** 20, window_left=2047 * 2 ** 20 - 1)


def test_set_kv_len_moves_the_host_lengths():
    """Full reads and plans made after it are for the lengths it gave."""
    b = d2sd.PagedBatch([0, 1, 2], [1000, 20], [0, 4096, 4100], np.zeros(4100, np.int32), 16, device="cpu")
    before = b.prepare_read()._reads[False]
    new = b.prepare_read(new_only=True)._reads[True]
    given = np.array([60000, 17])
    b.set_kv_len(given)
    given[:] = 0
    assert b.kv_len_host.tolist() == [60000, 17] and b.kv_indptr_host.tolist() == [0, 60000, 60017] and b.total_kv == 60017
    spans = b.prepare_read()._reads[False]
    assert spans is not before and int(spans[:, 1].sum()) == 60017 and int(spans[:, 4].max()) == 60016
    assert b.prepare_read(new_only=True)._reads[True] is new
    grown = d2sd.PagedChunkAttention("cpu").plan(b, 8, 2, 128, num_cus=256)
    fresh = _plan([1, 1], [60000, 17], [4096, 4])
    assert np.array_equal(grown.plan_host, fresh.plan_host)
    # batches over shared pages may hold more tokens than a read has rows
    b = d2sd.PagedBatch(range(65), [1] * 64, range(0, 64 * 2048 + 1, 2048), np.zeros(64 * 2048, np.int32), 2 ** 14, device="cpu")
    b.set_kv_len([2 ** 25] * 64)
    with pytest.raises(ValueError, match="2\\^31"):
        b.prepare_read()


@pytest.mark.parametrize("sm_scale", [1.9e-38, 1e-44, 1e-60, 3.5e38, float("inf")])
def test_scales_that_32_bits_do_not_hold_are_refused(sm_scale):
    """Below 2e-38 the rescaling's slack is infinite: rows whose keys were split got output 0 and lse -inf."""
    with pytest.raises(ValueError, match="sm_scale"):
        _plan([1], [3], [1], sm_scale=sm_scale)
    info, a = _plan([1], [3], [1]).info, _lib.ChunkRunArgs()
    a.cache.format, a.cache.num_pages, a.cache.page_size, a.cache.num_kv_heads, a.cache.head_dim = 0, 4, 16, 2, 128
    a.cache.stride_page, a.cache.stride_head, a.cache.stride_tok = 4096, 2048, 128
    a.cache.k = a.cache.v = a.plan = a.kv_len = a.page_table = a.q = a.out = a.lse = 4096  # (refused before any is used)
    a.sm_scale = sm_scale
    assert _lib.lib.d2sd_chunk_run(C.byref(info), C.byref(a), None) != 0
    assert b"sm_scale" in _lib.lib.d2sd_last_error()


def test_the_smallest_scale_is_planned():
    assert _plan([1], [3], [1], sm_scale=2e-38).sm_scale == 2e-38


def test_more_cus_than_the_planner_counts_are_refused():
    """Twice 2^30 workgroups wrapped to a negative number of places, which the schedule never filled."""
    for n in (2 ** 20 + 1, 2 ** 30, 2 ** 31 - 1):
        with pytest.raises(RuntimeError, match="num_cus"):
            _plan([1, 1], [1000, 2000], [63, 125], num_cus=n)
    assert _plan([1, 1], [1000, 2000], [63, 125], num_cus=2 ** 20).info.num_items > 0
