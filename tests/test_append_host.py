"""Host side of the cache's append: the C entry refuses what its kernel does not
take, before any launch, and its struct is the header's."""
import ctypes as C

import pytest
import torch

import d2sd
from d2sd import _lib
from test_paged_host import AT, _cache


def _args(**kw):
    a = _lib.CacheAppendArgs()
    a.cache = _cache(AT)
    a.items = a.kv_len = a.page_table = a.q = a.q_out = a.k = a.v = a.inv_freq = AT
    a.q_stride_n = a.qo_stride_n = 4096
    a.k_stride_n = a.v_stride_n = 1024
    a.q_stride_h = a.qo_stride_h = a.k_stride_h = a.v_stride_h = 128
    a.eps, a.scale, a.num_tokens, a.num_qo_heads, a.num_pairs = 1e-6, 1.0, 1, 32, 64
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("bad", [
    dict(items=None), dict(kv_len=None), dict(page_table=None), dict(q=None), dict(q_out=None), dict(k=None), dict(v=None),
    dict(inv_freq=None), dict(q=AT + 8), dict(q_out=AT + 2), dict(k=AT + 4), dict(v=AT + 8), dict(items=AT + 4),
    dict(q_norm=AT + 2), dict(k_norm=AT + 8), dict(num_tokens=-1), dict(num_qo_heads=-1), dict(num_qo_heads=2 ** 31 - 1), dict(num_pairs=0),
    dict(num_pairs=65), dict(num_pairs=1 << 30), dict(num_pairs=-1), dict(scale=float("nan")), dict(scale=float("inf")),
    dict(q_norm=AT, eps=0.0), dict(k_norm=AT, eps=float("inf")), dict(k_norm=AT, eps=-1.0), dict(q_stride_n=4),
    dict(q_stride_h=-8), dict(qo_stride_n=12), dict(k_stride_n=1023), dict(k_stride_h=-128), dict(v_stride_n=2),
    dict(v_stride_h=-8), dict(qo_stride_h=256)])
def test_append_refuses_bad_arguments(bad):
    a = _args(**bad)
    assert _lib.lib.d2sd_cache_append(C.byref(a), None) != 0
    assert b"cache_append" in _lib.lib.d2sd_last_error()
    assert _lib.lib.d2sd_cache_append(None, None) != 0


@pytest.mark.parametrize("fmt,bad", [(0, dict(format=4)), (0, dict(num_pages=0)), (0, dict(page_size=24)),
                                     (0, dict(head_dim=48)), (1, dict(k_scale=None)), (3, dict(v_scale=None)),
                                     (0, dict(stride_tok=4)), (2, dict(scale_stride_tok=-1)), (0, dict(k=AT + 8))])
def test_append_refuses_bad_caches(fmt, bad):
    a = _args(cache=_cache(AT, fmt, **bad))
    assert _lib.lib.d2sd_cache_append(C.byref(a), None) != 0
    assert b"cache_append" in _lib.lib.d2sd_last_error()


def test_nothing_to_do_needs_no_memory():
    a = _args(num_tokens=0, items=None, kv_len=None, page_table=None, q=None, q_out=None, k=None, v=None, inv_freq=None)
    assert _lib.lib.d2sd_cache_append(C.byref(a), None) == 0


def test_cpu_tensors_are_refused():
    x = torch.zeros(1, 8, 128, dtype=torch.bfloat16)
    pool = torch.zeros(2, 8, 16, 128, dtype=torch.bfloat16)
    i = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError):
        torch.ops.d2sd.cache_append(x, x, x, i, 1, i, i, pool, pool, None, None, 0, False, torch.ones(64, dtype=torch.float64),
                                    None, None, None, 1e-6, 1.0, False, x)


def test_struct_matches_the_header():
    import test_abi_layout as abi
    old, abi.STRUCTS = abi.STRUCTS, {"CacheAppendArgs": "d2sd_cache_append_args"}
    try:
        abi.test_ctypes_structs_name_every_c_field_in_order()
        abi.test_ctypes_structs_match_the_c_header()
    finally:
        abi.STRUCTS = old


def test_traced_by_meta_tensors():
    m = lambda *s, dt=torch.bfloat16: torch.empty(*s, dtype=dt, device="meta")  # noqa: E731
    pool, i = m(2, 8, 16, 128), m(4, dt=torch.int32)
    torch.ops.d2sd.cache_append(m(1, 32, 128), m(1, 8, 128), m(1, 8, 128), i, 1, i, i, pool, pool, None, None, 0, False,
                                m(64, dt=torch.float64), None, None, None, 1e-6, 1.0, False, m(1, 32, 128))
    assert "append" in dir(d2sd.PagedKVCache)
