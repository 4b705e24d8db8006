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


def _rows(base, tokens, heads, sn, sh, d):
    return {base + t * sn + h * sh + i for t in range(tokens) for h in range(heads) for i in range(d)}


@pytest.mark.skipif(torch.cuda.is_available(), reason="calls that are not refused would be launched, over no memory")
def test_outputs_that_overlap_an_input_are_refused():
    """q_out over a part of k, v or another place of q: refused; views of one buffer whose rows lie apart: not."""
    import random
    rng = random.Random(0)
    d, seen = 32, {True: 0, False: 0}
    for n in range(1500):
        T, hq, hkv = rng.randint(1, 5), rng.randint(1, 4), rng.randint(1, 3)
        style = rng.randrange(4)
        width = (hq + 2 * hkv) * d + 8 * rng.randrange(3)
        view = {  # token and head stride, start: of heads inside a token's row, or tokens inside a head's
            0: lambda first: (width, d, first * d),
            1: lambda first: (d, T * d, first * T * d),
            2: lambda first: (width, d, first * d + 8 * rng.randint(-2, 2)),
            3: lambda first: (8 * rng.randint(0, 40), 8 * rng.randint(0, 40), 8 * rng.randint(0, 200)),
        }[style]
        q, k, v = view(0), view(hq), view(hq + hkv)
        out = rng.choice([q, q, view(0), view(rng.randint(0, hq + 2 * hkv)), (hq * d, d, 20000), (hq * d, d, 8 * rng.randint(0, 300))])
        if out is q or out == q:
            q = out
        lo = min(x[2] for x in (q, k, v, out))
        q, k, v, out = ((sn, sh, at - lo) for sn, sh, at in (q, k, v, out))
        sets = {x: _rows(x[2], T, h, x[0], x[1], d) for x, h in ((k, hkv), (v, hkv), (q, hq))}
        mine = _rows(out[2], T, hq, out[0], out[1], d)
        apart = len(mine) == T * hq * d
        nested = (T < 2 or out[0] >= d) and (hq < 2 or out[1] >= d) and \
            (T < 2 or hq < 2 or out[0] >= (hq - 1) * out[1] + d or out[1] >= (T - 1) * out[0] + d)
        if apart and not nested:
            continue  # (rows of other orders are refused too)
        bad = not apart or bool(mine & sets[k]) or bool(mine & sets[v]) or (out != q and bool(mine & sets[q]))
        base = 1 << 30
        a = _args(num_tokens=T, num_qo_heads=hq, num_pairs=16, cache=_cache(AT, head_dim=d, num_kv_heads=hkv), q=base + 2 * q[2],
                  k=base + 2 * k[2], v=base + 2 * v[2], q_out=base + 2 * out[2], q_stride_n=q[0], q_stride_h=q[1],
                  qo_stride_n=out[0], qo_stride_h=out[1], k_stride_n=k[0], k_stride_h=k[1], v_stride_n=v[0], v_stride_h=v[1])
        assert _lib.lib.d2sd_cache_append(C.byref(a), None) != 0  # (no device: nothing is launched)
        said = _lib.lib.d2sd_last_error()
        if b"same strides" in said:
            continue
        assert (b"lie apart" in said) == bad, (n, style, T, hq, hkv, q, k, v, out, said)
        seen[bad] += 1
    assert min(seen.values()) > 200, seen


@pytest.mark.skipif(torch.cuda.is_available(), reason="calls that are not refused would be launched, over no memory")
def test_the_fused_projection_in_place_is_taken():
    """A long prompt's queries rotated inside the projection that holds keys and values too: heads of all three side by side,
    and the three behind each other."""
    T, hq, hkv, d = 1 << 20, 64, 8, 128
    base, row = 1 << 40, (hq + 2 * hkv) * d
    one = dict(q=base, q_out=base, k=base + 2 * hq * d, v=base + 2 * (hq + hkv) * d, q_stride_n=row, qo_stride_n=row,
               k_stride_n=row, v_stride_n=row)
    three = dict(q=base, q_out=base, k=base + 2 * T * hq * d, v=base + 2 * T * (hq + hkv) * d, q_stride_n=hq * d, qo_stride_n=hq * d,
                 k_stride_n=hkv * d, v_stride_n=hkv * d)
    for kw in (one, three):
        a = _args(num_tokens=T, num_qo_heads=hq, cache=_cache(AT, num_kv_heads=hkv), **kw)
        assert _lib.lib.d2sd_cache_append(C.byref(a), None) != 0 and b"launch" in _lib.lib.d2sd_last_error()
        for wrong in (dict(q_out=base + 16), dict(k=base + 2 * d * (hq - 1)), dict(v=base + 2 * (hq * d - 8))):
            a = _args(num_tokens=T, num_qo_heads=hq, cache=_cache(AT, num_kv_heads=hkv), **{**kw, **wrong})
            assert _lib.lib.d2sd_cache_append(C.byref(a), None) != 0 and b"lie apart" in _lib.lib.d2sd_last_error(), wrong
