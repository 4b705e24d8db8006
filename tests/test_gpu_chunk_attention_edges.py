"""PagedChunkAttention at the edges of what it accepts, against the 64-bit form
with the tolerances that test_gpu_chunk_attention.py derives."""
import math

import numpy as np
import pytest
import torch

import d2sd
from oracle import paged_oracle as po
from test_gpu_chunk_attention import DEV, Problem, U

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 2, 2 ** 31 - 41, 2 ** 30])
@pytest.mark.parametrize("fmt,d", [("bf16", 128), ("mxfp4", 64)])
def test_the_widest_windows_over_caches_cut_back(window, fmt, d):
    """Requests that hold fewer tokens than they have new ones start below position 0; a window as wide as an int
    changes nothing for their rows (chunks, and token items of one and two row blocks)."""
    qo, kv = [40, 3, 8, 1], [60, 300, 8, 5]
    wide, none = Problem(qo, kv, 8, 2, d, fmt, window=window), Problem(qo, kv, 8, 2, d, fmt)
    for lens in ([35, 1, 5, 0], [38, 2, 7, 5], kv):
        got = []
        for p in (wide, none):
            p.batch.set_kv_len(lens)
            got.append(p.run())
        torch.cuda.synchronize()
        wide.check(*got[0], kv=lens)
        assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])


@pytest.mark.parametrize("num_cus", [1, 256, 4096])
@pytest.mark.parametrize("fmt,d", [("bf16", 128), ("mxfp8", 64)])
def test_a_sink_of_minus_infinity_is_no_sink(fmt, d, num_cus):
    """Heads without a sink beside heads with one, plans with and without split keys: rows without a key get output 0
    and lse -inf from them too, the others the output of a plan without sinks."""
    qo, kv = [40, 3, 1, 6], [900, 2500, 2100, 2200]
    p, plain = (Problem(qo, kv, 8, 2, d, fmt, sinks=s, num_cus=num_cus) for s in (True, False))
    p.attn.sinks[::3] = -math.inf
    p.sinks[::3] = -1e30  # in the 64-bit form: the same, but for rows without a key, where -inf - -inf is no number
    assert (num_cus == 1) == (p.attn.info.num_merges == 0)
    for lens in (kv, [25, 1, 0, 3]):
        got = []
        for x in (p, plain):
            x.batch.set_kv_len(lens)
            got.append(x.run())
        torch.cuda.synchronize()
        p.check(*got[0], kv=lens)
        assert torch.equal(got[0][0][:, ::3], got[1][0][:, ::3]) and torch.equal(got[0][1], got[1][1])


@pytest.mark.parametrize("num_cus", [1, 4096])
@pytest.mark.parametrize("sm_scale", [2.1e-38, 1e-36, 1e-30])
@pytest.mark.parametrize("fmt,d", [("bf16", 128), ("mxfp4", 64)])
def test_scales_near_the_smallest_float(fmt, d, sm_scale, num_cus):
    """Every visible key weighs the same; the rescaling's slack, about 8 / sm_scale, is near the largest float."""
    p = Problem([40, 3, 1], [900, 1500, 2100], 8, 2, d, fmt, sm_scale=sm_scale, num_cus=num_cus)
    assert (num_cus == 1) == (p.attn.info.num_merges == 0)
    out, lse = p.run()
    torch.cuda.synchronize()
    p.check(out, lse)


def _expected(p):
    """Outputs and log-sums of the whole batch in 64 bits, and how far off each may be."""
    parts, q0, k0 = [], 0, 0
    for n, L in zip(p.qo, p.kv):
        o, s, A, size = po.attention_ref(p.q[q0:q0 + n], p.kr[k0:k0 + L], p.vr[k0:k0 + L], L - n, p.group, p.scale, p.window)
        e = (p.d + 4) * U * size
        parts.append((o, 2.0 ** -8 * o.abs() + A * (2.0 ** -8 + 2 * e + 2 * L * U + 32 * U)[..., None] + 1e-30,
                      s, 2 * e + L * U + 32 * U + 4 * U * s.abs()))
        q0, k0 = q0 + n, k0 + L
    return [torch.cat(x) for x in zip(*parts)]


def _poison(p, side, request, token, what):
    """Writes the cache with `what` in one token's key or value, head 1, dim 37.  The dims it spreads to there: a block
    of 32 in the block formats."""
    kv = [p.k.clone(), p.v.clone()]
    kv[side][sum(p.kv[:request]) + token, 1, 37] = what
    p.cache.write(*(x.to(DEV) for x in kv), d2sd.PagedBatch(
        np.concatenate([[0], np.cumsum(p.kv)]), p.kv, p.batch.page_indptr_host, p.table, p.cache.page_size, device=DEV))
    return range(32, 64) if p.fmt.startswith("mx") else range(37, 38)


@pytest.mark.parametrize("num_cus", [1, 4096])
@pytest.mark.parametrize("window", [-1, 70])
@pytest.mark.parametrize("fmt", ["bf16", "fp8", "mxfp8", "mxfp4"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("qo,kv", [([100, 8, 1], [160, 90, 300]), ([300, 6], [300, 1200]), ([1, 3, 4], [70, 300, 260]),
                                   ([60, 2], [1500, 2600])])
def test_what_a_row_does_not_see_may_be_infinite(qo, kv, d, fmt, window, num_cus):
    """An infinity or NaN in a key or value reaches the rows that see its token, whatever tile it shares with others:
    chunks, token items of one and two row blocks, split keys, both edges of a window."""
    p = Problem(qo, kv, 8, 2, d, fmt, window=window, num_cus=num_cus)
    o, most, s, lse_most = _expected(p)
    starts = np.concatenate([[0], np.cumsum(qo)])
    for r, (n, L) in enumerate(zip(qo, kv)):
        # the newest token, one amid the new ones, the first of them, and those that rows lose at a window's lower edge
        for token in sorted({L - 1, L - 1 - n // 3, L - n, max(L - n - 40, 0), max(L - n - 68, 0)}):
            for side, what in ((0, math.nan), (1, math.inf if fmt == "bf16" else math.nan)):
                dims = _poison(p, side, r, token, what)
                out, lse = (t.cpu().double() for t in p.run())
                pos = L - n + torch.arange(n)
                rows = starts[r] + torch.arange(n)[(pos >= token) & ((pos <= token + window) | (window < 0))]
                hit = torch.zeros(out.shape, dtype=torch.bool)
                for dim in dims if side else range(d):
                    hit[rows, 4:, dim] = True
                assert not torch.isfinite(out[hit]).any(), f"request {r} token {token} side {side}"
                off = torch.where(hit, 0.0, (out - o).abs() - most)
                assert bool((off <= 0).all()), f"request {r} token {token} side {side}: {off.max():.3g} beyond its bound"
                if side == 0:
                    assert torch.isnan(lse[rows, 4:]).all()
                    lse[rows, 4:] = s[rows, 4:]
                assert bool(((lse - s).abs() <= lse_most).all()), f"request {r} token {token} side {side}: lse"


@pytest.mark.parametrize("fmt", ["bf16", "mxfp4"])
def test_rows_without_a_key_beside_values_that_are_not_finite(fmt):
    """Rows of a cache cut back below its new tokens, in tiles whose only tokens hold infinities: output 0, lse -inf."""
    p = Problem([40, 4], [40, 4], 8, 2, 128, fmt)
    p.v[:] = math.inf
    _poison(p, 1, 0, 0, math.inf)
    p.batch.set_kv_len([25, 2])
    out, lse = (t.cpu() for t in p.run())
    empty = torch.cat([torch.arange(15), 40 + torch.arange(2)])
    assert bool((out[empty] == 0).all()) and bool((lse[empty] == -math.inf).all())
    rest = torch.cat([15 + torch.arange(25), 42 + torch.arange(2)])
    assert not torch.isfinite(out[rest]).any() and torch.isfinite(lse[rest]).all()


@pytest.mark.parametrize("num_cus", [1, 4096])
@pytest.mark.parametrize("fmt,d", [("bf16", 128), ("mxfp8", 64)])
def test_a_query_that_is_no_number_stays_in_its_row(fmt, d, num_cus):
    """Beside it: rows of the same wave, the same token's other heads, other tokens; output over the queries."""
    p = Problem([100, 3, 1], [1500, 300, 2000], 8, 2, d, fmt, num_cus=num_cus, window=400)
    o, most, s, lse_most = _expected(p)
    bad = torch.zeros(p.q.shape[:2], dtype=torch.bool)
    for row, head, what in ((0, 0, math.nan), (17, 5, math.inf), (99, 7, math.nan), (101, 2, -math.inf), (103, 6, math.nan)):
        p.qd[row, head, 3] = what
        bad[row, head] = True
    lse = torch.empty(p.q.shape[:2], device=DEV)
    out, lse = (t.cpu().double() for t in p.attn.run(p.qd, p.cache, out=p.qd, lse=lse))
    torch.cuda.synchronize()
    assert not torch.isfinite(out[bad]).any()
    assert bool(((out - o).abs() <= most)[~bad].all()) and bool(((lse - s).abs() <= lse_most)[~bad].all())
