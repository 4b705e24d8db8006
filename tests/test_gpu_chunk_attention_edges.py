"""PagedChunkAttention at the edges of what it accepts, against the 64-bit form
with the tolerances that test_gpu_chunk_attention.py derives."""
import math

import pytest
import torch

from test_gpu_chunk_attention import Problem

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
