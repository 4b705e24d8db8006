"""PagedChunkAttention at the edges of what it accepts, against the 64-bit form
with the tolerances that test_gpu_chunk_attention.py derives."""
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
