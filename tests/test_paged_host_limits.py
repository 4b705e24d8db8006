"""Host side of the paged-cache operators at the limits of their arguments.  CPU."""
import numpy as np
import pytest

import d2sd


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
