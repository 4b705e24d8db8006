"""PagedKVCache.read and PagedChunkAttention.plan after a batch's lengths moved."""
import numpy as np
import pytest
import torch

import d2sd
from oracle import paged_oracle as po

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _caches(fmt, P, hkv, d, room, seed):
    """Requests whose caches are filled as far as their pages go; their values as they read back."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // P) for n in room]
    pi = np.concatenate([[0], np.cumsum(need)])
    table = torch.randperm(int(pi[-1]), generator=g).to(torch.int32).to(DEV)
    scale = torch.full((hkv,), 0.02, device=DEV) if fmt == "fp8" else None
    c = d2sd.PagedKVCache.allocate(int(pi[-1]), P, hkv, d, fmt, k_scale=scale, v_scale=scale, device=DEV)
    total = sum(room)
    k, v = (torch.randn(total, hkv, d, generator=g).to(torch.bfloat16) for _ in range(2))
    c.write(k.to(DEV), v.to(DEV), d2sd.PagedBatch(np.concatenate([[0], np.cumsum(room)]), room, pi, table, P))
    sc = None if scale is None else scale.cpu()
    vals = [po.values_ref(*po.quantise_ref(x, fmt, sc), fmt, sc).to(torch.bfloat16) for x in (k, v)]
    start = np.concatenate([[0], np.cumsum(room)])
    rows = lambda lens: torch.cat([torch.arange(start[r], start[r] + n) for r, n in enumerate(lens)])  # noqa: E731
    return c, pi, table, vals, rows


@pytest.mark.parametrize("fmt", ["bf16", "fp8", "mxfp8", "mxfp4"])
def test_a_full_read_follows_set_kv_len(fmt):
    """Grown, cut back, emptied and grown again: every row of the lengths as they are, no others; given outputs too."""
    room = [40, 100, 33]
    c, pi, table, vals, rows = _caches(fmt, 16, 2, 64, room, 3)
    b = d2sd.PagedBatch([0, 1, 1, 3], [20, 50, 33], pi, table, 16)
    for lens in ([20, 50, 33], [21, 51, 33], [40, 100, 33], [3, 0, 17], [0, 0, 0], [40, 1, 2]):
        b.set_kv_len(lens)
        got = c.read(b)
        given = tuple(torch.full((sum(lens) + 2, 2, 64), 5.0, dtype=torch.bfloat16, device=DEV) for _ in range(2))
        c.read(b, out=given)
        torch.cuda.synchronize()
        for x, y, want in zip(got, given, vals):
            assert torch.equal(x.cpu(), want[rows(lens)]) and torch.equal(y[:sum(lens)].cpu(), want[rows(lens)])
            assert bool((y[sum(lens):] == 5.0).all())


def test_captured_reads_keep_their_rows_and_later_ones_follow():
    c, pi, table, vals, rows = _caches("mxfp8", 16, 2, 64, [40, 100], 4)
    b = d2sd.PagedBatch([0, 1, 2], [20, 50], pi, table, 16)
    out = tuple(torch.zeros(70, 2, 64, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    b.prepare_read()
    graph = d2sd.HipGraph()
    with graph.capture():
        c.read(b, out=out)
    for lens in ([30, 60], [40, 100], [20, 50]):
        b.set_kv_len(lens)
        for t in out:
            t.zero_()
        graph.replay()
        now = c.read(b)
        torch.cuda.synchronize()
        for x, y, want in zip(out, now, vals):
            assert torch.equal(x.cpu(), want[rows([20, 50])]) and torch.equal(y.cpu(), want[rows(lens)])


@pytest.mark.parametrize("hkv,d", [(2, 64), (8, 128)])
@pytest.mark.parametrize("fmt", ["bf16", "fp8", "mxfp8", "mxfp4"])
def test_rows_that_the_cache_does_not_hold_are_zero(fmt, hkv, d):
    """Tensors that a read allocates (in memory that held something else): zeros for tokens past a length that a device
    write shortened, before a cache's start, and in pages outside the pool; the others as they are."""
    room = [40, 100, 33]
    c, pi, table, vals, rows = _caches(fmt, 16, hkv, d, room, 5)
    b = d2sd.PagedBatch([0, 5, 5, 25], room, pi, table, 16)
    b.prepare_read().prepare_read(new_only=True)
    lens = [38, 61, 12]
    b.kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
    b.page_table[1] = 2 ** 31 - 1       # tokens 16 .. 31 of request 0
    b.page_table[int(pi[1])] = -1       # 0 .. 15 of request 1
    held = [torch.arange(n) < m for n, m in zip(room, lens)]
    held[0][16:32] = False
    held[1][:16] = False
    full = torch.cat(held)
    # new tokens of requests 0 and 2: 33 .. 37, and -8 .. 11 (of which 8 have no place)
    new = torch.cat([torch.arange(33, 38), torch.full((8,), -1), 140 + torch.arange(12)])
    for new_only in (False, True):
        n = b.total_q if new_only else b.total_kv
        for _ in range(3):
            stale = [torch.full((n, hkv, d), 7.0, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
            torch.cuda.synchronize()
            del stale
            got = c.read(b, new_only=new_only)
            torch.cuda.synchronize()
            for x, want in zip(got, vals):
                want = torch.where((new >= 0)[:, None, None], want[new], 0) if new_only else \
                    torch.where(full[:, None, None], want, 0)
                assert torch.equal(x.cpu(), want.to(torch.bfloat16))
            del got, x
