"""What a batch, a plan and a cache hold for their caller, used on another stream
than the one that they were made on and let go of while that is under way."""
import numpy as np
import pytest
import torch

import d2sd

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _setup(fmt):
    P, hkv, d = 16, 2, 64
    qo, kv = [1, 40], [5000, 700]
    pi = np.concatenate([[0], np.cumsum([-(-n // P) for n in kv])])
    scale = torch.full((hkv,), 0.02, device=DEV) if fmt == "fp8" else None
    c = d2sd.PagedKVCache.allocate(int(pi[-1]), P, hkv, d, fmt, k_scale=scale, v_scale=scale, device=DEV)
    for t in (c.k_pool, c.v_pool, c.k_scale, c.v_scale):
        if t is not None and t is not scale:
            t.view(torch.uint8).fill_(0x38)
    table = np.random.default_rng(1).permutation(int(pi[-1])).astype(np.int32)
    b = d2sd.PagedBatch([0, 1, 41], kv, pi, table, P, device=DEV)
    a = d2sd.PagedChunkAttention().plan(b, 8, hkv, d, kv_format=fmt, sinks=torch.zeros(8, device=DEV))
    b.prepare_read().prepare_read(new_only=True)
    return c, b, a


def _step(c, b, a, q, x):
    c.write(x, -x, b)
    out = a.run(q, c)
    return [*out, *c.read(b), *c.read(b, new_only=True)]


@pytest.mark.parametrize("fmt", ["bf16", "fp8", "mxfp8"])
def test_buffers_outlive_their_last_use_on_another_stream(fmt):
    """Plan, token records, read lists, lengths, page table, sinks and pools: their memory goes to nobody else before
    the side stream has come to its end."""
    g = torch.Generator().manual_seed(7)
    q, x = (torch.randn(41, h, 64, generator=g).to(torch.bfloat16).to(DEV) for h in (8, 2))
    ref = _step(*_setup(fmt), q, x)
    c, b, a = _setup(fmt)
    held = [a.plan_dev, b._tokens, b.page_table, a.sinks, c.k_pool, c.v_pool, *b._reads.values()]
    held += [] if fmt == "bf16" else [c.k_scale, c.v_scale]
    # (by storage: the lengths lie behind the token records)
    places = {t.untyped_storage().data_ptr(): t.untyped_storage().nbytes() for t in held}
    assert a.info.num_merges > 0
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(int(1e9))  # some 0.5 s
        got = _step(c, b, a, q, x)
    del held, c, b, a
    # as many tensors of each size as the pool may hand out (none is written to)
    taken = [torch.empty(n, dtype=torch.uint8, device=DEV) for n in places.values() for _ in range(8)]
    assert not side.query(), "the side stream ended before its buffers were let go of"
    spans = [(t.data_ptr(), t.data_ptr() + t.numel()) for t in taken]
    for at, n in places.items():
        assert not [s for s in spans if s[0] < at + n and at < s[1]]
    side.synchronize()
    for u, v in zip(got, ref):
        assert torch.equal(u, v)
    # and then it does come back
    del taken, got
    torch.cuda.synchronize()
    again = [torch.empty(n, dtype=torch.uint8, device=DEV) for n in places.values() for _ in range(8)]
    assert any(s.data_ptr() in places for s in again)


def test_a_re_planned_attention_and_moved_lengths_let_go_safely():
    """plan() and set_kv_len() replace the buffers that a side stream's calls still read."""
    g = torch.Generator().manual_seed(8)
    q, x = (torch.randn(41, h, 64, generator=g).to(torch.bfloat16).to(DEV) for h in (8, 2))
    ref = _step(*_setup("mxfp8"), q, x)
    c, b, a = _setup("mxfp8")
    places = {t.untyped_storage().data_ptr(): t.untyped_storage().nbytes() for t in (a.plan_dev, b._reads[False])}
    torch.cuda.synchronize()
    side, lens = torch.cuda.Stream(), b.kv_len_host.copy()
    with torch.cuda.stream(side):
        torch.cuda._sleep(int(1e9))
        got = _step(c, b, a, q, x)
        done = side.record_event()
    a.plan(b, 8, 2, 64, kv_format="mxfp8", sinks=a.sinks)
    b._host_lengths(lens)  # (what set_kv_len drops, without its write to the lengths in use)
    taken = [torch.empty(n, dtype=torch.uint8, device=DEV) for n in places.values() for _ in range(8)]
    assert not done.query()
    spans = [(t.data_ptr(), t.data_ptr() + t.numel()) for t in [*taken, a.plan_dev]]
    for at, n in places.items():
        assert not [s for s in spans if s[0] < at + n and at < s[1]]
    side.synchronize()
    for u, v in zip(got, ref):
        assert torch.equal(u, v)


def test_read_lists_made_on_another_stream_than_their_batch():
    g = torch.Generator().manual_seed(9)
    x = torch.randn(41, 2, 64, generator=g).to(torch.bfloat16).to(DEV)
    c, b, _ = _setup("mxfp8")
    c.write(x, -x, b)
    ref = c.read(b)
    lens = b.kv_len_host.copy()
    b._host_lengths(lens)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        b.prepare_read()
    at, n = b._reads[False].data_ptr(), b._reads[False].untyped_storage().nbytes()
    side.synchronize()
    torch.cuda._sleep(int(1e9))
    got = c.read(b)
    done = torch.cuda.current_stream().record_event()
    b._host_lengths(lens)
    with torch.cuda.stream(side):
        taken = [torch.empty(n, dtype=torch.uint8, device=DEV) for _ in range(8)]
    assert not done.query()
    assert not [t for t in taken if t.data_ptr() < at + n and at < t.data_ptr() + n]
    torch.cuda.synchronize()
    for u, v in zip(got, ref):
        assert torch.equal(u, v)
