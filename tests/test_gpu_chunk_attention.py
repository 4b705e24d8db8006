"""GPU parity of PagedChunkAttention against the 64-bit form over the values the
cache stands for.

Tolerance, from the arithmetic (u = 2^-24, n visible keys, A = sum_j p_j |v_j|):
  * a score is a 32-bit sum of D exact products: off by D u S, S the row's
    largest sum_i |q_i k_ij| sm_scale; scaling and subtracting the offset add
    4 u |score| <= 4 u S; so p_j is off by e = (D + 4) u S, and exp2 by 4 u;
  * a probability is rounded to bf16 for the second product: half a step, 2^-8;
  * the sums over keys (32-bit) are off by n u of A at most, the sum of
    probabilities by n u of itself, joining partial states by 16 u;
  * the output is rounded to bf16: 2^-8 of it.
So |o - ref| <= 2^-8 |ref| + A (2^-8 + 2 e + 2 n u + 32 u), each row's
|lse - ref| <= 2 e + n u + 32 u + 4 u |ref|."""
import math

import numpy as np
import pytest
import torch

import d2sd
from oracle import paged_oracle as po

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


class Problem:
    """A ragged batch over a cache whose other bytes are NaN patterns (0xFF)."""

    def __init__(self, qo, kv, hq, hkv, d, fmt="bf16", layout="HND", P=16, window=-1, sinks=False, seed=0, extra=0,
                 spread=1.0, pad=0, **plan):
        g = torch.Generator().manual_seed(seed + sum(kv) + hq + d)
        self.qo, self.kv, self.fmt, self.group, self.window, self.d = qo, list(kv), fmt, hq // hkv, window, d
        need = [-(-(n + extra) // P) for n in kv]
        pi = np.concatenate([[0], np.cumsum(need)]).astype(int)
        pages = int(pi[-1]) + 3
        table = torch.randperm(pages, generator=g)[:int(pi[-1])].to(torch.int32)
        self.table = table.to(DEV)
        starts = np.concatenate([[0], np.cumsum(qo)])
        scale = [None, None]
        if fmt == "fp8":
            scale = [torch.rand(hkv, generator=g) * 0.01 + 0.008, torch.rand(hkv, generator=g) * 0.01 + 0.008]
        self.cache = d2sd.PagedKVCache.allocate(pages, P, hkv, d, fmt, kv_layout=layout, device=DEV,
                                                k_scale=None if scale[0] is None else scale[0].to(DEV),
                                                v_scale=None if scale[1] is None else scale[1].to(DEV))
        c = self.cache
        for t in (c.k_pool, c.v_pool, *((c.k_scale, c.v_scale) if fmt.startswith("mx") else ())):
            t.view(torch.uint8).fill_(0xFF)
        # fill every request's cache through the write, as tokens that are all new
        total = sum(kv)
        self.k, self.v = (torch.randn(total, hkv, d, generator=g) * spread).to(torch.bfloat16), \
            torch.randn(total, hkv, d, generator=g).to(torch.bfloat16)
        fill = d2sd.PagedBatch(np.concatenate([[0], np.cumsum(kv)]), kv, pi, self.table, P, device=DEV)
        c.write(self.k.to(DEV), self.v.to(DEV), fill)
        self.batch = d2sd.PagedBatch(starts, kv, pi, self.table, P, device=DEV)
        self.q = torch.randn(int(starts[-1]) + pad, hq, d, generator=g).to(torch.bfloat16)
        self.qd = self.q.to(DEV)
        self.sinks = torch.randn(hq, generator=g) if sinks else None
        self.attn = d2sd.PagedChunkAttention().plan(
            self.batch, hq, hkv, d, kv_format=fmt, window_left=window,
            sinks=None if self.sinks is None else self.sinks.to(DEV), **plan)
        self.scale = plan.get("sm_scale") or d ** -0.5
        val = lambda x, s: po.values_ref(*po.quantise_ref(x, fmt, s), fmt, s)  # noqa: E731
        self.kr, self.vr = val(self.k, scale[0]), val(self.v, scale[1])

    def run(self, **kw):
        return self.attn.run(self.qd, self.cache, **kw)

    def check(self, out, lse, kv=None, base2=False):
        out, lse = out.cpu().double(), lse.cpu().double() * (math.log(2.0) if base2 else 1.0)
        q0 = k0 = 0
        for r, n in enumerate(self.qo):
            L, full = (self.kv if kv is None else kv)[r], self.kv[r]
            k, v = self.kr[k0:k0 + L], self.vr[k0:k0 + L]
            o, s, A, size = po.attention_ref(self.q[q0:q0 + n], k, v, L - n, self.group, self.scale, self.window, self.sinks)
            e = (self.d + 4) * U * size
            bound = 2.0 ** -8 * o.abs() + A * (2.0 ** -8 + 2 * e + 2 * L * U + 32 * U)[..., None]
            got = out[q0:q0 + n]
            assert torch.isfinite(got).all(), f"request {r}"
            off = (got - o).abs() - bound - 1e-30
            assert not n or off.max() <= 0, f"request {r}: {off.max():.3g} beyond its bound at {np.unravel_index(int(off.argmax()), off.shape)}"
            gl = lse[q0:q0 + n]
            empty = torch.isinf(s)
            assert torch.equal(empty, torch.isinf(gl)) and bool((got[empty] == 0).all()), f"request {r}: rows without a key"
            dl = (gl - s)[~empty].abs() - (2 * e + L * U + 32 * U + 4 * U * s.abs())[~empty]
            assert not dl.numel() or dl.max() <= 0, f"request {r}: lse {dl.max():.3g} beyond its bound"
            q0, k0 = q0 + n, k0 + full


def run_and_check(*a, **kw):
    p = Problem(*a, **kw)
    out, lse = p.run()
    torch.cuda.synchronize()
    p.check(out, lse, base2=kw.get("lse_base2", False))
    return p, out, lse


FORMATS = ["bf16", "fp8", "mxfp8", "mxfp4"]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("layout,P", [("HND", 16), ("NHD", 64), ("HND", 1)])
@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 128), (16, 2, 64)])
def test_tokens(fmt, layout, P, hq, hkv, d):
    """Decoding: one token of requests from one key to a few thousand."""
    run_and_check([1] * 8, [1, 2, 31, 32, 33, 255, 1000, 2500], hq, hkv, d, fmt, layout, P)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("layout,P", [("HND", 16), ("NHD", 128)])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (16, 2, 64)])
def test_chunks(fmt, layout, P, hq, hkv, d):
    """Chunks of prompts on both sides of the row tiles (32 and 256 packed rows), whole prompts among them."""
    run_and_check([65, 9, 8, 64, 130], [65, 500, 8, 1100, 131], hq, hkv, d, fmt, layout, P)


@pytest.mark.parametrize("hq,hkv,d", [(7, 1, 128), (28, 4, 128), (5, 5, 64), (12, 1, 64), (33, 1, 128), (64, 1, 64)])
def test_head_groups(hq, hkv, d):
    """Group sizes that divide nothing, one head per kv head, and more than a token item's 32 rows."""
    run_and_check([1, 3, 70], [100, 77, 300], hq, hkv, d, "mxfp8")


@pytest.mark.parametrize("window", [0, 1, 5, 63, 64, 127, 1000])
@pytest.mark.parametrize("fmt,d", [("bf16", 64), ("mxfp4", 128)])
def test_windows(window, fmt, d):
    run_and_check([1, 40, 100, 2], [700, 650, 100, 66], 8, 2, d, fmt, window=window, sinks=True)


@pytest.mark.parametrize("num_cus,max_splits", [(4096, 0), (256, 1), (64, 7)])
@pytest.mark.parametrize("fmt,d", [("bf16", 128), ("fp8", 64), ("mxfp4", 128)])
def test_splits(num_cus, max_splits, fmt, d):
    """Plans that split keys finely, not at all, and between; with sinks, base 2 and a window over some of it."""
    for window in (-1, 900):
        run_and_check([1, 300, 12], [3000, 2500, 2049], 8, 2, d, fmt, window=window, sinks=True, num_cus=num_cus,
                      max_splits=max_splits, lse_base2=True)


def test_sharp_and_flat_scores():
    """Scores of +-300 (one key takes all), and equal ones."""
    run_and_check([1, 50], [400, 300], 8, 2, 128, "bf16", spread=30.0)
    run_and_check([1, 50], [400, 300], 8, 2, 128, "mxfp8", spread=1e-3)


def test_rows_without_a_key_and_empty_requests():
    """More new tokens than cached keys (after a cache was cut back), requests without tokens or keys."""
    p = Problem([4, 0, 3, 40, 0], [4, 5, 3, 60, 0], 8, 2, 128, "mxfp8", sinks=True, num_cus=2048)
    for lens in ([1, 5, 0, 25, 0], [4, 5, 3, 60, 0], [0, 0, 0, 0, 0]):
        p.batch.set_kv_len(lens)
        out, lse = p.run()
        torch.cuda.synchronize()
        # (a cache cut back to L keeps its first L tokens)
        p.check(out, lse, kv=lens)
    none = Problem([], [], 8, 2, 64)
    assert none.run()[0].shape == (0, 8, 64)


def test_strides_padding_and_given_outputs():
    """q inside a fused projection, outputs with gaps; rows behind the last request stay as they were."""
    p = Problem([3, 50], [40, 90], 8, 2, 64, "mxfp8", pad=5)
    T = 53
    fused = torch.randn(T + 5, 12, 64).to(torch.bfloat16).to(DEV)
    fused[:, 2:10] = p.qd
    hold = torch.full((T + 5, 9, 64), 3.0, dtype=torch.bfloat16, device=DEV)
    ls = torch.full((T + 5, 9), 4.0, device=DEV)
    out, lse = p.attn.run(fused[:, 2:10], p.cache, out=hold[:, 1:], lse=ls[:, 1:], workspace=p.attn.workspace())
    torch.cuda.synchronize()
    p.check(out[:T], lse[:T])
    assert bool((hold[T:] == 3.0).all() and (ls[T:] == 4.0).all() and (hold[:, 0] == 3.0).all() and (ls[:, 0] == 4.0).all())
    out2, lse2 = p.run()
    assert torch.equal(out2[:T], out[:T]) and bool((out2[T:] == 0).all()) and bool((lse2[T:] == -math.inf).all())


def test_same_bits_every_time_and_at_once_on_two_streams():
    p = Problem([1, 200], [9000, 4000], 8, 2, 128, "mxfp8")
    assert p.attn.info.num_merges > 0
    ref = p.run()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            got.append(p.run())
    torch.cuda.synchronize()
    for o, l in got:
        assert torch.equal(o, ref[0]) and torch.equal(l, ref[1])


@pytest.mark.parametrize("fmt", ["bf16", "mxfp4"])
def test_a_captured_step_replays_while_caches_grow(fmt):
    """write + attention of one token a request, lengths advanced on the device."""
    p = Problem([1, 1, 2], [300, 40, 1000], 8, 2, 128, fmt, extra=64)
    g = torch.Generator().manual_seed(9)
    kn, vn = (torch.zeros(4, 2, 128, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    out, lse = torch.empty_like(p.qd), torch.empty(4, 8, device=DEV)
    ws = p.attn.workspace()
    graph = d2sd.HipGraph()
    with graph.capture():
        p.cache.write(kn, vn, p.batch)
        p.attn.run(p.qd, p.cache, out=out, lse=lse, workspace=ws)
    held = [[p.kr[:300], p.vr[:300]], [p.kr[300:340], p.vr[300:340]], [p.kr[340:], p.vr[340:]]]
    for step in range(4):
        lens = [300 + 1 + step, 40 + 1 + step, 1000 + 2 + 2 * step]
        x = torch.randn(2, 4, 2, 128, generator=g).to(torch.bfloat16)
        val = [po.values_ref(*po.quantise_ref(t, fmt), fmt) for t in x]
        for r, (a, b) in enumerate([(0, 1), (1, 2), (2, 4)]):
            held[r] = [torch.cat([held[r][s], val[s][a:b]]) for s in (0, 1)]
        kn.copy_(x[0])
        vn.copy_(x[1])
        p.batch.set_kv_len(lens)
        p.qd.copy_(torch.randn(p.q.shape, generator=g).to(torch.bfloat16))
        p.q = p.qd.cpu()
        graph.replay()
        torch.cuda.synchronize()
        p.kv = lens
        p.kr, p.vr = (torch.cat([h[s] for h in held]) for s in (0, 1))
        p.check(out, lse)
        eager = p.run()
        assert torch.equal(eager[0], out) and torch.equal(eager[1], lse)


FORMS = {"eight waves": 0, "four waves": 1, "tokens": 2}


@pytest.mark.parametrize("num_cus", [1, 4096])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("d", [64, 128])
def test_row_counts_around_the_tiles(d, fmt, num_cus):
    """One head per kv head, so rows are tokens: both sides of 16 and 32 (token items) and of 128 and 256 (tile items of
    four and of eight waves); both workgroup sizes of heads of 128."""
    rows = [1, 15, 16, 17, 31, 32, 33, 127, 128, 129, 255, 256, 257, 1024]
    p, _, _ = run_and_check(rows, [n + 37 * (n % 3) for n in rows[:-1]] + [4024], 2, 2, d, fmt, num_cus=num_cus)
    assert p.attn.info.form == FORMS["eight waves" if d == 128 and num_cus == 1 else "four waves"]


@pytest.mark.parametrize("P", [1, 2, 4, 8])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("d", [64, 128])
def test_small_pages(d, fmt, P):
    """Pages of fewer tokens than one load's rows, in items of both kinds."""
    run_and_check([70, 1, 5], [200, 333, 64], 8, 2, d, fmt, "NHD" if P == 2 else "HND", P)


@pytest.mark.parametrize("fmt", FORMATS)
def test_large_pages_and_long_caches(fmt):
    """Token tiles whose rows share pages wherever the window and the cache's end leave them whole."""
    for window in (-1, 1000, 31):
        run_and_check([1, 1, 4, 1], [4000, 4001, 2049, 30], 8, 2, 64, fmt, "HND", 64, window=window)
        run_and_check([1, 1, 4, 1], [4000, 4001, 2049, 30], 8, 2, 128, fmt, "NHD", 256, window=window)


def test_a_captured_run_holds_its_own_outputs_and_workspace():
    """run() without outputs or workspace inside a capture; eager runs, allocations and synchronisations between the
    replays."""
    p = Problem([1, 60], [6000, 3000], 8, 2, 128, "mxfp8")
    assert p.attn.info.num_merges > 0
    graph = d2sd.HipGraph()
    with graph.capture():
        out, lse = p.run()
    g = torch.Generator().manual_seed(12)
    for _ in range(4):
        p.qd.copy_(torch.randn(p.q.shape, generator=g).to(torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        eager = p.run()
        fill = [torch.full((1 << 20,), float("nan"), device=DEV) for _ in range(8)]
        torch.cuda.synchronize()
        assert torch.equal(eager[0], out) and torch.equal(eager[1], lse)
        del fill
    p.q = p.qd.cpu()
    p.check(out, lse)


def test_a_side_stream_orders_write_and_attention():
    """All of a step on a stream that is not the default one."""
    p = Problem([3, 40], [300, 700], 8, 2, 128, "mxfp4")
    ref = p.run()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    x = torch.randn(43, 2, 128).to(torch.bfloat16).to(DEV)
    with torch.cuda.stream(side):
        p.cache.write(x, x, p.batch)
        a = p.run()
        k, v = p.cache.read(p.batch, new_only=True)
    side.synchronize()
    b = p.run()
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and not torch.equal(a[0], ref[0])
    want = po.values_ref(*po.quantise_ref(x.cpu(), "mxfp4"), "mxfp4").to(torch.bfloat16)
    assert torch.equal(k.cpu(), want) and torch.equal(v.cpu(), want)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 128), (64, 8, 64)])
def test_reads_larger_than_the_caches_give_the_same_bits(fmt, hq, hkv, d):
    """Tokens over more than 128 MB of keys and values: read past the caches, and as smaller batches are read."""
    g = torch.Generator().manual_seed(17)
    row = {"bf16": 2 * d, "mxfp4": d // 2}.get(fmt, d)
    P, R = 16, 12
    L = [-(-150 * 2 ** 20 // (R * 2 * hkv * row)) + 61 * r for r in range(R)]
    pi = np.concatenate([[0], np.cumsum([-(-n // P) for n in L])]).astype(int)
    table = torch.randperm(int(pi[-1]), generator=g).to(torch.int32)
    scale = dict(k_scale=torch.full((hkv,), 0.01, device=DEV), v_scale=torch.full((hkv,), 0.01, device=DEV)) if fmt == "fp8" else {}
    c = d2sd.PagedKVCache.allocate(int(pi[-1]), P, hkv, d, fmt, device=DEV, **scale)
    for t in (c.k_pool, c.v_pool):
        if fmt == "bf16":
            t.normal_()
        else:  # any codes but NaN
            t.view(torch.uint8).random_(0, 256).bitwise_and_(0xFF if fmt == "mxfp4" else 0xBF)
    if fmt.startswith("mx"):
        for t in (c.k_scale, c.v_scale):
            t.random_(118, 124)
    b = d2sd.PagedBatch(np.arange(R + 1), L, pi, table.to(DEV), P)
    q = torch.randn(R, hq, d, generator=g).to(torch.bfloat16).to(DEV)
    a = d2sd.PagedChunkAttention().plan(b, hq, hkv, d, kv_format=fmt)
    assert a.info.form == 3
    past = a.run(q, c)
    a.info.form = 2
    a._info = torch.frombuffer(bytearray(bytes(a.info)), dtype=torch.uint8)
    kept = a.run(q, c)
    torch.cuda.synchronize()
    assert torch.isfinite(past[0]).all() and torch.equal(past[0], kept[0]) and torch.equal(past[1], kept[1])


def test_shared_pages_of_a_common_prefix():
    """Two requests whose tables begin with the same pages."""
    P, g = 16, torch.Generator().manual_seed(1)
    k, v = (torch.randn(64, 2, 64, generator=g).to(torch.bfloat16) for _ in range(2))
    c = d2sd.PagedKVCache.allocate(8, P, 2, 64, "bf16", device=DEV)
    d2sd_b = d2sd.PagedBatch([0, 40, 64], [40, 56], [0, 3, 7], [5, 1, 2, 5, 1, 4, 0], P, device=DEV)
    # request 0's 40 tokens in pages 5, 1, 2; request 1 shares 5 and 1 and brings its last 24 tokens in 4, 0
    c.write(k.to(DEV), v.to(DEV), d2sd_b)
    q = torch.randn(64, 4, 64, generator=g).to(torch.bfloat16)
    out, _ = d2sd.PagedChunkAttention().plan(d2sd_b, 4, 2, 64).run(q.to(DEV), c)
    torch.cuda.synchronize()
    k1, v1 = torch.cat([k[:32], k[40:]]), torch.cat([v[:32], v[40:]])
    for rows, kk, vv, pos0 in ((slice(0, 40), k[:40], v[:40], 0), (slice(40, 64), k1, v1, 32)):
        o, s, A, size = po.attention_ref(q[rows], kk, vv, pos0, 2, 64 ** -0.5)
        bound = 2.0 ** -8 * o.abs() + A * (2.0 ** -8 + (2 * 68 * U * size + 2 * 64 * U + 32 * U)[..., None])
        assert ((out[rows].cpu().double() - o).abs() <= bound).all()


def test_a_cache_of_a_quarter_million_tokens():
    """Keys split as far as a plan goes, and not at all."""
    for kw in (dict(), dict(max_splits=1)):
        run_and_check([1, 9], [250001, 131072], 4, 2, 64, "bf16", P=64, **kw)


def test_a_page_table_in_place_is_read_at_each_call():
    """Pages moved by device writes to the table and the pools: the same batch and plan follow."""
    p = Problem([2, 70], [100, 300], 8, 2, 64, "mxfp8")
    ref = p.run()
    torch.cuda.synchronize()
    assert p.batch.page_table.data_ptr() == p.table.data_ptr()
    n = p.cache.num_pages
    perm = torch.randperm(n, generator=torch.Generator().manual_seed(2)).to(DEV)
    for t in (p.cache.k_pool, p.cache.v_pool, p.cache.k_scale, p.cache.v_scale):
        old = t.view(torch.uint8).clone()
        t.view(torch.uint8)[perm] = old  # page i moves to perm[i]
    p.table.copy_(perm[p.table.long()].to(torch.int32))
    got = p.run()
    k, v = p.cache.read(p.batch)
    torch.cuda.synchronize()
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    assert torch.equal(k.cpu().double(), p.kr) and torch.equal(v.cpu().double(), p.vr)


def test_offsets_past_32_bits():
    """Pages beyond 4 GiB of a pool (token-major, so that rows of one head lie far apart as well)."""
    P, hkv, d, L = 16, 8, 128, 100
    pages = 2 ** 32 // (P * hkv * d * 2) + 40
    c = d2sd.PagedKVCache.allocate(pages, P, hkv, d, "bf16", kv_layout="NHD", device=DEV)
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(L, hkv, d, generator=g).to(torch.bfloat16) for _ in range(2))
    table = [pages - 1 - i for i in range(7)]
    c.write(k.to(DEV), v.to(DEV), d2sd.PagedBatch([0, L], [L], [0, 7], table, P, device=DEV))
    for n in (1, 50):
        q = torch.randn(n, 16, d, generator=g).to(torch.bfloat16)
        b = d2sd.PagedBatch([0, n], [L], [0, 7], table, P, device=DEV)
        out, _ = d2sd.PagedChunkAttention().plan(b, 16, hkv, d).run(q.to(DEV), c)
        torch.cuda.synchronize()
        o, s, A, size = po.attention_ref(q, k, v, L - n, 2, d ** -0.5)
        bound = 2.0 ** -8 * o.abs() + A * (2.0 ** -8 + (2 * 132 * U * size + 2 * L * U + 32 * U)[..., None])
        assert ((out.cpu().double() - o).abs() <= bound).all()


def test_page_ids_outside_the_pool_stay_in_bounds():
    """Clamped like the verify attention's: a wrong page is read, never memory outside the pool."""
    c = d2sd.PagedKVCache.allocate(4, 16, 2, 64, "mxfp8", device=DEV)
    for t in (c.k_pool, c.v_pool, c.k_scale, c.v_scale):
        t.view(torch.uint8).fill_(0x38)
    b = d2sd.PagedBatch([0, 1], [64], [0, 4], [0, 2 ** 31 - 1, -5, 4], 16, device=DEV)
    out, lse = d2sd.PagedChunkAttention().plan(b, 4, 2, 64, kv_format="mxfp8").run(
        torch.zeros(1, 4, 64, dtype=torch.bfloat16, device=DEV), c)
    torch.cuda.synchronize()
    assert torch.isfinite(out).all() and (lse - math.log(64)).abs().max() < 1e-5


def test_refusals_on_the_device():
    p = Problem([2], [20], 8, 2, 64, "mxfp8")
    q = p.qd
    for bad, err in (((q.float(), p.cache), TypeError), ((q[:1], p.cache), ValueError), ((q[:, :4], p.cache), ValueError),
                     ((q.cpu(), p.cache), ValueError)):
        with pytest.raises(err):
            p.attn.run(*bad)
    other = d2sd.PagedKVCache.allocate(2, 16, 2, 64, "mxfp4", device=DEV)
    with pytest.raises(ValueError):
        p.attn.run(q, other)
    with pytest.raises(ValueError):
        p.attn.run(q, d2sd.PagedKVCache.allocate(2, 32, 2, 64, "mxfp8", device=DEV))
    for kw in (dict(out=torch.empty_like(q)[:1]), dict(lse=torch.empty(2, 8, dtype=torch.float64, device=DEV)),
               dict(out=torch.empty_like(q).cpu())):
        with pytest.raises(ValueError):
            p.attn.run(q, p.cache, **kw)
    s = Problem([1], [20000], 8, 2, 64, "mxfp8")
    assert s.attn.info.workspace_bytes > 0
    with pytest.raises(ValueError, match="workspace"):
        s.attn.run(s.qd, s.cache, workspace=torch.empty(16, dtype=torch.uint8, device=DEV))
