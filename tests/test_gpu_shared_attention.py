"""GPU parity of PagedChunkAttention plans with shared keys against the 64-bit
form over each request's own keys.

Tolerance: that of the chunk attention's tests (its docstring has the
arithmetic), which does not depend on how a row's keys are split and joined.
The pages of what a request shares hold NaN patterns wherever they are not its
group's first request's: nobody reads them."""
import math

import numpy as np
import pytest
import torch

import d2sd
from oracle import paged_oracle as po

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
FORMATS = ["bf16", "fp8", "mxfp8", "mxfp4"]


class Problem:
    """Groups of requests: request r's cache is its group's shared tokens, then its own (own[r] of them)."""

    def __init__(self, groups, prefix, own, new, hq, hkv, d, fmt="bf16", layout="HND", P=16, window=-1, sinks=False, seed=0,
                 extra=0, pad=0, spread=1.0, keep_shared=True, **plan):
        g = torch.Generator().manual_seed(seed + sum(own) + sum(prefix) + hq + d)
        first = np.concatenate([[0], np.cumsum(groups)]).astype(int)
        share = [prefix[i] for i, n in enumerate(groups) for _ in range(n)]
        lead = [first[i] for i, n in enumerate(groups) for _ in range(n)]
        self.kv, self.qo = [a + b for a, b in zip(share, own)], list(new)
        self.fmt, self.group, self.window, self.d, self.hkv, self.P, self.layout = fmt, hq // hkv, window, d, hkv, P, layout
        R = len(self.kv)
        need = [-(-(n + extra) // P) for n in self.kv]
        pi = np.concatenate([[0], np.cumsum(need)]).astype(int)
        pages = int(pi[-1]) + 3
        table = torch.randperm(pages, generator=g)[:int(pi[-1])].to(torch.int32)
        scale = [torch.rand(hkv, generator=g) * 0.01 + 0.008 for _ in range(2)] if fmt == "fp8" else [None, None]
        kw = {} if fmt != "fp8" else dict(k_scale=scale[0].to(DEV), v_scale=scale[1].to(DEV))
        self.cache = c = d2sd.PagedKVCache.allocate(pages, P, hkv, d, fmt, kv_layout=layout, device=DEV, **kw)
        for t in (c.k_pool, c.v_pool, *((c.k_scale, c.v_scale) if fmt.startswith("mx") else ())):
            t.view(torch.uint8).fill_(0xFF)
        x = [(torch.randn(sum(prefix) + sum(own), hkv, d, generator=g) * s).to(torch.bfloat16) for s in (spread, 1.0)]
        self.raw = x
        # written once: a group's shared tokens as its first request's, every request's own behind them
        at, self.rows, pos = 0, [], {}
        for i in range(len(groups)):
            pos[i] = torch.arange(at, at + prefix[i])
            at += prefix[i]
        mine = []
        for r in range(R):
            mine.append(torch.arange(at, at + own[r]))
            at += own[r]
            self.rows.append(torch.cat([pos[int(np.searchsorted(first, r, side="right")) - 1], mine[r]]))
        for r in range(R):
            # (a write of all of the first one's tokens, of the own ones of the others)
            n = self.kv[r] if lead[r] == r else own[r]
            t = self.rows[r][len(self.rows[r]) - n:]
            b = d2sd.PagedBatch([0, n], [self.kv[r]], [0, need[r]], table[pi[r]:pi[r + 1]], P, device=DEV)
            c.write(x[0][t].to(DEV), x[1][t].to(DEV), b)
        # the others' entries for whole shared pages: any page
        for r in range(R):
            if lead[r] != r and groups[int(np.searchsorted(first, r, side="right")) - 1] > 1:
                table[pi[r]:pi[r] + share[r] // P] = 2 ** 30
        self.table = table.to(DEV)
        self.starts = np.concatenate([[0], np.cumsum(new)]).astype(int)
        self.batch = d2sd.PagedBatch(self.starts, self.kv, pi, self.table, P, device=DEV)
        self.q = torch.randn(int(self.starts[-1]) + pad, hq, d, generator=g).to(torch.bfloat16)
        self.qd = self.q.to(DEV)
        self.sinks = torch.randn(hq, generator=g) if sinks else None
        self.attn = d2sd.PagedChunkAttention().plan(
            self.batch, hq, hkv, d, kv_format=fmt, window_left=window, sinks=None if self.sinks is None else self.sinks.to(DEV),
            shared_indptr=first, shared_len=prefix, keep_shared=keep_shared, **plan)
        self.scale = plan.get("sm_scale") or d ** -0.5
        self.kr, self.vr = (po.values_ref(*po.quantise_ref(t, fmt, s), fmt, s) for t, s in zip(x, scale))

    def run(self, **kw):
        return self.attn.run(self.qd, self.cache, **kw)

    def check(self, out, lse, kv=None, base2=False, rows=None):
        out, lse = out.cpu().double(), lse.cpu().double() * (math.log(2.0) if base2 else 1.0)
        for r, n in enumerate(self.qo):
            L = (self.kv if kv is None else kv)[r]
            at, q0 = self.rows[r][:L], int(self.starts[r])
            k, v = self.kr[at], self.vr[at]
            o, s, A, size = po.attention_ref(self.q[q0:q0 + n], k, v, L - n, self.group, self.scale, self.window, self.sinks)
            e = (self.d + 4) * U * size
            bound = 2.0 ** -8 * o.abs() + A * (2.0 ** -8 + 2 * e + 2 * L * U + 32 * U)[..., None]
            got = out[q0:q0 + n]
            assert torch.isfinite(got).all(), f"request {r}"
            off = (got - o).abs() - bound - 1e-30
            assert not n or off.max() <= 0, \
                f"request {r}: {off.max():.3g} beyond its bound at {np.unravel_index(int(off.argmax()), off.shape)}"
            gl = lse[q0:q0 + n]
            empty = torch.isinf(s)
            assert torch.equal(empty, torch.isinf(gl)) and bool((got[empty] == 0).all()), f"request {r}: rows without a key"
            dl = (gl - s)[~empty].abs() - (2 * e + L * U + 32 * U + 4 * U * s.abs())[~empty]
            assert not dl.numel() or dl.max() <= 0, f"request {r}: lse {dl.max():.3g} beyond its bound"


def run_and_check(*a, **kw):
    p = Problem(*a, **kw)
    assert p.attn.info.form & 8
    out, lse = p.run()
    torch.cuda.synchronize()
    p.check(out, lse, base2=kw.get("lse_base2", False))
    return p, out, lse


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("layout,P", [("HND", 16), ("NHD", 64), ("HND", 1)])
@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 128), (16, 2, 64)])
def test_decoding(fmt, layout, P, hq, hkv, d):
    """One token of each of a few requests, own lengths from one key on; groups of every kind of item."""
    run_and_check([4], [515], [1, 2, 31, 200], [1] * 4, hq, hkv, d, fmt, layout, P)
    run_and_check([7, 1, 3], [300, 40, 1000], [1, 2, 31, 200, 33, 1, 64, 50, 7, 90, 3], [1] * 11, hq, hkv, d, fmt, layout, P)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (16, 2, 64)])
def test_many_requests(fmt, hq, hkv, d):
    """More rows than a row tile of either workgroup (128 and 256), of requests that cross its border."""
    n = 83
    run_and_check([n], [700], [1 + 3 * (i % 17) for i in range(n)], [1 + (i % 3 == 0 and i % 17 > 0) for i in range(n)], hq, hkv, d,
                  fmt)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("layout,P", [("HND", 16), ("NHD", 128)])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (16, 2, 64)])
def test_chunks(fmt, layout, P, hq, hkv, d):
    """Chunks of prompts and single tokens behind the same document, empty requests among them."""
    run_and_check([6], [333], [65, 9, 8, 80, 300, 5], [65, 9, 1, 64, 130, 0], hq, hkv, d, fmt, layout, P)


@pytest.mark.parametrize("hq,hkv,d", [(7, 1, 128), (28, 4, 128), (5, 5, 64), (12, 1, 64), (33, 1, 128), (64, 1, 64)])
def test_head_groups(hq, hkv, d):
    run_and_check([3, 2], [200, 100], [40, 3, 70, 9, 1], [1, 3, 70, 2, 1], hq, hkv, d, "mxfp8")


@pytest.mark.parametrize("window", [0, 1, 5, 63, 64, 127, 260, 400, 1000])
@pytest.mark.parametrize("fmt,d", [("bf16", 64), ("mxfp4", 128), ("mxfp8", 64)])
def test_windows(window, fmt, d):
    """Windows that leave all, a part or nothing of what is shared, for all rows or some of them."""
    run_and_check([4, 8], [300, 250], [1, 50, 100, 2, 1, 2, 3, 70, 5, 300, 9, 20], [1, 40, 100, 2, 1, 2, 3, 50, 5, 1, 9, 3], 8, 2, d,
                  fmt, window=window, sinks=True)


@pytest.mark.parametrize("num_cus,max_splits", [(4096, 0), (256, 1), (64, 7)])
@pytest.mark.parametrize("fmt,d", [("bf16", 128), ("fp8", 64), ("mxfp4", 128)])
def test_splits(num_cus, max_splits, fmt, d):
    for window in (-1, 900):
        run_and_check([3, 2], [2000, 1500], [1000, 500, 49, 700, 300], [1, 300, 12, 20, 1], 8, 2, d, fmt, window=window, sinks=True,
                      num_cus=num_cus, max_splits=max_splits, lse_base2=True)


@pytest.mark.parametrize("num_cus", [1, 4096])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("d", [64, 128])
def test_row_counts_around_the_tiles(d, fmt, num_cus):
    """Groups whose rows lie on both sides of 16, 32, 128 and 256."""
    groups = [2, 15, 16, 17, 2, 2, 2, 2]
    own = [1 + i % 5 for i in range(50)] + [3, 31, 16, 17, 128, 129, 200, 4024]
    new = [1] * 50 + [2, 30, 16, 16, 127, 1, 200, 1024]
    run_and_check(groups, [65, 40, 33, 64, 31, 100, 129, 1], own, new, 2, 2, d, fmt, num_cus=num_cus)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("window", [-1, 1500])
def test_workgroups_of_eight_waves(fmt, window):
    p, _, _ = run_and_check([4], [2000], [1500, 900, 400, 1], [500, 257, 300, 1], 8, 2, 128, fmt, num_cus=1, window=window)
    assert p.attn.info.form == 8


@pytest.mark.parametrize("P", [1, 2, 4, 8])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("d", [64, 128])
def test_small_pages(d, fmt, P):
    run_and_check([2, 20], [133, 70], [70, 1] + [3 + i for i in range(20)], [70, 1] + [1] * 20, 8, 2, d, fmt,
                  "NHD" if P == 2 else "HND", P)


def test_sharp_and_flat_scores():
    run_and_check([2, 12], [200, 200], [1, 50] + [9] * 12, [1, 50] + [1] * 12, 8, 2, 128, "bf16", spread=30.0)
    run_and_check([2, 12], [200, 200], [1, 50] + [9] * 12, [1, 50] + [1] * 12, 8, 2, 128, "mxfp8", spread=1e-3)


@pytest.mark.parametrize("window", [-1, 40])
@pytest.mark.parametrize("fmt", ["bf16", "mxfp8"])
def test_caches_cut_back(fmt, window):
    """Lengths below what is shared, below the new tokens, of nothing; the same plan."""
    p = Problem([3, 14, 1], [90, 65, 0], [30, 4, 9] + [2] * 14 + [6], [20, 4, 9] + [1] * 14 + [6], 8, 2, 128, fmt, sinks=True,
                window=window, num_cus=2048)
    full = p.kv
    for lens in ([100, 90, 70] + full[3:], [10, 94, 3] + [i for i in range(14)] + [3], [0] * 18, [119, 1, 99] + [66] * 14 + [0], full):
        p.batch.set_kv_len(lens)
        out, lse = p.run()
        torch.cuda.synchronize()
        p.check(out, lse, kv=lens)


def test_the_result_of_a_plan_without_groups():
    """Where every request's own table leads to the shared tokens too: both plans within the bound of one another."""
    for fmt, new in (("bf16", [1] * 5), ("mxfp4", [1, 40, 3, 1, 200])):
        p = Problem([5], [600], [80, 40, 3, 33, 200], new, 8, 2, 64, fmt)
        pi = p.batch.page_indptr_host
        for r in range(1, 5):  # whole shared pages: the first request's; the last, shared in part: its own copy
            p.batch.page_table[pi[r]:pi[r] + 600 // 16] = p.batch.page_table[:600 // 16]
            for t in (p.cache.k_pool, p.cache.v_pool, p.cache.k_scale, p.cache.v_scale):
                if t is not None:
                    t.view(torch.uint8)[p.table[pi[r] + 37].long(), :, :8] = t.view(torch.uint8)[p.table[37].long(), :, :8]
        out, lse = p.run()
        plain, plse = d2sd.PagedChunkAttention().plan(p.batch, 8, 2, 64, kv_format=fmt).run(p.qd, p.cache)
        torch.cuda.synchronize()
        p.check(out, lse)
        p.check(plain, plse)


def test_strides_padding_and_given_outputs():
    p = Problem([2, 3], [50, 40], [3, 50, 1, 2, 3], [3, 50, 1, 1, 2], 8, 2, 64, "mxfp8", pad=5)
    T = 57
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


@pytest.mark.parametrize("fmt", ["bf16", "mxfp8"])
def test_same_bits_every_time_and_at_once_on_two_streams(fmt):
    p = Problem([40, 2], [3000, 2000], [17] * 40 + [100, 300], [1] * 40 + [80, 1], 8, 2, 128, fmt)
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
    """append + attention of one or two tokens a request; lengths advance on the device."""
    own, new = [30, 4, 100], [1, 1, 2]
    p = Problem([3], [205], own, new, 8, 2, 128, fmt, extra=64)
    g = torch.Generator().manual_seed(9)
    f, s = d2sd.rotary_frequencies(128)
    fd = f.to(DEV)
    qkv = torch.zeros(4, 12, 128, dtype=torch.bfloat16, device=DEV)
    q_out, out, lse = torch.empty(4, 8, 128, dtype=torch.bfloat16, device=DEV), torch.empty_like(p.qd), torch.empty(4, 8, device=DEV)
    ws = p.attn.workspace()
    graph = d2sd.HipGraph()
    with graph.capture():
        p.cache.append(qkv[:, :8], qkv[:, 8:10], qkv[:, 10:], p.batch, fd, q_out=q_out)
        p.attn.run(q_out, p.cache, out=out, lse=lse, workspace=ws)
    for step in range(4):
        lens = [205 + own[0] + 1 + step, 205 + own[1] + 1 + step, 205 + own[2] + 2 + 2 * step]
        qkv.copy_(torch.randn(4, 12, 128, generator=g).to(torch.bfloat16))
        p.batch.set_kv_len(lens)
        graph.replay()
        torch.cuda.synchronize()
        # what the cache holds now of the new tokens joins the reference's keys
        k, v = (t.cpu().double() for t in p.cache.read(p.batch, new_only=True))
        at = torch.arange(len(p.kr), len(p.kr) + 4)
        p.kr, p.vr = torch.cat([p.kr, k]), torch.cat([p.vr, v])
        for r, (a, b) in enumerate([(0, 1), (1, 2), (2, 4)]):
            p.rows[r] = torch.cat([p.rows[r], at[a:b]])
        p.q, p.kv = q_out.cpu(), lens
        p.check(out, lse)
        eager = p.attn.run(q_out, p.cache)
        assert torch.equal(eager[0], out) and torch.equal(eager[1], lse)


def test_a_captured_run_holds_what_it_uses():
    """Outputs and workspace of its own inside a capture; the plan made again for other groups between the replays."""
    p = Problem([3, 30], [1000, 700], [50, 3, 9] + [5] * 30, [20, 1, 2] + [1] * 30, 8, 2, 128, "mxfp8")
    graph = d2sd.HipGraph()
    with graph.capture():
        out, lse = p.run()
    want = p.run()
    p.attn.plan(p.batch, 8, 2, 128, kv_format="mxfp8")
    g = torch.Generator().manual_seed(12)
    for i in range(4):
        fill = [torch.full((1 << 20,), float("nan"), device=DEV) for _ in range(8)]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(want[0], out) and torch.equal(want[1], lse)
        del fill
    del g
    p.check(out, lse)


NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("value", [NAN, INF])
@pytest.mark.parametrize("fmt", ["bf16", "mxfp8"])
@pytest.mark.parametrize("window", [-1, 60])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (16, 2, 64)])
def test_values_that_are_not_finite_reach_the_rows_that_see_them(value, fmt, window, hq, hkv, d):
    """In a shared value and in an own one; rows of items of both kinds, some of which do not see the token."""
    groups, prefix = [3, 20], [100, 90]
    own, new = [30, 5, 2] + [1 + 7 * (i % 4) for i in range(20)], [20, 5, 2] + [1] * 20
    p = Problem(groups, prefix, own, new, hq, hkv, d, fmt, window=window)
    clean = p.run()
    torch.cuda.synchronize()
    # (request, position) of the tokens; shared ones reach the whole group
    for r, pos in ((0, 80), (3, 40), (0, 110), (5, 90 + 2), (1, 99)):
        q = Problem(groups, prefix, own, new, hq, hkv, d, fmt, window=window)
        slot = p.table[p.batch.page_indptr_host[r if pos >= (100 if r < 3 else 90) else (0 if r < 3 else 3)] + pos // 16].long()
        if fmt == "bf16":
            q.cache.v_pool[slot, :, pos % 16] = value
        else:
            q.cache.v_scale[slot, :, pos % 16] = 255
        out, lse = q.run()
        torch.cuda.synchronize()
        hit = torch.zeros(out.shape[0], dtype=torch.bool)
        for m in range(23):
            same = m == r or (m < 3) == (r < 3) and pos < (100 if r < 3 else 90)
            for t in range(new[m]):
                at = p.kv[m] - new[m] + t
                hit[int(p.starts[m]) + t] = same and pos <= at and (window < 0 or pos >= at - window)
        hit = hit.to(DEV)
        assert not bool(out[hit].isfinite().any()), (r, pos)
        # (rows computed a second time add their keys in another order, each order within the bound of the lse)
        p.check(torch.where(hit[:, None, None], clean[0], out), lse)


def test_garbage_where_nobody_looks():
    """Caches cut back: the shared tokens behind every row's position hold NaN, in keys and values."""
    p = Problem([3, 20], [200, 150], [30, 5, 2] + [3] * 20, [20, 5, 2] + [1] * 20, 8, 2, 128, "bf16")
    lens = [100, 90, 60] + [70 + i for i in range(20)]
    p.batch.set_kv_len(lens)
    for r, last in ((0, 100), (3, 90)):
        for pos in range(last, 200 if r == 0 else 150):
            slot = int(p.table[p.batch.page_indptr_host[r] + pos // 16])
            p.cache.k_pool[slot, :, pos % 16] = NAN
            p.cache.v_pool[slot, :, pos % 16] = NAN
    out, lse = p.run()
    torch.cuda.synchronize()
    p.check(out, lse, kv=lens)


@pytest.mark.parametrize("fmt", FORMATS)
def test_long_shared_caches(fmt):
    """More than 128 MB of keys and values (read past the caches), and a quarter million shared tokens of few heads."""
    row = {"bf16": 256, "mxfp4": 64}.get(fmt, 128)
    p, _, _ = run_and_check([2], [130 * 2 ** 20 // (2 * 8 * row)], [9, 40], [1, 1], 8, 8, 128, fmt, P=64)
    assert p.attn.info.form == 8 + 3
    run_and_check([3, 2], [250001, 1000], [1, 40, 70, 9, 5], [1, 9, 70, 2, 1], 4, 2, 64, fmt, P=64)


def test_offsets_past_32_bits():
    """Shared and own pages beyond 4 GiB of a pool."""
    P, hkv, d, S = 16, 8, 128, 100
    pages = 2 ** 32 // (P * hkv * d * 2) + 40
    c = d2sd.PagedKVCache.allocate(pages, P, hkv, d, "bf16", kv_layout="NHD", device=DEV)
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(S + 60, hkv, d, generator=g).to(torch.bfloat16) for _ in range(2))
    table = [pages - 1 - i for i in range(20)]
    pi = [0, 9, 18]
    kv = [130, 130]
    c.write(k[:130].to(DEV), v[:130].to(DEV), d2sd.PagedBatch([0, 130], [130], [0, 9], table[:9], P, device=DEV))
    c.write(k[130:].to(DEV), v[130:].to(DEV), d2sd.PagedBatch([0, 30], [130], [0, 9], table[9:18], P, device=DEV))
    for n in (1, 25):
        q = torch.randn(2 * n, 16, d, generator=g).to(torch.bfloat16)
        b = d2sd.PagedBatch([0, n, 2 * n], kv, pi, table, P, device=DEV)
        out, _ = d2sd.PagedChunkAttention().plan(b, 16, hkv, d, shared_indptr=[0, 2], shared_len=[S],
                                                   keep_shared=True).run(q.to(DEV), c)
        torch.cuda.synchronize()
        for r, rows in ((0, torch.arange(130)), (1, torch.cat([torch.arange(S), torch.arange(130, 160)]))):
            o, s, A, size = po.attention_ref(q[r * n:r * n + n], k[rows], v[rows], 130 - n, 2, d ** -0.5)
            bound = 2.0 ** -8 * o.abs() + A * (2.0 ** -8 + (2 * 132 * U * size + 2 * 130 * U + 32 * U)[..., None])
            assert ((out[r * n:r * n + n].cpu().double() - o).abs() <= bound).all()


def test_page_ids_outside_the_pool_stay_in_bounds():
    c = d2sd.PagedKVCache.allocate(4, 16, 2, 64, "mxfp8", device=DEV)
    for t in (c.k_pool, c.v_pool, c.k_scale, c.v_scale):
        t.view(torch.uint8).fill_(0x38)
    R = 20
    b = d2sd.PagedBatch(np.arange(R + 1), [64] * R, 4 * np.arange(R + 1), [0, 2 ** 31 - 1, -5, 4] * R, 16, device=DEV)
    out, lse = d2sd.PagedChunkAttention().plan(b, 4, 2, 64, kv_format="mxfp8", shared_indptr=[0, R], shared_len=[40],
                                                 keep_shared=True).run(
        torch.zeros(R, 4, 64, dtype=torch.bfloat16, device=DEV), c)
    torch.cuda.synchronize()
    assert torch.isfinite(out).all() and (lse - math.log(64)).abs().max() < 1e-5


def test_a_side_stream_orders_append_and_attention():
    p = Problem([2, 30], [300, 200], [3, 40] + [5] * 30, [3, 40] + [1] * 30, 8, 2, 128, "mxfp4")
    ref = p.run()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    x = torch.randn(73, 2, 128).to(torch.bfloat16).to(DEV)
    f = d2sd.rotary_frequencies(128)[0].to(DEV)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        p.cache.append(None, x, x, p.batch, f)
        a = p.run()
    side.synchronize()
    b = p.run()
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and not torch.equal(a[0], ref[0])


def test_refusals_on_the_device():
    p = Problem([2], [100], [9, 20], [1, 2], 8, 2, 64, "mxfp8")
    assert p.attn.info.workspace_bytes > 0
    with pytest.raises(ValueError, match="workspace"):
        p.attn.run(p.qd, p.cache, workspace=torch.empty(16, dtype=torch.uint8, device=DEV))
    with pytest.raises(ValueError):
        p.attn.run(p.qd[:2], p.cache)
    with pytest.raises(RuntimeError, match="chunk_plan"):
        d2sd.PagedChunkAttention().plan(p.batch, 8, 2, 64, shared_indptr=[0, 2], shared_len=[113])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("window", [-1, 300])
def test_more_requests_in_a_row_tile_than_lanes(d, fmt, window):
    """One query head a kv head: a row tile of 128 or 256 rows has more requests than a wave has lanes."""
    n = 200
    run_and_check([n], [400], [1 + 2 * (i % 9) for i in range(n)], [1] * n, 2, 2, d, fmt, window=window, num_cus=64)


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("d", [64, 128])
def test_scales_off_the_boundaries_of_their_copies(d, fmt):
    """Block scales whose rows start at odd bytes: shared keys take another way through LDS, to the same result."""
    p = Problem([3, 40], [500, 300], [70, 5, 2] + [1 + i % 40 for i in range(40)], [60, 5, 2] + [1] * 40, 8, 2, d, fmt)
    assert p.attn.info.form & 8
    out, lse = p.run()
    c = p.cache

    def odd(t):
        wide = torch.full((*t.shape[:-1], t.shape[-1] + 1), 0xFF, dtype=torch.uint8, device=DEV)
        wide[..., :-1] = t.view(torch.uint8)
        return wide[..., :-1]

    moved = d2sd.PagedKVCache(c.k_pool, c.v_pool, fmt, k_scale=odd(c.k_scale), v_scale=odd(c.v_scale), kv_layout=p.layout)
    got, glse = p.attn.run(p.qd, moved)
    torch.cuda.synchronize()
    p.check(out, lse)
    p.check(got, glse)


def test_sharing_that_does_not_pay_gives_the_same_result():
    """Planned apart, requests read the shared tokens through pages of their own."""
    new, own = [60] * 8, [60 + 9 * i for i in range(8)]
    p = Problem([8], [48], own, new, 8, 2, 128, "mxfp8", num_cus=256)
    pi = p.batch.page_indptr_host
    for r in range(1, 8):
        p.batch.page_table[pi[r]:pi[r] + 3] = p.batch.page_table[:3]
    assert p.attn.info.form & 8
    a = p.run()
    p.attn.plan(p.batch, 8, 2, 128, kv_format="mxfp8", shared_indptr=[0, 8], shared_len=[48], num_cus=256)
    assert not p.attn.info.form & 8
    b = p.run()
    torch.cuda.synchronize()
    p.check(*a)
    p.check(*b)


def shared_states(p, ws):
    """Partial states over shared keys of tile items: outputs and sums, in the items' order."""
    i, d = p.attn.info, p.d
    items = p.attn.plan_host[:16 * i.num_items].reshape(-1, 16)
    room = i.workspace_bytes // ((d + 1) * 4)
    f = ws.view(torch.int32)
    o, lse = f[:room * d], f[room * d:room * (d + 1)]
    got = []
    for it in items[(items[:, 12] == 1) & (items[:, 11] == 0)].tolist():
        n = -(-it[5] // 32) * 32
        at = it[10] + it[8] * n
        got.append((o[at * d:(at + it[5] // 32 * 32) * d].clone(), lse[at:at + it[5]].clone()))
    return got


@pytest.mark.parametrize("fmt,d", [("bf16", 128), ("mxfp8", 128), ("bf16", 64), ("fp8", 64)])
def test_prompts_of_mixed_lengths_take_shared_keys_once(fmt, d):
    """New prompts of 1 to 60 tokens behind one system prompt, an idle request among them: the states over the shared
    keys are those that the same plan gives once every cache has grown far beyond them."""
    rng = np.random.default_rng(5)
    new = [int(n) for n in rng.integers(1, 61, 24)]
    new[7] = 0
    own = [max(n, 1) for n in new]
    p = Problem([24], [1500], own, new, 8, 2, d, fmt, extra=64, num_cus=64)
    ws = p.attn.workspace().fill_(0x7F)
    out, lse = p.run(workspace=ws)
    torch.cuda.synchronize()
    p.check(out, lse)
    planned = shared_states(p, ws)
    assert len(planned) > 4
    p.batch.set_kv_len([n + 60 for n in p.kv])
    p.run(workspace=ws.fill_(0x7F))
    torch.cuda.synchronize()
    for (o, l), (o2, l2) in zip(planned, shared_states(p, ws)):
        assert torch.equal(o, o2) and torch.equal(l, l2)
