"""GPU parity of PagedKVCache.append against the 64-bit forms of the norm, the
rotation and the cache's formats.

Tolerance, from the arithmetic (u = 2^-24; size: |a| + |b| of an element's pair
after the norm):
  * norm: the sum of D squares in runs of eight and log2 steps is off by 16 u of
    itself, its division by D and eps add 2 u: half of that on the square root,
    2 u of the reciprocal root, 2 u of the two products: 13 u of a normed value,
    a pass of 2^64 down and up for large ones is exact;
  * rotation: as in the rotary embedding's tests, 2^-20 of the size;
so a rotated value is off by E = scale * 2^-20 size + 13 u size * scale (without
a norm the first alone), one that is not rotated by 13 u of itself.  What is
rounded to bf16 adds half a step, 2^-8 of the value, or 2^-134 where bf16 is
subnormal (below 2^-126 its step is 2^-133 whatever the value).  A quantised key is the
element nearest to a value that E away: no further from the exact value than
its nearest element and 2 E (fp8: and 2 u of it, the quotient's rounding), on
the scale of a block whose largest magnitude is E away."""
import numpy as np
import pytest
import torch

import d2sd
from oracle import paged_oracle as po

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
TINY = 2.0 ** -134  # half a step of subnormal bf16
FORMATS = ["bf16", "fp8", "mxfp8", "mxfp4"]


def turned_ref(x, weight, pos, f, eps, interleaved, scale):
    """Normed and rotated heads in 64 bits and how far off they may be."""
    y, off = x.double(), torch.zeros(x.shape, dtype=torch.float64)
    if weight is not None:
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * weight.double()
        off = 13 * U * y.abs()
    z, size = po.rotary_ref(y, pos, f, interleaved=interleaved, scale=scale)
    r = 2 * f.numel()
    e = scale * (2.0 ** -20 + (13 * U if weight is not None else 0.0)) * size
    e[..., r:] = off[..., r:]
    return z, e


def exponents(amax, most, hi):
    """Exponent of the scale of blocks with these largest magnitudes."""
    m, e = torch.frexp(amax / most)
    e = torch.where(m == 0.5, e - 1, e)
    return torch.where(amax == 0, -117, e).clamp(-117, hi)


def check_keys(fmt, got, scale_bytes, scale, want, off):
    """got: values read back [rows, heads, D]; want, off: exact keys and how far computed ones may be."""
    if fmt == "bf16":
        over = (got - want).abs() - (2.0 ** -8 * (want.abs() + off) + off + TINY)
        assert over.max() <= 0, f"{over.max():.3g} beyond the bound"
        return
    grid = po.element_grid(fmt)
    if fmt == "fp8":
        unit = scale.double()[:, None].expand_as(want)
        off = off + 2 * U * want.abs()
        # (what is read back is the element times the scale in bf16)
        slack = 2.0 ** -8 * got.abs()
    else:
        most, hi = (6.0, 125) if fmt == "mxfp4" else (448.0, 119)
        amax = want.unflatten(-1, (-1, 32)).abs().amax(-1)
        far = off.unflatten(-1, (-1, 32)).amax(-1)
        e = scale_bytes.long() - 127
        assert bool(((e >= exponents((amax - far).clamp(min=0), most, hi)) & (e <= exponents(amax + far, most, hi))).all())
        unit = (2.0 ** e.double()).repeat_interleave(32, -1)
        slack = 0.0
    near = torch.zeros_like(want)
    for part, out in zip((want / unit).split(64), near.split(64)):
        code = po.nearest_code(part, grid)
        mag = grid[code % (8 if fmt == "mxfp4" else 128)]
        out.copy_((mag - part.abs()).abs())
    over = (got - want).abs() - (near * unit + 2 * off + slack)
    assert over.max() <= 0, f"{over.max():.3g} beyond the bound"


class Problem:
    def __init__(self, qo, kv, hq, hkv, d, r, fmt="bf16", layout="HND", P=16, interleaved=False, norm="qk", far=0, seed=0,
                 pad=0, wide_positions=False, spread=2.0):
        g = torch.Generator().manual_seed(seed + sum(kv) + hq + d + r)
        self.qo, self.kv, self.fmt, self.layout, self.P, self.d, self.hkv = qo, list(kv), fmt, layout, P, d, hkv
        self.interleaved, self.r = interleaved, r
        need = [-(-n // P) for n in kv]
        self.pi = np.concatenate([[0], np.cumsum(need)]).astype(int)
        pages = int(self.pi[-1]) + 3
        self.table = torch.randperm(pages, generator=g)[:int(self.pi[-1])].to(torch.int32)
        scale = [torch.rand(hkv, generator=g) * 0.05 + 0.02 for _ in range(2)] if fmt == "fp8" else [None, None]
        self.scale = scale
        kw = {} if fmt != "fp8" else dict(k_scale=scale[0].to(DEV), v_scale=scale[1].to(DEV))
        make = lambda: d2sd.PagedKVCache.allocate(pages, P, hkv, d, fmt, kv_layout=layout, device=DEV, **kw)  # noqa: E731
        self.cache, self.plain = make(), make()
        for c in (self.cache, self.plain):
            for t in (c.k_pool, c.v_pool, *((c.k_scale, c.v_scale) if fmt.startswith("mx") else ())):
                t.view(torch.uint8).fill_(0xA5)
        self.starts = np.concatenate([[0], np.cumsum(qo)]).astype(int)
        self.batch = d2sd.PagedBatch(self.starts, kv, self.pi, self.table.to(DEV), P, device=DEV)
        T = self.T = int(self.starts[-1])
        self.qkv = (torch.randn(T + pad, hq + 2 * hkv, d, generator=g) * spread).to(torch.bfloat16)
        self.hq = hq
        self.q_norm, self.k_norm = ((1 + 0.3 * torch.randn(d, generator=g)).to(torch.bfloat16) if n in norm else None
                                    for n in "qk")
        self.place = torch.tensor([kv[q] - n + i for q, n in enumerate(qo) for i in range(n)], dtype=torch.int64)
        self.pos = self.place
        self.given = None
        if far:
            self.pos = torch.randint(0, far, (T,), generator=g)
            self.given = torch.cat([self.pos, torch.zeros(pad, dtype=torch.int64)]).to(torch.int64 if wide_positions
                                                                                      else torch.int32).to(DEV)
        self.f, self.s = d2sd.rotary_frequencies(r, 1e6, dict(type="yarn", factor=8.0, original_max_position=4096)
                                                 if r > 2 else None)
        self.fd, self.dev = self.f.to(DEV), self.qkv.to(DEV)
        self.norms = [None if t is None else t.to(DEV) for t in (self.q_norm, self.k_norm)]

    def parts(self, t):
        return t[:, :self.hq], t[:, self.hq:self.hq + self.hkv], t[:, self.hq + self.hkv:]

    def run(self, queries=True, **kw):
        q, k, v = self.parts(self.dev)
        args = dict(scale=self.s, interleaved=self.interleaved, q_norm=self.norms[0], k_norm=self.norms[1])
        args.update(kw)
        return self.cache.append(q if queries else None, k, v, self.batch, self.fd, self.given, **args)

    def check_queries(self, got):
        q, _, _ = self.parts(self.qkv)
        want, off = turned_ref(q[:self.T], self.q_norm, self.pos, self.f, 1e-6, self.interleaved, self.s)
        over = (got[:self.T].cpu().double() - want).abs() - (2.0 ** -8 * (want.abs() + off) + off + TINY)
        assert not over.numel() or over.max() <= 0, f"queries {over.max():.3g} beyond their bound"

    def check_cache(self):
        """Keys within their bounds, values the bytes of write(), every other slot as it was."""
        _, k, v = self.parts(self.qkv)
        T, P = self.T, self.P
        dev = self.parts(self.dev)
        self.plain.write(dev[1], dev[2], self.batch)
        got, _ = self.cache.read(self.batch, new_only=True)
        at = [int(self.table[self.pi[q] + self.place[t] // P]) * P + int(self.place[t]) % P
              for q in range(len(self.qo)) for t in range(self.starts[q], self.starts[q + 1])]
        rows = lambda t: (t.transpose(1, 2) if self.layout == "HND" else t).reshape(-1, self.hkv, t.shape[-1]).cpu()  # noqa: E731
        mx = self.fmt.startswith("mx")
        want, off = turned_ref(k[:T], self.k_norm, self.pos, self.f, 1e-6, self.interleaved, self.s)
        check_keys(self.fmt, got.cpu().double(), rows(self.cache.k_scale)[at] if mx else None, self.scale[0], want, off)
        raw = lambda t: rows(t if t.dtype == torch.bfloat16 else t.view(torch.uint8))  # noqa: E731
        assert torch.equal(raw(self.cache.v_pool).view(torch.uint8), raw(self.plain.v_pool).view(torch.uint8))
        rest = torch.ones(self.cache.num_pages * P, dtype=torch.bool)
        rest[at] = False
        assert bool((raw(self.cache.k_pool)[rest].view(torch.uint8) == 0xA5).all())
        if mx:
            assert torch.equal(rows(self.cache.v_scale), rows(self.plain.v_scale))
            assert bool((rows(self.cache.k_scale)[rest] == 0xA5).all())


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("layout,P", [("HND", 16), ("NHD", 64), ("HND", 1)])
@pytest.mark.parametrize("hq,hkv,d,r", [(32, 8, 128, 128), (64, 8, 64, 64), (5, 1, 96, 32), (3, 3, 160, 34),
                                        (2, 2, 256, 256), (4, 2, 32, 2), (7, 1, 64, 58)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append_matches_the_formulas(fmt, layout, P, hq, hkv, d, r, interleaved):
    p = Problem([3, 0, 1, 40], [3, 5, 700, 77], hq, hkv, d, r, fmt, layout, P, interleaved,
                norm=["qk", "q", "k", ""][(d + r + interleaved) % 4])
    before = p.dev.clone()
    out = p.run(q_out=torch.empty(p.T, hq, d, dtype=torch.bfloat16, device=DEV))
    torch.cuda.synchronize()
    p.check_queries(out)
    p.check_cache()
    assert torch.equal(p.dev, before)  # the projection stays as it was


@pytest.mark.parametrize("d,r", [(32, 16), (32, 32), (64, 16), (64, 32), (64, 48), (96, 64), (128, 16), (128, 32), (128, 64),
                                 (128, 80), (160, 128), (256, 128), (256, 48), (256, 256)])
@pytest.mark.parametrize("fmt", ["bf16", "mxfp4"])
@pytest.mark.parametrize("norm", ["qk", ""])
def test_partners_in_any_lane(d, r, fmt, norm):
    """Dims that are paired 1 to 16 lanes apart, and distances that are no power of two."""
    p = Problem([2, 33], [9, 61], 5, 3, d, r, fmt, norm=norm)
    p.check_queries(p.run(q_out=torch.empty(p.T, 5, d, dtype=torch.bfloat16, device=DEV)))
    p.check_cache()


@pytest.mark.parametrize("fmt", ["bf16", "mxfp8"])
@pytest.mark.parametrize("norm", ["qk", ""])
def test_given_positions_and_long_batches(fmt, norm):
    """Far positions, int32 and int64; queries of more than 32 MB (stored past the caches)."""
    for wide in (False, True):
        p = Problem([17, 1], [400, 1], 8, 2, 128, 128, fmt, norm=norm, far=1 << 21, wide_positions=wide)
        out = p.run(q_out=torch.empty(p.T, 8, 128, dtype=torch.bfloat16, device=DEV))
        p.check_queries(out)
        p.check_cache()
    p = Problem([2100, 70], [2100, 70], 64, 1, 128, 128, fmt, norm=norm)
    p.check_queries(p.run(q_out=torch.empty(p.T, 64, 128, dtype=torch.bfloat16, device=DEV)))
    p.check_cache()


def test_in_place_padding_and_no_queries():
    """Queries back into the projection, rows behind the last request left alone; keys and values only."""
    p = Problem([2, 9], [30, 9], 6, 2, 64, 48, "mxfp4", pad=4, far=1000)
    before = p.dev.clone()
    out = p.run()
    assert out.data_ptr() == p.dev.data_ptr()
    p.check_queries(out)
    assert torch.equal(p.dev[p.T:], before[p.T:]) and torch.equal(p.dev[:, 6:], before[:, 6:])
    p.check_cache()
    p = Problem([2, 9], [30, 9], 6, 2, 64, 48, "mxfp4", pad=4)
    before = p.dev.clone()
    assert p.run(queries=False) is None
    p.check_cache()
    assert torch.equal(p.dev, before)
    none = Problem([0, 0], [4, 0], 6, 2, 64, 48)
    none.run()
    torch.cuda.synchronize()
    assert bool((none.cache.k_pool.view(torch.uint8) == 0xA5).all())


@pytest.mark.parametrize("fmt", FORMATS)
def test_strides_of_their_own(fmt):
    """Keys head-major, values with gaps, queries out into a wider tensor."""
    p = Problem([5, 3], [50, 3], 4, 2, 128, 64, fmt)
    q, k, v = p.parts(p.dev)
    kt = k.transpose(0, 1).contiguous().transpose(0, 1)
    wide = torch.full((p.T, 3, 256), 9.0, dtype=torch.bfloat16, device=DEV)
    wide[:, :2, 64:192] = v
    hold = torch.full((p.T, 6, 136), 3.0, dtype=torch.bfloat16, device=DEV)
    out = p.cache.append(q, kt, wide[:, :2, 64:192], p.batch, p.fd, scale=p.s, q_norm=p.q_norm.to(DEV),
                         k_norm=p.k_norm.to(DEV), q_out=hold[:, 1:5, 8:])
    p.check_queries(out)
    p.check_cache()
    assert bool((hold[:, 0] == 3.0).all() and (hold[:, 5] == 3.0).all() and (hold[:, :, :8] == 3.0).all())


@pytest.mark.parametrize("fmt", FORMATS)
def test_tokens_without_a_place(fmt):
    """Caches cut back below their new tokens, page ids outside the pool: no key is written, queries turn all the same."""
    p = Problem([6, 4], [6, 40], 4, 2, 64, 64, fmt)
    p.batch.set_kv_len([2, 3])
    p.batch.page_table[int(p.pi[1])] = -5
    out = p.run(q_out=torch.empty(p.T, 4, 64, dtype=torch.bfloat16, device=DEV))
    p.place = p.pos = torch.tensor([-4, -3, -2, -1, 0, 1, -1, 0, 1, 2])
    p.check_queries(out)
    torch.cuda.synchronize()
    rows = lambda t: (t.view(torch.uint8).transpose(1, 2)).reshape(p.cache.num_pages * p.P, -1)  # noqa: E731
    for t in (p.cache.k_pool, p.cache.v_pool):
        changed = (rows(t) != 0xA5).any(-1).nonzero().flatten().tolist()
        assert changed == [int(p.table[0]) * p.P + i for i in (0, 1)]
    p.batch.page_table[int(p.pi[1])] = p.cache.num_pages
    p.batch.page_table[0] = 1 << 30
    before = p.cache.k_pool.view(torch.uint8).clone()
    p.run(q_out=out)
    torch.cuda.synchronize()
    assert torch.equal(p.cache.k_pool.view(torch.uint8), before)


def test_norm_of_large_small_and_empty_heads():
    """Squares beyond 32 bits, tiny heads, zeros; eps is what keeps the small ones small."""
    p = Problem([4], [4], 3, 1, 64, 64)
    p.qkv[0] *= 1e30 / 4
    p.qkv[1] *= 1e-30
    p.qkv[2] = 0
    p.qkv[3, :, 0] = 3e38
    p.dev.copy_(p.qkv)
    p.check_queries(p.run(q_out=torch.empty(4, 3, 64, dtype=torch.bfloat16, device=DEV)))
    p.check_cache()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("norm", ["qk", ""])
def test_values_that_are_not_finite_stay_in_their_heads(fmt, norm):
    p = Problem([6], [6], 4, 2, 128, 128, fmt, norm=norm)
    clean_q = p.run(q_out=torch.empty(6, 4, 128, dtype=torch.bfloat16, device=DEV)).clone()
    clean = [x.clone() for x in p.cache.read(p.batch, new_only=True)]
    p.dev[1, 2, 5] = float("nan")        # a query's head
    p.dev[2, 4, 70] = float("nan")       # keys
    p.dev[3, 5, 3] = float("inf")
    p.dev[4, 7, 9] = float("nan")        # a value
    q = p.run(q_out=torch.empty(6, 4, 128, dtype=torch.bfloat16, device=DEV))
    k, v = p.cache.read(p.batch, new_only=True)
    bad = torch.zeros(6, 4, dtype=torch.bool, device=DEV)
    bad[1, 2] = True
    assert bool(q[1, 2].isnan().any()) and torch.equal(q[~bad], clean_q[~bad])
    bad = torch.zeros(6, 2, dtype=torch.bool, device=DEV)
    bad[2, 0] = bad[3, 1] = True
    # (fp8 elements saturate: an infinite key without a norm is +-448 times the scale)
    assert bool(k[2, 0].isnan().any()) and (fmt == "fp8" and not norm or not bool(k[3, 1].isfinite().all()))
    assert torch.equal(k[~bad], clean[0][~bad])
    assert bool(v[4, 1].isnan().any())
    good = torch.ones(6, 2, dtype=torch.bool, device=DEV)
    good[4, 1] = False
    assert torch.equal(v[good], clean[1][good])


def test_other_streams_and_replays_follow_the_lengths():
    p = Problem([1, 1, 1], [4, 20, 33], 8, 2, 128, 128, "mxfp8", P=64)
    q_out = torch.empty(3, 8, 128, dtype=torch.bfloat16, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        p.run(q_out=q_out)
    side.synchronize()
    p.check_queries(q_out)
    p.check_cache()
    g = d2sd.HipGraph()
    with g.capture():
        p.run(q_out=q_out)
    for lens in ([5, 21, 34], [40, 64, 1], [6, 7, 8], [4, 20, 33]):
        p.batch.set_kv_len(lens)
        for c in (p.cache, p.plain):
            for t in (c.k_pool, c.v_pool, c.k_scale, c.v_scale):
                t.view(torch.uint8).fill_(0xA5)
        q_out.zero_()
        g.replay()
        torch.cuda.synchronize()
        p.kv = lens
        p.place = p.pos = torch.tensor([n - 1 for n in lens])
        p.check_queries(q_out)
        p.check_cache()


def test_refusals():
    p = Problem([2], [5], 4, 2, 64, 64)
    q, k, v = p.parts(p.dev)
    f, run = p.fd, p.cache.append
    out = torch.empty(2, 4, 64, dtype=torch.bfloat16, device=DEV)
    for bad in (lambda: run(q.float(), k, v, p.batch, f), lambda: run(q, k.half(), v, p.batch, f),
                lambda: run(q, k, v, p.batch, f.float()), lambda: run(q, k, v, p.batch, f, torch.zeros(2, device=DEV)),
                lambda: run(q, k, v, p.batch, f, q_norm=torch.ones(64, device=DEV))):
        with pytest.raises(TypeError):
            bad()
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device=DEV)  # noqa: E731
    for bad in (lambda: run(q[:1], k, v, p.batch, f), lambda: run(q, k[:1], v, p.batch, f),
                lambda: run(q, k, z(2, 3, 64), p.batch, f), lambda: run(z(2, 4, 32), k, v, p.batch, f),
                lambda: run(q, k, v, p.batch, f, q_out=z(2, 4, 65)), lambda: run(q, k, v, p.batch, f, q_out=z(3, 4, 64)),
                lambda: run(q, k, v, p.batch, f, q_out=out[:, :1].expand(2, 4, 64)),
                lambda: run(q, k, v, p.batch, f, q_out=z(8, 64).as_strided((2, 4, 64), (64, 64, 1))),
                lambda: run(None, k, v, p.batch, f, q_out=out), lambda: run(q, k, v, p.batch, f.cpu()),
                lambda: run(q, k, v, p.batch, torch.ones(33, dtype=torch.float64, device=DEV)),
                lambda: run(q, k, v, p.batch, f, torch.zeros(1, dtype=torch.int32, device=DEV)),
                lambda: run(q, k, v, p.batch, f, torch.zeros(2, dtype=torch.int32)),
                lambda: run(q, k, v, p.batch, f, k_norm=z(32)), lambda: run(q.cpu(), k, v, p.batch, f)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: run(q, k, v, p.batch, f[:0]), lambda: run(q, k, v, p.batch, f, scale=float("inf")),
                lambda: run(q, k, v, p.batch, f, q_norm=z(64), eps=0.0),
                lambda: run(q, k, v, p.batch, f, q_norm=z(64), eps=float("nan")),
                lambda: run(q, z(2, 2, 65)[:, :, 1:], v, p.batch, f), lambda: run(q, k, v, p.batch, f, k_norm=z(65)[1:]),
                lambda: run(z(2, 4, 68)[:, :, :64], k, v, p.batch, f, q_out=out)):
        with pytest.raises(RuntimeError, match="cache_append"):
            bad()
    with pytest.raises(ValueError):
        run(q, k, v, d2sd.PagedBatch([0, 2], [5], [0, 1], [0], 32, device=DEV), f)
    torch.cuda.synchronize()
    assert bool((p.cache.k_pool.view(torch.uint8) == 0xA5).all())


def test_queries_over_other_inputs_are_refused():
    p = Problem([3, 2], [30, 9], 4, 4, 64, 64)
    q, k, v = p.parts(p.dev)
    hold = torch.zeros(p.T + 1, 12, 64, dtype=torch.bfloat16, device=DEV)
    hold[:p.T] = p.dev
    before = p.dev.clone()
    for bad in (lambda: p.cache.append(q, k, v, p.batch, p.fd, q_out=k), lambda: p.cache.append(q, k, v, p.batch, p.fd, q_out=v),
                lambda: p.cache.append(q, k, v, p.batch, p.fd, q_out=p.dev[:, 1:5]),
                lambda: p.cache.append(hold[:-1, :4], hold[:-1, 4:8], hold[:-1, 8:], p.batch, p.fd, q_out=hold[1:, :4])):
        with pytest.raises(RuntimeError, match="cache_append: .*lie apart"):
            bad()
    torch.cuda.synchronize()
    assert torch.equal(p.dev, before) and bool((p.cache.k_pool.view(torch.uint8) == 0xA5).all())
    # parts of one buffer that do lie apart
    out = p.cache.append(hold[:-1, :4], hold[:-1, 4:8], hold[:-1, 8:], p.batch, p.fd, scale=p.s, q_norm=p.norms[0],
                         k_norm=p.norms[1], q_out=hold[:-1, :4])
    p.check_queries(out)
    p.check_cache()
