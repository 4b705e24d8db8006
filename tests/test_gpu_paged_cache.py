"""GPU parity of PagedKVCache.write and read against the 64-bit forms: codes and
block scales bit for bit, values read back exactly (fp8: code * scale rounded
to bf16 once, so bit for bit as well)."""
import numpy as np
import pytest
import torch

import d2sd
from oracle import paged_oracle as po

pytestmark = pytest.mark.gpu
DEV = "cuda"
FORMATS = ["bf16", "fp8", "mxfp8", "mxfp4"]


def make(fmt, layout, pages, P, hkv, d, g=None, fill=True):
    """A cache with every byte set (a pattern no write leaves by chance)."""
    scale = None
    if fmt == "fp8":
        scale = torch.rand(hkv, generator=g) * 0.02 + 0.001
    c = d2sd.PagedKVCache.allocate(pages, P, hkv, d, fmt, kv_layout=layout, device=DEV,
                                   k_scale=None if scale is None else scale.to(DEV),
                                   v_scale=None if scale is None else (2 * scale).to(DEV))
    if fill:
        for t in (c.k_pool, c.v_pool, *((c.k_scale, c.v_scale) if fmt.startswith("mx") else ())):
            t.view(torch.uint8).fill_(0x5A)
    return c


def rows_of(t, layout, table, pos, P):
    """Pool rows [len(pos), Hkv, width] (bytes or bf16) of one request's positions."""
    t = t.cpu()
    t = t.transpose(1, 2) if layout == "HND" else t
    pos = torch.as_tensor(pos, dtype=torch.long)
    return t[table.long()[pos // P], pos % P]


def batch_of(qo, kv, P, g, spare=3, extra=0):
    need = [-(-(n + extra) // P) for n in kv]
    pi = np.concatenate([[0], np.cumsum(need)])
    table = torch.randperm(int(pi[-1]) + spare, generator=g)[:int(pi[-1])].to(torch.int32)
    b = d2sd.PagedBatch(np.concatenate([[0], np.cumsum(qo)]), kv, pi, table.to(DEV), P)
    return b, table, pi, int(pi[-1]) + spare


@pytest.mark.parametrize("layout", ["HND", "NHD"])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("qo,kv,P,hkv,d", [([1], [1], 16, 8, 128), ([3, 0, 17, 1], [3, 5, 40, 100], 16, 8, 128),
                                            ([1] * 9, list(range(1, 10)), 1, 2, 64), ([33, 2], [70, 2], 64, 3, 96),
                                            ([5], [300], 128, 1, 32), ([4, 4], [4, 9], 4, 2, 256)])
def test_write_and_read_match_the_definition(fmt, layout, qo, kv, P, hkv, d):
    g = torch.Generator().manual_seed(sum(kv) + d)
    b, table, pi, pages = batch_of(qo, kv, P, g)
    c = make(fmt, layout, pages, P, hkv, d, g)
    before = [t.clone() for t in (c.k_pool, c.v_pool)]
    T = b.total_q
    kvr = torch.randn(T + 2, hkv, 2, d, generator=g)
    kvr = (kvr * torch.exp2(torch.randint(-30, 20, kvr.shape[:3], generator=g).float())[..., None]).to(torch.bfloat16)
    if T > 1:
        kvr[1, 0] = 0.0                                     # a block of zeros
    dev = kvr.to(DEV)
    c.write(dev[:, :, 0], dev[:, :, 1], b)                  # strided views; rows behind the last request stay out
    k_new, v_new = c.read(b, new_only=True)
    full = [torch.full((b.total_kv + 1, hkv, d), 7.0, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    c.read(b, out=tuple(full))
    torch.cuda.synchronize()
    touched = torch.zeros(pages * P, dtype=torch.bool)
    for side, (pool, sc, new, whole, old) in enumerate(((c.k_pool, c.k_scale, k_new, full[0], before[0]),
                                                        (c.v_pool, c.v_scale, v_new, full[1], before[1]))):
        x = kvr[:T, :, side]
        scale = sc.cpu() if fmt == "fp8" else None
        codes, scales = po.quantise_ref(x, fmt, scale)
        want = po.values_ref(codes, scales, fmt, scale).to(torch.bfloat16)
        assert torch.equal(new.cpu(), want), f"side {side}: values read back"
        stored, q0 = po.pack_codes(codes, fmt), 0
        raw = pool if fmt == "bf16" else pool.view(torch.uint8)
        for r, n in enumerate(qo):
            pos = range(kv[r] - n, kv[r])
            t = table[pi[r]:pi[r + 1]]
            if n:
                assert torch.equal(rows_of(raw, layout, t, pos, P), stored[q0:q0 + n]), f"side {side} request {r}: codes"
                if scales is not None:
                    assert torch.equal(rows_of(sc, layout, t, pos, P).long(), scales[q0:q0 + n]), "block scales"
                at = b.kv_indptr_host[r] + kv[r] - n
                assert torch.equal(whole[at:at + n].cpu(), want[q0:q0 + n])
                touched[t.long()[torch.tensor(list(pos)) // P] * P + torch.tensor(list(pos)) % P] = True
            q0 += n
        assert bool((whole[b.total_kv:] == 7.0).all())
        # slots that no token went to keep their bytes
        a = (pool if fmt == "bf16" else pool.view(torch.uint8)).cpu()
        o = (old if fmt == "bf16" else old.view(torch.uint8)).cpu()
        if layout == "HND":
            a, o = a.transpose(1, 2), o.transpose(1, 2)
        a, o = a.reshape(pages * P, -1), o.reshape(pages * P, -1)
        assert torch.equal(a[~touched].view(torch.uint8), o[~touched].view(torch.uint8))


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4", "fp8"])
def test_every_bf16_value(fmt):
    """All 65536 bit patterns (infinities, NaNs and subnormals among them), in order (blocks of like size) and
    shuffled over exponents within a range of 2^12 and over everything."""
    bits = torch.arange(65536, dtype=torch.int32)
    g = torch.Generator().manual_seed(5)
    near = torch.argsort(bits % 32768 + torch.rand(65536, generator=g) * 12 * 128)
    wild = torch.randperm(65536, generator=g)
    x = torch.cat([bits, bits[near], bits[wild]]).to(torch.int16).view(torch.bfloat16).view(-1, 2, 128)
    T, P = x.shape[0], 64
    b = d2sd.PagedBatch([0, T], [T], [0, T // P], list(range(T // P)), P, device=DEV)
    c = make(fmt, "HND", T // P, P, 2, 128, g)
    xd = x.to(DEV)
    c.write(xd, xd, b)
    k, v = c.read(b)
    torch.cuda.synchronize()
    for pool, sc, got in ((c.k_pool, c.k_scale, k), (c.v_pool, c.v_scale, v)):
        scale = sc.cpu() if fmt == "fp8" else None
        codes, scales = po.quantise_ref(x, fmt, scale)
        stored = pool.view(torch.uint8).cpu().transpose(1, 2).reshape(T, 2, -1)
        nan = codes == 127 if fmt == "fp8" else torch.zeros_like(codes, dtype=torch.bool)
        if fmt == "fp8":  # a NaN's sign is not part of the format
            assert bool(((stored[nan] & 127) == 127).all())
            assert torch.equal(stored[~nan], codes[~nan].to(torch.uint8))
        else:
            assert torch.equal(stored, po.pack_codes(codes, fmt))
            assert torch.equal(sc.cpu().transpose(1, 2).reshape(T, 2, -1).long(), scales)
        want = po.values_ref(codes, scales, fmt, scale).to(torch.bfloat16)
        assert torch.equal(torch.isnan(got.cpu()), torch.isnan(want))
        ok = ~torch.isnan(want)
        assert torch.equal(got.cpu()[ok], want[ok])


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
def test_read_of_every_code_under_every_scale(fmt):
    """Caches written elsewhere: every element code under every scale byte that leaves it finite and normal."""
    hi = 246 if fmt == "mxfp8" else 252
    sb = torch.arange(10, hi + 1)
    n = sb.numel()
    codes = (torch.arange(256) if fmt == "mxfp8" else torch.arange(32) % 16).repeat(n, 1).view(n, 1, -1)
    codes = torch.where((codes % 128 == 127) & (fmt == "mxfp8"), 0, codes)
    d = codes.shape[-1]
    pages = -(-n // 16)
    c = make(fmt, "NHD", pages, 16, 1, d)
    pad = pages * 16 - n
    store = torch.cat([po.pack_codes(codes, fmt), torch.zeros(pad, 1, c.k_pool.shape[-1], dtype=torch.uint8)])
    scales = torch.cat([sb, torch.full((pad,), 255)]).to(torch.uint8).view(-1, 1, 1).expand(-1, 1, d // 32).contiguous()
    for pool, sc in ((c.k_pool, c.k_scale), (c.v_pool, c.v_scale)):
        pool.view(torch.uint8).copy_(store.view(pages, 16, 1, -1))
        sc.copy_(scales.view(pages, 16, 1, -1))
    b = d2sd.PagedBatch([0, 0], [n + pad], [0, pages], list(range(pages)), 16, device=DEV)
    k, v = c.read(b)
    torch.cuda.synchronize()
    want = po.values_ref(codes, sb.view(-1, 1, 1).expand(-1, 1, d // 32), fmt).to(torch.bfloat16)
    for got in (k.cpu(), v.cpu()):
        assert torch.equal(got[:n], want)
        assert bool(torch.isnan(got[n:]).all())  # scale 255


def test_lengths_move_on_the_device_and_bad_pages_are_skipped():
    g = torch.Generator().manual_seed(2)
    P, hkv, d = 16, 2, 64
    b, table, pi, pages = batch_of([2, 2], [2, 20], P, g, extra=20)
    c = make("mxfp8", "HND", pages, P, hkv, d)
    x = torch.randn(4, hkv, d, generator=g).to(torch.bfloat16).to(DEV)
    graph = d2sd.HipGraph()
    c.write(x, x, b)
    out = tuple(torch.zeros(4, hkv, d, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    b.prepare_read(new_only=True)
    with graph.capture():
        c.write(x, x, b)
        c.read(b, new_only=True, out=out)
    for lens in ([5, 33], [1, 22], [22, 40]):  # [1, ..]: the request's first token has no place
        b.set_kv_len(lens)
        x.copy_(torch.randn(4, hkv, d, generator=g))
        for t in out:
            t.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        want = po.values_ref(*po.quantise_ref(x.cpu(), "mxfp8"), "mxfp8").to(torch.bfloat16)
        for t in out:
            got = t.cpu()
            if lens[0] == 1:
                assert bool((got[0] == 9.0).all())
                got = got[1:]
            assert torch.equal(got, want[4 - got.shape[0]:])
    # page ids outside the pool: those tokens are neither written nor read, the others are
    bad = torch.tensor([0, pages, -1, 1], dtype=torch.int32, device=DEV)
    b2 = d2sd.PagedBatch([0, 64], [64], [0, 4], bad, P)
    y = torch.randn(64, hkv, d, generator=g).to(torch.bfloat16).to(DEV)
    c.write(y, y, b2)
    got = tuple(torch.full((64, hkv, d), 9.0, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    c.read(b2, out=got)
    torch.cuda.synchronize()
    want = po.values_ref(*po.quantise_ref(y.cpu(), "mxfp8"), "mxfp8").to(torch.bfloat16)
    for t in got:
        assert bool((t[16:48] == 9.0).all())
        assert torch.equal(t[:16].cpu(), want[:16]) and torch.equal(t[48:].cpu(), want[48:])


def test_offsets_past_32_bits():
    """The last pages of a pool of 4.5 GB a side."""
    P, hkv, d = 64, 8, 128
    pages = 4700000000 // (P * hkv * d)
    c = make("mxfp8", "HND", pages, P, hkv, d, fill=False)
    g = torch.Generator().manual_seed(8)
    b = d2sd.PagedBatch([0, 70], [70], [0, 2], [pages - 1, pages - 2], P, device=DEV)
    x = torch.randn(70, hkv, d, generator=g).to(torch.bfloat16)
    c.write(x.to(DEV), x.to(DEV), b)
    k, v = c.read(b)
    torch.cuda.synchronize()
    want = po.values_ref(*po.quantise_ref(x, "mxfp8"), "mxfp8").to(torch.bfloat16)
    assert torch.equal(k.cpu(), want) and torch.equal(v.cpu(), want)
    assert c.k_pool.numel() > 2 ** 32


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("hkv,d,layout", [(3, 96, "HND"), (1, 64, "NHD")])
def test_prompts_of_many_tokens(fmt, hkv, d, layout):
    """Thousands of tokens of ragged requests, one of which holds fewer tokens than it has new ones; a padded batch."""
    g = torch.Generator().manual_seed(d)
    P = 16
    qo, kv = [4001, 0, 2, 4190, 40], [4001, 7, 5000, 4200, 25]
    b, table, pi, pages = batch_of(qo, kv, P, g)
    c = make(fmt, layout, pages, P, hkv, d, g)
    T = b.total_q
    x = torch.randn(T + 5, hkv, d, generator=g).to(torch.bfloat16)
    c.write(x.to(DEV), (-x).to(DEV), b)
    out = tuple(torch.full((T + 3, hkv, d), 9.0, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    c.read(b, new_only=True, out=out)
    torch.cuda.synchronize()
    lost = T - 40 + torch.arange(15)  # the last request's first tokens have no place
    for got, pool, sc, s in ((out[0], c.k_pool, c.k_scale, 1), (out[1], c.v_pool, c.v_scale, -1)):
        scale = sc.cpu() if fmt == "fp8" else None
        want = po.values_ref(*po.quantise_ref(s * x[:T], fmt, scale), fmt, scale).to(torch.bfloat16)
        want[lost] = 9.0
        assert torch.equal(got[:T].cpu(), want)
        assert bool((got[T:] == 9.0).all())


@pytest.mark.parametrize("fmt", FORMATS)
def test_reads_of_more_than_the_caches_hold(fmt):
    """0.14 GB of results, stored past the caches: every row is there."""
    g = torch.Generator().manual_seed(6)
    P, hkv, d = 64, 8, 128
    kv = [16001, 3, 18500]
    b, table, pi, pages = batch_of([0, 0, 0], kv, P, g)
    c = make(fmt, "HND", pages, P, hkv, d, g)
    fill = d2sd.PagedBatch(np.concatenate([[0], np.cumsum(kv)]), kv, pi, table.to(DEV), P)
    x = torch.randn(500, hkv, d, generator=g).to(torch.bfloat16)  # token t holds row t % 500
    rows = torch.arange(b.total_kv) % 500
    xd = x.to(DEV)[rows.to(DEV)]
    c.write(xd, -xd, fill)
    k, v = c.read(b)
    torch.cuda.synchronize()
    for got, s, sc in ((k, 1, c.k_scale), (v, -1, c.v_scale)):
        scale = sc.cpu() if fmt == "fp8" else None
        want = po.values_ref(*po.quantise_ref(s * x, fmt, scale), fmt, scale).to(torch.bfloat16)
        assert torch.equal(got, want.to(DEV)[rows.to(DEV)])


def test_pools_serve_the_kv_commit_and_the_other_way_round():
    """fp8 and bf16 pools are PagedKVCommit's: the same bytes from either."""
    g = torch.Generator().manual_seed(4)
    for fmt in ("bf16", "fp8"):
        P, hkv, d, L, n = 16, 8, 128, 30, 7
        b, table, pi, pages = batch_of([n], [L + n], P, g)
        c, c2 = make(fmt, "HND", pages, P, hkv, d, g), make(fmt, "HND", pages, P, hkv, d, g)
        if fmt == "fp8":
            c2.k_scale.copy_(c.k_scale)
            c2.v_scale.copy_(c.v_scale)
        x = torch.randn(n, hkv, d, generator=g).to(torch.bfloat16).to(DEV)
        c.write(x, -x, b)
        kw = dict(k_scales=c2.k_scale, v_scales=c2.v_scale) if fmt == "fp8" else {}
        d2sd.PagedKVCommit([c2.k_pool], [c2.v_pool], [x], [-x], **kw).commit(
            table.to(DEV), L, torch.arange(n, dtype=torch.int32, device=DEV))
        torch.cuda.synchronize()
        for a, z in ((c.k_pool, c2.k_pool), (c.v_pool, c2.v_pool)):
            assert torch.equal(a.view(torch.uint8), z.view(torch.uint8))


def test_refusals_on_the_device():
    c = make("mxfp4", "HND", 4, 16, 2, 64)
    b = d2sd.PagedBatch([0, 2], [2], [0, 1], [0], 16, device=DEV)
    x = torch.zeros(2, 2, 64, dtype=torch.bfloat16, device=DEV)
    for bad in ((x.float(), x), (x, x.float())):
        with pytest.raises(TypeError):
            c.write(*bad, b)
    for bad in ((x[:1], x[:1]), (x[:, :1], x[:, :1]), (x, x.transpose(0, 1).contiguous().transpose(0, 1)),
                (x.cpu(), x.cpu()), (x[..., :32], x[..., :32])):
        with pytest.raises(ValueError):
            c.write(*bad, b)
    with pytest.raises(ValueError):
        c.write(x, x, d2sd.PagedBatch([0, 2], [2], [0, 1], [0], 32, device=DEV))
    with pytest.raises(ValueError):
        c.write(x, x, d2sd.PagedBatch([0, 2], [2], [0, 1], [0], 16, device="cpu"))
    with pytest.raises(RuntimeError):  # rows off 16-byte boundaries
        y = torch.zeros(2 * 2 * 64 + 8, dtype=torch.bfloat16, device=DEV)[1:2 * 2 * 64 + 1].view(2, 2, 64)
        c.write(y, y, b)
    p8 = torch.zeros(4, 2, 16, 64, dtype=torch.float8_e4m3fn, device=DEV)
    s = torch.ones(2, device=DEV)
    for args, kw, err in (((p8, p8, "bf16"), {}, TypeError), ((p8, p8, "fp8"), {}, ValueError),
                          ((p8, p8, "fp8"), dict(k_scale=s, v_scale=s[:1]), ValueError),
                          ((p8, p8[:2], "fp8"), dict(k_scale=s, v_scale=s), ValueError),
                          ((p8, p8, "mxfp8"), dict(k_scale=s, v_scale=s), TypeError),
                          ((p8[:, :, :12], p8[:, :, :12], "fp8"), dict(k_scale=s, v_scale=s), ValueError)):
        with pytest.raises(err):
            d2sd.PagedKVCache(*args, **kw)
    graph = d2sd.HipGraph()
    b3 = d2sd.PagedBatch([0, 2], [2], [0, 1], [0], 16, device=DEV)
    with graph.capture():
        with pytest.raises(RuntimeError, match="prepare_read"):
            c.read(b3)
        c.write(x, x, b)
