"""GPU parity of rotary_embedding against the 64-bit form.

Tolerance: one rounding to bf16, half a step (2^-8 of the value), and 32-bit
arithmetic before it: the fraction of a turn is rounded to 2^-25 (2^-22 as an
angle), the sine and cosine are good to 2^-22, the factor and the two products
and their sum add 2^-23 each: together under 2^-20 of |a| + |b|, the pair's size."""
import pytest
import torch

import d2sd
from oracle import paged_oracle as po

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _check(got, x, pos, f, tag, **kw):
    ref, size = po.rotary_ref(x, pos, f, **kw)
    got = got.cpu().double()
    bound = 2.0 ** -8 * ref.abs() + 2.0 ** -20 * kw.get("scale", 1.0) * size
    r = 2 * f.numel()
    assert torch.equal(got[..., r:], x.double()[..., r:]), f"{tag}: the dims behind the rotated ones changed"
    worst = ((got - ref).abs() - bound).max().item()
    assert worst <= 0, f"{tag}: {worst:.3g} beyond its bound"


@pytest.mark.parametrize("tokens,hq,hkv,d,r", [(1, 32, 8, 128, 128), (48, 64, 8, 64, 64), (150, 32, 8, 128, 64),
                                                (1500, 28, 4, 128, 128), (7, 5, 1, 96, 32), (3, 2, 2, 256, 256),
                                                (9, 3, 1, 80, 20), (2, 1, 1, 6, 2), (1100, 3, 1, 34, 18)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_matches_the_formula(tokens, hq, hkv, d, r, interleaved):
    g = torch.Generator().manual_seed(tokens + d + r)
    q = (torch.randn(tokens, hq, d, generator=g) * 2).to(torch.bfloat16)
    k = (torch.randn(tokens, hkv, d, generator=g) * 2).to(torch.bfloat16)
    pos = torch.randint(0, 1 << 21, (tokens,), generator=g, dtype=torch.int32)
    pos[0] = 0
    f, s = d2sd.rotary_frequencies(r, 1e6, dict(type="yarn", factor=32.0, original_max_position=4096) if r > 2 else None)
    qd, kd, pd, fd = q.to(DEV), k.to(DEV), pos.to(DEV), f.to(DEV)
    for inverse in (False, True):
        for p in (pd, pd.long()):
            qo, ko = d2sd.rotary_embedding(qd, kd, p, fd, interleaved=interleaved, scale=s, inverse=inverse,
                                           out=(torch.empty_like(qd), torch.empty_like(kd)))
            for name, got, x in (("q", qo, q), ("k", ko, k)):
                _check(got, x, pos, f, f"{name} inverse={inverse} {p.dtype}", interleaved=interleaved, scale=s,
                       inverse=inverse)
        assert torch.equal(qd.cpu(), q) and torch.equal(kd.cpu(), k)
    # in place, queries only: the same bits
    q2 = qd.clone()
    d2sd.rotary_embedding(q2, None, pd, fd, interleaved=interleaved, scale=s, inverse=True)
    assert torch.equal(q2, qo)


def test_fused_projection_views_and_unaligned_rows():
    """q and k as views of one projection output, and rows off 16-byte boundaries; what lies between stays."""
    g = torch.Generator().manual_seed(3)
    for pad in (0, 1):
        base = torch.randn(60, 12 * 64 + pad, generator=g).to(torch.bfloat16)
        pos = torch.arange(60, dtype=torch.int32) * 1000
        f, _ = d2sd.rotary_frequencies(64)
        dev = base.to(DEV)
        heads = dev[:, pad:].unflatten(1, (12, 64))
        d2sd.rotary_embedding(heads[:, :8], heads[:, 8:10], pos.to(DEV), f.to(DEV))
        x = base[:, pad:].unflatten(1, (12, 64))
        _check(heads[:, :8], x[:, :8], pos, f, "q")
        _check(heads[:, 8:10], x[:, 8:10], pos, f, "k")
        assert torch.equal(heads[:, 10:].cpu(), x[:, 10:]) and torch.equal(dev[:, :pad].cpu(), base[:, :pad])


@pytest.mark.parametrize("interleaved", [False, True])
def test_results_larger_than_the_caches(interleaved):
    """Prompts whose results are stored past the caches: sampled tokens against the formula, in place and out of it."""
    g = torch.Generator().manual_seed(21)
    tokens, hq, hkv, d = 2500, 56, 8, 128
    q = torch.randn(tokens, hq, d, generator=g).to(torch.bfloat16)
    k = torch.randn(tokens, hkv, d, generator=g).to(torch.bfloat16)
    pos = torch.randperm(1 << 20, generator=g)[:tokens]
    f, s = d2sd.rotary_frequencies(96)
    qd, kd = q.to(DEV), k.to(DEV)
    out = d2sd.rotary_embedding(qd, kd, pos.to(DEV), f.to(DEV), interleaved=interleaved,
                                out=(torch.empty_like(qd), torch.empty_like(kd)))
    some = torch.cat([torch.randperm(tokens, generator=g)[:60], torch.tensor([0, tokens - 1])])
    for name, got, x in (("q", out[0], q), ("k", out[1], k)):
        _check(got[some.to(DEV)], x[some], pos[some], f, name, interleaved=interleaved)
    q2, k2 = d2sd.rotary_embedding(qd, kd, pos.to(DEV), f.to(DEV), interleaved=interleaved)
    assert q2.data_ptr() == qd.data_ptr() and torch.equal(q2, out[0]) and torch.equal(k2, out[1])


def test_far_and_negative_positions():
    """Positions beyond 32 bits: the angle's error stays that of a near one (64-bit products: 2^-53 of the
    turns, under 2^-22 up to 2^31 turns)."""
    x = torch.ones(4, 1, 64, dtype=torch.bfloat16)
    pos = torch.tensor([-5, 2 ** 31 - 1, 2 ** 33 + 1, -2 ** 20], dtype=torch.int64)
    f, _ = d2sd.rotary_frequencies(64)
    f = f[1:].contiguous()  # 31 pairs: single elements
    y, _ = d2sd.rotary_embedding(x.to(DEV), None, pos.to(DEV), f.to(DEV), out=(torch.empty_like(x, device=DEV), None))
    ref, size = po.rotary_ref(x, pos, f)
    # (the 64-bit reference's own angle is off by 2^-53 of it)
    extra = (pos.abs().double()[:, None, None] * 2.0 ** -51)
    assert ((y.cpu().double() - ref).abs() <= 2.0 ** -8 * ref.abs() + (2.0 ** -20 + extra) * size).all()


def test_rotation_and_its_inverse_differ_from_the_start_by_roundings():
    """Turned forth and back: two roundings of the pair's parts, 2^-8 of |a| + |b| each at most."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(33, 4, 128, generator=g).to(torch.bfloat16)
    pos, (f, _) = torch.arange(33, dtype=torch.int32) * 777, d2sd.rotary_frequencies(128)
    y = x.to(DEV)
    d2sd.rotary_embedding(y, None, pos.to(DEV), f.to(DEV))
    d2sd.rotary_embedding(y, None, pos.to(DEV), f.to(DEV), inverse=True)
    a, b = x.double()[..., :64].abs(), x.double()[..., 64:].abs()
    size = torch.cat([a + b, a + b], -1)
    assert ((y.cpu().double() - x.double()).abs() <= (3 * 2.0 ** -8) * size).all()


def test_replays_in_a_graph_with_new_positions():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(5, 6, 64, generator=g).to(torch.bfloat16)
    f, _ = d2sd.rotary_frequencies(64)
    xd, out, pos, fd = x.to(DEV), torch.empty_like(x, device=DEV), torch.zeros(5, dtype=torch.int32, device=DEV), f.to(DEV)
    graph = d2sd.HipGraph()
    with graph.capture():
        d2sd.rotary_embedding(xd, None, pos, fd, out=(out, None))
    for rep in range(3):
        p = torch.randint(0, 100000, (5,), generator=g, dtype=torch.int32)
        pos.copy_(p)
        graph.replay()
        torch.cuda.synchronize()
        _check(out, x, p, f, f"replay {rep}")


def test_refusals_on_the_device():
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16, device=DEV)
    pos, f = torch.zeros(3, dtype=torch.int32, device=DEV), torch.zeros(32, dtype=torch.float64, device=DEV)
    with pytest.raises(TypeError):
        d2sd.rotary_embedding(q, None, pos, f.float())
    with pytest.raises(ValueError):
        d2sd.rotary_embedding(q, None, pos[:2], f)
    with pytest.raises(ValueError):
        d2sd.rotary_embedding(q, None, pos.cpu(), f)
    with pytest.raises(RuntimeError):
        d2sd.rotary_embedding(q, None, pos, torch.zeros(33, dtype=torch.float64, device=DEV))
    with pytest.raises(ValueError):
        d2sd.rotary_embedding(q, q[:, :, :32], pos, f)
    e = q[:0]
    assert d2sd.rotary_embedding(e, None, pos[:0], f)[0].shape == (0, 4, 64)
