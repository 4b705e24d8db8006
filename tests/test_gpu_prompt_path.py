"""The operators together, as a server uses them: a prompt in chunks (rotary,
cache write, attention over the cache), decoding steps, then a verify step of
CascadeVerifyAttention over the same pool and the commit of what it accepts."""
import numpy as np
import pytest
import torch

import d2sd
from oracle import paged_oracle as po

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


@pytest.mark.parametrize("fmt,hq,hkv,d", [("bf16", 8, 2, 128), ("fp8", 8, 2, 64), ("mxfp8", 16, 2, 64), ("mxfp4", 8, 2, 128)])
def test_prompt_decode_verify_commit(fmt, hq, hkv, d):
    g = torch.Generator().manual_seed(hq + d)
    P, lens = 16, [300, 37]          # two prompts, in chunks of 128 tokens, then 3 decoding steps
    total = [n + 3 for n in lens]
    pi = np.concatenate([[0], np.cumsum([-(-(n + 40) // P) for n in total])])
    table = torch.randperm(int(pi[-1]), generator=g).to(torch.int32).to(DEV)
    scale = torch.full((hkv,), 0.02, device=DEV) if fmt == "fp8" else None
    cache = d2sd.PagedKVCache.allocate(int(pi[-1]), P, hkv, d, fmt, k_scale=scale, v_scale=scale, device=DEV)
    f, s = d2sd.rotary_frequencies(d, 1e4)
    f = f.to(DEV)
    q, k, v = (torch.randn(2, max(total), h, d, generator=g).to(torch.bfloat16) for h in (hq, hkv, hkv))
    outs = [[], []]
    held = [0, 0]
    while held != total:
        take = [min(128, lens[r] - held[r]) if held[r] < lens[r] else int(held[r] < total[r]) for r in (0, 1)]
        rows = [(r, held[r] + i) for r in (0, 1) for i in range(take[r])]
        pick = lambda t: torch.stack([t[r, i] for r, i in rows]).to(DEV)  # noqa: E731
        qs, ks, vs = pick(q), pick(k), pick(v)
        pos = torch.tensor([i for _, i in rows], dtype=torch.int32, device=DEV)
        d2sd.rotary_embedding(qs, ks, pos, f, scale=s)
        held = [held[r] + take[r] for r in (0, 1)]
        batch = d2sd.PagedBatch([0, take[0], sum(take)], held, pi, table, P, device=DEV)
        cache.write(ks, vs, batch)
        o, _ = d2sd.PagedChunkAttention().plan(batch, hq, hkv, d, kv_format=fmt).run(qs, cache)
        outs[0].append(o[:take[0]])
        outs[1].append(o[take[0]:])
    kc, vc = cache.read(batch)
    torch.cuda.synchronize()
    for r in (0, 1):
        got = torch.cat(outs[r]).cpu().double()
        a, b = batch.kv_indptr_host[r], batch.kv_indptr_host[r + 1]
        # the queries as the rotary call rounds them (tested by itself)
        qr = q[r, :total[r]].to(DEV).contiguous()
        d2sd.rotary_embedding(qr, None, torch.arange(total[r], dtype=torch.int32, device=DEV), f, scale=s)
        kr, vr = kc[a:b].cpu(), vc[a:b].cpu()
        o, _, A, size = po.attention_ref(qr.cpu(), kr, vr, 0, hq // hkv, d ** -0.5)
        # as in the chunk attention's tests; fp8 (the attention keeps the scale apart from the codes): the values read back are rounded to bf16, 2^-8 of a
        # key's products (S 2^-8 on the scores, both ways of the softmax) and of a value
        e = (d + 4) * U * size + (2.0 ** -8 * size if fmt == "fp8" else 0.0)
        bound = 2.0 ** -8 * o.abs() + A * (2.0 ** -8 + 2 * e + 2 * total[r] * U + 32 * U
                                           + (2.0 ** -8 if fmt == "fp8" else 0.0))[..., None]
        assert ((got - o).abs() <= bound).all(), f"request {r}"

    # a verify step of a 20-token chain (the causal case) over the cache, both ways
    n = 20
    qv, kv_, vv = (torch.randn(2 * n, h, d, generator=g).to(torch.bfloat16).to(DEV) for h in (hq, hkv, hkv))
    casc = d2sd.CascadeVerifyAttention(DEV)
    if fmt in ("bf16", "fp8"):
        casc.plan([0, n, 2 * n], total, hq, hkv, d, mask_mode="causal", page_size=P, page_indptr=pi, page_table=table,
                  kv_dtype=cache.k_pool.dtype, k_scale=scale, v_scale=scale)
        ov, lv = casc.run(qv, kv_, vv, cache.k_pool, cache.v_pool)
    else:  # the block formats are read back for it
        kc2, vc2 = cache.read(batch)
        casc.plan([0, n, 2 * n], total, hq, hkv, d, mask_mode="causal", prefix_tok_indptr=[0, total[0]], kv_layout="NHD")
        ov, lv = casc.run(qv, kv_, vv, kc2, vc2)
    after = d2sd.PagedBatch([0, n, 2 * n], [t + n for t in total], pi, table, P, device=DEV)
    cache.write(kv_, vv, after)
    oc, lc = d2sd.PagedChunkAttention().plan(after, hq, hkv, d, kv_format=fmt).run(qv, cache)
    torch.cuda.synchronize()
    if fmt == "bf16":  # same keys and values either way: two roundings of P and one of O each, and 32-bit sums
        spread = vv.float().abs().amax() + vc.float().abs().amax()
        assert ((ov.float() - oc.float()).abs() <= 4 * 2.0 ** -8 * spread).all()
        assert ((lv - lc).abs() <= 1e-3).all()
    else:  # the chain's own keys were quantised on the way into the cache: finite, and the lse of the same order
        assert torch.isfinite(oc).all() and ((lv - lc).abs() < 1.0).all()

    # and the commit of three accepted tokens of request 0 to the pool the attention read
    if fmt in ("bf16", "fp8"):
        kw = dict(k_scales=scale, v_scales=scale) if fmt == "fp8" else {}
        nodes = torch.tensor([0, 4, 7], dtype=torch.int32, device=DEV)
        d2sd.PagedKVCommit([cache.k_pool], [cache.v_pool], [kv_], [vv], **kw).commit(table[:int(pi[1])], total[0], nodes)
        now = d2sd.PagedBatch([0, 0, 0], [total[0] + 3, total[1]], pi, table, P, device=DEV)
        kb, vb = cache.read(now)
        torch.cuda.synchronize()
        sc = None if scale is None else scale.cpu()
        for x, got in ((kv_, kb), (vv, vb)):
            want = po.values_ref(*po.quantise_ref(x[nodes.long()].cpu(), fmt, sc), fmt, sc).to(torch.bfloat16)
            assert torch.equal(got[total[0]:total[0] + 3].cpu(), want)
        assert torch.equal(kb[:total[0]], kc[:total[0]]) and torch.equal(vb[:total[0]], vc[:total[0]])
