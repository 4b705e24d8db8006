"""What the paged-cache operators are timed on: the calls between a prompt (or a step's new tokens) and the
attention that reads them back from the cache.

Kinds of case
  rope   rotary embedding of new queries and keys at their positions: half or interleaved layout, part of the
         head, frequencies stretched for long contexts
  write  new keys and values of a ragged batch quantised into a paged cache, then read back as the values that
         later steps will see (the tokens of the step only)
  read   the whole cache of a ragged batch read back into contiguous keys and values
  attn   causal attention of each request's newest tokens over its paged cache, which already holds them: one
         token (decoding), a chunk of a prompt, or a batch of both

Cache formats: "bf16"; "fp8" (e4m3fn bytes with one fp32 scale per kv head); "mxfp8" and "mxfp4" (e4m3fn bytes or
e2m1 nibbles, even element low, in blocks of 32 head dims with a power-of-two scale byte e8m0 each).  A block's
scale is the smallest power of two that keeps its largest magnitude in the elements' range (448 or 6), within
2^-117 and 2^119 (mxfp8) or 2^125 (mxfp4); elements are rounded to nearest even.
"""
import math
import random
import sys
from pathlib import Path

import numpy as np
import torch

own = False

if str(Path(__file__).resolve().parents[1] / "d2-sd_amd") not in sys.path:
    sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "d2-sd_amd"))

DEV = "cuda"
BLOCK = 32  # head dims of one block scale


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _paged(kind, name, **c):
    c = dict(dict(kind=kind, hq=32, hkv=8, d=128, fmt="bf16", layout="HND", page=16, reqs=1, kv_lo=1, kv_hi=1, new=1,
                  chunks=0, chunk=0, window=-1, sinks=False, shape=0), **c)
    return dict(name=name, **c) if name else c


def _rope(name, **c):
    c = dict(dict(kind="rope", tokens=1, hq=32, hkv=8, d=128, rotary=128, interleaved=False, base=1e6, stretch="none",
                  factor=1.0, trained=4096, far=4096, inverse=False), **c)
    return dict(name=name, **c) if name else c


def listed():
    return [
        # a decoding step of 48 conversations, one token each
        _rope("rope_decode_48", tokens=48, far=32768),
        # an 8K prompt at head size 64, frequencies stretched 32 times beyond the 4K they were trained at
        _rope("rope_prompt_8k_yarn", tokens=8192, hq=64, d=64, rotary=64, base=150000.0, stretch="yarn", factor=32.0,
              far=131072),
        # interleaved pairs over half of each head, positions of a million-token document
        _rope("rope_partial_interleaved", tokens=2111, rotary=64, interleaved=True, base=10000.0, stretch="linear",
              factor=8.0, far=1000000),
        # the cache write of a decoding step
        _paged("write", "write_decode_64_mxfp8", fmt="mxfp8", reqs=64, kv_lo=200, kv_hi=4000),
        # a prefill batch's write, the smallest cache
        _paged("write", "write_prompts_mxfp4", fmt="mxfp4", reqs=5, kv_lo=1000, kv_hi=6000, new=0),
        # the caches of a ragged batch, for code that wants contiguous bf16
        _paged("read", "read_16_requests_mxfp8", fmt="mxfp8", reqs=16, kv_lo=100, kv_hi=8000),
        # one conversation at head size 64 in token-major pages, the smallest cache
        _paged("read", "read_one_mxfp4_d64", hq=64, d=64, fmt="mxfp4", layout="NHD", page=64, kv_lo=4099, kv_hi=4099),
        # the smallest attention: one token of one short conversation
        _paged("attn", "attn_decode_one_1k", kv_lo=1000, kv_hi=1000),
        # a server decoding 32 long conversations
        _paged("attn", "attn_decode_32_mxfp8", hq=64, fmt="mxfp8", reqs=32, kv_lo=8192, kv_hi=32768),
        # 23 decoding requests and one 1000-token chunk of a prompt in the same call
        _paged("attn", "attn_mixed_mxfp4", fmt="mxfp4", reqs=24, kv_lo=1200, kv_hi=5000, chunks=1, chunk=1000, shape=3),
        # head size 64 with sinks and a window of 128 keys: four chunks of prompts
        _paged("attn", "attn_chunks_d64_window", hq=64, d=64, reqs=4, kv_lo=2000, kv_hi=8000, chunks=4, chunk=1024,
               window=127, sinks=True, shape=1),
        # the largest: two 2K chunks of long prompts
        _paged("attn", "attn_chunks_2k_at_16k", reqs=2, kv_lo=15000, kv_hi=16384, chunks=2, chunk=2048),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(32, 8, 128), (32, 8, 128), (64, 8, 128), (64, 8, 64), (28, 4, 128), (16, 16, 64)]
MOST_SCORES = 2.5e9  # padded score matrix of the plain form
MOST_TOKENS = 3e5  # padded cache of the plain form


def draw(rng):
    kind = rng.choices(["rope", "write", "read", "attn"], [2, 2, 2, 6])[0]
    hq, hkv, d = rng.choice(HEADS)
    if kind == "rope":
        stretch = rng.choice(["none", "linear", "yarn", "wavelength"])
        return _rope(None, tokens=_log(rng, 1, 8192), hq=hq, hkv=hkv, d=d, rotary=rng.choice([d, d, d // 2, d // 4]),
                     interleaved=rng.random() < 0.5, base=rng.choice([1e4, 1.5e5, 1e6]), stretch=stretch,
                     factor=1.0 if stretch == "none" else rng.choice([2.0, 8.0, 32.0]), far=_log(rng, 8192, 1000000),
                     inverse=rng.random() < 0.25)
    c = dict(hq=hq, hkv=hkv, d=d, fmt=rng.choice(["bf16", "fp8", "mxfp8", "mxfp8", "mxfp4", "mxfp4"]),
             layout=rng.choice(["HND", "HND", "NHD"]), page=rng.choice([16, 16, 32, 64, 128]),
             reqs=_log(rng, 1, 64), shape=rng.randrange(1 << 16))
    c["kv_lo"] = _log(rng, 16, 12000)
    c["kv_hi"] = min(32768, int(c["kv_lo"] * rng.uniform(1.0, 4.0)))
    c["new"] = rng.choice([1, 1, 1, 0, rng.randint(2, 9)])
    if kind == "attn":
        c["window"] = rng.choice([-1, -1, -1, 127, rng.randint(0, 4000)])
        c["sinks"] = rng.random() < 0.3
        c["new"] = max(1, c["new"])
        if rng.random() < 0.5:
            c["chunk"] = _log(rng, 10, 2048)
            c["chunks"] = rng.randint(1, c["reqs"])
    else:
        c["reqs"] = min(c["reqs"], 24)
    while True:
        qo, kv = _lens(c)
        if kind == "attn" and c["reqs"] * c["hq"] * max(qo) * max(kv) > MOST_SCORES or c["reqs"] * max(kv) > MOST_TOKENS \
                or kind != "attn" and c["reqs"] * max(kv) > 6e4:
            if c["reqs"] > 2:
                c["reqs"] = c["reqs"] * 2 // 3
                c["chunks"] = min(c.get("chunks", 0), c["reqs"])
            else:
                c["kv_lo"], c["kv_hi"] = c["kv_lo"] // 2 + 1, c["kv_hi"] // 2 + 1
                c["chunk"] = c.get("chunk", 0) * 2 // 3
            continue
        return _paged(kind, None, **c)


def _lens(case):
    """New tokens and cache lengths (the new tokens included) of each request; new == 0: every token is new.
    The first `chunks` requests bring a chunk of their prompt."""
    rng = random.Random(case.get("shape", 0))
    kv = [rng.randint(case["kv_lo"], case["kv_hi"]) for _ in range(case["reqs"])]
    qo = [min(L, case["chunk"] if r < case.get("chunks", 0) else case["new"] or L) for r, L in enumerate(kv)]
    return qo, kv


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _states(gen, *shape):
    """Keys and values as projections give them: unit scale, some head dims several times larger than the rest."""
    x = torch.randn(shape, generator=gen, device=DEV)
    lift = 1.0 + 5.0 * (torch.rand(shape[-2:], generator=gen, device=DEV) < 0.03).float()
    return (x * lift).to(torch.bfloat16)


def _frequencies(case):
    """Radians per position of each rotated pair (64 bits) and the factor on cos and sin."""
    i = torch.arange(0, case["rotary"], 2, dtype=torch.float64)
    f = case["base"] ** (-i / case["rotary"])
    factor, n0 = case["factor"], case["trained"]
    if case["stretch"] == "linear":
        return f / factor, 1.0
    if case["stretch"] == "yarn":  # slow pairs interpolated, fast ones kept, a ramp between 32 turns and 1
        at = lambda turns: case["rotary"] * math.log(n0 / (turns * 2 * math.pi)) / (2 * math.log(case["base"]))  # noqa: E731
        lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), case["rotary"] - 1)
        ramp = ((i / 2 - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1.0
    if case["stretch"] == "wavelength":  # pairs longer than the trained length interpolated, those under a quarter kept
        turns = n0 * f / (2 * math.pi)
        smooth = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return f / factor * (1 - smooth) + f * smooth, 1.0
    return f, 1.0


class _State:
    pass


def prepare(case, seed):
    s, gen = _State(), _gen(seed)
    s.case = case
    if case["kind"] == "rope":
        n = case["tokens"]
        s.q = torch.randn((n, case["hq"], case["d"]), generator=gen, device=DEV).to(torch.bfloat16)
        s.k = torch.randn((n, case["hkv"], case["d"]), generator=gen, device=DEV).to(torch.bfloat16)
        s.q_out, s.k_out = torch.empty_like(s.q), torch.empty_like(s.k)
        first = int(torch.randint(0, max(1, case["far"] - n), (1,), generator=gen, device=DEV))
        s.positions = (first + torch.arange(n, device=DEV)).to(torch.int32)
        if n <= 64:  # one token of each of n conversations
            s.positions = torch.randint(0, case["far"], (n,), generator=gen, device=DEV, dtype=torch.int32)
        f, s.scale = _frequencies(case)
        s.inv_freq = f.to(DEV)
        return s
    hkv, d, P, fmt = case["hkv"], case["d"], case["page"], case["fmt"]
    qo, kv = _lens(case)
    s.qo_indptr, s.page_indptr = [0], [0]
    for a, b in zip(qo, kv):
        s.qo_indptr.append(s.qo_indptr[-1] + a)
        s.page_indptr.append(s.page_indptr[-1] + -(-b // P))
    s.kv_len, s.max_qo, s.max_kv = kv, max(qo), max(kv)
    n = s.page_indptr[-1]
    pages = n + 4
    s.page_table = torch.from_numpy(np.random.default_rng(seed).permutation(pages)[:n].astype(np.int32)).to(DEV)
    at = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    s.qo_indptr_dev, s.page_indptr_dev, s.kv_len_dev = at(s.qo_indptr), at(s.page_indptr), at(kv)
    total = s.qo_indptr[-1]
    # pools with every page in use filled through the plain quantiser
    heads = lambda w: (pages, hkv, P, w) if case["layout"] == "HND" else (pages, P, hkv, w)  # noqa: E731
    pools = []
    for _ in range(2):
        x = _states(gen, pages, P, hkv, d)
        scale = None
        if fmt == "fp8":
            scale = (x.float().abs().amax(dim=(0, 1, 3)) / 448.0).contiguous()
        codes, scales = _encode(x, fmt, scale)
        x = None
        if case["layout"] == "HND":
            codes = codes.transpose(1, 2).contiguous()
            scales = scales.transpose(1, 2).contiguous() if scales is not None else None
        assert tuple(codes.shape) == heads(codes.shape[-1])
        pools.append((codes, scale if fmt == "fp8" else scales))
    (s.k_pool, s.k_scale), (s.v_pool, s.v_scale) = pools
    s.q = s.k = s.v = s.sinks = None
    if case["kind"] == "attn":
        s.q = torch.randn((total, case["hq"], d), generator=gen, device=DEV).to(torch.bfloat16)
        s.sinks = torch.randn(case["hq"], generator=gen, device=DEV) if case["sinks"] else None
    if case["kind"] == "write":
        s.k, s.v = _states(gen, total, hkv, d), _states(gen, total, hkv, d)
    if own:
        import d2sd
        s.cache = d2sd.PagedKVCache(s.k_pool, s.v_pool, fmt, k_scale=s.k_scale, v_scale=s.v_scale,
                                    kv_layout=case["layout"])
        s.batch = d2sd.PagedBatch(s.qo_indptr, s.kv_len, s.page_indptr, s.page_table, P)
        if case["kind"] == "attn":
            s.attn = d2sd.PagedChunkAttention().plan(s.batch, case["hq"], hkv, d, kv_format=fmt,
                                                     window_left=case["window"], sinks=s.sinks)
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    case = s.case
    if not own:
        return _PLAIN[case["kind"]](s)
    if case["kind"] == "rope":
        import d2sd
        return d2sd.rotary_embedding(s.q, s.k, s.positions, s.inv_freq, interleaved=case["interleaved"], scale=s.scale,
                                     inverse=case["inverse"], out=(s.q_out, s.k_out))
    if case["kind"] == "write":
        s.cache.write(s.k, s.v, s.batch)
        return s.cache.read(s.batch, new_only=True)
    if case["kind"] == "read":
        return s.cache.read(s.batch)
    return s.attn.run(s.q, s.cache)


def _rotate_plain(x, cos, sin, case):
    """Pairs (a, b) -> (a cos - b sin, b cos + a sin) in 32 bits; the rest of the head passes through."""
    n, r = x.shape[0], case["rotary"]
    y = x.float()
    part = y[..., :r].reshape(n, -1, r // 2, 2) if case["interleaved"] else \
        y[..., :r].reshape(n, -1, 2, r // 2).transpose(2, 3)
    a, b = part[..., 0], part[..., 1]
    c, t = cos[:, None], sin[:, None]
    z = torch.stack([a * c - b * t, b * c + a * t], dim=-1)
    z = z.reshape(n, -1, r) if case["interleaved"] else z.transpose(2, 3).reshape(n, -1, r)
    return torch.cat([z, y[..., r:]], dim=-1).to(x.dtype)


def _rope_plain(s):
    angle = s.positions.double()[:, None] * s.inv_freq[None]
    cos, sin = (angle.cos() * s.scale).float(), (angle.sin() * s.scale).float()
    sin = -sin if s.case["inverse"] else sin
    return _rotate_plain(s.q, cos, sin, s.case), _rotate_plain(s.k, cos, sin, s.case)


_E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
_RANGE = {"mxfp8": (448.0, 8, 1.75, 119), "mxfp4": (6.0, 2, 1.5, 125)}  # largest, its exponent, its fraction, top scale


def _two_to(e):
    """2^e in 32 bits, exactly (e from -126 to 127)."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _encode(x, fmt, scale=None):
    """Codes (and block scale bytes) of bf16 rows [..., heads, d]."""
    if fmt == "bf16":
        return x, None
    y = x.float()
    if fmt == "fp8":
        return (y / scale[:, None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn), None
    most, top, frac, hi = _RANGE[fmt]
    y = y.unflatten(-1, (-1, BLOCK))
    amax = y.abs().amax(-1)
    m, e = torch.frexp(amax)
    e = (e - 1 - top + (2 * m > frac).int()).clamp(-117, hi)
    e = torch.where(amax == 0, -117, e)
    finite = torch.isfinite(amax)
    y = (y * _two_to(-e)[..., None]).clamp(-most, most)
    y = torch.where(finite[..., None], y, torch.zeros_like(y)).flatten(-2)
    scales = torch.where(finite, e + 127, 255).to(torch.uint8)
    if fmt == "mxfp8":
        return y.to(torch.float8_e4m3fn), scales
    a = y.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = torch.round(a / step) * step
    code = torch.bucketize(a, torch.tensor(_E2M1, device=x.device)).to(torch.uint8)
    code = code | (torch.signbit(y).to(torch.uint8) << 3)
    return code[..., 0::2] | (code[..., 1::2] << 4), scales


def _decode(codes, scales, fmt):
    """32-bit values of cache rows [..., heads, width]; scales: per head (fp8) or of the same rows (mx)."""
    if fmt == "bf16":
        return codes.float()
    if fmt == "fp8":
        return codes.float() * scales[:, None]
    if fmt == "mxfp4":
        both = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2)
        values = torch.tensor(_E2M1 + [-v for v in _E2M1], device=codes.device)[both.int()]
    else:
        values = codes.float()
    factor = torch.where(scales == 255, torch.nan, _two_to(scales.int() - 127))
    return (values.unflatten(-1, (-1, BLOCK)) * factor[..., None]).flatten(-2)


def _rows(s, r, pos):
    """Pool pages and slots of positions `pos` of requests `r` (page ids of places past the end: the last one's)."""
    P = s.case["page"]
    at = s.page_indptr_dev.long()[r] + pos // P
    return s.page_table.long()[at.clamp(max=s.page_table.numel() - 1)], pos % P


def _fetch(s, page, slot):
    """Cache rows as [..., heads, d] values in 32 bits, keys and values."""
    take = lambda t: t[page, :, slot] if s.case["layout"] == "HND" else t[page, slot]  # noqa: E731
    got = []
    for pool, scale in ((s.k_pool, s.k_scale), (s.v_pool, s.v_scale)):
        codes = take(pool.view(torch.uint8)).view(pool.dtype) if pool.element_size() == 1 else take(pool)
        got.append(_decode(codes, take(scale) if s.case["fmt"].startswith("mx") else scale, s.case["fmt"]))
    return got


def _new_tokens(s):
    """Request and position of every new token."""
    t = torch.arange(s.qo_indptr[-1], device=DEV)
    ends = s.qo_indptr_dev.long()
    r = torch.searchsorted(ends[1:].contiguous(), t, right=True)
    return r, s.kv_len_dev.long()[r] - ends[r + 1] + t


def _write_plain(s):
    fmt, hnd = s.case["fmt"], s.case["layout"] == "HND"
    page, slot = _rows(s, *_new_tokens(s))
    for x, pool, scale in ((s.k, s.k_pool, s.k_scale), (s.v, s.v_pool, s.v_scale)):
        codes, scales = _encode(x, fmt, scale)
        if pool.element_size() == 1:
            pool, codes = pool.view(torch.uint8), codes.view(torch.uint8)
        if hnd:
            pool[page, :, slot] = codes
        else:
            pool[page, slot] = codes
        if scales is not None and hnd:
            scale[page, :, slot] = scales
        elif scales is not None:
            scale[page, slot] = scales
    k, v = _fetch(s, page, slot)
    return k.to(torch.bfloat16), v.to(torch.bfloat16)


def _read_plain(s):
    L = s.kv_len_dev.long()
    r = torch.repeat_interleave(torch.arange(L.numel(), device=DEV), L)
    pos = torch.arange(r.numel(), device=DEV) - (L.cumsum(0) - L)[r]
    k, v = _fetch(s, *_rows(s, r, pos))
    return k.to(torch.bfloat16), v.to(torch.bfloat16)


def _attn_plain(s):
    """Padded to the longest chunk and cache; hidden scores are -inf, places behind a cache's end 0."""
    c = s.case
    hq, hkv, d, g = c["hq"], c["hkv"], c["d"], c["hq"] // c["hkv"]
    ends, L = s.qo_indptr_dev.long(), s.kv_len_dev.long()
    R, T, N = L.numel(), s.max_qo, s.max_kv
    qlen = ends[1:] - ends[:-1]
    row = (ends[:-1, None] + torch.arange(T, device=DEV)).clamp(max=s.q.shape[0] - 1)
    q = s.q[row].float().view(R, T, hkv, g, d).permute(0, 2, 3, 1, 4).reshape(R, hkv, g * T, d)
    key = torch.arange(N, device=DEV)
    k, v = _fetch(s, *_rows(s, torch.arange(R, device=DEV)[:, None].expand(R, N), key.expand(R, N)))
    held = (key < L[:, None])[..., None, None]
    k = torch.where(held, k, 0.0).permute(0, 2, 3, 1).contiguous()
    v = torch.where(held, v, 0.0).transpose(1, 2).contiguous()
    x = torch.matmul(q, k).mul_(d ** -0.5)
    pos = (L - qlen)[:, None] + torch.arange(T, device=DEV)
    seen = key <= pos[..., None]
    if c["window"] >= 0:
        seen &= key > pos[..., None] - c["window"] - 1
    x = x.view(R, hkv, g, T, N).masked_fill_(~seen[:, None, None], -torch.inf)
    top = x.amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, 0.0)
    p = x.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(R, hkv, g * T, N), v).view(R, hkv, g, T, d) / total.clamp(min=1e-30)
    lse = (top + total.log())[..., 0]
    if s.sinks is not None:
        o = o * torch.sigmoid(lse - s.sinks.view(hkv, g, 1))[..., None]
    r, t = _new_tokens(s)
    t = t - (L - qlen)[r]
    o, lse = o.permute(0, 3, 1, 2, 4).reshape(R, T, hq, d)[r, t], lse.permute(0, 3, 1, 2).reshape(R, T, hq)[r, t]
    return o.to(torch.bfloat16), lse


_PLAIN = {"rope": _rope_plain, "write": _write_plain, "read": _read_plain, "attn": _attn_plain}


# ---------------------------------------------------------------------------
# what a pass cannot do without, and its results in 64 bits
# ---------------------------------------------------------------------------
_ROW = {"bf16": lambda d: 2 * d, "fp8": lambda d: d, "mxfp8": lambda d: d + d // BLOCK,
        "mxfp4": lambda d: d // 2 + d // BLOCK}


def work(case):
    d, hkv, hq = case["d"], case["hkv"], case["hq"]
    if case["kind"] == "rope":
        n = case["tokens"]
        return {"bytes": 2 * 2 * n * (hq + hkv) * d + 4 * n + 8 * (case["rotary"] // 2), "flops": 3.0 * n * (hq + hkv) * case["rotary"]}
    row, (qo, kv) = _ROW[case["fmt"]](d), _lens(case)
    if case["kind"] == "write":  # bf16 in, codes out, the values they stand for out
        return {"bytes": 2 * sum(qo) * hkv * (2 * d + row + 2 * d), "flops": 2.0 * sum(qo) * hkv * d}
    if case["kind"] == "read":
        return {"bytes": 2 * sum(kv) * hkv * (row + 2 * d), "flops": 0.0}
    keys = pairs = 0
    for n, L in zip(qo, kv):
        w = min(L, case["window"] + 1) if case["window"] >= 0 else L
        keys += min(L, w + n - 1)
        short = max(0, min(n, w - (L - n) - 1))  # queries whose window is not full
        pairs += (n - short) * w + sum(L - n + i + 1 for i in range(short))
    return {"bytes": 2 * keys * hkv * row + sum(qo) * hq * (4 * d + 4), "flops": 4.0 * pairs * hq * d}


def _grid(fmt):
    """The non-negative values of the elements, in the order of their codes."""
    if fmt == "mxfp4":
        return torch.tensor(_E2M1, dtype=torch.float64, device=DEV)
    codes = torch.arange(127)
    e, m = codes // 8, (codes % 8).double()
    return torch.where(e > 0, (1 + m / 8) * 2.0 ** (e - 7).double(), m / 8 * 2.0 ** -6).to(DEV)


def _nearest(y, grid):
    """|y| to the nearest value of the grid, ties to the even code, y's sign kept."""
    a = y.abs().clamp(max=float(grid[-1]))
    hi = torch.searchsorted(grid, a.contiguous()).clamp(1, grid.numel() - 1)
    lo = hi - 1
    down, up = a - grid[lo], grid[hi] - a
    take_lo = (down < up) | ((down == up) & (lo % 2 == 0))
    return torch.copysign(torch.where(take_lo, grid[lo], grid[hi]), y)


def _exact_values(x, fmt, scale):
    """What the cache stands for after bf16 rows [tokens, heads, d] were written to it."""
    y = x.double()
    if fmt == "bf16":
        return y
    if fmt == "fp8":
        return _nearest(y / scale.double()[:, None], _grid("mxfp8")) * scale.double()[:, None]
    grid = _grid(fmt)
    most, _, _, hi = _RANGE[fmt]
    y = y.reshape(*y.shape[:-1], -1, BLOCK)
    m, e = torch.frexp(y.abs().amax(-1) / most)
    e = torch.where(m == 0.5, e - 1, e).clamp(-117, hi)
    unit = ((e.long() + 1023) << 52).view(torch.float64)[..., None]
    return (_nearest(y / unit, grid) * unit).reshape(x.shape)


def _exact_cache(s, r):
    """Keys and values of request r, [len, heads, d] in 64 bits."""
    c, L, P = s.case, s.kv_len[r], s.case["page"]
    pages = s.page_table[s.page_indptr[r]:s.page_indptr[r + 1]].long()
    got = []
    for pool, scale in ((s.k_pool, s.k_scale), (s.v_pool, s.v_scale)):
        rows = lambda t: (t[pages].transpose(1, 2) if c["layout"] == "HND" else t[pages]).reshape(  # noqa: E731
            -1, c["hkv"], t.shape[-1])[:L]
        if c["fmt"] == "bf16":
            got.append(rows(pool).double())
            continue
        byte = rows(pool.view(torch.uint8)).long()
        if c["fmt"] == "mxfp4":
            byte = torch.stack([byte % 16, byte // 16], -1).reshape(L, c["hkv"], -1)
            x = _grid("mxfp4")[byte % 8] * torch.where(byte >= 8, -1.0, 1.0)
        else:
            x = _grid("mxfp8")[(byte % 128).clamp(max=126)] * torch.where(byte >= 128, -1.0, 1.0)
        if c["fmt"] == "fp8":
            got.append(x * scale.double()[:, None])
        else:
            got.append(x * ((rows(scale).long() + 896) << 52).view(torch.float64).repeat_interleave(BLOCK, -1))
    return got


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rope":
        r, outs = case["rotary"], []
        f = s.positions.double()[:, None] * s.inv_freq
        turn = torch.polar(torch.full_like(f, s.scale), -f if case["inverse"] else f)[:, None]
        for x in (s.q, s.k):
            y = x.double().clone()
            a, b = (y[..., 0:r:2], y[..., 1:r:2]) if case["interleaved"] else (y[..., :r // 2], y[..., r // 2:r])
            z = torch.complex(a, b) * turn
            a.copy_(z.real)
            b.copy_(z.imag)
            outs.append(y)
        return tuple(outs)
    if case["kind"] == "write":
        return _exact_values(s.k, case["fmt"], s.k_scale), _exact_values(s.v, case["fmt"], s.v_scale)
    if case["kind"] == "read":
        each = [_exact_cache(s, r) for r in range(case["reqs"])]
        return torch.cat([k for k, _ in each]), torch.cat([v for _, v in each])
    hq, g = case["hq"], case["hq"] // case["hkv"]
    out = torch.zeros((s.qo_indptr[-1], hq, case["d"]), dtype=torch.float64, device=DEV)
    lse = torch.full((s.qo_indptr[-1], hq), -torch.inf, dtype=torch.float64, device=DEV)
    for r in range(case["reqs"]):
        k, v = _exact_cache(s, r)
        a, b = s.qo_indptr[r], s.qo_indptr[r + 1]
        back = (s.kv_len[r] - (b - a) + torch.arange(b - a, device=DEV))[:, None] - torch.arange(s.kv_len[r], device=DEV)
        hidden = (back < 0) | (back > case["window"]) if case["window"] >= 0 else back < 0
        for h in range(hq):
            x = s.q[a:b, h].double() @ k[:, h // g].T.contiguous() / math.sqrt(case["d"])
            x = x.masked_fill(hidden, -torch.inf)
            lse[a:b, h] = torch.logsumexp(x, -1)
            out[a:b, h] = torch.softmax(x, -1) @ v[:, h // g].contiguous()
    if s.sinks is not None:
        out *= torch.sigmoid(lse - s.sinks.double())[..., None]
    return out, lse
