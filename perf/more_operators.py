"""What a layer does with its new tokens on the way into a paged cache, and attention for requests whose caches begin
alike: the calls of a serving loop whose conversations share a system prompt or a document.

Kinds of case
  append  new queries, keys and values from the projection: (RMS norm of each query and key head,) both rotated at
          their positions, queries out, keys and values into their pages, quantised if the cache is.  What the cache
          holds of a bf16 cache is the pools themselves; of the others, the step's tokens read back
  shared  causal attention of each request's newest tokens over its paged cache, which already holds them, where
          groups of neighbouring requests hold the same first tokens

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
EPS = 1e-6


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _append(name, **c):
    c = dict(dict(kind="append", hq=32, hkv=8, d=128, fmt="bf16", layout="HND", page=16, reqs=1, kv_lo=1, kv_hi=1, new=1,
                  norm=False, rotary=128, interleaved=False, base=1e6, stretch="none", factor=1.0, trained=4096, far=0,
                  shape=0), **c)
    return dict(name=name, **c) if name else c


def _shared(name, **c):
    """groups: requests of each group; prefix: tokens that a group's requests share; own_lo .. own_hi: tokens of a
    request behind them, the new ones (new_lo .. new_hi) included."""
    c = dict(dict(kind="shared", hq=32, hkv=8, d=128, fmt="bf16", layout="HND", page=16, groups="1", prefix="0",
                  own_lo=1, own_hi=1, new_lo=1, new_hi=1, window=-1, sinks=False, shape=0), **c)
    return dict(name=name, **c) if name else c


def listed():
    return [
        # the smallest step: one conversation's next token, queries and keys normed
        _append("append_decode_one", kv_lo=1000, kv_hi=1000, norm=True),
        # a decoding step of 48 conversations into a quantised cache
        _append("append_decode_48_mxfp8", fmt="mxfp8", reqs=48, kv_lo=200, kv_hi=1500, norm=True),
        # interleaved pairs over half of each head, at positions far inside a document that other caches hold the
        # rest of; token-major pages, odd lengths
        _append("append_document_fp8", hq=28, hkv=4, fmt="fp8", layout="NHD", page=64, reqs=3, kv_lo=300, kv_hi=1100,
                new=0, rotary=64, interleaved=True, base=10000.0, stretch="linear", factor=8.0, far=1000000),
        # a prefill batch at head size 64, frequencies stretched 32 times, into the smallest cache
        _append("append_prompts_mxfp4_d64", hq=64, d=64, fmt="mxfp4", reqs=5, kv_lo=1000, kv_hi=3000, new=0, rotary=64,
                base=150000.0, stretch="yarn", factor=32.0),
        # the largest: an 8K prompt
        _append("append_prompt_8k", hq=64, kv_lo=8192, kv_hi=8192, new=0, norm=True),
        # the smallest attention: four conversations under one short system prompt
        _shared("shared_decode_4", groups="4", prefix="2003", own_lo=20, own_hi=300),
        # a server decoding 32 conversations under a system prompt with tools
        _shared("shared_decode_32_mxfp8", fmt="mxfp8", groups="32", prefix="8192", own_lo=100, own_hi=1200),
        # 64 short questions about one long document
        _shared("shared_decode_64_bf16", groups="64", prefix="16384", own_lo=50, own_hi=500),
        # head size 64 with sinks: 12 conversations whose drafts of 7 tokens are verified
        _shared("shared_drafts_d64_sinks", hq=64, d=64, fmt="fp8", groups="12", prefix="5000", own_lo=100, own_hi=900,
                new_lo=7, new_hi=7, sinks=True, shape=1),
        # two prompts shared by several, one conversation by itself, a window that hides a part of what is shared
        _shared("shared_two_groups_window", fmt="mxfp4", groups="9,1,14", prefix="3100,0,6001", own_lo=300, own_hi=2500,
                window=4095, shape=2),
        # chunks of prompts that go on from the same document
        _shared("shared_chunks_mxfp4", fmt="mxfp4", groups="6", prefix="8192", own_lo=100, own_hi=700, new_lo=100,
                new_hi=700, shape=3),
        # the largest: 96 conversations about a 32K document
        _shared("shared_decode_96_32k", hq=64, fmt="mxfp8", groups="96", prefix="32768", own_lo=200, own_hi=3000, shape=4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(32, 8, 128), (32, 8, 128), (64, 8, 128), (64, 8, 64), (28, 4, 128), (16, 16, 64)]
MOST_SCORES = 2e9    # padded score matrix of the plain form
MOST_FLOPS = 1.2e11
MOST_TOKENS = 2.5e5  # of all caches


def draw(rng):
    hq, hkv, d = rng.choice(HEADS)
    c = dict(hq=hq, hkv=hkv, d=d, fmt=rng.choice(["bf16", "bf16", "fp8", "mxfp8", "mxfp8", "mxfp4"]),
             layout=rng.choice(["HND", "HND", "NHD"]), page=rng.choice([16, 16, 32, 64, 128]), shape=rng.randrange(1 << 16))
    if rng.random() < 0.45:
        c["stretch"] = rng.choice(["none", "linear", "yarn", "wavelength"])
        c.update(norm=rng.random() < 0.5, rotary=rng.choice([d, d, d // 2, d // 4]), interleaved=rng.random() < 0.4,
                 base=rng.choice([1e4, 1.5e5, 1e6]), factor=1.0 if c["stretch"] == "none" else rng.choice([2.0, 8.0, 32.0]),
                 far=rng.choice([0, 0, _log(rng, 8192, 1000000)]), reqs=_log(rng, 1, 64), kv_lo=_log(rng, 16, 8192))
        c["kv_hi"] = min(8192, int(c["kv_lo"] * rng.uniform(1.0, 4.0)))
        c["new"] = rng.choice([1, 1, 0, 0, rng.randint(2, 9)])
        while c["reqs"] * c["kv_hi"] > (8192 if c["new"] == 0 else 60000):
            if c["reqs"] > 2:
                c["reqs"] = c["reqs"] * 2 // 3
            else:
                c["kv_lo"], c["kv_hi"] = c["kv_lo"] // 2 + 1, c["kv_hi"] // 2 + 1
        return _append(None, **c)
    reqs = _log(rng, 2, 96)
    cuts = sorted(rng.sample(range(1, reqs), min(reqs - 1, rng.choice([0, 0, 0, 1, 2, 3]))))
    groups = [b - a for a, b in zip([0] + cuts, cuts + [reqs])]
    prefix = [_log(rng, 64, 32768) if n > 1 else rng.choice([0, _log(rng, 64, 4096)]) for n in groups]
    c["own_lo"] = _log(rng, 1, 1000)
    c["own_hi"] = min(4000, int(c["own_lo"] * rng.uniform(1.0, 6.0)))
    c["new_lo"] = c["new_hi"] = 1
    if rng.random() < 0.35:
        c["new_lo"], c["new_hi"] = 1, rng.randint(2, 9)
    elif rng.random() < 0.3:
        c["new_hi"] = _log(rng, 10, 1000)
        c["new_lo"] = rng.randint(1, c["new_hi"])
    c["window"] = rng.choice([-1, -1, -1, -1, rng.randint(0, 8000)])
    c["sinks"] = rng.random() < 0.3
    while True:
        case = _shared(None, groups=",".join(map(str, groups)), prefix=",".join(map(str, prefix)), **c)
        first, lens, new, _ = _lens(case)
        scores = max((b - a) * max(new[a:b]) * (p + max(lens[a:b])) for a, b, p in zip(first, first[1:], prefix)) * hq
        flops = sum(sum(new[a:b]) * (p + max(lens[a:b])) for a, b, p in zip(first, first[1:], prefix)) * 4.0 * hq * d
        if scores <= MOST_SCORES and flops <= MOST_FLOPS and sum(lens) + sum(prefix) <= MOST_TOKENS:
            return case
        if c["new_hi"] > 32:
            c["new_lo"], c["new_hi"] = c["new_lo"] * 2 // 3 + 1, c["new_hi"] * 2 // 3
        elif sum(lens) > sum(prefix):
            c["own_lo"], c["own_hi"] = c["own_lo"] // 2 + 1, c["own_hi"] // 2 + 1
        else:
            prefix = [p * 3 // 4 for p in prefix]


def _lens(case):
    """append: (new tokens, cache lengths) of each request, new == 0: every token is new.  shared: (first request of
    each group and the end, own tokens, new tokens, shared tokens of each request)."""
    rng = random.Random(case["shape"])
    if case["kind"] == "append":
        kv = [rng.randint(case["kv_lo"], case["kv_hi"]) for _ in range(case["reqs"])]
        return [min(n, case["new"] or n) for n in kv], kv
    groups, prefix = ([int(x) for x in case[k].split(",")] for k in ("groups", "prefix"))
    first = [0]
    for n in groups:
        first.append(first[-1] + n)
    lens = [rng.randint(case["own_lo"], case["own_hi"]) for _ in range(first[-1])]
    new = [min(n, rng.randint(case["new_lo"], case["new_hi"])) for n in lens]
    return first, lens, new, [p for n, p in zip(groups, prefix) for _ in range(n)]


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
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
    s, gen = _State(), torch.Generator(device=DEV).manual_seed(int(seed))
    s.case = case
    hq, hkv, d, P, fmt = case["hq"], case["hkv"], case["d"], case["page"], case["fmt"]
    if case["kind"] == "append":
        new, kv = _lens(case)
        shared = [0] * len(kv)
    else:
        s.first, own_len, new, shared = _lens(case)
        kv = [a + b for a, b in zip(own_len, shared)]
    # pages in random order; the full pages of what a group shares are in the tables of all its requests, and the
    # page that it ends in is in each one's own
    s.qo_indptr, s.page_indptr, table, used, at_page = [0], [0], [], 0, []
    for r in range(len(kv)):
        n = -(-kv[r] // P)
        full = shared[r] // P if case["kind"] == "shared" and r not in s.first else 0
        lead = table[s.page_indptr[s.first[_group(s, r)]]:][:full] if full else []
        table += lead + list(range(used, used + n - full))
        at_page.append(used - full)
        used += n - full
        s.qo_indptr.append(s.qo_indptr[-1] + new[r])
        s.page_indptr.append(len(table))
    pages = used + 4
    order = np.random.default_rng(seed).permutation(pages).astype(np.int32)
    s.page_table = torch.from_numpy(order[np.asarray(table)]).to(DEV)
    at = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    s.qo_indptr_dev, s.page_indptr_dev, s.kv_len_dev = at(s.qo_indptr), at(s.page_indptr), at(kv)
    s.kv_len, s.new, s.shared = kv, new, shared
    total = s.qo_indptr[-1]
    # pools with every page in use filled through the plain quantiser
    pools = []
    for _ in range(2):
        x = _states(gen, pages, P, hkv, d)
        for r in range(len(kv)):
            tail = shared[r] % P
            if case["kind"] == "shared" and r not in s.first and tail:
                src = order[table[s.page_indptr[s.first[_group(s, r)]] + shared[r] // P]]
                x[int(order[table[s.page_indptr[r] + shared[r] // P]]), :tail] = x[int(src), :tail]
        scale = (x.float().abs().amax(dim=(0, 1, 3)) / 448.0).contiguous() if fmt == "fp8" else None
        codes, scales = _encode(x, fmt, scale)
        x = None
        if case["layout"] == "HND":
            codes = codes.transpose(1, 2).contiguous()
            scales = scales.transpose(1, 2).contiguous() if scales is not None else None
        pools.append((codes, scale if fmt == "fp8" else scales))
    (s.k_pool, s.k_scale), (s.v_pool, s.v_scale) = pools
    if case["kind"] == "append":
        qkv = torch.randn((total, hq + 2 * hkv, d), generator=gen, device=DEV)
        lift = 1.0 + 5.0 * (torch.rand((hq + 2 * hkv, d), generator=gen, device=DEV) < 0.03).float()
        qkv = (qkv * lift).to(torch.bfloat16)  # the fused projection's output; its parts are views
        s.q, s.k, s.v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        s.q_out = torch.empty((total, hq, d), dtype=torch.bfloat16, device=DEV)
        s.q_norm = s.k_norm = s.positions = None
        if case["norm"]:
            s.q_norm, s.k_norm = ((1.0 + 0.3 * torch.randn(d, generator=gen, device=DEV)).to(torch.bfloat16) for _ in range(2))
        if case["far"]:  # this batch's caches begin at a position of their own
            start = torch.randint(0, case["far"], (len(kv),), generator=gen, device=DEV)
            r, pos = _new_tokens(s)
            s.positions = (start[r] + pos).to(torch.int32)
        f, s.scale = _frequencies(case)
        s.inv_freq = f.to(DEV)
    else:
        s.q = torch.randn((total, hq, d), generator=gen, device=DEV).to(torch.bfloat16)
        s.sinks = torch.randn(hq, generator=gen, device=DEV) if case["sinks"] else None
    if own:
        import d2sd
        s.cache = d2sd.PagedKVCache(s.k_pool, s.v_pool, fmt, k_scale=s.k_scale, v_scale=s.v_scale,
                                    kv_layout=case["layout"])
        s.batch = d2sd.PagedBatch(s.qo_indptr, s.kv_len, s.page_indptr, s.page_table, P)
        if case["kind"] == "shared":
            s.attn = d2sd.PagedChunkAttention().plan(s.batch, hq, hkv, d, kv_format=fmt, window_left=case["window"],
                                                     sinks=s.sinks, shared_indptr=s.first,
                                                     shared_len=[shared[a] for a in s.first[:-1]])
    return s


def _group(s, r):
    return max(i for i, a in enumerate(s.first[:-1]) if a <= r)


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    case = s.case
    if not own:
        return _append_plain(s) if case["kind"] == "append" else _shared_plain(s)
    if case["kind"] == "shared":
        return s.attn.run(s.q, s.cache)
    s.cache.append(s.q, s.k, s.v, s.batch, s.inv_freq, s.positions, scale=s.scale, interleaved=case["interleaved"],
                   q_norm=s.q_norm, k_norm=s.k_norm, eps=EPS, q_out=s.q_out)
    if case["fmt"] == "bf16":
        return s.q_out, s.k_pool, s.v_pool
    return (s.q_out, *s.cache.read(s.batch, new_only=True))


_E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
_RANGE = {"mxfp8": (448.0, 8, 1.75, 119), "mxfp4": (6.0, 2, 1.5, 125)}  # largest, its exponent, its fraction, top scale


def _two_to(e):
    """2^e in 32 bits, exactly (e from -126 to 127)."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _encode(x, fmt, scale=None):
    """Codes (and block scale bytes) of rows [..., heads, d] in 32 bits or bf16."""
    if fmt == "bf16":
        return x.to(torch.bfloat16), None
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


def _turned(x, weight, cos, sin, case):
    """Rows [tokens, heads, d] normed (with a weight) and rotated, in 32 bits."""
    n, r = x.shape[0], case["rotary"]
    y = x.float()
    if weight is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * weight.float()
    part = y[..., :r].reshape(n, -1, r // 2, 2) if case["interleaved"] else \
        y[..., :r].reshape(n, -1, 2, r // 2).transpose(2, 3)
    a, b = part[..., 0], part[..., 1]
    c, t = cos[:, None], sin[:, None]
    z = torch.stack([a * c - b * t, b * c + a * t], dim=-1)
    z = z.reshape(n, -1, r) if case["interleaved"] else z.transpose(2, 3).reshape(n, -1, r)
    return torch.cat([z, y[..., r:]], dim=-1)


def _append_plain(s):
    case, fmt, hnd = s.case, s.case["fmt"], s.case["layout"] == "HND"
    r, pos = _new_tokens(s)
    angle = (pos if s.positions is None else s.positions).double()[:, None] * s.inv_freq[None]
    cos, sin = (angle.cos() * s.scale).float(), (angle.sin() * s.scale).float()
    s.q_out.copy_(_turned(s.q, s.q_norm, cos, sin, case).to(torch.bfloat16))
    page, slot = _rows(s, r, pos)
    for x, pool, scale in ((_turned(s.k, s.k_norm, cos, sin, case), s.k_pool, s.k_scale), (s.v, s.v_pool, s.v_scale)):
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
    if fmt == "bf16":
        return s.q_out, s.k_pool, s.v_pool
    k, v = _fetch(s, page, slot)
    return s.q_out, k.to(torch.bfloat16), v.to(torch.bfloat16)


def _shared_plain(s):
    """Each group's shared keys once, for the queries of all its requests, and their own keys padded to the longest;
    hidden scores are -inf, places behind a cache's end 0."""
    c = s.case
    hq, hkv, d, g = c["hq"], c["hkv"], c["d"], c["hq"] // c["hkv"]
    ends, L = s.qo_indptr_dev.long(), s.kv_len_dev.long()
    out = torch.empty_like(s.q)
    lse_out = torch.empty(s.q.shape[:2], device=DEV)
    for a, b in zip(s.first, s.first[1:]):
        R, T, S = b - a, max(s.new[a:b]), s.shared[a]
        N = max(s.kv_len[a:b]) - S
        left, length, begin = ends[a + 1:b + 1] - ends[a:b], L[a:b], ends[a:b]
        row = (begin[:, None] + torch.arange(T, device=DEV)).clamp(max=s.q.shape[0] - 1)
        q = s.q[row].float().view(R, T, hkv, g, d).permute(2, 0, 3, 1, 4)  # [hkv, R, g, T, d]
        q = q.contiguous().mul_(d ** -0.5)
        pos = (length - left)[:, None] + torch.arange(T, device=DEV)      # [R, T]

        def hidden(key):  # keys [..., n] against positions: [..., T, n]
            h = key > pos[..., None]
            return h | (key < pos[..., None] - c["window"]) if c["window"] >= 0 else h

        # own keys
        key = S + torch.arange(N, device=DEV)
        k, v = _fetch(s, *_rows(s, torch.arange(a, b, device=DEV)[:, None].expand(R, N), key.expand(R, N)))
        held = (key < length[:, None])[..., None, None]
        k = torch.where(held, k, 0.0).permute(2, 0, 3, 1).contiguous()    # [hkv, R, d, N]
        v = torch.where(held, v, 0.0).permute(2, 0, 1, 3).contiguous()    # [hkv, R, N, d]
        x = torch.matmul(q.view(hkv, R, g * T, d), k).view(hkv, R, g, T, N)
        x.masked_fill_(hidden(key)[:, None], -torch.inf)
        top = x.amax(-1, keepdim=True)
        if S:  # shared keys
            key = torch.arange(S, device=DEV)
            ks, vs = _fetch(s, *_rows(s, torch.full((S,), a, device=DEV), key))
            ks, vs = ks.permute(1, 2, 0).contiguous(), vs.transpose(0, 1).contiguous()
            y = torch.matmul(q.view(hkv, R * g * T, d), ks).view(hkv, R, g, T, S)
            y.masked_fill_(hidden(key)[:, None], -torch.inf)
            top = torch.maximum(top, y.amax(-1, keepdim=True))
        top = torch.where(torch.isfinite(top), top, 0.0)
        p = x.sub_(top).exp_()
        total = p.sum(-1, keepdim=True)
        o = torch.matmul(p.view(hkv, R, g * T, N), v).view(hkv, R, g, T, d)
        if S:
            p = y.sub_(top).exp_()
            total = total + p.sum(-1, keepdim=True)
            o = o + torch.matmul(p.view(hkv, R * g * T, S), vs).view(hkv, R, g, T, d)
        o = o / total.clamp(min=1e-30)
        lse = (top + total.log())[..., 0]
        if s.sinks is not None:
            o = o * torch.sigmoid(lse - s.sinks.view(hkv, 1, g, 1))[..., None]
        r = torch.repeat_interleave(torch.arange(R, device=DEV), left)
        t = torch.arange(s.qo_indptr[a], s.qo_indptr[b], device=DEV) - begin[r]
        rows = slice(s.qo_indptr[a], s.qo_indptr[b])
        out[rows] = o.permute(1, 3, 0, 2, 4).reshape(R, T, hq, d)[r, t].to(torch.bfloat16)
        lse_out[rows] = lse.permute(1, 3, 0, 2).reshape(R, T, hq)[r, t]
    return out, lse_out


# ---------------------------------------------------------------------------
# what a pass cannot do without, and its results in 64 bits
# ---------------------------------------------------------------------------
_ROW = {"bf16": lambda d: 2 * d, "fp8": lambda d: d, "mxfp8": lambda d: d + d // BLOCK,
        "mxfp4": lambda d: d // 2 + d // BLOCK}


def work(case):
    d, hkv, hq = case["d"], case["hkv"], case["hq"]
    row = _ROW[case["fmt"]](d)
    if case["kind"] == "append":
        n, rotated = sum(_lens(case)[0]), case["rotary"] + (4 * d if case["norm"] else 0)
        back = 0 if case["fmt"] == "bf16" else 2 * d  # read back as the values they stand for
        return {"bytes": n * (hq * 4 * d + hkv * 2 * (2 * d + row + back) + 16),
                "flops": 3.0 * n * (hq + hkv) * rotated + 2.0 * n * hkv * d}
    first, own_len, new, shared = _lens(case)
    keys, pairs = 0, 0
    for a, b in zip(first, first[1:]):
        seen = [[], []]  # of the shared keys: first and end that some row sees
        for r in range(a, b):
            n, L, S = new[r], own_len[r] + shared[r], shared[r]
            lo = max(0, L - n - case["window"]) if case["window"] >= 0 else 0
            keys += L - max(lo, S)
            if S > lo:
                seen[0].append(lo)
                seen[1].append(S)
            w = min(L, case["window"] + 1) if case["window"] >= 0 else L
            short = max(0, min(n, w - (L - n) - 1))  # queries whose window is not full
            pairs += (n - short) * w + sum(L - n + i + 1 for i in range(short))
        keys += max(seen[1]) - min(seen[0]) if seen[0] else 0
    return {"bytes": 2 * keys * hkv * row + sum(new) * hq * (4 * d + 4), "flops": 4.0 * pairs * hq * d}


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


def _exact_values(y, fmt, scale):
    """What the cache stands for after rows [tokens, heads, d] in 64 bits were written to it."""
    if fmt == "bf16":
        return y
    if fmt == "fp8":  # (the format's quotient is one of 32 bits: on ties of the elements it decides)
        return _nearest((y / scale.double()[:, None]).float().double(), _grid("mxfp8")) * scale.double()[:, None]
    grid = _grid(fmt)
    most, _, _, hi = _RANGE[fmt]
    x = y.reshape(*y.shape[:-1], -1, BLOCK)
    m, e = torch.frexp(x.abs().amax(-1) / most)
    e = torch.where(m == 0.5, e - 1, e).clamp(-117, hi)
    unit = ((e.long() + 1023) << 52).view(torch.float64)[..., None]
    return (_nearest(x / unit, grid) * unit).reshape(y.shape)


def _exact_cache(s, r):
    """Keys and values of request r through its own table, [len, heads, d] in 64 bits."""
    c, L = s.case, s.kv_len[r]
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


def _exact_turned(x, weight, turn, case):
    y, r = x.double().clone(), case["rotary"]
    if weight is not None:
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + EPS) * weight.double()
    a, b = (y[..., 0:r:2], y[..., 1:r:2]) if case["interleaved"] else (y[..., :r // 2], y[..., r // 2:r])
    z = torch.complex(a, b) * turn
    a.copy_(z.real)
    b.copy_(z.imag)
    return y


def exact(case, seed):
    s = prepare(case, seed)
    R = len(s.kv_len)
    if case["kind"] == "append":
        where = [(r, s.kv_len[r] - s.new[r] + i) for r in range(R) for i in range(s.new[r])]
        pos = torch.tensor([p for _, p in where], dtype=torch.float64, device=DEV)
        f = (pos if s.positions is None else s.positions.double())[:, None] * s.inv_freq
        turn = torch.polar(torch.full_like(f, s.scale), f)[:, None]
        q = _exact_turned(s.q, s.q_norm, turn, case)
        k = _exact_values(_exact_turned(s.k, s.k_norm, turn, case), case["fmt"], s.k_scale)
        v = _exact_values(s.v.double(), case["fmt"], s.v_scale)
        if case["fmt"] != "bf16":
            return q, k, v
        table = s.page_table.tolist()
        page = torch.tensor([table[s.page_indptr[r] + p // case["page"]] for r, p in where], device=DEV)
        slot = torch.tensor([p % case["page"] for _, p in where], device=DEV)
        pools = s.k_pool.double(), s.v_pool.double()
        for pool, x in zip(pools, (k, v)):
            (pool.transpose(1, 2) if case["layout"] == "HND" else pool)[page, slot] = x
        return q, *pools
    hq, g = case["hq"], case["hq"] // case["hkv"]
    out = torch.zeros((s.qo_indptr[-1], hq, case["d"]), dtype=torch.float64, device=DEV)
    lse = torch.full((s.qo_indptr[-1], hq), -torch.inf, dtype=torch.float64, device=DEV)
    for r in range(R):
        k, v = (x.transpose(0, 1).contiguous() for x in _exact_cache(s, r))
        a, b = s.qo_indptr[r], s.qo_indptr[r + 1]
        back = (s.kv_len[r] - (b - a) + torch.arange(b - a, device=DEV))[:, None] - torch.arange(s.kv_len[r], device=DEV)
        hidden = (back < 0) | (back > case["window"]) if case["window"] >= 0 else back < 0
        for h in range(case["hkv"]):
            q = s.q[a:b, h * g:(h + 1) * g].transpose(0, 1).double().reshape(g * (b - a), -1)
            x = (q @ k[h].T.contiguous() / math.sqrt(case["d"])).view(g, b - a, -1)
            x = x.masked_fill(hidden, -torch.inf)
            lse[a:b, h * g:(h + 1) * g] = torch.logsumexp(x, -1).T
            o = torch.softmax(x, -1).view(g * (b - a), -1) @ v[h]
            out[a:b, h * g:(h + 1) * g] = o.view(g, b - a, -1).transpose(0, 1)
    if s.sinks is not None:
        out *= torch.sigmoid(lse - s.sinks.double())[..., None]
    return out, lse
