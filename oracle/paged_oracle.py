"""Plain 64-bit forms of the paged-cache operators (rotary embedding, cache write
and read, attention of new tokens over the cache), written from their formulas.
CPU, float64; test infrastructure only, like cascade_oracle.
"""
from __future__ import annotations

import math

import torch

BLOCK = 32
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def rotary_ref(x, positions, inv_freq, interleaved=False, scale=1.0, inverse=False):
    """Rotated heads [tokens, heads, D] (float64) and the size sum |a| + |b| of each element's pair."""
    r = 2 * inv_freq.numel()
    y = x.double().clone()
    size = torch.zeros_like(y)
    t = positions.double()[:, None] * inv_freq.double()[None]
    c, s = (t.cos() * scale)[:, None], (t.sin() * scale * (-1.0 if inverse else 1.0))[:, None]
    first = slice(0, r, 2) if interleaved else slice(0, r // 2)
    second = slice(1, r, 2) if interleaved else slice(r // 2, r)
    a, b = y[..., first].clone(), y[..., second].clone()
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    size[..., first] = size[..., second] = a.abs() + b.abs()
    return y, size


def element_grid(fmt):
    """Non-negative element values in code order."""
    if fmt == "mxfp4":
        return torch.tensor(E2M1, dtype=torch.float64)
    return torch.tensor([m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
                         for e in range(16) for m in range(8) if (e, m) != (15, 7)], dtype=torch.float64)


def nearest_code(y, grid):
    """Code (sign in the bit above) of the grid value nearest to y, ties to the even code, saturating."""
    a = y.abs().clamp(max=float(grid[-1]))
    hi = torch.searchsorted(grid, a.contiguous()).clamp(1, grid.numel() - 1)
    lo = hi - 1
    down, up = a - grid[lo], grid[hi] - a
    code = torch.where((down < up) | ((down == up) & (lo % 2 == 0)), lo, hi)
    return code + torch.signbit(y).long() * (128 if grid.numel() > 8 else 8)


def quantise_ref(x, fmt, scale=None):
    """(codes, scale bytes) that bf16 rows [..., heads, D] become in the cache.
    Codes: bf16 values, e4m3fn bytes or e2m1 codes (one per element), int64 bytes."""
    if fmt == "bf16":
        return x.clone(), None
    y = x.double()
    if fmt == "fp8":
        q = (x.float() / scale.float()[:, None]).double()  # the quotient is rounded to 32 bits first
        code = nearest_code(torch.nan_to_num(q, nan=0.0, posinf=448.0, neginf=-448.0), element_grid(fmt))
        return torch.where(torch.isnan(q), 127, code), None
    most, hi = (6.0, 125) if fmt == "mxfp4" else (448.0, 119)
    y = y.unflatten(-1, (-1, BLOCK))
    amax = y.abs().amax(-1)
    bad = ~torch.isfinite(y).all(-1)
    m, e = torch.frexp(torch.where(bad, 0.0, amax) / most)  # amax / most = m 2^e, m in [1/2, 1)
    e = torch.where(m == 0.5, e - 1, e)
    e = torch.where(amax == 0, -117, e).clamp(-117, hi)
    y = torch.where(bad[..., None], 0.0, y * 2.0 ** -e.double()[..., None])
    return nearest_code(y, element_grid(fmt)).flatten(-2), torch.where(bad, 255, e + 127)


def values_ref(codes, scales, fmt, scale=None):
    """float64 values of codes as quantise_ref gives them."""
    if fmt == "bf16":
        return codes.double()
    grid, sign = element_grid(fmt), 8 if fmt == "mxfp4" else 128
    mag = codes % sign
    v = torch.where(mag >= grid.numel(), math.nan, grid[mag.clamp(max=grid.numel() - 1)])
    v = torch.where(codes >= sign, -v, v)
    if fmt == "fp8":
        return v * scale.double()[:, None]
    f = torch.where(scales == 255, math.nan, 2.0 ** (scales.double() - 127))
    return (v.unflatten(-1, (-1, BLOCK)) * f[..., None]).flatten(-2)


def pack_codes(codes, fmt):
    """Codes as the cache stores them (bytes; mxfp4 two to a byte, even element low)."""
    if fmt == "mxfp4":
        return (codes[..., 0::2] + 16 * codes[..., 1::2]).to(torch.uint8)
    return codes if fmt == "bf16" else codes.to(torch.uint8)


def attention_ref(q, k, v, pos0, group, sm_scale, window_left=-1, sinks=None):
    """One request: q [n, Hq, D] at positions pos0 .., keys and values
    [len, Hkv, D] (float64).  Returns o, lse (natural log) and, for tolerances,
    sum_j p_j |v_j| and the largest sum_i |q_i k_ij| sm_scale of each row."""
    n, hq, d = q.shape
    L = k.shape[0]
    pos = pos0 + torch.arange(n)[:, None]
    key = torch.arange(L)[None]
    seen = key <= pos
    if window_left >= 0:
        seen &= key >= pos - window_left
    o, spread = torch.zeros(n, hq, d, dtype=torch.float64), torch.zeros(n, hq, d, dtype=torch.float64)
    lse = torch.full((n, hq), -math.inf, dtype=torch.float64)
    size = torch.zeros(n, hq, dtype=torch.float64)
    if L:
        for h in range(hq):
            kh, vh = k[:, h // group].double(), v[:, h // group].double()
            qh = q[:, h].double()
            x = torch.where(seen, qh @ kh.T * sm_scale, -math.inf)
            lse[:, h] = torch.logsumexp(x, -1)
            p = torch.where(seen, torch.exp(x - torch.where(torch.isfinite(lse[:, h]), lse[:, h], 0.0)[:, None]), 0.0)
            o[:, h], spread[:, h] = p @ vh, p @ vh.abs()
            size[:, h] = (torch.where(seen, qh.abs() @ kh.abs().T, 0.0) * sm_scale).amax(-1)
    if sinks is not None:
        f = torch.sigmoid(lse - sinks.double())[..., None]
        o, spread = o * f, spread * f
    return o, lse, spread, size
