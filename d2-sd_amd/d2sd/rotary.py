"""Rotary embedding of new queries and keys at their positions (libd2sd.so).

qk_norm_rope rotates with the reference's bf16 table and its rounding steps
(generation/verification.py:113-123).  rotary_embedding takes positions and
frequencies instead: half or interleaved pairs, part of the head, any position
(per token, as far as a long document goes), in place or not, forwards or
back.  The angles are computed in the kernel, in turns, from 64-bit products;
cos and sin are 32-bit and the result is rounded to bf16 once.
"""
from __future__ import annotations

import math
from typing import Mapping, Optional, Tuple

import torch

from . import _lib  # noqa: F401  (registers torch.ops.d2sd)
from .graph import keep_alive

_rotary = torch.ops.d2sd.rotary_embedding.default


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: Optional[Mapping] = None,
                       device=None) -> Tuple[torch.Tensor, float]:
    """(inv_freq [rotary_dim / 2] float64 radians per position, factor on cos
    and sin) for rotary_embedding: base ** (-2i / rotary_dim), stretched for
    contexts longer than the trained one by `scaling`, a mapping with "type":

      "linear"      factor: every frequency divided by it
      "ntk"         factor: base times factor ** (d / (d - 2)), d = rotary_dim
      "dynamic"     factor, original_max_position, seq_len: "ntk" with
                    factor * seq_len / original_max_position - (factor - 1),
                    from the trained length on
      "yarn"        factor, original_max_position, beta_fast=32, beta_slow=1,
                    attention_factor=0.1 ln(factor) + 1, truncate=True: pairs
                    that make fewer than beta_slow turns over the trained
                    length are divided by factor, those with more than
                    beta_fast kept, a linear ramp over the pair index between
      "wavelength"  factor, low_freq_factor, high_freq_factor,
                    original_max_position: the same by turns: below
                    low_freq_factor divided, above high_freq_factor kept, a
                    linear blend in the number of turns between
      "per_pair"    factors [rotary_dim / 2], attention_factor=1: each
                    frequency divided by its own factor
    """
    d = int(rotary_dim)
    if d < 2 or d % 2:
        raise ValueError("rotary_dim must be positive and even")
    base = float(base)
    if not (base > 1.0 and math.isfinite(base)):
        raise ValueError("base must be finite and above 1")
    s = dict(scaling) if scaling else {"type": "none"}
    kind = s.pop("type", None)
    scale = 1.0
    i = torch.arange(0, d, 2, dtype=torch.float64)

    def take(name, default=None):
        v = s.pop(name, default)
        if v is None:
            raise ValueError(f"scaling {kind!r} needs {name!r}")
        return v

    def positive(name, default=None):
        v = float(take(name, default))
        if not (v > 0.0 and math.isfinite(v)):
            raise ValueError(f"scaling {kind!r}: {name} must be positive and finite")
        return v

    if kind in ("ntk", "dynamic"):
        if d == 2:
            raise ValueError(f"scaling {kind!r} needs a rotary_dim above 2")
        factor = positive("factor")
        if kind == "dynamic":
            n0 = positive("original_max_position")
            factor = factor * max(positive("seq_len"), n0) / n0 - (factor - 1.0)
        base = base * factor ** (d / (d - 2))
    f = base ** (-i / d)
    if kind == "linear":
        f = f / positive("factor")
    elif kind == "yarn":
        factor, n0 = positive("factor"), positive("original_max_position")
        fast, slow = positive("beta_fast", 32.0), positive("beta_slow", 1.0)
        scale = positive("attention_factor", 0.1 * math.log(factor) + 1.0 if factor > 1.0 else 1.0)
        # the (real) pair index that makes `turns` turns over n0 positions
        pair = lambda turns: d * math.log(n0 / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))  # noqa: E731
        lo, hi = pair(fast), pair(slow)
        if bool(take("truncate", True)):
            lo, hi = math.floor(lo), math.ceil(hi)
        lo, hi = max(lo, 0), min(hi, d - 1)
        ramp = ((i / 2 - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
        f = f / factor * ramp + f * (1.0 - ramp)
    elif kind == "wavelength":
        factor, n0 = positive("factor"), positive("original_max_position")
        low, high = positive("low_freq_factor"), positive("high_freq_factor")
        if not high > low:
            raise ValueError("scaling 'wavelength': high_freq_factor must be above low_freq_factor")
        keep = ((n0 * f / (2.0 * math.pi) - low) / (high - low)).clamp(0.0, 1.0)
        f = f / factor * (1.0 - keep) + f * keep
    elif kind == "per_pair":
        factors = torch.as_tensor(take("factors"), dtype=torch.float64, device="cpu").reshape(-1)
        if factors.numel() != d // 2 or not bool((factors > 0).all()):
            raise ValueError("scaling 'per_pair' needs one positive factor per pair")
        scale = positive("attention_factor", 1.0)
        f = f / factors
    elif kind not in ("none", "default", "ntk", "dynamic"):
        raise ValueError(f"unknown scaling type {kind!r}")
    if s:
        raise ValueError(f"scaling {kind!r}: unknown entries {sorted(s)}")
    return (f if device is None else f.to(device)), scale


def rotary_embedding(q: Optional[torch.Tensor], k: Optional[torch.Tensor], positions: torch.Tensor,
                     inv_freq: torch.Tensor, *, interleaved: bool = False, scale: float = 1.0, inverse: bool = False,
                     out: Optional[Tuple[Optional[torch.Tensor], Optional[torch.Tensor]]] = None
                     ) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor]]:
    """Rotates head dims [0, 2 * inv_freq.numel()) of q [tokens, Hq, D] and k
    [tokens, Hkv, D] (bf16; either may be None) by positions [tokens] (int32 or
    int64) times inv_freq (float64, on the device; rotary_frequencies): pairs
    (x[i], x[i + r/2]), or (x[2i], x[2i + 1]) when interleaved; cos and sin are
    multiplied by `scale`; inverse turns back (the gradient of the rotation,
    or keys moved to other positions).  In place, or into out = (q_out, k_out)
    of the same shapes.  Returns (q, k) or out."""
    outs = (q, k) if out is None else tuple(out)
    if len(outs) != 2:
        raise ValueError("out must be (q_out, k_out)")
    _rotary(q, k, positions, inv_freq, outs[0], outs[1], interleaved, scale, inverse)
    keep_alive(q, k, positions, inv_freq, *outs)
    return outs
