"""rotary_frequencies against transformers' frequency initialisers (their
outputs, 32-bit: relative 2^-20 covers their powers and ramps), and the
refusals of rotary_embedding and rotary_frequencies.  CPU."""
import ctypes as C
import math

import pytest
import torch

import d2sd
from d2sd import _lib


def _config(d, base, scaling, n0=4096, longest=131072):
    transformers = pytest.importorskip("transformers")
    return transformers.Qwen3Config(hidden_size=4 * d, num_attention_heads=4, head_dim=d, rope_theta=base,
                                    max_position_embeddings=longest, rope_scaling=scaling)


@pytest.mark.parametrize("kind,theirs,ours", [
    ("default", None, None),
    ("linear", dict(factor=8.0), dict(type="linear", factor=8.0)),
    ("yarn", dict(factor=32.0, original_max_position_embeddings=4096),
     dict(type="yarn", factor=32.0, original_max_position=4096)),
    ("yarn", dict(factor=4.0, original_max_position_embeddings=8192, beta_fast=16.0, beta_slow=2.0,
                  attention_factor=1.5, truncate=False),
     dict(type="yarn", factor=4.0, original_max_position=8192, beta_fast=16, beta_slow=2, attention_factor=1.5,
          truncate=False)),
    ("llama3", dict(factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0, original_max_position_embeddings=8192),
     dict(type="wavelength", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0, original_max_position=8192)),
])
@pytest.mark.parametrize("d,base", [(128, 10000.0), (64, 150000.0)])
def test_frequencies_match_transformers(kind, theirs, ours, d, base):
    mod = pytest.importorskip("transformers.modeling_rope_utils")
    scaling = None if theirs is None else dict(rope_type=kind, **theirs)
    fns = mod.ROPE_INIT_FUNCTIONS
    if kind not in fns:
        pytest.skip(f"this transformers has no {kind!r} initialiser")
    ref, factor = fns[kind](_config(d, base, scaling), torch.device("cpu"))
    got, scale = d2sd.rotary_frequencies(d, base, ours)
    assert got.dtype == torch.float64 and got.shape == (d // 2,)
    assert ((got - ref.double()).abs() <= 2.0 ** -20 * got).all()
    assert math.isclose(scale, factor, rel_tol=1e-6)


def test_frequencies_by_formula():
    f, s = d2sd.rotary_frequencies(8, 100.0)
    assert s == 1.0 and torch.allclose(f, torch.tensor([100.0 ** (-i / 8) for i in (0, 2, 4, 6)], dtype=torch.float64),
                                       rtol=1e-15)
    f, _ = d2sd.rotary_frequencies(8, 100.0, dict(type="ntk", factor=4.0))
    assert torch.allclose(f[-1], torch.tensor((100.0 * 4.0 ** (8 / 6)) ** (-6 / 8), dtype=torch.float64), rtol=1e-14)
    # dynamic: untouched up to the trained length
    g, _ = d2sd.rotary_frequencies(8, 100.0, dict(type="dynamic", factor=4.0, original_max_position=64, seq_len=50))
    assert torch.equal(g, d2sd.rotary_frequencies(8, 100.0)[0])
    g, _ = d2sd.rotary_frequencies(8, 100.0, dict(type="dynamic", factor=4.0, original_max_position=64, seq_len=128))
    assert torch.allclose(g, d2sd.rotary_frequencies(8, 100.0, dict(type="ntk", factor=5.0))[0], rtol=1e-14)
    h, s = d2sd.rotary_frequencies(4, 100.0, dict(type="per_pair", factors=[1.0, 2.0], attention_factor=1.25))
    assert s == 1.25 and torch.allclose(h, torch.tensor([1.0, 0.05], dtype=torch.float64), rtol=1e-15)


@pytest.mark.parametrize("args", [(0,), (7,), (8, 1.0), (8, math.inf), (8, 1e4, dict(type="cubic")), (8, 1e4, dict(type="linear")),
                                  (8, 1e4, dict(type="linear", factor=0.0)), (8, 1e4, dict(type="linear", factor=2.0, turns=3)),
                                  (8, 1e4, dict(type="per_pair", factors=[1.0])), (2, 1e4, dict(type="ntk", factor=2.0)),
                                  (8, 1e4, dict(type="wavelength", factor=8.0, low_freq_factor=4.0, high_freq_factor=4.0,
                                                original_max_position=10))])
def test_frequencies_refuse(args):
    with pytest.raises(ValueError):
        d2sd.rotary_frequencies(*args)


def test_rotary_refuses_cpu_tensors_and_mismatches():
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16)
    pos, f = torch.zeros(3, dtype=torch.int32), torch.zeros(32, dtype=torch.float64)
    with pytest.raises(ValueError):
        d2sd.rotary_embedding(q, None, pos, f)          # CPU tensors
    with pytest.raises(ValueError):
        d2sd.rotary_embedding(None, None, pos, f)
    with pytest.raises(TypeError):
        d2sd.rotary_embedding(q.float(), None, pos, f)
    with pytest.raises(ValueError):
        d2sd.rotary_embedding(q, None, pos, f, out=(q,))
    with pytest.raises(ValueError):
        d2sd.rotary_embedding(q, None, pos, f, out=(None, None))


def _args(**kw):
    buf = C.cast(C.create_string_buffer(4096), C.c_void_p).value
    a = _lib.RotaryArgs()
    a.q = a.q_out = a.positions = a.inv_freq = buf
    a.q_stride_n = a.qo_stride_n = 256
    a.q_stride_h = a.qo_stride_h = 64
    a.scale, a.num_tokens, a.num_qo_heads, a.head_dim, a.num_pairs = 1.0, 1, 4, 64, 32
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("bad", [dict(num_tokens=-1), dict(num_kv_heads=-1), dict(num_kv_heads=1), dict(head_dim=63),
                                 dict(head_dim=258), dict(num_pairs=33), dict(num_pairs=0), dict(q=None), dict(q_out=None),
                                 dict(positions=None), dict(inv_freq=None), dict(scale=math.inf), dict(scale=math.nan),
                                 dict(qo_stride_n=512)])
def test_c_entry_refuses_without_launching(bad):
    assert _lib.lib.d2sd_rotary_embedding(C.byref(_args(**bad)), None) != 0
    assert b"rotary_embedding" in _lib.lib.d2sd_last_error()


def test_c_entry_with_no_tokens_launches_nothing():
    assert _lib.lib.d2sd_rotary_embedding(C.byref(_args(num_tokens=0)), None) == 0
    assert _lib.lib.d2sd_rotary_embedding(None, None) != 0
