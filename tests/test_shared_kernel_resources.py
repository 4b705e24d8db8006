"""The kernels of appended tokens and of shared keys keep their state in registers: no
loop of theirs touches scratch memory, and the workgroups that a CU is planned to hold
fit its registers and LDS.  Read from the code objects' metadata, no GPU."""
import pytest

import d2sd
from test_kernel_resources import _code_objects, _kernels

pytest.importorskip("msgpack")


def _named(name):
    with open(d2sd.LIB_PATH, "rb") as f:
        return [k for elf in _code_objects(f.read()) for k in _kernels(elf) if name in k[".name"]]


# formats x (partners in registers or read again; queries kept or streamed); formats x (heads of 64: four waves, tokens kept or streamed; heads of 128: eight
# waves too, four where their rings fit); merges by head dim and order of the partial states
@pytest.mark.parametrize("name,n", [("cache_append_kernel", 16), ("shared_attn_kernel", 25), ("shared_merge_kernel", 4)])
def test_no_scratch_in_loops(name, n):
    kernels = _named(name)
    assert len(kernels) == n
    for k in kernels:
        # (one register set aside across the loop of one kernel: stored before it, read after it)
        assert k[".vgpr_spill_count"] <= 1 and k[".private_segment_fixed_size"] <= 8, k[".name"]


def test_workgroups_fit_beside_each_other():
    for k in _named("shared_attn_kernel"):
        waves = k[".max_flat_workgroup_size"] // 64
        assert waves in (4, 8)
        # (a workgroup of 8, or two of 4: two waves on each SIMD)
        assert k[".vgpr_count"] <= 256 and k[".group_segment_fixed_size"] <= (160 if waves == 8 else 80) * 1024, k[".name"]
