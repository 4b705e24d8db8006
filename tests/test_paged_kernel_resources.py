"""The kernels of the paged cache, the rotary embedding and the chunk attention keep
their state in registers: no loop of theirs touches scratch memory.  Read from the
code objects' metadata, no GPU."""
import pytest

import d2sd
from test_kernel_resources import _code_objects, _kernels

pytest.importorskip("msgpack")


def test_no_scratch_in_loops():
    with open(d2sd.LIB_PATH, "rb") as f:
        kernels = [k for elf in _code_objects(f.read()) for k in _kernels(elf)]
    count = lambda name: [k for k in kernels if name in k[".name"]]  # noqa: E731
    # formats x (heads of 64: four waves, tokens kept or streamed; heads of 128: eight waves too); merges by head dim
    for name, n in (("chunk_attn_kernel", 28), ("chunk_merge_kernel", 2), ("cache_write_kernel", 8), ("cache_read_kernel", 8),
                    ("rotary_kernel", 6)):
        assert len(count(name)) == n, name
        for k in count(name):
            # (one register set aside across the loop of one kernel: stored before it, read after it)
            assert k[".vgpr_spill_count"] <= 1 and k[".private_segment_fixed_size"] <= 8, k[".name"]
