"""PagedChunkAttention — attention of each request's newest tokens over its
paged KV cache, which already holds them (libd2sd.so).

CascadeVerifyAttention reads a prefix and, apart from it, the suffix of a
verify step under its tree mask.  A prompt's chunks and plain decoding steps
are causal and write their keys first (PagedKVCache.write, quantised if the
cache is): this operator reads keys and values from the cache only, for
batches that mix chunks and single tokens, in every cache format, with a
window that follows each token and attention sinks.  Where groups of requests
begin with the same tokens, plan() takes them and their keys are read and
multiplied once for all rows of the group.

plan() does the host work once for a batch's shape; run() launches one kernel,
and a second that joins partial states where a request's keys were split.
Both read the current lengths from batch.kv_len on the device, so a captured
step replays while the caches grow.  run() may be captured into a HipGraph;
unless `workspace` is given, each run takes scratch memory of its own, so runs
may overlap on different streams.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Sequence, Tuple, Union

import numpy as np
import torch

from . import _lib
from ._lib import check, lib
from .graph import _CAPTURING, home_stream, keep_alive
from .paged import KV_FORMATS, PagedBatch, PagedKVCache, _device, _i32

_attention, _attention_out = (torch.ops.d2sd.chunk_attention.default, torch.ops.d2sd.chunk_attention_out.default)


class PagedChunkAttention:
    def __init__(self, device: Union[str, torch.device, None] = None):
        self._want_device = device
        self.batch: Optional[PagedBatch] = None

    def plan(self, batch: PagedBatch, num_qo_heads: int, num_kv_heads: int, head_dim: int, *, kv_format: str = "bf16",
             sm_scale: Optional[float] = None, window_left: int = -1, sinks: Optional[torch.Tensor] = None,
             lse_base2: bool = False, max_splits: int = 0, num_cus: int = 0,
             shared_indptr: Optional[Sequence[int]] = None, shared_len: Optional[Sequence[int]] = None,
             keep_shared: bool = False) -> "PagedChunkAttention":
        """Plans the batch (its kv_len_host, of its making or the last
        set_kv_len: the work is shared out for those lengths, and right for any
        within the requests' pages).

        Query i of request r sits at position kv_len[r] - n_r + i and sees the
        cached keys up to it; window_left >= 0 keeps the window_left keys
        before it and its own.  sm_scale defaults to head_dim ** -0.5 and must
        be at least 2e-38 (over fp8 caches, times each k_scale too).  sinks [Hq] fp32 applies O *= sigmoid(lse - sink).  Rows
        that see no key (a request whose kv_len is below its new tokens) get
        output 0 and lse -inf.  A NaN or infinity in K or V reaches the rows
        that see its token and no others.

        Requests whose caches begin alike (a system prompt, a document):
        requests shared_indptr[i] .. shared_indptr[i + 1] - 1 hold the same
        tokens in their first shared_len[i] positions (0: none).  Those keys
        are read once for all of them, through the first one's pages, where
        that is faster by the plan's estimate (joining partial states costs
        time; few shared keys, or many new tokens, do not repay it), else by
        each request through its own.  The states take workspace too, 8 bytes
        for each element of the output where nothing is split: they have to
        gain 1%, and 1% more for each 128 MB.  keep_shared=True shares the keys
        in any case; the others' pages of that range are then never looked at.
        shared_indptr starts at 0 and ends at the number of requests; a
        group's shared_len is any number that its first request's pages hold.
        The result is that of a plan without groups, whatever lengths the
        caches have later, as long as the first request's pages keep the shared
        tokens (also where it is cut back below them: plan again before other
        tokens are written there)."""
        if kv_format not in KV_FORMATS:
            raise ValueError(f"kv_format must be one of {sorted(KV_FORMATS)}")
        if self._want_device is not None and _device(self._want_device) != batch.device:
            raise ValueError("the batch is on another device")
        if sinks is not None:
            if sinks.dtype != torch.float32 or tuple(sinks.shape) != (num_qo_heads,) or not sinks.is_contiguous() \
                    or sinks.device != batch.device:
                raise ValueError("sinks must be a contiguous float32 [num_qo_heads] tensor on the batch's device")
        scale = head_dim ** -0.5 if sm_scale is None else float(sm_scale)
        if not (scale >= 2e-38 and scale <= torch.finfo(torch.float32).max):
            raise ValueError("sm_scale must be at least 2e-38 and finite")
        as_p = lambda x: x.ctypes.data_as(C.POINTER(C.c_int32))  # noqa: E731
        desc = _lib.ChunkPlanDesc()
        desc.num_reqs = batch.num_reqs
        desc.qo_indptr, desc.kv_len = as_p(batch.qo_indptr_host), as_p(batch.kv_len_host)
        desc.page_indptr = as_p(batch.page_indptr_host)
        desc.num_qo_heads, desc.num_kv_heads, desc.head_dim = num_qo_heads, num_kv_heads, head_dim
        desc.format, desc.page_size, desc.window_left = KV_FORMATS[kv_format], batch.page_size, window_left
        desc.num_cus, desc.max_splits = num_cus, max_splits
        if (shared_indptr is None) != (shared_len is None):
            raise ValueError("shared_indptr and shared_len go together")
        groups, indptr, shared = 0, None, None
        if shared_len is not None:
            ip, n = _i32(shared_indptr), _i32(shared_len)
            if ip.ndim != 1 or n.ndim != 1 or ip.size != n.size + 1:
                raise ValueError("shared_indptr must have len(shared_len) + 1 entries")
            groups, indptr, shared = n.size, as_p(ip), as_p(n)
            if not groups and batch.num_reqs:
                raise ValueError("shared_indptr must hold every request")
        info = _lib.ChunkPlanInfo()
        # (too small a buffer means planning twice: merges of 12 ints for 1024 elements of the output, and items)
        merges = 24 * (batch.total_q * max(num_qo_heads, 0) * max(head_dim, 0) >> 10)
        host = np.empty((1 << 18) + min(merges, 1 << 24), dtype=np.int32)
        plan = lambda: lib.d2sd_chunk_plan_shared(C.byref(desc), groups, indptr, shared, bool(keep_shared), as_p(host),  # noqa: E731
                                                  host.size, C.byref(info))
        with torch.cuda.device(batch.device) if batch.device.type == "cuda" else torch.no_grad():
            rc = plan()
            if rc == _lib.D2SD_ERR_WORKSPACE and info.plan_ints > host.size:
                host = np.empty(info.plan_ints, dtype=np.int32)
                rc = plan()
        check(rc, "chunk_plan")
        self.info, self.batch, self.sinks = info, batch, sinks
        # (a small plan does not hold the whole buffer)
        self.plan_host = host[:info.plan_ints] if 2 * info.plan_ints > host.size else host[:info.plan_ints].copy()
        self.plan_dev = torch.from_numpy(self.plan_host).to(batch.device)
        self._home = home_stream(batch.device)
        self.kv_format, self.sm_scale, self.lse_base2 = kv_format, scale, bool(lse_base2)
        self.num_qo_heads, self.num_kv_heads, self.head_dim = num_qo_heads, num_kv_heads, head_dim
        self._info = torch.frombuffer(bytearray(bytes(info)), dtype=torch.uint8)
        return self

    def workspace(self) -> torch.Tensor:
        """Scratch memory for run(workspace=...): one for all runs that never
        overlap (the layers of a step)."""
        if self.batch is None:
            raise RuntimeError("workspace() before plan()")
        return torch.empty(max(int(self.info.workspace_bytes), 16), dtype=torch.uint8, device=self.batch.device)

    def run(self, q: torch.Tensor, cache: PagedKVCache, out: Optional[torch.Tensor] = None,
            lse: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None
            ) -> Tuple[torch.Tensor, torch.Tensor]:
        """q [total_q, Hq, D] (bf16; rows behind the last request's are left
        alone, and so are those of out and lse) over `cache`.  Returns (out
        [total_q, Hq, D] bf16, lse [total_q, Hq] fp32, natural log unless
        planned with lse_base2)."""
        batch = self.batch
        if batch is None:
            raise RuntimeError("run() before plan()")
        cache._check_batch(batch)
        if cache.kv_format != self.kv_format:
            raise ValueError(f"the plan is for a {self.kv_format} cache, not {cache.kv_format}")
        rest = (self._info, self.plan_dev, batch.kv_len, batch.page_table, *cache._pools, self.sinks, self.sm_scale,
                self.lse_base2, self._home if self._home == batch._home == cache._home else -1)
        if workspace is None and self.info.workspace_bytes and _CAPTURING:
            workspace = self.workspace()  # the graph holds it
        if out is None and lse is None:
            out, lse = _attention(q, workspace, *rest)
        else:
            if out is None:
                out = torch.empty_like(q, memory_format=torch.contiguous_format)
                out[batch.total_q:].zero_()
            if lse is None:
                lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
                lse[batch.total_q:].fill_(-float("inf"))
            _attention_out(q, out, lse, workspace, *rest)
        if _CAPTURING:
            keep_alive(self.plan_dev, batch.kv_len, batch.page_table, self.sinks, q, out, lse, workspace, *cache._pools[:4])
        return out, lse
