"""Paged KV cache of a ragged batch (libd2sd.so): new keys and values written
into their pages, quantised on the way, and cached tokens read back.

PagedKVCommit writes one request's accepted tree nodes; a prompt, or one step
of many requests, is written here: token i of request r goes to the cache
position that the batch says, whatever the requests' lengths.  "bf16" and
"fp8" pools are the ones CascadeVerifyAttention and PagedKVCommit work on; the
block formats halve and quarter a cache's bytes without scales to calibrate.

    kv_format  pools                                scales
    "bf16"     bf16                                 none
    "fp8"      float8_e4m3fn, value / scale[head]   fp32 [Hkv] each for K and V,
                                                    positive
    "mxfp8"    float8_e4m3fn                        uint8, one per 32 head dims
    "mxfp4"    uint8, two e2m1 elements a byte      uint8, one per 32 head dims
               (the even one low)

Pools are [pages, Hkv, P, D] (kv_layout "HND") or [pages, P, Hkv, D] ("NHD"),
mxfp4 with D / 2 bytes in the place of D; block scales have the pools' shape
with D / 32 last.  A block's scale byte b stands for 2^(b - 127) (255: NaN).
Writing takes the smallest power of two that keeps the block's largest
magnitude within the elements' range, from 2^-117 on, and rounds to nearest
even, so that reading back gives exact bf16 values and a block holding a NaN
or infinity reads back as NaN.
"""
from __future__ import annotations

from typing import Optional, Sequence, Tuple, Union

import numpy as np
import torch

from . import _lib
from .graph import _CAPTURING, capturing, home_stream, keep_alive

_write, _read, _read_out = (getattr(torch.ops.d2sd, n).default for n in ("cache_write", "cache_read", "cache_read_out"))
KV_FORMATS = {"bf16": _lib.D2SD_CACHE_BF16, "fp8": _lib.D2SD_CACHE_FP8, "mxfp8": _lib.D2SD_CACHE_MXFP8,
              "mxfp4": _lib.D2SD_CACHE_MXFP4}
_BLOCK = 32


def _i32(x) -> np.ndarray:
    if isinstance(x, torch.Tensor):
        x = x.cpu().numpy()
    a = np.asarray(x)
    if a.size and (a.min() < -2 ** 31 or a.max() >= 2 ** 31):
        raise ValueError("lengths and offsets must fit 32 bits")
    return np.ascontiguousarray(a.astype(np.int32))


def _device(device) -> torch.device:
    dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
    if dev.type == "cuda" and dev.index is None:
        dev = torch.device("cuda", torch.cuda.current_device())
    return dev


def _spans(first, count, row, req, from_end, pi) -> np.ndarray:
    """d2sd_cache_span records that cover tokens first .. of each request."""
    per = _lib.READ_TOKENS
    n = -(-count // per)                       # records per request
    r = np.repeat(np.arange(len(count)), n)
    j = (np.arange(len(r)) - np.repeat(np.cumsum(n) - n, n)) * per
    out = np.zeros((len(r), 8), dtype=np.int32)
    out[:, 0] = req[r]
    out[:, 1] = np.minimum(count[r] - j, per)
    out[:, 2] = first[r] - j if from_end else first[r] + j
    out[:, 3] = int(from_end)
    out[:, 4] = row[r] + j
    out[:, 5], out[:, 6] = pi[req[r]], pi[req[r] + 1]
    return out


class PagedBatch:
    """The ragged batch of one step: request r brings new tokens
    qo_indptr[r] .. qo_indptr[r+1] - 1 (rows of q, k and v), has a cache of
    kv_len[r] tokens with them, and the pages
    page_table[page_indptr[r] : page_indptr[r+1]] of page_size tokens each.

    `kv_len` (int32, on the device) holds the current lengths and is what the
    kernels read: update it in place (set_kv_len, or any device write) and the
    same batch, and graphs captured with it, serve the next step, as long as
    the new tokens stay as many and the pages suffice.  kv_len_host,
    kv_indptr_host and total_kv are the host's lengths, those of the last
    set_kv_len (a device write does not move them): full reads cover them, and
    plans made from now on share out work for them.  A contiguous int32 device
    tensor given as page_table is used in place."""

    def __init__(self, qo_indptr: Sequence[int], kv_len: Sequence[int], page_indptr: Sequence[int],
                 page_table: Union[Sequence[int], torch.Tensor], page_size: int,
                 device: Union[str, torch.device, None] = None):
        if device is None and isinstance(page_table, torch.Tensor) and page_table.is_cuda:
            device = page_table.device
        qo, kv, pi = _i32(qo_indptr), _i32(kv_len), _i32(page_indptr)
        P, R = int(page_size), kv.size
        if qo.ndim != 1 or kv.ndim != 1 or pi.ndim != 1 or qo.size != R + 1 or pi.size != R + 1:
            raise ValueError("qo_indptr and page_indptr must have len(kv_len) + 1 entries")
        if P <= 0 or P & (P - 1):
            raise ValueError("page_size must be a power of two")
        if qo[0] != 0 or pi[0] < 0 or (np.diff(qo) < 0).any() or (np.diff(pi) < 0).any() or (kv < 0).any():
            raise ValueError("qo_indptr starts at 0, indptrs must not decrease, lengths must not be negative")
        if (kv.astype(np.int64) > np.diff(pi).astype(np.int64) * P).any():
            raise ValueError("page_indptr gives a request too few pages for its kv_len")
        n = page_table.numel() if isinstance(page_table, torch.Tensor) else len(page_table)
        if n < pi[-1]:
            raise ValueError("page_table shorter than page_indptr[-1]")
        self.device = _device(device)
        self._home = home_stream(self.device)  # of the batch's tensors (-1: of several)
        self.page_size, self.num_reqs, self.total_q = P, R, int(qo[-1])
        self.qo_indptr_host, self.page_indptr_host = qo, pi
        self._reads = {}
        self._host_lengths(kv)
        if self.total_kv >= 2 ** 31:
            raise ValueError("the batch's caches hold 2^31 tokens or more")
        # one upload: a record per new token, then the lengths
        req = np.repeat(np.arange(R, dtype=np.int32), np.diff(qo))
        tokens = np.stack([req, qo[req + 1] - np.arange(self.total_q, dtype=np.int32), pi[req], pi[req + 1]],
                          axis=1).astype(np.int32)
        up = torch.from_numpy(np.concatenate([tokens.reshape(-1), kv])).to(self.device)
        self._tokens = up[:4 * self.total_q]
        self.kv_len = up[4 * self.total_q:]
        if isinstance(page_table, torch.Tensor) and page_table.dtype == torch.int32 and page_table.is_contiguous() \
                and page_table.device == self.device:
            self.page_table = page_table.reshape(-1)
        else:
            self.page_table = torch.from_numpy(_i32(page_table).reshape(-1)).to(self.device)

    def _host_lengths(self, kv: np.ndarray) -> None:
        self.kv_len_host = kv
        self.kv_indptr_host = np.concatenate([[0], np.cumsum(kv, dtype=np.int64)])
        self.total_kv = int(self.kv_indptr_host[-1])
        self._reads.pop(False, None)  # (those of the new tokens count from a cache's end)

    def set_kv_len(self, kv_len: Sequence[int]) -> None:
        """Current cache lengths (host write into `kv_len`).  The next full read
        covers them; one captured before keeps the rows that it was captured
        with."""
        v = _i32(kv_len)
        if v.shape != (self.num_reqs,) or (v < 0).any() or \
                (v.astype(np.int64) > np.diff(self.page_indptr_host).astype(np.int64) * self.page_size).any():
            raise ValueError("one length per request, within its pages")
        self.kv_len.copy_(torch.from_numpy(v))
        self._host_lengths(v)

    def prepare_read(self, new_only: bool = False) -> "PagedBatch":
        """Builds what PagedKVCache.read needs of this batch (done by the first
        read, and the first full one after set_kv_len; call it before a read
        that is captured into a graph)."""
        if new_only not in self._reads:
            if self.device.type == "cuda" and capturing():
                raise RuntimeError("PagedKVCache.read: call batch.prepare_read() before capturing a read")
            req = np.arange(self.num_reqs)
            if new_only:
                n = np.diff(self.qo_indptr_host)
                spans = _spans(n, n, self.qo_indptr_host[:-1], req, True, self.page_indptr_host)
            else:
                if self.total_kv >= 2 ** 31:
                    raise ValueError("the batch's caches hold 2^31 tokens or more")
                spans = _spans(np.zeros_like(self.kv_len_host), self.kv_len_host, self.kv_indptr_host[:-1], req, False,
                               self.page_indptr_host)
            self._reads[new_only] = torch.from_numpy(spans).to(self.device)
            if home_stream(self.device) != self._home:
                self._home = -1
        return self


class PagedKVCache:
    """One layer's paged keys and values in one of the formats above."""

    def __init__(self, k_pool: torch.Tensor, v_pool: torch.Tensor, kv_format: str = "bf16", *,
                 k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None,
                 kv_layout: str = "HND"):
        if kv_format not in KV_FORMATS:
            raise ValueError(f"kv_format must be one of {sorted(KV_FORMATS)}")
        if kv_layout not in ("HND", "NHD"):
            raise ValueError("kv_layout must be 'HND' or 'NHD'")
        mx = kv_format.startswith("mx")
        dtypes = {"bf16": (torch.bfloat16,), "fp8": (torch.float8_e4m3fn,),
                  "mxfp8": (torch.float8_e4m3fn, torch.uint8), "mxfp4": (torch.uint8,)}[kv_format]
        for name, t in (("k_pool", k_pool), ("v_pool", v_pool)):
            if t.dtype not in dtypes:
                raise TypeError(f"{name} of a {kv_format} cache must be {dtypes[0]} (got {t.dtype})")
            if t.dim() != 4 or t.stride(-1) != 1 or t.shape != k_pool.shape or t.stride() != k_pool.stride() \
                    or t.device != k_pool.device or not t.is_cuda:
                raise ValueError("k_pool and v_pool must be 4-D device tensors of one shape and stride with a "
                                 "contiguous last dimension")
        tok, head = (2, 1) if kv_layout == "HND" else (1, 2)
        P, hkv = k_pool.shape[tok], k_pool.shape[head]
        d = k_pool.shape[3] * (2 if kv_format == "mxfp4" else 1)
        if kv_format == "bf16":
            if k_scale is not None or v_scale is not None:
                raise ValueError("a bf16 cache has no scales")
        else:
            if k_scale is None or v_scale is None:
                raise ValueError(f"a {kv_format} cache needs k_scale and v_scale")
            shape = (hkv,) if not mx else (*k_pool.shape[:3], d // _BLOCK)
            dtype = torch.uint8 if mx else torch.float32
            for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
                if t.dtype != dtype:
                    raise TypeError(f"{name} of a {kv_format} cache must be {dtype} (got {t.dtype})")
                if tuple(t.shape) != shape or t.stride() != k_scale.stride() or t.stride(-1) != 1 \
                        or t.device != k_pool.device:
                    raise ValueError(f"{name} must be {list(shape)} on the pools' device, contiguous in its last "
                                     "dimension, both alike")
        if P & (P - 1) or P == 0:
            raise ValueError("page_size must be a power of two")
        if d % _BLOCK or not 0 < d <= 256:
            raise ValueError("head_dim must be a multiple of 32 up to 256")
        # what every operator over the cache takes of it
        self._pools = (k_pool, v_pool, k_scale, v_scale, KV_FORMATS[kv_format], kv_layout == "NHD")
        self.k_pool, self.v_pool, self.k_scale, self.v_scale = k_pool, v_pool, k_scale, v_scale
        self.kv_format, self.kv_layout, self.device = kv_format, kv_layout, k_pool.device
        self._home = home_stream(self.device)
        self.num_pages, self.page_size, self.num_kv_heads, self.head_dim = k_pool.shape[0], P, hkv, d

    @classmethod
    def allocate(cls, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int, kv_format: str = "bf16", *,
                 k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None,
                 kv_layout: str = "HND", device: Union[str, torch.device, None] = None) -> "PagedKVCache":
        """A cache of num_pages pages, its contents unset (fp8: with the given
        per-head scales)."""
        if kv_format not in KV_FORMATS:
            raise ValueError(f"kv_format must be one of {sorted(KV_FORMATS)}")
        dev = _device(device)
        lead = (num_pages, num_kv_heads, page_size) if kv_layout == "HND" else (num_pages, page_size, num_kv_heads)
        width = head_dim // 2 if kv_format == "mxfp4" else head_dim
        dtype = {"bf16": torch.bfloat16, "mxfp4": torch.uint8}.get(kv_format, torch.float8_e4m3fn)
        k, v = (torch.empty((*lead, width), dtype=dtype, device=dev) for _ in range(2))
        if kv_format.startswith("mx"):
            if k_scale is not None or v_scale is not None:
                raise ValueError("block scales are part of the cache")
            k_scale, v_scale = (torch.empty((*lead, head_dim // _BLOCK), dtype=torch.uint8, device=dev)
                                for _ in range(2))
        return cls(k, v, kv_format, k_scale=k_scale, v_scale=v_scale, kv_layout=kv_layout)

    def _check_batch(self, batch: PagedBatch) -> None:
        if batch.page_size != self.page_size:
            raise ValueError(f"the batch's page_size {batch.page_size} is not the cache's {self.page_size}")

    def write(self, k: torch.Tensor, v: torch.Tensor, batch: PagedBatch) -> None:
        """Writes the batch's new tokens, rows of k and v [total_q, Hkv, D]
        (bf16; rows behind the last request's are left alone), to the cache
        positions kv_len[r] - n_r .. kv_len[r] - 1 of each request.  Page ids
        outside the pool are skipped.  Two tokens of one call must not share a
        slot."""
        self._check_batch(batch)
        home = self._home if self._home == batch._home else -1
        _write(k, v, batch._tokens, batch.total_q, batch.kv_len, batch.page_table, *self._pools, home)
        if _CAPTURING:
            keep_alive(k, v, batch._tokens, batch.kv_len, batch.page_table, *self._pools[:4])

    def read(self, batch: PagedBatch, new_only: bool = False,
             out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """The batch's cached keys and values as contiguous bf16 [rows, Hkv, D]:
        request r's tokens are rows kv_indptr_host[r] .. of the batch (the
        host's lengths: set_kv_len's), or, with new_only, the batch's new tokens
        in the rows of q.  Rows of tokens that the cache does not hold now (a
        shorter kv_len, a page id outside the pool) are zero; in a given `out`
        they are left alone.  out: (k, v) of any token and head strides, alike."""
        self._check_batch(batch)
        rows = batch.total_q if new_only else batch.total_kv
        if new_only not in batch._reads:
            batch.prepare_read(new_only)
        items = batch._reads[new_only]
        home = self._home if self._home == batch._home else -1
        if out is None:
            out = _read(rows, items, items.shape[0], batch.kv_len, batch.page_table, *self._pools, home)
        else:
            k, v = out
            _read_out(k, v, rows, items, items.shape[0], batch.kv_len, batch.page_table, *self._pools, home)
        if _CAPTURING:
            keep_alive(*out, items, batch.kv_len, batch.page_table, *self._pools[:4])
        return out
