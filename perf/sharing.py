"""Whether requests that begin with the same tokens are better attended with their first keys shared or apart, and which
of the two PagedChunkAttention.plan takes by itself: 330 batches, each timed planned apart, with all groups shared
(keep_shared) and as plan() chooses.

    python3 perf/sharing.py [FILE]     # a table in markdown, to FILE or the standard output

Batches: 2 to 64 requests of some new tokens (as many each, or 1 to so many), each with 200 to 400 cached tokens of its
own behind a shared prompt (prompts: none but the new ones), in one group; and several groups of unequal prompts.
Times: the smallest of five averages of 20 calls, the three plans in turn.  Every batch's caches hold the same tokens
in every plan: the others' page tables name the first request's shared pages.
"""
import sys
import time
from pathlib import Path

import numpy as np
import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "d2-sd_amd"))

import d2sd  # noqa: E402

PAGE = 16
KINDS = [("bf16", 32, 8, 128), ("mxfp8", 32, 8, 128), ("bf16", 64, 8, 64)]
MOST_NEW = 6000  # new tokens of a batch


def batches():
    """(format, query heads, kv heads, head dim, what, requests of each group, shared keys of each, new tokens of each
    request, cached ones of its own with them)"""
    out = []

    def add(kind, what, groups, shared, new, cached):
        rng = np.random.default_rng(len(out))
        new = [int(n) for n in (new(rng) if callable(new) else new)]
        own = [n + int(rng.integers(200, 401)) if cached else n for n in new]
        out.append((*kind, what, list(groups), [s // PAGE * PAGE for s in shared], new, own))

    for kind in KINDS:
        for reqs in (2, 4, 16, 64):
            for n in (1, 5, 32, 200):
                for shared in (64, 512, 4096):
                    if reqs * n <= 4000:
                        add(kind, f"{n}", [reqs], [shared], [n] * reqs, True)
            for most in (9, 60, 400):
                for shared in (512, 4096, 16384):
                    if reqs * most <= 2 * MOST_NEW:
                        add(kind, f"1..{most}", [reqs], [shared], lambda r: r.integers(1, most + 1, reqs), True)
                        if reqs > 2:
                            add(kind, f"1..{most}, prompts", [reqs], [shared], lambda r: r.integers(1, most + 1, reqs), False)
        for groups, shared in (([8] * 4, [4096] * 4), ([16, 4, 30, 2], [8000, 300, 2000, 16000]), ([4] * 16, [1000] * 16),
                               ([2, 5, 9, 20, 3, 7], [512, 1024, 2048, 4096, 8192, 640])):
            n = sum(groups)
            add(kind, "1", groups, shared, [1] * n, True)
            add(kind, "1, each seventh 200", groups, shared, [200 if i % 7 == 3 else 1 for i in range(n)], True)
    return out


def plans(hq, hkv, d, fmt, groups, shared, new, own, device="cuda", **kw):
    """The batch, and its page count; a request's table begins with the shared pages of its group's first."""
    table, indptr, used, at = [], [0], 0, 0
    for g, n in enumerate(groups):
        full = shared[g] // PAGE
        lead = list(range(used, used + full))
        used += full
        for _ in range(n):
            m = -(-own[at] // PAGE)
            table += lead + list(range(used, used + m))
            used += m
            indptr.append(len(table))
            at += 1
    kv = [o + s for o, s in zip(own, np.repeat(shared, groups))]
    batch = d2sd.PagedBatch(np.concatenate([[0], np.cumsum(new)]), kv, indptr, np.asarray(table, dtype=np.int32), PAGE,
                            device=device)
    return batch, used


def cache(pages, hkv, d, fmt):
    gen = torch.Generator(device="cuda").manual_seed(2)
    shape = (pages, hkv, PAGE, d)
    if fmt == "bf16":
        return d2sd.PagedKVCache(*(torch.randn(shape, generator=gen, device="cuda").to(torch.bfloat16) for _ in range(2)))
    c = d2sd.PagedKVCache.allocate(pages, PAGE, hkv, d, fmt)
    for codes, scale in ((c.k_pool, c.k_scale), (c.v_pool, c.v_scale)):
        codes.view(torch.uint8).copy_(torch.randint(0, 0x70, shape, generator=gen, device="cuda"))
        scale.fill_(120)
    return c


def average(fn, calls=20):
    a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    a.record()
    for _ in range(calls):
        fn()
    b.record()
    b.synchronize()
    return a.elapsed_time(b) / calls * 1e3


def main():
    out = open(sys.argv[1], "w") if len(sys.argv) > 1 else sys.stdout
    print("| cache | heads | groups | shared keys | new tokens | apart us | shared us | chosen us | shared? | states MB | plan ms |",
          "|---|---|---|---|---|---|---|---|---|---|---|", sep="\n", file=out, flush=True)
    for fmt, hq, hkv, d, what, groups, shared, new, own in batches():
        batch, pages = plans(hq, hkv, d, fmt, groups, shared, new, own)
        c = cache(pages, hkv, d, fmt)
        q = torch.randn(sum(new), hq, d, device="cuda").to(torch.bfloat16)
        kw = dict(shared_indptr=np.concatenate([[0], np.cumsum(groups)]), shared_len=shared)
        attn = []
        for extra in ({}, dict(kw, keep_shared=True), kw):
            t0 = time.perf_counter()
            attn.append(d2sd.PagedChunkAttention().plan(batch, hq, hkv, d, kv_format=fmt, **extra))
            took = time.perf_counter() - t0
        for a in attn:
            average(lambda: a.run(q, c), 3)
        us = np.min([[average(lambda: a.run(q, c)) for a in attn] for _ in range(5)], axis=0)
        of = lambda x: str(x[0]) if len(set(x)) == 1 else ", ".join(map(str, x))  # noqa: E731
        n = f"{len(groups)} of {of(groups)}" if len(groups) > 1 else f"{groups[0]}"
        print(f"| {fmt} | {hq} + {hkv} of {d} | {n} | {of(shared)} | {what} | {us[0]:.1f} | {us[1]:.1f} | {us[2]:.1f} | "
              f"{'yes' if attn[2].info.form & 8 else 'no'} | {attn[1].info.workspace_bytes / 1e6:.1f} | {took * 1e3:.2f} |",
              file=out, flush=True)


if __name__ == "__main__":
    main()
