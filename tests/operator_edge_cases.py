"""Cases of the cross attention and the 8-bit product at values that are not numbers, shared by the emulator suite and the GPU suite."""
from __future__ import annotations

import math

import torch

import operator_cases as oc
from humanvid_amd import ops

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
NAN, INF = float("nan"), float("inf")

# (Lq, Lk, heads, kv_heads, D): one for each way the work is cut
CROSS_KERNELS = [
    (70, 77, 4, 4, 40),     # states in registers, several tiles of queries
    (35, 33, 4, 1, 80),     # the same, four heads on one key head
    (20, 64, 8, 4, 64),
    (2, 150, 4, 2, 40),     # at most 16 rows
    (1, 1100, 2, 1, 128),   # the same, keys cut into ranges
    (33, 130, 2, 2, 64),    # at most 64 rows: chunks of 64 keys
    (20, 600, 2, 2, 80),    # the same, keys cut into ranges
    (70, 130, 1, 1, 160),   # more rows: chunks of 32 keys
]


def _states(B, Lq, Lk, heads, kv_heads, D, seed):
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(B, Lq, heads * D, generator=g) * 1.5).to(BF16)
    k, v = (torch.randn(B, Lk, kv_heads * D, generator=g).to(BF16) for _ in range(2))
    return g, q, k, v


def _run(cx, q, k, v, heads, kv_heads, kv_len=None, key_mask=None):
    o = torch.full(q.shape, 7.0, dtype=BF16, device=cx.device)
    put = lambda t: None if t is None else t.to(cx.device)  # noqa: E731
    oc.run_cross(cx, put(q), put(k), put(v), o, heads, kv_heads, put(kv_len), put(key_mask))
    cx.sync()
    return o.cpu()


def case_empty_entries(cx, Lq, Lk, heads, kv_heads, D, how, seed=0):
    """Entries that attend to nothing are zero whatever their queries (and states) hold, and leave the others alone.
    how: "len" | "mask" | "part" (a length, and a mask over what the length leaves)."""
    g, q, k, v = _states(4, Lq, Lk, heads, kv_heads, D, seed)
    kv_len = key_mask = None
    if how in ("len", "part"):
        kv_len = torch.tensor([Lk, 0, 0, max(1, Lk // 2)], dtype=torch.int32)
        if how == "part":
            kv_len[1:3] = max(1, Lk // 2)
    if how in ("mask", "part"):
        key_mask = torch.rand(4, Lk, generator=g) < 0.7
        key_mask[[0, 3], 0] = True
        key_mask[1:3] = False
        if how == "part":
            key_mask[1:3, int(kv_len[1]):] = True
    want = _run(cx, q, k, v, heads, kv_heads, kv_len, key_mask)
    assert bool((want[1:3] == 0).all()) and bool(torch.isfinite(want).all()) and bool((want[[0, 3]] != 0).any())
    q[1] = NAN
    q[2, :, 0::3], q[2, :, 1::3], q[2, :, 2::3] = INF, -INF, 3e38
    k[1], v[2] = INF, NAN
    got = _run(cx, q, k, v, heads, kv_heads, kv_len, key_mask)
    assert torch.equal(got, want)


def case_masked_stretches(cx, Lq, Lk, heads, kv_heads, D, seed=0):
    """masks that leave whole stretches of states out, at the beginning, in the middle and at the end"""
    g, q, k, v = _states(3, Lq, Lk, heads, kv_heads, D, seed)
    keep = torch.ones(3, Lk, dtype=torch.bool)
    keep[0, :Lk - 1] = False                              # only the last state
    keep[1, 1:] = False                                   # only the first
    keep[2, Lk // 8:Lk - Lk // 8] = False                 # the middle left out
    k[~keep], v[~keep] = NAN, INF
    ref, tol = oc.cross_reference(q, k, v, heads, kv_heads, keep, 1 / math.sqrt(D))
    got = _run(cx, q, k, v, heads, kv_heads, key_mask=keep)
    assert bool(((got.to(F64) - ref).abs() <= tol).all())
