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


def case_query_values(cx, Lq, Lk, heads, kv_heads, D, masked, seed=0):
    """A query that holds NaN or infinities spoils its own row of its own head, and nothing else.  (Scores of both signs, so that an
    infinite query has no softmax either.)"""
    g, q, k, v = _states(2, Lq, Lk, heads, kv_heads, D, seed)
    key_mask = None
    if masked:
        key_mask = torch.rand(2, Lk, generator=g) < 0.7
        key_mask[:, :4] = True
    want = _run(cx, q, k, v, heads, kv_heads, key_mask=key_mask)
    bad = torch.zeros(2, Lq, heads, D, dtype=torch.bool)
    for i, x in enumerate((NAN, INF, -INF)):
        b, row, h = i % 2, (i * 7) % Lq, (i * 3) % heads
        q.view(2, Lq, heads, D)[b, row, h, 5 + i] = x
        bad[b, row, h] = True
    got = _run(cx, q, k, v, heads, kv_heads, key_mask=key_mask)
    bad = bad.view(2, Lq, -1)
    assert bool(got[bad].isnan().all())
    assert torch.equal(got[~bad], want[~bad])


def case_state_values(cx, Lq, Lk, heads, kv_heads, D, masked, seed=0):
    """Attended states that hold infinities and NaN, against the definition: an infinite key takes a weight of zero where its score is
    -inf and leaves NaN where it is +inf; an infinite value reaches its own column of the rows that give it weight; a NaN key leaves
    NaN in every row of its head, a NaN value in its column."""
    g, q, k, v = _states(4, Lq, Lk, heads, kv_heads, D, seed)
    keep = torch.ones(4, Lk, dtype=torch.bool)
    if masked:
        keep = torch.rand(4, Lk, generator=g) < 0.7
        keep[:, 1] = keep[:, Lk - 1] = True
        k[~keep], v[~keep] = NAN, NAN
    G, h0 = heads // kv_heads, heads - 1
    c0 = (h0 // G) * D  # columns of the last key head
    rest = keep.clone()
    rest[0, Lk - 1] = False
    ref, tol = oc.cross_reference(q, k, v, heads, kv_heads, rest, 1 / math.sqrt(D))  # entry 0 without its infinite key
    k[0, Lk - 1, c0 + 3] = INF
    v[1, 1, c0 + 2] = -INF
    k[2, 1, c0 + 7] = NAN
    v[3, Lk - 1, c0 + 4] = NAN
    full, ftol = oc.cross_reference(q, k.nan_to_num(0, 0, 0), v.nan_to_num(0, 0, 0), heads, kv_heads, keep, 1 / math.sqrt(D))
    got = _run(cx, q, k, v, heads, kv_heads, key_mask=keep if masked else None).to(F64).view(4, Lq, heads, D)
    ref, tol, full, ftol = (t.view(4, Lq, heads, D) for t in (ref, tol, full, ftol))
    hit = torch.arange(heads) // G == h0 // G  # heads that read those columns
    ok = torch.zeros(4, Lq, heads, D, dtype=torch.bool)

    def near(b, x, t):
        return (got[b] - x[b]).abs() <= t[b]

    ok[0] = near(0, full, ftol)
    plus = (q[0].view(Lq, heads, D)[:, hit, 3] > 0)[..., None]  # (no query is zero there)
    ok[0][:, hit] = torch.where(plus, got[0][:, hit].isnan(), near(0, ref, tol)[:, hit])
    ok[1] = near(1, full, ftol)
    ok[1][:, hit, 2] = got[1][:, hit, 2] == -INF
    ok[2] = near(2, full, ftol)
    ok[2][:, hit] = got[2][:, hit].isnan()
    ok[3] = near(3, full, ftol)
    ok[3][:, hit, 4] = got[3][:, hit, 4].isnan()
    assert bool((q[0].view(Lq, heads, D)[:, hit, 3] != 0).all())
    assert bool(ok.all()), [int((~ok[b]).sum()) for b in range(4)]


def case_gemm_values(cx, M, N, K, out, seed=0):
    """NaN operands and scales reach their own row or column and nothing else, wherever in a block they lie."""
    x, xs, w, ws, bias, res = oc.gemm_operands(M, N, K, seed)

    def run():
        put = lambda t: t.to(cx.device)  # noqa: E731
        y = torch.full((M, N), 7.0, dtype=out, device=cx.device)
        a = (cx.lib, cx.stream, put(x), put(xs), put(w), put(ws), y)
        kw = dict(bias=put(bias), residual=put(res))
        n = ops.gemm_fp8(*a, query_workspace=True, **kw)
        ops.gemm_fp8(*a, workspace=torch.full((n,), NAN, device=cx.device) if n else None, **kw)
        cx.sync()
        return y.cpu()

    want = run()
    bad = torch.zeros(M, N, dtype=torch.bool)
    xb, wb = x.view(torch.uint8), w.view(torch.uint8)
    for row, k in ((0, 0), (M // 2, K - 1), (M - 1, K // 2)):
        xb[row, k] = 0x7f
        bad[row] = True
    for col, k in ((0, K - 1), (N // 2, 0), (N - 1, max(0, K - 17))):
        wb[col, k] = 0xff
        bad[:, col] = True
    if M > 8:
        xs[3, -1] = INF
        xs[5, 0] = NAN
        bad[5] = True
    got = run()
    if M > 8:  # a row of infinite scale: infinite or NaN, never a number
        assert not bool(torch.isfinite(got[3]).any())
        bad[3] = True
        assert bool(got[5].isnan().all())
    rows = torch.zeros(M, dtype=torch.bool)
    rows[[0, M // 2, M - 1]] = True
    assert bool(got[rows].isnan().all()) and bool(got[:, [0, N // 2, N - 1]].isnan().all())
    assert torch.equal(got[~bad], want[~bad]) and bool(torch.isfinite(got[~bad]).all())


def ranges_tensors(cx, seed, M=100, N=320, K=2560):
    """operands of a product whose reduction is cut into ranges, with its scratch"""
    g = torch.Generator().manual_seed(seed)
    t = dict(x=torch.randn(M, K, generator=g).to(BF16).to(cx.device), kb=-(-K // 128))
    w = (torch.randn(N, K, generator=g) * K**-0.5).to(BF16).to(cx.device)
    t["x8"], t["xs"] = torch.empty(M, K, dtype=oc.FP8, device=cx.device), torch.empty(t["kb"], M, device=cx.device).t()
    t["w8"], t["ws"] = torch.empty(N, K, dtype=oc.FP8, device=cx.device), torch.empty(-(-N // 128), t["kb"], device=cx.device)
    ops.fp8_quantize(cx.lib, cx.stream, w, t["w8"], t["ws"], block_rows=128)
    t["bias"] = torch.randn(N, generator=g).to(cx.device)
    t["residual"] = torch.randn(M, N, generator=g).to(BF16).to(cx.device)
    t["y"], t["y32"] = torch.zeros(M, N, dtype=BF16, device=cx.device), torch.zeros(M, N, device=cx.device)
    n = ops.gemm_fp8(cx.lib, cx.stream, t["x8"], t["xs"], t["w8"], t["ws"], t["y"], query_workspace=True)
    assert n > 0
    t["work"] = torch.empty(n, device=cx.device)
    return t


def ranges_run(lib, stream, t):
    """quantise, and both kinds of results through the same scratch, one after the other"""
    ops.fp8_quantize(lib, stream, t["x"], t["x8"], t["xs"])
    a = (lib, stream, t["x8"], t["xs"], t["w8"], t["ws"])
    ops.gemm_fp8(*a, t["y"], bias=t["bias"], residual=t["residual"], workspace=t["work"])
    ops.gemm_fp8(*a, t["y32"], bias=t["bias"], workspace=t["work"])


def case_ranges_command_list(cx, **sizes):
    """the product in ranges recorded into a command list: a replay recomputes from what the buffers then hold"""
    import ctypes

    t = ranges_tensors(cx, 21, **sizes)
    h = ctypes.c_void_p()
    cx.lib.call("hv_cmdlist_begin")
    try:
        ranges_run(cx.lib, cx.stream, t)
    finally:
        cx.lib.call("hv_cmdlist_end", ctypes.byref(h))
    g = torch.Generator().manual_seed(22)
    try:
        for _ in range(2):
            t["x"].copy_(torch.randn(t["x"].shape, generator=g))
            t["work"].fill_(NAN)
            t["y"].zero_()
            t["y32"].zero_()
            cx.lib.call("hv_cmdlist_run", h, cx.stream)
            cx.sync()
            got = t["y"].clone(), t["y32"].clone()
            t["work"].fill_(NAN)
            ranges_run(cx.lib, cx.stream, t)
            cx.sync()
            assert torch.equal(got[0], t["y"]) and torch.equal(got[1], t["y32"]) and bool((t["y32"] != 0).any())
    finally:
        cx.lib.call("hv_cmdlist_destroy", h)
