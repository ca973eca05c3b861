"""The cross attention and 8-bit projection operators on a real MI355X through the C ABI."""
import math

import pytest
import torch

import kernel_cases as kc
import operator_cases as oc
from humanvid_amd import ops

pytestmark = pytest.mark.gpu
BF16, F32, F64, FP8 = torch.bfloat16, torch.float32, torch.float64, torch.float8_e4m3fn


@pytest.fixture(scope="module")
def cx():
    from humanvid_amd import lib

    lib.require_gpu()
    return kc.Ctx(lib.load(), "cuda", lib.current_stream())


@pytest.mark.parametrize("B,Lq,Lk,heads,kv_heads,D,mask,layout", [
    (1, 1, 1, 8, 8, 40, None, "plain"),
    (2, 1, 4, 8, 8, 40, "len", "plain"),
    (2, 777, 77, 8, 8, 40, None, "fused"),
    (2, 1000, 77, 8, 8, 40, "mask", "wide"),
    (2, 384, 96, 8, 4, 80, "len", "inplace"),
    (3, 130, 65, 4, 4, 64, "both", "plain"),
    (2, 96, 257, 8, 8, 160, None, "fused"),
    (2, 96, 257, 8, 8, 160, "both", "shared"),
    (2, 200, 1025, 16, 4, 128, "len", "fused"),
    (4, 1, 4109, 16, 4, 128, "both", "fused"),
    (2, 3, 8192, 8, 2, 40, "len", "plain"),
    (1, 17, 3001, 4, 4, 160, "mask", "wide"),
    (3, 64, 0, 8, 8, 80, None, "plain"),
    (1, 40000, 33, 8, 8, 40, "mask", "plain"),
    (2, 600, 700, 8, 8, 80, "mask", "plain"),
])
def test_cross_attention(cx, B, Lq, Lk, heads, kv_heads, D, mask, layout):
    oc.case_cross(cx, B, Lq, Lk, heads, kv_heads, D, mask, seed=Lk + D, layout=layout)


def test_cross_attention_large_scores(cx):
    oc.case_cross(cx, 2, 200, 500, 4, 4, 64, seed=3, scale=8.0)


def test_cross_attention_offsets_past_32_bits(cx):
    """states whose rows are 2 MiB apart: byte offsets up to 9 GiB inside one entry"""
    Lk, H, D = 4500, 2, 80
    C = H * D
    g = torch.Generator().manual_seed(9)
    ks, vs, q = (torch.randn(1, n, C, generator=g).to(BF16) for n in (Lk, Lk, 100))
    far = torch.empty(Lk << 20, dtype=BF16, device="cuda").view(1, Lk, 1 << 20)
    k, v = far[..., :C], far[..., 1 << 19:(1 << 19) + C]
    k.copy_(ks)
    v.copy_(vs)
    ref, tol = oc.cross_reference(q, ks, vs, H, H, torch.ones(1, Lk, dtype=torch.bool), 1 / math.sqrt(D))
    for rows in (1, 100):  # cut into ranges, and not
        o = torch.empty(1, rows, C, dtype=BF16, device="cuda")
        oc.run_cross(cx, q[:, :rows].cuda(), k, v, o, H, H)
        cx.sync()
        assert bool(((o.cpu().to(F64) - ref[:, :rows]).abs() <= tol[:, :rows]).all())


@pytest.mark.parametrize("M,K,rows,kw", [
    (1, 16, 1, {}), (1000, 320, 1, dict(wide=True)), (257, 1040, 1, dict(transposed=False, as_bytes=True)), (300, 5120, 1, {}),
    (100, 144, 1, dict(special=True)), (1280, 1280, 128, {}), (130, 272, 128, dict(wide=True)), (128, 128, 128, dict(special=True, transposed=False)),
])
def test_fp8_quantize(cx, M, K, rows, kw):
    oc.case_quantize(cx, M, K, rows, seed=M + K, **kw)


@pytest.mark.parametrize("M,N,K,kw", [
    (1, 8, 16, {}),
    (1, 1280, 5120, dict(out=F32)),
    (17, 1000, 1040, dict(residual=True)),
    (33, 321, 320, dict(layout="wide", residual=True)),
    (64, 2560, 640, dict(layout="odd", bias=False)),
    (65, 70, 320, dict(residual=True)),
    (1000, 1333, 272, dict(layout="wide", residual=True, out=F32)),
    (700, 640, 2560, dict(layout="inplace")),
    (4099, 2050, 1296, dict(layout="odd")),
    (9216, 4096, 640, {}),
    (20000, 960, 320, dict(residual=True)),
    (100, 200, 5120, dict(residual=True)),
    (700, 333, 4112, dict(layout="wide", out=F32, residual=True)),
    (129, 640, 2560, dict(layout="inplace")),
    (300, 70, 5104, dict(layout="odd")),
])
def test_gemm_fp8(cx, M, N, K, kw):
    oc.case_gemm_fp8(cx, M, N, K, seed=M + N + K, ref_device="cuda", **kw)


@pytest.mark.parametrize("tile", [64, 128, 256])
def test_gemm_fp8_tiles(cx, tile):
    cx.lib.call("hv_set_tuning", 16, tile)
    try:
        oc.case_gemm_fp8(cx, 1541, 1000, 1040, seed=tile, residual=True, ref_device="cuda")
        oc.case_gemm_fp8(cx, 4100, 1288, 400, seed=tile + 2, layout="inplace", ref_device="cuda")
        oc.case_gemm_fp8(cx, 2100, 1288, 400, seed=tile + 3, residual=True, out=F32, ref_device="cuda")
        oc.case_gemm_fp8(cx, 300, 330, 144, seed=tile + 1, layout="wide", residual=True, out=F32, ref_device="cuda")
    finally:
        cx.lib.call("hv_set_tuning", 16, 0)


def test_operators_together(cx):
    oc.case_chain(cx, B=2, Lq=500, Lk=77, heads=8, D=40, cdim=768)
    oc.case_chain(cx, B=2, Lq=96, Lk=257, heads=8, D=160, cdim=1024, seed=1)


def test_command_list(cx):
    oc.case_command_list(cx)


def _everything(lib, stream, t):
    ops.cross_attention(lib, stream, t["q"], t["k"], t["v"], t["o"], heads=8, key_mask=t["mask"], workspace=t["work"])
    ops.fp8_quantize(lib, stream, t["o"].view(-1, 320), t["x8"], t["xs"])
    ops.gemm_fp8(lib, stream, t["x8"], t["xs"], t["w8"], t["ws"], t["y"], workspace=t["gwork"])


def _tensors(cx, B, Lq, Lk, seed):
    g = torch.Generator().manual_seed(seed)
    t = {n: torch.randn(B, L, 320, generator=g).to(BF16).cuda() for n, L in (("q", Lq), ("k", Lk), ("v", Lk))}
    t["mask"] = (torch.rand(B, Lk, generator=g) < 0.8).cuda()
    t["o"] = torch.zeros_like(t["q"])
    n = ops.cross_attention(cx.lib, cx.stream, t["q"], t["k"], t["v"], t["o"], heads=8, query_workspace=True)
    t["work"] = torch.empty(n, device="cuda") if n else None
    t["x8"], t["xs"] = torch.empty(B * Lq, 320, dtype=FP8, device="cuda"), torch.empty(3, B * Lq, device="cuda").t()
    w = torch.randn(640, 320, generator=g).to(BF16).cuda()
    t["w8"], t["ws"] = torch.empty(640, 320, dtype=FP8, device="cuda"), torch.empty(5, 3, device="cuda")
    ops.fp8_quantize(cx.lib, cx.stream, w, t["w8"], t["ws"], block_rows=128)
    t["y"] = torch.zeros(B * Lq, 640, device="cuda")
    n = ops.gemm_fp8(cx.lib, cx.stream, t["x8"], t["xs"], t["w8"], t["ws"], t["y"], query_workspace=True)
    t["gwork"] = torch.empty(n, device="cuda") if n else None
    return t


@pytest.mark.parametrize("Lq,Lk", [(2, 2000), (500, 77)])
def test_graph_replays(cx, Lq, Lk):
    """captured once, replayed on new data, with eager calls of other data between the replays"""
    t, other = _tensors(cx, 2, Lq, Lk, 1), _tensors(cx, 2, Lq, Lk, 2)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        _everything(cx.lib, s.cuda_stream, t)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _everything(cx.lib, torch.cuda.current_stream().cuda_stream, t)
    for i in range(4):
        t["q"].normal_()
        t["mask"].copy_(torch.rand(t["mask"].shape, device="cuda") < 0.5)
        graph.replay()
        torch.cuda.synchronize()
        got = t["o"].clone(), t["y"].clone()
        _everything(cx.lib, cx.stream, other)
        t["o"].zero_()
        t["y"].zero_()
        _everything(cx.lib, cx.stream, t)
        torch.cuda.synchronize()
        assert torch.equal(got[0], t["o"]) and torch.equal(got[1], t["y"]) and bool((t["y"] != 0).any())


def test_two_streams_at_once(cx):
    """two runs at the same time, each with its own workspace, give what each gives alone; twice the same bits"""
    a, b = _tensors(cx, 2, 3, 3000, 3), _tensors(cx, 2, 3, 3000, 4)
    want = []
    for t in (a, b):
        _everything(cx.lib, cx.stream, t)
        torch.cuda.synchronize()
        want.append((t["o"].clone(), t["y"].clone()))
        t["o"].zero_()
        t["y"].zero_()
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(20):
        _everything(cx.lib, s1.cuda_stream, a)
        _everything(cx.lib, s2.cuda_stream, b)
    torch.cuda.synchronize()
    for t, w in zip((a, b), want):
        assert torch.equal(t["o"], w[0]) and torch.equal(t["y"], w[1])


def test_current_stream_is_torchs():
    from humanvid_amd import lib

    side = torch.cuda.Stream()
    assert lib.current_stream() == torch.cuda.current_stream().cuda_stream
    with torch.cuda.stream(side):
        assert lib.current_stream() == side.cuda_stream == torch.cuda.current_stream().cuda_stream
    assert lib.current_stream() == torch.cuda.current_stream().cuda_stream
