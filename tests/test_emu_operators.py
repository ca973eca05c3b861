"""The cross attention and 8-bit projection operators on the host emulator: the kernels' indexing, masks, refusals (no GPU)."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(__file__), "emu"))
import build_emu  # noqa: E402

import kernel_cases as kc  # noqa: E402
import operator_cases as oc  # noqa: E402
from humanvid_amd import _abi as A  # noqa: E402
from humanvid_amd import ops  # noqa: E402

BF16, F32, FP8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


@pytest.fixture(scope="module")
def cx():
    return kc.Ctx(A.HvLibrary(build_emu.build()), "cpu", None)


@pytest.mark.parametrize("B,Lq,Lk,heads,kv_heads,D,mask,layout", [
    (1, 1, 1, 1, 1, 40, None, "plain"),
    (2, 1, 4, 2, 2, 40, "len", "plain"),
    (2, 5, 17, 2, 1, 40, "mask", "fused"),
    (1, 70, 77, 1, 1, 40, "mask", "wide"),       # one chunk of 96 keys, two query tiles per wave, ragged rows
    (2, 66, 96, 1, 1, 80, "len", "inplace"),
    (1, 33, 65, 2, 2, 64, "both", "plain"),
    (2, 20, 97, 2, 2, 128, "both", "shared"),    # two chunks of 64
    (1, 130, 130, 1, 1, 160, "mask", "fused"),
    (2, 9, 257, 2, 2, 160, "len", "plain"),      # at most 16 rows: each wave its own keys
    (2, 1, 530, 4, 1, 128, "both", "fused"),     # shared key head, one query
    (3, 2, 1100, 1, 1, 40, "len", "plain"),      # the same, keys cut into ranges
    (1, 5, 1300, 3, 1, 64, "mask", "wide"),      # three heads to a key head
    (3, 20, 600, 1, 1, 80, "both", "fused"),     # ranges of a chunked row block
    (2, 70, 640, 1, 1, 40, "len", "plain"),
    (3, 2, 0, 2, 2, 40, None, "plain"),          # no states at all
    (2, 1, 3, 4, 4, 40, "len", "plain"),         # four heads a workgroup, states in registers
    (1, 131, 77, 4, 4, 40, "mask", "wide"),      # several tiles, the last one ragged
    (2, 70, 33, 4, 2, 64, "both", "fused"),      # shared key heads: two waves of rows each
    (1, 35, 96, 4, 1, 80, "len", "inplace"),     # one key head for all four
    (1, 33, 80, 8, 8, 64, None, "shared"),
    (2, 40, 17, 4, 4, 80, "mask", "plain"),
    (3, 5, 0, 4, 4, 40, None, "plain"),
])
def test_cross_attention(cx, B, Lq, Lk, heads, kv_heads, D, mask, layout):
    oc.case_cross(cx, B, Lq, Lk, heads, kv_heads, D, mask, seed=Lk + D, layout=layout)


def test_cross_attention_large_scores(cx):
    """scores of hundreds: one state takes a row, no overflow"""
    oc.case_cross(cx, 1, 18, 100, 1, 1, 64, seed=3, scale=8.0)


def test_cross_attention_length_out_of_range_is_clamped(cx):
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(3, n, 40, generator=g).to(BF16) for n in (2, 8, 8))
    o, want = torch.empty_like(q), torch.empty_like(q)
    ops.cross_attention(cx.lib, cx.stream, q, k, v, o, heads=1, kv_len=torch.tensor([-5, 2**31 - 1, 3], dtype=torch.int32))
    ops.cross_attention(cx.lib, cx.stream, q, k, v, want, heads=1, kv_len=torch.tensor([0, 8, 3], dtype=torch.int32))
    assert torch.equal(o, want) and bool((o[0] == 0).all())


def test_cross_attention_nan_query_stays_in_its_row(cx):
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(1, n, 40, generator=g).to(BF16) for n in (20, 50, 50))
    o, want = torch.empty_like(q), torch.empty_like(q)
    ops.cross_attention(cx.lib, cx.stream, q, k, v, want, heads=1)
    q[0, 7, 3] = float("nan")
    ops.cross_attention(cx.lib, cx.stream, q, k, v, o, heads=1)
    assert bool(o[0, 7].isnan().all())
    rest = [i for i in range(20) if i != 7]
    assert torch.equal(o[0, rest], want[0, rest])


def test_empty_calls(cx):
    e = torch.empty
    ops.cross_attention(cx.lib, cx.stream, e(0, 4, 40, dtype=BF16), e(0, 3, 40, dtype=BF16), e(0, 3, 40, dtype=BF16), e(0, 4, 40, dtype=BF16), heads=1)
    ops.cross_attention(cx.lib, cx.stream, e(2, 0, 40, dtype=BF16), e(2, 3, 40, dtype=BF16), e(2, 3, 40, dtype=BF16), e(2, 0, 40, dtype=BF16), heads=1)
    ops.fp8_quantize(cx.lib, cx.stream, e(0, 32, dtype=BF16), e(0, 32, dtype=FP8), e(0, 1))
    ops.gemm_fp8(cx.lib, cx.stream, e(0, 32, dtype=FP8), e(0, 1), e(8, 32, dtype=FP8), e(1, 1), e(0, 8))
    ops.gemm_fp8(cx.lib, cx.stream, e(3, 32, dtype=FP8), e(3, 1), e(0, 32, dtype=FP8), e(0, 1), e(3, 0))


@pytest.mark.parametrize("M,K,rows,kw", [
    (1, 16, 1, {}),
    (5, 320, 1, dict(wide=True)),
    (17, 1040, 1, dict(transposed=False, as_bytes=True)),
    (9, 144, 1, dict(special=True)),
    (1, 128, 128, {}),
    (130, 272, 128, dict(wide=True)),
    (128, 128, 128, dict(special=True, transposed=False)),
])
def test_fp8_quantize(cx, M, K, rows, kw):
    oc.case_quantize(cx, M, K, rows, seed=M + K, **kw)


def test_fp8_quantize_every_quotient(cx):
    """every bf16 mantissa against every amax mantissa: 128 x 128 quotients over three binades, middles among them"""
    for lo in range(0, 128, 16):
        rows = []
        for a in range(lo, lo + 16):
            top = 1 + a / 128
            for sh in (0, 3, 9):
                m = (1 + torch.arange(128) / 128) * 2.0**-sh
                rows.append(torch.cat([torch.full((16,), top), torch.where(m > top, m / 2, m), torch.zeros(112)]))
        x = torch.stack(rows).to(BF16)
        want, wscale = oc.e4m3_exact(x, 1)
        q, s = torch.empty_like(want), torch.empty_like(wscale)
        ops.fp8_quantize(cx.lib, cx.stream, x, q, s)
        assert torch.equal(oc.bits(q), oc.bits(want)) and torch.equal(s, wscale)


def test_fp8_quantize_infinity(cx):
    x = torch.ones(2, 256, dtype=BF16)
    x[0, 5] = float("inf")
    q, s = torch.empty(2, 256, dtype=FP8), torch.empty(2, 2)
    ops.fp8_quantize(cx.lib, cx.stream, x, q, s)
    assert bool((q.float() * s.repeat_interleave(128, dim=1))[0, :128].isnan().all())
    assert bool((q.float()[0, 128:] == 448).all()) and bool((q.float()[1] == 448).all())


@pytest.mark.parametrize("M,N,K,kw", [
    (1, 8, 16, {}),
    (1, 40, 1040, dict(out=F32)),
    (17, 130, 320, dict(residual=True)),
    (33, 24, 144, dict(layout="wide", residual=True)),
    (64, 16, 128, dict(layout="odd", bias=False)),
    (65, 70, 320, dict(residual=True)),
    (100, 133, 272, dict(layout="wide", residual=True, out=F32)),
    (70, 64, 128, dict(layout="inplace")),
    (130, 65, 16, dict(layout="odd")),
    (70, 50, 2064, dict(residual=True)),                     # the reduction in ranges, joined
    (66, 40, 2048, dict(layout="wide", out=F32, residual=True)),
    (65, 70, 2560, dict(layout="inplace")),
])
def test_gemm_fp8(cx, M, N, K, kw):
    oc.case_gemm_fp8(cx, M, N, K, seed=M + N + K, **kw)


@pytest.mark.parametrize("tile", [64, 128, 256])
def test_gemm_fp8_tiles(cx, tile):
    cx.lib.call("hv_set_tuning", 16, tile)
    try:
        oc.case_gemm_fp8(cx, 270, 200, 272, seed=tile, residual=True)
        oc.case_gemm_fp8(cx, 260, 264, 144, seed=tile + 2, layout="inplace")
        oc.case_gemm_fp8(cx, 140, 136, 144, seed=tile + 3, residual=True, out=F32)
        oc.case_gemm_fp8(cx, 65, 330, 144, seed=tile + 1, layout="wide", residual=True, out=F32)
    finally:
        cx.lib.call("hv_set_tuning", 16, 0)


def test_gemm_fp8_ranges_need_their_workspace(cx):
    z = torch.zeros
    x, w = z(70, 2048, dtype=FP8), z(50, 2048, dtype=FP8)
    a = (cx.lib, cx.stream, x, z(70, 16), w, z(1, 16), z(70, 50))
    n = ops.gemm_fp8(*a, query_workspace=True)
    assert n > 0
    for bad in (None, z(n - 1)):
        with pytest.raises(ValueError):
            ops.gemm_fp8(*a, workspace=bad)
    ops.gemm_fp8(*a, workspace=z(n))


def test_operators_together(cx):
    oc.case_chain(cx, B=2, Lq=10, Lk=7, heads=2, D=40, cdim=96)


def test_command_list(cx):
    oc.case_command_list(cx)


def _cross(cx, q=(1, 2, 40), k=(1, 3, 40), v=None, o=None, dtype=BF16, **kw):
    e = lambda s: torch.zeros(*s, dtype=dtype)  # noqa: E731
    ops.cross_attention(cx.lib, cx.stream, e(q), e(k), e(v or k), e(o or q), **dict(dict(heads=1), **kw))


@pytest.mark.parametrize("error,kw", [
    (NotImplementedError, dict(q=(1, 2, 48), k=(1, 3, 48))),
    (ValueError, dict(heads=3, q=(1, 2, 120), k=(1, 3, 80), kv_heads=2)),
    (ValueError, dict(heads=0)),
    (ValueError, dict(kv_heads=2)),
    (ValueError, dict(k=(2, 3, 40))),
    (ValueError, dict(v=(1, 4, 40))),
    (ValueError, dict(o=(1, 3, 40))),
    (ValueError, dict(dtype=torch.float16)),
    (ValueError, dict(scale=0.0)),
    (ValueError, dict(scale=-1.0)),
    (ValueError, dict(scale=float("nan"))),
    (ValueError, dict(scale=float("inf"))),
    (ValueError, dict(kv_len=torch.zeros(1, dtype=torch.int64))),
    (ValueError, dict(kv_len=torch.zeros(2, dtype=torch.int32))),
    (ValueError, dict(key_mask=torch.zeros(1, 3))),
    (ValueError, dict(key_mask=torch.zeros(1, 4, dtype=torch.uint8))),
    (ValueError, dict(key_mask=torch.zeros(1, 6, dtype=torch.uint8)[:, ::2])),
    (ValueError, dict(k=(1, 2000, 40))),                                         # cut into ranges: a workspace is needed
    (ValueError, dict(k=(1, 2000, 40), workspace=torch.zeros(10))),
    (ValueError, dict(workspace=torch.zeros(10, dtype=torch.float64))),
])
def test_cross_attention_refuses(cx, error, kw):
    with pytest.raises(error):
        _cross(cx, **kw)


def test_cross_attention_refuses_strides(cx):
    q, k = torch.zeros(1, 2, 44, dtype=BF16)[..., :40], torch.zeros(1, 3, 40, dtype=BF16)
    with pytest.raises(ValueError):
        ops.cross_attention(cx.lib, cx.stream, q, k, k, torch.zeros(1, 2, 40, dtype=BF16), heads=1)  # rows of 88 bytes
    q = torch.zeros(1, 2, 48, dtype=BF16)[..., 1:41]
    with pytest.raises(ValueError):
        ops.cross_attention(cx.lib, cx.stream, q, k, k, torch.zeros(1, 2, 40, dtype=BF16), heads=1)  # 2 bytes off
    q = torch.zeros(1, 2, 80, dtype=BF16)[..., ::2]
    with pytest.raises(ValueError):
        ops.cross_attention(cx.lib, cx.stream, q, k, k, torch.zeros(1, 2, 40, dtype=BF16), heads=1)


def test_outputs_that_overlap_themselves_are_refused(cx):
    q, k = torch.zeros(2, 3, 40, dtype=BF16), torch.zeros(2, 3, 40, dtype=BF16)
    for o in (torch.zeros(1, 3, 40, dtype=BF16).expand(2, -1, -1), torch.zeros(2, 1, 40, dtype=BF16).expand(-1, 3, -1)):
        with pytest.raises(ValueError):
            ops.cross_attention(cx.lib, cx.stream, q, k, k, o, heads=1)
    o = torch.zeros(3, 2, 40, dtype=BF16).transpose(0, 1)  # queries outside, entries inside: fine
    ops.cross_attention(cx.lib, cx.stream, q, k, k, o, heads=1)
    x, w = torch.zeros(4, 64, dtype=FP8), torch.zeros(8, 64, dtype=FP8)
    with pytest.raises(ValueError):
        ops.gemm_fp8(cx.lib, cx.stream, x, torch.zeros(4, 1), w, torch.zeros(1, 1), torch.zeros(1, 8).expand(4, -1))
    with pytest.raises(ValueError):
        ops.fp8_quantize(cx.lib, cx.stream, torch.zeros(4, 256, dtype=BF16), torch.zeros(4, 256, dtype=FP8), torch.zeros(1, 2).expand(4, -1))


def test_gemm_fp8_residual_of_one_row(cx):
    """a residual that is the same row for all (stride 0)"""
    x, xs, w, ws, _, res = oc.gemm_operands(70, 64, 128, 3)
    y, want = torch.empty(70, 64), torch.empty(70, 64)
    ops.gemm_fp8(cx.lib, cx.stream, x, xs, w, ws, y, residual=res[:1].expand(70, -1))
    ops.gemm_fp8(cx.lib, cx.stream, x, xs, w, ws, want, residual=res[:1].expand(70, -1).contiguous())
    assert torch.equal(y, want)


def _quant(cx, x=(4, 64), xt=BF16, q=None, qt=FP8, scale=(4, 1), st=F32, **kw):
    ops.fp8_quantize(cx.lib, cx.stream, torch.zeros(*x, dtype=xt), torch.zeros(*(q or x), dtype=qt), torch.zeros(*scale, dtype=st), **kw)


@pytest.mark.parametrize("kw", [
    dict(x=(4, 40)), dict(x=(4, 0), scale=(4, 0)), dict(xt=F32), dict(qt=torch.float8_e5m2), dict(qt=torch.int8), dict(st=torch.float64),
    dict(scale=(4, 2)), dict(scale=(1, 1)), dict(block_rows=64), dict(q=(4, 80)), dict(block_rows=128, scale=(4, 1)),
])
def test_fp8_quantize_refuses(cx, kw):
    with pytest.raises(ValueError):
        _quant(cx, **kw)


def _gemm(cx, x=(4, 64), w=(8, 64), y=(4, 8), xt=FP8, wt=FP8, yt=F32, xs=(4, 1), ws=(1, 1), st=F32, **kw):
    z = torch.zeros
    ops.gemm_fp8(cx.lib, cx.stream, z(*x, dtype=xt), z(*xs, dtype=st), z(*w, dtype=wt), z(*ws, dtype=st), z(*y, dtype=yt), **kw)


@pytest.mark.parametrize("kw", [
    dict(x=(4, 40), w=(8, 40)), dict(w=(8, 80)), dict(y=(4, 9)), dict(xt=BF16), dict(wt=torch.float8_e5m2), dict(yt=torch.float16),
    dict(xs=(4, 2)), dict(xs=(1, 1)), dict(ws=(2, 1)), dict(st=BF16), dict(bias=torch.zeros(9)), dict(bias=torch.zeros(8, dtype=BF16)),
    dict(residual=torch.zeros(4, 8)), dict(residual=torch.zeros(4, 9, dtype=BF16)), dict(workspace=torch.zeros(4, dtype=BF16)),
])
def test_gemm_fp8_refuses(cx, kw):
    with pytest.raises(ValueError):
        _gemm(cx, **kw)


def test_null_operands_are_refused(cx):
    import ctypes as C

    p = A.CrossAttentionParams(B=1, Lq=1, Lk=1, heads=1, kv_heads=1, D=40, scale=1.0)
    assert cx.lib.cdll.hv_cross_attention(C.byref(p), None) == A.HV_EINVAL
    assert cx.lib.cdll.hv_cross_attention(None, None) == A.HV_EINVAL
    p.Lq = -1
    assert cx.lib.cdll.hv_cross_attention(C.byref(p), None) == A.HV_EINVAL
    assert cx.lib.cdll.hv_cross_attention_workspace(C.byref(p), C.byref(C.c_long())) == A.HV_EINVAL
    for field, value in (("ldq", -8), ("k_stride_b", -40), ("ldk", 1 << 25), ("mask_stride_b", -1)):
        buf = torch.zeros(64, dtype=BF16)
        p = A.CrossAttentionParams(B=1, Lq=1, Lk=1, heads=1, kv_heads=1, D=40, scale=1.0, Q=buf.data_ptr(), K=buf.data_ptr(), V=buf.data_ptr(),
                                   O=buf.data_ptr(), ldq=40, ldk=40, ldv=40, ldo=40)
        assert cx.lib.cdll.hv_cross_attention(C.byref(p), None) == A.HV_OK
        setattr(p, field, value)
        assert cx.lib.cdll.hv_cross_attention(C.byref(p), None) == A.HV_EINVAL, field
    r = A.GemmFp8Params(M=1, N=1, K=16)
    assert cx.lib.cdll.hv_gemm_fp8(C.byref(r), None) == A.HV_EINVAL
    assert cx.lib.cdll.hv_gemm_fp8(None, None) == A.HV_EINVAL
    assert cx.lib.cdll.hv_fp8_quantize(None, 0, 1, 16, 1, None, 0, None, 0, 0, None) == A.HV_EINVAL
