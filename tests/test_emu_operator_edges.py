"""The cross attention and 8-bit projection operators at values that are not numbers, on the host emulator."""
import pytest

import operator_edge_cases as ec
from test_emu_operators import cx  # noqa: F401  (the fixture)


@pytest.mark.parametrize("how", ["len", "mask", "part"])
@pytest.mark.parametrize("Lq,Lk,heads,kv_heads,D", ec.CROSS_KERNELS)
def test_empty_entries_are_zero_whatever_they_hold(cx, Lq, Lk, heads, kv_heads, D, how):  # noqa: F811
    ec.case_empty_entries(cx, Lq, Lk, heads, kv_heads, D, how, seed=Lk)


@pytest.mark.parametrize("Lq,Lk,heads,kv_heads,D", ec.CROSS_KERNELS)
def test_masks_that_leave_whole_stretches_out(cx, Lq, Lk, heads, kv_heads, D):  # noqa: F811
    ec.case_masked_stretches(cx, Lq, Lk, heads, kv_heads, D, seed=Lk)


def _rc(cx, name, *args):  # noqa: F811
    return getattr(cx.lib.cdll, name)(*args)


def test_sizes_past_one_launch_are_refused(cx):  # noqa: F811
    """a launch has less than 2^32 threads, keys are counted in 32 bits: refused before anything is launched or read"""
    import ctypes as C

    import torch

    from humanvid_amd import _abi as A

    buf = torch.zeros(64, dtype=torch.uint8)
    at = (buf.data_ptr() + 15) // 16 * 16
    # single queries of very many entries that share their states
    p = A.CrossAttentionParams(Q=at, ldq=320, q_stride_b=320, K=at, ldk=320, V=at, ldv=320, O=at, ldo=320, o_stride_b=320,
                               B=2097152, Lq=1, Lk=100, heads=8, kv_heads=8, D=40, scale=1.0)
    for field, value in (("B", 2097152), ("Lk", 0x40000000)):
        p.B, p.Lk = 1, 100
        setattr(p, field, value)
        assert _rc(cx, "hv_cross_attention", C.byref(p), None) == A.HV_EINVAL, field
        assert b"2^32" in cx.lib.cdll.hv_last_error()
        assert _rc(cx, "hv_cross_attention_workspace", C.byref(p), C.byref(C.c_long())) == A.HV_EINVAL, field
    # a row onto more columns than a launch of 16 a workgroup covers
    r = A.GemmFp8Params(X=at, ldx=16, x_scale=at, x_scale_row=1, x_scale_k=1, W=at, ldw=16, w_scale=at, w_scale_row=1, w_scale_k=1,
                        Y=at, ldy=1 << 27, M=1, N=1 << 27, K=16)
    assert _rc(cx, "hv_gemm_fp8", C.byref(r), None) == A.HV_EINVAL and b"2^32" in cx.lib.cdll.hv_last_error()
    assert _rc(cx, "hv_gemm_fp8_workspace", C.byref(r), C.byref(C.c_long())) == A.HV_EINVAL
    for rows, M in ((1, 1 << 28), (128, 65536 * 128)):
        assert _rc(cx, "hv_fp8_quantize", at, 16, M, 16, rows, at, 16, at, 1, 1, None) == A.HV_EINVAL
        assert b"2^32" in cx.lib.cdll.hv_last_error()


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("Lq,Lk,heads,kv_heads,D", ec.CROSS_KERNELS)
def test_a_query_that_is_no_number_stays_in_its_row(cx, Lq, Lk, heads, kv_heads, D, masked):  # noqa: F811
    ec.case_query_values(cx, Lq, Lk, heads, kv_heads, D, masked, seed=Lk + 1)


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("Lq,Lk,heads,kv_heads,D", ec.CROSS_KERNELS)
def test_attended_states_that_are_no_numbers(cx, Lq, Lk, heads, kv_heads, D, masked):  # noqa: F811
    ec.case_state_values(cx, Lq, Lk, heads, kv_heads, D, masked, seed=Lk + 2)


GEMMS = [(5, 40, 272), (33, 24, 144), (100, 133, 272), (70, 50, 2064)]


@pytest.mark.parametrize("out", [ec.BF16, ec.F32])
@pytest.mark.parametrize("M,N,K", GEMMS)
def test_gemm_fp8_operands_that_are_no_numbers(cx, M, N, K, out):  # noqa: F811
    ec.case_gemm_values(cx, M, N, K, out, seed=M)


@pytest.mark.parametrize("out", [ec.BF16, ec.F32])
@pytest.mark.parametrize("tile", [64, 128, 256])
def test_gemm_fp8_tiles_operands_that_are_no_numbers(cx, tile, out):  # noqa: F811
    cx.lib.call("hv_set_tuning", 16, tile)
    try:
        ec.case_gemm_values(cx, 270, 140, 144, out, seed=tile)
    finally:
        cx.lib.call("hv_set_tuning", 16, 0)


def test_command_list_of_a_product_in_ranges(cx):  # noqa: F811
    ec.case_ranges_command_list(cx, M=66, N=40, K=2048)


def test_scratch_that_is_not_aligned_is_named(cx):  # noqa: F811
    import torch

    q, k = torch.zeros(1, 2, 40, dtype=ec.BF16), torch.zeros(1, 2000, 40, dtype=ec.BF16)
    n = ec.ops.cross_attention(cx.lib, cx.stream, q, k, k, q.clone(), heads=1, query_workspace=True)
    with pytest.raises(ValueError, match="16-byte aligned"):
        ec.ops.cross_attention(cx.lib, cx.stream, q, k, k, q.clone(), heads=1, workspace=torch.zeros(n + 1)[1:])
