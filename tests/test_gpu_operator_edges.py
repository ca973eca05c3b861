"""The cross attention and 8-bit projection operators at values that are not numbers, on a real MI355X."""
import pytest

import operator_edge_cases as ec
from test_gpu_operators import cx  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu
SIZES = ec.CROSS_KERNELS + [(1000, 77, 8, 2, 40), (300, 700, 8, 8, 160), (8, 4109, 16, 4, 128), (200, 3000, 4, 4, 80)]


@pytest.mark.parametrize("how", ["len", "mask", "part"])
@pytest.mark.parametrize("Lq,Lk,heads,kv_heads,D", SIZES)
def test_empty_entries_are_zero_whatever_they_hold(cx, Lq, Lk, heads, kv_heads, D, how):  # noqa: F811
    ec.case_empty_entries(cx, Lq, Lk, heads, kv_heads, D, how, seed=Lk)


@pytest.mark.parametrize("Lq,Lk,heads,kv_heads,D", SIZES)
def test_masks_that_leave_whole_stretches_out(cx, Lq, Lk, heads, kv_heads, D):  # noqa: F811
    ec.case_masked_stretches(cx, Lq, Lk, heads, kv_heads, D, seed=Lk)


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("Lq,Lk,heads,kv_heads,D", SIZES)
def test_a_query_that_is_no_number_stays_in_its_row(cx, Lq, Lk, heads, kv_heads, D, masked):  # noqa: F811
    ec.case_query_values(cx, Lq, Lk, heads, kv_heads, D, masked, seed=Lk + 1)


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("Lq,Lk,heads,kv_heads,D", SIZES)
def test_attended_states_that_are_no_numbers(cx, Lq, Lk, heads, kv_heads, D, masked):  # noqa: F811
    ec.case_state_values(cx, Lq, Lk, heads, kv_heads, D, masked, seed=Lk + 2)


@pytest.mark.parametrize("out", [ec.BF16, ec.F32])
@pytest.mark.parametrize("M,N,K", [(5, 40, 272), (33, 24, 144), (100, 133, 272), (70, 50, 2064), (4100, 2050, 400)])
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
