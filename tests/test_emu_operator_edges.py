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
