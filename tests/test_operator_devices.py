"""Operands in host memory are refused by the GPU library before anything is launched (no GPU is used: a library that launches fails)."""
import os

import pytest
import torch

from humanvid_amd import _abi as A
from humanvid_amd import build as hvbuild
from humanvid_amd import ops

BF16, F32, FP8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


class _NoLaunch:
    host = False  # as the GPU library

    def call(self, name, *args):
        raise AssertionError(f"{name} was called")


def _cross(lib, **kw):
    t = [torch.zeros(1, n, 40, dtype=BF16) for n in (2, 3, 3, 2)]
    ops.cross_attention(lib, 0, *t, heads=1, **kw)


def _quantize(lib):
    ops.fp8_quantize(lib, 0, torch.zeros(4, 64, dtype=BF16), torch.zeros(4, 64, dtype=FP8), torch.zeros(4, 1))


def _gemm(lib, **kw):
    ops.gemm_fp8(lib, 0, torch.zeros(4, 64, dtype=FP8), torch.zeros(4, 1), torch.zeros(8, 64, dtype=FP8), torch.zeros(1, 1), torch.zeros(4, 8), **kw)


@pytest.mark.parametrize("call", [
    _cross, _quantize, _gemm,
    lambda lib: _cross(lib, kv_len=torch.zeros(1, dtype=torch.int32), key_mask=torch.ones(1, 3, dtype=torch.uint8)),
    lambda lib: _gemm(lib, bias=torch.zeros(8), residual=torch.zeros(4, 8, dtype=BF16)),
])
def test_host_tensors_are_refused(call):
    with pytest.raises(ValueError, match="cpu"):
        call(_NoLaunch())


def test_the_built_library_is_the_gpu_library():
    if not os.path.exists(hvbuild.LIB):
        hvbuild.build()
    lib = A.HvLibrary(hvbuild.LIB)
    assert lib.host is False
    for call in (_cross, _quantize, _gemm):
        with pytest.raises(ValueError, match="cpu"):
            call(lib)


def test_the_emulated_library_takes_host_tensors():
    import sys

    sys.path.insert(0, os.path.join(os.path.dirname(__file__), "emu"))
    import build_emu

    lib = A.HvLibrary(build_emu.build())
    assert lib.host is True
    for call in (_cross, _quantize, _gemm):
        call(lib)
