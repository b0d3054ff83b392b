"""What the 8-bit matrices' entries take and refuse, beside test_fp8.py's."""

import pytest

from furykernel_amd import fp8, runtime
from furykernel_amd.kernels import LaunchError
from test_fp8 import FakeMatrix
from test_serve import DEVICE, FakeBuffer


def test_cut_sums_are_of_products_to_16_bits():
    a, b, c = FakeMatrix(9, 1000), FakeMatrix(40, 1000), FakeBuffer(9 * 40 * 4)
    for kind in ("f16", "bf16"):
        fp8.Gemm(DEVICE, a, b, c, c_type=kind, cut_sums=True)
        for s in ((1, 16, 32), (100, 5000, 3080), (8192, 8192, 2048)):
            assert fp8.gemm_form(*s, kind, cut_sums=True) and fp8.gemm_form(*s, kind)
    with pytest.raises(LaunchError):
        fp8.Gemm(DEVICE, a, b, c, cut_sums=True)
    with pytest.raises(LaunchError):
        fp8.gemm_form(9, 40, 1000, "f32", cut_sums=True)
    args = fp8.GemmArgs(1 << 20, 1 << 21, 1 << 22, 1 << 23, 1 << 24, 40, 9, 40, 1000, 0)
    for c_type, taken in ((0, True), (1, True), (2, True), (0x101, True), (0x102, True), (3, False), (0x100, False),
                          (0x103, False), (0x201, False), (0x301, False), (1 << 31, False)):
        args.c_type = c_type
        form = runtime.library().fk_fp8_gemm_form(9, 40, 1000, c_type)
        if taken:
            runtime.serve_check("fk_fp8_gemm", args)
            assert form
        else:
            with pytest.raises(runtime.FkError):
                runtime.serve_check("fk_fp8_gemm", args)
            assert form == b""
