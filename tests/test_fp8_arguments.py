"""What the 8-bit matrices' entries take and refuse, beside test_fp8.py's."""

import pytest

from furykernel_amd import fp8, mx4, runtime
from furykernel_amd.kernels import LaunchError
from test_fp8 import FakeMatrix, norm
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
            with pytest.raises(runtime.FkError) as refusal:
                runtime.serve_check("fk_fp8_gemm", args)
            assert form == b"" and refusal.value.status == -2   # FK_ERR_ARG


def test_a_norm_s_sum_lies_over_rows_of_its_own_stride_only():
    """x and the residual in one buffer at two strides: the sum's row 2 would be the
    other's row 1, which another threadgroup reads."""
    x = FakeBuffer(9 * 2000 * 4)
    both = dict(x=x, residual=x, sum=x)
    norm(**both)
    norm(**both, x_stride=2000, residual_stride=2000, sum_stride=2000)
    for over in (dict(residual_stride=2000), dict(x_stride=2000), dict(sum_stride=2000),
                 dict(x_stride=2000, sum_stride=2000), dict(residual_stride=2000, sum_stride=2000),
                 dict(x_stride=1001, residual_stride=2000, sum_stride=1001)):
        with pytest.raises(LaunchError):
            norm(**both, **over)
    r = FakeBuffer(9 * 1000 * 4, ptr=x.ptr)
    for over in (dict(sum=x, sum_stride=2000), dict(sum=r), dict(sum=r, residual_stride=1001)):
        with pytest.raises(LaunchError):
            norm(x=x, x_stride=2000, residual=r, **over)
    norm(x=x, x_stride=2000, residual=r)               # read only
    one = FakeBuffer(1000 * 4)                         # (a row has no stride)
    norm(x=one, x_stride=2000, residual=one, sum=one, to=FakeMatrix(1, 1000))


def test_a_norm_whose_launch_would_be_2_to_32_threads():
    """Row tiles go by eights, one an XCD: their rounding up counts."""
    def taken(rows, k):
        args = fp8.AddNormArgs(x=1 << 45, codes=1 << 46, scales=1 << 47, x_stride=k, rows=rows, k=k, x_type=2, eps=1e-5)
        try:
            runtime.serve_check("fk_fp8_add_norm", args)
        except runtime.FkError:
            return False
        return True

    most = 16 * ((1 << 18) - 8)
    for k in (16384, 15361, 32768, 30721):              # threadgroups of 1024 threads, a row each
        assert taken(most, k) and not taken(most + 1, k) and not taken(most + 16 * 7, k)
    for k in (15360, 8192, 2048, 1):                    # fewer threads
        assert taken(most + 1, k) and taken(most + 16 * 7, k) and not taken(most + 16 * 7 + 1, k)


@pytest.mark.parametrize("kind", [fp8.Fp8Matrix, mx4.Mx4Matrix])
def test_a_matrix_whose_scales_find_no_memory_leaves_none_taken(kind):
    class Device:
        taken = 0

        def alloc(self, nbytes):
            if self.taken:
                raise runtime.FkError(1, "no memory")
            self.taken += 1
            buf = FakeBuffer(nbytes, self)
            buf.free = lambda: setattr(self, "taken", self.taken - 1)
            return buf

    device = Device()
    with pytest.raises(runtime.FkError):
        kind(device, 100, 1000)
    assert device.taken == 0
