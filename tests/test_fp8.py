"""The 8-bit matrices without a GPU: the C structs' layouts, the checks that
their entries make of the arguments, the bindings' checks of their buffers (no
launch is made of what they refuse), and the oracle's own format."""

import ctypes
import re
from pathlib import Path

import numpy as np
import pytest

import fp8_cases as F
from furykernel_amd import fp8, runtime
from furykernel_amd.kernels import LaunchError
from test_serve import DEVICE, FakeBuffer, FakeDevice

HEADER = (Path(__file__).resolve().parents[1] / "include" / "fkrocm_fp8.h").read_text()
STRUCTS = {"fk_fp8_quantize_args": fp8.QuantizeArgs, "fk_fp8_dequantize_args": fp8.DequantizeArgs,
           "fk_fp8_add_norm_args": fp8.AddNormArgs, "fk_fp8_gemm_args": fp8.GemmArgs}


def fields_of(header, name):
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), header, re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    fields = []
    for decl in filter(None, (d.strip() for d in body.split(";"))):
        kind, names = decl.split(None, 1)
        fields += [(n.strip(), {"uint64_t": ctypes.c_uint64, "uint32_t": ctypes.c_uint32,
                                "float": ctypes.c_float}[kind]) for n in names.split(",")]
    return fields


@pytest.mark.parametrize("name", sorted(STRUCTS))
def test_the_structs_fields_are_the_headers(name):
    assert STRUCTS[name]._fields_ == fields_of(HEADER, name)


def test_the_oracles_codes_are_the_formats():
    assert F.MAGNITUDES[-1] == 448 and F.MAGNITUDES[1] == 2.0 ** -9 and F.MAGNITUDES[8] == 2.0 ** -6
    assert np.array_equal(F.encode(F.MAGNITUDES), np.arange(127)) and np.array_equal(F.encode(-F.MAGNITUDES[1:]),
                                                                                      np.arange(129, 255))
    mid = (F.MAGNITUDES[1:] + F.MAGNITUDES[:-1]) / 2
    even = np.arange(126) + np.arange(126) % 2
    assert np.array_equal(F.encode(mid), even)
    assert np.array_equal(F.encode(np.nextafter(mid, 0)), np.arange(126))
    assert np.array_equal(F.encode(np.nextafter(mid, 500)), np.arange(1, 127))
    assert F.scale_of(448.0) == 1 and F.scale_of(np.nextafter(448.0, 500)) == 2 and F.scale_of(224.0) == 0.5
    assert F.scale_of(0.0) == 2.0 ** -126 and F.scale_of(2.0 ** -140) == 2.0 ** -126
    codes, scale = F.quantize(np.random.default_rng(0).standard_normal((21, 700)))
    back = F.unpack(*F.pack(codes, scale), 21, 700)
    assert np.array_equal(back[0], codes) and np.array_equal(back[1], scale)


class FakeMatrix(fp8.Fp8Matrix):
    def __init__(self, rows, k, device=DEVICE):
        lib = runtime.library()
        self.device, self.rows, self.k = device, rows, k
        self.codes = FakeBuffer(max(lib.fk_fp8_codes_bytes(rows, k), 16), device)
        self.scales = FakeBuffer(max(lib.fk_fp8_scales_bytes(rows, k), 16), device)


def test_sizes_of_matrices():
    lib = runtime.library()
    assert lib.fk_fp8_codes_bytes(1, 1) == 16 * 128 and lib.fk_fp8_scales_bytes(1, 1) == 64
    assert lib.fk_fp8_codes_bytes(17, 129) == 32 * 256 and lib.fk_fp8_scales_bytes(17, 513) == 2 * 2 * 64
    for rows, k in ((0, 8), (8, 0), (1 << 31, 1), (1, 1 << 31), (1 << 20, 1 << 20), (512, 128 * ((1 << 21) - 1) + 1)):
        assert lib.fk_fp8_codes_bytes(rows, k) == 0 and lib.fk_fp8_scales_bytes(rows, k) == 0
        with pytest.raises(LaunchError):
            fp8.Fp8Matrix(DEVICE, rows, k)
    assert lib.fk_fp8_codes_bytes(512, 128 * ((1 << 21) - 1)) == 512 * 128 * ((1 << 21) - 1)


def test_quantize_and_back_take_what_they_say_and_refuse_the_rest():
    m = FakeMatrix(9, 1000)
    x = FakeBuffer(9 * 1000 * 4)
    fp8.Quantize(DEVICE, x, m)
    fp8.Quantize(DEVICE, FakeBuffer(9 * 1003 * 2), m, x_type="bf16", x_stride=1003, x_offset=3)
    fp8.Dequantize(DEVICE, m, FakeBuffer(9 * 1000 * 4), scales=FakeBuffer(9 * 8 * 4))
    for bad in (lambda: fp8.Quantize(DEVICE, FakeBuffer(9 * 1000 * 4 - 1), m),
                lambda: fp8.Quantize(DEVICE, x, m, x_type="f64"),
                lambda: fp8.Quantize(DEVICE, x, m, x_stride=999),
                lambda: fp8.Quantize(DEVICE, x, m, x_offset=1),
                lambda: fp8.Quantize(DEVICE, x, m, x_offset=-1),
                lambda: fp8.Quantize(DEVICE, FakeBuffer(9 * 1000 * 4, ptr=x.ptr + 2), m),
                lambda: fp8.Quantize(DEVICE, FakeBuffer(9 * 1000 * 4, ptr=m.codes.ptr), m),
                lambda: fp8.Quantize(DEVICE, FakeBuffer(9 * 1000 * 4, FakeDevice()), m),
                lambda: fp8.Dequantize(DEVICE, m, FakeBuffer(9 * 1000 * 2)),
                lambda: fp8.Dequantize(DEVICE, m, FakeBuffer(9 * 1000 * 4), y_stride=10),
                lambda: fp8.Dequantize(DEVICE, m, x, scales=FakeBuffer(9 * 8 * 4 - 1)),
                lambda: fp8.Dequantize(DEVICE, m, x, scales=FakeBuffer(9 * 8 * 4, ptr=x.ptr)),
                lambda: fp8.Dequantize(DEVICE, m, FakeBuffer(9 * 1000 * 4, ptr=m.scales.ptr))):
        with pytest.raises(LaunchError):
            bad()


def norm(**over):
    n = dict(rows=9, k=1000, wide=4)
    bufs = dict(x=FakeBuffer(n["rows"] * n["k"] * 4), gamma=FakeBuffer(n["k"] * 4), to=FakeMatrix(n["rows"], n["k"]),
                eps=1e-5)
    return fp8.AddNorm(DEVICE, **(bufs | over))


def test_add_norm_takes_what_it_says_and_refuses_the_rest():
    size = 9 * 1000 * 4
    x, r = FakeBuffer(size), FakeBuffer(size)
    norm()
    norm(gamma=None)
    norm(residual=r, sum=FakeBuffer(size))
    norm(x=x, residual=r, sum=r)                       # the stream in place
    norm(x=x, residual=r, sum=x)
    norm(x=x, sum=x)
    norm(x=x, residual=x, sum=x)
    norm(residual=r)
    norm(x=FakeBuffer(9 * 1003 * 2), x_type="f16", x_stride=1003, x_offset=1)
    norm(to=FakeMatrix(1, 32768), x=FakeBuffer(1 << 20), gamma=None)
    m = FakeMatrix(9, 1000)
    for over in (dict(x=FakeBuffer(size - 4)), dict(gamma=FakeBuffer(3996)), dict(residual=FakeBuffer(size - 4)),
                 dict(sum=FakeBuffer(size - 4)), dict(x_type="f8"), dict(eps=-1e-5), dict(eps=float("nan")),
                 dict(eps=float("inf")), dict(x_stride=999), dict(residual=r, residual_stride=999),
                 dict(sum=FakeBuffer(size), sum_stride=999),
                 dict(x=x, sum=FakeBuffer(size, ptr=x.ptr + 4)),
                 dict(x=FakeBuffer(9 * 1003 * 4, ptr=x.ptr), x_stride=1003, sum=FakeBuffer(size, ptr=x.ptr)),
                 dict(residual=r, sum=FakeBuffer(size, ptr=r.ptr - 4)),
                 dict(x=x, residual=FakeBuffer(size, ptr=x.ptr + 4000), sum=x),
                 dict(to=m, x=FakeBuffer(size, ptr=m.codes.ptr)), dict(to=m, sum=FakeBuffer(size, ptr=m.scales.ptr)),
                 dict(to=m, gamma=FakeBuffer(4000, ptr=m.codes.ptr)),
                 dict(gamma=FakeBuffer(4000, ptr=x.ptr), sum=x),
                 dict(gamma=FakeBuffer(4000, ptr=x.ptr + 4)),
                 dict(to=FakeMatrix(1, 32769), x=FakeBuffer(1 << 20), gamma=None),
                 dict(to=FakeMatrix(1 << 22, 8), x=FakeBuffer(1 << 27), gamma=None)):
        with pytest.raises(LaunchError):
            norm(**over)


def test_products_take_what_they_say_and_refuse_the_rest():
    a, b = FakeMatrix(9, 1000), FakeMatrix(40, 1000)
    fp8.Gemm(DEVICE, a, b, FakeBuffer(9 * 40 * 4))
    fp8.Gemm(DEVICE, a, b, FakeBuffer(9 * 41 * 2), c_type="bf16", c_stride=41)
    for bad in (lambda: fp8.Gemm(DEVICE, a, FakeMatrix(40, 1001), FakeBuffer(9 * 40 * 4)),
                lambda: fp8.Gemm(DEVICE, a, b, FakeBuffer(9 * 40 * 4 - 1)),
                lambda: fp8.Gemm(DEVICE, a, b, FakeBuffer(9 * 40 * 4), c_stride=39),
                lambda: fp8.Gemm(DEVICE, a, b, FakeBuffer(9 * 40 * 4), c_type="i8"),
                lambda: fp8.Gemm(DEVICE, a, b, FakeBuffer(9 * 40 * 4, ptr=a.codes.ptr)),
                lambda: fp8.Gemm(DEVICE, a, b, FakeBuffer(9 * 40 * 4, ptr=b.scales.ptr)),
                lambda: fp8.Gemm(DEVICE, a, b, FakeBuffer(9 * 40 * 4, FakeDevice()))):
        with pytest.raises(LaunchError):
            bad()
    assert fp8.gemm_form(0, 8, 8) == "" and fp8.gemm_form(1 << 29, 1 << 29, 8, "f16") == ""
    for c in ("f32", "f16", "bf16"):
        assert fp8.gemm_form(8, 8192, 2048, c).startswith("few")
        assert fp8.gemm_form(8192, 8192, 2048, c).startswith("many")


def test_a_null_address_a_bad_type_and_an_unknown_size_of_arguments():
    args = fp8.GemmArgs(0, 1 << 20, 1 << 21, 1 << 22, 1 << 23, 40, 9, 40, 1000, 0)
    for over in ({}, {"a_codes": 1 << 24, "c_type": 3}, {"a_codes": 1 << 24, "c": 0}, {"a_codes": (1 << 24) + 8}):
        for k, v in over.items():
            setattr(args, k, v)
        with pytest.raises(runtime.FkError):
            runtime.serve_check("fk_fp8_gemm", args)
    with pytest.raises(runtime.FkError):
        runtime.serve_check("fk_fp8_gemm", fp8.QuantizeArgs())
