"""8-bit matrices with a scale for each block of 128 (include/fkrocm_fp8.h):
a model's weights and activations as e4m3 values over powers of two, their
products on the matrix cores.

* ``Fp8Matrix`` — a matrix's codes and scales in device memory.
* ``Quantize``, ``Dequantize`` — rows of f32, f16 or bf16 to it and back.
* ``AddNorm`` — the residual's addition, RMSNorm, and that to 8 bits.
* ``Gemm`` — C = A Bᵀ of two of them.

The operations are bound to their buffers once and queued by
``enqueue(stream)``.
"""

from __future__ import annotations

import ctypes

from . import runtime
from .kernels import LaunchError
from .paged import _U32, _U64, TYPES, admit, element, need, row_stride, whole


class QuantizeArgs(ctypes.Structure):
    """fk_fp8_quantize_args."""
    _fields_ = [(f, _U64) for f in ("x", "codes", "scales", "x_stride")] + \
        [(f, _U32) for f in ("rows", "k", "x_type")]


class DequantizeArgs(ctypes.Structure):
    """fk_fp8_dequantize_args."""
    _fields_ = [(f, _U64) for f in ("codes", "scales", "y", "scales_out", "y_stride")] + \
        [(f, _U32) for f in ("rows", "k", "y_type")]


class AddNormArgs(ctypes.Structure):
    """fk_fp8_add_norm_args."""
    _fields_ = [(f, _U64) for f in ("x", "residual", "sum", "gamma", "codes", "scales", "x_stride",
                                    "residual_stride", "sum_stride")] + \
        [(f, _U32) for f in ("rows", "k", "x_type")] + [("eps", ctypes.c_float)]


class GemmArgs(ctypes.Structure):
    """fk_fp8_gemm_args."""
    _fields_ = [(f, _U64) for f in ("a_codes", "a_scales", "b_codes", "b_scales", "c", "c_stride")] + \
        [(f, _U32) for f in ("m", "n", "k", "c_type")]


class Fp8Matrix:
    """[rows, k] at 8 bits: its codes and scales, of which ``Quantize`` and
    ``AddNorm`` write every byte (padding included) and nothing before holds
    anything."""

    def __init__(self, device: runtime.Device, rows: int, k: int):
        whole("Fp8Matrix", rows=rows, k=k)
        lib = runtime.library()
        sizes = lib.fk_fp8_codes_bytes(rows, k), lib.fk_fp8_scales_bytes(rows, k)
        if not all(sizes):
            raise LaunchError(f"Fp8Matrix: no matrix of {rows} rows of {k}")
        self.device, self.rows, self.k = device, rows, k
        self.codes = device.alloc(sizes[0])
        try:
            self.scales = device.alloc(sizes[1])
        except runtime.FkError:
            self.codes.free()
            raise

    def free(self) -> None:
        self.codes.free()
        self.scales.free()

    def _held(self, entry: str, name: str, device: runtime.Device) -> tuple[int, int]:
        lib = runtime.library()
        return (need(entry, f"{name}'s codes", self.codes, lib.fk_fp8_codes_bytes(self.rows, self.k), device),
                need(entry, f"{name}'s scales", self.scales, lib.fk_fp8_scales_bytes(self.rows, self.k), device))


class Quantize(runtime.Operation):
    """Rows x [rows][k] of `x_type`, `x_stride` elements apart and `x_offset`
    elements into their buffer, to `to` (fk_fp8_quantize)."""

    def __init__(self, device, x: runtime.Buffer, to: Fp8Matrix, x_type: str = "f32", x_stride: int | None = None,
                 x_offset: int = 0):
        e = "fk_fp8_quantize"
        wide = element(e, x_type)
        x_stride = row_stride(e, "x_stride", x_stride, to.k)
        codes, scales = to._held(e, "the matrix", device)
        at = need(e, "x", x, ((to.rows - 1) * x_stride + to.k) * wide, device, x_offset * wide)
        args = QuantizeArgs(at, codes, scales, x_stride, to.rows, to.k, TYPES[x_type])
        admit(e, args)
        super().__init__(device, e, args, (x, to))


class Dequantize(runtime.Operation):
    """The values of a matrix into y [rows][k] of `y_type`, each rounded once,
    and with `scales` (f32 [rows][ceil(k / 128)]) its scales
    (fk_fp8_dequantize)."""

    def __init__(self, device, held: Fp8Matrix, y: runtime.Buffer, y_type: str = "f32", y_stride: int | None = None,
                 scales: runtime.Buffer | None = None):
        e = "fk_fp8_dequantize"
        wide = element(e, y_type)
        y_stride = row_stride(e, "y_stride", y_stride, held.k)
        codes, from_scales = held._held(e, "the matrix", device)
        at = need(e, "y", y, ((held.rows - 1) * y_stride + held.k) * wide, device)
        out = 0 if scales is None else need(e, "scales", scales, 4 * held.rows * -(-held.k // 128), device)
        args = DequantizeArgs(codes, from_scales, at, out, y_stride, held.rows, held.k, TYPES[y_type])
        admit(e, args)
        super().__init__(device, e, args, (held, y, scales))


class AddNorm(runtime.Operation):
    """h = x + residual, rounded to `x_type` and kept in `sum` (which may be the
    residual's buffer or x's); h / sqrt(mean h² + eps) · gamma (f32 [k]) to `to`
    (fk_fp8_add_norm).  Without `residual` h is x, without `sum` it is not
    kept, without `gamma` its elements are 1."""

    def __init__(self, device, x: runtime.Buffer, to: Fp8Matrix, eps: float, gamma: runtime.Buffer | None = None,
                 residual: runtime.Buffer | None = None, sum: runtime.Buffer | None = None, x_type: str = "f32",
                 x_stride: int | None = None, residual_stride: int | None = None, sum_stride: int | None = None,
                 x_offset: int = 0):
        e = "fk_fp8_add_norm"
        wide = element(e, x_type)
        codes, scales = to._held(e, "the matrix", device)
        at, strides = {}, {}
        for name, buf, stride, offset in (("x", x, x_stride, x_offset), ("residual", residual, residual_stride, 0),
                                          ("sum", sum, sum_stride, 0)):
            strides[f"{name}_stride"] = s = row_stride(e, f"{name}_stride", stride, to.k)
            at[name] = 0 if buf is None else need(e, name, buf, ((to.rows - 1) * s + to.k) * wide, device,
                                                  offset * wide)
        at["gamma"] = 0 if gamma is None else need(e, "gamma", gamma, 4 * to.k, device)
        args = AddNormArgs(**at, codes=codes, scales=scales, **strides, rows=to.rows, k=to.k, x_type=TYPES[x_type],
                           eps=eps)
        admit(e, args)
        super().__init__(device, e, args, (x, residual, sum, gamma, to))


CUT_SUMS = 0x100   # FK_FP8_CUT_SUMS


def _c_type(entry: str, c_type: str, cut_sums: bool) -> tuple[int, int]:
    """C's type as the call has it, and its elements' bytes."""
    wide = element(entry, c_type, ("f16", "bf16") if cut_sums else ("f32", "f16", "bf16"))
    return TYPES[c_type] | (CUT_SUMS if cut_sums else 0), wide


def gemm_form(m: int, n: int, k: int, c_type: str = "f32", cut_sums: bool = False) -> str:
    """The kernel that a Gemm of these sizes takes (fk_fp8_gemm_form)."""
    whole("fk_fp8_gemm", m=m, n=n, k=k)
    return runtime.library().fk_fp8_gemm_form(m, n, k, _c_type("fk_fp8_gemm", c_type, cut_sums)[0]).decode()


class Gemm(runtime.Operation):
    """C [m][n] = A Bᵀ of A [m, k] and B [n, k] (a weight, outputs first), in
    rows of `c_type` `c_stride` elements apart (fk_fp8_gemm).  Sums are
    binary32's; with `cut_sums` those of C of f16 or bf16 are the matrix cores'
    8-bit operations' own, off by up to 7 2^-14 of Σ |a b|, at up to twice the
    rate (FK_FP8_CUT_SUMS)."""

    def __init__(self, device, a: Fp8Matrix, b: Fp8Matrix, c: runtime.Buffer, c_type: str = "f32",
                 c_stride: int | None = None, cut_sums: bool = False):
        e = "fk_fp8_gemm"
        kind, wide = _c_type(e, c_type, cut_sums)
        if a.k != b.k:
            raise LaunchError(f"{e}: rows of {a.k} and of {b.k}")
        c_stride = row_stride(e, "c_stride", c_stride, b.rows)
        at = need(e, "c", c, ((a.rows - 1) * c_stride + b.rows) * wide, device)
        args = GemmArgs(*a._held(e, "A", device), *b._held(e, "B", device), at, c_stride, a.rows, b.rows, a.k, kind)
        admit(e, args)
        super().__init__(device, e, args, (a, b, c))
