"""4-bit microscaled matrices (include/fkrocm_mx4.h, the OCP MX format MXFP4):
a model's weights at 4.25 bits an element, its activations brought to the
same form as they come, their products on the matrix cores.

* ``Mx4Matrix`` — a matrix's codes and scales in device memory.
* ``Quantize``, ``Dequantize`` — rows of f32, f16 or bf16 to it and back.
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
    """fk_mx4_quantize_args."""
    _fields_ = [(f, _U64) for f in ("x", "codes", "scales", "x_stride")] + \
        [(f, _U32) for f in ("rows", "k", "x_type")]


class DequantizeArgs(ctypes.Structure):
    """fk_mx4_dequantize_args."""
    _fields_ = [(f, _U64) for f in ("codes", "scales", "y", "scales_out", "y_stride")] + \
        [(f, _U32) for f in ("rows", "k", "y_type")]


class GemmArgs(ctypes.Structure):
    """fk_mx4_gemm_args."""
    _fields_ = [(f, _U64) for f in ("a_codes", "a_scales", "b_codes", "b_scales", "c", "c_stride")] + \
        [(f, _U32) for f in ("m", "n", "k", "c_type")]


class Mx4Matrix:
    """[rows, k] at 4 bits: its codes and scales, of which ``Quantize`` writes
    every byte (padding included) and nothing before holds anything."""

    def __init__(self, device: runtime.Device, rows: int, k: int):
        whole("Mx4Matrix", rows=rows, k=k)
        lib = runtime.library()
        sizes = lib.fk_mx4_codes_bytes(rows, k), lib.fk_mx4_scales_bytes(rows, k)
        if not all(sizes):
            raise LaunchError(f"Mx4Matrix: no matrix of {rows} rows of {k}")
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
        return (need(entry, f"{name}'s codes", self.codes, lib.fk_mx4_codes_bytes(self.rows, self.k), device),
                need(entry, f"{name}'s scales", self.scales, lib.fk_mx4_scales_bytes(self.rows, self.k), device))


class Quantize(runtime.Operation):
    """Rows x [rows][k] of `x_type`, `x_stride` elements apart and `x_offset`
    elements into their buffer, to `to` (fk_mx4_quantize)."""

    def __init__(self, device, x: runtime.Buffer, to: Mx4Matrix, x_type: str = "f32", x_stride: int | None = None,
                 x_offset: int = 0):
        e = "fk_mx4_quantize"
        wide = element(e, x_type)
        x_stride = row_stride(e, "x_stride", x_stride, to.k)
        codes, scales = to._held(e, "the matrix", device)
        at = need(e, "x", x, ((to.rows - 1) * x_stride + to.k) * wide, device, x_offset * wide)
        args = QuantizeArgs(at, codes, scales, x_stride, to.rows, to.k, TYPES[x_type])
        admit(e, args)
        super().__init__(device, e, args, (x, to))


class Dequantize(runtime.Operation):
    """The values of a matrix into y [rows][k] of `y_type`, each rounded once,
    and with `scales` (f32 [rows][ceil(k / 32)]) its scales
    (fk_mx4_dequantize)."""

    def __init__(self, device, held: Mx4Matrix, y: runtime.Buffer, y_type: str = "f32", y_stride: int | None = None,
                 scales: runtime.Buffer | None = None):
        e = "fk_mx4_dequantize"
        wide = element(e, y_type)
        y_stride = row_stride(e, "y_stride", y_stride, held.k)
        codes, from_scales = held._held(e, "the matrix", device)
        at = need(e, "y", y, ((held.rows - 1) * y_stride + held.k) * wide, device)
        out = 0 if scales is None else need(e, "scales", scales, 4 * held.rows * -(-held.k // 32), device)
        args = DequantizeArgs(codes, from_scales, at, out, y_stride, held.rows, held.k, TYPES[y_type])
        admit(e, args)
        super().__init__(device, e, args, (held, y, scales))


class Gemm(runtime.Operation):
    """C [m][n] = A Bᵀ of A [m, k] and B [n, k] (a weight, outputs first), in
    rows of `c_type` `c_stride` elements apart (fk_mx4_gemm)."""

    def __init__(self, device, a: Mx4Matrix, b: Mx4Matrix, c: runtime.Buffer, c_type: str = "f32",
                 c_stride: int | None = None):
        e = "fk_mx4_gemm"
        wide = element(e, c_type)
        if a.k != b.k:
            raise LaunchError(f"{e}: rows of {a.k} and of {b.k}")
        c_stride = row_stride(e, "c_stride", c_stride, b.rows)
        at = need(e, "c", c, ((a.rows - 1) * c_stride + b.rows) * wide, device)
        args = GemmArgs(*a._held(e, "A", device), *b._held(e, "B", device), at, c_stride, a.rows, b.rows, a.k,
                        TYPES[c_type])
        admit(e, args)
        super().__init__(device, e, args, (a, b, c))
