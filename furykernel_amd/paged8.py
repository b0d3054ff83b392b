"""The operators over paged KV caches held in 8 bits (include/
fkrocm_paged8.h), the counterparts of ``paged``'s for the same ``PagePlan``.

* ``PagedStore8`` — q, k, v rows: RoPE, k and v in 8 bits into the pools.
* ``PagedLoad8`` — cached positions as rows.
* ``PagedAttend8`` — attention of one new token a request over its pages.

Pools are [blocks][kv_heads][block_size][head_dim] of e4m3; `scales` is f32
[blocks][kv_heads][2], a block and head's scale of its keys and of its values
(powers of two).  Heads are of a multiple of 16, at most 256; blocks of a
multiple of 8.  Each operation is bound to its buffers once and queued by
``enqueue(stream)``.
"""

from __future__ import annotations

import ctypes

from . import runtime
from .kernels import LaunchError
from .paged import _U32, _U64, TYPES, admit, element, need, row_stride, whole


class PagedStore8Args(ctypes.Structure):
    """fk_paged_store8_args."""
    _fields_ = [(f, _U64) for f in ("q", "k", "v", "slots", "positions", "rope", "qr", "kpool", "vpool", "scales",
                                    "q_stride", "k_stride", "v_stride")] + \
        [(f, _U32) for f in ("tokens", "heads", "kv_heads", "head_dim", "block_size", "blocks", "rotated",
                             "rope_rows", "rows_type", "q_bf16")]


class PagedLoad8Args(ctypes.Structure):
    """fk_paged_load8_args."""
    _fields_ = [(f, _U64) for f in ("slots", "kpool", "vpool", "scales", "k", "v", "k_stride", "v_stride")] + \
        [(f, _U32) for f in ("tokens", "kv_heads", "head_dim", "block_size", "blocks", "rows_type")]


class PagedAttend8Args(ctypes.Structure):
    """fk_paged_attend8_args."""
    _fields_ = [(f, _U64) for f in ("q", "kpool", "vpool", "scales", "table", "lengths", "starts", "out", "workspace",
                                    "workspace_bytes", "q_stride", "out_stride")] + \
        [(f, _U32) for f in ("requests", "heads", "kv_heads", "head_dim", "block_size", "blocks", "table_len",
                             "window", "q_rows", "q_bf16", "out_f32")] + [("scale", ctypes.c_float)]


def _pools(e: str, device, kpool, vpool, scales, kv_heads: int, head_dim: int, block_size: int, blocks: int) -> dict:
    pool = blocks * block_size * kv_heads * head_dim
    return {"kpool": need(e, "kpool", kpool, pool, device), "vpool": need(e, "vpool", vpool, pool, device),
            "scales": need(e, "scales", scales, 8 * blocks * kv_heads, device)}


class PagedStore8(runtime.Operation):
    """A step's rows into 8-bit caches (fk_paged_store8): for each token with a
    slot of the pools, q and k turned by RoPE at positions[t] (`rotated` pairs
    of NeoX halves; 0: none), q rounded into `qr` [tokens][heads][head_dim] of
    `q_type`, k and v to 8 bits.  The tokens of a block follow one another in
    the order of their places, as a plan's do.  A block whose place 0 is written
    begins anew; another keeps its scale or takes a larger one, to which the
    rows it holds before the new ones are then brought.  Without q only k and v
    are stored.

    q, k and v are rows of `rows_type`, `*_stride` elements apart and
    `*_offset` elements into their buffers: both multiples of 16 bytes."""

    def __init__(self, device, k, v, slots, kpool, vpool, scales, tokens: int, kv_heads: int, head_dim: int,
                 block_size: int, blocks: int, q=None, qr=None, heads: int = 0, positions=None, rope=None,
                 rope_rows: int = 0, rotated: int = 0, rows_type: str = "f32", q_type: str = "f16",
                 q_stride: int | None = None, k_stride: int | None = None, v_stride: int | None = None,
                 q_offset: int = 0, k_offset: int = 0, v_offset: int = 0):
        e = "fk_paged_store8"
        whole(e, tokens=tokens, heads=heads, kv_heads=kv_heads, head_dim=head_dim, block_size=block_size,
              blocks=blocks, rope_rows=rope_rows, rotated=rotated)
        wide = element(e, rows_type)
        element(e, q_type, ("f16", "bf16"))
        if (q is None) != (qr is None) or (q is not None and heads == 0):
            raise LaunchError(f"{e}: q, its heads and qr go together")
        if rotated and (positions is None or rope is None):
            raise LaunchError(f"{e}: RoPE needs positions and the table")
        qw, kw = heads * head_dim, kv_heads * head_dim
        at, strides = {}, {}
        for name, buf, width, stride, offset in (("q", q, qw, q_stride, q_offset), ("k", k, kw, k_stride, k_offset),
                                                 ("v", v, kw, v_stride, v_offset)):
            strides[f"{name}_stride"] = s = row_stride(e, f"{name}_stride", stride, width)
            rows = (tokens - 1) * s + width if tokens else 0
            at[name] = 0 if buf is None else need(e, name, buf, rows * wide, device, offset * wide)
        at["slots"] = need(e, "slots", slots, 4 * tokens, device)
        at["positions"] = need(e, "positions", positions, 4 * tokens, device) if rotated else 0
        at["rope"] = need(e, "rope", rope, 8 * rope_rows * rotated, device) if rotated else 0
        at["qr"] = 0 if q is None else need(e, "qr", qr, tokens * qw * 2, device)
        at |= _pools(e, device, kpool, vpool, scales, kv_heads, head_dim, block_size, blocks)
        args = PagedStore8Args(**at, **strides, tokens=tokens, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                               block_size=block_size, blocks=blocks, rotated=rotated, rope_rows=rope_rows,
                               rows_type=TYPES[rows_type], q_bf16=int(q_type == "bf16"))
        admit(e, args)
        super().__init__(device, e, args, (q, k, v, slots, positions, rope, qr, kpool, vpool, scales))


class PagedLoad8(runtime.Operation):
    """Cached positions as rows (fk_paged_load8): for each t with a slot of the
    pools, its keys and values into row t of `k` and `v`, [kv_heads][head_dim]
    of `rows_type`, `*_stride` elements apart (a multiple of 16 bytes), each
    rounded once.  Rows without a slot stay as they were."""

    def __init__(self, device, slots, kpool, vpool, scales, k, v, tokens: int, kv_heads: int, head_dim: int,
                 block_size: int, blocks: int, rows_type: str = "f16", k_stride: int | None = None,
                 v_stride: int | None = None):
        e = "fk_paged_load8"
        whole(e, tokens=tokens, kv_heads=kv_heads, head_dim=head_dim, block_size=block_size, blocks=blocks)
        wide, w = element(e, rows_type), kv_heads * head_dim
        at, strides = {"slots": need(e, "slots", slots, 4 * tokens, device)}, {}
        for name, buf, stride in (("k", k, k_stride), ("v", v, v_stride)):
            strides[f"{name}_stride"] = s = row_stride(e, f"{name}_stride", stride, w)
            at[name] = need(e, name, buf, ((tokens - 1) * s + w) * wide if tokens else 0, device)
        at |= _pools(e, device, kpool, vpool, scales, kv_heads, head_dim, block_size, blocks)
        args = PagedLoad8Args(**at, **strides, tokens=tokens, kv_heads=kv_heads, head_dim=head_dim,
                              block_size=block_size, blocks=blocks, rows_type=TYPES[rows_type])
        admit(e, args)
        super().__init__(device, e, args, (slots, kpool, vpool, scales, k, v))


def attend8_workspace(requests: int, heads: int, kv_heads: int, head_dim: int, block_size: int, blocks: int,
                      table_len: int, window: int = 0) -> int:
    """The bytes of a PagedAttend8's workspace (fk_paged_attend8_workspace)."""
    sizes = dict(requests=requests, heads=heads, kv_heads=kv_heads, head_dim=head_dim, block_size=block_size,
                 blocks=blocks, table_len=table_len, window=window)
    whole("fk_paged_attend8", **sizes)
    n = int(runtime.library().fk_paged_attend8_workspace(ctypes.byref(PagedAttend8Args(**sizes))))
    if n == 0:
        raise LaunchError(f"fk_paged_attend8: it does not take {sizes}")
    return n


def attend8_form(**sizes: int) -> str:
    """How a PagedAttend8 of ``attend8_workspace``'s sizes is shared out
    (fk_paged_attend8_form)."""
    attend8_workspace(**sizes)
    return runtime.library().fk_paged_attend8_form(ctypes.byref(PagedAttend8Args(**sizes))).decode()


class PagedAttend8(runtime.Operation):
    """Attention of one new token a request over 8-bit pages
    (fk_paged_attend8), as ``paged.PagedAttend``'s: out[r] = softmax(scale q[r]
    Kᵀ) V over positions 0 .. lengths[r] - 1 (with a `window` the last of
    them), q and out rows [heads][head_dim] of `q_type` (out also f32),
    `*_stride` elements apart.  With a plan's `starts` q has `q_rows` rows, a
    step's tokens: request r's is that of its last new token, and a request
    without one counts as empty.  A length of 0 gives zeros.  `workspace` holds
    ``attend8_workspace`` bytes; two calls that may run at once take one each."""

    def __init__(self, device, q, kpool, vpool, scales, table, lengths, out, workspace, requests: int, heads: int,
                 kv_heads: int, head_dim: int, block_size: int, blocks: int, table_len: int, scale: float,
                 window: int = 0, q_type: str = "f16", out_type: str | None = None, q_stride: int | None = None,
                 out_stride: int | None = None, starts=None, q_rows: int = 0):
        e = "fk_paged_attend8"
        whole(e, q_rows=q_rows)
        element(e, q_type, ("f16", "bf16"))
        wide = element(e, q_type if out_type is None else out_type, (q_type, "f32"))
        sizes = dict(requests=requests, heads=heads, kv_heads=kv_heads, head_dim=head_dim, block_size=block_size,
                     blocks=blocks, table_len=table_len, window=window)
        nbytes = attend8_workspace(**sizes)
        w = heads * head_dim
        q_stride, out_stride = (row_stride(e, n, s, w) for n, s in (("q_stride", q_stride), ("out_stride", out_stride)))
        rows = requests if starts is None else q_rows
        at = {"q": need(e, "q", q, (max(rows - 1, 0) * q_stride + w) * 2, device),
              "starts": 0 if starts is None else need(e, "starts", starts, 4 * (requests + 1), device),
              "table": need(e, "table", table, 4 * requests * table_len, device),
              "lengths": need(e, "lengths", lengths, 4 * requests, device),
              "out": need(e, "out", out, ((requests - 1) * out_stride + w) * wide, device),
              "workspace": need(e, "workspace", workspace, nbytes, device),
              **_pools(e, device, kpool, vpool, scales, kv_heads, head_dim, block_size, blocks)}
        args = PagedAttend8Args(**at, workspace_bytes=workspace.size, q_stride=q_stride, out_stride=out_stride,
                                **sizes, q_bf16=int(q_type == "bf16"), out_f32=int(out_type == "f32"), scale=scale,
                                q_rows=0 if starts is None else q_rows)
        admit(e, args)
        super().__init__(device, e, args, (q, kpool, vpool, scales, table, lengths, starts, out, workspace))
