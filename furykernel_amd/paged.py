"""The operators of a served batch over paged KV caches
(include/fkrocm_serve.h): what a step of requests that come and go, each with
its own length, does beside its model's launches.

* ``PagePlan`` — block tables and slot maps from the requests' lengths.
* ``PagedStore`` — q, k, v rows: RoPE, k and v into the pools at their slots.
* ``PagedAttend`` — attention of one new token a request over its pages.

Each is bound to its buffers once, which checks that they hold what the
kernels touch, and queued by ``enqueue(stream)`` (one C call; it may be
captured into a graph).  Pools are [blocks][kv_heads][block_size][head_dim] of
f16 or bf16 (src/FuryKernel/Program/Graph.hs:144-152).
"""

from __future__ import annotations

import ctypes

from . import runtime
from .kernels import LaunchError

# FK_T_* and the bytes of an element.
TYPES = {"f32": 0, "f16": 1, "bf16": 2}
ELEM_BYTES = {"f32": 4, "f16": 2, "bf16": 2}
NO_SLOT = 0xFFFFFFFF
_U32, _U64 = ctypes.c_uint32, ctypes.c_uint64


def need(entry: str, name: str, buf: runtime.Buffer, nbytes: int, device: runtime.Device, offset: int = 0) -> int:
    """The address `offset` bytes into a buffer of `device` that holds
    `nbytes` from there on."""
    if buf.device is not device:
        raise LaunchError(f"{entry}: {name} is another device's buffer")
    if offset < 0 or buf.size < offset + nbytes:
        raise LaunchError(f"{entry}: {name} holds {buf.size - offset} bytes, the launch reads or writes {nbytes}")
    return buf.ptr + offset


def whole(entry: str, **values: int) -> None:
    """Each a whole number that its 32-bit field holds."""
    for name, v in values.items():
        if not 0 <= v < 1 << 32:
            raise LaunchError(f"{entry}: {name} = {v} is not a 32-bit count")


def element(entry: str, name: str, types=("f32", "f16", "bf16")) -> int:
    if name not in types:
        raise LaunchError(f"{entry}: type {name!r} is none of {', '.join(types)}")
    return ELEM_BYTES[name]


def row_stride(entry: str, name: str, stride: int | None, width: int) -> int:
    """Elements from row to row: the width, or what holds a row."""
    stride = width if stride is None else stride
    if not width <= stride < 1 << 40:
        raise LaunchError(f"{entry}: {name} = {stride} of rows of {width}")
    return stride


def admit(entry: str, args: ctypes.Structure) -> None:
    """The library's own checks of a call's arguments (fk_serve_check)."""
    try:
        runtime.serve_check(entry, args)
    except runtime.FkError as err:
        raise LaunchError(err.message) from None


class PagePlanArgs(ctypes.Structure):
    """fk_page_plan_args."""
    _fields_ = [(f, _U64) for f in ("cached", "fresh", "free_blocks", "head", "table", "lengths", "starts", "slots",
                                    "positions", "owner", "counts")] + \
        [(f, _U32) for f in ("requests", "tokens", "table_len", "block_size", "free_len")]


class PagedStoreArgs(ctypes.Structure):
    """fk_paged_store_args."""
    _fields_ = [(f, _U64) for f in ("q", "k", "v", "slots", "positions", "rope", "qr", "kpool", "vpool", "q_stride",
                                    "k_stride", "v_stride")] + \
        [(f, _U32) for f in ("tokens", "heads", "kv_heads", "head_dim", "block_size", "blocks", "rotated",
                             "rope_rows", "rows_type", "cache_bf16")]


class PagedAttendArgs(ctypes.Structure):
    """fk_paged_attend_args."""
    _fields_ = [(f, _U64) for f in ("q", "kpool", "vpool", "table", "lengths", "starts", "out", "workspace",
                                    "workspace_bytes",
                                    "q_stride", "out_stride")] + \
        [(f, _U32) for f in ("requests", "heads", "kv_heads", "head_dim", "block_size", "blocks", "table_len",
                             "window", "q_rows", "cache_bf16", "out_f32")] + [("scale", ctypes.c_float)]


class PagePlan(runtime.Operation):
    """The block tables and slot maps of a step (fk_page_plan): requests of
    cached[r] positions that bring fresh[r] tokens each (u32), `tokens` the
    step's fixed count, padding included.  Blocks that requests need come
    from `free` (u32 [free_len]), from entry head[0] on, in the order of the
    requests, and go into their rows of `table` (u32 [requests][table_len]).

    Out: lengths [requests] = cached + fresh, starts [requests + 1], and for
    each token its slot (block · block_size + place), position and request
    (`owner`); behind the last token NO_SLOT, 0 and NO_SLOT.  counts [4]:
    tokens, blocks taken, requests that do not fit (their tokens have no
    slot, their length stays), the next step's head (a graph that steps by
    itself copies it to `head`)."""

    def __init__(self, device, cached, fresh, free, head, table, lengths, starts, slots, positions, owner, counts,
                 requests: int, tokens: int, table_len: int, block_size: int, free_len: int):
        e = "fk_page_plan"
        whole(e, requests=requests, tokens=tokens, table_len=table_len, block_size=block_size, free_len=free_len)
        bufs = {"cached": (cached, requests), "fresh": (fresh, requests), "free_blocks": (free, free_len),
                "head": (head, 1), "table": (table, requests * table_len), "lengths": (lengths, requests),
                "starts": (starts, requests + 1), "slots": (slots, tokens), "positions": (positions, tokens),
                "owner": (owner, tokens), "counts": (counts, 4)}
        at = {name: need(e, name, buf, 4 * count, device) for name, (buf, count) in bufs.items()}
        args = PagePlanArgs(**at, requests=requests, tokens=tokens, table_len=table_len, block_size=block_size,
                            free_len=free_len)
        admit(e, args)
        super().__init__(device, e, args, tuple(buf for buf, _ in bufs.values()))


class PagedStore(runtime.Operation):
    """A step's rows into the caches (fk_paged_store): for each token with a
    slot of the pools, q and k turned by RoPE at positions[t] (`rotated`
    pairs of NeoX halves; 0: none), q rounded into `qr` [tokens][heads]
    [head_dim] of the caches' type, k and v into the pools.  Without q only k
    and v are stored.

    q, k and v are rows of `rows_type`, `*_stride` elements apart and
    `*_offset` elements into their buffers (a fused product's rows): both
    multiples of 16 bytes."""

    def __init__(self, device, k, v, slots, kpool, vpool, tokens: int, kv_heads: int, head_dim: int, block_size: int,
                 blocks: int, q=None, qr=None, heads: int = 0, positions=None, rope=None, rope_rows: int = 0,
                 rotated: int = 0, rows_type: str = "f32", cache: str = "f16", q_stride: int | None = None,
                 k_stride: int | None = None, v_stride: int | None = None, q_offset: int = 0, k_offset: int = 0,
                 v_offset: int = 0):
        e = "fk_paged_store"
        whole(e, tokens=tokens, heads=heads, kv_heads=kv_heads, head_dim=head_dim, block_size=block_size,
              blocks=blocks, rope_rows=rope_rows, rotated=rotated)
        wide = element(e, rows_type)
        element(e, cache, ("f16", "bf16"))
        if (q is None) != (qr is None) or (q is not None and heads == 0):
            raise LaunchError(f"{e}: q, its heads and qr go together")
        if rotated and (positions is None or rope is None):
            raise LaunchError(f"{e}: RoPE needs positions and the table")
        qw, kw = heads * head_dim, kv_heads * head_dim
        strides = {"q": qw if q_stride is None else q_stride, "k": kw if k_stride is None else k_stride,
                   "v": kw if v_stride is None else v_stride}
        at = {}
        for name, buf, width, offset in (("q", q, qw, q_offset), ("k", k, kw, k_offset), ("v", v, kw, v_offset)):
            if not 0 <= strides[name] < 1 << 40:
                raise LaunchError(f"{e}: {name}_stride = {strides[name]}")
            rows = (tokens - 1) * strides[name] + width if tokens else 0
            at[name] = 0 if buf is None else need(e, name, buf, rows * wide, device, offset * wide)
        at["slots"] = need(e, "slots", slots, 4 * tokens, device)
        at["positions"] = need(e, "positions", positions, 4 * tokens, device) if rotated else 0
        at["rope"] = need(e, "rope", rope, 8 * rope_rows * rotated, device) if rotated else 0
        at["qr"] = 0 if q is None else need(e, "qr", qr, tokens * qw * 2, device)
        pool = blocks * block_size * kw * 2
        at["kpool"], at["vpool"] = need(e, "kpool", kpool, pool, device), need(e, "vpool", vpool, pool, device)
        args = PagedStoreArgs(**at, **{f"{n}_stride": s for n, s in strides.items()}, tokens=tokens, heads=heads,
                              kv_heads=kv_heads, head_dim=head_dim, block_size=block_size, blocks=blocks,
                              rotated=rotated, rope_rows=rope_rows, rows_type=TYPES[rows_type],
                              cache_bf16=int(cache == "bf16"))
        admit(e, args)
        super().__init__(device, e, args, (q, k, v, slots, positions, rope, qr, kpool, vpool))


def attend_workspace(requests: int, heads: int, kv_heads: int, head_dim: int, block_size: int, blocks: int,
                     table_len: int, window: int = 0) -> int:
    """The bytes of a PagedAttend's workspace (fk_paged_attend_workspace)."""
    sizes = dict(requests=requests, heads=heads, kv_heads=kv_heads, head_dim=head_dim, block_size=block_size,
                 blocks=blocks, table_len=table_len, window=window)
    whole("fk_paged_attend", **sizes)
    args = PagedAttendArgs(**sizes)
    n = int(runtime.library().fk_paged_attend_workspace(ctypes.byref(args)))
    if n == 0:
        raise LaunchError(f"fk_paged_attend: it does not take {sizes}")
    return n


def attend_form(**sizes: int) -> str:
    """How a PagedAttend of ``attend_workspace``'s sizes is shared out
    (fk_paged_attend_form)."""
    attend_workspace(**sizes)
    return runtime.library().fk_paged_attend_form(ctypes.byref(PagedAttendArgs(**sizes))).decode()


class PagedAttend(runtime.Operation):
    """Attention of one new token a request over its pages (fk_paged_attend):
    out[r] = softmax(scale q[r] Kᵀ) V over positions 0 .. lengths[r] - 1 (with
    a `window` the last of them), q and out rows [heads][head_dim], `*_stride`
    elements apart; out of the caches' type, or f32.  With a plan's `starts`
    q has `q_rows` rows, a step's tokens: request r's is that of its last new
    token, and a request without one counts as empty.  A length of 0 gives
    zeros.  `workspace` holds ``attend_workspace`` bytes; two calls that may
    run at once take one each."""

    def __init__(self, device, q, kpool, vpool, table, lengths, out, workspace, requests: int, heads: int,
                 kv_heads: int, head_dim: int, block_size: int, blocks: int, table_len: int, scale: float,
                 window: int = 0, cache: str = "f16", out_type: str | None = None, q_stride: int | None = None,
                 out_stride: int | None = None, starts=None, q_rows: int = 0):
        e = "fk_paged_attend"
        whole(e, q_rows=q_rows)
        element(e, cache, ("f16", "bf16"))
        wide = element(e, cache if out_type is None else out_type, (cache, "f32"))
        sizes = dict(requests=requests, heads=heads, kv_heads=kv_heads, head_dim=head_dim, block_size=block_size,
                     blocks=blocks, table_len=table_len, window=window)
        nbytes = attend_workspace(**sizes)
        w = heads * head_dim
        q_stride, out_stride = (w if s is None else s for s in (q_stride, out_stride))
        if not (w <= q_stride < 1 << 40 and w <= out_stride < 1 << 40):
            raise LaunchError(f"{e}: row strides {q_stride} and {out_stride} of rows of {w}")
        pool = blocks * block_size * kv_heads * head_dim * 2
        rows = requests if starts is None else q_rows
        at = {"q": need(e, "q", q, (max(rows - 1, 0) * q_stride + w) * 2, device),
              "starts": 0 if starts is None else need(e, "starts", starts, 4 * (requests + 1), device),
              "kpool": need(e, "kpool", kpool, pool, device), "vpool": need(e, "vpool", vpool, pool, device),
              "table": need(e, "table", table, 4 * requests * table_len, device),
              "lengths": need(e, "lengths", lengths, 4 * requests, device),
              "out": need(e, "out", out, ((requests - 1) * out_stride + w) * wide, device),
              "workspace": need(e, "workspace", workspace, nbytes, device)}
        args = PagedAttendArgs(**at, workspace_bytes=workspace.size, q_stride=q_stride, out_stride=out_stride, **sizes,
                               cache_bf16=int(cache == "bf16"), out_f32=int(out_type == "f32"), scale=scale,
                               q_rows=0 if starts is None else q_rows)
        admit(e, args)
        super().__init__(device, e, args, (q, kpool, vpool, table, lengths, starts, out, workspace))
