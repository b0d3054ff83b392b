"""The operators of a served batch (include/fkrocm_serve.h) as their
definitions say, in whole numbers and binary64 on the host: what
tests/test_serve.py and tests/test_gpu_serve.py hold the kernels to."""

import numpy as np

NO_SLOT = 0xFFFFFFFF


def plan(cached, fresh, free, head, table, tokens, block):
    """fk_page_plan a request at a time: (its outputs by name, u32)."""
    n = len(cached)
    table = np.array(table, np.int64)
    lengths, starts = np.array(cached, np.int64), np.zeros(n + 1, np.int64)
    slots, owner = np.full(tokens, NO_SLOT, np.int64), np.full(tokens, NO_SLOT, np.int64)
    positions = np.zeros(tokens, np.int64)
    at = wanted = taken = refused = 0
    for r in range(n):
        c, f = int(cached[r]), int(fresh[r])
        held, pages = -(-c // block), -(-(c + f) // block)
        ok = pages <= table.shape[1] and c + f <= table.shape[1] * block and at + f <= tokens
        if ok and pages > held:
            wanted += pages - held
            ok = wanted <= max(0, len(free) - head)
            if ok:
                table[r, held:pages] = np.asarray(free)[head + wanted - (pages - held):head + wanted]
                taken = wanted
        live = range(at, min(at + f, tokens))
        for t in live:
            p = c + t - at
            owner[t], positions[t] = r, p & NO_SLOT
            if ok:
                slots[t] = min(table[r, p // block] * block + p % block, NO_SLOT)
        if ok:
            lengths[r] = c + f
        refused += not ok
        at += f
        starts[r + 1] = at
    counts = [min(at, NO_SLOT), taken, refused, head + taken]
    out = {"table": table, "lengths": lengths, "starts": np.minimum(starts, NO_SLOT), "slots": slots,
           "positions": positions, "owner": owner, "counts": counts}
    return {k: np.asarray(v, np.int64).astype(np.uint32) for k, v in out.items()}


def attend(q, k, v, table, lengths, block, scale, window=0):
    """fk_paged_attend in binary64: q [n, heads, d], pools [blocks, kv heads,
    block, d].  Also, for the error's bound, Σ p |v| of each element and each
    head's Σ |q k| at its largest (in score units)."""
    n, heads, d = q.shape
    kv = k.shape[1]
    out, spread = np.zeros((n, heads, d)), np.zeros((n, heads, d))
    reach = np.zeros((n, heads, 1))
    for r in range(n):
        length = min(int(lengths[r]), table.shape[1] * block)
        first = max(0, length - window) if window else 0
        if length == 0:
            continue
        at = np.arange(first, length)
        page = np.minimum(table[r, at // block].astype(np.int64), k.shape[0] - 1)
        for h in range(heads):
            g = h // (heads // kv)
            kk, vv = k[page, g, at % block].astype(np.float64), v[page, g, at % block].astype(np.float64)
            qq = q[r, h].astype(np.float64)
            s = kk @ qq * scale
            e = np.exp(s - s.max())
            e /= e.sum()
            out[r, h], spread[r, h] = e @ vv, e @ np.abs(vv)
            reach[r, h] = (np.abs(kk) @ np.abs(qq)).max() * abs(scale)
    return out, spread, reach


def attend_tolerance(out, spread, reach, lengths, d, half_step):
    """How far a row may be from binary64's.  A score's error: d + 1 binary32
    operations on terms whose sizes add to `reach`, the scale and the change
    to log2 units (3 roundings of at most reach): (d + 4) 2^-24 reach; the
    exponential's: 2 ulp of its value (2^-23 each way).  The probability's two
    16-bit parts: cut off, bf16 leaves up to 2^-7 of p, whose rounding is off by
    2^-9 of that, 2^-16 (f16 2^-10 and 2^-12, and half its smallest step at
    2^-40 of the largest: less).  Sums: one rounding
    a tile and key, at most the keys of one quarter of a threadgroup's run and
    64 joins, n / 4 + 64 of 2^-24, twice (the values' and the sum's).  All of
    them relative to Σ p |v|, and the result's rounding to its own type."""
    n = np.asarray(lengths, np.float64)[:, None, None]
    rel = 2 * ((d + 4) * 2.0 ** -24 * reach + 2.0 ** -22) + 2.0 ** -16 + 2 * (n / 4 + 64) * 2.0 ** -24
    return half_step * np.abs(out) + rel * spread * (1 + half_step) + 2.0 ** -25


def rope(x, cs, rotated):
    """NeoX halves: x [tokens, heads, d] by cs [tokens, rotated, 2], in binary64."""
    x = x.astype(np.float64)
    half = x.shape[-1] // 2
    a, b = x[..., :rotated].copy(), x[..., half:half + rotated].copy()
    c, s = (cs[:, None, :, i].astype(np.float64) for i in (0, 1))
    x[..., :rotated], x[..., half:half + rotated] = a * c - b * s, b * c + a * s
    return x


def widen(bits, bf16):
    """16-bit elements' values, binary64."""
    if bf16:
        return (bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return bits.view(np.float16).astype(np.float64)


def narrow(x, bf16):
    """binary32 values to 16 bits, to nearest even."""
    x = np.ascontiguousarray(x, np.float32)
    if not bf16:
        return x.astype(np.float16).view(np.uint16)
    w = x.view(np.uint32)
    return ((w + 0x7FFF + ((w >> 16) & 1)) >> 16).astype(np.uint16)


def half_step(kind):
    """Half a step of a type relative to the value."""
    return {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[kind]
