"""8-bit values with scales that are powers of two (include/fkrocm_fp8.h,
fkrocm_paged8.h) as their definitions say, on the host: what the tests of the
8-bit operators hold the kernels to."""

import numpy as np

# The values of the codes 0 .. 126 (e4m3: 4 exponent bits of bias 7, 3 of mantissa), ascending.
MAGNITUDES = np.array([(m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7))
                       for e in range(16) for m in range(8)][:127])
VALUES = np.concatenate([MAGNITUDES, [np.nan], -MAGNITUDES, [np.nan]])   # by code
SMALLEST = 2.0 ** -126


def encode(y):
    """Codes of binary64 values over their scale: to the nearest, halfway cases
    to the even code, NaN where not finite."""
    y = np.asarray(y, np.float64)
    a = np.where(np.isfinite(y), np.abs(y), 0.0)
    step = np.exp2(np.maximum(np.frexp(a)[1] - 1, -6) - 3.0)
    code = np.searchsorted(MAGNITUDES, np.rint(a / step) * step).astype(np.uint8)
    return np.where(np.isfinite(y), code | (np.signbit(y).astype(np.uint8) << 7), np.uint8(0x7F)).astype(np.uint8)


def scale_of(big):
    """The smallest power of two, from 2^-126 on, that keeps `big` (binary64,
    finite) within 448."""
    big = np.asarray(big, np.float64)
    m, e = np.frexp(big)                       # big = m 2^e, m in [1/2, 1); 448 = 7/8 2^9
    e = np.where(m > 0.875, e - 8, e - 9)
    return np.exp2(np.maximum(np.where(big > 0, e, -126), -126).astype(np.float64))


def largest(x, axis):
    x = np.abs(np.asarray(x, np.float64))
    return np.where(np.isfinite(x), x, 0.0).max(axis)


def blocks(x):
    """Rows by blocks of 128, zeros behind them."""
    x = np.asarray(x, np.float64)
    x = np.concatenate([x, np.zeros((x.shape[0], -x.shape[1] % 128))], 1)
    return x.reshape(x.shape[0], -1, 128)


def quantize(x):
    """(codes [rows, blocks, 128], scales [rows, blocks]) of rows."""
    b = blocks(x)
    scale = scale_of(largest(b, -1))
    return encode(b / scale[..., None]), scale


def values(codes, scale, k):
    return (VALUES[codes] * scale[..., None]).reshape(codes.shape[0], -1)[:, :k]


def pack(codes, scale):
    """(codes, scales) as an Fp8Matrix holds them, bytes."""
    rows, n = scale.shape
    pad = -rows % 16
    codes = np.concatenate([codes, np.zeros((pad, n, 128), np.uint8)])
    # rows by 16, elements by 64 by pieces of 16
    held = codes.reshape(-1, 16, 2 * n, 4, 16).transpose(0, 2, 3, 1, 4)
    b = np.full((rows + pad, n + -n % 4), 127, np.uint8)
    b[:rows, :n] = (np.log2(scale) + 127).astype(np.uint8)
    return held.reshape(-1).copy(), b.reshape(-1, 16, b.shape[1] // 4, 4).transpose(0, 2, 1, 3).reshape(-1).copy()


def unpack(codes, scales, rows, k):
    """pack's other way: (codes [rows, blocks, 128], scales [rows, blocks])."""
    n = -(-k // 128)
    c = codes.reshape(-1, 2 * n, 4, 16, 16).transpose(0, 3, 1, 2, 4).reshape(-1, n, 128)[:rows]
    b = scales.reshape(-1, -(-n // 4), 16, 4).transpose(0, 2, 1, 3).reshape(c.shape[0] + -rows % 16, -1)[:rows, :n]
    return c, np.exp2(b.astype(np.float64) - 127)


def same_codes(got, want):
    """Equal byte for byte, a NaN of either sign a NaN."""
    return (got == want) | (((got & 0x7F) == 0x7F) & ((want & 0x7F) == 0x7F))


def turn(x, cs, rotated):
    """NeoX halves of binary32 heads [tokens, heads, d] by cs [tokens, rotated,
    2], each operation rounded, as the kernels make them."""
    x = np.array(x, np.float32)
    if rotated == 0:
        return x
    half = x.shape[-1] // 2
    a, b = x[..., :rotated].copy(), x[..., half:half + rotated].copy()
    c, s = (cs[:, None, :, i].astype(np.float32) for i in (0, 1))
    x[..., :rotated], x[..., half:half + rotated] = a * c - b * s, b * c + a * s
    return x


def store(rows, slots, pool, scales, block):
    """fk_paged_store8 of one of k and v, a run at a time: rows [tokens, kv
    heads, d] (turned), pool [blocks, kv heads, block, d] of codes and scales
    [blocks, kv heads], both written."""
    places = pool.shape[0] * block
    t = 0
    while t < len(slots):
        if slots[t] >= places:
            t += 1
            continue
        b, n = int(slots[t]) // block, 1
        while t + n < len(slots) and slots[t + n] < places and int(slots[t + n]) // block == b:
            n += 1
        x = np.asarray(rows[t:t + n], np.float64)
        place = int(slots[t]) % block
        scale = scale_of(largest(x, (0, 2)))
        if place:
            scale = np.maximum(scale, scales[b])
            for h in np.flatnonzero(scale != scales[b]):
                pool[b, h, :place] = encode(VALUES[pool[b, h, :place]] * (scales[b, h] / scale[h]))
        scales[b] = scale
        for i in range(n):
            pool[b, :, int(slots[t + i]) % block] = encode(x[i] / scale[:, None])
        t += n


def norm(h, gamma, eps):
    """h / sqrt(mean h^2 + eps) gamma in binary64."""
    h = np.asarray(h, np.float64)
    y = h / np.sqrt((h * h).mean(1, keepdims=True) + eps)
    return y if gamma is None else y * np.asarray(gamma, np.float64)


def norm_relative(k):
    """How far a normed element may be from binary64's, relative to it: the sum
    of k squares, all positive, in any order of at most k / 8 + 16 additions a
    term goes through after its own rounding and square, halved by the square
    root; then the mean, eps, the root, the reciprocal and two products, 2^-24
    each."""
    return ((k / 8 + 18) / 2 + 6) * 2.0 ** -24
