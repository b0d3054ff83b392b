"""4-bit microscaled matrices (include/fkrocm_mx4.h) as the format says, in
binary64 on the host, and the order they are held in."""

import numpy as np

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def quantize(x):
    """x [rows, k] to (codes [rows, blocks, 32], scale bytes [rows, blocks]),
    k counted up to whole blocks."""
    x = np.asarray(x, np.float64)
    rows, k = x.shape
    x = np.pad(x, ((0, 0), (0, -k % 32))).reshape(rows, -1, 32)
    big = np.abs(x).max(-1)
    finite = np.isfinite(x).all(-1)
    exp = np.frexp(np.where(finite & (big > 0), big, 1.0))[1] - 1       # floor(log2 big)
    b = np.where(finite, np.where(big > 0, np.maximum(exp - 2, -127) + 127, 127), 255).astype(np.int64)
    y = np.where(finite[..., None], np.abs(x) / np.exp2(np.where(finite, b, 127) - 127.0)[..., None], 0.0)
    codes = np.zeros(y.shape, np.uint8)
    for i in range(7):
        mid = (GRID[i] + GRID[i + 1]) / 2
        codes += ((y > mid) if i % 2 == 0 else (y >= mid)).astype(np.uint8)
    codes |= (np.signbit(x) & finite[..., None]).astype(np.uint8) << 3
    return codes, b.astype(np.uint8)


def scale_of(b):
    return np.where(b == 255, np.nan, np.exp2(np.where(b == 255, 127, b) - 127.0))


def values(codes, b, k):
    """What they stand for, [rows, k]."""
    v = np.where(codes & 8, -1.0, 1.0) * GRID[codes & 7] * scale_of(b.astype(np.int64))[..., None]
    return v.reshape(v.shape[0], -1)[:, :k]


def pack(codes, b):
    """(codes' bytes, scales' bytes) in the order they are held in."""
    rows, blocks, _ = codes.shape
    rt, pairs = -(-rows // 16), -(-blocks // 8)
    c = np.zeros((rt * 16, pairs * 8, 32), np.uint8)
    s = np.full((rt * 16, pairs * 8), 127, np.uint8)
    c[:rows, :blocks], s[:rows, :blocks] = codes, b
    c = (c[..., ::2] | c[..., 1::2] << 4).reshape(rt, 16, pairs, 2, 4, 16).transpose(0, 2, 3, 4, 1, 5)
    s = s.reshape(rt, 16, pairs, 2, 4).transpose(0, 2, 4, 1, 3)
    return np.ascontiguousarray(c).ravel(), np.ascontiguousarray(s).ravel()
