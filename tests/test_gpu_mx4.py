"""4-bit microscaled matrices (include/fkrocm_mx4.h) on the GPU: the codes and
scales byte for byte, the values they stand for, and products: exact where
every partial sum fits binary32, elsewhere within the accumulation's bound."""

import numpy as np
import pytest

import mx4_cases as M
import serve_cases as S
from furykernel_amd import mx4, runtime
from test_gpu_serve import SENTINEL, Memory, mem  # noqa: F401  (mem is a fixture)

pytestmark = pytest.mark.gpu


def held(rows, kind):
    """(the elements' bytes, their values) of binary32 rows rounded to a type."""
    if kind == "f32":
        rows = np.ascontiguousarray(rows, np.float32)
        return rows, rows.astype(np.float64)
    bits = S.narrow(rows, kind == "bf16")
    return bits, S.widen(bits, kind == "bf16")


def matrix(device, mem, rows, k):
    m = mx4.Mx4Matrix(device, rows, k)
    mem.keep(m)
    for b in (m.codes, m.scales):
        b.write(np.full(b.size, 0x5A, np.uint8))
    return m


def put_matrix(device, mem, codes, b, k):
    m = matrix(device, mem, codes.shape[0], k)
    for buf, data in zip((m.codes, m.scales), M.pack(codes, b)):
        buf.write(data)
    return m


def hold_quantize(device, mem, rows, kind, stride=None, offset=0):
    n, k = rows.shape
    bits, x = held(rows, kind)
    stride = k if stride is None else stride
    fill, of = (0x7E7E7E7E, np.uint32) if kind == "f32" else (0x7E7E, np.uint16)
    src = np.full(offset + n * stride, fill, of)
    src[offset:].reshape(n, stride)[:, :k] = bits.view(src.dtype)
    m = matrix(device, mem, n, k)
    mx4.Quantize(device, mem.put(src), m, x_type=kind, x_stride=stride, x_offset=offset).enqueue()
    device.sync()
    codes, b = M.quantize(x)
    for buf, want, what in zip((m.codes, m.scales), M.pack(codes, b), ("codes", "scales")):
        got = buf.read(np.uint8)
        assert np.array_equal(got, want), (what, int((got != want).sum()), np.flatnonzero(got != want)[:8],
                                           got[got != want][:8], want[got != want][:8])
    return m, codes, b


SIZES = [(1, 1), (1, 32), (3, 31), (16, 256), (17, 257), (9, 1000), (5, 40), (33, 136), (100, 3080), (257, 520),
         (64, 2048), (2053, 2056), (2100, 2052)]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,k", SIZES)
def test_quantize_byte_for_byte(device, mem, n, k, kind):
    print(f"quantize {n} {k} {kind}", flush=True)
    rng = np.random.default_rng(n * k)
    rows = rng.standard_normal((n, k)) * np.exp2(rng.integers(-12, 8, (n, 1)))
    rows[rng.random((n, k)) < 0.1] = 0
    hold_quantize(device, mem, rows.astype(np.float32), kind)


def test_quantize_rows_apart_and_off_alignment(device, mem):
    rng = np.random.default_rng(2)
    for kind in ("f32", "f16", "bf16"):
        for n, k, stride, offset in ((20, 64, 72, 8), (20, 64, 65, 0), (7, 64, 64, 3), (5, 1000, 1003, 1)):
            print(f"quantize apart {kind} {n} {k} {stride} {offset}", flush=True)
            hold_quantize(device, mem, rng.standard_normal((n, k)).astype(np.float32), kind, stride, offset)


def test_quantize_halfway_and_every_scale(device, mem):
    """Every halfway point and its neighbours, in blocks of every scale that a
    binary32 block can have, the subnormal ones too."""
    points = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0], np.float32)
    near = np.concatenate([points, np.nextafter(points, np.float32(0)), np.nextafter(points, np.float32(9)), [0, 4]])
    block = np.concatenate([near, -near[:3]]).astype(np.float32)[:32]
    assert block.size == 32
    exps = np.arange(-149, 126)
    rows = np.ldexp(block[None].astype(np.float64), exps[:, None])
    rows = np.where(np.abs(rows) < 3.4e38, rows, 3.4e38 * np.sign(rows)).astype(np.float32)
    hold_quantize(device, mem, rows, "f32")
    hold_quantize(device, mem, rows[100:190], "bf16")
    hold_quantize(device, mem, rows[125:164], "f16")


def test_quantize_blocks_that_are_not_finite_or_zero(device, mem):
    rng = np.random.default_rng(3)
    rows = rng.standard_normal((20, 128)).astype(np.float32)
    rows[1, 40], rows[2, 3], rows[3, 127], rows[4, 64:96] = np.nan, np.inf, -np.inf, 0
    rows[5] = -0.0
    for kind in ("f32", "f16", "bf16"):
        m, codes, b = hold_quantize(device, mem, rows, kind)
        assert (b == 255).sum() == 3
        y, sc = mem.empty(20 * 128 * 4), mem.empty(20 * 4 * 4)
        mx4.Dequantize(device, m, y, "f32", scales=sc).enqueue()
        device.sync()
        assert np.array_equal(y.read(np.float32).reshape(20, 128), M.values(codes, b, 128).astype(np.float32),
                              equal_nan=True)
        assert np.array_equal(sc.read(np.float32).reshape(20, 4), M.scale_of(b.astype(int)).astype(np.float32),
                              equal_nan=True)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,k,pad", [(1, 1, 0), (9, 1000, 0), (17, 264, 8), (33, 100, 3), (64, 2048, 0)])
def test_dequantize_rounds_each_value_once(device, mem, n, k, pad, kind):
    print(f"dequantize {n} {k} {pad} {kind}", flush=True)
    rng = np.random.default_rng(n + k)
    codes = rng.integers(0, 16, (n, -(-k // 32), 32)).astype(np.uint8)
    b = rng.integers(0, 256, codes.shape[:2]).astype(np.uint8) if kind == "f32" else \
        rng.integers(127 - 30, 127 + 17, codes.shape[:2]).astype(np.uint8)
    codes.reshape(n, -1)[:, k:] = 0
    m = put_matrix(device, mem, codes, b, k)
    wide = np.uint32 if kind == "f32" else np.uint16
    y, sc = mem.empty(n * (k + pad) * wide().itemsize), mem.empty(4 * (n * codes.shape[1] + 1))
    mx4.Dequantize(device, m, y, kind, y_stride=k + pad, scales=sc).enqueue()
    device.sync()
    bits = y.read(wide, n * (k + pad)).reshape(n, k + pad)
    assert np.all(bits[:-1, k:] == wide(SENTINEL & np.iinfo(wide).max)), "written between rows"
    want = M.values(codes, b, k)
    with np.errstate(over="ignore"):
        want = want.astype(np.float32)
        got = np.ascontiguousarray(bits[:, :k])
        if kind == "f32":
            assert np.array_equal(got.view(np.float32), want, equal_nan=True)
        else:
            assert np.array_equal(got, S.narrow(want, kind == "bf16"))
    sc = sc.read(np.float32)
    assert np.array_equal(sc[:-1].reshape(b.shape), M.scale_of(b.astype(int)).astype(np.float32), equal_nan=True)
    assert sc[-1:].view(np.uint32)[0] == SENTINEL


# Products ----------------------------------------------------------------------


def random_matrix(rng, n, k, spread):
    codes = rng.integers(0, 16, (n, -(-k // 32), 32)).astype(np.uint8)
    codes.reshape(n, -1)[:, k:] = 0
    return codes, (127 + rng.integers(-spread, spread + 1, codes.shape[:2])).astype(np.uint8)


def product(device, mem, a, b, m, n, kind, pad=0):
    wide = np.uint32 if kind == "f32" else np.uint16
    c = mem.empty((m * (n + pad) + 8) * wide().itemsize)
    mx4.Gemm(device, a, b, c, c_type=kind, c_stride=n + pad).enqueue()
    device.sync()
    bits = c.read(wide)
    last = bits[(m - 1) * (n + pad) + n:m * (n + pad) + 8]
    assert np.all(last == wide(SENTINEL & np.iinfo(wide).max)), "written past the product"
    bits = bits[:m * (n + pad)].reshape(m, n + pad)
    assert np.all(bits[:, n:] == wide(SENTINEL & np.iinfo(wide).max)), "written between rows"
    return np.ascontiguousarray(bits[:, :n])


SHAPES = [(1, 1, 1), (1, 16, 32), (2, 17, 300), (3, 100, 128), (8, 8192, 2048), (15, 48, 4100), (16, 250, 777),
          (17, 33, 64), (31, 130, 1000), (33, 64, 512), (64, 512, 256), (65, 257, 513), (100, 1001, 3080),
          (128, 512, 96), (129, 384, 2048), (200, 100, 5000), (255, 300, 1536), (256, 256, 128), (257, 513, 640),
          (300, 1030, 2304), (512, 768, 4096), (1000, 40, 130), (1030, 2050, 300), (250, 2040, 2048),
          (500, 2030, 1900), (200, 8192, 2048), (201, 8191, 2049), (30, 16380, 2040), (27, 16001, 700),
          (500, 8190, 2048), (4000, 2050, 1900), (5000, 8192, 3080), (4097, 8111, 2500), (4090, 4090, 8190)]


def test_the_products_shapes_reach_every_form():
    forms = {runtime.library().fk_mx4_gemm_form(*s).decode() for s in SHAPES}
    assert forms == {"few 1x1", "few 4x1", "few 4x2", "few 8x2", "mid 8x8", "many 16x16"}


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_products_whose_sums_fit_are_exact(device, mem, m, n, k):
    """Scales of 1 and 2: every product is a multiple of 1/4 of at most 144 and
    the sums stay below 2^21, so binary32 holds each partial sum of any order
    (the host's too)."""
    print(f"gemm exact {m} {n} {k}", flush=True)
    rng = np.random.default_rng(m + n + k)
    (ca, sa), (cb, sb) = random_matrix(rng, m, k, 0), random_matrix(rng, n, k, 0)
    sa += rng.integers(0, 2, sa.shape).astype(np.uint8)
    sb += rng.integers(0, 2, sb.shape).astype(np.uint8)
    want = M.values(ca, sa, k).astype(np.float32) @ M.values(cb, sb, k).T.astype(np.float32)
    a, b = put_matrix(device, mem, ca, sa, k), put_matrix(device, mem, cb, sb, k)
    for kind, pad in (("f32", 0), ("f16", 3 if n % 8 else 0), ("bf16", 4 if n % 8 else 8)):
        got = product(device, mem, a, b, m, n, kind, pad)
        bits = want.view(np.uint32) if kind == "f32" else S.narrow(want, kind == "bf16")
        # +0 and -0 alike: a sum's zero has either sign
        same = (got == bits) | ((want == 0) & ((got & (0x7FFFFFFF if kind == "f32" else 0x7FFF)) == 0))
        assert same.all(), (kind, int((~same).sum()), np.argwhere(~same)[:4].tolist())


# Of each form whose wavefronts share k: sizes, and the wavefronts.
TURNS = [("few 1x1", 5, 200, 8), ("few 4x1", 100, 1000, 8), ("few 4x2", 100, 2500, 4), ("few 8x2", 500, 1500, 4)]


@pytest.mark.parametrize("form,m,n,w", TURNS)
def test_products_of_one_to_six_pairs_of_tiles_a_wavefront(device, mem, form, m, n, w):
    """As above, k ending in each turn of a wavefront's loop."""
    rng = np.random.default_rng(m)
    for pairs in (w + 1, 2 * w - 1, 2 * w, 2 * w + 1, 3 * w, 3 * w + 2, 4 * w, 4 * w + 1, 5 * w, 6 * w - 1):
        k = 256 * pairs - 37
        print(f"gemm turns {form} {m} {n} {k}", flush=True)
        assert runtime.library().fk_mx4_gemm_form(m, n, k).decode() == form
        (ca, sa), (cb, sb) = random_matrix(rng, m, k, 0), random_matrix(rng, n, k, 0)
        want = M.values(ca, sa, k).astype(np.float32) @ M.values(cb, sb, k).T.astype(np.float32)
        got = product(device, mem, put_matrix(device, mem, ca, sa, k), put_matrix(device, mem, cb, sb, k), m, n, "f32")
        assert np.array_equal(got.view(np.float32), want)


@pytest.mark.parametrize("m,n,k", [(1, 64, 4096), (9, 300, 2048), (40, 200, 1000), (256, 512, 2048), (300, 700, 900)])
def test_products_over_scales_apart(device, mem, m, n, k):
    """Scales 2^-20 .. 2^20: off by the additions' roundings, k of them of at
    most 2^-23 of the terms' sizes together, and the result's own."""
    print(f"gemm scales {m} {n} {k}", flush=True)
    rng = np.random.default_rng(k)
    (ca, sa), (cb, sb) = random_matrix(rng, m, k, 20), random_matrix(rng, n, k, 20)
    va, vb = M.values(ca, sa, k), M.values(cb, sb, k)
    want, size = va @ vb.T, np.abs(va) @ np.abs(vb).T
    got = product(device, mem, put_matrix(device, mem, ca, sa, k), put_matrix(device, mem, cb, sb, k), m, n, "f32")
    err = np.abs(got.view(np.float32).astype(np.float64) - want)
    assert np.all(err <= k * 2.0 ** -23 * size + 2.0 ** -24 * np.abs(want)), (err / size).max()


def test_products_of_rows_that_are_not_numbers(device, mem):
    """A block of scale NaN makes its own row's products NaN and no other's."""
    rng = np.random.default_rng(8)
    for m, n, k in ((5, 40, 512), (300, 260, 512)):
        (ca, sa), (cb, sb) = random_matrix(rng, m, k, 2), random_matrix(rng, n, k, 2)
        sa[3, 5], sb[17, 0] = 255, 255
        want = M.values(ca, sa, k) @ M.values(cb, sb, k).T
        got = product(device, mem, put_matrix(device, mem, ca, sa, k), put_matrix(device, mem, cb, sb, k), m, n, "f32")
        assert np.array_equal(np.isnan(got.view(np.float32)), np.isnan(want))


def test_a_linear_captured_with_its_quantisation(device, mem):
    """Rows quantised and multiplied in one graph, replayed over other rows and
    beside eager calls: each replay's result the eager one's bits, within the
    accumulation's bound of the definition."""
    rng = np.random.default_rng(9)
    m, n, k = 20, 300, 1000
    weights = matrix(device, mem, n, k)
    w = rng.standard_normal((n, k)).astype(np.float32)
    mx4.Quantize(device, mem.put(w), weights).enqueue()
    x, rows, y = mem.empty(4 * m * k), matrix(device, mem, m, k), mem.empty(4 * m * n)
    ops = [mx4.Quantize(device, x, rows), mx4.Gemm(device, rows, weights, y)]
    vw = M.values(*M.quantize(w), k)
    stream = device.new_stream()
    device.sync()
    with device.capture(stream) as captured:
        for op in ops:
            op.enqueue(stream)
    for turn in range(4):
        data = rng.standard_normal((m, k)).astype(np.float32) * 2.0 ** turn
        x.write(data)
        captured[0].replay(stream)
        device.sync(stream)
        got = y.read(np.float32).reshape(m, n)
        vx = M.values(*M.quantize(data), k)
        assert np.all(np.abs(got - vx @ vw.T) <= k * 2.0 ** -23 * (np.abs(vx) @ np.abs(vw).T))
        y.write(np.zeros(m * n, np.float32))
        for op in ops:
            op.enqueue()
        device.sync()
        assert np.array_equal(y.read(np.uint32), got.view(np.uint32).ravel())
    captured[0].destroy()


def test_products_on_two_streams_at_once(device, mem):
    """Products of one weight by two streams, of different forms: each one's
    bits those it has alone."""
    rng = np.random.default_rng(17)
    n, k = 2050, 1900
    weights = matrix(device, mem, n, k)
    mx4.Quantize(device, mem.put(rng.standard_normal((n, k)).astype(np.float32)), weights).enqueue()
    ops, outs = [], []
    for m in (8, 1000):
        rows, y = matrix(device, mem, m, k), mem.empty(4 * m * n)
        ops.append([mx4.Quantize(device, mem.put(rng.standard_normal((m, k)).astype(np.float32)), rows),
                    mx4.Gemm(device, rows, weights, y)])
        outs.append(y)
    alone = []
    for pair, y in zip(ops, outs):
        for op in pair:
            op.enqueue()
        device.sync()
        alone.append(y.read(np.uint32).copy())
        y.write(np.zeros_like(alone[-1]))
    device.sync()
    streams = [device.new_stream(), device.new_stream()]
    for _ in range(5):
        for i in range(2):
            for pair, stream in zip(ops, streams):
                pair[i].enqueue(stream)
    for s in streams:
        device.sync(s)
    for y, want in zip(outs, alone):
        assert np.array_equal(y.read(np.uint32), want)
