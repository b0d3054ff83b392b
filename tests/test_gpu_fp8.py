"""8-bit matrices (include/fkrocm_fp8.h) on the GPU: the codes and scales byte
for byte, the values they stand for, the norm within what its binary32 sums
leave open, and products: exact where every partial sum fits, elsewhere within
the accumulation's bound."""

import numpy as np
import pytest

import fp8_cases as F
import serve_cases as S
from furykernel_amd import fp8, runtime
from test_gpu_mx4 import held
from test_gpu_serve import SENTINEL, Memory, mem  # noqa: F401  (mem is a fixture)

pytestmark = pytest.mark.gpu


def matrix(device, mem, rows, k):
    m = fp8.Fp8Matrix(device, rows, k)
    mem.keep(m)
    for b in (m.codes, m.scales):
        b.write(np.full(b.size, 0x5A, np.uint8))
    return m


def put_matrix(device, mem, codes, scale, k):
    m = matrix(device, mem, codes.shape[0], k)
    for buf, data in zip((m.codes, m.scales), F.pack(codes, scale)):
        buf.write(data)
    return m


def placed(bits, kind, stride, offset=0):
    """Rows' bits apart, something else between them."""
    fill, of = (0x7E7E7E7E, np.uint32) if kind == "f32" else (0x7E7E, np.uint16)
    n, k = bits.shape
    src = np.full(offset + n * stride, fill, of)
    src[offset:].reshape(n, stride)[:, :k] = bits.view(of)
    return src


def hold_quantize(device, mem, rows, kind, stride=None, offset=0):
    n, k = rows.shape
    bits, x = held(rows, kind)
    stride = k if stride is None else stride
    m = matrix(device, mem, n, k)
    fp8.Quantize(device, mem.put(placed(bits, kind, stride, offset)), m, x_type=kind, x_stride=stride,
                 x_offset=offset).enqueue()
    device.sync()
    codes, scale = F.quantize(x)
    want = F.pack(codes, scale)
    got = m.codes.read(np.uint8)
    bad = np.flatnonzero(~F.same_codes(got, want[0]))
    assert not bad.size, (bad.size, bad[:8], got[bad[:8]], want[0][bad[:8]])
    got = m.scales.read(np.uint8)
    assert np.array_equal(got, want[1]), (np.flatnonzero(got != want[1])[:8], got[got != want[1]][:8])
    return m, codes, scale


SIZES = [(1, 1), (1, 128), (3, 127), (16, 256), (17, 129), (9, 1000), (5, 40), (33, 136), (100, 3080), (257, 520),
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
    """Every halfway point between two codes and its neighbours in binary32, in
    blocks of every scale that a binary32 block can have, the subnormal ones
    too; and largest magnitudes on both sides of a scale's limit."""
    mid = ((F.MAGNITUDES[1:] + F.MAGNITUDES[:-1]) / 2).astype(np.float32)
    near = np.concatenate([mid, np.nextafter(mid, np.float32(0)), np.nextafter(mid, np.float32(500))])
    near = np.concatenate([near, np.zeros(-near.size % 127, np.float32)]).reshape(-1, 127)
    block = np.concatenate([np.full((len(near), 1), 448, np.float32), near * np.where(np.arange(127) % 3, 1, -1)], 1)
    exps = np.arange(-157, 120)
    rows = np.ldexp(block.reshape(1, -1).astype(np.float64), exps[:, None]).astype(np.float32)
    hold_quantize(device, mem, rows, "f32")
    hold_quantize(device, mem, rows[60:200], "bf16")
    hold_quantize(device, mem, rows[135:160], "f16")
    tops = np.ldexp(np.array([448, 449, 256, 447.99, 224, 225], np.float64)[None], np.arange(-140, 119)[:, None])
    rows = np.zeros((tops.size, 130), np.float32)
    rows[:, 5], rows[:, 129] = tops.ravel(), -tops.ravel()
    hold_quantize(device, mem, rows, "f32")
    hold_quantize(device, mem, np.nextafter(rows, np.float32(np.inf)), "f32")


def test_quantize_blocks_that_are_not_finite_or_zero(device, mem):
    rng = np.random.default_rng(3)
    rows = rng.standard_normal((20, 300)).astype(np.float32)
    rows[1, 40], rows[2, 3], rows[3, 299], rows[4, 128:256] = np.nan, np.inf, -np.inf, 0
    rows[5], rows[6], rows[7, 128:256] = -0.0, np.nan, np.inf
    for kind in ("f32", "f16", "bf16"):
        m, codes, scale = hold_quantize(device, mem, rows, kind)
        y, sc = mem.empty(20 * 300 * 4), mem.empty(20 * 3 * 4)
        fp8.Dequantize(device, m, y, "f32", scales=sc).enqueue()
        device.sync()
        got, want = y.read(np.float32).reshape(20, 300), F.values(codes, scale, 300).astype(np.float32)
        assert np.array_equal(got, want, equal_nan=True) and np.array_equal(np.signbit(got[5]), np.signbit(want[5]))
        assert np.isnan(got[6]).all() and np.isnan(got).sum() == 3 + 300 + 128
        assert np.array_equal(sc.read(np.float32).reshape(20, 3), scale.astype(np.float32))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,k,pad", [(1, 1, 0), (9, 1000, 0), (17, 264, 8), (33, 100, 3), (64, 2048, 0)])
def test_dequantize_rounds_each_value_once(device, mem, n, k, pad, kind):
    print(f"dequantize {n} {k} {pad} {kind}", flush=True)
    rng = np.random.default_rng(n + k)
    codes = rng.integers(0, 256, (n, -(-k // 128), 128)).astype(np.uint8)
    codes[(codes & 0x7F) == 0x7F] = 0x7E
    exps = rng.integers(-126, 120, codes.shape[:2]) if kind == "f32" else rng.integers(-26, 9, codes.shape[:2])
    scale = np.exp2(exps.astype(np.float64))
    codes.reshape(n, -1)[:, k:] = 0
    m = put_matrix(device, mem, codes, scale, k)
    wide = np.uint32 if kind == "f32" else np.uint16
    y, sc = mem.empty(n * (k + pad) * wide().itemsize), mem.empty(4 * (n * codes.shape[1] + 1))
    fp8.Dequantize(device, m, y, kind, y_stride=k + pad, scales=sc).enqueue()
    device.sync()
    bits = y.read(wide, n * (k + pad)).reshape(n, k + pad)
    assert np.all(bits[:-1, k:] == wide(SENTINEL & np.iinfo(wide).max)), "written between rows"
    with np.errstate(over="ignore"):
        want = F.values(codes, scale, k).astype(np.float32)
        want = want.view(np.uint32) if kind == "f32" else S.narrow(want, kind == "bf16")
    assert np.array_equal(bits[:, :k], want)
    sc = sc.read(np.float32)
    assert np.array_equal(sc[:-1].reshape(scale.shape), scale.astype(np.float32)) and sc[-1:].view(np.uint32)[0] == SENTINEL


# The norm ------------------------------------------------------------------------


def add(x, r, kind):
    """(bits, values) of x + r rounded to their type."""
    with np.errstate(over="ignore", invalid="ignore"):
        return held((x.astype(np.float32) + r.astype(np.float32)).astype(np.float32), kind)


def hold_norm(device, mem, rng, n, k, kind, residual=True, gamma=True, over="", pads=(0, 0, 0), eps=1e-5, rows=None):
    """`over`: which input the sum is written over; pads: rows' strides past k."""
    xb, x = held(rng.standard_normal((n, k)) * np.exp2(rng.integers(-9, 9, (n, 1))) if rows is None else rows, kind)
    rb, r = held(rng.standard_normal((n, k)) * 3, kind)
    hb, h = add(x, r, kind) if residual else (xb, x)
    g = (1 + 0.2 * rng.standard_normal(k)).astype(np.float32) if gamma else None
    px, pr, ps = (k + p for p in pads)
    bx = mem.put(placed(xb, kind, px))
    br = mem.put(placed(rb, kind, pr)) if residual else None
    word = np.uint32 if kind == "f32" else np.uint16
    bs = {"x": bx, "residual": br, "": mem.put(placed(np.full((n, k), 0x55, word), kind, ps)), "none": None}[over]
    ps = {"x": px, "residual": pr}.get(over, ps)
    m = matrix(device, mem, n, k)
    fp8.AddNorm(device, bx, m, eps, gamma=None if g is None else mem.put(g), residual=br, sum=bs, x_type=kind,
                x_stride=px, residual_stride=pr, sum_stride=ps).enqueue()
    device.sync()
    if bs is not None:
        got = bs.read(word, n * ps).reshape(n, ps)
        assert np.array_equal(got[:, :k], hb.view(word)), "the sum"
        assert np.all(got[:, k:] == word(0x7E7E7E7E & np.iinfo(word).max)), "written between rows"
    raw = m.codes.read(np.uint8), m.scales.read(np.uint8)
    codes, scale = F.unpack(*raw, n, k)
    for got, again in zip(raw, F.pack(codes, scale)):   # the padding is what pack makes of it
        assert np.array_equal(got, again)
    assert not codes.reshape(n, -1)[:, k:].any()
    y, rel = F.norm(h, g, eps), F.norm_relative(k)
    big = F.largest(F.blocks(y), -1)
    lo, hi = F.scale_of(big * (1 - rel)), F.scale_of(big * (1 + rel))
    assert np.all((scale == lo) | (scale == hi)), "a scale"
    # half a step of the code: 2^-4 of the value, or of the smallest normal code
    wide = np.repeat(scale, 128, 1)[:, :k]
    tol = np.maximum(2.0 ** -4 * np.abs(y), 2.0 ** -10 * wide) * (1 + 2 * rel) + rel * np.abs(y)
    bad = ~(np.abs(F.values(codes, scale, k) - y) <= tol)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist())
    return m


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,k", [(1, 1), (1, 8), (3, 127), (5, 128), (17, 129), (8, 2048), (33, 1000), (200, 2056),
                                 (5, 4097), (129, 5000), (2, 8192), (3, 16384), (2, 32768), (1, 32761)])
def test_add_norm(device, mem, n, k, kind):
    print(f"norm {n} {k} {kind}", flush=True)
    hold_norm(device, mem, np.random.default_rng(n + k), n, k, kind)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,k", [(1024, 2049), (1033, 2600), (2049, 4100), (1030, 8192), (1025, 2048)])
def test_add_norm_of_rows_that_fill_the_card(device, mem, n, k, kind):
    print(f"norm {n} {k} {kind}", flush=True)
    hold_norm(device, mem, np.random.default_rng(n + k), n, k, kind, gamma=kind != "f16", pads=(0, 8, 16))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("residual,gamma,over,pads", [
    (False, True, "none", (0, 0, 0)), (False, False, "", (3, 0, 5)), (True, True, "none", (1, 3, 0)),
    (True, False, "x", (7, 2, 0)), (True, True, "residual", (1, 8, 0)), (False, True, "x", (0, 0, 0)),
    (True, True, "", (9, 8, 7))])
def test_add_norm_forms(device, mem, residual, gamma, over, pads, kind):
    for n, k in ((19, 1000), (4, 2500)):
        print(f"norm {n} {k} {kind} {residual} {gamma} {over} {pads}", flush=True)
        hold_norm(device, mem, np.random.default_rng(k), n, k, kind, residual, gamma, over, pads)


def test_add_norm_of_zeros_large_and_small_rows(device, mem):
    rng = np.random.default_rng(4)
    rows = rng.standard_normal((6, 300))
    rows[0], rows[1], rows[2], rows[3], rows[4, 7:] = 0, rows[1] * 1e-30, rows[2] * 1e17, 1e-44, 0
    hold_norm(device, mem, rng, 6, 300, "f32", residual=False, rows=rows.astype(np.float32))
    hold_norm(device, mem, rng, 6, 300, "bf16", residual=False, rows=rows, eps=1e-30)
    rows[0] = 1.0
    hold_norm(device, mem, rng, 6, 300, "f16", residual=False, rows=rows * (np.abs(rows) < 100), eps=0.5)


@pytest.mark.parametrize("kind,n,k,size,eps", [
    ("bf16", 1100, 5000, 0, 1e-5), ("f16", 8000, 533, 0, 1e-5), ("f16", 1025, 1, 0, 1e-5), ("f32", 3000, 130, 0, 1e-5), ("f32", 1030, 4096, 0, 1e-5), ("f32", 1500, 2048, 0, 0.0),
    ("bf16", 40, 30001, 0, 1e-5), ("f32", 300, 1000, 100, 0.0), ("f32", 300, 9000, -100, 0.0), ("f32", 64, 700, -60, 1e-30)])
def test_add_norm_s_codes_are_the_exact_value_s(device, mem, kind, n, k, size, eps):
    """Byte for byte: in binary32 a few in a million would be others.  `size`:
    of the rows, a power of two, whose squares binary32 does not hold."""
    rng = np.random.default_rng(n + k)
    xb, x = held(rng.standard_normal((n, k)) * 2.0 ** size, kind)
    rb, r = held(rng.standard_normal((n, k)) * 2.0 ** size, kind)
    hb, h = add(x, r, kind)
    g = (1 + 0.1 * rng.standard_normal(k)).astype(np.float32)
    m = matrix(device, mem, n, k)
    fp8.AddNorm(device, mem.put(xb), m, eps, gamma=mem.put(g), residual=mem.put(rb), x_type=kind).enqueue()
    device.sync()
    for got, want in zip((m.codes, m.scales), F.pack(*F.quantize(F.norm(h, g, np.float64(np.float32(eps)))))):
        assert np.array_equal(got.read(np.uint8), want)


def test_add_norm_of_rows_that_are_not_finite(device, mem):
    """A row with a NaN or an infinity is NaN where the formula is; the others are
    as ever."""
    rng = np.random.default_rng(5)
    x = rng.standard_normal((5, 200)).astype(np.float32)
    clean = x.copy()
    x[1, 3], x[3, 150] = np.nan, np.inf
    ms = []
    for rows in (x, clean):
        m = matrix(device, mem, 5, 200)
        fp8.AddNorm(device, mem.put(rows), m, 1e-5).enqueue()
        device.sync()
        ms.append(F.values(*F.unpack(m.codes.read(np.uint8), m.scales.read(np.uint8), 5, 200), 200))
    assert np.isnan(ms[0][1]).all() and np.isnan(ms[0][3, 150])
    assert not np.delete(ms[0][3], 150).any()             # a finite element over an infinite root
    keep = [0, 2, 4]
    assert np.array_equal(ms[0][keep], ms[1][keep])


# Products ----------------------------------------------------------------------


def random_matrix(rng, n, k, spread):
    codes, _ = F.quantize(rng.standard_normal((n, k)))
    return codes, np.exp2(rng.integers(-spread, spread + 1, codes.shape[:2]).astype(np.float64))


def product(device, mem, a, b, m, n, k, kind, pad=0):
    c = mem.empty(m * (n + pad) * (4 if kind == "f32" else 2))
    fp8.Gemm(device, put_matrix(device, mem, *a, k), put_matrix(device, mem, *b, k), c, c_type=kind,
             c_stride=n + pad).enqueue()
    device.sync()
    word = np.uint32 if kind == "f32" else np.uint16
    bits = c.read(word, m * (n + pad)).reshape(m, n + pad)
    assert np.all(bits[:, n:] == word(SENTINEL & np.iinfo(word).max)), "written between rows"
    bits = np.ascontiguousarray(bits[:, :n])
    return bits.view(np.float32).astype(np.float64) if kind == "f32" else S.widen(bits, kind == "bf16")


def hold_product(device, mem, rng, m, n, k, kind, pad=0, spread=3):
    a, b = random_matrix(rng, m, k, spread), random_matrix(rng, n, k, spread)
    hold_values(device, mem, a, b, m, n, k, kind, pad)
    if kind == "f16":   # (most of which f16 does not hold: and what it holds)
        hold_values(device, mem, (a[0], a[1] * 2.0 ** -16), b, m, n, k, kind, pad)


def hold_values(device, mem, a, b, m, n, k, kind, pad, rows=slice(None)):
    print(f"product {m} {n} {k} {kind} {fp8.gemm_form(m, n, k, kind)}", flush=True)
    got = product(device, mem, a, b, m, n, k, kind, pad)[rows]
    av, bv = F.values(a[0][rows], a[1][rows], k), F.values(*b, k)
    want, size = av @ bv.T, np.abs(av) @ np.abs(bv).T
    # k additions of binary32, cut off or rounded (2^-23 each); of 16 bits the cut
    # of eight products of k, and the result's rounding
    rel = k * 2.0 ** -23 + (0 if kind == "f32" else 7 * 2.0 ** -14)
    tol = rel * size + (0 if kind == "f32" else S.half_step(kind) * np.abs(want) * (1 + rel) + 2.0 ** -25)  # (f16's smallest step)
    with np.errstate(invalid="ignore"):
        bad = ~(np.abs(got - want) <= tol)
    if kind == "f16":   # 65520 is the least that rounds to infinity
        bad &= ~((np.abs(got) == np.inf) & (np.sign(got) == np.sign(want)) & (np.abs(want) + rel * size >= 65520))
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist(), got[bad][:4], want[bad][:4])


PRODUCTS = [(1, 1, 1), (1, 16, 32), (3, 5, 127), (16, 16, 128), (17, 33, 129), (8, 1000, 520), (40, 100, 1000),
            (100, 300, 3080), (129, 257, 640), (300, 500, 264), (513, 700, 512), (2000, 900, 384), (1100, 1300, 2048)]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_products(device, mem, m, n, k, kind):
    hold_product(device, mem, np.random.default_rng(m + n + k), m, n, k, kind, pad=(m + n) % 3)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_products_of_every_form(device, mem, kind):
    """Sizes of each kernel that the rule may take, odd ones among them."""
    seen = set()
    for m, n, k in ((5, 70, 300), (60, 3000, 130), (60, 9000, 200), (120, 9001, 260), (250, 8200, 250),
                    (700, 1500, 400), (2100, 1700, 200), (4100, 4200, 136), (9000, 300, 250), (6200, 8300, 520)):
        seen.add(fp8.gemm_form(m, n, k, kind).split()[0])
        hold_product(device, mem, np.random.default_rng(m), m, n, k, kind)
    for m, n, k in ((4000, 4090, 1030), (4090, 8100, 1160), (8190, 8190, 1290), (8190, 16300, 2000)):
        if not fp8.gemm_form(m, n, k, kind).startswith("many"):
            continue
        seen.add("many")
        rng = np.random.default_rng(m)
        rows = np.unique(np.concatenate([rng.integers(0, m, 60), [0, m - 1]]))
        a, b = random_matrix(rng, m, k, 3), random_matrix(rng, n, k, 3)
        hold_values(device, mem, (a[0], a[1] * 2.0 ** -14), b, m, n, k, kind, 1, rows)
        break
    assert seen == {"few", "mid", "many"}


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_each_forms_products(device, mem, kind):
    """Odd sizes of every form of the rule's, by its name."""
    sizes = [(3, 509, 130), (17, 509, 515), (3, 16390, 130), (17, 3001, 130), (17, 5003, 130), (3, 8190, 1030),
             (47, 5003, 130), (17, 16390, 130), (17, 8190, 300), (47, 9001, 130), (17, 16390, 300), (17, 12001, 515),
             (17, 16390, 515), (97, 8190, 300), (97, 8190, 515), (299, 3001, 515), (4099, 3001, 130),
             (97, 16390, 1030), (97, 16390, 2060)]
    names = {"few 1x1", "few 1x2", "few 2x1", "few 2x2", "few 4x2", "few 4x3", "few 4x4", "mid 8x8", "mid 8x8 deep",
             "mid 4x8 deep", "many 16x16"} | (set() if kind == "f32" else {"few 8x2"})
    assert {fp8.gemm_form(*s, kind) for s in sizes} == names
    for s in sizes:
        rng = np.random.default_rng(s[1])
        a, b = random_matrix(rng, s[0], s[2], 3), random_matrix(rng, s[1], s[2], 3)
        hold_values(device, mem, (a[0], a[1] * 2.0 ** -14), b, *s, kind, 3)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m,n,k", [(7, 130, 1100), (130, 260, 1100), (600, 700, 1100), (2050, 1030, 1100)])
def test_whole_number_products_are_exact(device, mem, m, n, k, kind):
    """Small whole numbers, scales of 1/2 to 2 a block: every product and partial
    sum is exact, so the product is, to the bit (16 bits: rounded once)."""
    print(f"exact product {m} {n} {k} {kind} {fp8.gemm_form(m, n, k, kind)}", flush=True)
    rng = np.random.default_rng(m * n)
    mats = []
    for rows in (m, n):
        blocks = -(-k // 128)
        x = rng.integers(-4, 5, (rows, blocks * 128)).astype(np.float64)
        x[:, k:] = 0
        mats.append((F.encode(x.reshape(rows, blocks, 128)),
                     np.exp2(rng.integers(-1, 2, (rows, blocks)).astype(np.float64))))
    got = product(device, mem, *mats, m, n, k, kind)
    want = (F.values(*mats[0], k) @ F.values(*mats[1], k).T).astype(np.float32)
    if kind == "f32":
        assert np.array_equal(got, want)
    else:
        assert np.array_equal(got, S.widen(S.narrow(want, kind == "bf16"), kind == "bf16"))


@pytest.mark.parametrize("m,n", [(8, 40), (130, 300), (600, 700), (1200, 1100)])
def test_f32_products_keep_small_terms_beside_large_ones(device, mem, m, n):
    """448 448, its negative, and terms down to 2^-18 of them: sums that 8-bit
    operations alone would cut off."""
    print(f"small terms {m} {n} {fp8.gemm_form(m, n, 256, 'f32')}", flush=True)
    rng = np.random.default_rng(6)
    x, w = np.zeros((m, 256)), np.zeros((n, 256))
    x[:, 0] = x[:, 1] = w[:, 0] = 448
    w[:, 1] = -448
    x[:, 2:] = np.exp2(rng.integers(-9, 0, (m, 254)))
    w[:, 2:] = rng.choice([-1.0, 1.0], (n, 254))
    a, b = F.quantize(x), F.quantize(w)
    got, want = product(device, mem, a, b, m, n, 256, "f32"), F.values(*a, 256) @ F.values(*b, 256).T
    assert np.abs(got - want).max() <= 2.0 ** -23 * 448 ** 2 * 2


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_products_of_scales_at_their_ends(device, mem, kind):
    """Scales whose product is within a binary32 though they are not."""
    rng = np.random.default_rng(7)
    a, b = random_matrix(rng, 20, 256, 0), random_matrix(rng, 40, 256, 0)
    a = (a[0], np.full_like(a[1], 2.0 ** -110))
    b = (b[0], np.full_like(b[1], 2.0 ** 100))
    got, want = product(device, mem, a, b, 20, 40, 256, kind), F.values(*a, 256) @ F.values(*b, 256).T
    size = np.abs(F.values(*a, 256)) @ np.abs(F.values(*b, 256)).T
    assert np.all(np.abs(got - want) <= (2.0 ** -7 if kind == "bf16" else 2.0 ** -15) * size)


@pytest.mark.parametrize("m,n", [(20, 40), (300, 520), (1100, 1030)])
def test_f32_products_of_the_smallest_scale(device, mem, m, n):
    """Elements below 2^-126, which bfloat16 holds in part or not at all: 2^-126
    times the other operand's at most from each."""
    rng = np.random.default_rng(9)
    a, b = random_matrix(rng, m, 256, 0), random_matrix(rng, n, 256, 0)
    a, b = (a[0], np.full_like(a[1], 2.0 ** -126)), (b[0], np.full_like(b[1], 2.0 ** 112))
    got, (av, bv) = product(device, mem, a, b, m, n, 256, "f32"), (F.values(*x, 256) for x in (a, b))
    tol = 256 * 2.0 ** -23 * (np.abs(av) @ np.abs(bv).T) + 2.0 ** -126 * np.abs(bv).sum(1)
    assert np.all(np.abs(got - av @ bv.T) <= tol)


def test_a_nan_is_its_row_and_columns_only(device, mem):
    rng = np.random.default_rng(8)
    for m, n, kind in ((20, 50, "f32"), (20, 50, "f16"), (600, 700, "f32"), (600, 700, "bf16")):
        a, b = random_matrix(rng, m, 300, 1), random_matrix(rng, n, 300, 1)
        clean = product(device, mem, a, b, m, n, 300, kind)
        a[0][3, 1, 7] = 0x7F
        b[0][17, 0, 100] = 0xFF
        got = product(device, mem, a, b, m, n, 300, kind)
        hit = np.zeros((m, n), bool)
        hit[3], hit[:, 17] = True, True
        assert np.isnan(got[hit]).all() and np.array_equal(got[~hit], clean[~hit])


# A run of them ---------------------------------------------------------------------


@pytest.mark.parametrize("kind,n,k,wide", [("f32", 8, 512, 700), ("bf16", 45, 1000, 264), ("f16", 300, 264, 1000)])
def test_a_captured_layer(device, mem, kind, n, k, wide):
    """The stream's addition and norm, a product up, its norm, a product down
    onto a row, captured on a stream of its own and replayed over new rows with
    eager calls between: every replay bit for bit the eager one."""
    rng = np.random.default_rng(9)
    up, down = (matrix(device, mem, *s) for s in ((wide, k), (k, wide)))
    for m in (up, down):
        fp8.Quantize(device, mem.put(rng.standard_normal((m.rows, m.k)).astype(np.float32) * 0.1), m).enqueue()
    word = 4 if kind == "f32" else 2
    x, r, h1, h2 = (mem.empty(n * c * word) for c in (k, k, wide, k))
    a1, a2 = matrix(device, mem, n, k), matrix(device, mem, n, wide)
    gamma = mem.put(rng.standard_normal(k).astype(np.float32))
    ops = [fp8.AddNorm(device, x, a1, 1e-5, gamma=gamma, residual=r, sum=r, x_type=kind),
           fp8.Gemm(device, a1, up, h1, c_type=kind), fp8.AddNorm(device, h1, a2, 1e-5, x_type=kind),
           fp8.Gemm(device, a2, down, h2, c_type=kind)]
    stream = device.new_stream()
    device.sync()
    with device.capture(stream) as captured:
        for op in ops:
            op.enqueue(stream)
    for step in range(4):
        xs, rs = (held(rng.standard_normal((n, k)), kind)[0] for _ in "xr")
        got = []
        for go in (lambda: captured[0].replay(stream), lambda: [op.enqueue() for op in ops]):
            x.write(xs)
            r.write(rs)
            h2.write(np.zeros(h2.size, np.uint8))
            device.sync()
            go()
            device.sync(stream)
            device.sync()
            got.append([b.read(np.uint8, n * k * word) for b in (r, h2)])
        assert all(np.array_equal(p, q) for p, q in zip(*got)), step
        assert got[0][1].any()
    captured[0].destroy()


def test_two_streams_and_a_step_s_outputs_of_their_own(device, mem):
    rng = np.random.default_rng(10)
    k, ops, outs = 1000, [], []
    for n in (9, 200):
        m, w = matrix(device, mem, n, k), matrix(device, mem, 300, k)
        x, y = (mem.put(rng.standard_normal((rows, k)).astype(np.float32)) for rows in (n, 300))
        c = mem.empty(n * 300 * 4)
        ops.append([fp8.Quantize(device, x, m), fp8.Quantize(device, y, w), fp8.Gemm(device, m, w, c)])
        outs.append(c)
    for run in ops:
        for op in run:
            op.enqueue()
    device.sync()
    want = [c.read(np.uint32) for c in outs]
    streams = [device.new_stream() for _ in ops]
    for c in outs:
        c.write(np.zeros(c.size, np.uint8))
    for i in range(3):
        for run, s in zip(ops, streams):
            run[i].enqueue(s)
    for s in streams:
        device.sync(s)
    assert all(np.array_equal(c.read(np.uint32), w) for c, w in zip(outs, want))


def test_an_earlier_calls_error_is_not_theirs(device, mem):
    m = matrix(device, mem, 5, 40)
    op = fp8.Quantize(device, mem.put(np.ones((5, 40), np.float32)), m)
    with pytest.raises(runtime.FkError):
        device.alloc(1 << 50)
    op.enqueue()
    device.sync()
