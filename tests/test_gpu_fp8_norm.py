"""The norm to 8 bits (include/fkrocm_fp8.h: fk_fp8_add_norm) byte for byte: the
codes and scales of the exact value, at every size and form and at the ends of
binary32."""

import numpy as np
import pytest

import fp8_cases as F
from furykernel_amd import fp8
from test_gpu_fp8 import add, matrix, placed
from test_gpu_mx4 import held
from test_gpu_serve import Memory, mem  # noqa: F401  (mem is a fixture)

pytestmark = pytest.mark.gpu


def hold(device, mem, xb, h, g, kind, eps=1e-5, residual=None, total=False, pads=(0, 0, 0)):  # noqa: F811
    """The norm of rows `xb` (and `residual`), whose sum's values are `h`, against
    binary64's."""
    n, k = xb.shape
    px, pr, ps = (k + p for p in pads)
    m = matrix(device, mem, n, k)
    word = np.uint32 if kind == "f32" else np.uint16
    bs = mem.put(placed(np.full((n, k), 0x55, word), kind, ps)) if total else None
    fp8.AddNorm(device, mem.put(placed(xb, kind, px)), m, eps, gamma=None if g is None else mem.put(g), x_type=kind,
                residual=None if residual is None else mem.put(placed(residual, kind, pr)), sum=bs,
                x_stride=px, residual_stride=pr, sum_stride=ps).enqueue()
    device.sync()
    with np.errstate(all="ignore"):
        y = F.norm(h, g, np.float64(np.float32(eps)))
        y = np.where(np.isinf(y.astype(np.float32)), np.inf, y)   # past binary32's range: not finite
        codes, scales = F.pack(*F.quantize(y))
    got = m.codes.read(np.uint8), m.scales.read(np.uint8)
    bad = ~F.same_codes(got[0], codes)
    assert not bad.any(), (int(bad.sum()), bad.size, got[0][bad][:6], codes[bad][:6])
    assert np.array_equal(got[1], scales), int((got[1] != scales).sum())


def rows_of(rng, n, k, kind, size=0):
    return held(rng.standard_normal((n, k)) * np.exp2(rng.integers(-9, 9, (n, 1)) + float(size)), kind)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,k", [(1, 1), (1, 8), (3, 127), (5, 128), (17, 129), (8, 2048), (33, 1000), (200, 2056),
                                 (5, 4097), (129, 5000), (2, 8192), (3, 16384), (2, 32768), (1, 32761), (1024, 2049),
                                 (1033, 2600), (2049, 4100), (1030, 8192), (1025, 2048), (1024, 1), (3000, 300)])
def test_every_size(device, mem, n, k, kind):  # noqa: F811
    print(f"exact norm {n} {k} {kind}", flush=True)
    rng = np.random.default_rng(n + k)
    (xb, x), (rb, r) = rows_of(rng, n, k, kind), held(rng.standard_normal((n, k)) * 3, kind)
    g = (1 + 0.2 * rng.standard_normal(k)).astype(np.float32)
    hold(device, mem, xb, add(x, r, kind)[1], g, kind, residual=rb, total=True, pads=(n % 3, 8, k % 5))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("residual,gamma,total", [(False, False, False), (False, True, True), (True, False, False)])
def test_every_form(device, mem, residual, gamma, total, kind):  # noqa: F811
    rng = np.random.default_rng(3)
    for n, k in ((19, 1000), (4, 2500), (1100, 700)):
        print(f"exact norm {n} {k} {kind} {residual} {gamma} {total}", flush=True)
        (xb, x), (rb, r) = rows_of(rng, n, k, kind), held(rng.standard_normal((n, k)) * 3, kind)
        g = (1 + 0.2 * rng.standard_normal(k)).astype(np.float32) if gamma else None
        hold(device, mem, xb, add(x, r, kind)[1] if residual else x, g, kind, residual=rb if residual else None,
             total=total)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_rows_with_zeros(device, mem, kind):  # noqa: F811
    """Sparse rows, rows of zeros but one, gammas of zero; signs of zeros too."""
    rng = np.random.default_rng(4)
    x = rng.standard_normal((1100, 1000)) * (rng.random((1100, 1000)) < 0.3)
    x[:40], x[:40, 5], x[40:60, :500] = -0.0, 3, 0
    g = np.where(rng.random(1000) < 0.2, 0, 1 + 0.1 * rng.standard_normal(1000)).astype(np.float32)
    xb, x = held(x, kind)
    for n in (60, 1100):
        hold(device, mem, xb[:n], x[:n], g, kind)
        hold(device, mem, xb[:n], x[:n], None, kind, eps=0.0)


@pytest.mark.parametrize("n", [64, 1100])
def test_a_gamma_that_is_not_finite_and_values_past_the_range(device, mem, n):  # noqa: F811
    """NaN where the formula is infinite, NaN or past binary32's range, the rest of
    the block by its own largest."""
    rng = np.random.default_rng(5)
    x = rng.standard_normal((n, 1000)).astype(np.float32)
    x[3, 10:400:7] = 0
    g = (1 + 0.1 * rng.standard_normal(1000)).astype(np.float32)
    g[[10, 150, 151]], g[[24, 300, 500]], g[[38, 640]] = np.inf, -np.inf, np.nan
    hold(device, mem, x, x, g, "f32")
    x[5, 3:900:31], g = x[5, 3:900:31] * 20, np.full(1000, 1.5 * 2.0 ** 126, np.float32)
    hold(device, mem, x, x, g, "f32")
    hold(device, mem, x, x, -g, "f32")


@pytest.mark.parametrize("n", [64, 1100])
@pytest.mark.parametrize("gamma", [0, -120, -126, -130, -135])
def test_values_below_the_normal_range(device, mem, n, gamma):  # noqa: F811
    """Results, products on their way and rows below 2^-126, where a binary32 has
    fewer bits than its largest ones."""
    rng = np.random.default_rng(6 - gamma)
    g = np.ldexp(1 + 0.2 * rng.standard_normal(1000), gamma).astype(np.float32)
    for size, eps in ((0, 1e-5), (-126, 1e-5), (-130, 1e-5), (-136, 1e-5), (-140, 1e-5), (-140, 0.0)):
        print(f"exact norm below the range {n} {gamma} {size} {eps}", flush=True)
        xb, x = held(rng.standard_normal((n, 1000)) * 2.0 ** size, "f32")
        hold(device, mem, xb, x, g, "f32", eps)
    # some far below their row's others, a large gamma over them
    x = (rng.standard_normal((n, 1000)) * np.exp2(rng.choice([0, -126, -130, -138], (n, 1000)))).astype(np.float32)
    hold(device, mem, x, x, np.ldexp(g.astype(np.float64), 40 - 2 * gamma // 3).astype(np.float32), "f32")


@pytest.mark.parametrize("n", [64, 1100])
def test_rows_at_the_upper_end(device, mem, n):  # noqa: F811
    """Rows whose root binary32 holds in part or not at all, large and small
    elements among them."""
    rng = np.random.default_rng(7)
    for size in (120, 125, 126, 127):
        x = np.ldexp(np.clip(rng.standard_normal((n, 1000)), -1.9, 1.9), size - rng.integers(0, 2, (n, 1000)) * 20)
        xb, x = held(x, "f32")
        for g in (0, 30, 100):
            print(f"exact norm at the upper end {n} {size} {g}", flush=True)
            hold(device, mem, xb, x, np.ldexp(1 + 0.2 * rng.standard_normal(1000), g).astype(np.float32), "f32")
    xb, x = held(np.ldexp(rng.standard_normal((n, 1000)) * 0.5, 127), "bf16")
    hold(device, mem, xb, x, None, "bf16")
