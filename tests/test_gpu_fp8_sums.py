"""The sums of the 8-bit products (include/fkrocm_fp8.h: fk_fp8_gemm): whole in
C of every type, cut off where a caller asks for that."""

import numpy as np
import pytest

import fp8_cases as F
import serve_cases as S
from furykernel_amd import fp8
from test_gpu_fp8 import put_matrix, random_matrix
from test_gpu_serve import SENTINEL, Memory, mem  # noqa: F401  (mem is a fixture)

pytestmark = pytest.mark.gpu


def product(device, mem, a, b, m, n, k, kind, cut=False, pad=0):  # noqa: F811
    print(f"product {m} {n} {k} {kind} {cut} {fp8.gemm_form(m, n, k, kind, cut)}", flush=True)
    c = mem.empty(m * (n + pad) * 2)
    fp8.Gemm(device, put_matrix(device, mem, *a, k), put_matrix(device, mem, *b, k), c, c_type=kind,
             c_stride=n + pad, cut_sums=cut).enqueue()
    device.sync()
    bits = c.read(np.uint16, m * (n + pad)).reshape(m, n + pad)
    assert np.all(bits[:, n:] == SENTINEL & 0xFFFF), "written between rows"
    return S.widen(np.ascontiguousarray(bits[:, :n]), kind == "bf16")


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("m,n,k", [(8, 40, 256), (100, 5000, 256), (97, 8190, 515), (130, 300, 256), (600, 700, 256),
                                   (300, 3001, 256), (600, 3000, 520), (97, 16390, 1030), (4099, 3001, 256)])
def test_products_to_16_bits_keep_small_terms_beside_large_ones(device, mem, m, n, k, kind):  # noqa: F811
    """448 448, its negative, and terms down to 2^-18 of them, six of them among
    the eight products that hold both: what is left is the small terms' sum,
    rounded once (the large ones' sum is exact: 2^-23 of it for each of the two)."""
    rng = np.random.default_rng(6)
    x, w = np.zeros((m, k)), np.zeros((n, k))
    x[:, 0] = x[:, 1] = w[:, 0] = 448
    w[:, 1] = -448
    x[:, 2:] = np.exp2(rng.integers(-9, 0, (m, k - 2)))
    w[:, 2:] = rng.choice([-1.0, 1.0], (n, k - 2))
    a, b = F.quantize(x), F.quantize(w)
    got, want = product(device, mem, a, b, m, n, k, kind), F.values(*a, k) @ F.values(*b, k).T
    off = 2.0 ** -23 * 448 ** 2 * 2
    assert np.all(np.abs(got - want) <= off + S.half_step(kind) * (np.abs(want) + off))


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_each_forms_products_of_cut_sums(device, mem, kind):  # noqa: F811
    """Odd sizes of every form, by its name: within what eight products lose."""
    sizes = [(3, 509, 130), (17, 3001, 130), (3, 8190, 1030), (17, 8190, 300), (47, 5003, 130), (97, 8190, 515),
             (17, 12001, 515), (299, 3001, 515), (17, 16390, 300), (97, 16390, 1030), (17, 16390, 515),
             (4099, 3001, 130)]
    assert {fp8.gemm_form(*s, kind, True) for s in sizes} == {
        "few 1x1", "few 1x2", "few 2x1", "few 2x2", "few 4x2", "few 8x2", "few 4x3", "few 4x4", "mid 8x8",
        "mid 8x8 deep", "mid 4x8 deep", "many 16x16"}
    for m, n, k in sizes:
        rng = np.random.default_rng(n)
        a, b = random_matrix(rng, m, k, 3), random_matrix(rng, n, k, 3)
        a = (a[0], a[1] * 2.0 ** -14)
        got = product(device, mem, a, b, m, n, k, kind, True, 3)
        av, bv = F.values(*a, k), F.values(*b, k)
        want, size = av @ bv.T, np.abs(av) @ np.abs(bv).T
        rel = k * 2.0 ** -23 + 7 * 2.0 ** -14
        tol = rel * size + S.half_step(kind) * np.abs(want) * (1 + rel) + 2.0 ** -25   # (f16's smallest step)
        bad = ~(np.abs(got - want) <= tol)
        assert not bad.any(), (m, n, k, int(bad.sum()), np.argwhere(bad)[:4].tolist())


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("m,n,k", [(7, 130, 1100), (600, 700, 1100), (2050, 1030, 1100)])
def test_whole_number_products_of_cut_sums_are_exact(device, mem, m, n, k, kind):  # noqa: F811
    """Whole numbers up to 4: no product is below 2^-14 of another, so none is cut."""
    rng = np.random.default_rng(m * n)
    mats = []
    for rows in (m, n):
        blocks = -(-k // 128)
        x = rng.integers(-4, 5, (rows, blocks * 128)).astype(np.float64)
        x[:, k:] = 0
        mats.append((F.encode(x.reshape(rows, blocks, 128)), np.ones((rows, blocks))))
    want = (F.values(*mats[0], k) @ F.values(*mats[1], k).T).astype(np.float32)
    want = S.widen(S.narrow(want, kind == "bf16"), kind == "bf16")
    assert np.array_equal(product(device, mem, *mats, m, n, k, kind, True), want)
