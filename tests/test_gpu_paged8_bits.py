"""Attention over 8-bit pages (include/fkrocm_paged8.h): what its outputs of 16
bits keep of the probabilities."""

import numpy as np
import pytest

import fp8_cases as F
import serve_cases as S
from test_gpu_paged8 import attend_inputs, bind_attend
from test_gpu_serve import Memory, mem  # noqa: F401  (mem is a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("q_type", ["f16", "bf16"])
def test_small_differences_of_weighted_values(device, mem, d, q_type):  # noqa: F811
    """Two keys, of score 0 and value -u and of score x and value v, u and v of 1 ..
    15/8 and p = e^x beside u / v: out = (v p - u) / (1 + p), a small difference.
    Roundings of 2^-24: the scale to log2 units and the score 1 each (of |x| < 0.65:
    1.3 together), the exponential 1 ulp (2), of v p < 1.9; the sum of u and p's
    three parts, exact ones, 3, of u < 1.9: 12 in all, over 1 + p > 1.5; and the
    result's half step."""
    print(f"attend8 differences {d} {q_type}", flush=True)
    pairs = [(8 + i, 8 + j) for j in range(8) for i in range(j)]
    n, heads, bf16 = len(pairs), 4, q_type == "bf16"
    u, v = np.array(pairs, np.float64).T / 8
    x = attend_inputs(np.random.default_rng(d), [2] * n, heads, 1, d, 16, q_type)
    near = S.narrow(np.log(u / v), bf16)
    q = near[:, None] + np.arange(-2, 2).astype(np.uint16)     # neighbours of the type
    x["q"][:] = 0
    x["q"][:, :, 0] = q
    for r in range(n):
        b = x["table"][r, 0]
        x["k"][b], x["v"][b], x["scales"][b] = 0, 0, 1
        x["k"][b, 0, 1, 0] = F.encode(np.array(1.0))
        x["v"][b, 0, 0], x["v"][b, 0, 1] = F.encode(-u[r]), F.encode(v[r])
    op, read, _ = bind_attend(device, mem, x, 1.0)
    op.enqueue()
    device.sync()
    p = np.exp(S.widen(q, bf16))
    want = ((v[:, None] * p - u[:, None]) / (1 + p))[..., None]
    off = 12 * 2.0 ** -24 / 1.5
    tol = off + S.half_step(q_type) * (np.abs(want) + off) + 2.0 ** -25   # (f16's smallest step)
    bad = np.abs(read() - want) > tol
    assert not bad.any(), (int(bad.sum()), bad.size)
