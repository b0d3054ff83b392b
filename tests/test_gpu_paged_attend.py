"""The paged attention (include/fkrocm_serve.h: fk_paged_attend) on the GPU
at the edges of its numbers: the bits its probabilities keep, infinities of
unlikely keys."""

import numpy as np
import pytest

import serve_cases as S
from test_gpu_serve import attend_inputs, bind_attend, hold_attend, mem  # noqa: F401  (mem is a fixture)

pytestmark = pytest.mark.gpu


def position(x, r, p):
    """Where the pools hold position p of request r: (block, place in it)."""
    return x["table"][r, p // x["block"]], p % x["block"]


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("cache", ["f16", "bf16"])
def test_probabilities_keep_their_bits(device, mem, d, cache):
    """Two keys, of score 0 and value 0 and of score x in -2 .. 0 and value v,
    both exact: out = v p / (1 + p), p = e^x, in f32.  Roundings of 2^-24: the
    scale to log2 units 2 and the score 1 (of |x| at most: 6 together), the
    reference's subtraction from at most 16 log2 units 6 (half of 2^-20, times ln 2),
    the exponential 1 ulp (2); p's parts exact (bf16) or off by 2^-11 of the
    2^-10 of p that the first leaves (f16: 8); their sum 3, the sum 1 + p 1, the
    quotient 1, the result 1."""
    print(f"attend bits {d} {cache}", flush=True)
    bf16, n, heads = cache == "bf16", 300, 16
    rng = np.random.default_rng(d)
    x = attend_inputs(rng, [2] * n, heads, 1, d, 16, cache)
    x["q"][:] = 0
    x["q"][:, np.arange(heads), np.arange(heads)] = S.narrow(np.ones(heads), bf16)
    score, value = S.narrow(-2 * rng.random((n, d)), bf16), S.narrow(1 + rng.random((n, d)), bf16)
    for r in range(n):
        b = x["table"][r, 0]
        x["k"][b, 0, 0], x["v"][b, 0, 0] = 0, 0
        x["k"][b, 0, 1], x["v"][b, 0, 1] = score[r], value[r]
    op, read, _ = bind_attend(device, mem, x, 1.0, out_type="f32")
    op.enqueue()
    device.sync()
    p = np.exp(S.widen(score, bf16)[:, :heads, None])
    want = S.widen(value, bf16)[:, None] * p / (1 + p)
    err = np.abs(read() / want - 1).max()
    assert err <= (20 if bf16 else 28) * 2.0 ** -24, np.log2(err)


# Request 0's keys of chosen scores, below one of 0 by as much; past 87 a
# weight is no normal binary32, past 103 none at all.
BELOW = [0.0, 5.0, 13.5, 14.25, 17.5, 20.0, 27.0, 40.0, 60.0, 86.0, 95.0, 120.0]


@pytest.mark.parametrize("cache", ["f16", "bf16"])
@pytest.mark.parametrize("d,lengths,table_len", [(64, [90, 40], 6), (128, [90, 40], 6), (256, [30, 17], 4),
                                                 (80, [90, 40], 6), (64, [5000, 300], 320), (128, [5000, 9], 320),
                                                 (256, [3000, 5], 200), (200, [3000, 64], 200)])
def test_infinite_values_of_unlikely_keys(device, mem, d, lengths, table_len, cache):
    """An infinite value gives infinity whatever its key's weight: any finite
    score's is above 0.  A key of score -infinity has a weight of 0, and 0
    times infinity is no number; both infinities in one element are none
    either.  Elsewhere the finite values' attention, within its bound."""
    print(f"attend infinities {d} {lengths} {cache}", flush=True)
    bf16 = cache == "bf16"
    rng = np.random.default_rng(d + len(lengths))
    x = attend_inputs(rng, lengths, 2, 1, d, 16, cache, table_len=table_len)
    top = lengths[0]
    # scores from element 0 alone: -64 of every key but the chosen, which
    # lie over the whole length
    at = np.linspace(0, top - 1, len(BELOW)).round().astype(int)[::-1]
    lost = next(p for p in range(top // 2, top) if p not in at)
    assert len(set(at)) == len(BELOW)
    x["q"][0] = S.narrow(np.zeros((2, d)), bf16)
    x["q"][0, :, 0] = S.narrow(np.ones(2), bf16)
    for p in range(top):
        b, i = position(x, 0, p)
        x["k"][b, 0, i, 0] = S.narrow([-64.0], bf16)[0]
    inf = 0x7F80 if bf16 else 0x7C00
    for j, (p, below) in enumerate(zip(at, BELOW)):
        b, i = position(x, 0, p)
        x["k"][b, 0, i, 0] = S.narrow([-below], bf16)[0]
        x["v"][b, 0, i, 2 * j] = inf | (0x8000 if j % 3 == 0 else 0)
    both, none, nought = 30, 31, 33
    for p, column, bits in ((at[2], both, inf), (at[7], both, inf | 0x8000), (at[9], none, inf + 1),
                            (lost, nought, inf)):
        b, i = position(x, 0, p)
        x["v"][b, 0, i, column] = bits
    b, i = position(x, 0, lost)
    x["k"][b, 0, i, 0] = inf | 0x8000
    op, read, _ = bind_attend(device, mem, x, 1.0, out_type="f32")
    op.enqueue()
    device.sync()
    got = read()
    columns = 2 * np.arange(len(BELOW))
    want = np.where(np.arange(len(BELOW)) % 3 == 0, -np.inf, np.inf)
    assert np.array_equal(got[0][:, columns], np.broadcast_to(want, (2, len(BELOW)))), got[0][:, columns]
    assert np.isnan(got[0][:, [both, none, nought]]).all()
    rest = np.setdiff1d(np.arange(d), np.concatenate([columns, [both, none, nought]]))
    wide = {i: S.widen(x[i], bf16) for i in ("q", "k", "v")}
    b, i = position(x, 0, lost)
    wide["k"][b, 0, i, 0] = -1e5               # (the oracle's weight: 0 all the same)
    with np.errstate(invalid="ignore"):
        out, spread, reach = S.attend(*wide.values(), x["table"], x["lengths"], 16, 1.0)
    # a key's parts that would be 0 stand at 2^-39 of the largest weight (f16),
    # two of them, of values below 5
    reach = np.minimum(reach, 130.0)
    tol = S.attend_tolerance(out, spread, reach, x["lengths"], d, 2.0 ** -24) + top * 2 * 2.0 ** -39 * 5
    for r in range(2):
        cols = rest if r == 0 else np.arange(d)
        err = np.abs(got[r][:, cols] - out[r][:, cols])
        assert np.all(err <= tol[r][:, cols]), (r, err.max())


def test_rows_of_infinite_scores_and_values(device, mem):
    """A row all of whose scores are -infinity, and one with a score of
    infinity, are no numbers, with infinite values in their keys too."""
    x = attend_inputs(np.random.default_rng(4), [40, 40], 2, 1, 64, 16, "f16")
    x["q"][:] = S.narrow(np.zeros((2, 2, 64)), False)
    x["q"][:, :, 0] = S.narrow(np.ones(2), False)
    for p in range(40):
        b, i = position(x, 0, p)
        x["k"][b, 0, i, 0] = 0xFC00
    b, i = position(x, 1, 7)
    x["k"][b, 0, i, 0] = 0x7C00
    for r in range(2):
        b, i = position(x, r, 20)
        x["v"][b, 0, i, 3] = 0x7C00
    op, read, _ = bind_attend(device, mem, x, 1.0)
    op.enqueue()
    device.sync()
    assert np.isnan(read()).all()


@pytest.mark.parametrize("out_type", [None, "f32"])
@pytest.mark.parametrize("d,lengths", [(64, [1, 2, 40, 300]), (128, [1, 2, 40, 300]), (256, [1, 300, 5]),
                                       (64, [3000, 7]), (128, [3000])])
def test_values_near_the_largest_bf16(device, mem, d, lengths, out_type):
    """Values of about 2^115 (2^112 of 3000 keys): a row's weights of 1 and
    less times them add to less than 2^128, so the row is finite."""
    print(f"attend large values {d} {lengths} {out_type}", flush=True)
    x = attend_inputs(np.random.default_rng(d), lengths, 4, 2, d, 16, "bf16")
    x["v"] = S.narrow(S.widen(x["v"], True) * 2.0 ** (115 if max(lengths) < 1000 else 112), True)
    hold_attend(device, mem, x, d ** -0.5, out_type=out_type)
