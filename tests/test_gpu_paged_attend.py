"""The paged attention (include/fkrocm_serve.h: fk_paged_attend) on the GPU
at the edges of its numbers: the bits its probabilities keep, infinities of
unlikely keys, large values; and where its keys are split over threadgroups,
with a plan's starts, in windows, and captured."""

import numpy as np
import pytest

import serve_cases as S
from furykernel_amd import paged
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
@pytest.mark.parametrize("d,lengths,table_len,block", [
    (64, [90, 40], 6, 16), (128, [90, 40], 6, 16), (256, [30, 17], 4, 16), (80, [90, 40], 6, 16),
    (64, [5000, 300], 320, 16), (128, [5000, 9], 320, 16), (256, [3000, 5], 200, 16), (200, [3000, 64], 200, 16),
    (64, [700, 40], 700, 1), (128, [500, 3], 500, 1), (64, [2000, 40], 2000, 1), (128, [5000, 40], 2, 2500)])
def test_infinite_values_of_unlikely_keys(device, mem, d, lengths, table_len, block, cache):
    """An infinite value gives infinity whatever its key's weight: any finite
    score's is above 0.  A key of score -infinity has a weight of 0, and 0
    times infinity is no number; both infinities in one element are none
    either.  Elsewhere the finite values' attention, within its bound."""
    print(f"attend infinities {d} {lengths} {block} {cache}", flush=True)
    bf16 = cache == "bf16"
    rng = np.random.default_rng(d + len(lengths))
    x = attend_inputs(rng, lengths, 2, 1, d, block, cache, table_len=table_len)
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
        out, spread, reach = S.attend(*wide.values(), x["table"], x["lengths"], block, 1.0)
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


# The attention whose keys are split over threadgroups and joined --------------------


def sizes_of(x, window=0):
    return dict(requests=len(x["lengths"]), heads=x["heads"], kv_heads=x["kv"], head_dim=x["d"],
                block_size=x["block"], blocks=x["k"].shape[0], table_len=x["table"].shape[1], window=window)


@pytest.mark.parametrize("d,cache", [(64, "f16"), (128, "bf16"), (256, "f16")])
@pytest.mark.parametrize("lengths,kv", [([3000, 0, 9000, 5, 700, 64, 2048], 2), ([1], 1),
                                        ([40, 0, 300, 7, 2100, 90] * 60, 2)])
def test_split_attention_takes_queries_by_a_plans_starts(device, mem, d, cache, lengths, kv):
    """As the whole one: a request's last token's row, nothing of a request
    without one or with tokens past the rows there are; pairs fewer and more
    than the threadgroups, twice into one workspace with other requests empty."""
    print(f"attend split starts {len(lengths)} {kv} {d} {cache}", flush=True)
    bf16, n, heads = cache == "bf16", len(lengths), 3 * kv
    rng = np.random.default_rng(n + d)
    x = attend_inputs(rng, lengths, heads, kv, d, 16, cache, table_len=max(130, -(-max(lengths) // 16)))
    sizes = sizes_of(x)
    assert paged.attend_form(**sizes) == "split"
    w, q_rows = heads * d, 2 * n
    rows = S.narrow(rng.standard_normal((q_rows, heads, d)), bf16)
    starts, out = mem.empty(4 * n + 4), mem.empty(2 * n * w)
    op = paged.PagedAttend(device, q=mem.put(rows), kpool=mem.put(x["k"]), vpool=mem.put(x["v"]),
                           table=mem.put(x["table"]), lengths=mem.put(x["lengths"]), starts=starts, q_rows=q_rows,
                           out=out, workspace=mem.empty(paged.attend_workspace(**sizes)), scale=d ** -0.5, cache=cache,
                           **sizes)
    wide = [S.widen(x[i], bf16) for i in ("k", "v")]
    for turn in range(2):
        fresh = rng.integers(0, 4, n)
        fresh[0] = turn + 1 if n > 1 else 1
        begin = np.concatenate([[0], fresh.cumsum()])
        if n > 1:
            begin[-1] = max(begin[-1], q_rows + 3)      # the last one's tokens end past the rows
        starts.write(begin.astype(np.uint32))
        op.enqueue()
        device.sync()
        seen = np.where((np.diff(begin) > 0) & (begin[1:] <= q_rows), x["lengths"], 0)
        q = S.widen(rows[np.clip(begin[1:] - 1, 0, q_rows - 1)], bf16)
        o, spread, reach = S.attend(q, *wide, x["table"], seen, 16, d ** -0.5)
        got = S.widen(out.read(np.uint16, n * w).reshape(n, heads, d), bf16)
        tol = S.attend_tolerance(o, spread, reach, seen, d, S.half_step(cache))
        bad = ~(np.abs(got - o) <= tol)
        assert not bad.any(), (turn, int(bad.sum()), np.argwhere(bad)[:4].tolist())
        assert np.all(got[seen == 0] == 0) and (n == 1 or (seen == 0).sum() > 1)


@pytest.mark.parametrize("window", [1500, 2049, 3000])
@pytest.mark.parametrize("d,block,cache", [(64, 16, "bf16"), (128, 24, "f16"), (256, 16, "bf16"), (72, 7, "f16")])
def test_split_attention_in_a_window(device, mem, window, d, block, cache):
    print(f"attend split window {window} {d} {block} {cache}", flush=True)
    lengths = [3000, 0, 9000, 5, window, window + 1, 1, 6000]
    x = attend_inputs(np.random.default_rng(window), lengths, 6, 2, d, block, cache)
    assert paged.attend_form(**sizes_of(x, window)) == "split"
    hold_attend(device, mem, x, d ** -0.5, window=window)


@pytest.mark.parametrize("heads,kv,d,block,cache", [(40, 2, 64, 16, "f16"), (17, 1, 128, 16, "bf16"),
                                                    (33, 1, 256, 24, "f16"), (6, 2, 64, 4096, "bf16"),
                                                    (48, 3, 72, 1, "bf16"), (512, 16, 64, 16, "f16")])
@pytest.mark.parametrize("lengths", [[9000, 0, 5, 700, 2500], [3000]])
def test_split_attention_of_many_heads_a_kv_head(device, mem, heads, kv, d, block, cache, lengths):
    """Groups of more than 16 query heads, the last ones few; large blocks and
    ones of a position."""
    print(f"attend split heads {heads} {kv} {d} {block} {cache} {lengths}", flush=True)
    x = attend_inputs(np.random.default_rng(heads), lengths, heads, kv, d, block, cache)
    assert paged.attend_form(**sizes_of(x)) == "split"
    hold_attend(device, mem, x, d ** -0.5)


@pytest.mark.parametrize("cache,d,block,window", [("f16", 64, 16, 0), ("bf16", 128, 24, 0), ("bf16", 64, 16, 1600)])
def test_a_captured_step_of_split_attention(device, mem, cache, d, block, window):
    """Plan, store and attend, whose two launches share a workspace, captured
    once and replayed over requests of up to 3000 positions that grow, rest and
    come in, with eager calls on the same buffers between: every replay's rows
    those of the definition over the caches as they then are."""
    rng = np.random.default_rng(21)
    bf16 = cache == "bf16"
    heads, kv, tokens = 4, 2, 9
    cached = np.array([0, 1900, block * 40, 3000, 5], np.uint32)
    n, table_len = len(cached), -(-3040 // block)
    x = attend_inputs(rng, [int(c) for c in cached], heads, kv, d, block, cache, spare=30, table_len=table_len)
    sizes = sizes_of(x, window)
    assert paged.attend_form(**sizes) == "split"
    blocks = sizes["blocks"]
    used = {int(b) for r in range(n) for b in x["table"][r, :-(-int(cached[r]) // block)]}
    free = np.array([b for b in range(blocks) if b not in used], np.uint32)
    head, table, width = 0, x["table"], (heads + 2 * kv) * d
    b = dict(cached=mem.put(cached), fresh=mem.put(np.ones(n, np.uint32)), free=mem.put(free),
             head=mem.put(np.zeros(1, np.uint32)), table=mem.put(table), lengths=mem.empty(4 * n),
             starts=mem.empty(4 * n + 4), slots=mem.empty(4 * tokens), positions=mem.empty(4 * tokens),
             owner=mem.empty(4 * tokens), counts=mem.put(np.zeros(4, np.uint32)))
    rows, qr, out = mem.empty(4 * tokens * width), mem.empty(2 * tokens * heads * d), mem.empty(2 * n * heads * d)
    kpool, vpool = mem.put(x["k"]), mem.put(x["v"])
    plan = paged.PagePlan(device, **b, requests=n, tokens=tokens, table_len=table_len, block_size=block,
                          free_len=len(free))
    store = paged.PagedStore(device, q=rows, k=rows, v=rows, k_offset=heads * d, v_offset=(heads + kv) * d,
                             q_stride=width, k_stride=width, v_stride=width, slots=b["slots"], qr=qr, kpool=kpool,
                             vpool=vpool, tokens=tokens, heads=heads, kv_heads=kv, head_dim=d, block_size=block,
                             blocks=blocks, rows_type="f32", cache=cache)
    attend = paged.PagedAttend(device, q=qr, kpool=kpool, vpool=vpool, table=b["table"], lengths=b["lengths"], out=out,
                               workspace=mem.empty(paged.attend_workspace(**sizes)), scale=d ** -0.5, cache=cache,
                               starts=b["starts"], q_rows=tokens, **sizes)
    stream = device.new_stream()
    with device.capture(stream) as captured:
        for op in (plan, store, attend):
            op.enqueue(stream)
        b["cached"].copy_from(b["lengths"], 4 * n, stream=stream)
        b["head"].copy_from(b["counts"], 4, src_offset=12, stream=stream)
    for step in range(5):
        fresh = np.ones(n, np.uint32)
        fresh[step] = step % 3                      # a request rests, another brings two tokens
        new = rng.standard_normal((tokens, width)).astype(np.float32)
        rows.write(new)
        b["fresh"].write(fresh)
        device.sync()
        captured[0].replay(stream)
        device.sync(stream)
        want = S.plan(cached, fresh, free, head, table, tokens, block)
        for k in ("lengths", "starts", "slots"):
            assert np.array_equal(b[k].read(np.uint32, want[k].size), want[k]), (step, k)
        table, head, cached = want["table"], int(want["counts"][3]), want["lengths"]
        for t in range(int(want["counts"][0])):
            at, within = divmod(int(want["slots"][t]), block)
            for pool, first in ((x["k"], heads), (x["v"], heads + kv)):
                pool[at, :, within] = S.narrow(new[t, first * d:(first + kv) * d].reshape(kv, d), bf16)
        qs = S.widen(S.narrow(new[:, :heads * d], bf16), bf16).reshape(tokens, heads, d)
        seen = np.where(fresh > 0, cached, 0)
        o, spread, reach = S.attend(qs[np.maximum(want["starts"][1:].astype(int) - 1, 0)], S.widen(x["k"], bf16),
                                    S.widen(x["v"], bf16), table, seen, block, d ** -0.5, window)
        got = out.read(np.uint16, n * heads * d)
        tol = S.attend_tolerance(o, spread, reach, cached, d, S.half_step(cache))
        bad = ~(np.abs(S.widen(got.reshape(n, heads, d), bf16) - o) <= tol)
        assert not bad.any(), (step, int(bad.sum()), np.argwhere(bad)[:4].tolist())
        out.write(np.zeros_like(got))
        attend.enqueue()
        device.sync()
        assert np.array_equal(out.read(np.uint16, n * heads * d), got)
    captured[0].destroy()
