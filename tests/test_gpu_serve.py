"""The operators of a served batch (include/fkrocm_serve.h) on the GPU: the
page plan word for word against its definition, the paged store bit for bit
where nothing is turned, the paged attention against binary64 within a bound
derived beside the oracle (serve_cases.py).

The pools hold NaN wherever no request's position lies, outputs a sentinel
wherever nothing is written."""

import numpy as np
import pytest

import serve_cases as S
from furykernel_amd import paged

pytestmark = pytest.mark.gpu
SENTINEL = 0x7E7E7E7E


class Memory:
    """Buffers of one test, freed with it."""

    def __init__(self, device):
        self.device, self.held = device, []

    def put(self, array):
        return self.keep(self.device.upload(array))

    def empty(self, nbytes):
        return self.put(np.full(-(-max(nbytes, 4) // 4), SENTINEL, np.uint32))

    def keep(self, buf):
        self.held.append(buf)
        return buf


@pytest.fixture
def mem(device):
    m = Memory(device)
    yield m
    device.sync()
    for b in m.held:
        b.free()


# The page plan -----------------------------------------------------------------


def plan_case(seed, n, longest, chunk, block, table_len, spare_tokens=0, spare_blocks=5, head=3):
    rng = np.random.default_rng(seed)
    cached = rng.integers(0, longest + 1, n)
    fresh = np.where(rng.random(n) < 0.3, rng.integers(0, chunk + 1, n), 1)
    held, need = -(-cached // block), -(-(cached + fresh) // block) - -(-cached // block)
    order = rng.permutation(int(held.sum() + need.sum()) + head + max(spare_blocks, 0) + 1)
    table = rng.integers(0, 1 << 32, (n, table_len), dtype=np.uint64).astype(np.uint32)  # entries past: anything
    at = 0
    for r in range(n):
        k = min(held[r], table_len)
        table[r, :k] = order[at:at + k]
        at += held[r]
    free = order[at:at + head + int(need.sum()) + spare_blocks]
    return dict(cached=cached.astype(np.uint32), fresh=fresh.astype(np.uint32), free=free.astype(np.uint32),
                head=head, table=table, tokens=max(0, int(fresh.sum()) + spare_tokens), block=block)


def run_plan(device, mem, x):
    n, tokens, table_len = len(x["cached"]), x["tokens"], x["table"].shape[1]
    free = x["free"] if len(x["free"]) else np.zeros(1, np.uint32)
    bufs = {"cached": mem.put(x["cached"]), "fresh": mem.put(x["fresh"]), "free": mem.put(free),
            "head": mem.put(np.array([x["head"]], np.uint32)), "table": mem.put(x["table"])}
    sizes = {"lengths": n, "starts": n + 1, "slots": tokens, "positions": tokens, "owner": tokens, "counts": 4}
    # a word more than the call may write, each
    outs = {k: mem.empty(4 * (c + 1)) for k, c in sizes.items()}
    op = paged.PagePlan(device, **bufs, **outs, requests=n, tokens=tokens, table_len=table_len, block_size=x["block"],
                        free_len=len(x["free"]))
    op.enqueue()
    device.sync()
    got = {k: outs[k].read(np.uint32) for k in sizes}
    for k, c in sizes.items():
        assert got[k][c] == SENTINEL, f"{k} written past its end"
    return {"table": bufs["table"].read(np.uint32).reshape(n, table_len), **{k: got[k][:c] for k, c in sizes.items()}}


def hold_plan(device, mem, x):
    want = S.plan(x["cached"], x["fresh"], x["free"], x["head"], x["table"], x["tokens"], x["block"])
    got = run_plan(device, mem, x)
    for k in want:
        assert np.array_equal(got[k], want[k]), (k, np.flatnonzero(got[k].ravel() != want[k].ravel())[:8])
    return want


@pytest.mark.parametrize("n,longest,chunk,block,spare", [
    (1, 0, 1, 16, 0), (1, 0, 1, 1, 3), (1, 5000, 3000, 16, 100), (2, 31, 33, 16, 0), (63, 40, 9, 7, 5),
    (256, 300, 1, 16, 0), (257, 60, 4, 5, 3), (512, 60, 4, 5, 0), (513, 60, 4, 11, 9),
    (1000, 100, 40, 24, 17), (1023, 9, 3, 1, 0), (1024, 50, 20, 8, 1), (1025, 50, 20, 128, 2), (2048, 40, 5, 3, 0),
    (2049, 40, 5, 3, 70), (1500, 700, 80, 16, 777), (3001, 30, 7, 16, 999), (20000, 20, 12, 16, 50)])
def test_plan_is_its_definition(device, mem, n, longest, chunk, block, spare):
    print(f"plan {n} {longest} {chunk} {block} {spare}", flush=True)
    x = plan_case(n + block, n, longest, chunk, block, -(-(longest + chunk) // block) + 1, spare)
    want = hold_plan(device, mem, x)
    assert want["counts"][2] == 0 and want["counts"][0] == x["fresh"].sum()


@pytest.mark.parametrize("why,over", [
    ("blocks", dict(spare_blocks=-9)), ("no blocks", dict(spare_blocks=-10 ** 6)), ("table", dict(table_len=2)),
    ("tokens", dict(spare_tokens=-30)), ("no tokens", dict(spare_tokens=-10 ** 6)),
    ("all", dict(spare_blocks=-30, table_len=3, spare_tokens=-100))])
@pytest.mark.parametrize("n", [150, 300, 700, 1500, 2500])
def test_plan_refuses_requests_that_do_not_fit(device, mem, why, over, n):
    x = plan_case(5, n, 60, 30, 16, **{"table_len": 7, **over})
    if why == "no blocks":
        x["free"] = x["free"][:2]     # fewer than are taken already
    want = hold_plan(device, mem, x)
    assert 0 < want["counts"][2] <= n


@pytest.mark.parametrize("n", [40, 400, 1000, 2000, 2500])
def test_plan_of_lengths_that_are_nonsense(device, mem, n):
    x = plan_case(6, n, 60, 30, 16, 7)
    rng = np.random.default_rng(1)
    for name in ("cached", "fresh"):
        x[name][rng.integers(0, n, 5)] = rng.choice([0xFFFFFFFF, 0x80000000, 113], 5)
    x["table"][:, :3] = 0xFFFFFFF0    # slots past 32 bits are no slots
    hold_plan(device, mem, x)


@pytest.mark.parametrize("n", [40, 400, 1000, 2000, 3000])
def test_plan_of_a_free_list_taken_past_its_end(device, mem, n):
    """No block is left; requests whose pages hold their new tokens go on."""
    x = plan_case(8, n, 60, 3, 16, 7)
    x["head"] = 0xFFFFFFFF
    want = hold_plan(device, mem, x)
    assert 0 < want["counts"][2] < n and np.any(want["slots"] != S.NO_SLOT)


@pytest.mark.parametrize("block", [1, 2, 3, 5, 7, 11, 16, 24, 100, 641, 1000, 4095, 65537])
def test_plan_of_blocks_of_any_size(device, mem, block):
    x = plan_case(9, 70, 9000, 3, block, -(-9003 // block) + 1, 5)
    hold_plan(device, mem, x)


def test_plan_of_nothing(device, mem):
    x = plan_case(7, 5, 60, 0, 16, 7)
    x["fresh"][:] = 0
    x["tokens"] = 0
    assert hold_plan(device, mem, x)["counts"].tolist() == [0, 0, 0, 3]


# The paged store -----------------------------------------------------------------


def run_store(device, mem, rng, tokens, heads, kv, d, block, rows_type, cache, rotated, queries=True, pad=0):
    """(got, want, the values' size) of qr and the pools: [tokens or slots, heads, d]."""
    blocks = -(-tokens // block) + 2
    slots = rng.permutation(blocks * block)[:tokens].astype(np.uint32)
    slots[rng.random(tokens) < 0.1] = S.NO_SLOT
    if tokens > 3:
        slots[1] = blocks * block         # the first slot past the pool
    rope_rows = 50
    positions = rng.integers(0, rope_rows + 20, tokens).astype(np.uint32)
    angle = rng.uniform(-4, 4, (rope_rows, max(rotated, 1)))
    cs = np.stack([np.cos(angle), np.sin(angle)], -1).astype(np.float32)
    width = (heads + 2 * kv) * d + pad
    rows = rng.standard_normal((tokens, width)).astype(np.float32)
    bf16 = cache == "bf16"
    if rows_type == "f32":
        held, values = rows, rows.astype(np.float64)
    else:
        held = S.narrow(rows, rows_type == "bf16")
        values = S.widen(held, rows_type == "bf16")
    fused = mem.put(held)
    qr = mem.empty(2 * tokens * heads * d)
    pools = [mem.empty(2 * blocks * block * kv * d) for _ in range(2)]
    kw = dict(q=fused, qr=qr, heads=heads, q_stride=width) if queries else dict(heads=0)
    op = paged.PagedStore(device, k=fused, v=fused, k_offset=heads * d, v_offset=(heads + kv) * d, k_stride=width,
                          v_stride=width, slots=mem.put(slots), positions=mem.put(positions), rope=mem.put(cs),
                          rope_rows=rope_rows, rotated=rotated, kpool=pools[0], vpool=pools[1], tokens=tokens,
                          kv_heads=kv, head_dim=d, block_size=block, blocks=blocks, rows_type=rows_type, cache=cache,
                          **kw)
    op.enqueue()
    device.sync()
    got = [qr.read(np.uint16, tokens * heads * d).reshape(tokens, heads, d)]
    for p in pools:
        p = p.read(np.uint16, blocks * block * kv * d).reshape(blocks, kv, block, d)
        got.append(p.transpose(0, 2, 1, 3).reshape(blocks * block, kv, d))
    q, k, v = (values[:, a:b].reshape(tokens, -1, d) for a, b in
               ((0, heads * d), (heads * d, (heads + kv) * d), ((heads + kv) * d, (heads + 2 * kv) * d)))
    turn = cs[np.minimum(positions, rope_rows - 1)]
    live = slots < blocks * block
    untouched = np.uint16(SENTINEL & 0xFFFF)
    want = []
    for got_x, x, size, where in ((got[0], q, tokens, np.arange(tokens)), (got[1], k, blocks * block, slots),
                                  (got[2], v, blocks * block, slots)):
        full = np.full(got_x.shape, np.nan)
        if not (x is q and not queries):
            full[where[live]] = (x if x is v else S.rope(x, turn, rotated))[live]
        want.append(full)
        assert np.all(got_x[np.isnan(full)] == untouched), "a row without a slot was written"
    return got, want, bf16


@pytest.mark.parametrize("tokens,heads,kv,d,block", [(1, 4, 4, 16, 16), (7, 8, 2, 64, 7), (41, 3, 1, 80, 1),
                                                     (130, 6, 2, 128, 24), (9, 2, 2, 256, 64)])
@pytest.mark.parametrize("rows_type,cache", [("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16"),
                                             ("f16", "bf16"), ("bf16", "f16")])
def test_store_rounds_each_element_once(device, mem, tokens, heads, kv, d, block, rows_type, cache):
    """Elements that nothing turns are the value's own nearest, bit for bit;
    a turned one is two products and a difference in binary32, each a half
    step of 2^-24 (of the products' sizes, at most |x| + |y|), then one
    rounding."""
    rng = np.random.default_rng(tokens + d)
    for rotated, pad in ((0, 0), (d // 2, 16), (d // 4 - 1, 8)):
        print(f"store {tokens} {heads} {kv} {d} {block} {rows_type} {cache} {rotated}", flush=True)
        got, want, bf16 = run_store(device, mem, rng, tokens, heads, kv, d, block, rows_type, cache, rotated, pad=pad)
        for g, w, turned in zip(got, want, (rotated, rotated, 0)):
            there = ~np.isnan(w)
            still = there.copy()
            still[..., :turned] = False
            still[..., d // 2:d // 2 + turned] = False
            assert np.array_equal(g[still], S.narrow(w[still].astype(np.float32), bf16))
            err = np.abs(S.widen(g, bf16)[there] - w[there])
            least = 2.0 ** -25 if not bf16 else 2.0 ** -130   # half f16's smallest step
            assert np.all(err <= S.half_step(cache) * np.abs(w[there]) * (1 + 2.0 ** -10) + 3 * 2.0 ** -24 * 10 + least)


def test_store_without_queries_and_of_no_tokens(device, mem):
    rng = np.random.default_rng(4)
    got, want, _ = run_store(device, mem, rng, 33, 4, 2, 64, 16, "f32", "f16", 32, queries=False)
    assert np.isnan(want[0]).all()
    b = mem.empty(4096)
    paged.PagedStore(device, k=b, v=b, slots=b, kpool=mem.empty(4096), vpool=mem.empty(4096), tokens=0, kv_heads=1,
                     head_dim=16, block_size=16, blocks=4).enqueue()
    device.sync()


# The paged attention ----------------------------------------------------------------


def attend_inputs(rng, lengths, heads, kv, d, block, cache, spare=3, table_len=None, size=1.0):
    n, bf16 = len(lengths), cache == "bf16"
    pages = [-(-int(x) // block) for x in lengths]
    table_len = max(1, *pages) if table_len is None else table_len
    blocks = sum(pages) + spare
    order = rng.permutation(blocks)
    table = rng.integers(0, 1 << 32, (n, table_len), dtype=np.uint64).astype(np.uint32)  # behind a length: anything
    nan = np.uint16(0x7FC1 if bf16 else 0x7E01)
    pools = [np.full((blocks, kv, block, d), nan, np.uint16) for _ in range(2)]
    at = 0
    for r, length in enumerate(lengths):
        mine = order[at:at + pages[r]]
        at += pages[r]
        table[r, :pages[r]] = mine
        for i, b in enumerate(mine):
            live = min(block, int(length) - i * block)
            for p in pools:
                p[b, :, :live] = S.narrow(rng.standard_normal((kv, live, d)) * size, bf16)
    q = S.narrow(rng.standard_normal((n, heads, d)), bf16)
    return dict(q=q, k=pools[0], v=pools[1], table=table, lengths=np.asarray(lengths, np.uint32), block=block,
                heads=heads, kv=kv, d=d, cache=cache)


def bind_attend(device, mem, x, scale, window=0, out_type=None, q_pad=0, out_pad=0, bufs=None):
    n, w = len(x["lengths"]), x["heads"] * x["d"]
    wide = np.uint32 if out_type == "f32" else np.uint16
    if bufs is None:
        q = np.full((n, w + q_pad), 0x7FC1, np.uint16)
        q[:, :w] = x["q"].reshape(n, w)
        bufs = dict(q=mem.put(q), kpool=mem.put(x["k"]), vpool=mem.put(x["v"]), table=mem.put(x["table"]),
                    lengths=mem.put(x["lengths"]))
    sizes = dict(requests=n, heads=x["heads"], kv_heads=x["kv"], head_dim=x["d"], block_size=x["block"],
                 blocks=x["k"].shape[0], table_len=x["table"].shape[1], window=window)
    out = mem.empty(n * (w + out_pad) * np.dtype(wide).itemsize)
    workspace = mem.empty(paged.attend_workspace(**sizes) + 64)
    op = paged.PagedAttend(device, **bufs, out=out, workspace=workspace, scale=scale, cache=x["cache"],
                           out_type=out_type, q_stride=w + q_pad, out_stride=w + out_pad, **sizes)

    def read():
        bits = out.read(wide, n * (w + out_pad)).reshape(n, w + out_pad)
        if out_pad:
            assert np.all(bits[:-1, w:] == wide(SENTINEL & np.iinfo(wide).max)), "written between rows"
        assert np.all(workspace.read(np.uint32)[-16:] == SENTINEL), "written past the workspace"
        bits = np.ascontiguousarray(bits[:, :w]).reshape(n, x["heads"], x["d"])
        return bits.view(np.float32).astype(np.float64) if out_type == "f32" else S.widen(bits, x["cache"] == "bf16")

    return op, read, bufs


def hold_attend(device, mem, x, scale, window=0, out_type=None, **kw):
    op, read, _ = bind_attend(device, mem, x, scale, window, out_type, **kw)
    op.enqueue()
    device.sync()
    got = read()
    bf16 = x["cache"] == "bf16"
    out, spread, reach = S.attend(*(S.widen(x[i], bf16) for i in ("q", "k", "v")), x["table"], x["lengths"], x["block"],
                                  scale, window)
    tol = S.attend_tolerance(out, spread, reach, x["lengths"], x["d"], S.half_step(out_type or x["cache"]))
    bad = ~(np.abs(got - out) <= tol)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist(), got[bad][:4], out[bad][:4], tol[bad][:4])
    empty = x["lengths"] == 0
    assert np.all(got[empty] == 0)


RAGGED = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 0, 127, 128, 129, 255, 256, 257, 300, 511, 513, 700, 0]


@pytest.mark.parametrize("cache", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv,d,block", [
    (4, 4, 64, 16), (8, 2, 64, 7), (7, 1, 64, 1), (16, 1, 128, 16), (12, 4, 128, 24), (17, 1, 128, 64),
    (40, 1, 64, 16), (2, 2, 8, 16), (4, 2, 72, 16), (6, 2, 80, 5), (8, 8, 96, 128), (3, 1, 136, 16), (4, 1, 256, 16),
    (34, 2, 256, 3), (4, 2, 64, 1000), (300, 300, 8, 16)])
def test_attend_of_ragged_requests(device, mem, heads, kv, d, block, cache):
    print(f"attend {heads} {kv} {d} {block} {cache}", flush=True)
    x = attend_inputs(np.random.default_rng(heads + d), RAGGED, heads, kv, d, block, cache)
    hold_attend(device, mem, x, d ** -0.5)


@pytest.mark.parametrize("pages", [2, 4, 8, 12, 16, 17, 24, 32, 40, 48, 49, 64, 65, 80, 96, 97, 100])
@pytest.mark.parametrize("d,kv", [(64, 2), (128, 1), (256, 2), (64, 64), (64, 16), (128, 16), (128, 50)])
def test_attend_of_tables_of_every_length(device, mem, pages, d, kv):
    """Tables of few units go whole to the threadgroups, longer ones split:
    each side of each rule, the lengths short and up to the table's."""
    print(f"attend table {pages} {d} {kv}", flush=True)
    top = pages * 16
    lengths = [x for x in (0, 1, 33, top // 2, top - 1, top, 17) if x <= top]
    x = attend_inputs(np.random.default_rng(pages), lengths, 2 * kv, kv, d, 16, "bf16", table_len=pages)
    hold_attend(device, mem, x, d ** -0.5)
    hold_attend(device, mem, x, d ** -0.5, window=40)


@pytest.mark.parametrize("window", [1, 7, 64, 100, 256, 5000])
@pytest.mark.parametrize("d,block", [(64, 16), (128, 24), (256, 16)])
def test_attend_in_a_window(device, mem, window, d, block):
    print(f"attend window {window} {d} {block}", flush=True)
    x = attend_inputs(np.random.default_rng(window), RAGGED, 6, 2, d, block, "f16")
    hold_attend(device, mem, x, d ** -0.5, window=window)


@pytest.mark.parametrize("lengths", [[1], [20000], [9000, 1, 0, 4000], [3000] * 70, [5] * 900, [0, 0], [0] * 600 + [3]])
@pytest.mark.parametrize("d,cache", [(64, "bf16"), (128, "f16"), (256, "bf16")])
def test_attend_of_batches(device, mem, lengths, d, cache):
    """One long request over many threadgroups, a few, more than there are
    threadgroups, more requests than threads, none with a key."""
    print(f"attend batch {len(lengths)} {max(lengths)} {d} {cache}", flush=True)
    x = attend_inputs(np.random.default_rng(len(lengths)), lengths, 4, 2, d, 16, cache)
    hold_attend(device, mem, x, d ** -0.5)


def test_attend_of_one_request_with_many_heads(device, mem):
    """More (request, kv head) pairs than threads, split, whole and empty."""
    for lengths, table_len in (([2000], 125), ([0], 125), ([90], 6)):
        print(f"attend many heads {lengths}", flush=True)
        x = attend_inputs(np.random.default_rng(5), lengths, 300, 300, 16, 16, "bf16", table_len=table_len)
        hold_attend(device, mem, x, 0.25)


def test_attend_rows_apart_and_f32_out(device, mem):
    for d, heads, cache in ((64, 6, "f16"), (128, 4, "bf16"), (80, 2, "f16")):
        print(f"attend rows apart {d}", flush=True)
        x = attend_inputs(np.random.default_rng(d), RAGGED[:20], heads, 2, d, 16, cache)
        hold_attend(device, mem, x, d ** -0.5, out_type="f32", q_pad=24, out_pad=5)
        hold_attend(device, mem, x, d ** -0.5, q_pad=8, out_pad=3)


def test_attend_large_and_small_scores(device, mem):
    """Scores far apart (one key takes all), all alike, and of scale 0 and below."""
    for size, scale in ((30.0, 0.125), (1.0, 0.0), (1.0, -0.125), (1e-3, 1.0)):
        print(f"attend scores {size} {scale}", flush=True)
        x = attend_inputs(np.random.default_rng(3), RAGGED, 4, 2, 64, 16, "f16", size=size)
        hold_attend(device, mem, x, scale)


def test_attend_lengths_past_the_table_and_blocks_past_the_pool(device, mem):
    x = attend_inputs(np.random.default_rng(8), [40, 64, 33], 4, 2, 64, 16, "f16", table_len=4)
    x["k"][:], x["v"][:] = (S.narrow(np.random.default_rng(i).standard_normal(x["k"].shape), False) for i in (1, 2))
    x["table"][0, 3] = 0
    x["table"][2, 2] = 0xFFFFFFFF            # a block past the pool: its last
    x["lengths"] = np.array([0xFFFFFFFF, 65, 48], np.uint32)
    x["table"][0, 2:] = x["table"][0, :2]
    hold_attend(device, mem, x, 0.125)


def test_attend_values_that_are_not_finite(device, mem):
    """A request's own infinity or NaN reaches its own outputs, as the formula
    has it, and no other's."""
    x = attend_inputs(np.random.default_rng(9), [100, 70, 130], 4, 2, 64, 16, "f16")
    inf, nan = 0x7C00, 0x7E00
    x["v"][x["table"][0, 1], 0, 3, 5] = inf          # request 0, kv head 0, position 19, element 5
    x["k"][x["table"][2, 4], 1, 1, 7] = nan          # request 2, kv head 1
    op, read, _ = bind_attend(device, mem, x, 0.125)
    op.enqueue()
    device.sync()
    got = read()
    assert np.isinf(got[0, :2, 5]).all() and np.isnan(got[2, 2:]).all()
    got[0, :2, 5], got[2, 2:] = 0, 0
    assert np.isfinite(got).all()


def test_attend_past_4_gib_of_pool(device, mem):
    """Blocks whose bytes lie past 32 bits of offset."""
    kv, d, block, blocks = 8, 128, 64, 40000           # 5.2 GB a pool
    x = attend_inputs(np.random.default_rng(10), [150, 64], 16, kv, d, block, "f16")
    far = np.array([39999, 33000, 1, 39000, 2, 3, 4, 5], np.uint32)[:x["k"].shape[0]]
    bufs = {}
    bytes_of = kv * block * d * 2
    for name, src in (("kpool", "k"), ("vpool", "v")):
        bufs[name] = mem.keep(device.alloc(blocks * bytes_of))
        for i, b in enumerate(far):
            bufs[name].write(x[src][i], offset=int(b) * bytes_of)
    want = dict(x)
    live = x["table"] < len(far)
    table = np.where(live, far[np.minimum(x["table"], len(far) - 1)], 0).astype(np.uint32)
    bufs.update(q=mem.put(x["q"]), table=mem.put(table), lengths=mem.put(x["lengths"]))
    n, w = 2, 16 * d
    sizes = dict(requests=n, heads=16, kv_heads=kv, head_dim=d, block_size=block, blocks=blocks,
                 table_len=table.shape[1])
    out = mem.empty(n * w * 2)
    paged.PagedAttend(device, **bufs, out=out, workspace=mem.empty(paged.attend_workspace(**sizes)), scale=0.1,
                      **sizes).enqueue()
    device.sync()
    got = S.widen(out.read(np.uint16, n * w).reshape(n, 16, d), False)
    o, spread, reach = S.attend(*(S.widen(want[i], False) for i in ("q", "k", "v")), want["table"], want["lengths"],
                                block, 0.1)
    assert np.all(np.abs(got - o) <= S.attend_tolerance(o, spread, reach, want["lengths"], d, 2.0 ** -11))


def test_attend_gives_the_same_bits_again_and_on_other_streams(device, mem):
    x = attend_inputs(np.random.default_rng(11), [3000, 5, 900, 0, 7000], 8, 2, 128, 16, "bf16")
    op, read, bufs = bind_attend(device, mem, x, 0.09)
    other, read_other, _ = bind_attend(device, mem, x, 0.09, bufs=bufs)
    op.enqueue()
    device.sync()
    first = read()
    streams = [device.new_stream(), device.new_stream()]
    for _ in range(5):
        op.enqueue(streams[0])
        other.enqueue(streams[1])
    for s in streams:
        device.sync(s)
    assert np.array_equal(read(), first) and np.array_equal(read_other(), first)


def test_attend_takes_queries_by_a_plans_starts(device, mem):
    """A request's last token's row; requests without one, or with tokens past
    the rows there are, count as empty."""
    x = attend_inputs(np.random.default_rng(13), [100, 300, 65, 7, 33, 90], 4, 2, 64, 16, "f16")
    starts = np.array([0, 1, 1, 4, 4, 6, 9], np.uint32)
    rows = S.narrow(np.random.default_rng(14).standard_normal((6, 4, 64)), False)
    lengths = np.where((np.diff(starts.astype(int)) > 0) & (starts[1:] <= 6), x["lengths"], 0)
    n, w = 6, 256
    sizes = dict(requests=n, heads=4, kv_heads=2, head_dim=64, block_size=16, blocks=x["k"].shape[0],
                 table_len=x["table"].shape[1])
    out = mem.empty(n * w * 2)
    paged.PagedAttend(device, q=mem.put(rows), kpool=mem.put(x["k"]), vpool=mem.put(x["v"]),
                      table=mem.put(x["table"]), lengths=mem.put(x["lengths"]), starts=mem.put(starts), q_rows=6,
                      out=out, workspace=mem.empty(paged.attend_workspace(**sizes)), scale=0.125, **sizes).enqueue()
    device.sync()
    got = S.widen(out.read(np.uint16, n * w).reshape(n, 4, 64), False)
    q = S.widen(rows[np.minimum(starts[1:].astype(int) - 1, 5)], False)
    o, spread, reach = S.attend(q, S.widen(x["k"], False), S.widen(x["v"], False), x["table"], lengths, 16, 0.125)
    assert np.all(np.abs(got - o) <= S.attend_tolerance(o, spread, reach, lengths, 64, 2.0 ** -11))
    assert np.all(got[lengths == 0] == 0) and np.sum(lengths == 0) == 3


def test_index_arrays_a_word_off(device, mem):
    """Tables, lengths, starts, slots and positions at any word of a buffer:
    the same bits as from its start."""
    def shifted(array):
        return mem.put(np.concatenate([np.uint32([0xDEADBEEF]), np.ravel(array), np.uint32([0xDEADBEEF])]))

    x = attend_inputs(np.random.default_rng(15), [40, 500, 1, 77], 8, 2, 64, 16, "f16")
    starts = np.arange(5, dtype=np.uint32)
    op, read, _ = bind_attend(device, mem, x, 0.1)
    op.enqueue()
    device.sync()
    want = read()
    for name, array in (("table", x["table"]), ("lengths", x["lengths"]), ("starts", starts)):
        setattr(op.args, name, shifted(array).ptr + 4)
    op.args.q_rows = 4
    op.enqueue()
    device.sync()
    assert np.array_equal(read(), want)

    rng = np.random.default_rng(16)
    tokens, d = 5, 16
    slots, positions = np.uint32([3, 9, 0, 30, 7]), np.uint32([1, 0, 4, 2, 2])
    rows, cs = mem.put(rng.standard_normal((2, tokens, d)).astype(np.float32)), rng.standard_normal((5, 8, 2))
    got = []
    for put, off in ((mem.put, 0), (shifted, 4)):
        pools = [mem.empty(2 * 32 * d) for _ in range(2)]
        op = paged.PagedStore(device, k=rows, v=rows, v_offset=tokens * d, slots=put(slots), positions=put(positions),
                              rope=mem.put(cs.astype(np.float32)), rope_rows=5, rotated=8, kpool=pools[0],
                              vpool=pools[1], tokens=tokens, kv_heads=1, head_dim=d, block_size=16, blocks=2)
        op.args.slots += off
        op.args.positions += off
        op.enqueue()
        device.sync()
        got.append([p.read(np.uint16).copy() for p in pools])
    assert all(np.array_equal(p, q) for p, q in zip(*got))


# A step of them together ------------------------------------------------------------


@pytest.mark.parametrize("cache,d,block", [("f16", 64, 16), ("bf16", 128, 24)])
def test_a_captured_step_serves_requests_that_grow(device, mem, cache, d, block):
    """Plan, store and attend captured once and replayed for six steps, the
    host changing the new rows between: every replay's plan, caches and rows
    those of the definitions, over requests that grow through their pages."""
    rng = np.random.default_rng(12)
    bf16 = cache == "bf16"
    n, heads, kv, tokens, table_len = 5, 4, 2, 7, 12
    cached = np.array([0, block - 2, 3 * block, 100, 5], np.uint32)
    blocks = 60
    order = rng.permutation(blocks).astype(np.uint32)
    table = np.zeros((n, table_len), np.uint32)
    at = 0
    for r in range(n):
        held = -(-int(cached[r]) // block)
        table[r, :held] = order[at:at + held]
        at += held
    free = order[at:]
    hist = [[S.widen(S.narrow(rng.standard_normal((int(c), kv, d)), bf16), bf16) for c in cached] for _ in range(2)]
    pools = [np.full((blocks, kv, block, d), 0x7FC1, np.uint16) for _ in range(2)]
    for p, h in zip(pools, hist):
        for r in range(n):
            for i in range(int(cached[r])):
                p[table[r, i // block], :, i % block] = S.narrow(h[r][i], bf16)
    angle = rng.uniform(-4, 4, (table_len * block, d // 2))
    cs = np.stack([np.cos(angle), np.sin(angle)], -1).astype(np.float32)
    width = (heads + 2 * kv) * d
    b = dict(cached=mem.put(cached), fresh=mem.put(np.ones(n, np.uint32)), free=mem.put(free),
             head=mem.put(np.zeros(1, np.uint32)), table=mem.put(table), lengths=mem.empty(4 * n),
             starts=mem.empty(4 * n + 4), slots=mem.empty(4 * tokens), positions=mem.empty(4 * tokens),
             owner=mem.empty(4 * tokens), counts=mem.put(np.zeros(4, np.uint32)))
    rows, qr = mem.empty(4 * tokens * width), mem.empty(2 * tokens * heads * d)
    out = mem.empty(2 * n * heads * d)
    kpool, vpool = (mem.put(p) for p in pools)
    sizes = dict(requests=n, heads=heads, kv_heads=kv, head_dim=d, block_size=block, blocks=blocks, table_len=table_len)
    ops = [paged.PagePlan(device, **b, requests=n, tokens=tokens, table_len=table_len, block_size=block,
                          free_len=len(free)),
           paged.PagedStore(device, q=rows, k=rows, v=rows, k_offset=heads * d, v_offset=(heads + kv) * d,
                            q_stride=width, k_stride=width, v_stride=width, slots=b["slots"],
                            positions=b["positions"], rope=mem.put(cs), rope_rows=table_len * block, rotated=d // 2,
                            qr=qr, kpool=kpool, vpool=vpool, tokens=tokens, heads=heads, kv_heads=kv, head_dim=d,
                            block_size=block, blocks=blocks, rows_type="f32", cache=cache),
           paged.PagedAttend(device, q=qr, kpool=kpool, vpool=vpool, table=b["table"], lengths=b["lengths"], out=out,
                             workspace=mem.empty(paged.attend_workspace(**sizes)), scale=d ** -0.5, cache=cache,
                             starts=b["starts"], q_rows=tokens, **sizes)]
    stream = device.new_stream()
    with device.capture(stream) as captured:
        for op in ops:
            op.enqueue(stream)
        b["cached"].copy_from(b["lengths"], 4 * n, stream=stream)
        b["head"].copy_from(b["counts"], 4, src_offset=12, stream=stream)
    graph = captured[0]
    head = 0
    for step in range(6):
        fresh = np.ones(n, np.uint32)
        fresh[step % n] = step % 3                   # a request rests, another brings two tokens
        x = rng.standard_normal((tokens, width)).astype(np.float32)
        rows.write(x)
        b["fresh"].write(fresh)
        graph.replay(stream)
        device.sync(stream)
        want = S.plan(cached, fresh, free, head, table, tokens, block)
        for k in ("lengths", "starts", "slots", "positions", "owner", "counts"):
            assert np.array_equal(b[k].read(np.uint32, want[k].size), want[k]), (step, k)
        table, head = want["table"], int(want["counts"][3])
        assert np.array_equal(b["table"].read(np.uint32).reshape(n, -1), table)
        turn = cs[want["positions"]]
        q, k, v = (x[:, i:j].reshape(tokens, -1, d) for i, j in
                   ((0, heads * d), (heads * d, (heads + kv) * d), ((heads + kv) * d, width)))
        q, k = (S.rope(t, turn, d // 2) for t in (q, k))
        stored = [p.read(np.uint16, blocks * kv * block * d).reshape(blocks, kv, block, d) for p in (kpool, vpool)]
        half = S.half_step(cache)
        for t in range(int(want["counts"][0])):
            at, within = divmod(int(want["slots"][t]), block)
            for p, made in zip(stored, (k[t], v[t].astype(np.float64))):
                assert np.all(np.abs(S.widen(p[at, :, within], bf16) - made) <= half * np.abs(made) + 2.0 ** -20)
        # the attention of the rows and caches as stored: a request's last
        # token's, nothing of one that rests
        qs = S.widen(qr.read(np.uint16, tokens * heads * d).reshape(tokens, heads, d), bf16)
        seen = np.where(fresh > 0, want["lengths"], 0)
        o, spread, reach = S.attend(qs[np.maximum(want["starts"][1:].astype(int) - 1, 0)], S.widen(stored[0], bf16),
                                    S.widen(stored[1], bf16), table, seen, block, d ** -0.5)
        got = S.widen(out.read(np.uint16, n * heads * d).reshape(n, heads, d), bf16)
        tol = S.attend_tolerance(o, spread, reach, want["lengths"], d, half)
        bad = ~(np.abs(got - o) <= tol)
        assert not bad.any(), (step, int(bad.sum()), np.argwhere(bad)[:4].tolist())
        cached = want["lengths"]
        device.sync()
    graph.destroy()
