"""The operators over 8-bit paged caches (include/fkrocm_paged8.h) on the GPU:
the store's codes and scales and the load's rows bit for bit, the attention
against binary64 within the bound derived beside the oracle (serve_cases.py).

Pools hold NaN wherever no request's position lies, scales NaN where no block
is held, outputs a sentinel wherever nothing is written."""

import numpy as np
import pytest

import fp8_cases as F
import serve_cases as S
from furykernel_amd import fp8, paged, paged8
from test_gpu_fp8 import matrix as mem_matrix
from test_gpu_mx4 import held
from test_gpu_serve import SENTINEL, Memory, mem  # noqa: F401  (mem is a fixture)

pytestmark = pytest.mark.gpu
NONE = S.NO_SLOT


# The store ----------------------------------------------------------------------


def runs(rng, wants, block, lost=0.1, spare=3, pad=0):
    """(slots, blocks, places begun by block) of requests that bring so many
    tokens, most into a block that holds some; some requests have no slots."""
    pages = [-(-(block - 1 + n) // block) for n in wants]
    blocks = sum(pages) + spare
    order, at, slots, begun = rng.permutation(blocks), 0, [], np.zeros(blocks, int)
    for n, p in zip(wants, pages):
        first = int(rng.integers(0, block)) if rng.random() < 0.7 else 0
        place = first + np.arange(n)
        if n and rng.random() >= lost:
            slots += (order[at + place // block] * block + place % block).tolist()
            begun[order[at]] = first
        else:
            slots += [NONE] * n
        at += p
    return np.array(slots + [NONE] * pad, np.int64).astype(np.uint32), blocks, begun


def held_pool(rng, blocks, kv, block, d, begun, size):
    """Codes and scales of blocks that hold places before `begun`: normals of
    the block's size; NaN behind, and as a scale where nothing is held."""
    x = rng.standard_normal((blocks, kv, block, d)) * size[:, None, None, None]
    scale = F.scale_of(F.largest(x, (2, 3)))
    pool = F.encode(x / scale[..., None, None])
    behind = np.broadcast_to((np.arange(block)[None] >= begun[:, None])[:, None], (blocks, kv, block))
    pool[behind] = 0x7F
    scale[begun == 0] = np.nan
    return pool, scale


def hold_store(device, mem, rng, wants, heads, kv, d, block, rows_type, q_type, rotated, pad=0, queries=True,
               loud=6, rows=None, steps=1):
    slots, blocks, begun = runs(rng, wants, block, pad=3)
    T, half = len(slots), d // 2
    size = np.exp2(rng.integers(-loud, loud + 1, blocks).astype(np.float64))
    pools, scales = zip(*(held_pool(rng, blocks, kv, block, d, begun, size) for _ in "kv"))
    width = (heads + 2 * kv) * d + pad
    x = rng.standard_normal((T, width)) * np.exp2(rng.integers(-loud, loud + 1, (T, 1))) if rows is None else rows(T, width)
    bits, x = held(x, rows_type)
    x = x.astype(np.float32)
    cs = rng.standard_normal((64, max(rotated, 1), 2)).astype(np.float32)
    positions = rng.integers(0, 70, T).astype(np.uint32)       # past the table's rows: its last
    turned = cs[np.minimum(positions, 63)]
    q, k, v = (x[:, a * d:b * d].reshape(T, b - a, d) for a, b in ((0, heads), (heads, heads + kv),
                                                                   (heads + kv, heads + 2 * kv)))
    q, k = F.turn(q, turned, rotated), F.turn(k, turned, rotated)
    want = [p.copy() for p in pools]
    want_scales = [s.copy() for s in scales]
    for _ in range(steps):
        for rows_of, pool, scale in zip((k, v), want, want_scales):
            F.store(rows_of, slots, pool, scale, block)
    word = 4 if rows_type == "f32" else 2
    buf = mem.put(bits)
    bufs = dict(kpool=mem.put(pools[0]), vpool=mem.put(pools[1]),
                scales=mem.put(np.stack(scales, -1).astype(np.float32)), slots=mem.put(slots))
    qr = mem.empty(2 * T * heads * d)
    more = dict(q=buf, qr=qr, heads=heads, q_stride=width) if queries else {}
    if rotated:
        more.update(positions=mem.put(positions), rope=mem.put(cs), rope_rows=64, rotated=rotated)
    op = paged8.PagedStore8(device, k=buf, v=buf, **bufs, **more, k_offset=heads * d, v_offset=(heads + kv) * d,
                            k_stride=width, v_stride=width, tokens=T, kv_heads=kv, head_dim=d, block_size=block,
                            blocks=blocks, rows_type=rows_type, q_type=q_type)
    for _ in range(steps):
        op.enqueue()
    device.sync()
    for name, w in zip(("kpool", "vpool"), want):
        got = bufs[name].read(np.uint8).reshape(w.shape)
        bad = ~F.same_codes(got, w)
        assert not bad.any(), (name, int(bad.sum()), np.argwhere(bad)[:4].tolist(), got[bad][:6], w[bad][:6])
    got = bufs["scales"].read(np.float32).reshape(blocks, kv, 2)
    assert np.array_equal(got, np.stack(want_scales, -1).astype(np.float32), equal_nan=True)
    live = slots != NONE
    got = qr.read(np.uint16, T * heads * d).reshape(T, heads, d)
    if not queries:
        live[:] = False
    assert np.all(got[~live] == np.uint16(SENTINEL & 0xFFFF)), "a row without a slot"
    assert np.array_equal(got[live], S.narrow(q[live], q_type == "bf16"))


@pytest.mark.parametrize("rows_type,q_type", [("f32", "f16"), ("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("wants,heads,kv,d,block", [
    ([1], 1, 1, 16, 8), ([1] * 9, 4, 2, 64, 16), ([1, 0, 5, 40, 17, 1, 16], 8, 2, 64, 16), ([300, 7], 4, 4, 128, 24),
    ([64, 64, 63], 6, 2, 80, 64), ([200, 1, 9], 2, 1, 256, 128), ([33] * 20, 4, 4, 96, 8), ([1] * 700, 2, 2, 32, 16),
    ([700], 3, 3, 48, 256), ([1000, 1, 1, 900], 4, 2, 64, 1000), ([2500] * 2, 2, 8, 128, 16)])
def test_store_bit_for_bit(device, mem, wants, heads, kv, d, block, rows_type, q_type):
    rng = np.random.default_rng(sum(wants) + d)
    for rotated, pad in ((0, 0), (d // 2, 16), (d // 4 - 1, 8)):
        print(f"store8 {wants[:8]} {heads} {kv} {d} {block} {rows_type} {rotated}", flush=True)
        hold_store(device, mem, rng, wants, heads, kv, d, block, rows_type, q_type, rotated, pad)


@pytest.mark.parametrize("wants,kv,d,block", [
    ([700, 1, 64, 39, 41, 1] * 12, 32, 16, 40), ([130, 1, 1, 63] * 50, 32, 16, 64), ([900, 2] * 10, 33, 32, 136),
    ([1] * 9000, 32, 16, 8), ([3000, 1, 77], 64, 48, 72)])
def test_store_of_many_tokens_a_wavefront(device, mem, wants, kv, d, block):
    """Up to 64 tokens whose runs a wavefront takes, runs within them and past them."""
    print(f"store8 {wants[:6]} {kv} {d} {block}", flush=True)
    hold_store(device, mem, np.random.default_rng(block), wants, 2, kv, d, block, "bf16", "f16", d // 4)


def test_store_without_queries_again_and_of_no_tokens(device, mem):
    rng = np.random.default_rng(4)
    hold_store(device, mem, rng, [5, 40, 1], 2, 2, 64, 16, "f32", "f16", 32, queries=False)
    hold_store(device, mem, rng, [5, 40, 1], 2, 2, 64, 16, "bf16", "bf16", 32, steps=3)
    b = mem.empty(8192)
    paged8.PagedStore8(device, k=b, v=b, slots=b, kpool=mem.empty(1024), vpool=mem.empty(1024), scales=mem.empty(32),
                       tokens=0, kv_heads=1, head_dim=16, block_size=16, blocks=4).enqueue()
    device.sync()


def test_store_of_zeros_tiny_large_and_not_finite_rows(device, mem):
    for loud in (0, 60, 100):
        hold_store(device, mem, np.random.default_rng(loud), [3, 20, 40, 1, 1], 2, 2, 64, 16, "f32", "f16", 0, loud=loud)

    def odd(T, width):
        rng = np.random.default_rng(6)
        x = rng.standard_normal((T, width)) * np.exp2(rng.integers(-140, 100, (T, 1)).astype(np.float64))
        x[rng.random((T, width)) < 0.2] = 0
        x[::5] = 0
        with np.errstate(invalid="ignore"):
            x[1::7, ::9], x[2::7, 5], x[3::7, ::3] = np.nan, np.inf, -np.inf
        return x

    for block in (8, 64):
        hold_store(device, mem, np.random.default_rng(block), [30, 1, 1, 9, 70], 2, 2, 64, block, "f32", "bf16", 0, rows=odd)


def test_a_scale_that_grows_brings_the_held_rows_along(device, mem):
    """A token a step into one block, each louder than the last, then quiet ones:
    the codes are those of the definition, step after step."""
    rng = np.random.default_rng(11)
    kv, d, block = 2, 32, 16
    pool, scale = [np.full((2, kv, block, d), 0x7F, np.uint8) for _ in "kv"], [np.full((2, kv), np.nan) for _ in "kv"]
    kp, vp, sc = mem.put(pool[0]), mem.put(pool[1]), mem.put(np.full((2, kv, 2), np.nan, np.float32))
    rows, slots = mem.empty(4 * 2 * kv * d), mem.empty(4)
    op = paged8.PagedStore8(device, k=rows, v=rows, v_offset=kv * d, k_stride=2 * kv * d, v_stride=2 * kv * d,
                            slots=slots, kpool=kp, vpool=vp, scales=sc, tokens=1, kv_heads=kv, head_dim=d,
                            block_size=block, blocks=2)
    for place in range(block):
        x = (rng.standard_normal((1, 2 * kv, d)) * 2.0 ** (min(place, 9) * 1.5)).astype(np.float32)
        rows.write(x)
        slots.write(np.array([block + place], np.uint32))
        op.enqueue()
        device.sync()
        for i, buf in enumerate((kp, vp)):
            F.store(x[:, i * kv:(i + 1) * kv], [block + place], pool[i], scale[i], block)
            assert F.same_codes(buf.read(np.uint8).reshape(pool[i].shape), pool[i]).all(), place
        assert np.array_equal(sc.read(np.float32).reshape(2, kv, 2), np.stack(scale, -1).astype(np.float32), equal_nan=True)


# The load -----------------------------------------------------------------------


def random_pools(rng, blocks, kv, block, d, spread=6):
    codes = [rng.integers(0, 256, (blocks, kv, block, d)).astype(np.uint8) for _ in "kv"]
    scales = np.exp2(rng.integers(-spread, spread + 1, (blocks, kv, 2)).astype(np.float64))
    return codes, scales


@pytest.mark.parametrize("rows_type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("T,kv,d,block,pad", [(1, 1, 16, 8, 0), (9, 2, 64, 16, 8), (100, 3, 80, 24, 16),
                                              (1000, 8, 128, 16, 0), (77, 1, 256, 128, 0), (5000, 2, 96, 64, 24)])
def test_load_bit_for_bit(device, mem, T, kv, d, block, pad, rows_type):
    print(f"load8 {T} {kv} {d} {block} {rows_type}", flush=True)
    rng = np.random.default_rng(T + d)
    blocks, w = -(-T // block) + 2, kv * d
    codes, scales = random_pools(rng, blocks, kv, block, d)
    slots = rng.permutation(blocks * block)[:T].astype(np.uint32)
    slots[rng.random(T) < 0.1] = NONE
    if T > 3:
        slots[:3] = slots[3], blocks * block, slots[4]       # a position twice, one past the pool
    bufs = dict(kpool=mem.put(codes[0]), vpool=mem.put(codes[1]), scales=mem.put(scales.astype(np.float32)))
    word = np.uint32 if rows_type == "f32" else np.uint16
    outs = [mem.empty(T * (w + p) * word().itemsize) for p in (pad, 2 * pad)]
    paged8.PagedLoad8(device, slots=mem.put(slots), **bufs, k=outs[0], v=outs[1], tokens=T, kv_heads=kv, head_dim=d,
                      block_size=block, blocks=blocks, rows_type=rows_type, k_stride=w + pad,
                      v_stride=w + 2 * pad).enqueue()
    device.sync()
    live = slots < blocks * block
    at, place = (slots[live] // block).astype(int), slots[live] % block
    for i, (out, p) in enumerate(zip(outs, (pad, 2 * pad))):
        got = out.read(word, T * (w + p)).reshape(T, w + p)
        gap = word(SENTINEL & np.iinfo(word).max)
        assert np.all(got[:, w:] == gap) and np.all(got[~live] == gap)
        want = (F.VALUES[codes[i]] * scales[..., i, None, None])[at, :, place].reshape(-1, w).astype(np.float32)
        got = np.ascontiguousarray(got[live, :w])
        nan = np.isnan(want)
        if rows_type == "f32":
            assert np.array_equal(got.view(np.float32), want, equal_nan=True)
        else:
            assert np.array_equal(got[~nan], S.narrow(want, rows_type == "bf16")[~nan])
            assert np.isnan(S.widen(got, rows_type == "bf16")[nan]).all()


# The attention ------------------------------------------------------------------


def attend_inputs(rng, lengths, heads, kv, d, block, q_type, spare=3, table_len=None, size=1.0, spread=2):
    n, bf16 = len(lengths), q_type == "bf16"
    pages = [-(-int(x) // block) for x in lengths]
    table_len = max(1, *pages) if table_len is None else table_len
    blocks = sum(pages) + spare
    order = rng.permutation(blocks)
    table = rng.integers(0, 1 << 32, (n, table_len), dtype=np.uint64).astype(np.uint32)  # behind a length: anything
    pools = [np.full((blocks, kv, block, d), 0x7F, np.uint8) for _ in range(2)]
    scales = np.full((blocks, kv, 2), np.nan)
    at = 0
    for r, length in enumerate(lengths):
        mine = order[at:at + pages[r]]
        at += pages[r]
        table[r, :pages[r]] = mine
        for i, b in enumerate(mine):
            live = min(block, int(length) - i * block)
            for s, p in enumerate(pools):
                x = rng.standard_normal((kv, live, d)) * size * np.exp2(rng.integers(-spread, spread + 1, (kv, 1, 1)))
                scale = F.scale_of(F.largest(x, (1, 2)))
                p[b, :, :live], scales[b, :, s] = F.encode(x / scale[:, None, None]), scale
    q = S.narrow(rng.standard_normal((n, heads, d)), bf16)
    return dict(q=q, k=pools[0], v=pools[1], scales=scales, table=table, lengths=np.asarray(lengths, np.uint32),
                block=block, heads=heads, kv=kv, d=d, q_type=q_type)


def sizes_of(x, window=0):
    return dict(requests=len(x["lengths"]), heads=x["heads"], kv_heads=x["kv"], head_dim=x["d"], block_size=x["block"],
                blocks=x["k"].shape[0], table_len=x["table"].shape[1], window=window)


def bind_attend(device, mem, x, scale, window=0, out_type=None, q_pad=0, out_pad=0):
    n, w = len(x["lengths"]), x["heads"] * x["d"]
    wide = np.uint32 if out_type == "f32" else np.uint16
    q = np.full((n, w + q_pad), 0x7FC1, np.uint16)
    q[:, :w] = x["q"].reshape(n, w)
    bufs = dict(q=mem.put(q), kpool=mem.put(x["k"]), vpool=mem.put(x["v"]), table=mem.put(x["table"]),
                scales=mem.put(x["scales"].astype(np.float32)), lengths=mem.put(x["lengths"]))
    sizes = sizes_of(x, window)
    out = mem.empty(n * (w + out_pad) * np.dtype(wide).itemsize)
    nbytes = paged8.attend8_workspace(**sizes)
    workspace = mem.empty(nbytes + 64)
    op = paged8.PagedAttend8(device, **bufs, out=out, workspace=workspace, scale=scale, q_type=x["q_type"],
                             out_type=out_type, q_stride=w + q_pad, out_stride=w + out_pad, **sizes)

    def read():
        bits = out.read(wide, n * (w + out_pad)).reshape(n, w + out_pad)
        if out_pad:
            assert np.all(bits[:-1, w:] == wide(SENTINEL & np.iinfo(wide).max)), "written between rows"
        assert np.all(workspace.read(np.uint32)[-16:] == SENTINEL), "written past the workspace"
        bits = np.ascontiguousarray(bits[:, :w]).reshape(n, x["heads"], x["d"])
        return bits.view(np.float32).astype(np.float64) if out_type == "f32" else S.widen(bits, x["q_type"] == "bf16")

    return op, read, bufs


def pools_of(x):
    """The pools' values, binary64."""
    return [F.VALUES[x[name]] * x["scales"][..., i, None, None] for i, name in enumerate("kv")]


def definition(x, scale, window=0):
    """(rows, tolerance of a kind's half step): binary64's attention, whose
    bound holds with a bit to spare (the probabilities' parts hold all of theirs)."""
    o, spread, reach = S.attend(S.widen(x["q"], x["q_type"] == "bf16"), *pools_of(x), x["table"], x["lengths"],
                                x["block"], scale, window)
    return o, lambda half: S.attend_tolerance(o, spread, reach, x["lengths"], x["d"], half)


def hold_attend(device, mem, x, scale, window=0, out_type=None, **kw):
    op, read, _ = bind_attend(device, mem, x, scale, window, out_type, **kw)
    op.enqueue()
    device.sync()
    got = read()
    out, tolerance = definition(x, scale, window)
    tol = tolerance(S.half_step(out_type or x["q_type"]))
    bad = ~(np.abs(got - out) <= tol)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist(), got[bad][:4], out[bad][:4], tol[bad][:4])
    assert np.all(got[x["lengths"] == 0] == 0)


RAGGED = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 0, 127, 128, 129, 255, 256, 257, 300, 511, 513, 700, 0]


@pytest.mark.parametrize("q_type", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv,d,block", [
    (4, 4, 64, 16), (8, 2, 64, 8), (7, 1, 64, 24), (16, 1, 128, 16), (12, 4, 128, 24), (17, 1, 128, 64),
    (40, 1, 64, 16), (2, 2, 16, 16), (4, 2, 48, 16), (6, 2, 80, 40), (8, 8, 96, 128), (3, 1, 144, 16), (4, 1, 256, 16),
    (34, 2, 256, 8), (4, 2, 64, 1000), (300, 300, 16, 16)])
def test_attend_of_ragged_requests(device, mem, heads, kv, d, block, q_type):
    print(f"attend8 {heads} {kv} {d} {block} {q_type}", flush=True)
    x = attend_inputs(np.random.default_rng(heads + d), RAGGED, heads, kv, d, block, q_type)
    hold_attend(device, mem, x, d ** -0.5)


@pytest.mark.parametrize("pages", [2, 4, 8, 12, 16, 17, 24, 32, 40, 48, 49, 64, 65, 80, 96, 97, 100])
@pytest.mark.parametrize("d,kv", [(64, 2), (128, 1), (256, 2), (64, 64), (64, 16), (128, 16), (128, 50)])
def test_attend_of_tables_of_every_length(device, mem, pages, d, kv):
    """Tables of few units go whole to the threadgroups, longer ones split:
    each side of each rule, the lengths short and up to the table's."""
    print(f"attend8 table {pages} {d} {kv}", flush=True)
    top = pages * 16
    lengths = [x for x in (0, 1, 33, top // 2, top - 1, top, 17) if x <= top]
    x = attend_inputs(np.random.default_rng(pages), lengths, 2 * kv, kv, d, 16, "bf16", table_len=pages)
    hold_attend(device, mem, x, d ** -0.5)
    hold_attend(device, mem, x, d ** -0.5, window=40)


@pytest.mark.parametrize("window", [1, 7, 64, 100, 256, 5000])
@pytest.mark.parametrize("d,block", [(64, 16), (128, 24), (256, 8)])
def test_attend_in_a_window(device, mem, window, d, block):
    print(f"attend8 window {window} {d} {block}", flush=True)
    x = attend_inputs(np.random.default_rng(window), RAGGED + [3000, 2049], 6, 2, d, block, "f16")
    hold_attend(device, mem, x, d ** -0.5, window=window)
    if window < 5000:      # blocks that have left the window may be anything
        for r, length in enumerate(x["lengths"]):
            gone = max(0, int(length) - window) // block
            x["table"][r, :gone] = 0xFFFFFFFF
        hold_attend(device, mem, x, d ** -0.5, window=window)


@pytest.mark.parametrize("lengths", [[1], [20000], [9000, 1, 0, 4000], [3000] * 70, [5] * 900, [0, 0], [0] * 600 + [3],
                                     [9000, 0] + [7] * 300])
@pytest.mark.parametrize("d,q_type,block", [(64, "bf16", 16), (128, "f16", 8), (256, "bf16", 16)])
def test_attend_of_batches(device, mem, lengths, d, q_type, block):
    """One long request over many threadgroups, a few, more than there are
    threadgroups, more requests than threads, none with a key."""
    print(f"attend8 batch {len(lengths)} {max(lengths)} {d} {q_type}", flush=True)
    x = attend_inputs(np.random.default_rng(len(lengths)), lengths, 4, 2, d, block, q_type)
    hold_attend(device, mem, x, d ** -0.5)


@pytest.mark.parametrize("heads,kv,d,block,q_type", [(40, 2, 64, 16, "f16"), (17, 1, 128, 16, "bf16"),
                                                     (33, 1, 256, 24, "f16"), (6, 2, 64, 4096, "bf16"),
                                                     (48, 3, 80, 8, "bf16"), (512, 16, 64, 16, "f16")])
@pytest.mark.parametrize("lengths", [[9000, 0, 5, 700, 2500], [3000]])
def test_split_attention_of_many_heads_a_kv_head(device, mem, heads, kv, d, block, q_type, lengths):
    print(f"attend8 heads {heads} {kv} {d} {block} {q_type} {lengths}", flush=True)
    x = attend_inputs(np.random.default_rng(heads), lengths, heads, kv, d, block, q_type)
    assert paged8.attend8_form(**sizes_of(x)) == "split"
    hold_attend(device, mem, x, d ** -0.5)


def test_attend_of_one_request_with_many_heads(device, mem):
    for lengths, table_len in (([2000], 125), ([0], 125), ([90], 6)):
        print(f"attend8 many heads {lengths}", flush=True)
        x = attend_inputs(np.random.default_rng(5), lengths, 300, 300, 16, 16, "bf16", table_len=table_len)
        hold_attend(device, mem, x, 0.25)


def test_attend_rows_apart_and_f32_out(device, mem):
    for d, heads, q_type in ((64, 6, "f16"), (128, 4, "bf16"), (80, 2, "f16"), (256, 2, "bf16")):
        print(f"attend8 rows apart {d}", flush=True)
        x = attend_inputs(np.random.default_rng(d), RAGGED[:20], heads, 2, d, 16, q_type)
        hold_attend(device, mem, x, d ** -0.5, out_type="f32", q_pad=24, out_pad=5)
        hold_attend(device, mem, x, d ** -0.5, q_pad=8, out_pad=3)


def test_attend_large_and_small_scores_and_scales(device, mem):
    """Scores far apart (one key takes all), all alike, and of scale 0 and below;
    values far larger and smaller than 1."""
    for size, scale in ((30.0, 0.125), (1.0, 0.0), (1.0, -0.125), (1e-3, 1.0)):
        print(f"attend8 scores {size} {scale}", flush=True)
        x = attend_inputs(np.random.default_rng(3), RAGGED, 4, 2, 64, 16, "f16", size=size)
        hold_attend(device, mem, x, scale)
    x = attend_inputs(np.random.default_rng(4), RAGGED, 4, 2, 64, 16, "bf16", spread=0)
    for by in (2.0 ** 100, 2.0 ** -100):
        x["scales"][..., 1] *= by
        op, read, _ = bind_attend(device, mem, x, 0.125, out_type="f32")
        op.enqueue()
        device.sync()
        got = read()
        x["scales"][..., 1] /= by
        out, tolerance = definition(x, 0.125)
        assert np.all(np.abs(got / by - out) <= tolerance(2.0 ** -24))


def test_attend_lengths_past_the_table_and_blocks_past_the_pool(device, mem):
    x = attend_inputs(np.random.default_rng(8), [40, 64, 33], 4, 2, 64, 16, "f16", table_len=4)
    rng = np.random.default_rng(1)
    x["k"][:], x["v"][:] = (F.encode(rng.standard_normal(x["k"].shape) * 100) for _ in "kv")
    x["scales"][:] = 2.0 ** -7
    x["table"][0, 3] = 0
    x["table"][2, 2] = 0xFFFFFFFF            # a block past the pool: its last
    x["lengths"] = np.array([0xFFFFFFFF, 65, 48], np.uint32)
    x["table"][0, 2:] = x["table"][0, :2]
    hold_attend(device, mem, x, 0.125)


def test_attend_values_that_are_not_numbers(device, mem):
    """A request's own NaN reaches its own outputs and no other's."""
    for lengths in ([100, 70, 130], [5000, 70, 3000]):
        x = attend_inputs(np.random.default_rng(9), lengths, 4, 2, 64, 16, "f16")
        x["v"][x["table"][0, 1], 0, 3, 5] = 0xFF
        x["k"][x["table"][2, 4], 1, 1, 7] = 0x7F
        op, read, _ = bind_attend(device, mem, x, 0.125)
        op.enqueue()
        device.sync()
        got = read()
        assert np.isnan(got[0, :2, 5]).all() and np.isnan(got[2, 2:]).all()
        got[0, :2, 5], got[2, 2:] = 0, 0
        assert np.isfinite(got).all()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("q_type", ["f16", "bf16"])
def test_probabilities_keep_their_bits(device, mem, d, q_type):
    """Two keys, of score 0 and value 0 and of score x in -2 .. 0 and value v,
    both exact: out = v p / (1 + p), p = e^x, in f32.  Roundings of 2^-24: the
    scale to log2 units 2 and the score 1 (of |x| at most: 6 together), the
    reference's subtraction 0 (it is 0), the exponential 1 ulp (2), p's parts
    exact, their sum 3, the sum 1 + p 1, the quotient 1, the result 1."""
    print(f"attend8 bits {d} {q_type}", flush=True)
    n, heads = 300, 16
    rng = np.random.default_rng(d)
    x = attend_inputs(rng, [2] * n, heads, 1, d, 16, q_type)
    x["q"][:] = 0
    x["q"][:, np.arange(heads), np.arange(heads)] = S.narrow(np.ones(heads), q_type == "bf16")
    score, value = F.encode(-2 * rng.random((n, d))), F.encode(1 + rng.random((n, d)))
    for r in range(n):
        b = x["table"][r, 0]
        x["k"][b, 0, 0], x["v"][b, 0, 0] = 0, 0
        x["k"][b, 0, 1], x["v"][b, 0, 1], x["scales"][b, 0] = score[r], value[r], (1, 4)
    op, read, _ = bind_attend(device, mem, x, 1.0, out_type="f32")
    op.enqueue()
    device.sync()
    p = np.exp(F.VALUES[score][:, :heads, None])
    want = 4 * F.VALUES[value][:, None] * p / (1 + p)
    err = np.abs(read() / want - 1).max()
    assert err <= 14 * 2.0 ** -24, np.log2(err)


def test_attend_past_4_gib_of_pool(device, mem):
    """Blocks whose bytes lie past 32 bits of offset."""
    kv, d, block, blocks = 8, 128, 64, 80000           # 5.2 GB a pool
    x = attend_inputs(np.random.default_rng(10), [150, 64], 16, kv, d, block, "f16")
    far = np.array([79999, 67000, 1, 78000, 2, 3, 4, 5], np.uint32)[:x["k"].shape[0]]
    bufs = {"scales": mem.put(np.full((blocks, kv, 2), np.nan, np.float32))}
    bytes_of = kv * block * d
    for name, src in (("kpool", "k"), ("vpool", "v")):
        bufs[name] = mem.keep(device.alloc(blocks * bytes_of))
        for i, b in enumerate(far):
            bufs[name].write(x[src][i], offset=int(b) * bytes_of)
    for i, b in enumerate(far):
        bufs["scales"].write(x["scales"][i].astype(np.float32), offset=int(b) * kv * 8)
    table = np.where(x["table"] < len(far), far[np.minimum(x["table"], len(far) - 1)], 0).astype(np.uint32)
    bufs.update(q=mem.put(x["q"]), table=mem.put(table), lengths=mem.put(x["lengths"]))
    sizes = sizes_of(x) | dict(blocks=blocks)
    out = mem.empty(2 * 16 * d * 2)
    paged8.PagedAttend8(device, **bufs, out=out, workspace=mem.empty(paged8.attend8_workspace(**sizes)), scale=0.1,
                        **sizes).enqueue()
    device.sync()
    got = S.widen(out.read(np.uint16, 2 * 16 * d).reshape(2, 16, d), False)
    want, tolerance = definition(x, 0.1)
    assert np.all(np.abs(got - want) <= tolerance(S.half_step("f16")))
    # and the rows read back from there
    slots = np.array([79999 * 64 + 5, 1 * 64 + 63, 67000 * 64], np.uint32)
    rows = [mem.empty(3 * kv * d * 4) for _ in "kv"]
    paged8.PagedLoad8(device, slots=mem.put(slots), kpool=bufs["kpool"], vpool=bufs["vpool"], scales=bufs["scales"],
                      k=rows[0], v=rows[1], tokens=3, kv_heads=kv, head_dim=d, block_size=block, blocks=blocks,
                      rows_type="f32").enqueue()
    device.sync()
    for i, (buf, values) in enumerate(zip(rows, pools_of(x))):
        got = buf.read(np.float32, 3 * kv * d).reshape(3, kv, d)
        for g, (b, place) in zip(got, ((0, 5), (2, 63), (1, 0))):
            assert np.array_equal(g, values[b, :, place].astype(np.float32), equal_nan=True), i


@pytest.mark.parametrize("block", [16, 64])
def test_store_past_4_gib_of_pool(device, mem, block):
    """Runs that begin a block and that go on in one, past 32 bits of offset."""
    kv, d, blocks = 8, 128, 5200000 // block           # 5.3 GB a pool
    rng, bytes_of = np.random.default_rng(11), kv * block * d
    far, begun = [blocks - 1, blocks - 70000 // block, 1], np.array([0, 5, 7])
    codes, scales = zip(*(held_pool(rng, 3, kv, block, d, begun, np.ones(3)) for _ in "kv"))
    bufs = {n: mem.keep(device.alloc(blocks * bytes_of)) for n in ("kpool", "vpool")}
    bufs["scales"] = mem.keep(device.alloc(blocks * kv * 8))
    for i, b in enumerate(far):
        for n, c in zip(("kpool", "vpool"), codes):
            bufs[n].write(c[i], offset=b * bytes_of)
        bufs["scales"].write(np.stack([s[i] for s in scales], -1).astype(np.float32), offset=b * kv * 8)
    place = [(i, p) for i, first in enumerate(begun) for p in range(first, 8)]
    x = (rng.standard_normal((len(place), 2 * kv * d)) * 4).astype(np.float32)
    want = [c.copy() for c in codes]
    want_scales = [s.copy() for s in scales]
    for j, (w, s) in enumerate(zip(want, want_scales)):
        F.store(x[:, j * kv * d:(j + 1) * kv * d].reshape(-1, kv, d),
                np.array([i * block + p for i, p in place], np.uint32), w, s, block)
    slots = np.array([far[i] * block + p for i, p in place], np.uint32)
    row = mem.put(x)
    paged8.PagedStore8(device, k=row, v=row, **bufs, slots=mem.put(slots), v_offset=kv * d, k_stride=2 * kv * d,
                       v_stride=2 * kv * d, tokens=len(place), kv_heads=kv, head_dim=d, block_size=block,
                       blocks=blocks).enqueue()
    device.sync()
    for i, b in enumerate(far):
        for n, w in zip(("kpool", "vpool"), want):
            got = bufs[n].read(np.uint8, bytes_of, offset=b * bytes_of).reshape(w[i].shape)
            assert np.all(F.same_codes(got, w[i])), (i, n)
        got = bufs["scales"].read(np.float32, 2 * kv, offset=b * kv * 8).reshape(kv, 2)
        assert np.array_equal(got, np.stack([s[i] for s in want_scales], -1).astype(np.float32)), i


# A run of them ---------------------------------------------------------------------


@pytest.mark.parametrize("q_type,d,block,window", [("f16", 64, 16, 0), ("bf16", 128, 24, 0), ("bf16", 64, 16, 1600)])
def test_a_captured_step_of_8_bit_caches(device, mem, q_type, d, block, window):
    """Plan, store and attend, whose two launches share a workspace, and a load of
    the step's own rows, captured once and replayed over requests of up to 3000
    positions that grow, rest and come in, with eager calls between: every
    replay's caches those of the definition, its rows those of the definition
    over the caches as they then are."""
    rng = np.random.default_rng(21)
    bf16 = q_type == "bf16"
    heads, kv, tokens = 4, 2, 9
    cached = np.array([0, 1900, block * 40, 3000, 5], np.uint32)
    n, table_len = len(cached), -(-3040 // block)
    x = attend_inputs(rng, [int(c) for c in cached], heads, kv, d, block, q_type, spare=30, table_len=table_len)
    sizes = sizes_of(x, window)
    assert paged8.attend8_form(**sizes) == "split"
    blocks = sizes["blocks"]
    used = {int(b) for r in range(n) for b in x["table"][r, :-(-int(cached[r]) // block)]}
    free = np.array([b for b in range(blocks) if b not in used], np.uint32)
    head, table, width = 0, x["table"], (heads + 2 * kv) * d
    b = dict(cached=mem.put(cached), fresh=mem.put(np.ones(n, np.uint32)), free=mem.put(free),
             head=mem.put(np.zeros(1, np.uint32)), table=mem.put(table), lengths=mem.empty(4 * n),
             starts=mem.empty(4 * n + 4), slots=mem.empty(4 * tokens), positions=mem.empty(4 * tokens),
             owner=mem.empty(4 * tokens), counts=mem.put(np.zeros(4, np.uint32)))
    rows, qr, out = mem.empty(4 * tokens * width), mem.empty(2 * tokens * heads * d), mem.empty(2 * n * heads * d)
    pool = dict(kpool=mem.put(x["k"]), vpool=mem.put(x["v"]), scales=mem.put(x["scales"].astype(np.float32)))
    back = [mem.empty(4 * tokens * kv * d) for _ in "kv"]
    shape = dict(kv_heads=kv, head_dim=d, block_size=block, blocks=blocks)
    plan = paged.PagePlan(device, **b, requests=n, tokens=tokens, table_len=table_len, block_size=block,
                          free_len=len(free))
    store = paged8.PagedStore8(device, q=rows, k=rows, v=rows, k_offset=heads * d, v_offset=(heads + kv) * d,
                               q_stride=width, k_stride=width, v_stride=width, slots=b["slots"], qr=qr, **pool,
                               tokens=tokens, heads=heads, rows_type="f32", q_type=q_type, **shape)
    attend = paged8.PagedAttend8(device, q=qr, **pool, table=b["table"], lengths=b["lengths"], out=out,
                                 workspace=mem.empty(paged8.attend8_workspace(**sizes)), scale=d ** -0.5,
                                 q_type=q_type, starts=b["starts"], q_rows=tokens, **sizes)
    load = paged8.PagedLoad8(device, slots=b["slots"], **pool, k=back[0], v=back[1], tokens=tokens, rows_type="f32",
                             **shape)
    stream = device.new_stream()
    with device.capture(stream) as captured:
        for op in (plan, store, attend, load):
            op.enqueue(stream)
        b["cached"].copy_from(b["lengths"], 4 * n, stream=stream)
        b["head"].copy_from(b["counts"], 4, src_offset=12, stream=stream)
    for step in range(6):
        fresh = np.ones(n, np.uint32)
        fresh[step % n] = step % 3                  # a request rests, another brings two tokens
        new = (rng.standard_normal((tokens, width)) * 2.0 ** step).astype(np.float32)
        rows.write(new)
        b["fresh"].write(fresh)
        device.sync()
        captured[0].replay(stream)
        device.sync(stream)
        want = S.plan(cached, fresh, free, head, table, tokens, block)
        for k in ("lengths", "starts", "slots"):
            assert np.array_equal(b[k].read(np.uint32, want[k].size), want[k]), (step, k)
        table, head, cached = want["table"], int(want["counts"][3]), want["lengths"]
        x["table"], x["lengths"] = table, np.where(fresh > 0, cached, 0)
        for i, (name, first) in enumerate((("k", heads), ("v", heads + kv))):
            scale = x["scales"][..., i]
            F.store(new[:, first * d:(first + kv) * d].reshape(tokens, kv, d), want["slots"], x[name], scale, block)
            assert F.same_codes(pool[name + "pool"].read(np.uint8).reshape(x[name].shape), x[name]).all(), (step, name)
        assert np.array_equal(pool["scales"].read(np.float32).reshape(x["scales"].shape), x["scales"].astype(np.float32),
                              equal_nan=True)
        qs = S.narrow(new[:, :heads * d], bf16).reshape(tokens, heads, d)
        x["q"] = qs[np.maximum(want["starts"][1:].astype(int) - 1, 0)]
        o, tolerance = definition(x, d ** -0.5, window)
        got = out.read(np.uint16, n * heads * d)
        bad = ~(np.abs(S.widen(got.reshape(n, heads, d), bf16) - o) <= tolerance(S.half_step(q_type)))
        assert not bad.any(), (step, int(bad.sum()), np.argwhere(bad)[:4].tolist())
        live = want["slots"] != NONE
        at, place = (want["slots"][live] // block).astype(int), want["slots"][live] % block
        for buf, values in zip(back, pools_of(x)):
            assert np.array_equal(buf.read(np.float32, tokens * kv * d).reshape(tokens, kv, d)[live],
                                  values[at, :, place].astype(np.float32))
        out.write(np.zeros_like(got))
        attend.enqueue()
        device.sync()
        assert np.array_equal(out.read(np.uint16, n * heads * d), got)
    captured[0].destroy()


@pytest.mark.parametrize("kind,out_type", [("f32", "f16"), ("bf16", "bf16")])
def test_a_captured_layer_over_8_bit_caches(device, mem, kind, out_type):
    """A layer as a server runs it: plan, the stream's norm, q k v, store,
    attention, its product onto the stream, the next norm and a product.
    Captured and replayed over requests that grow from nothing, with the same
    calls made eagerly over buffers of their own between: the same bits, codes
    and scales after every step."""
    rng = np.random.default_rng(31)
    n, hidden, heads, kv, d, block, table_len = 5, 200, 6, 2, 64, 8, 6
    tokens, blocks, width, wide = 9, 40, (heads + 2 * kv) * d, 264
    word = 4 if kind == "f32" else 2
    weights = {name: (rng.standard_normal(shape) * shape[1] ** -0.5).astype(np.float32)
               for name, shape in (("qkv", (width, hidden)), ("o", (hidden, heads * d)), ("up", (wide, hidden)))}
    gamma = (1 + 0.1 * rng.standard_normal((2, hidden))).astype(np.float32)
    cs = rng.standard_normal((64, d // 2, 2)).astype(np.float32)

    def layer():
        m = {}
        for name, w in weights.items():
            m[name] = mem_matrix(device, mem, *w.shape)
            fp8.Quantize(device, mem.put(w), m[name]).enqueue()
        b = dict(cached=mem.put(np.zeros(n, np.uint32)), fresh=mem.put(np.ones(n, np.uint32)),
                 free=mem.put(np.arange(blocks, dtype=np.uint32)), head=mem.put(np.zeros(1, np.uint32)),
                 table=mem.put(np.zeros((n, table_len), np.uint32)), lengths=mem.empty(4 * n),
                 starts=mem.empty(4 * n + 4), slots=mem.empty(4 * tokens), positions=mem.empty(4 * tokens),
                 owner=mem.empty(4 * tokens), counts=mem.put(np.zeros(4, np.uint32)))
        x, rows, o = (mem.put(np.zeros(tokens * c * word, np.uint8)) for c in (hidden, width, hidden))
        qr, y = (mem.put(np.zeros(2 * c * heads * d, np.uint8)) for c in (tokens, n))
        up = mem.put(np.zeros(n * wide * 4, np.uint8))
        pool = dict(kpool=mem.put(np.zeros(blocks * block * kv * d, np.uint8)),
                    vpool=mem.put(np.zeros(blocks * block * kv * d, np.uint8)),
                    scales=mem.put(np.zeros(blocks * kv * 2, np.float32)))
        h, ym, h2 = (mem_matrix(device, mem, *s) for s in ((tokens, hidden), (n, heads * d), (n, hidden)))
        sizes = dict(requests=n, heads=heads, kv_heads=kv, head_dim=d, block_size=block, blocks=blocks,
                     table_len=table_len)
        ops = [paged.PagePlan(device, **b, requests=n, tokens=tokens, table_len=table_len, block_size=block,
                              free_len=blocks),
               fp8.AddNorm(device, x, h, 1e-5, gamma=mem.put(gamma[0]), x_type=kind),
               fp8.Gemm(device, h, m["qkv"], rows, c_type=kind),
               paged8.PagedStore8(device, q=rows, k=rows, v=rows, k_offset=heads * d, v_offset=(heads + kv) * d,
                                  q_stride=width, k_stride=width, v_stride=width, slots=b["slots"],
                                  positions=b["positions"], rope=mem.put(cs), rope_rows=64, rotated=d // 2, qr=qr,
                                  **pool, tokens=tokens, heads=heads, kv_heads=kv, head_dim=d, block_size=block,
                                  blocks=blocks, rows_type=kind, q_type=out_type),
               paged8.PagedAttend8(device, q=qr, **pool, table=b["table"], lengths=b["lengths"], out=y,
                                   workspace=mem.empty(paged8.attend8_workspace(**sizes)), scale=d ** -0.5,
                                   q_type=out_type, starts=b["starts"], q_rows=tokens, **sizes),
               fp8.Quantize(device, y, ym, x_type=out_type), fp8.Gemm(device, ym, m["o"], o, c_type=kind),
               fp8.AddNorm(device, o, h2, 1e-5, gamma=mem.put(gamma[1]), x_type=kind),
               fp8.Gemm(device, h2, m["up"], up)]
        return b, x, ops, [rows, qr, y, o, up, h.codes, h.scales, h2.codes, h2.scales, *pool.values(), b["lengths"]]

    (cb, cx, cops, cheld), (eb, ex, eops, eheld) = layer(), layer()
    stream = device.new_stream()
    device.sync()
    with device.capture(stream) as captured:
        for op in cops:
            op.enqueue(stream)
        cb["cached"].copy_from(cb["lengths"], 4 * n, stream=stream)
        cb["head"].copy_from(cb["counts"], 4, src_offset=12, stream=stream)
    for step in range(12):
        fresh = np.ones(n, np.uint32)
        fresh[step % n] = step % 4
        xs = held(rng.standard_normal((tokens, hidden)) * 2.0 ** (step % 3), kind)[0]
        for b, x in ((cb, cx), (eb, ex)):
            b["fresh"].write(fresh)
            x.write(xs)
        device.sync()
        captured[0].replay(stream)
        for op in eops:
            op.enqueue()
        eb["cached"].copy_from(eb["lengths"], 4 * n)
        eb["head"].copy_from(eb["counts"], 4, src_offset=12)
        device.sync(stream)
        device.sync()
        for i, (p, q) in enumerate(zip(cheld, eheld)):
            assert np.array_equal(p.read(np.uint8), q.read(np.uint8)), (step, i)
        got = cheld[4].read(np.float32, n * wide)
        assert np.isfinite(got).all() and got.any()
    assert cheld[-1].read(np.uint32, n).max() > block
    captured[0].destroy()


def test_two_attentions_at_once_with_a_workspace_each(device, mem):
    rng = np.random.default_rng(31)
    bound = [bind_attend(device, mem, attend_inputs(rng, lengths, 8, 2, d, 16, "bf16"), d ** -0.5)
             for lengths, d in (([9000, 40, 2000], 128), ([5000] * 5, 64))]
    for op, _, _ in bound:
        op.enqueue()
    device.sync()
    want = [read() for _, read, _ in bound]
    streams = [device.new_stream() for _ in bound]
    for _ in range(3):
        for (op, _, _), s in zip(bound, streams):
            op.enqueue(s)
    for s in streams:
        device.sync(s)
    assert all(np.array_equal(read(), w) for (_, read, _), w in zip(bound, want))
