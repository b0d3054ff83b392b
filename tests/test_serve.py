"""The operators of a served batch without a GPU: the C structs' layouts, the
checks that their entries make of the arguments, and the bindings' checks of
their buffers (no launch is made of what they refuse)."""

import ctypes
import re
from pathlib import Path

import pytest

from furykernel_amd import mx4, paged, runtime
from furykernel_amd.kernels import LaunchError

INCLUDE = Path(__file__).resolve().parents[1] / "include"
HEADER = (INCLUDE / "fkrocm_serve.h").read_text() + (INCLUDE / "fkrocm_mx4.h").read_text()
STRUCTS = {"fk_mx4_quantize_args": mx4.QuantizeArgs, "fk_mx4_dequantize_args": mx4.DequantizeArgs,
           "fk_mx4_gemm_args": mx4.GemmArgs, "fk_page_plan_args": paged.PagePlanArgs,
           "fk_paged_store_args": paged.PagedStoreArgs, "fk_paged_attend_args": paged.PagedAttendArgs}


class FakeDevice:
    ctx = None


DEVICE = FakeDevice()


class FakeBuffer:
    """A buffer of this size at an address of its own, with nothing behind it."""
    at = 1 << 40

    def __init__(self, size, device=DEVICE, ptr=None):
        self.size, self.device = size, device
        self.ptr = FakeBuffer.at if ptr is None else ptr
        FakeBuffer.at += (size + 511) // 256 * 256


@pytest.mark.parametrize("name", sorted(STRUCTS))
def test_the_structs_fields_are_the_headers(name):
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), HEADER, re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    fields = []
    for decl in filter(None, (d.strip() for d in body.split(";"))):
        kind, names = decl.split(None, 1)
        fields += [(n.strip(), {"uint64_t": ctypes.c_uint64, "uint32_t": ctypes.c_uint32,
                                "float": ctypes.c_float}[kind]) for n in names.split(",")]
    assert STRUCTS[name]._fields_ == fields


def attend_sizes(**over):
    return {**dict(requests=5, heads=8, kv_heads=2, head_dim=64, block_size=16, blocks=20, table_len=5), **over}


def attend(over=(), sizes=(), **kw):
    z = attend_sizes(**dict(sizes))
    n, w = z["requests"], z["heads"] * z["head_dim"]
    pool = z["blocks"] * z["block_size"] * z["kv_heads"] * z["head_dim"] * 2
    bufs = dict(q=FakeBuffer(n * w * 2), kpool=FakeBuffer(pool), vpool=FakeBuffer(pool),
                table=FakeBuffer(4 * n * z["table_len"]), lengths=FakeBuffer(4 * n), out=FakeBuffer(n * w * 2),
                workspace=FakeBuffer(1 << 26))
    bufs.update(dict(over))
    return paged.PagedAttend(DEVICE, **bufs, **z, scale=0.125, **kw)


def test_attend_takes_what_it_says():
    attend()
    attend(out_type="f32", over={"out": FakeBuffer(5 * 512 * 4)})
    attend(q_stride=520, over={"q": FakeBuffer((4 * 520 + 512) * 2)})
    for d in (8, 72, 128, 200, 256):
        attend(sizes={"head_dim": d})
    attend(sizes={"heads": 34, "window": 7})


@pytest.mark.parametrize("sizes", [
    {"requests": 0}, {"heads": 0}, {"kv_heads": 0}, {"heads": 7}, {"head_dim": 0}, {"head_dim": 12},
    {"head_dim": 264}, {"block_size": 0}, {"blocks": 0}, {"table_len": 0}, {"table_len": 1 << 28},
    {"blocks": 1 << 28}, {"requests": 1 << 24}, {"requests": 1 << 23, "table_len": 1 << 20}, {"requests": -1},
    {"window": 1 << 32}])
def test_attend_refuses_sizes(sizes):
    with pytest.raises(LaunchError):
        attend(sizes=sizes)


@pytest.mark.parametrize("name", ["q", "kpool", "vpool", "table", "lengths", "out", "workspace"])
def test_attend_refuses_buffers(name):
    sizes = attend_sizes()
    full = {"q": 5120, "kpool": 81920, "vpool": 81920, "table": 100, "lengths": 20, "out": 5120,
            "workspace": paged.attend_workspace(**sizes)}[name]
    attend({name: FakeBuffer(full)})
    off = 2 if name in ("table", "lengths") else 8
    for bad in (FakeBuffer(full - 1), FakeBuffer(full, FakeDevice()), FakeBuffer(full, ptr=FakeBuffer.at + off)):
        with pytest.raises(LaunchError):
            attend({name: bad})


def test_attend_refuses_overlaps_strides_and_types():
    q = FakeBuffer(5 * 512 * 4)
    for over, kw in (({"q": q, "out": q}, {}), ({"lengths": q, "workspace": q}, {}), ({}, {"q_stride": 504}),
                     ({"q": q}, {"q_stride": 516}), ({}, {"out_stride": 511}), ({}, {"cache": "f32"}),
                     ({}, {"cache": "bf16", "out_type": "f16"}), ({}, {"out_stride": 513})):
        with pytest.raises(LaunchError):
            attend(over, **kw)


def test_attend_refuses_starts_without_rows():
    starts, q = FakeBuffer(24), FakeBuffer(7 * 512 * 2)
    attend({"starts": starts, "q": q}, q_rows=7)
    for over, rows in (({"starts": starts, "q": q}, 0), ({"starts": starts, "q": q}, 8),
                       ({"starts": starts, "q": q}, -1), ({"starts": FakeBuffer(20), "q": q}, 7)):
        with pytest.raises(LaunchError):
            attend(over, q_rows=rows)


def plan(over=(), **sizes):
    z = {**dict(requests=4, tokens=9, table_len=3, block_size=16, free_len=5), **sizes}
    n, t = z["requests"], z["tokens"]
    words = dict(cached=n, fresh=n, free=z["free_len"], head=1, table=n * z["table_len"], lengths=n, starts=n + 1,
                 slots=t, positions=t, owner=t, counts=4)
    bufs = {k: FakeBuffer(4 * max(v, 0)) for k, v in words.items()}
    bufs.update(dict(over))
    return paged.PagePlan(DEVICE, **bufs, **z)


def test_plan_takes_what_it_says():
    plan()
    plan(tokens=0)
    plan(free_len=0)
    plan(requests=100000, tokens=1 << 20)


@pytest.mark.parametrize("sizes", [{"requests": 0}, {"requests": 1 << 24}, {"table_len": 0}, {"block_size": 0},
                                   {"block_size": 1 << 31, "table_len": 2}, {"tokens": -1}, {"tokens": 0xFFFFFFFF}])
def test_plan_refuses_sizes(sizes):
    with pytest.raises(LaunchError):
        plan(**sizes)


def test_plan_refuses_buffers_and_overlaps():
    words = dict(cached=4, fresh=4, free=5, head=1, table=12, lengths=4, starts=5, slots=9, positions=9, owner=9,
                 counts=4)
    for name, count in words.items():
        for bad in (FakeBuffer(4 * count - 1), FakeBuffer(4 * count, FakeDevice()),
                    FakeBuffer(4 * count, ptr=FakeBuffer.at + 2)):
            with pytest.raises(LaunchError):
                plan({name: bad})
    one = FakeBuffer(4096)
    for a, b in (("cached", "lengths"), ("head", "counts"), ("free", "table"), ("slots", "owner")):
        with pytest.raises(LaunchError, match="overlaps"):
            plan({a: one, b: one})
    counts = FakeBuffer(16)
    with pytest.raises(LaunchError, match="overlaps"):   # the next head is not this step's
        plan({"counts": counts, "head": FakeBuffer(4, ptr=counts.ptr + 12)})


def store(over=(), sizes=(), **kw):
    z = {**dict(tokens=5, heads=4, kv_heads=2, head_dim=64, block_size=16, blocks=3, rotated=32, rope_rows=100),
         **dict(sizes)}
    T, d = z["tokens"], z["head_dim"]
    pool = z["blocks"] * z["block_size"] * z["kv_heads"] * d * 2
    bufs = dict(q=FakeBuffer(4 * T * z["heads"] * d), k=FakeBuffer(4 * T * z["kv_heads"] * d),
                v=FakeBuffer(4 * T * z["kv_heads"] * d), slots=FakeBuffer(4 * T), positions=FakeBuffer(4 * T),
                rope=FakeBuffer(8 * z["rope_rows"] * max(z["rotated"], 0)), qr=FakeBuffer(2 * T * z["heads"] * d),
                kpool=FakeBuffer(pool), vpool=FakeBuffer(pool))
    bufs.update(dict(over))
    return paged.PagedStore(DEVICE, **bufs, **z, **kw)


def test_store_takes_what_it_says():
    store()
    store(sizes={"rotated": 0}, over={"rope": None, "positions": None})
    store(sizes={"heads": 0}, over={"q": None, "qr": None})
    store(sizes={"tokens": 0})
    store(sizes={"head_dim": 16, "rotated": 8})
    store(sizes={"head_dim": 256}, rows_type="bf16", cache="bf16")
    fused = FakeBuffer(4 * 5 * 520)
    store({"q": fused, "k": fused, "v": fused}, q_stride=520, k_stride=520, v_stride=520, k_offset=256, v_offset=384)


@pytest.mark.parametrize("sizes", [
    {"kv_heads": 0}, {"head_dim": 8}, {"head_dim": 40}, {"head_dim": 272}, {"block_size": 0}, {"blocks": 0},
    {"blocks": 1 << 31}, {"rotated": 33}, {"rope_rows": 0}, {"tokens": 1 << 28}, {"tokens": -3},
    {"tokens": 1, "heads": 1 << 25}, {"tokens": 1, "kv_heads": 1 << 25, "blocks": 1}])
def test_store_refuses_sizes(sizes):
    with pytest.raises(LaunchError):
        store(sizes=sizes)


def test_store_refuses_buffers_strides_and_types():
    for name in ("q", "k", "v", "slots", "positions", "rope", "qr", "kpool", "vpool"):
        good = store().held[("q", "k", "v", "slots", "positions", "rope", "qr", "kpool", "vpool").index(name)]
        off = 2 if name in ("slots", "positions") else 4
        for bad in (FakeBuffer(good.size - 1), FakeBuffer(good.size, FakeDevice()),
                    FakeBuffer(good.size, ptr=FakeBuffer.at + off)):
            with pytest.raises(LaunchError):
                store({name: bad})
    big = FakeBuffer(1 << 20)
    for over, kw in (({"q": None}, {}), ({"qr": None}, {}), ({"rope": None}, {}), ({"positions": None}, {}),
                     ({"k": big}, {"k_stride": 130}), ({"k": big}, {"k_stride": 64}), ({"v": big}, {"v_offset": 2}),
                     ({"v": big}, {"v_offset": -4}), ({}, {"rows_type": "i8"}), ({}, {"cache": "f32"}),
                     ({"kpool": big, "vpool": big}, {}), ({"q": big, "kpool": big}, {}), ({"q": big}, {"q_offset": 1})):
        with pytest.raises(LaunchError):
            store(over, **kw)


def test_the_arrays_of_a_step_may_lie_together():
    # (a plan's outputs in one buffer, a word apart)
    store({"slots": FakeBuffer(20, ptr=FakeBuffer.at + 4), "positions": FakeBuffer(20, ptr=FakeBuffer.at + 324)})
    attend({"lengths": FakeBuffer(20, ptr=FakeBuffer.at + 4), "table": FakeBuffer(100, ptr=FakeBuffer.at + 324)})


def test_the_checks_refuse_spans_past_any_memory():
    huge = FakeBuffer(1 << 80)   # what a wrapped size would let through
    with pytest.raises(LaunchError, match="spans 2"):
        store({"k": huge}, sizes={"tokens": 1 << 24, "heads": 1, "head_dim": 16, "rotated": 8}, k_stride=1 << 39)
    with pytest.raises(LaunchError, match="spans 2"):
        attend({"q": huge, "starts": FakeBuffer(24)}, q_rows=1 << 31, q_stride=1 << 36)
    with pytest.raises(LaunchError, match="spans 2"):
        mx4.Quantize(DEVICE, huge, matrix(1 << 24, 32), x_stride=1 << 39)


def test_the_check_refuses_unknown_entries_and_sizes_of_arguments():
    lib = runtime.library()
    err = ctypes.create_string_buffer(200)
    args = paged.PagePlanArgs()
    for entry, n, status in ((b"fk_nothing", 8, -4), (b"fk_page_plan", 8, -2), (None, 8, -4)):
        assert lib.fk_serve_check(entry, ctypes.byref(args), n, err, 200) == status and err.value
    assert lib.fk_serve_check(b"fk_page_plan", None, ctypes.sizeof(args), err, 200) == -2
    for entry in (lib.fk_page_plan, lib.fk_paged_store, lib.fk_paged_attend):
        assert entry(None, ctypes.byref(args), None) == -2
    assert lib.fk_paged_attend_workspace(None) == 0


# 4-bit microscaled matrices ----------------------------------------------------


def matrix(rows, k):
    m = mx4.Mx4Matrix.__new__(mx4.Mx4Matrix)
    lib = runtime.library()
    m.device, m.rows, m.k = DEVICE, rows, k
    m.codes, m.scales = FakeBuffer(lib.fk_mx4_codes_bytes(rows, k)), FakeBuffer(lib.fk_mx4_scales_bytes(rows, k))
    return m


def test_mx4_matrices_hold_whole_tiles():
    lib = runtime.library()
    for rows, k, tiles in ((1, 1, 1), (16, 256, 1), (17, 256, 2), (16, 257, 2), (100, 3080, 7 * 13)):
        assert lib.fk_mx4_codes_bytes(rows, k) == tiles * 2048 and lib.fk_mx4_scales_bytes(rows, k) == tiles * 128
    for rows, k in ((0, 5), (5, 0), (0xFFFFFFFF, 32), (1 << 30, 1 << 30)):
        assert lib.fk_mx4_codes_bytes(rows, k) == 0 == lib.fk_mx4_scales_bytes(rows, k)


def test_mx4_operations_refuse_what_does_not_fit():
    a, b = matrix(20, 100), matrix(33, 100)
    mx4.Quantize(DEVICE, FakeBuffer(4 * 2000), a)
    mx4.Quantize(DEVICE, FakeBuffer(2 * (19 * 101 + 100 + 3)), a, "bf16", x_stride=101, x_offset=3)
    mx4.Dequantize(DEVICE, a, FakeBuffer(4 * 2000), scales=FakeBuffer(4 * 20 * 4))
    mx4.Gemm(DEVICE, a, b, FakeBuffer(4 * 20 * 33))
    big = FakeBuffer(1 << 20)
    short = matrix(20, 100)
    short.codes = FakeBuffer(short.codes.size - 1)
    bad = [lambda: mx4.Quantize(DEVICE, FakeBuffer(4 * 2000 - 1), a),
           lambda: mx4.Quantize(DEVICE, big, a, "i8"), lambda: mx4.Quantize(DEVICE, big, a, x_stride=99),
           lambda: mx4.Quantize(DEVICE, big, a, x_offset=-1), lambda: mx4.Quantize(DEVICE, big, short),
           lambda: mx4.Quantize(DEVICE, FakeBuffer(8000, ptr=FakeBuffer.at + 2), a),
           lambda: mx4.Quantize(DEVICE, FakeBuffer(8000, FakeDevice()), a),
           lambda: mx4.Quantize(DEVICE, FakeBuffer(8000, ptr=a.codes.ptr), a),
           lambda: mx4.Dequantize(DEVICE, a, FakeBuffer(4 * 2000 - 1)),
           lambda: mx4.Dequantize(DEVICE, a, big, y_stride=99),
           lambda: mx4.Dequantize(DEVICE, a, big, scales=FakeBuffer(4 * 20 * 4 - 1)),
           lambda: mx4.Dequantize(DEVICE, a, big, scales=big),
           lambda: mx4.Dequantize(DEVICE, a, FakeBuffer(8000, ptr=a.scales.ptr)),
           lambda: mx4.Gemm(DEVICE, a, b, FakeBuffer(4 * 20 * 33 - 1)),
           lambda: mx4.Gemm(DEVICE, a, matrix(33, 101), big), lambda: mx4.Gemm(DEVICE, a, b, big, "i8"),
           lambda: mx4.Gemm(DEVICE, a, b, big, c_stride=32), lambda: mx4.Gemm(DEVICE, short, b, big),
           lambda: mx4.Gemm(DEVICE, a, b, FakeBuffer(1 << 13, ptr=b.codes.ptr)), lambda: mx4.Mx4Matrix(DEVICE, 0, 5),
           lambda: mx4.Mx4Matrix(DEVICE, -1, 5)]
    for i, call in enumerate(bad):
        with pytest.raises(LaunchError):
            call()
            print(f"call {i} was taken")
    lib = runtime.library()
    for entry in (lib.fk_mx4_quantize, lib.fk_mx4_dequantize, lib.fk_mx4_gemm):
        assert entry(None, None, None) == -2


def test_the_form_of_a_refused_product_is_none():
    """Products that fk_mx4_gemm refuses for their sizes, and one that it takes."""
    lib = runtime.library()
    for m, n, k in ((1 << 27, 1 << 27, 32), (1 << 20, 1 << 20, 32), (0, 5, 32), (5, 0, 32), (5, 5, 0),
                    (1 << 30, 5, 512), (100, 200, 300)):
        print(f"product {m} {n} {k}", flush=True)
        args = mx4.GemmArgs(*(i << 44 for i in range(1, 6)), n, m, n, k, 0)
        taken = lib.fk_serve_check(b"fk_mx4_gemm", ctypes.byref(args), ctypes.sizeof(args), None, 0) == 0
        assert bool(lib.fk_mx4_gemm_form(m, n, k)) == taken


def test_no_matrix_takes_a_launch_of_more_threads_than_there_are():
    """A wavefront of 64 threads a tile, two tiles a pair, whole threadgroups of
    four: fewer than 2^32 threads."""
    lib = runtime.library()
    for tiles, taken in (((1 << 25) - 3, True), ((1 << 25) - 2, True), ((1 << 25) - 1, False), (1 << 25, False)):
        assert bool(lib.fk_mx4_codes_bytes(16 * tiles, 1)) == taken == bool(lib.fk_mx4_scales_bytes(16 * tiles, 1))


def test_the_attentions_form_by_its_sizes():
    for form, over in (("whole 4", {"table_len": 16}), ("whole 8", {"table_len": 32}), ("split", {"table_len": 400}),
                       ("whole 8", {"table_len": 400, "window": 200}), ("split", {"head_dim": 256, "table_len": 17})):
        assert paged.attend_form(**attend_sizes(**over)) == form
    with pytest.raises(LaunchError):
        paged.attend_form(**attend_sizes(heads=7))
    lib = runtime.library()
    assert lib.fk_paged_attend_form(None) == b"" == lib.fk_paged_attend_form(ctypes.byref(paged.PagedAttendArgs()))
