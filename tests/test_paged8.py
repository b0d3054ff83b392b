"""The operators over 8-bit paged caches without a GPU: the C structs'
layouts, the checks that their entries make of the arguments, the bindings'
checks of their buffers (no launch is made of what they refuse)."""

from pathlib import Path

import pytest

from furykernel_amd import paged8, runtime
from furykernel_amd.kernels import LaunchError
from test_fp8 import fields_of
from test_serve import DEVICE, FakeBuffer, FakeDevice

HEADER = (Path(__file__).resolve().parents[1] / "include" / "fkrocm_paged8.h").read_text()
STRUCTS = {"fk_paged_store8_args": paged8.PagedStore8Args, "fk_paged_load8_args": paged8.PagedLoad8Args,
           "fk_paged_attend8_args": paged8.PagedAttend8Args}


@pytest.mark.parametrize("name", sorted(STRUCTS))
def test_the_structs_fields_are_the_headers(name):
    assert STRUCTS[name]._fields_ == fields_of(HEADER, name)


def pools(z):
    n = z["blocks"] * z["kv_heads"]
    size = max(0, n * z["block_size"] * z["head_dim"])
    return dict(kpool=FakeBuffer(size), vpool=FakeBuffer(size), scales=FakeBuffer(max(0, 8 * n)))


def attend(over=(), sizes=(), **kw):
    z = {**dict(requests=5, heads=8, kv_heads=2, head_dim=64, block_size=16, blocks=20, table_len=5), **dict(sizes)}
    n, w = z["requests"], z["heads"] * z["head_dim"]
    bufs = dict(q=FakeBuffer(max(0, n * w * 2)), table=FakeBuffer(max(0, 4 * n * z["table_len"])),
                lengths=FakeBuffer(max(0, 4 * n)), out=FakeBuffer(max(0, n * w * 2)), workspace=FakeBuffer(1 << 26))
    return paged8.PagedAttend8(DEVICE, **(bufs | pools(z) | dict(over)), **z, scale=0.125, **kw)


def test_attend_takes_what_it_says():
    attend()
    attend(out_type="f32", over={"out": FakeBuffer(5 * 512 * 4)}, q_type="bf16")
    attend(q_stride=520, over={"q": FakeBuffer((4 * 520 + 512) * 2)})
    for d in (16, 80, 128, 208, 256):
        attend(sizes={"head_dim": d})
    attend(sizes={"heads": 34, "window": 7, "block_size": 8})
    attend(starts=FakeBuffer(24), q_rows=9, over={"q": FakeBuffer(9 * 1024)})
    assert paged8.attend8_form(requests=1, heads=8, kv_heads=2, head_dim=64, block_size=16, blocks=9999,
                               table_len=8000) == "split"
    assert paged8.attend8_form(requests=1, heads=8, kv_heads=2, head_dim=64, block_size=16, blocks=9,
                               table_len=8) == "whole"


@pytest.mark.parametrize("sizes", [
    {"requests": 0}, {"heads": 0}, {"kv_heads": 0}, {"heads": 7}, {"head_dim": 0}, {"head_dim": 8}, {"head_dim": 72},
    {"head_dim": 272}, {"block_size": 0}, {"block_size": 4}, {"block_size": 12}, {"blocks": 0}, {"table_len": 0},
    {"table_len": 1 << 28}, {"blocks": 1 << 28}, {"requests": 1 << 24}, {"requests": 1 << 23, "table_len": 1 << 20},
    {"requests": -1}, {"window": 1 << 32}])
def test_attend_refuses_sizes(sizes):
    with pytest.raises(LaunchError):
        attend(sizes=sizes)


def test_attend_refuses_buffers_and_rows():
    b = FakeBuffer(1 << 20)
    w = FakeBuffer(1 << 26)
    for over in ({"q": FakeBuffer(5119)}, {"kpool": FakeBuffer(20 * 2 * 16 * 64 - 1)}, {"scales": FakeBuffer(319)},
                 {"vpool": FakeBuffer(100)}, {"table": FakeBuffer(99)}, {"lengths": FakeBuffer(19)},
                 {"out": FakeBuffer(5119)}, {"workspace": FakeBuffer(1000)}, {"scales": FakeBuffer(320, ptr=b.ptr + 4)},
                 {"kpool": FakeBuffer(1 << 16, ptr=b.ptr + 8)}, {"out": b, "q": b}, {"out": b, "scales": b},
                 {"workspace": w, "out": w}, {"workspace": w, "kpool": w}, {"q": FakeBuffer(5120, FakeDevice())}):
        with pytest.raises(LaunchError):
            attend(over=over)
    for kw in ({"q_type": "f32"}, {"out_type": "bf16"}, {"q_stride": 511}, {"q_stride": 513}, {"out_stride": 511},
               {"starts": FakeBuffer(24), "q_rows": 0}, {"starts": FakeBuffer(23), "q_rows": 5},
               {"starts": FakeBuffer(24), "q_rows": 6}):
        with pytest.raises(LaunchError):
            attend(**kw)


def store(over=(), **kw):
    z = {**dict(tokens=9, kv_heads=2, head_dim=64, block_size=16, blocks=20, heads=4), **kw}
    wide = 4 if z.get("rows_type", "f32") == "f32" else 2
    row = z["kv_heads"] * z["head_dim"] * wide * z["tokens"]
    bufs = dict(q=FakeBuffer(z["heads"] * z["head_dim"] * wide * z["tokens"]), k=FakeBuffer(row), v=FakeBuffer(row),
                slots=FakeBuffer(4 * z["tokens"]), qr=FakeBuffer(2 * z["heads"] * z["head_dim"] * z["tokens"]))
    return paged8.PagedStore8(DEVICE, **(bufs | pools(z) | dict(over)), **z)


ROPE = dict(positions=FakeBuffer(36), rope=FakeBuffer(100 * 32 * 8))


def test_store_takes_what_it_says_and_refuses_the_rest():
    store()
    store(over=ROPE, rotated=32, rope_rows=100)
    store(over={"q": None, "qr": None}, heads=0)
    store(tokens=0)
    for d in (16, 80, 256):
        store(head_dim=d, rows_type="bf16", q_type="bf16")
    fused = FakeBuffer(9 * 512 * 4)
    store(over={"q": fused, "k": fused, "v": fused}, q_stride=512, k_stride=512, v_stride=512, k_offset=256, v_offset=384)
    b = FakeBuffer(1 << 20)
    for kw in (dict(head_dim=72), dict(head_dim=272), dict(head_dim=0), dict(block_size=12), dict(block_size=0),
               dict(blocks=0), dict(blocks=1 << 28), dict(kv_heads=0), dict(rows_type="e4m3"), dict(q_type="f32"),
               dict(heads=0), dict(q_stride=255), dict(k_stride=130), dict(v_stride=127), dict(rotated=33),
               dict(over=ROPE, rotated=33, rope_rows=100), dict(over=ROPE, rotated=32, rope_rows=0),
               dict(over=ROPE, rotated=32, rope_rows=101), dict(rotated=32, rope_rows=100),
               dict(over={"qr": None}), dict(over={"slots": FakeBuffer(35)}), dict(over={"kpool": FakeBuffer(9)}),
               dict(over={"scales": FakeBuffer(319)}), dict(over={"qr": FakeBuffer(9 * 512 - 1)}),
               dict(over={"k": FakeBuffer(9 * 512 - 1)}), dict(over={"kpool": b, "vpool": b}),
               dict(over={"kpool": b, "k": b}), dict(over={"qr": b, "scales": b}), dict(over={"scales": b, "slots": b}),
               dict(over={"scales": FakeBuffer(320, ptr=b.ptr + 4)}), dict(k_offset=3), dict(q_offset=-4),
               dict(tokens=1 << 30, heads=1 << 20), dict(tokens=-1)):
        with pytest.raises(LaunchError):
            store(**{"over": (), **kw})


def load(over=(), **kw):
    z = {**dict(tokens=9, kv_heads=2, head_dim=64, block_size=16, blocks=20), **kw}
    row = z["kv_heads"] * z["head_dim"] * (4 if z.get("rows_type") == "f32" else 2) * z["tokens"]
    bufs = dict(slots=FakeBuffer(4 * z["tokens"]), k=FakeBuffer(row), v=FakeBuffer(row))
    return paged8.PagedLoad8(DEVICE, **(bufs | pools(z) | dict(over)), **z)


def test_load_takes_what_it_says_and_refuses_the_rest():
    load()
    load(rows_type="f32")
    load(tokens=0)
    load(over={"k": FakeBuffer(9 * 272), "v": FakeBuffer(9 * 288)}, k_stride=136, v_stride=144)
    b = FakeBuffer(1 << 20)
    for kw in (dict(head_dim=72), dict(block_size=12), dict(blocks=0), dict(kv_heads=0), dict(rows_type="f64"),
               dict(k_stride=127), dict(v_stride=132), dict(over={"slots": FakeBuffer(35)}),
               dict(over={"vpool": FakeBuffer(9)}), dict(over={"k": FakeBuffer(9 * 256 - 1)}),
               dict(over={"k": b, "v": b}), dict(over={"k": b, "kpool": b}), dict(over={"v": b, "scales": b}),
               dict(over={"v": b, "slots": b}), dict(tokens=1 << 31, kv_heads=1 << 16)):
        with pytest.raises(LaunchError):
            load(**{"over": (), **kw})


def test_unknown_sizes_of_arguments_are_refused():
    for entry in ("fk_paged_store8", "fk_paged_load8", "fk_paged_attend8"):
        with pytest.raises(runtime.FkError):
            runtime.serve_check(entry, type("Args", (paged8.ctypes.Structure,), {"_fields_": [("x", paged8._U32)]})())
