"""What the one-call operators' kernels leave in flight at their barriers, from
the instructions of the library's own code objects: a wavefront whose reads of
LDS are still out when it arrives may have them overwritten by another's loads
behind the barrier.

The large product (op_mx4_gemm_many) is left out: it arrives with reads out, of
a stage that is loaded again two barriers later, behind the products that wait
for them."""

import re
import subprocess

import pytest

from furykernel_amd.runtime import LIBRARY
from test_code_objects import device_elf
from test_serve_objects import MAGIC

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"


def instructions(text):
    """{function: [(address, mnemonic, operands, first word)]} of a listing."""
    out, now = {}, None
    for line in text.splitlines():
        if m := re.match(r"[0-9a-f]+ <(.+)>:$", line):
            now = out.setdefault(m.group(1), [])
        elif m := re.match(r"\s+(\S+)\s*(.*?)\s*// ([0-9A-F]+): ([0-9A-F]{8})", line):
            now.append((int(m.group(3), 16), m.group(1), m.group(2), int(m.group(4), 16)))
    return out


def reads_out_at_barriers(code):
    """The most LDS operations that may be in flight at each barrier, over
    every path to it: (address, how many)."""
    index = {at: i for i, (at, *_) in enumerate(code)}
    entry, work, found = {0: 0}, [0], {}
    while work:
        i = work.pop()
        n = entry[i]
        while i < len(code):
            at, op, operands, word = code[i]
            if op.startswith("ds_"):
                n = min(n + 1, 15)    # (all that the counter tells apart)
            elif op == "s_waitcnt" and (m := re.search(r"lgkmcnt\((\d+)\)", operands)):
                n = min(n, int(m.group(1)))
            elif op == "s_barrier":
                found[at] = max(found.get(at, 0), n)
            go = []
            if op.startswith("s_cbranch") or op == "s_branch":
                step = (word & 0xFFFF) - ((word & 0x8000) << 1)
                go.append(index[at + 4 + 4 * step])
            if op not in ("s_branch", "s_endpgm"):
                go.append(i + 1)
            if len(go) == 1 and go[0] == i + 1:
                i += 1
                continue
            for j in go:
                if j not in entry or entry[j] < n:
                    entry[j] = n
                    work.append(j)
            break
    return sorted(found.items())


@pytest.fixture(scope="module")
def listing(tmp_path_factory):
    if not LIBRARY.exists():
        pytest.skip("the library is not built (run __graft_entry__.build())")
    data, out = LIBRARY.read_bytes(), {}
    for i, m in enumerate(re.finditer(re.escape(MAGIC), data)):
        path = tmp_path_factory.mktemp("objects") / f"{i}.elf"
        path.write_bytes(device_elf(data[m.start():]))
        text = subprocess.run([OBJDUMP, "-d", str(path)], capture_output=True, text=True, check=True).stdout
        out.update({k: v for k, v in instructions(text).items() if re.search(r"op_(page|paged|mx4)_", k)})
    return out


@pytest.mark.parametrize("kernel,count", [("op_mx4_gemm_mid", 3), ("op_mx4_gemm_few", 12), ("op_paged_attendI", 20),
                                          ("op_paged_attend_join", 6), ("op_page_plan", 5)])
def test_no_wavefront_arrives_with_reads_of_lds_in_flight(listing, kernel, count):
    found = {k: reads_out_at_barriers(v) for k, v in listing.items() if kernel in k}
    assert len(found) == count and all(found.values())
    late = {k: [(hex(at), n) for at, n in v if n] for k, v in found.items()}
    assert not any(late.values()), {k: v for k, v in late.items() if v}


def test_a_planted_read_is_found():
    """The walk itself: a read that a loop's end leaves out reaches the barrier
    at its head; a wait before the barrier takes it away."""
    loop = [(0, "s_barrier", "", 0), (4, "ds_read_b128", "v[0:3], v4", 0), (12, "s_waitcnt", "lgkmcnt(1)", 0),
            (16, "s_cbranch_scc1", "65531", 0xBF85FFFB), (20, "s_endpgm", "", 0)]
    assert reads_out_at_barriers(loop) == [(0, 1)]
    loop[2] = (12, "s_waitcnt", "vmcnt(0) lgkmcnt(0)", 0)
    assert reads_out_at_barriers(loop) == [(0, 0)]
