"""The one-call operators' kernels (include/fkrocm_serve.h, fkrocm_mx4.h) as
compiled into the C ABI's library, from their own metadata: none keeps
anything in private memory (arguments chosen by pointer, sums rounded ahead of
their turn: still correct, many times slower), and each is there."""

import re

import pytest

from furykernel_amd.runtime import LIBRARY
from test_code_objects import kernel_metadata

MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"


class Bundle:
    """One translation unit's code objects, as kernel_metadata reads a file."""

    def __init__(self, data):
        self.data = data

    def read_bytes(self):
        return self.data


@pytest.fixture(scope="module")
def kernels():
    if not LIBRARY.exists():
        pytest.skip("the library is not built (run __graft_entry__.build())")
    data = LIBRARY.read_bytes()
    out = {}
    for m in re.finditer(re.escape(MAGIC), data):
        out.update(kernel_metadata(Bundle(data[m.start():])))
    return out


def test_the_operators_kernels_use_no_private_memory(kernels):
    found = {k: v for k, v in kernels.items() if re.search(r"op_(page|paged|mx4)_", k)}
    kinds = {re.search(r"op_(page_plan_held|page_plan|paged_store|paged_attend_join|paged_attend|mx4_quantize|"
                       r"mx4_dequantize|mx4_gemm_few|mx4_gemm_mid|mx4_gemm_many)", k).group(1) for k in found}
    assert len(kinds) == 10
    for name, k in found.items():
        assert k[".private_segment_fixed_size"] == 0 and k[".vgpr_spill_count"] == 0, name


def test_the_large_products_sums_stay_in_accumulation_registers(kernels):
    many = [v for k, v in kernels.items() if "op_mx4_gemm_many" in k]
    assert len(many) == 3 and all(k[".agpr_count"] == 256 for k in many)
