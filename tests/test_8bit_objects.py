"""The 8-bit operators' kernels (include/fkrocm_fp8.h, fkrocm_paged8.h) as
compiled into the C ABI's library, from their own metadata: none keeps anything
in private memory, and each is there."""

import re

from test_serve_objects import kernels  # noqa: F401  (a fixture)


def test_the_operators_kernels_use_no_private_memory(kernels):  # noqa: F811
    found = {k: v for k, v in kernels.items() if re.search(r"op_(fp8|pages8)_", k)}
    kinds = {re.search(r"op_((?:fp8|pages8)_(?:quantize|dequantize|add_norm|gemm_few|gemm_mid|gemm_many|store|load|"
                       r"attend|join))", k).group(1) for k in found}
    assert len(kinds) == 10
    for name, k in found.items():
        assert k[".private_segment_fixed_size"] == 0 and k[".vgpr_spill_count"] == 0, name


def test_the_large_products_sums_stay_in_accumulation_registers(kernels):  # noqa: F811
    many = [v for k, v in kernels.items() if "op_fp8_gemm_many" in k]
    assert len(many) == 3 and all(k[".agpr_count"] == 256 for k in many)
