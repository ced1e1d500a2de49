"""The machine code of the reorder's second launch, on the CPU: no spilled registers, no private stack."""
import pytest

from test_isa import device_asm, kernels, no_spills


@pytest.mark.timeout(600)
def test_no_spills(tmp_path):
    found = 0
    for n, _, meta in kernels(device_asm(tmp_path, "block_tables"), "tables_finish_kernel"):
        no_spills(meta, n)
        found += 1
    assert found == 1
