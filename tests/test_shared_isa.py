"""The machine code of the kernels for shared prefixes, beams and block tables, on the CPU: no spilled
registers, no private stack, and every K/V load from a scalar descriptor."""
import pytest

from test_isa import device_asm, kernels, no_spills


@pytest.mark.timeout(600)
@pytest.mark.parametrize("src,prefix,streams", [
    ("shared_decode", "shared_read_kernel", True), ("shared_decode", "shared_join_kernel", False),
    ("beam_select", "beam_rows_kernel", False), ("beam_select", "beam_merge_kernel", False),
    ("block_tables", "tables_plan_kernel", False), ("block_tables", "tables_apply_kernel", False),
    ("block_tables", "tables_reorder_kernel", False), ("block_tables", "tables_init_kernel", False)])
def test_no_spills_and_scalar_descriptors(tmp_path, src, prefix, streams):
    for n, body, meta in kernels(device_asm(tmp_path, src), prefix):
        no_spills(meta, n)
        lines = body.splitlines()
        loads = [k for k, line in enumerate(lines) if "buffer_load_dwordx4" in line]
        assert bool(loads) == streams, n
        for k in loads:
            assert "s_and_saveexec" not in " ".join(lines[max(0, k - 3):k]), f"{n}: a load in a loop over lanes"
