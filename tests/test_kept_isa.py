"""The machine code of the gkv_kept_* kernels and the block copy, on the CPU: no spilled
registers, no private stack, and every buffer load from a scalar descriptor."""
import pytest

from test_isa import device_asm, kernels, no_spills


@pytest.mark.timeout(600)
@pytest.mark.parametrize("src,prefix,streams", [
    ("kept_append", "kept_append_kernel", False), ("kept_decode", "kept_decode_whole_kernel", True),
    ("kept_decode", "kept_decode_split_kernel", True), ("kept_decode", "kept_decode_merge_kernel", False),
    ("kept_prefill", "kept_prefill_kernel", True), ("block_copy", "copy_blocks_kernel", False)])
def test_no_spills_and_scalar_descriptors(tmp_path, src, prefix, streams):
    for n, body, meta in kernels(device_asm(tmp_path, src), prefix):
        no_spills(meta, n)
        lines = body.splitlines()
        loads = [k for k, line in enumerate(lines) if "buffer_load_dwordx4" in line]
        assert bool(loads) == streams, n
        for k in loads:
            assert "s_and_saveexec" not in " ".join(lines[max(0, k - 3):k]), f"{n}: a load in a loop over lanes"
