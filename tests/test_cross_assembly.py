"""The bf16 stages of the attention to an encoder's states go from global memory straight into LDS by inline assembly, where the
compiler's hazard handling does not reach: a scalar register written by a vector instruction must not be read by a memory instruction
within five wait states.  The device assembly of that source is emitted and every block scanned (half a minute of compilation)."""
import os

from spion_amd import build


def test_no_assembly_block_reads_a_vector_written_scalar_too_early(tmp_path):
    out = build.emit_device_asm("cross_attention.hip", os.path.join(tmp_path, "cross_attention.s"))
    blocks, found = build.scan_sgpr_hazards(open(out).read())
    assert blocks > 100, blocks  # the loads into LDS are there and were seen
    assert not found, f"{len(found)} sites, first: {found[0]}"
