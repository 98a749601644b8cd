"""Registers, LDS and K loops of the compiled kernels of the int8 linear and
of the linears grouped by expert (CPU: hipcc cross-compiles for gfx950).

Their copies are counted by waits of their own (inline asm); a wait of the
compiler's in a K loop, or a spilled register read back there, would wait for
the copies just issued.  The 256 x 256 kernels keep a few registers of their
stores in scratch memory, outside the K loops.
"""

import re

import pytest
from test_kernel_resources import CSRC, kernel_metadata


def mfma_loops(asm, name):
    """The innermost loops of `name` that hold an MFMA: (instruction, inside
    inline asm) of the blocks that the listing's comments give to each."""

    start = asm.index(name + ":")
    loops, header, inasm = {}, None, False
    for line in asm[start:asm.index(".Lfunc_end", start)].split("\n"):
        s = line.strip()
        if s.startswith(";;#ASM"):
            inasm = s.startswith(";;#ASMSTART")
        elif s.startswith((".LBB", "; %bb.")):
            inside = re.search(r"in Loop: Header=(BB\d+_\d+)", s)
            header = s.split(":")[0][2:] if "Loop Header" in s else inside and inside.group(1)
        elif header and s and not s.startswith((";", ".")):
            loops.setdefault(header, []).append((s, inasm))
    return [lp for lp in loops.values() if any(t.startswith("v_mfma") for t, _ in lp)]


@pytest.mark.parametrize("source", ["grouped", "int8_linear"])
def test_product_kernels(source, tmp_path):
    src = CSRC / f"{source}.hip"
    meta = kernel_metadata(src, tmp_path)
    asm = (tmp_path / f"{source}.s").read_text()
    products = [k for k in meta if "product_tile_kernel" in k or "product_gemm_kernel" in k or "int8_few_kernel" in k]
    assert len(products) >= 8
    for name in products:
        m = meta[name]
        assert m["group_segment_fixed_size"] <= 160 * 1024, name
        if "product_tile_kernel" in name:  # two workgroups per CU and more
            assert m["group_segment_fixed_size"] <= 80 * 1024 and m["vgpr_count"] <= 128, name
        assert m["vgpr_spill_count"] == 0 or "Li256ELi256E" in name, name
        loops = mfma_loops(asm, name)
        assert loops, name
        for body in loops:
            assert [s for s, _ in body if s.startswith("scratch_")] == [], name
            if "few" not in name:  # reads the scales of a strip at its end
                assert [s for s, a in body if not a and s.startswith("s_waitcnt") and "vmcnt" in s] == [], name
