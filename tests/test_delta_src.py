"""Orderings in csrc/delta.hip that no result shows while the hardware and the compiler happen to keep them: each is asked
of the source."""
import os

import pytest

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "startlux-prism_amd", "csrc", "delta.hip")


def body(name):
    """The code of the function, comments taken out."""
    src = "\n".join(line.split("//")[0] for line in open(PATH).read().splitlines())
    at = src.index("{", src.index(name + "("))
    depth = 0
    for i in range(at, len(src)):
        depth += {"{": 1, "}": -1}.get(src[i], 0)
        if depth == 0:
            return src[at:i]
    raise AssertionError(name)


@pytest.mark.parametrize("name,write,read", [
    ("delta_rec_kernel", "kq[wave][1][e * 64 + lane] =", "= kq[wave][0][rg"),
    ("delta_prep_kernel", "const v4f row = *reinterpret_cast<const v4f*>(d +", "d[i * LD + col] ="),
])
def test_lanes_of_a_wave_exchange_in_order(name, write, read):
    """Between a wave's LDS accesses of one side and the other lanes' of the same words stands the wave's ordering point."""
    code = body(name)
    assert code.count(write) == code.count(read) == 1
    assert "wave_lds_order();" in code[code.index(write):code.index(read)]
    order = body("wave_lds_order")
    assert "__builtin_amdgcn_fence(__ATOMIC_ACQ_REL" in order and "__builtin_amdgcn_wave_barrier()" in order


def test_the_last_touches_have_landed_before_the_workgroup_ends():
    """scan_out's touched lines come by DMA into LDS that nobody reads: they are waited for before its last barrier, outside
    the loop over the chunks."""
    code = body("scan_out")
    loop = code.index("for (int c = 0; c < at.nc; c++) {")
    end = code.rindex("lds_barrier();")
    assert loop < code.index("touch(rec +") < code.rindex("vm_wait<0>();", 0, end) < end
    between = code[code.rindex("}", 0, end):end]
    assert "vm_wait<0>();" in between
