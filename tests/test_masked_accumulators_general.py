"""The wait states that test_masked_accumulators.py reads the built library for, in the masked attention kernels that it passes
over: those that bring their tiles through registers (csrc/masked_attention_bwd.h, bf16 heads past 128), which have no direct
load to be found by."""
import glob
import os
import re
import shutil
import subprocess

import pytest

from test_masked_accumulators import OP
from test_masked_accumulators import test_accumulators_are_settled as settled
from test_wait_states import KERNEL, LLVM, Code

pytestmark = pytest.mark.skipif(not os.path.exists(LLVM + "llvm-objdump"), reason="no disassembler here")


# the instances that mma_kept is in
KINDS = {"masked_dkdv_kernelIDF16bLi256E": 12, "masked_dkdv_heads_kernel": 16, "masked_fwd_heads_kernel": 20}


@pytest.fixture(scope="module")
def bodies(ffk, tmp_path_factory):
    """{name: text} of the masked attention kernels whose matrix instructions are written out."""
    where, found = tmp_path_factory.mktemp("library"), {}
    shutil.copy(ffk.LIB_PATH, where / "lib.so")
    subprocess.run([LLVM + "llvm-objdump", "--offloading", "lib.so"], cwd=where, check=True, capture_output=True)
    for path in sorted(glob.glob(str(where / "lib.so.*gfx950"))):
        text = subprocess.run([LLVM + "llvm-objdump", "-d", "--no-show-raw-insn", path], check=True, capture_output=True, text=True).stdout
        found.update({name: body for name, body in KERNEL.findall(text) if any(kind in name for kind in KINDS) and OP + " a[" in body})
    return found


def general(bodies):
    return {n: b for n, b in bodies.items() if "masked_dkdv_kernel" in n}


def test_every_kind_of_kernel_is_read(bodies):
    """Score variants times head sizes of each; dV and dK of heads past 128 are instances of their own, with three kinds of cap."""
    assert {kind: sum(kind in n for n in bodies) for kind in KINDS} == KINDS


def test_general_kernels_are_settled(bodies):
    settled([(n, Code(b)) for n, b in general(bodies).items()])


def test_a_missing_wait_is_found(bodies):
    """The same kernels with a result read right behind the instruction that computes it, in the text."""
    line = re.compile(r"^\t" + OP + r" a\[(\d+):\d+\].*?// ([0-9A-F]+):.*$", re.M)
    planted = {n: line.sub(lambda m: m.group(0) + "\n\tv_accvgpr_read_b32 v0, a%s // %s: 00000000" % m.groups(), b, count=1)
               for n, b in general(bodies).items()}
    assert all(planted[n] != b for n, b in general(bodies).items())
    with pytest.raises(AssertionError, match="^%d of " % len(planted)):
        settled([(n, Code(b)) for n, b in planted.items()])
