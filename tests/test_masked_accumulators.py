"""The accumulators of the masked attention kernels that matrix instructions written out keep in accumulation registers
(csrc/masked_attention_heads_*.hip, mma_kept): the compiler neither sees that their results take time nor puts wait states
in front of them, so the built library is read for the distances."""
import os

import pytest

from test_wait_states import LLVM, disassembled, registers

pytestmark = pytest.mark.skipif(not os.path.exists(LLVM + "llvm-objdump"), reason="no disassembler here")
OP = "v_mfma_f32_32x32x16_bf16"


@pytest.fixture(scope="module")
def kernels(ffk, tmp_path_factory):
    return [(n, c) for n, c in disassembled(ffk.LIB_PATH, tmp_path_factory.mktemp("library")) if "masked" in n]


def test_accumulators_are_settled(kernels):
    """v_mfma_f32_32x32x16_bf16 takes eight passes: eleven wait states before anything but another of them touches a result
    (sixteen are asked for), two behind a vector instruction that writes an operand (four)."""
    checked, wrong, seen_kernels = 0, [], 0
    for name, code in kernels:
        results = {i: registers(code.args[i][0]) for i, op in enumerate(code.op) if op == OP and code.args[i][0].startswith("a[")}
        if not results:
            continue
        seen_kernels += 1
        used = [frozenset().union(*map(registers, args)) for args in code.args]
        touches = frozenset().union(*results.values())
        for i, op in enumerate(code.op):
            if i in results:
                wanted, states = frozenset().union(*(registers(a) for a in code.args[i][1:4])), 4
            elif not op.startswith("s_") and used[i] & touches:
                wanted, states = used[i] & touches, 16
            else:
                continue
            checked += 1
            work, seen = [(p, 0) for p in code.before[i]], set()
            while work:
                at, passed = work.pop()
                if (at, passed) in seen or passed >= states:
                    continue
                seen.add((at, passed))
                if i in results:
                    bad = code.op[at].startswith("v_") and not code.op[at].startswith("v_mfma") and registers(code.args[at][0]) & wanted
                else:
                    bad = at in results and results[at] & wanted
                if bad:
                    wrong.append((name, code.op[at], code.args[at], op, code.args[i], passed))
                work += [(p, passed + code.wait_states(at)) for p in code.before[at]]
    assert seen_kernels >= 8 and checked > 500
    assert not wrong, "%d of %d, for instance %s" % (len(wrong), checked, wrong[:3])
