"""The windows of keys that masked attention's loops run over are integers all the way: some of its files are compiled with
NaNs left out of account (build.py), and there a negative integer's bits, carried as a float, are a value that the compiler may
take for any other.  Read from the compiler's output before any optimization, for the flags of those files."""
import importlib.util
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOURCE = """
#include "masked_attention.h"
namespace ffk {
extern "C" __global__ void windows(int const *in, int *out) {
  out[0] = wave_min_int(in[threadIdx.x]);
  out[1] = wave_max_int(in[threadIdx.x]);
}
}
"""


def builder():
    spec = importlib.util.spec_from_file_location("ffk_build", os.path.join(ROOT, "flexflow-train_amd", "build.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("name", ["masked_attention_heads_fwd.hip", "masked_attention_heads_rows.hip"])
def test_windows_are_integers(name, tmp_path):
    build = builder()
    assert "-fno-honor-nans" in build.EXTRA_FLAGS[name]
    (tmp_path / "windows.hip").write_text(SOURCE)
    subprocess.run([build.HIPCC] + build.HIP_FLAGS + build.EXTRA_FLAGS[name]
                   + ["-I" + build.CSRC, "--cuda-device-only", "-S", "-emit-llvm", "-Xclang", "-disable-llvm-passes",
                      str(tmp_path / "windows.hip"), "-o", str(tmp_path / "windows.ll")], check=True, capture_output=True)
    text = (tmp_path / "windows.ll").read_text()
    functions = {m.group(1).strip('"'): m.group(0) for m in re.finditer(r'^define [^\n]*@("[^"]+"|[\w.$]+)\(.*?^}', text, re.S | re.M)}
    reached, work = set(), ["windows"]
    while work:
        at = work.pop()
        if at in reached or at not in functions:
            continue
        reached.add(at)
        work += [n.strip('"') for n in re.findall(r'@("[^"]+"|[\w.$]+)', functions[at])]
    assert len(reached) >= 3, reached  # the two reductions, and what they call
    wrong = sorted(n for n in reached if re.search(r"\b(float|double|half|bfloat)\b", functions[n]))
    assert not wrong, wrong
