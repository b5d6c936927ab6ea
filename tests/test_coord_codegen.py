"""What the compiler is told about the coordinator-side kernels' exchanges through LDS (no GPU): in the wave that turns rows
round in a corner of its own, writes and other lanes' reads are kept apart by a fence in both directions."""
import os
import subprocess

import pytest

from mimo26f_afd_amd import build

PROGRAM = """#include "w4_kernels.h"
template __global__ void m26g::w4_streamed_kernel<8, 1>(const m26g::W4Args, int);
template __global__ void m26g::w4_resident_kernel<1, 2, 16, false, float>(const m26g::W4Args, int, int, int, int, int);
"""


@pytest.fixture(scope="module")
def functions(tmp_path_factory):
    """Name -> lines of the optimised intermediate code."""
    at = tmp_path_factory.mktemp("w4")
    (at / "w4.hip").write_text(PROGRAM)
    flags = [f for f in build.FLAGS if f not in ("-shared", "-fPIC")]
    out = at / "w4.ll"
    subprocess.run([build.hipcc(), *flags, "-I", os.path.join(build.HERE, "csrc"), "--cuda-device-only", "-S", "-emit-llvm", str(at / "w4.hip"), "-o", str(out)],
                   check=True, capture_output=True)
    found, lines = {}, None
    for line in out.read_text().splitlines():
        if line.startswith("define "):
            lines = found.setdefault(line.split("@")[1].split("(")[0], [])
        elif line == "}":
            lines = None
        elif lines is not None:
            lines.append(line.strip())
    return found


@pytest.mark.parametrize("kernel", ["w4_streamed_kernel", "w4_resident_kernel"])
def test_rows_turned_round_in_lds_are_fenced_both_ways(functions, kernel):
    lines = next(v for k, v in functions.items() if kernel in k)
    last, turns, bare = None, 0, []
    for line in lines:
        if line.startswith("fence ") or "s.barrier" in line:
            last = None
        elif "ptr addrspace(3)" in line and (line.startswith("store ") or " = load " in line):
            kind = "write" if line.startswith("store ") else "read"
            if last and last != kind:
                bare.append(line)
            turns += last != kind
            last = kind
    assert turns >= 4, "no exchange through LDS found"
    assert not bare, bare[:4]
