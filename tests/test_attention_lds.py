"""Where objects in LDS lie: what a kernel reads and writes 8 or 16 bytes at a time starts on such a boundary, behind whatever
else a kernel keeps there."""
import os
import re
import shutil
import subprocess

import pytest

from test_beam_barriers import PKG, _flags

SOURCE = """#include "attend_step.h"
#include "attend_many.h"
static_assert(alignof(ChooseLds<1>) %% 16 == 0 && sizeof(ChooseLds<1>) %% 16 == 0, "counts are read 16 bytes at a time, in an array of these");
static_assert(alignof(ChooseLds<8>) %% 16 == 0, "counts are read 16 bytes at a time");
static_assert(sizeof(JoinLds<4>::sum[0]) %% 8 == 0 && sizeof(JoinLds<8>::sum[0]) %% 8 == 0 && kJoinPad %% 2 == 0, "sums are written 8 bytes at a time");
template __global__ void %s;
"""


@pytest.mark.skipif(shutil.which("hipcc") is None, reason="needs hipcc")
@pytest.mark.parametrize("kernel", ["attend_step_kernel<32, 1, 4>(AttendArgs, SelectArgs)", "attend_few_kernel<32, 1, 8, 4>(AttendArgs, int)",
                                    "attend_few_kernel<256, 3, 4, 16>(AttendArgs, int)", "attend_many_kernel<32, 1, 8, 2>(AttendArgs, int)"])
def test_vectors_in_lds_lie_on_their_boundaries(tmp_path, kernel):
    (src, ir) = (tmp_path / "kernels.hip", tmp_path / "kernels.ll")
    src.write_text(SOURCE % kernel)
    r = subprocess.run(["hipcc", "-x", "hip", *_flags(), "-I", os.path.join(PKG, "csrc"), "--cuda-device-only", "-S", "-emit-llvm",
                        str(src), "-o", str(ir)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-1000:]
    text = ir.read_text()
    arrays = re.findall(r"^@(\S+) = external .*addrspace\(3\) global \[0 x i8\].*align (\d+)", text, re.M)
    assert len(arrays) == 1 and int(arrays[0][1]) >= 16, arrays
