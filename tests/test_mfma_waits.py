"""Build-time guard for the matrix-instruction kernels: no vector instruction may read the result of a
v_mfma before the wait states it needs (scripts/audit_mfma_waits.py).  hipcc cross-compiles without a GPU, so this
runs in the CPU suite; the audit is also checked to catch a planted violation."""
import glob
import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

import pytest

from conftest import ROOT

sys.path.insert(0, os.path.join(ROOT, "scripts"))
import audit_mfma_waits as A  # noqa: E402

HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
FLAGS = ["-O3", "-std=c++17", "--offload-arch=gfx950", "-munsafe-fp-atomics", "-Xclang", "-target-feature",
         "-Xclang", "-packed-fp32-ops", "--cuda-device-only", "-S"]


def test_no_kernel_reads_a_matrix_result_too_early(tmp_path):
    if not os.path.exists(HIPCC):
        pytest.skip("no hipcc")
    srcs = [s for s in sorted(glob.glob(os.path.join(ROOT, "kge-1_amd", "csrc", "*.hip")))
            if "mfma" in open(s).read()]
    assert len(srcs) >= 5

    def build(src):
        out = tmp_path / (os.path.basename(src) + ".s")
        subprocess.run([HIPCC] + FLAGS + [src, "-o", str(out)], check=True, capture_output=True)
        return out

    with ThreadPoolExecutor(max_workers=4) as pool:
        outs = list(pool.map(build, srcs))
    assert sum(open(out).read().count("v_mfma") for out in outs) > 1000
    bad = {out.name: found for out in outs if (found := A.audit_file(str(out)))}
    assert not bad, bad


def _findings(body):
    lines = body.split("\n")
    (name, a, b), = A.functions(lines)
    return A.audit(lines, a, b)


BODY = """k:
.LBB0_1:
\tv_mfma_f32_16x16x32_bf16 a[0:3], v[0:3], v[4:7], a[0:3]
\ts_cbranch_scc0 .LBB0_1
.LBB0_2:
%s\tv_accvgpr_read_b32 v8, a0
\ts_endpgm
.Lfunc_end0:
"""


def test_audit_flags_a_read_without_its_wait():
    (found,) = _findings(BODY % "")
    assert found[1] == "v_accvgpr_read_b32 v8, a0" and found[2] == 6  # 7 needed, the branch is one
    assert _findings(BODY % "\ts_nop 4\n") and not _findings(BODY % "\ts_nop 5\n")
    # across the loop's own edge, and for the operands (not the accumulator) of another matrix instruction
    assert _findings((BODY % "\ts_nop 5\n").replace(".LBB0_1:\n", ".LBB0_1:\n\tv_mov_b32_e32 v9, a2\n"))
    assert _findings((BODY % "\ts_nop 5\n").replace("v[4:7], a[0:3]\n\ts_c", "v[4:7], a[0:3]\n"
                                                    "\tv_mfma_f32_16x16x32_bf16 v[12:15], a[0:3], v[4:7], v[12:15]\n\ts_c"))
    # fp32 inputs: 8 passes
    slow = (BODY % "\ts_nop 7\n").replace("16x16x32_bf16", "16x16x4_f32")
    assert _findings(slow) and not _findings(slow.replace("s_nop 7", "s_nop 8"))
