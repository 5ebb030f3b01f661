"""The kernels of the operators around a block share two code objects: those
hold them, the direct-to-LDS loads of the cross entropy's products follow the
rule for M0 (gemm's code object), and none has packed fp32 instructions."""
import os
import re
import shutil
import subprocess

import pytest

from bwpp import _lib
from test_codeobj_m0 import LIB, LLVM, _asm
from test_codeobj_m0 import test_m0_written_only_by_lds_dma_asm as check_m0


@pytest.mark.parametrize("kernel", ["gemm", "rowops"])
def test_instructions(kernel, tmp_path):
    check_m0(kernel, tmp_path)
    assert not [ln for ln in _asm(kernel, tmp_path) if ln.startswith(("v_pk_add_f32", "v_pk_mul_f32", "v_pk_fma_f32"))]


def test_kernels_are_in_their_code_objects(tmp_path):
    src = open(os.path.join(_lib.PKG_DIR, "csrc", "runtime", "bwpp_lm.cpp")).read()
    names = set(re.findall(r'"(bwpp_(?:rotary|resnorm|xent)_\w+)"', src))
    assert len(names) > 60
    have = set()
    dump = os.path.join(LLVM, "llvm-objdump")
    for kernel in ("gemm", "rowops"):
        bundle, obj = os.path.join(LIB, f"bwpp_{kernel}.hsaco"), tmp_path / f"{kernel}.o"
        if not (os.path.exists(bundle) and shutil.which(dump)):
            pytest.skip("code object or ROCm LLVM tools not present")
        subprocess.run([os.path.join(LLVM, "clang-offload-bundler"), "--unbundle", "--type=o", f"--input={bundle}",
                        "--targets=hipv4-amdgcn-amd-amdhsa--gfx950", f"--output={obj}"], check=True)
        out = subprocess.run([dump, "--syms", str(obj)], check=True, capture_output=True, text=True).stdout
        have |= {ln.split()[-1] for ln in out.splitlines() if " F .text" in ln}
    assert names <= have, names - have
    # and no such kernel that nothing names
    assert {k for k in have if re.match(r"bwpp_(rotary|resnorm|xent)_", k)} == names
