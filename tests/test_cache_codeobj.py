"""The code objects that hold the paged cache's and the rules' kernels hold those
that the runtime names and no others of them, their direct-to-LDS loads follow the
rule for M0, and they have no packed fp32 instructions."""
import os
import re
import shutil
import subprocess

import pytest

from bwpp import _lib
from test_codeobj_m0 import LIB, LLVM, _asm
from test_codeobj_m0 import test_m0_written_only_by_lds_dma_asm as check_m0

OBJECTS = ("rowops", "attention_f32")


def kernel_names():
    src = open(os.path.join(_lib.PKG_DIR, "csrc", "runtime", "bwpp_cache.cpp")).read()
    return re.findall(r'^    "(bwpp_(?:cache|logit)_\w+)",$', src, flags=re.M)


@pytest.mark.parametrize("kernel", OBJECTS)
def test_instructions(kernel, tmp_path):
    check_m0(kernel, tmp_path)
    lines = _asm(kernel, tmp_path)
    assert not [ln for ln in lines if ln.startswith(("v_pk_add_f32", "v_pk_mul_f32", "v_pk_fma_f32"))]


def test_kernels_are_in_their_code_objects(tmp_path):
    names, have = kernel_names(), []
    assert len(names) > 50 and len(set(names)) == len(names)
    dump = os.path.join(LLVM, "llvm-objdump")
    for kernel in OBJECTS:
        bundle, obj = os.path.join(LIB, f"bwpp_{kernel}.hsaco"), tmp_path / f"{kernel}.o"
        if not (os.path.exists(bundle) and shutil.which(dump)):
            pytest.skip("code object or ROCm LLVM tools not present")
        subprocess.run([os.path.join(LLVM, "clang-offload-bundler"), "--unbundle", "--type=o", f"--input={bundle}",
                        "--targets=hipv4-amdgcn-amd-amdhsa--gfx950", f"--output={obj}"], check=True)
        out = subprocess.run([dump, "--syms", str(obj)], check=True, capture_output=True, text=True).stdout
        have += [n for n in (ln.split()[-1] for ln in out.splitlines() if " F .text" in ln)
                 if n.startswith(("bwpp_cache", "bwpp_logit"))]
    assert sorted(have) == sorted(names)
