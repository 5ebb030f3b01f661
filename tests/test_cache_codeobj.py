"""The code objects of the paged cache and the rules on logits hold the kernels
that the runtime names and no others, their direct-to-LDS loads follow the rule
for M0, and they have no packed fp32 instructions."""
import os
import re
import shutil
import subprocess

import pytest

from bwpp import _lib
from test_codeobj_m0 import IMPLICIT, LIB, LLVM, _asm

OBJECTS = ("cache", "cache_bf16")


def kernel_names():
    src = open(os.path.join(_lib.PKG_DIR, "csrc", "runtime", "bwpp_cache.cpp")).read()
    return re.findall(r'^    "(bwpp_(?:cache|logit)_\w+)",$', src, flags=re.M)


@pytest.mark.parametrize("kernel", OBJECTS)
def test_instructions(kernel, tmp_path):
    lines = _asm(kernel, tmp_path)
    assert len(lines) > 100
    for i, ins in enumerate(lines):
        assert not IMPLICIT.search(ins), f"instruction reads M0 implicitly: {ins}"
        after = lines[i + 1] if i + 1 < len(lines) else ""
        if re.search(r"\bm0\b", ins):  # from a scalar register (VCC is one), right before its load
            assert re.match(r"s_mov_b32 m0, (s\d+|vcc_lo|vcc_hi)$", ins) and after.startswith("global_load_lds_dwordx4"), (ins, after)
        if ins.startswith("global_load_lds_dwordx4"):
            assert i > 0 and lines[i - 1].startswith("s_mov_b32 m0,"), ins
    assert not [ln for ln in lines if ln.startswith(("v_pk_add_f32", "v_pk_mul_f32", "v_pk_fma_f32"))]
    assert any(ln.startswith("global_load_lds_dwordx4") for ln in lines) == (kernel == "cache_bf16")


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
        have += [ln.split()[-1] for ln in out.splitlines() if " F .text" in ln]
    assert sorted(have) == sorted(names)
