"""The cross entropy's code object has the matrix products' direct-to-LDS loads:
the same check of M0 as theirs.  The other two have none."""
import pytest

from test_codeobj_m0 import _asm
from test_codeobj_m0 import test_m0_written_only_by_lds_dma_asm as check_m0  # noqa: F401


@pytest.mark.parametrize("kernel", ["xent", "rotary", "resnorm"])
def test_m0(kernel, tmp_path):
    check_m0(kernel, tmp_path)
    has = any(ln.startswith("global_load_lds_dwordx4") for ln in _asm(kernel, tmp_path))
    assert has == (kernel == "xent")


def test_no_packed_fp32(tmp_path):
    """Compiled without packed fp32 instructions."""
    for kernel in ("xent", "rotary", "resnorm"):
        assert not [ln for ln in _asm(kernel, tmp_path) if ln.startswith(("v_pk_add_f32", "v_pk_mul_f32", "v_pk_fma_f32"))]
