"""Which kernels ragged products of the bf16 gradient run on: the last four
launches are dx's product on the wide tiles, what is left of its K (vocabulary)
past a multiple of 32 on others, dW's, and dx's rounding; where dx's tiles are too
few for the wide ones, its product is one on the others."""
import pytest

from test_gpu_linear_xent import BF16, _case, _forward, _gradient

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("wide", ["vd", "dv"])
@pytest.mark.parametrize("T,D,V,dx_wide,left", [(2048, 1024, 8205, True, True), (2050, 1040, 8200, True, True),
                                                (2048, 1024, 8224, True, False), (1500, 2056, 4100, False, False)])
def test_ragged_products(be, wide, T, D, V, dx_wide, left):
    x, w, t = _case(T, D, V, BF16, wide, 14, (0, -V % 8 if wide == "dv" else 0))
    t[::11] = -1
    _, lse, _ = _forward(be, x, w, t, BF16, wide)
    _gradient(be, x, w, t, lse, None, BF16, wide)
    last = [be.recent_kernel(i) for i in range(4)]
    tb = "t01" if wide == "dv" else "t00"  # dx reads W the other way round
    assert last[0].startswith("bwpp_xent_round_bf16") and last[1] == "bwpp_xent_rows_p_t10", last
    if left:
        assert last[2].startswith("bwpp_xent_sums_r") and f"_{tb}" in last[2], last
    product = last[3 if left else 2]
    assert product == f"bwpp_xent_sums_p_{tb}" if dx_wide else product.startswith("bwpp_xent_sums_r"), last
