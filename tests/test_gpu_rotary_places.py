"""Rotary in place in a fused buffer whose heads lie before its tokens, and for a
single token without token strides: the bits of the call into other buffers; v's
heads stay."""
import pytest
import torch

import bwpp

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("B,T,Hq,Hk,d,rot", [(2, 33, 4, 2, 64, 64), (3, 7, 3, 1, 40, 20), (4, 1, 8, 2, 128, 128)])
def test_heads_first_in_place(be, dtype, grad, B, T, Hq, Hk, d, rot):
    H = Hq + 2 * Hk
    buf = torch.randn(B, H, T, d, device="cuda").to(dtype)
    before = buf.clone()
    call = be.dispatch_rotary_grad if grad else be.dispatch_rotary
    ld = d if T > 1 else 0

    def params(hs, qb, kb):
        kw = {}
        for n in ("q", "k", "qo", "ko"):
            kw.update({f"ld{n}": ld, f"{n}_head_stride": hs, f"{n}_batch_stride": qb if n[0] == "q" else kb})
        return bwpp.RotaryParams(tokens=T, q_heads=Hq, k_heads=Hk, dim=d, batch=B, rot_dim=rot, dtype=int(dtype == torch.bfloat16),
                                 pos_offset=100, **kw)

    q, k = before[:, :Hq].contiguous(), before[:, Hq:Hq + Hk].contiguous()
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    call(q, k, None, qo, ko, params(T * d, Hq * T * d, Hk * T * d))
    call(buf, buf[:, Hq:], None, buf, buf[:, Hq:], params(T * d, H * T * d, H * T * d))
    assert torch.equal(buf[:, :Hq], qo) and torch.equal(buf[:, Hq:Hq + Hk], ko)
    assert torch.equal(buf[:, Hq + Hk:], before[:, Hq + Hk:])
