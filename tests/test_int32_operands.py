"""Targets and positions are 32-bit integers; torch's own are 64-bit, and are
refused before any address is taken.  (No GPU: tensors that say they are on one,
and a backend without a handle, which the library refuses behind the checks.)"""
import pytest
import torch

import bwpp
from bwpp import _lib, plan

ADDR = [0x100000000 * (i + 1) for i in range(6)]


class OnDevice:
    """A CPU tensor that says it is on the GPU; its address is never read."""
    is_cuda = True

    def __init__(self, t):
        self.t = t

    def __getattr__(self, name):
        return getattr(self.t, name)


@pytest.fixture
def backend():
    b = object.__new__(bwpp.HipBackend)
    b.lib, b._h = _lib.load(), None
    return b


def _calls(b, ints):
    x, w, o, p, q, r = ADDR
    rot = bwpp.RotaryParams(tokens=4, q_heads=2, dim=8, batch=2, pos_batch_stride=4)
    xe = bwpp.LinearXentParams(rows=8, vocab=10, dim=8, trans_w=1)
    return {"positions": [lambda: b.dispatch_rotary(x, None, ints, o, None, rot),
                          lambda: b.dispatch_rotary_grad(x, None, ints, o, None, rot)],
            "targets": [lambda: b.dispatch_linear_xent(x, w, ints, o, None, None, xe),
                        lambda: b.dispatch_linear_xent_grad(x, w, ints, p, None, q, r, xe)]}


@pytest.mark.parametrize("dtype", [torch.int64, torch.int16, torch.float32])
@pytest.mark.parametrize("what", ["targets", "positions"])
def test_other_types(backend, what, dtype):
    for call in _calls(backend, OnDevice(torch.zeros(2, 4, dtype=dtype)))[what]:
        with pytest.raises(ValueError) as e:
            call()
        assert what in str(e.value) and str(dtype) in str(e.value)


@pytest.mark.parametrize("what", ["targets", "positions"])
def test_strides(backend, what):
    t = torch.zeros(4, 16, dtype=torch.int32)
    for bad in (t[:2, :8:2], t[:, :2].t()):
        for call in _calls(backend, OnDevice(bad))[what]:
            with pytest.raises(ValueError) as e:
                call()
            assert what in str(e.value) and "contiguous" in str(e.value)
    apart = OnDevice(t[:2, :4])  # rows apart: positions have a batch stride
    for call in _calls(backend, apart)[what]:
        with pytest.raises(ValueError if what == "targets" else bwpp.BwppError):
            call()


@pytest.mark.parametrize("what", ["targets", "positions"])
def test_taken(backend, what):
    for t in (OnDevice(torch.zeros(8, dtype=torch.int32)), OnDevice(torch.zeros(2, 4, dtype=torch.int32)), ADDR[5] + 0x100000000):
        for call in _calls(backend, t)[what]:
            with pytest.raises(bwpp.BwppError) as e:
                call()
            assert e.value.status == bwpp.Status.INVALID_ARG and "handle" in str(e.value)


def test_plan_values():
    p = plan.Plan(None, "bwpp.plan 1\nvalue x f32 [4,8] input\nvalue w f32 [9,8] param\nvalue t i32 [4] input\n"
                        "value l f32 [4] output\nop linear_xent out=l in=x,w,t gives=loss trans_w=1\n")
    with pytest.raises(ValueError) as e:
        p.bind("t", torch.zeros(4, dtype=torch.int64))
    assert "'t'" in str(e.value)
    p.bind("t", torch.zeros(4, dtype=torch.int32))
    p.close()
