"""Numeric attributes of plan ops: products of integers and dims, or one decimal
number, negative ones too; anything else, or a value that its place does not
take, is an error of the plan."""
import pytest

from bwpp import plan

HEAD = """bwpp.plan 1
dim T 6
dim D 32
value x f32 [T,D] input
value o f32 [T,D] input
value w f32 [D,D] param
value wv f32 [50,D] param
value t i32 [T] input
value r f32 [T,D] output
value y f32 [T,D] output
value l f32 [T] output
"""
ROTARY, NORM, XENT = "op rotary out=r in=x heads=2 ", "op residual_norm out=r,y in=x,o ", "op linear_xent out=l in=x,wv,t gives=loss trans_w=1 "
ATT, MATMUL = "op attention out=r in=x,o,x heads=2 ", "op matmul out=r in=x,w "
RMS, SUM = "op rmsnorm out=r in=x ", "op reduce_max out=l in=x "


@pytest.mark.parametrize("op", [
    ROTARY + "offset=-7", ROTARY + "offset=-2147483648 magnitude=-2", ROTARY + "base=1e6 rot=8", ROTARY + "rot=T*2",
    NORM + "stream_scale=-1 branch_scale=-2.5e-1 eps=1e-6", NORM + "gate_rows=T", XENT + "scale=-1", XENT + "scale=+2",
    ATT + "scale=-1 causal=1", ATT + "scale=auto", RMS + "eps=1e-05", SUM + "axis=-1"])
def test_taken(op):
    plan.Plan(None, HEAD + op + "\n").close()


@pytest.mark.parametrize("op,key", [
    (ROTARY + "offset=abc", "offset"), (ROTARY + "offset=2147483648", "offset"), (ROTARY + "offset=1.5", "offset"),
    (ROTARY + "offset=-2147483649", "offset"), (ROTARY + "rot=-2", "rot"), (ROTARY + "rot=8x", "rot"),
    (ROTARY + "base=theta", "base"), (ROTARY + "magnitude=nan", "magnitude"), (ROTARY + "magnitude=1,5", "magnitude"),
    (ROTARY + "context=4294967296", "context"), (ROTARY + "batch=-1", "batch"), (ROTARY + "factor=", "factor"),
    (NORM + "post_norm=yes", "post_norm"), (NORM + "gate_rows=-1", "gate_rows"), (NORM + "stream_scale=--1", "stream_scale"),
    (NORM + "eps=small", "eps"), (XENT + "scale=1/2", "scale"), (XENT.replace("trans_w=1", "trans_w=true"), "trans_w"),
    (ATT + "scale=sqrt", "scale"), (ATT + "causal=true", "causal"), (ATT + "batch=1.5", "batch"), (MATMUL + "tb=-1", "tb"),
    (RMS + "eps=1e-5f", "eps"), (SUM + "axis=rows", "axis")])
def test_named(op, key):
    with pytest.raises(plan.PlanError) as e:
        plan.Plan(None, HEAD + op + "\n")
    assert key + "=" in str(e.value) and "number" in str(e.value), str(e.value)


def test_batches_times_heads_of_2_to_the_64():
    for op in ("op rotary out=r in=x layout=bhsd batch=4294967296 heads=4294967296",
               "op attention out=r in=x,o,x layout=bhsd batch=4294967296 heads=4294967296",
               "op attention out=r in=x,o,x layout=bhsd batch=4294967295 heads=4294967295"):
        with pytest.raises(plan.PlanError):
            plan.Plan(None, HEAD + op + "\n")


def test_dims_are_not_negative():
    with pytest.raises(plan.PlanError) as e:
        plan.Plan(None, HEAD.replace("dim T 6", "dim T -6"))
    assert "bad dim" in str(e.value)
    with pytest.raises(plan.PlanError) as e:
        plan.Plan(None, HEAD + "value z f32 [T*-1] input\n")
    assert "unknown dim" in str(e.value)
