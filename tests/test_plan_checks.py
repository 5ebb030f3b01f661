"""What the entry points would refuse at every run of a plan is refused when the
plan is created."""
import pytest

from bwpp import plan

HEAD = """bwpp.plan 1
dim T 6
value x f32 [T,32] input
value o f32 [T,32] input
value b bf16 [T,4] input
value wb bf16 [50,4] param
value wv f32 [50,32] param
value t i32 [T] input
value g f32 [32] param
value r f32 [T,32] output
value y f32 [T,32] output
value l f32 [T] output
value dg f32 [32] output
value big f32 [4294967302,32] input
value rbig f32 [4294967302,32] output
value wide f32 [1,4294967300] input
value rwide f32 [1,4294967300] output
value tbig i32 [4294967302] input
"""


@pytest.mark.parametrize("op,text", [
    ("op rotary out=r in=x heads=2 rot=7", "rot_dim"), ("op rotary out=r in=x heads=2 rot=18", "rot_dim"),
    ("op rotary_grad out=r in=x heads=2 rot=7", "rot_dim"), ("op rotary out=r in=x heads=32", "rot_dim"),
    ("op rotary out=r in=x heads=2 scaling=parts factor=4", "context"),
    ("op rotary out=r in=x heads=2 scaling=parts factor=4 context=64 low=4 high=4", "low_turns"),
    ("op rotary out=r in=x heads=2 base=-1", "base"), ("op rotary out=r in=x heads=2 factor=-2", "factor"),
    ("op residual_norm out=r,y in=x,o eps=-1", "eps"),
    ("op residual_norm_grad out=y,dg in=x,o,x with=dr gives=dx,dpost", "post-norm"),
    ("op residual_norm_grad out=y,dg in=x,o,g,x with=post,dr gives=dx,dpost post_norm=0", "post-norm"),
    ("op linear_xent out=l in=b,wb,t gives=loss trans_w=1", "8 elements"),
    ("op rotary out=rbig in=big heads=2", "32 bits"), ("op rotary out=rwide in=wide heads=2", "32 bits"),
    ("op residual_norm out=rbig in=big,big", "32 bits"), ("op residual_norm out=rwide in=wide,wide", "32 bits"),
    ("op linear_xent out=rbig in=big,wv,tbig gives=loss trans_w=1", "32 bits"),
    ("op linear_xent out=l in=x,big,t gives=loss trans_w=1", "32 bits")])
def test_refused(op, text):
    with pytest.raises(plan.PlanError) as e:
        plan.Plan(None, HEAD + op + "\n")
    assert text in str(e.value), str(e.value)


@pytest.mark.parametrize("op", [
    "op rotary out=r in=x heads=2 rot=6", "op rotary out=r in=x heads=2 scaling=parts factor=4 context=64 low=1 high=4",
    "op residual_norm out=r,y in=x,o eps=0", "op residual_norm_grad out=y,dg in=x,o,g,x with=post,dr gives=dx,dpost",
    "op linear_xent out=l in=x,wv,t gives=loss trans_w=1"])
def test_taken(op):
    plan.Plan(None, HEAD + op + "\n").close()
