"""Plan ops of the operators around the block, parsed and checked without a
GPU: the training step's plan is taken, mistakes in it are named."""
import pytest

from bwpp import plan
from lmplan import TRAIN


def test_train_plan_is_taken():
    p = plan.Plan(None, TRAIN)
    assert p.arena_bytes > 0
    p.close()


@pytest.mark.parametrize("old,new,text", [
    ("in=q,k,pos batch=B heads=HEADS rot=8", "in=q,k,pos batch=B heads=7 rot=8", "batch / heads"),
    ("in=q,k,pos batch", "in=q,pos batch", "in=Q"),
    ("op rotary out=q,k in=q,k,pos batch=B", "op rotary out=q,k in=q,k,x batch=B", "in=Q"),
    ("rot=8 scaling=parts factor=4 context=64 low=0.5 high=4 magnitude=1.125\nop attention",
     "rot=8 scaling=most\nop attention", "scaling"),
    ("rot=8 scaling=parts factor=4 context=64 low=0.5 high=4 magnitude=1.125\nop attention",
     "rot=8 pairs=odd\nop attention", "pairs"),
    ("in=x,o0,gpre0 with=pre", "in=x,o0,gpre0", "with="),
    ("in=x,o0,gpre0 with=pre", "in=x,o0,gpre0 with=pre,pre", "with="),
    ("in=x,o0,gpre0 with=pre", "in=x,o0,wqkv with=pre", "shape"),
    ("in=r0,ao,gpost1,gate1,gpre1 with=post,gate,pre branch", "in=r0,ao,gpost1,gate2,gpre1 with=post,gate,pre branch", "gate"),
    ("gives=dx,do,dpre\n", "gives=dx,do,dgamma\n", "gives="),
    ("with=pre,dr,dy gives=dx,do,dpre", "with=pre,dr,gate gives=dx,do,dpre", "gate"),
    ("in=y2,wv,targets gives=loss,lse,sums trans_w=1", "in=y2,wv,targets gives=loss,lse,sums", "columns"),
    ("in=y2,wv,targets gives", "in=y2,wv,loss gives", "i32"),
    ("in=y2,wv,targets gives=loss,lse,sums", "in=y2,wv,pos gives=loss,lse,sums", "one element a row"),
    ("out=loss,xlse,sums in", "out=loss,xlse,dl in", "shapes"),
    ("in=y2,wv,targets,xlse,dl gives=dx,dw", "in=y2,wv,targets,xlse,h gives=dx,dw", "shapes"),
    ("out=dy2,dwv in", "out=dwv,dy2 in", "shapes"),
    ("value targets i32 [B*T] input", "value targets i32 [B*T] temp", "i32"),
    ("op matmul out=qkv in=y0,wqkv", "op matmul out=qkv in=targets,wqkv", "f32 or bf16"),
    ("op silu out=h in=hpre", "op silu out=h in=targets", "f32"),
])
def test_mistakes_are_named(old, new, text):
    assert TRAIN.count(old) == 1
    with pytest.raises(plan.PlanError) as e:
        plan.Plan(None, TRAIN.replace(old, new))
    assert text in str(e.value), str(e.value)


def test_positions_of_each_batch_are_taken():
    plan.Plan(None, TRAIN.replace("in=q,k,pos batch=B heads=HEADS rot=8 scaling=parts factor=4 context=64 low=0.5 high=4 "
                                  "magnitude=1.125\nop attention", "in=q,k,targets batch=B heads=HEADS\nop attention")).close()
