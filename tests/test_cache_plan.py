"""Plan ops of the paged cache and the rules on logits, parsed and checked
without a GPU: a decoding step is taken, mistakes in it are named."""
import pytest

from bwpp import plan
from cacheplan import DECODE

KEEP = DECODE + "value kept i32 [S,3] input\nvalue counts i32 [S] input\nop cache_keep out=kc,vc in=kc,vc,table,held,kept,counts\n"
TREE = DECODE.replace("starts,held scale=auto", "starts,held,mask scale=0.25")


@pytest.mark.parametrize("text", [
    DECODE, KEEP, TREE, DECODE.replace("rot=8 scaling=linear factor=2", "rotate=0"),
    DECODE.replace("value kc f32 [PAGES,HK,PAGE,E]", "value kc f32 [PAGES,PAGE,HK,E]").replace("value vc f32 [PAGES,HK,PAGE,E]",
                   "value vc f32 [PAGES,PAGE,HK,E]").replace("held rot=8", "held cache=pthd rot=8").replace("scale=auto", "scale=auto cache=pthd"),
    DECODE.replace("out=ctx,lse", "out=ctx"),
    DECODE.replace("in=z,history,hstarts,rep,mask with=history,starts,repetition,mask", "in=z")])
def test_taken(text):
    plan.Plan(None, text).close()


@pytest.mark.parametrize("old,new,text", [
    ("out=q,kc,vc in=q,k,v", "out=q in=q,k,v", "in=Q,K,V"), ("out=q,kc,vc in", "out=q,vc,kc in", "in place"),
    ("in=q,k,v,kc,vc,table,starts,held rot", "in=q,k,v,kc,vc,table,starts rot", "in=Q,K,V"),
    ("held rot=8", "held rot=7", "rot_dim"), ("held rot=8", "held rot=18", "rot_dim"), ("scaling=linear", "scaling=most", "scaling"),
    ("factor=2", "factor=two", "factor"), ("factor=2", "factor=2 pairs=odd", "pairs"), ("factor=2", "factor=2 cache=thpd", "phtd"),
    ("factor=2", "factor=-2", "factor"),
    ("value vc f32 [PAGES,HK,PAGE,E]", "value vc f32 [PAGES,HK,PAGE,8]", "4-D shape"),
    ("value vc f32 [PAGES,HK,PAGE,E]", "value vc bf16 [PAGES,HK,PAGE,E]", "4-D shape"),
    ("value kc f32 [PAGES,HK,PAGE,E] param\nvalue vc f32 [PAGES,HK,PAGE,E] param",
     "value kc f32 [PAGES,HK,PAGE,E] temp\nvalue vc f32 [PAGES,HK,PAGE,E] temp", "inputs or params"),
    ("dim PAGE 8", "dim PAGE 12", "power of two"), ("value table i32 [S,COLS]", "value table i32 [S*COLS]", "TABLE"),
    ("value table i32 [S,COLS]", "value table f32 [S,COLS]", "TABLE"), ("value starts i32 [4]", "value starts i32 [3]", "STARTS"),
    ("value held i32 [S]", "value held i32 [2]", "HELD"),
    ("view v of=qkv offset=96 ld=128 shape=[S,32]", "view v of=qkv offset=96 ld=128 shape=[S,16]", "K and V"),
    ("dim E 16", "dim E 15", "heads of the pools"), ("scale=auto", "scale=large", "scale"), ("out=ctx,lse", "out=ctx,z", "LSE"),
    ("in=q,kc,vc,table,starts,held scale", "in=q,kc,vc,table,starts scale", "in=Q,KC"),
    ("in=q,kc,vc,table,starts,held scale", "in=q,kc,vc,table,starts,held,history scale", "MASK"),
    ("with=history,starts,repetition,mask", "with=history,starts,repetition", "with="),
    ("with=history,starts,repetition,mask", "with=history,starts,repetition,grammar", "with="),
    ("in=z,history,hstarts,rep,mask with=history,starts,repetition,mask", "in=z,history,rep,mask with=history,repetition,mask", "together"),
    ("value rep f32 [S]", "value rep f32 [2]", "one element a row"), ("value hstarts i32 [4]", "value hstarts i32 [3]", "rows + 1"),
    ("value mask i32 [S,4]", "value mask i32 [S,3]", "mask"), ("value y f32 [S,V]", "value y f32 [V,S]", "shape"),
])
def test_mistakes_are_named(old, new, text):
    assert DECODE.count(old) == 1
    with pytest.raises(plan.PlanError) as e:
        plan.Plan(None, DECODE.replace(old, new))
    assert text in str(e.value), str(e.value)


@pytest.mark.parametrize("old,new,text", [
    ("out=kc,vc in=kc,vc,table,held,kept", "out=kc in=kc,vc,table,held,kept", "in=KC"),
    ("value kept i32 [S,3]", "value kept i32 [2,3]", "KEPT"), ("value counts i32 [S]", "value counts i32 [4]", "COUNTS")])
def test_mistakes_in_keep_are_named(old, new, text):
    with pytest.raises(plan.PlanError) as e:
        plan.Plan(None, KEEP.replace(old, new))
    assert text in str(e.value), str(e.value)
