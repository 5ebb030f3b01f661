"""A decoding step of one block's attention as a launch plan: projection of the
new tokens, positions and append, attention over the cache, projection to a
vocabulary, rules for the next token, its greedy choice."""

DECODE = """bwpp.plan 1
dim S 3
dim D 64
dim HQ 4
dim HK 2
dim E 16
dim PAGES 12
dim PAGE 8
dim COLS 4
dim V 100
value x f32 [S,D] input
value wqkv f32 [D,128] param
value wv f32 [HQ*E,V] param
value kc f32 [PAGES,HK,PAGE,E] param
value vc f32 [PAGES,HK,PAGE,E] param
value table i32 [S,COLS] input
value starts i32 [4] input
value held i32 [S] input
value history i32 [20] input
value hstarts i32 [4] input
value rep f32 [S] input
value mask i32 [S,4] input
value qkv f32 [S,128] temp
view q of=qkv offset=0 ld=128 shape=[S,64]
view k of=qkv offset=64 ld=128 shape=[S,32]
view v of=qkv offset=96 ld=128 shape=[S,32]
value ctx f32 [S,HQ*E] output
value lse f32 [S,HQ] output
value z f32 [S,V] temp
value y f32 [S,V] output
op matmul out=qkv in=x,wqkv
op cache_append out=q,kc,vc in=q,k,v,kc,vc,table,starts,held rot=8 scaling=linear factor=2
op cache_attention out=ctx,lse in=q,kc,vc,table,starts,held scale=auto
op matmul out=z in=ctx,wv
op logit_rules out=y in=z,history,hstarts,rep,mask with=history,starts,repetition,mask
"""
