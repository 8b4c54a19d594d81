"""Refusals of the token-model operators (layer norm, embedding, 8-bit
activation checkpoints): arguments are checked before the context and any
device work, so every refusal shows without a GPU."""
import pytest

import ferrograd_amd as fa
from ferrograd_amd import _lib

P = 4096  # a non-NULL pointer; nothing may read it
INVALID, SHAPE, BOUNDS = 1, 5, 9
BIG = (1 << 23) + 1  # columns: one more than any of these takes
NAN, INF = float("nan"), float("inf")

# name -> (argument names, a call that only lacks its context)
CALLS = {
    "fg_layer_norm": dict(ctx=None, dtype=2, x=P, ldx=64, gamma=P, beta=P, eps=1e-5, R=4, C=64,
                          y=P, ldy=64, mean=P, rstd=P),
    "fg_layer_norm_bwd": dict(ctx=None, dtype=2, x=P, ldx=64, dy=P, lddy=64, gamma=P, mean=P,
                              rstd=P, R=4, C=64, dx=P, lddx=64, acc=0, dgamma=P, acc_g=0,
                              dbeta=2 * P, acc_b=0),
    "fg_embedding": dict(ctx=None, dtype=1, tokens=P, T=8, V=10, C=64, table=P, ldt=64, scale=1.0,
                         out=2 * P, ldo=64),
    "fg_embedding_bwd": dict(ctx=None, dtype=1, tokens=P, T=8, V=10, C=64, dout=P, lddo=64,
                             scale=1.0, dtable=2 * P, lddt=64, acc=0),
    "fg_ckpt8_save": dict(ctx=None, dtype=0, x=P, ldx=65, R=4, C=65, q=P, ldq=65, e=P, lde=3),
    "fg_ckpt8_load": dict(ctx=None, dtype=0, act=2, q=P, ldq=65, e=P, lde=3, R=4, C=65, z=P,
                          ldz=65, h=2 * P, ldh=65),
    "fg_act_bwd_ckpt8": dict(ctx=None, dtype=0, act=2, dH=P, lddh=65, q=P, ldq=65, e=P, lde=3, R=4,
                             C=65, dZ=P, lddz=65),
    "fg_matmul_bwd_ckpt8": dict(ctx=None, dtype=2, M=4, N=8, K=65, act=2, q=P, ldq=65, e=P, lde=3,
                                W=P, ldw=8, dZ=P, lddz=8, Zr=4 * P, Xr=2 * P, dX=3 * P, lddx=65,
                                dW=P, lddw=8, dbias=P, acc=0),
}

MANY = (1 << 31) - 1  # rows

REFUSED = [
    ("fg_layer_norm", dict(R=MANY, C=8200, ldx=8200, ldy=8200), BOUNDS),
    ("fg_layer_norm_bwd", dict(R=MANY, C=8200, ldx=8200, lddy=8200, lddx=8200), BOUNDS),
    ("fg_embedding", dict(T=MANY, C=2048, ldt=2048, ldo=2048), BOUNDS),
    ("fg_embedding_bwd", dict(T=(1 << 30) + 1), BOUNDS),
    ("fg_ckpt8_load", dict(R=MANY, C=4096, ldq=4096, lde=128, ldz=4096, ldh=4096), BOUNDS),
    # Outputs that are inputs, of another leading dimension or added to.
    ("fg_layer_norm", dict(ldx=65), INVALID), ("fg_layer_norm_bwd", dict(ldx=65), INVALID),
    ("fg_layer_norm_bwd", dict(lddy=65, x=2 * P), INVALID),
    ("fg_layer_norm_bwd", dict(acc=1), INVALID),
    ("fg_layer_norm_bwd", dict(acc=1, dy=2 * P), INVALID),
    ("fg_act_bwd_ckpt8", dict(lddh=66), INVALID),
    ("fg_layer_norm_bwd", dict(dbeta=P), INVALID), ("fg_embedding", dict(out=P), INVALID),
    ("fg_embedding_bwd", dict(dtable=P), INVALID), ("fg_ckpt8_load", dict(h=P), INVALID),
    ("fg_matmul_bwd_ckpt8", dict(Zr=3 * P), INVALID),
    ("fg_matmul_bwd_ckpt8", dict(Xr=P), INVALID), ("fg_matmul_bwd_ckpt8", dict(Zr=P), INVALID),
    ("fg_layer_norm", dict(C=BIG, ldx=BIG, ldy=BIG), BOUNDS),
    ("fg_layer_norm_bwd", dict(C=BIG, ldx=BIG, lddy=BIG, lddx=BIG), BOUNDS),
    ("fg_embedding", dict(C=BIG, ldt=BIG, ldo=BIG), BOUNDS),
    ("fg_embedding_bwd", dict(C=BIG, lddo=BIG, lddt=BIG), BOUNDS),
    ("fg_ckpt8_save", dict(C=BIG, ldx=BIG, ldq=BIG, lde=BIG), BOUNDS),
    ("fg_matmul_bwd_ckpt8", dict(K=BIG, ldq=BIG, lde=BIG, lddx=BIG), BOUNDS),
    ("fg_layer_norm", dict(dtype=3), INVALID), ("fg_layer_norm", dict(dtype=-1), INVALID),
    ("fg_layer_norm", dict(R=-1), SHAPE), ("fg_layer_norm", dict(C=0), SHAPE),
    ("fg_layer_norm", dict(ldx=63), SHAPE), ("fg_layer_norm", dict(ldy=63), SHAPE),
    ("fg_layer_norm", dict(eps=0.0), INVALID), ("fg_layer_norm", dict(eps=-1e-5), INVALID),
    ("fg_layer_norm", dict(eps=NAN), INVALID), ("fg_layer_norm", dict(eps=INF), INVALID),
    ("fg_layer_norm", dict(x=None), INVALID), ("fg_layer_norm", dict(y=None), INVALID),
    ("fg_layer_norm_bwd", dict(dtype=7), INVALID), ("fg_layer_norm_bwd", dict(C=-4), SHAPE),
    ("fg_layer_norm_bwd", dict(lddy=63), SHAPE), ("fg_layer_norm_bwd", dict(lddx=63), SHAPE),
    ("fg_layer_norm_bwd", dict(mean=None), INVALID),
    ("fg_layer_norm_bwd", dict(rstd=None), INVALID), ("fg_layer_norm_bwd", dict(dy=None), INVALID),
    ("fg_embedding", dict(dtype=4), INVALID), ("fg_embedding", dict(T=-1), SHAPE),
    ("fg_embedding", dict(V=0), SHAPE), ("fg_embedding", dict(C=0), SHAPE),
    ("fg_embedding", dict(ldt=63), SHAPE), ("fg_embedding", dict(ldo=10), SHAPE),
    ("fg_embedding", dict(tokens=None), INVALID), ("fg_embedding", dict(out=None), INVALID),
    ("fg_embedding_bwd", dict(V=-3), SHAPE), ("fg_embedding_bwd", dict(lddt=1), SHAPE),
    ("fg_embedding_bwd", dict(lddo=63), SHAPE), ("fg_embedding_bwd", dict(dtable=None), INVALID),
    ("fg_embedding_bwd", dict(dout=None), INVALID),
    ("fg_embedding_bwd", dict(T=0, dtable=None), INVALID),
    ("fg_ckpt8_save", dict(dtype=5), INVALID), ("fg_ckpt8_save", dict(lde=2), SHAPE),
    ("fg_ckpt8_save", dict(ldq=64), SHAPE), ("fg_ckpt8_save", dict(ldx=64), SHAPE),
    ("fg_ckpt8_save", dict(C=0), SHAPE), ("fg_ckpt8_save", dict(e=None), INVALID),
    ("fg_ckpt8_load", dict(act=3), INVALID), ("fg_ckpt8_load", dict(z=None, h=None), INVALID),
    ("fg_ckpt8_load", dict(ldh=64), SHAPE), ("fg_ckpt8_load", dict(q=None), INVALID),
    ("fg_act_bwd_ckpt8", dict(act=-1), INVALID), ("fg_act_bwd_ckpt8", dict(lddh=64), SHAPE),
    ("fg_act_bwd_ckpt8", dict(dZ=None), INVALID), ("fg_act_bwd_ckpt8", dict(R=-1), SHAPE),
    ("fg_matmul_bwd_ckpt8", dict(M=0), SHAPE), ("fg_matmul_bwd_ckpt8", dict(N=0), SHAPE),
    ("fg_matmul_bwd_ckpt8", dict(lde=2), SHAPE), ("fg_matmul_bwd_ckpt8", dict(lddx=64), SHAPE),
    ("fg_matmul_bwd_ckpt8", dict(Xr=None), INVALID),
    ("fg_matmul_bwd_ckpt8", dict(Zr=None), INVALID),
    ("fg_matmul_bwd_ckpt8", dict(Zr=2 * P), INVALID),
    ("fg_matmul_bwd_ckpt8", dict(dX=2 * P), INVALID),
    ("fg_matmul_bwd_ckpt8", dict(act=9), INVALID),
]


@pytest.mark.parametrize("fn,change,code", REFUSED,
                         ids=[f"{f[3:]}-{'-'.join(f'{k}={v}' for k, v in c.items())}"
                              for f, c, _ in REFUSED])
def test_refuses(fn, change, code):
    args = dict(CALLS[fn])
    assert set(change) <= set(args)
    args.update(change)
    with pytest.raises(fa.FgError) as e:
        _lib.call(fn, *args.values())
    assert e.value.code == code
    assert fn in str(e.value) and "ctx is NULL" not in str(e.value)


@pytest.mark.parametrize("fn", sorted(CALLS))
def test_refuses_a_null_context_last(fn):
    with pytest.raises(fa.FgError) as e:
        _lib.call(fn, *CALLS[fn].values())
    assert e.value.code == INVALID and f"{fn}: ctx is NULL" in str(e.value)
