"""Refusals of attention, RMS norm and token log probabilities: arguments are checked
before the context and any device work, so every refusal shows without a GPU.  Outputs
that are an input or another output are told apart once there is a context; that one has
no device, and the calls that are let through have nothing to do."""
import ctypes

import pytest

import ferrograd_amd as fa
from ferrograd_amd import _lib

P = 4096  # a non-NULL pointer; nothing may read it
INVALID, UNSUPPORTED, SHAPE, BOUNDS = 1, 3, 5, 9
BIG = (1 << 23) + 1  # columns: one more than any row operator takes
MANY = (1 << 31) - 1
NAN, INF = float("nan"), float("inf")
KEEP = ctypes.create_string_buffer(b"\xff" * 4096)  # a context of device -1
NO_DEVICE = ctypes.addressof(KEEP)

# name -> a call that only lacks its context
CALLS = {
    "fg_rms_norm": dict(ctx=None, dtype=2, x=P, ldx=64, r=2 * P, ldr=64, gamma=3 * P, eps=1e-5, R=4,
                        C=64, s=4 * P, lds=64, y=5 * P, ldy=64, q=6 * P, ldq=64, e=7 * P, lde=2,
                        rstd=8 * P),
    "fg_rms_norm_bwd": dict(ctx=None, dtype=2, s=P, lds=64, dy=2 * P, lddy=64, gamma=3 * P,
                            rstd=4 * P, R=4, C=64, ds=5 * P, ldds=64, dx=6 * P, lddx=64,
                            dgamma=7 * P, acc=0),
    "fg_token_logprobs": dict(ctx=None, dtype=1, logits=P, ldx=64, tokens=2 * P, R=4, C=64, scale=1.0,
                              logp=3 * P, entropy=4 * P, lse=5 * P, top=5, ids=6 * P, tops=7 * P),
    "fg_token_logprobs_bwd": dict(ctx=None, dtype=1, logits=P, ldx=64, tokens=2 * P, R=4, C=64,
                                  scale=1.0, lse=3 * P, entropy=4 * P, dlogp=5 * P, dentropy=6 * P,
                                  dlogits=7 * P, ldd=64),
    "fg_attention": dict(ctx=None, dtype=2, q=P, ldq=256, k=2 * P, ldk=128, v=3 * P, ldv=128,
                         qs=4 * P, ks=5 * P, kl=6 * P, n=2, Tq=10, Tk=12, heads=4, kv=2, D=64,
                         scale=0.125, causal=1, out=7 * P, ldo=256, lse=8 * P),
    "fg_attention_bwd": dict(ctx=None, dtype=2, q=P, ldq=256, k=2 * P, ldk=128, v=3 * P, ldv=128,
                             out=4 * P, ldo=256, dout=5 * P, lddo=256, lse=6 * P, qs=7 * P, ks=8 * P,
                             n=2, Tq=10, Tk=12, heads=4, kv=2, D=64, scale=0.125, causal=1,
                             dq=9 * P, lddq=256, dk=10 * P, lddk=128, dv=11 * P, lddv=128, acc=0),
}

REFUSED = [
    ("fg_rms_norm", dict(dtype=3), INVALID), ("fg_rms_norm", dict(R=-1), SHAPE),
    ("fg_rms_norm", dict(C=0), SHAPE),
    ("fg_rms_norm", dict(C=BIG, ldx=BIG, ldr=BIG, lds=BIG, ldy=BIG, ldq=BIG, lde=BIG), BOUNDS),
    ("fg_rms_norm", dict(R=MANY), BOUNDS), ("fg_rms_norm", dict(x=None), INVALID),
    ("fg_rms_norm", dict(y=None, q=None, e=None), INVALID),
    ("fg_rms_norm", dict(q=None), INVALID), ("fg_rms_norm", dict(e=None), INVALID),
    ("fg_rms_norm", dict(r=None), INVALID), ("fg_rms_norm", dict(s=None), INVALID),
    ("fg_rms_norm", dict(ldx=63), SHAPE), ("fg_rms_norm", dict(ldr=63), SHAPE),
    ("fg_rms_norm", dict(lds=63), SHAPE), ("fg_rms_norm", dict(ldy=63), SHAPE),
    ("fg_rms_norm", dict(ldq=63), SHAPE), ("fg_rms_norm", dict(lde=1), SHAPE),
    ("fg_rms_norm", dict(eps=0.0), INVALID), ("fg_rms_norm", dict(eps=-1.0), INVALID),
    ("fg_rms_norm", dict(eps=NAN), INVALID), ("fg_rms_norm", dict(eps=INF), INVALID),
    ("fg_rms_norm", dict(s=P, lds=65), INVALID), ("fg_rms_norm", dict(s=2 * P, lds=65), INVALID),
    ("fg_rms_norm", dict(y=P, ldy=65), INVALID), ("fg_rms_norm", dict(y=2 * P, ldy=65), INVALID),
    ("fg_rms_norm_bwd", dict(dtype=-1), INVALID), ("fg_rms_norm_bwd", dict(C=-2), SHAPE),
    ("fg_rms_norm_bwd", dict(lds=63), SHAPE), ("fg_rms_norm_bwd", dict(lddy=1), SHAPE),
    ("fg_rms_norm_bwd", dict(ldds=63), SHAPE), ("fg_rms_norm_bwd", dict(lddx=63), SHAPE),
    ("fg_rms_norm_bwd", dict(s=None), INVALID), ("fg_rms_norm_bwd", dict(dy=None), INVALID),
    ("fg_rms_norm_bwd", dict(rstd=None), INVALID), ("fg_rms_norm_bwd", dict(dx=None), INVALID),
    ("fg_rms_norm_bwd", dict(dx=P, lddx=65), INVALID),
    ("fg_rms_norm_bwd", dict(dx=2 * P, lddx=65), INVALID),
    ("fg_rms_norm_bwd", dict(dx=5 * P, lddx=65), INVALID),
    ("fg_rms_norm_bwd", dict(R=MANY), BOUNDS),
    ("fg_rms_norm_bwd", dict(C=BIG, lds=BIG, lddy=BIG, ldds=BIG, lddx=BIG), BOUNDS),
    ("fg_token_logprobs", dict(dtype=3), INVALID), ("fg_token_logprobs", dict(R=-1), SHAPE),
    ("fg_token_logprobs", dict(C=0), SHAPE), ("fg_token_logprobs", dict(ldx=63), SHAPE),
    ("fg_token_logprobs", dict(C=BIG, ldx=BIG), BOUNDS), ("fg_token_logprobs", dict(R=MANY), BOUNDS),
    ("fg_token_logprobs", dict(top=33), BOUNDS), ("fg_token_logprobs", dict(top=-1), BOUNDS),
    ("fg_token_logprobs", dict(top=9, C=8), BOUNDS),
    ("fg_token_logprobs", dict(top=0), INVALID),
    ("fg_token_logprobs", dict(ids=None, tops=None), INVALID),
    ("fg_token_logprobs", dict(scale=0.0), INVALID), ("fg_token_logprobs", dict(scale=INF), INVALID),
    ("fg_token_logprobs", dict(scale=NAN), INVALID), ("fg_token_logprobs", dict(logits=None), INVALID),
    ("fg_token_logprobs", dict(tokens=None), INVALID),
    ("fg_token_logprobs",
     dict(logp=None, entropy=None, lse=None, top=0, ids=None, tops=None), INVALID),
    ("fg_token_logprobs_bwd", dict(dtype=7), INVALID), ("fg_token_logprobs_bwd", dict(C=0), SHAPE),
    ("fg_token_logprobs_bwd", dict(ldx=63), SHAPE), ("fg_token_logprobs_bwd", dict(ldd=63), SHAPE),
    ("fg_token_logprobs_bwd", dict(scale=-1.0), INVALID),
    ("fg_token_logprobs_bwd", dict(lse=None), INVALID),
    ("fg_token_logprobs_bwd", dict(dlogits=None), INVALID),
    ("fg_token_logprobs_bwd", dict(dlogp=None, dentropy=None), INVALID),
    ("fg_token_logprobs_bwd", dict(entropy=None), INVALID),
    ("fg_token_logprobs_bwd", dict(dlogits=P, ldd=65), INVALID),
    ("fg_token_logprobs_bwd", dict(R=MANY), BOUNDS),
    ("fg_attention", dict(dtype=3), INVALID), ("fg_attention", dict(n=-1), SHAPE),
    ("fg_attention", dict(Tq=-1), SHAPE), ("fg_attention", dict(Tk=-1), SHAPE),
    ("fg_attention", dict(heads=0), SHAPE), ("fg_attention", dict(kv=0), SHAPE),
    ("fg_attention", dict(kv=3), SHAPE), ("fg_attention", dict(D=0), SHAPE),
    ("fg_attention", dict(D=129, ldq=600, ldk=600, ldv=600, ldo=600), UNSUPPORTED),
    ("fg_attention", dict(ldq=255), SHAPE), ("fg_attention", dict(ldk=127), SHAPE),
    ("fg_attention", dict(ldv=127), SHAPE), ("fg_attention", dict(ldo=255), SHAPE),
    ("fg_attention", dict(scale=0.0), INVALID), ("fg_attention", dict(scale=-0.1), INVALID),
    ("fg_attention", dict(scale=NAN), INVALID), ("fg_attention", dict(scale=INF), INVALID),
    ("fg_attention", dict(q=None), INVALID), ("fg_attention", dict(k=None), INVALID),
    ("fg_attention", dict(v=None), INVALID), ("fg_attention", dict(qs=None), INVALID),
    ("fg_attention", dict(ks=None), INVALID), ("fg_attention", dict(out=None), INVALID),
    ("fg_attention", dict(Tq=MANY), BOUNDS), ("fg_attention", dict(Tk=MANY), BOUNDS),
    ("fg_attention", dict(n=1 << 24), BOUNDS),
    ("fg_attention_bwd", dict(dtype=-1), INVALID), ("fg_attention_bwd", dict(kv=3), SHAPE),
    ("fg_attention_bwd", dict(lddo=255), SHAPE), ("fg_attention_bwd", dict(lddq=255), SHAPE),
    ("fg_attention_bwd", dict(lddk=127), SHAPE), ("fg_attention_bwd", dict(lddv=127), SHAPE),
    ("fg_attention_bwd", dict(lse=None), INVALID), ("fg_attention_bwd", dict(dout=None), INVALID),
    ("fg_attention_bwd", dict(dq=None), INVALID), ("fg_attention_bwd", dict(dk=None), INVALID),
    ("fg_attention_bwd", dict(dv=None), INVALID), ("fg_attention_bwd", dict(Tq=MANY), BOUNDS),
    ("fg_attention_bwd", dict(D=200, ldq=800, ldk=800, ldv=800, ldo=800, lddo=800, lddq=800,
                              lddk=800, lddv=800), UNSUPPORTED),
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


# name -> outputs, inputs, what leaves the call nothing to do (none: refused or not before
# the device is looked at), pairs that may be one buffer
ALIASES = {
    "fg_rms_norm": (["s", "y", "q", "e", "rstd"], ["x", "r", "gamma"], dict(R=0),
                    [("s", "x"), ("s", "r"), ("y", "x"), ("y", "r")]),
    "fg_rms_norm_bwd": (["dx", "dgamma"], ["s", "dy", "gamma", "rstd", "ds"], None,
                        [("dx", "s"), ("dx", "dy"), ("dx", "ds")]),
    "fg_token_logprobs": (["logp", "entropy", "lse", "ids", "tops"], ["logits", "tokens"],
                          dict(R=0), []),
    "fg_token_logprobs_bwd": (["dlogits"], ["logits", "tokens", "lse", "entropy", "dlogp",
                                            "dentropy"], dict(R=0), [("dlogits", "logits")]),
    "fg_attention": (["out", "lse"], ["q", "k", "v", "qs", "ks", "kl"], dict(n=0), []),
    "fg_attention_bwd": (["dq", "dk", "dv"], ["q", "k", "v", "out", "dout", "lse", "qs", "ks"],
                         dict(n=0), []),
}


def alias_call(fn, **same):
    args = dict(CALLS[fn], ctx=NO_DEVICE, **(ALIASES[fn][2] or {}))
    args.update({a: args[b] for a, b in same.items()})
    try:
        _lib.call(fn, *args.values())
    except fa.FgError as e:
        return e


@pytest.mark.parametrize("fn,a,b", [(f, o, x) for f, (outs, ins, _, _) in ALIASES.items()
                                    for i, o in enumerate(outs) for x in ins + outs[i + 1:]])
def test_refuses_an_output_that_is_another_buffer(fn, a, b):
    _, _, idle, free = ALIASES[fn]
    if (a, b) in free:
        if idle:
            assert alias_call(fn, **{a: b}) is None
        return
    e = alias_call(fn, **{a: b})
    assert e is not None and e.code == INVALID
    assert f"{fn}: " in str(e) and "ctx is NULL" not in str(e)


@pytest.mark.parametrize("fn", [f for f, c in ALIASES.items() if c[2]])
def test_takes_buffers_that_are_apart(fn):
    assert alias_call(fn) is None
