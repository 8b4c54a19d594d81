"""Outputs of the token-model calls that are an input, or another output, are
refused: a kernel would overwrite what other workgroups have yet to read.  (Buffers are
told apart once there is a context; this one has no device, and the calls that are let
through have no rows.)"""
import ctypes

import numpy as np
import pytest

import ferrograd_amd as fa
from ferrograd_amd import _lib
from test_token_ops import CALLS, INVALID

KEEP = ctypes.create_string_buffer(b"\xff" * 4096)  # a context of device -1
NO_DEVICE = ctypes.addressof(KEEP)

# name -> outputs, inputs, arguments that go with them (none: refused before the context
# is looked at), pairs that may be one buffer
CASES = {
    "fg_ckpt8_save": (["q", "e"], ["x"], dict(ctx=NO_DEVICE, R=0), []),
    "fg_ckpt8_load": (["z", "h"], ["q", "e"], dict(ctx=NO_DEVICE, R=0), []),
    "fg_act_bwd_ckpt8": (["dZ"], ["dH", "q", "e"], dict(ctx=NO_DEVICE, R=0), [("dZ", "dH")]),
    "fg_layer_norm": (["y", "mean", "rstd"], ["x", "gamma", "beta"], dict(ctx=NO_DEVICE, R=0),
                      [("y", "x")]),
    "fg_layer_norm_bwd": (["dx", "dgamma", "dbeta"], ["x", "dy", "gamma", "mean", "rstd"],
                          dict(ctx=NO_DEVICE), [("dx", "x"), ("dx", "dy")]),
    "fg_embedding": (["out"], ["tokens", "table"], dict(ctx=NO_DEVICE, T=0), []),
    "fg_embedding_bwd": (["dtable"], ["tokens", "dout"], dict(ctx=NO_DEVICE), []),
    # (Its scratch: overwritten before the products read their operands.)
    "fg_matmul_bwd_ckpt8": (["Zr", "Xr"], ["q", "e", "W", "dZ", "dX", "dW", "dbias"], {}, []),
}


def pairs():
    for fn, (outs, ins, _, _) in CASES.items():
        for i, o in enumerate(outs):
            for other in ins + outs[i + 1:]:
                yield fn, o, other


def call(fn, **same):
    """The call with every buffer apart but for a = b in `same`: FgError, or None."""
    outs, ins, more, _ = CASES[fn]
    args = dict(CALLS[fn], **more)
    args.update({n: (k + 1) << 12 for k, n in enumerate(outs + ins)})
    args.update({a: args[b] for a, b in same.items()})
    try:
        _lib.call(fn, *args.values())
    except fa.FgError as e:
        return e


@pytest.mark.parametrize("fn,a,b", list(pairs()))
def test_refuses_an_output_that_is_another_buffer(fn, a, b):
    _, _, more, free = CASES[fn]
    if (a, b) in free:
        if more.get("R") == 0:
            assert call(fn, **{a: b}) is None
        return
    e = call(fn, **{a: b})
    assert e is not None and e.code == INVALID
    assert f"{fn}: " in str(e) and "ctx is NULL" not in str(e)


def test_addresses_that_are_no_python_ints():
    """An object whose data_ptr() gives another integer type is taken as it was."""
    class Buffer:
        def data_ptr(self):
            return np.uint64(1 << 40)

    with pytest.raises(fa.FgError) as e:
        _lib.call("fg_softmax_f32", None, fa._ptr(Buffer()), 4, 4, fa._ptr(Buffer()))
    assert e.value.code == INVALID
    assert fa._ptr(Buffer()) == 1 << 40 and fa._ptr(None) is None and fa._ptr(7) == 7


@pytest.mark.parametrize("fn", [f for f, c in CASES.items() if c[2].get("R", c[2].get("T")) == 0])
def test_takes_buffers_that_are_apart(fn):
    assert call(fn) is None
