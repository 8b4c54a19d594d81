"""CPU tests of attention's scale: the one that a node has where none is given, that of the direct
call, 1/sqrt(columns of a head), and the smallest that a backward takes."""
import pytest

from ferrograd_amd import FgError, _lib
from ferrograd_amd import graph as G
from test_block_ops import CALLS, NO_DEVICE, UNSUPPORTED

U32 = G.SimpleDType.U32


def scales_of(monkeypatch, build, sizes):
    """The scales of a graph's attention nodes for a binding of the sizes."""
    seen, real = [], G.call

    def call(name, *args):
        if name == "fg_graph_attention":
            seen.append(args[8])
        return real(name, *args)

    monkeypatch.setattr(G, "call", call)
    g, meta = G.Graph(G.MEAN_SQUARED_ERROR, G.Optim.sgd().lower), G.Metadata.new()
    f = [meta.new_field() for _ in sizes]
    with g.define_ops() as ops:
        build(ops, f)
    g.describe([G.f32_bits(0.1), *sizes])
    return seen


def inputs(ops, t, c, n):
    return [ops.input([t, c]) for _ in range(3)] + [ops.input([n], U32)]


@pytest.mark.parametrize("heads", [1, 4, 8])
def test_scale_follows_the_columns_of_a_head(monkeypatch, heads):
    for C in (64, 128):
        got = scales_of(monkeypatch, lambda o, f: o.attention(*inputs(o, *f), heads), (32, C, 3))
        assert got == [pytest.approx((C // heads) ** -0.5)]


def test_scale_that_is_given_stays(monkeypatch):
    got = scales_of(monkeypatch, lambda o, f: o.attention(*inputs(o, *f), 4, scale=1.0), (32, 64, 3))
    assert got == [1.0]


def test_columns_are_found_through_operations(monkeypatch):
    """q behind a product, a bias, norms, a lookup, sums with a constant on either side and
    another attention."""
    def build(o, f):
        t, c, n, v = f
        starts, tokens = o.input([n], U32), o.input([t], U32)
        k, w = (o.input([t, c]) for _ in range(2))
        x = o.embedding(o.input([v, c]), tokens)
        x = o.rms_norm(x, o.input([c]))
        x = o.bias_add(o.matmul(x, o.input([c, c])), o.input([c]))
        x = o.gelu(o.layer_norm(x, o.input([c]), o.input([c])))
        x = o.add(o.constant_f32(1.0), x)
        x = o.mul(x, o.constant_f32(0.5))
        x = o.attention(x, k, w, starts, 2)
        o.attention(o.softmax(x), k, w, starts, 8)

    got = scales_of(monkeypatch, build, (48, 96, 3, 50))
    assert got == [pytest.approx(48 ** -0.5), pytest.approx(12 ** -0.5)]


def test_default_binding_validates():
    g, meta = G.Graph(G.MEAN_SQUARED_ERROR, G.Optim.sgd().lower), G.Metadata.new()
    f = [meta.new_field() for _ in range(3)]
    with g.define_ops() as ops:
        ops.attention(*inputs(ops, *f), 4)
    g.validate(meta)


def test_columns_of_a_long_chain_of_sums(monkeypatch):
    """Sums of a node with itself, one over the other: each is looked at once."""
    def build(o, f):
        q, k, v, starts = inputs(o, *f)
        for _ in range(200):
            q = o.add(q, q)
        o.attention(q, k, v, starts, 4)

    assert scales_of(monkeypatch, build, (32, 64, 3)) == [0.25]


@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_backward_in_16_bits_refuses_scales_whose_reciprocal_is_past_fp32(dtype):
    """The rows' log-sums enter its products in units of the scale."""
    args = dict(CALLS["fg_attention_bwd"], dtype=dtype, ctx=NO_DEVICE, n=0)
    for scale, refused in ((2.0 ** -120, False), (2.0 ** -121, dtype != 0), (1e-44, dtype != 0)):
        args["scale"] = scale
        if refused:
            with pytest.raises(FgError) as e:
                _lib.call("fg_attention_bwd", *args.values())
            assert e.value.code == UNSUPPORTED and "scale" in str(e.value)
        else:
            _lib.call("fg_attention_bwd", *args.values())
    fwd = dict(CALLS["fg_attention"], dtype=dtype, ctx=NO_DEVICE, n=0, scale=1e-44)
    _lib.call("fg_attention", *fwd.values())
