"""CPU tests of the scale that attention nodes have where none is given: that of the direct
call, 1/sqrt(columns of a head)."""
import pytest

from ferrograd_amd import graph as G

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
