"""CPU tests of layer norm, embedding and 8-bit activation checkpoints in the
graph planner: what dry plans lower to, and what is refused."""
import re

import pytest

from ferrograd_amd import FgError
from ferrograd_amd.graph import (CROSS_ENTROPY, MEAN_SQUARED_ERROR, Graph, Metadata, Optim,
                                 SimpleDType, f32_bits)
from test_planner import section


def token_model(T, V, C, H, K, dtype=SimpleDType.F32, ckpt=(), optim=None, act="gelu", layers=2):
    """tokens -> embedding -> layer norm -> `layers` Linear + act -> Linear -> softmax."""
    g, meta = Graph(CROSS_ENTROPY, (optim or Optim.adam()).lower), Metadata.new()
    fT, fV, fC, fH, fK = (meta.new_field() for _ in range(5))
    with g.define_ops() as ops:
        tok = ops.input([fT], SimpleDType.U32)
        table = ops.input([fV, fC], dtype)
        gamma, beta = ops.input([fC], dtype), ops.input([fC], dtype)
        h = ops.layer_norm(ops.embedding(table, tok, scale=2.0), gamma, beta, eps=1e-5)
        fin = fC
        for l in range(layers):
            W, b = ops.input([fin, fH], dtype), ops.input([fH], dtype)
            h = getattr(ops, act)(ops.bias_add(ops.matmul(h, W), b))
            if l in ckpt:
                ops.ckpt8(h)
            fin = fH
        W, b = ops.input([fin, fK], dtype), ops.input([fK], dtype)
        ops.softmax(ops.bias_add(ops.matmul(h, W), b))
    return g, [f32_bits(1e-3), T, V, C, H, K]


def test_token_model_lowers_to_its_own_launches():
    g, meta = token_model(512, 1000, 64, 256, 100)
    desc = g.describe(meta)
    n, fwd = section(desc, "forward")
    assert n == 6
    assert fwd[0].startswith("forward embedding 512x64x1000")
    assert fwd[1].startswith("forward layer_norm 512x64")
    assert [l.split(" ")[1] for l in fwd[2:]] == ["gemm", "gemm", "gemm", "softmax"]
    n, bwd = section(desc, "backward(ce-fused)")
    assert bwd[-2].startswith("backward layer_norm 512x64 -> grad of node")
    assert bwd[-1].startswith("backward embedding 512x64x1000 -> grad of node 1")
    assert "eltwise" not in desc and "zero grad" not in desc
    # Tokens are not updated: the table, gamma, beta and three Linear layers are.
    assert "adam over 9 inputs" in desc
    # The backwards of layer norm and of the table are one launch each, of a large batch
    # two and three.
    kernels = r"kernels per step: (\d+) \(forward (\d+), loss (\d+), backward (\d+), optim"
    m = re.search(kernels, desc)
    assert m and m.group(2) == "5" and m.group(4) == str(6 + 1 + 1)
    g, meta = token_model(8192, 1000, 64, 256, 100)
    m = re.search(kernels, g.describe(meta))
    assert m and m.group(2) == "5" and m.group(4) == str(6 + 2 + 3)


@pytest.mark.parametrize("dtype", [SimpleDType.F32, SimpleDType.BF16])
@pytest.mark.parametrize("act", ["relu", "gelu"])
def test_ckpt8_adds_a_save_and_a_load_and_shrinks_the_arena(act, dtype):
    size = (4096, 100, 128, 2048, 10, dtype)
    plain, meta = token_model(*size, act=act, layers=4)
    kept, _ = token_model(*size, act=act, layers=4, ckpt=(0, 1, 2, 3))
    d0, d1 = plain.describe(meta), kept.describe(meta)
    n0, f0 = section(d0, "forward")
    n1, f1 = section(d1, "forward")
    assert n1 == n0 + 4
    assert [l for l in f1 if "ckpt8" not in l] == f0
    assert [f1[i + 1].startswith("forward ckpt8 save 4096x2048") for i, l in enumerate(f1)
            if f"+{act}" in l] == [True] * 4
    n0, b0 = section(d0, "backward(ce-fused)")
    n1, b1 = section(d1, "backward(ce-fused)")
    assert n1 == n0 + 4 and [l for l in b1 if "ckpt8" not in l] == b0
    loads = [i for i, l in enumerate(b1) if "ckpt8 load" in l]
    assert all("gemm TN" in b1[i + 1] and "gemm NT" in b1[i + 2] for i in loads)
    arena = [int(re.search(r"arena: (\d+) bytes", d).group(1)) for d in (d0, d1)]
    # Of each layer's product, z and h (a plain plan lays out all three, the product
    # before the bias included) 33/32 bytes an element stay; three tensors (z, and two
    # of h in turn) are shared by all; padding is under 64 KiB a slot.
    MN, e = 4096 * 2048, 4 if dtype == SimpleDType.F32 else 2
    want = 4 * 3 * MN * e - 4 * MN * 33 // 32 - 3 * MN * e
    assert abs(arena[0] - arena[1] - want) < 32 * 65536


def test_layers_that_do_not_follow_one_another_share_no_live_memory():
    """Two branches whose activations are both read at the end: each keeps its
    own memory (a third, later one may take theirs)."""
    g, meta = Graph(MEAN_SQUARED_ERROR, Optim.sgd().lower), Metadata.new()
    f = meta.new_field()
    with g.define_ops() as ops:
        x = ops.input([f, f])
        W = [ops.input([f, f]) for _ in range(4)]
        a = ops.ckpt8(ops.gelu(ops.matmul(x, W[0])))
        b = ops.ckpt8(ops.gelu(ops.matmul(x, W[1])))
        ops.add(ops.matmul(a, W[2]), ops.matmul(b, W[3]))
    big, small = (int(re.search(r"arena: (\d+) bytes", g.describe([f32_bits(0.1), n])).group(1))
                  for n in (1024, 8))
    # z, two activations: 3 fp32; q: 2 bytes; e; per node value and gradient the rest:
    # values of two products and the sum, their gradients (5: two dz, two da merged
    # into dz ones, ...) are in both, so only a bound is asked: two live activations.
    assert big - small > (3 * 4 + 2) * 1024 * 1024


def refuse(code, text, build):
    g, meta = Graph(MEAN_SQUARED_ERROR, Optim.sgd().lower), Metadata.new()
    f = [meta.new_field() for _ in range(3)]
    with pytest.raises(FgError) as e:
        with g.define_ops() as ops:
            build(ops, f)
        g.describe([f32_bits(0.1), 4, 8, 16])
    assert e.value.code == code and text in str(e.value)


def test_refusals():
    U, B = SimpleDType.U32, SimpleDType.BF16
    refuse(5, "needs x[..., N], gamma[N], beta[N]", lambda o, f: o.layer_norm(
        o.input([f[0], f[1]]), o.input([f[0]]), o.input([f[1]])))
    refuse(5, "needs x[..., N], gamma[N], beta[N]", lambda o, f: o.layer_norm(
        o.input([f[0], f[1]]), o.input([f[1], f[1]]), o.input([f[1]])))
    refuse(3, "different element types", lambda o, f: o.layer_norm(
        o.input([f[0], f[1]], B), o.input([f[1]]), o.input([f[1]], B)))
    for eps in (0.0, -1.0, float("nan"), float("inf")):
        refuse(1, "eps must be positive", lambda o, f: o.layer_norm(
            o.input([f[0], f[1]]), o.input([f[1]]), o.input([f[1]]), eps=eps))

    def same(o, f):
        g = o.input([f[1]])
        return o.layer_norm(o.input([f[0], f[1]]), g, g)
    refuse(3, "must be different nodes", same)
    refuse(3, "is not a u32 input", lambda o, f: o.embedding(
        o.input([f[0], f[1]]), o.input([f[2]])))
    refuse(5, "the table must be a matrix", lambda o, f: o.embedding(
        o.input([f[0]]), o.input([f[2]], U)))
    refuse(3, "u32 inputs are the tokens", lambda o, f: o.relu(o.input([f[0], f[1]], U)))
    refuse(3, "u32 inputs are the tokens", lambda o, f: o.matmul(
        o.input([f[0], f[1]]), o.input([f[1], f[2]], U)))
    refuse(3, "u32 inputs are the tokens", lambda o, f: o.embedding(
        o.input([f[0], f[1]], U), o.input([f[2]], U)))

    def ck(build):
        refuse(3, "fg_graph_set_ckpt8", build)
    mm = lambda o, f: o.gelu(o.matmul(o.input([f[0], f[1]]), o.input([f[1], f[1]])))
    ck(lambda o, f: o.ckpt8(mm(o, f)))  # the last node
    ck(lambda o, f: o.tanh(o.ckpt8(mm(o, f))))  # read by no matmul
    ck(lambda o, f: o.matmul(o.ckpt8(o.gelu(o.input([f[0], f[1]]))), o.input([f[1], f[2]])))

    def twice(o, f):
        h = o.ckpt8(mm(o, f))
        return o.add(o.matmul(h, o.input([f[1], f[2]])), o.matmul(h, o.input([f[1], f[2]])))
    ck(twice)

    def second(o, f):
        return o.matmul(o.input([f[1], f[0]]), o.ckpt8(mm(o, f)))
    ck(second)
    refuse(1, "is not a relu or gelu", lambda o, f: o.ckpt8(o.tanh(o.input([f[0], f[1]]))))
