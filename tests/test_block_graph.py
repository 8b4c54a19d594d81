"""CPU tests of RMS norm and attention in the graph planner: what dry plans lower to, and
what is refused."""
import re

import pytest

from ferrograd_amd import FgError
from ferrograd_amd.graph import (CROSS_ENTROPY, MEAN_SQUARED_ERROR, Graph, Metadata, Optim,
                                 SimpleDType, f32_bits)
from test_planner import section

U = SimpleDType.U32


def block(ops, fields, heads, kv, dtype=SimpleDType.F32):
    """x[T][C] -> norm -> q, k, v -> attention -> projection, added to x."""
    T, C, KV, N = fields
    x, starts = ops.input([T, C], dtype), ops.input([N], U)
    h = ops.rms_norm(x, ops.input([C], dtype))
    q = ops.matmul(h, ops.input([C, C], dtype))
    k, v = (ops.matmul(h, ops.input([C, KV], dtype)) for _ in range(2))
    a = ops.attention(q, k, v, starts, heads, kv, scale=0.125)
    return ops.add(x, ops.matmul(a, ops.input([C, C], dtype)))


def described(heads, kv, T, C, KV, N, dtype=SimpleDType.F32):
    g, meta = Graph(MEAN_SQUARED_ERROR, Optim.sgd().lower), Metadata.new()
    fields = [meta.new_field() for _ in range(4)]
    with g.define_ops() as ops:
        block(ops, fields, heads, kv, dtype)
    return g.describe([f32_bits(1e-3), T, C, KV, N])


def test_block_lowers_to_its_own_launches():
    desc = described(8, 2, 8192, 512, 128, 5)
    n, fwd = section(desc, "forward")
    kinds = [" ".join(l.split(" ")[1:3]) for l in fwd]
    assert kinds[0].startswith("rms_norm 8192x512") and "gemm" in kinds[1]
    att = [l for l in fwd if "forward attention" in l]
    assert len(att) == 1 and "4 sequences 8192x8192 heads 8/2x64 causal" in att[0]
    assert sum("zero rows of no sequence" in l for l in fwd) == 1
    n, bwd = section(desc, "backward(seed)")
    assert sum("backward attention" in l for l in bwd) == 1
    assert sum("zero grad" in l for l in bwd) == 3  # of q, k and v, for rows of no sequence
    norm = [l for l in bwd if "backward rms_norm" in l]
    assert len(norm) == 1 and norm[0] == bwd[-1]
    # The norm's: two launches; attention's passes over the rows and over the keys.
    m = re.search(r"kernels per step: \d+ \(forward (\d+), loss \d+, backward (\d+), optim", desc)
    assert m and int(m.group(1)) >= len(fwd) and int(m.group(2)) >= len(bwd) + 2


def test_long_keys_are_split_with_a_launch_that_joins_them():
    """The plan's workspace holds the splits of few rows over long keys."""
    small, long = (described(4, 4, T, 256, 256, 2) for T in (64, 4096))
    arena = [int(re.search(r"arena: (\d+) bytes", d).group(1)) for d in (small, long)]
    assert arena[1] > arena[0]


def refuse(code, text, build, sizes=(32, 64, 16, 4, 48)):
    g, meta = Graph(MEAN_SQUARED_ERROR, Optim.sgd().lower), Metadata.new()
    f = [meta.new_field() for _ in range(5)]
    with pytest.raises(FgError) as e:
        with g.define_ops() as ops:
            build(ops, f)
        g.describe([f32_bits(0.1), *sizes])
    assert e.value.code == code and text in str(e.value)


def att(q=(0, 1), k=(0, 1), v=(0, 1), starts=(3,), heads=4, kv=4, types=("F32",) * 3, **kw):
    def build(o, f):
        t = [o.input([f[i] for i in dims], getattr(SimpleDType, ty))
             for dims, ty in zip((q, k, v), types)]
        return o.attention(*t, o.input([f[i] for i in starts], U), heads, kv, **kw)
    return build


def test_refusals_of_attention():
    refuse(5, "needs q[Tq, 4 D], k[Tk, 4 D], v[Tk, 4 D]", att(k=(0, 2)))
    refuse(5, "needs q[Tq, 4 D], k[Tk, 4 D], v[Tk, 4 D]", att(v=(3, 1)))
    refuse(5, "needs q[Tq, 5 D]", att(heads=5, kv=5))
    refuse(5, "q, k and v must be matrices", att(q=(1,)))
    refuse(5, "the starts are n + 1 numbers", att(starts=(3, 3)))
    refuse(5, "the starts are n + 1 numbers", att(), sizes=(32, 64, 16, 1, 48))
    refuse(1, "no multiple of 3 key heads", att(heads=4, kv=3))
    refuse(1, "no multiple of 0 key heads", att(heads=4, kv=0))
    refuse(3, "different element types", att(types=("BF16", "BF16", "F32")))
    refuse(3, "heads of 192 columns, at most 128", att(), sizes=(32, 768, 16, 4, 48))
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        refuse(1, "scale must be positive", att(scale=scale))

    def two_starts(o, f):
        x = [o.input([f[0], f[1]]) for _ in range(3)]
        return o.attention(*x, o.input([f[3]], U), 4, k_starts=o.input([f[4]], U))
    refuse(5, "the starts are n + 1 numbers", two_starts)

    def no_tokens(o, f):
        x = [o.input([f[0], f[1]]) for _ in range(3)]
        return o.attention(*x, o.input([f[3]]), 4)
    refuse(3, "is not a u32 input", no_tokens)

    def same(o, f):
        x = o.input([f[0], f[1]])
        return o.attention(o.input([f[0], f[1]]), x, x, o.input([f[3]], U), 4)
    refuse(3, "must be different nodes", same)

    def scalar(o, f):
        x = [o.input([f[0], f[1]]) for _ in range(2)]
        return o.attention(*x, o.constant_f32(1.0), o.input([f[3]], U), 4)
    refuse(5, "q, k and v must be matrices", scalar)
    refuse(3, "u32 inputs are the tokens", lambda o, f: o.add(
        o.input([f[0], f[1]]), o.input([f[0], f[1]], U)))


def test_refusals_of_rms_norm():
    refuse(5, "needs x[..., N], gamma[N]", lambda o, f: o.rms_norm(
        o.input([f[0], f[1]]), o.input([f[0]])))
    refuse(5, "needs x[..., N], gamma[N]", lambda o, f: o.rms_norm(
        o.input([f[0], f[1]]), o.input([f[1], f[1]])))
    refuse(5, "needs x[..., N], gamma[N]", lambda o, f: o.rms_norm(
        o.constant_f32(2.0), o.input([f[1]])))
    refuse(3, "different element types", lambda o, f: o.rms_norm(
        o.input([f[0], f[1]], SimpleDType.BF16), o.input([f[1]])))
    for eps in (0.0, -1.0, float("nan"), float("inf")):
        refuse(1, "eps must be positive", lambda o, f: o.rms_norm(
            o.input([f[0], f[1]]), o.input([f[1]]), eps=eps))

    def same(o, f):
        x = o.input([f[1]])
        return o.rms_norm(x, x)
    refuse(3, "must be different nodes", same)
