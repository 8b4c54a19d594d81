"""Two attention layers of different sizes whose keys or values need no gradient: what the
backward writes of those shares one memory, and the others' gradients are as they should be."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from conftest import normwise_rel  # noqa: E402
from ferrograd_amd import graph as G  # noqa: E402
from test_block_graph_gpu import attention64, gctx  # noqa: E402,F401

U32 = G.SimpleDType.U32


@pytest.mark.parametrize("frozen", [("k", "v"), ("k",), ("v",)])
def test_layers_with_frozen_operands(gctx, frozen):  # noqa: F811
    T, C, heads = 70, 48, 3
    sizes, starts = (40, 90), ([0, 20, 40], [0, 33, 90])  # keys of the two layers
    qs = [0, 30, 70]
    g, meta = G.Graph(G.MEAN_SQUARED_ERROR, G.Optim.sgd().lower), G.Metadata.new()
    fT, fC, fN, fK0, fK1 = (meta.new_field() for _ in range(5))
    with g.define_ops() as ops:
        s = [ops.input([fN], U32) for _ in range(3)]
        x = ops.input([fT, fC])
        for i, f in enumerate((fK0, fK1)):
            k, v = (ops.input([f, fC], requires_grad=n not in frozen) for n in "kv")
            x = ops.attention(x, k, v, s[0], heads, causal=False, scale=0.25, k_starts=s[1 + i])
    rng = np.random.default_rng(11)
    shapes = [(T, C)] + [(n, C) for n in sizes for _ in range(2)]
    par = [rng.standard_normal(sh).astype(np.float32) for sh in shapes]
    want = rng.standard_normal((T, C)).astype(np.float32)
    mb = [G.f32_bits(1e-2), T, C, 3, *sizes]
    st = gctx.alloc_tensors(g, g.compute_saved_nodes(), mb)
    ins = [gctx.init_tensor_u32((3,), np.array(v, np.uint32)) for v in (qs, *starts)]
    ins += [gctx.init_tensor_f32(p.shape, p) for p in par]
    sch = gctx.schedule(g.lower(meta), mb, ins, st)
    gctx.dispatch_forward(sch)
    gctx.dispatch_loss(sch, gctx.init_tensor_f32((T, C), want))
    gctx.dispatch_backward(sch)
    gctx.sync()
    p = [torch.from_numpy(a).double().requires_grad_() for a in par]
    y = p[0]
    for i in range(2):
        y = attention64(y, p[1 + 2 * i], p[2 + 2 * i], qs, starts[i], heads, heads, 0.25, False)
    ((y - torch.from_numpy(want).double()) ** 2).sum().backward()
    by = {t.node: gctx.download(t) for t in st.grad_tensors}
    nodes = [3, 4, 5, 7, 8]  # x, then k and v of each layer around its attention node
    for n, name, a in zip(nodes, ("x", "k", "v", "k", "v"), p):
        assert (n in by) == (name not in frozen)
        if n in by:
            assert normwise_rel(by[n].reshape(a.shape), a.grad.numpy()) < 1e-5 * math.sqrt(T), n
    st.plan.close()
