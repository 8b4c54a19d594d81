"""Layer norm, embedding and 8-bit activation checkpoints in graphs, as a token
model's training step uses them together, on the GPU against fp64 torch."""
import math

import numpy as np
import pytest

from conftest import normwise_rel

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from ferrograd_amd import graph as G  # noqa: E402
from test_token_ops_gpu import C0, C1, quantise  # noqa: E402

U32 = G.SimpleDType.U32
WORD = {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}
ROUND = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def gelu(z):
    return 0.5 * z * (1.0 + torch.tanh(C0 * (z + C1 * z ** 3)))


def to_dtype(a, dt):
    """Host float values rounded to dt (as the tensors hold them), float64."""
    t = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dt]
    return torch.from_numpy(np.asarray(a, np.float32)).to(t).double()


class Model:
    """tokens -> scale * table[tokens] -> layer norm -> [Linear + act (kept in 8
    bits where asked) -> layer norm] x layers -> Linear -> softmax, cross entropy."""

    def __init__(self, gctx, dt, T, V, C, H, K, layers=2, ckpt=(), act="gelu", optim=None,
                 tied=False, norm=True, seed=5, weights=None, scale=2.0):
        self.dt, self.act, self.scale, self.norm = dt, act, scale, norm
        self.graph, meta = G.Graph(G.CROSS_ENTROPY, (optim or G.Optim.adam()).lower), G.Metadata.new()
        fT, fV, fC, fH, fK = (meta.new_field() for _ in range(5))
        d = {"f32": G.SimpleDType.F32, "f16": G.SimpleDType.F16, "bf16": G.SimpleDType.BF16}[dt]
        rng = np.random.default_rng(seed)
        self.host, self.names = [], []

        def param(name, shape, make):
            a = weights(name, shape) if weights else make(shape)
            self.host.append(to_dtype(a, dt))
            self.names.append(name)

        near1 = lambda s: 1.0 + 0.2 * rng.standard_normal(s)
        near0 = lambda s: 0.1 * rng.standard_normal(s)
        dense = lambda s: rng.standard_normal(s) * math.sqrt(2.0 / s[0])
        with self.graph.define_ops() as ops:
            tok = ops.input([fT], U32)
            table = ops.input([fV, fC], d)
            param("table", (V, C), lambda s: rng.standard_normal(s))

            def ln(h, f, n, tag):
                if not norm:
                    return h
                param("gamma" + tag, (n,), near1)
                param("beta" + tag, (n,), near0)
                return ops.layer_norm(h, ops.input([f], d), ops.input([f], d), eps=1e-5)

            h = ln(ops.embedding(table, tok, scale=scale), fC, C, "")
            fin, nin = fC, C
            for l in range(layers):
                W, b = ops.input([fin, fH], d), ops.input([fH], d)
                param(f"W{l}", (nin, H), dense)
                param(f"b{l}", (H,), near0)
                h = getattr(ops, act)(ops.bias_add(ops.matmul(h, W), b))
                fin, nin = fH, H
                if l in ckpt:
                    ops.ckpt8(h)
            W = ops.input([fin, fK], d)
            param("Wo", (nin, K), dense)
            h = ops.matmul(h, W)
            if norm:
                h = ln(h, fK, K, "o")
            ops.softmax(h)
        self.layers = layers
        self.tokens = rng.integers(0, V, T).astype(np.uint32)
        self.tokens[: T // 3] = V // 2  # a frequent token
        self.labels = rng.integers(0, K, T).astype(np.uint32)
        self.gctx = gctx
        mb = [G.f32_bits(1e-2), T, V, C, H, K]
        self.st = gctx.alloc_tensors(self.graph, self.graph.compute_saved_nodes(), mb)
        init = {"f32": gctx.init_tensor_f32, "f16": gctx.init_tensor_f16,
                "bf16": gctx.init_tensor_bf16}[dt]
        self.ins = [gctx.init_tensor_u32(self.tokens.shape, self.tokens)]
        self.ins += [init(tuple(a.shape), a.float().numpy()) for a in self.host]
        self.sch = gctx.schedule(self.graph.lower(meta), mb, self.ins, self.st)
        self.target = gctx.new_onehot_init(self.labels)

    def value(self, t):
        a = self.gctx.download(t)
        return G.bf16_to_f32(a) if a.dtype == np.uint16 else a.astype(np.float32)

    def step(self):
        self.gctx.dispatch_forward(self.sch)
        self.gctx.dispatch_loss(self.sch, self.target)
        self.gctx.dispatch_backward(self.sch)
        self.gctx.sync()

    def grads(self):
        nodes = [i for i, nd in enumerate(self.graph.nodes) if nd.op == G.OP_INPUT][1:]
        by = {t.node: t for t in self.st.grad_tensors}
        return [self.value(by[n]).reshape(tuple(a.shape)) for n, a in zip(nodes, self.host)]

    def reference(self, kept=()):
        """fp64 loss and gradients; layers in `kept` use z restored from 8 bits in
        the backward (and the exact z in the forward)."""
        p = [a.clone().cuda().requires_grad_() for a in self.host]
        it = iter(p)
        tok = torch.from_numpy(self.tokens.astype(np.int64)).cuda()

        def ln(h):
            if not self.norm:
                return h
            g, b = next(it), next(it)
            c = h - h.mean(1, keepdim=True)
            return c / torch.sqrt((c * c).mean(1, keepdim=True) + float(np.float32(1e-5))) * g + b

        class Kept(torch.autograd.Function):
            """act(z).W whose backward reads z as 8 bits restore it."""
            @staticmethod
            def forward(ctx, z, W, act):
                ctx.save_for_backward(quantise(z)[2], W)
                ctx.act = act
                return (act(z)) @ W

            @staticmethod
            def backward(ctx, d):
                z, W = ctx.saved_tensors
                with torch.enable_grad():
                    zz = z.clone().requires_grad_()
                    h = ctx.act(zz)
                dz, = torch.autograd.grad(h, zz, d @ W.t())
                return dz, h.detach().t() @ d, None

        act = gelu if self.act == "gelu" else torch.relu
        h = ln(next(it)[tok] * self.scale)
        z = None
        for l in range(self.layers):
            W, b = next(it), next(it)
            if z is None:
                z = h @ W + b
            else:
                z = (Kept.apply(z, W, act) if l - 1 in kept else act(z) @ W) + b
        W = next(it)
        h = Kept.apply(z, W, act) if self.layers - 1 in kept else act(z) @ W
        h = ln(h)
        lab = torch.from_numpy(self.labels.astype(np.int64)).cuda()
        # The loss's gradient is per row, not of the mean.
        rows = torch.logsumexp(h, 1) - h.gather(1, lab[:, None])[:, 0]
        rows.sum().backward()
        return float(rows.mean().detach()), [a.grad.cpu().numpy() for a in p]

    def close(self):
        self.st.plan.close()
        for t in self.ins + [self.target]:
            t.free()


@pytest.fixture(scope="module")
def gctx(gpu_ctx):
    return G.GpuContext(gpu_ctx)


@pytest.mark.parametrize("size", [(64, 50, 32, 48, 10), (700, 301, 100, 130, 77),
                                  (4096, 1000, 256, 512, 100)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("act", ["relu", "gelu"])
def test_token_model_gradients_fp32(gctx, size, act):
    """Normwise error of every gradient against fp64: 1e-5 sqrt of the longest sum,
    the bar of the path's products."""
    m = Model(gctx, "f32", *size, act=act)
    m.step()
    loss, ref = m.reference()
    tol = 1e-5 * math.sqrt(max(size))
    assert abs(float(m.value(m.st.mean_loss)[0]) - loss) < 1e-5 * max(1.0, abs(loss))
    errs = {n: normwise_rel(g, r) for n, g, r in zip(m.names, m.grads(), ref)}
    print(errs, flush=True)
    assert all(e < tol for e in errs.values()), errs
    m.close()


@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_token_model_gradients_16_bit(gctx, dt):
    """Every tensor rounds once per node; the chain from a weight's gradient back is
    at most 12 nodes long, each off by half a step of its type, and a layer norm's
    backward at most doubles what enters it (its projection is of norm 1, its
    statistics come from rounded values)."""
    m = Model(gctx, dt, 600, 90, 128, 192, 40)
    m.step()
    loss, ref = m.reference()
    tol = 12 * 2 * 2 * ROUND[dt]
    assert abs(float(m.value(m.st.mean_loss)[0]) - loss) < tol * max(1.0, abs(loss))
    errs = {n: normwise_rel(g, r) for n, g, r in zip(m.names, m.grads(), ref)}
    print(errs, flush=True)
    assert all(e < tol for e in errs.values()), errs
    m.close()


def exact_weights(top):
    """Integers (up to `top`) and eighths: every pre-activation of the first layer is
    exact in fp32, so that fp64 rounds the same values to 8 bits.  Up to 3 they are
    sums of a few eighths that 7 bits hold; up to 40 they need more."""
    def make(name, shape):
        rng = np.random.default_rng(sum(map(ord, name)))
        if name == "Wo":
            return rng.standard_normal(shape) * math.sqrt(2.0 / shape[0]) * 3.0 / top
        return rng.integers(-top, top + 1, shape) * (1.0 if name == "table" else 0.125)
    return make


@pytest.mark.parametrize("act", ["relu", "gelu"])
@pytest.mark.parametrize("top", [3, 40])
@pytest.mark.parametrize("size", [(64, 50, 32, 48, 10), (900, 301, 40, 515, 33)],
                         ids=lambda s: "x".join(map(str, s)))
def test_ckpt8_gradients_are_those_of_the_restored_values(gctx, size, top, act):
    """One layer kept, its pre-activation exact: the gradients agree with fp64's from
    the restored values as closely as the path's products do; where 8 bits lose
    something, they differ from the exact values' gradients by more."""
    m = Model(gctx, "f32", *size, layers=1, ckpt=(0,), act=act, norm=False, scale=1.0,
              weights=exact_weights(top))
    m.step()
    loss, ref = m.reference(kept=(0,))
    _, plain = m.reference()
    assert abs(float(m.value(m.st.mean_loss)[0]) - loss) < 1e-5 * max(1.0, abs(loss))
    got = m.grads()
    tol = 1e-5 * math.sqrt(max(size))
    errs = {n: normwise_rel(g, r) for n, g, r in zip(m.names, got, ref)}
    off = {n: normwise_rel(g, r) for n, g, r in zip(m.names, got, plain)}
    print(errs, off, flush=True)
    assert all(e < tol for e in errs.values()), errs
    if top > 3:
        assert off["Wo"] > 2 * tol
    m.close()


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_ckpt8_forward_is_unchanged_and_backward_repeats(gctx, dt):
    """The same loss and probabilities to the bit with layers kept in 8 bits or not;
    a second backward of the same forward (restored again) gives the same bits;
    gradients stay within a step's share of the exact ones."""
    size = (300, 64, 96, 160, 24)
    a = Model(gctx, dt, *size, layers=4)
    b = Model(gctx, dt, *size, layers=4, ckpt=(0, 1, 2, 3))
    for m in (a, b):
        m.step()
    assert np.array_equal(a.gctx.download(a.st.forward_out), b.gctx.download(b.st.forward_out))
    assert np.array_equal(a.gctx.download(a.st.mean_loss), b.gctx.download(b.st.mean_loss))
    first = b.grads()
    b.gctx.dispatch_loss(b.sch, b.target)
    b.gctx.dispatch_backward(b.sch)
    b.gctx.sync()
    for x, y in zip(first, b.grads()):
        assert np.array_equal(x, y)
    # Four layers; each restored value is off by at most a 128th of its block's
    # largest, act' by as much times |act''| < 1, seen through norms: a few times that.
    for x, y, n in zip(a.grads(), first, a.names):
        assert normwise_rel(y, x) < 4 * 4 * 2.0 ** -7 + 48 * ROUND[dt], n
    a.close()
    b.close()


@pytest.mark.parametrize("optim", ["sgd", "adam"])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_captured_steps_give_the_eager_bits(gctx, dt, optim):
    """Two models of the same seed, one stepped eagerly, one by replays of a captured
    step with eager work of other sizes between them: the same parameters after each
    of four steps."""
    size = (400, 70, 64, 130, 20)
    opt = getattr(G.Optim, optim)
    a = Model(gctx, dt, *size, ckpt=(0, 1), optim=opt())
    b = Model(gctx, dt, *size, ckpt=(0, 1), optim=opt())
    other = Model(gctx, "f32", 90, 300, 40, 50, 12, optim=opt())
    gctx.capture_step(b.sch, b.target)
    for k in range(4):
        a.step()
        gctx.dispatch_optim(a.sch)
        gctx.launch_step(b.sch)
        gctx.sync()
        for x, y, n in zip(a.ins[1:], b.ins[1:], a.names):
            assert np.array_equal(gctx.download(x), gctx.download(y)), (k, n)
        other.step()
        gctx.dispatch_optim(other.sch)
    for m in (a, b, other):
        m.close()


@pytest.mark.parametrize("ckpt", [(), (0,), (1,), (0, 1)])
def test_captured_small_layers_beside_kept_ones(gctx, ckpt):
    """A long first product, a small hidden layer and a head of few classes, as a captured
    SGD step runs them (split, chained, the loss in the head's product), with each layer
    kept in 8 bits or not: the eager parameters after each of three steps."""
    size = (64, 40, 784, 64, 10)
    make = lambda: Model(gctx, "f32", *size, ckpt=ckpt, optim=G.Optim.sgd(), norm=False)
    a, b = make(), make()
    gctx.capture_step(b.sch, b.target)
    for k in range(3):
        a.step()
        gctx.dispatch_optim(a.sch)
        gctx.launch_step(b.sch)
        gctx.sync()
        for x, y, n in zip(a.ins[1:], b.ins[1:], a.names):
            assert np.array_equal(gctx.download(x), gctx.download(y)), (k, n)
    a.close()
    b.close()


def test_tied_table_and_shared_gamma_add_their_gradients(gctx):
    """A table read by two lookups and a gamma by two layer norms: gradients add."""
    T, V, C = 130, 40, 24
    g, meta = G.Graph(G.MEAN_SQUARED_ERROR, G.Optim.sgd().lower), G.Metadata.new()
    fT, fV, fC = (meta.new_field() for _ in range(3))
    with g.define_ops() as ops:
        t0, t1 = ops.input([fT], U32), ops.input([fT], U32)
        table, gamma = ops.input([fV, fC]), ops.input([fC])
        b0, b1 = ops.input([fC]), ops.input([fC])
        h = ops.layer_norm(ops.embedding(table, t0), gamma, b0)
        ops.add(h, ops.layer_norm(ops.embedding(table, t1, scale=-0.5), gamma, b1))
    rng = np.random.default_rng(9)
    tok = [rng.integers(0, V, T).astype(np.uint32) for _ in range(2)]
    par = [rng.standard_normal(s).astype(np.float32) for s in ((V, C), (C,), (C,), (C,))]
    want = rng.standard_normal((T, C)).astype(np.float32)
    mb = [G.f32_bits(1e-2), T, V, C]
    st = gctx.alloc_tensors(g, g.compute_saved_nodes(), mb)
    ins = [gctx.init_tensor_u32((T,), t) for t in tok]
    ins += [gctx.init_tensor_f32(p.shape, p) for p in par]
    sch = gctx.schedule(g.lower(meta), mb, ins, st)
    gctx.dispatch_forward(sch)
    gctx.dispatch_loss(sch, gctx.init_tensor_f32((T, C), want))
    gctx.dispatch_backward(sch)
    gctx.sync()
    p = [torch.from_numpy(a).double().requires_grad_() for a in par]

    def ln(h, b):
        c = h - h.mean(1, keepdim=True)
        return c / torch.sqrt((c * c).mean(1, keepdim=True) + float(np.float32(1e-5))) * p[1] + b

    y = ln(p[0][torch.from_numpy(tok[0].astype(np.int64))], p[2])
    y = y + ln(-0.5 * p[0][torch.from_numpy(tok[1].astype(np.int64))], p[3])
    ((y - torch.from_numpy(want).double()) ** 2).sum().backward()
    by = {t.node: gctx.download(t) for t in st.grad_tensors}
    for n, a in zip((2, 3, 4, 5), p):
        assert normwise_rel(by[n].reshape(a.shape), a.grad.numpy()) < 1e-5 * math.sqrt(T)
    st.plan.close()


def test_plan_checkpoint_leaves_tokens_out(gctx, tmp_path):
    from ferrograd_amd._lib import call

    path = str(tmp_path / "m.bpat").encode()
    a = Model(gctx, "f32", 64, 50, 32, 48, 10, seed=5)
    a.step()
    gctx.dispatch_optim(a.sch)
    call("fg_plan_save", a.st.plan.handle, path, 5)
    b = Model(gctx, "f32", 64, 50, 32, 48, 10, seed=6)
    was = gctx.download(b.ins[0]).copy()
    call("fg_plan_load", b.st.plan.handle, path)
    for x, y in zip(a.ins[1:], b.ins[1:]):
        assert np.array_equal(gctx.download(x), gctx.download(y))
    assert np.array_equal(gctx.download(b.ins[0]), was)
    a.close()
    b.close()
