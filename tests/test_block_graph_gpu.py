"""RMS norm, attention and token log probabilities as they are used together: nodes of a
token model's graph, and direct calls around the path's products, eager and captured.

Gradients are held normwise (max error over max value).  fp32: 1e-5 sqrt of the longest
sum, the bar of the path's products.  16 bits: every tensor rounds once per node, half a
step of its type; from a weight's gradient back through the loss the chain is at most 26
nodes (of the forward: lookup, norm, projection, P, attention, projection, residual, norm,
two products and activation, residual, norm, logits; of the backward as many less two), and
a norm's backward, or the softmax's difference, at most doubles what enters it, from
either side: 26 * 2 * 2 half steps.
"""
import math

import numpy as np
import pytest

from conftest import normwise_rel

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from ferrograd_amd import graph as G  # noqa: E402
from test_token_graph_gpu import ROUND, gelu, to_dtype  # noqa: E402
from test_token_ops_gpu import DTS, note, rand  # noqa: E402

U32 = G.SimpleDType.U32
EPS = float(np.float32(1e-5))
TOL16 = {dt: 26 * 2 * 2 * ROUND[dt] for dt in ("f16", "bf16")}


def norm64(x, gamma):
    return x / torch.sqrt((x * x).mean(1, keepdim=True) + EPS) * gamma


def attention64(q, k, v, qs, ks, heads, kv, scale, causal):
    """Packed sequences in fp64, differentiable; rows of no sequence are 0."""
    D, rows = q.shape[1] // heads, []
    out = torch.zeros_like(q)
    for a, b, c, d in zip(qs[:-1], qs[1:], ks[:-1], ks[1:]):
        if b == a or d == c:
            continue
        see = torch.ones(b - a, d - c, dtype=torch.bool, device=q.device)
        if causal:
            see = see.tril((d - c) - (b - a))
        none = ~see.any(1)
        for h in range(heads):
            g = h // (heads // kv)
            z = q[a:b, h * D:h * D + D] @ k[c:d, g * D:g * D + D].t() * scale
            z = torch.where(see | none[:, None], z, -math.inf)
            p = torch.where(none[:, None], 0.0, torch.softmax(z, 1))
            rows.append((slice(a, b), slice(h * D, h * D + D), p @ v[c:d, g * D:g * D + D]))
    for r, col, val in rows:
        out = out.index_put((torch.arange(r.start, r.stop, device=q.device)[:, None],
                             torch.arange(col.start, col.stop, device=q.device)[None]), val)
    return out


class Model:
    """tokens -> table -> layers of [norm, q k v, attention, projection, added; norm,
    Linear + gelu, Linear, added] -> norm -> Linear -> softmax, cross entropy."""

    def __init__(self, gctx, dt, starts, T, V, C, heads, kv, H, K, layers=1, optim=None, seed=5):
        self.gctx, self.dt, self.starts, self.layers = gctx, dt, starts, layers
        self.heads, self.kv, self.C = heads, kv, C
        D = C // heads
        self.scale = float(np.float32(1.0 / math.sqrt(D)))
        self.graph, meta = G.Graph(G.CROSS_ENTROPY, (optim or G.Optim.sgd()).lower), G.Metadata.new()
        dims = dict(T=T, V=V, C=C, E=kv * D, H=H, K=K, N=len(starts))
        f = {k: meta.new_field() for k in dims}
        d = {"f32": G.SimpleDType.F32, "f16": G.SimpleDType.F16, "bf16": G.SimpleDType.BF16}[dt]
        rng = np.random.default_rng(seed)
        self.host, self.names = [], []
        with self.graph.define_ops() as ops:
            tok, st = ops.input([f["T"]], U32), ops.input([f["N"]], U32)

            def par(name, shape):
                s = tuple(dims[c] for c in shape)
                a = rng.standard_normal(s)
                a = 1.0 + 0.2 * a if len(s) == 1 else a if name == "table" else a / math.sqrt(s[0])
                self.host.append(to_dtype(a, dt))
                self.names.append(name)
                return ops.input([f[c] for c in shape], d)

            x = ops.embedding(par("table", "VC"), tok)
            for l in range(layers):
                h = ops.rms_norm(x, par(f"g{l}", "C"), eps=EPS)
                q, k, v = (ops.matmul(h, par(f"{n}{l}", s)) for n, s in (("q", "CC"), ("k", "CE"),
                                                                        ("v", "CE")))
                a = ops.attention(q, k, v, st, heads, kv, scale=self.scale)
                x = ops.add(x, ops.matmul(a, par(f"o{l}", "CC")))
                h = ops.rms_norm(x, par(f"m{l}", "C"), eps=EPS)
                x = ops.add(x, ops.matmul(ops.gelu(ops.matmul(h, par(f"u{l}", "CH"))),
                                          par(f"d{l}", "HC")))
            ops.softmax(ops.matmul(ops.rms_norm(x, par("g", "C"), eps=EPS), par("out", "CK")))
        self.tokens = rng.integers(0, V, T).astype(np.uint32)
        self.labels = rng.integers(0, K, T).astype(np.uint32)
        mb = [G.f32_bits(1e-3)] + list(dims.values())
        self.st = gctx.alloc_tensors(self.graph, self.graph.compute_saved_nodes(), mb)
        init = {"f32": gctx.init_tensor_f32, "f16": gctx.init_tensor_f16,
                "bf16": gctx.init_tensor_bf16}[dt]
        self.ins = [gctx.init_tensor_u32((T,), self.tokens),
                    gctx.init_tensor_u32((len(starts),), np.array(starts, np.uint32))]
        self.ins += [init(tuple(a.shape), a.float().numpy()) for a in self.host]
        self.sch = gctx.schedule(self.graph.lower(meta), mb, self.ins, self.st)
        self.target = gctx.new_onehot_init(self.labels)

    def step(self):
        self.gctx.dispatch_forward(self.sch)
        self.gctx.dispatch_loss(self.sch, self.target)
        self.gctx.dispatch_backward(self.sch)
        self.gctx.sync()

    def grads(self):
        nodes = [i for i, nd in enumerate(self.graph.nodes) if nd.op == G.OP_INPUT][2:]
        by = {t.node: t for t in self.st.grad_tensors}
        out = []
        for n, a in zip(nodes, self.host):
            g = self.gctx.download(by[n])
            g = G.bf16_to_f32(g) if g.dtype == np.uint16 else g.astype(np.float32)
            out.append(g.reshape(tuple(a.shape)))
        return out

    def reference(self):
        p = [a.clone().cuda().requires_grad_() for a in self.host]
        it = iter(p)
        x = next(it)[torch.from_numpy(self.tokens.astype(np.int64)).cuda()]
        terms = []
        for _ in range(self.layers):
            h = norm64(x, next(it))
            q, k, v = (h @ next(it) for _ in range(3))
            terms.append((h, q, k, v))
            a = attention64(q, k, v, self.starts, self.starts, self.heads, self.kv, self.scale, True)
            a.retain_grad()
            terms[-1] += (a,)
            x = x + a @ next(it)
            h = norm64(x, next(it))
            x = x + gelu(h @ next(it)) @ next(it)
        z = norm64(x, next(it)) @ next(it)
        lab = torch.from_numpy(self.labels.astype(np.int64)).cuda()
        rows = torch.logsumexp(z, 1) - z.gather(1, lab[:, None])[:, 0]
        rows.sum().backward()
        # What the terms of q's and k's gradients can reach (errors).
        self.reach = [len(h) * self.scale * (self.C // self.heads) * float(
            (h.abs().max() * torch.maximum(q.abs().max(), k.abs().max()) * v.abs().max()
             * a.grad.abs().max()).detach()) for h, q, k, v, a in terms]
        return float(rows.mean().detach()), [a.grad.cpu().numpy() for a in p]

    def errors(self, ref):
        """Normwise, but for gradients that are 0: a batch of one token throughout has equal
        rows of v, so that dP - delta cancels and q's and k's weights get none.  Nothing is
        to be divided by then; the gradient is T sums of products h dq, dq = scale * sum
        over keys of P (dout . v - delta) k, in which the terms that cancel are at most
        D max|dout| max|v|, so that what rounding leaves is a tolerance's share of
        T max|h| scale D max|dout| max|v| max|k| (or |q|)."""
        out = {}
        for n, g, r in zip(self.names, self.grads(), ref):
            exact0 = n[0] in "qk" and len(set(self.tokens)) == 1
            out[n] = np.abs(g).max() / self.reach[int(n[1:])] if exact0 else normwise_rel(g, r)
        return out

    def close(self):
        self.st.plan.close()
        for t in self.ins + [self.target]:
            t.free()


@pytest.fixture(scope="module")
def gctx(gpu_ctx):
    return G.GpuContext(gpu_ctx)


# starts, T, V, C, heads, kv, H, K, layers
MODELS = [
    ([0, 3], 3, 5, 8, 2, 1, 16, 4, 1),
    ([0, 40, 40, 61], 64, 50, 32, 4, 2, 48, 10, 2),              # rows of no sequence
    ([5, 300, 301, 690], 700, 301, 96, 2, 2, 130, 77, 1),
    ([0, 1000, 2048], 2048, 500, 512, 8, 2, 256, 100, 1),
]


@pytest.mark.parametrize("case", MODELS, ids=lambda c: f"T{c[1]}xC{c[3]}")
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_model_gradients(gctx, dt, case):
    note("model", dt, case)
    starts, *size, layers = case
    m = Model(gctx, dt, starts, *size, layers=layers)
    m.step()
    loss, ref = m.reference()
    tol = 1e-5 * math.sqrt(max(size)) if dt == "f32" else TOL16[dt] * layers
    got_loss = float(gctx.download(m.st.mean_loss)[0])
    errs = m.errors(ref)
    print(errs, flush=True)
    assert abs(got_loss - loss) < (1e-5 if dt == "f32" else tol) * max(1.0, abs(loss))
    assert all(e < tol for e in errs.values()), errs
    m.close()


@pytest.mark.parametrize("optim", ["sgd", "adam"])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_captured_steps_give_the_eager_bits(gctx, dt, optim):
    starts, *size, layers = MODELS[2]
    opt = getattr(G.Optim, optim)
    a, b = (Model(gctx, dt, starts, *size, layers=layers, optim=opt()) for _ in range(2))
    other = Model(gctx, "f32", *MODELS[1][:-1], optim=opt())
    gctx.capture_step(b.sch, b.target)
    for k in range(4):
        a.step()
        gctx.dispatch_optim(a.sch)
        gctx.launch_step(b.sch)
        gctx.sync()
        for x, y, n in zip(a.ins[2:], b.ins[2:], a.names):
            assert np.array_equal(gctx.download(x), gctx.download(y)), (k, n)
        other.step()
        gctx.dispatch_optim(other.sch)
    for m in (a, b, other):
        m.close()


@pytest.mark.parametrize("frozen", [(), (0,), (1, 2), (2,)])
def test_gradients_that_are_added_and_inputs_that_need_none(gctx, frozen):
    """k feeds a sum beside attention, x a norm and a sum: the gradients add.  Queries of
    other lengths than the keys, and inputs without a gradient."""
    T, C, heads = 90, 48, 3
    qs, ks = [2, 30, 31, 80], [0, 33, 60, 77]
    g, meta = G.Graph(G.MEAN_SQUARED_ERROR, G.Optim.sgd().lower), G.Metadata.new()
    fT, fC, fN = (meta.new_field() for _ in range(3))
    with g.define_ops() as ops:
        s0, s1 = ops.input([fN], U32), ops.input([fN], U32)
        q, k, v = (ops.input([fT, fC], requires_grad=i not in frozen) for i in range(3))
        gamma = ops.input([fC])
        a = ops.attention(q, k, v, s0, heads, causal=False, scale=0.25, k_starts=s1)
        y = ops.add(a, k)
        ops.add(y, ops.rms_norm(y, gamma, eps=EPS))
    rng = np.random.default_rng(9)
    par = [rng.standard_normal(s).astype(np.float32) for s in [(T, C)] * 3 + [(C,)]]
    want = rng.standard_normal((T, C)).astype(np.float32)
    mb = [G.f32_bits(1e-2), T, C, len(qs)]
    st = gctx.alloc_tensors(g, g.compute_saved_nodes(), mb)
    ins = [gctx.init_tensor_u32((4,), np.array(s, np.uint32)) for s in (qs, ks)]
    ins += [gctx.init_tensor_f32(p.shape, p) for p in par]
    sch = gctx.schedule(g.lower(meta), mb, ins, st)
    gctx.dispatch_forward(sch)
    gctx.dispatch_loss(sch, gctx.init_tensor_f32((T, C), want))
    gctx.dispatch_backward(sch)
    gctx.sync()
    p = [torch.from_numpy(a).double().requires_grad_() for a in par]
    y = attention64(p[0], p[1], p[2], qs, ks, heads, heads, 0.25, False) + p[1]
    y = y + norm64(y, p[3])
    ((y - torch.from_numpy(want).double()) ** 2).sum().backward()
    by = {t.node: gctx.download(t) for t in st.grad_tensors}
    assert {2, 3, 4, 5} & set(by) == {2, 3, 4, 5} - {2 + i for i in frozen}
    for n, a in zip((2, 3, 4, 5), p):
        if n - 2 not in frozen:
            assert normwise_rel(by[n].reshape(a.shape), a.grad.numpy()) < 1e-5 * math.sqrt(T), n
    st.plan.close()


class Block:
    """One attention layer and the head of a model by direct calls, forward and backward,
    on 16-bit tensors: the norms with the residual, the second one's output kept in 8 bits
    for its product's gradient, q, k and v from one product."""

    def __init__(self, ctx, dt, starts, T, C, heads, kv, V, seed=3):
        self.ctx, self.code, self.dt, self.starts = ctx, DTS[dt][0], dt, starts
        self.T, self.C, self.heads, self.kv, self.V = T, C, heads, kv, V
        self.D, self.W = C // heads, C + 2 * kv * (C // heads)
        new = lambda *s: torch.zeros(s, dtype=DTS[dt][1], device="cuda")
        f32 = lambda *s: torch.zeros(s, device="cuda")
        self.x, self.r = rand((T, C), dt, seed), rand((T, C), dt, seed + 1)
        self.g0, self.g1 = (rand((1, C), dt, seed + 2 + i, 0.2, 1.0)[0] for i in range(2))
        self.wqkv = rand((C, self.W), dt, seed + 4, C ** -0.5)
        self.wo, self.wv = (rand((C, n), dt, seed + 5 + i, C ** -0.5) for i, n in ((0, C), (1, V)))
        self.tok = torch.randint(0, V, (T,), generator=torch.Generator().manual_seed(seed),
                                 dtype=torch.int32).cuda()
        self.qs = torch.tensor(starts, dtype=torch.int32, device="cuda")
        self.s0, self.y0, self.o, self.s1, self.y1, self.a = (new(T, C) for _ in range(6))
        self.qkv, self.z = new(T, self.W), new(T, V)
        self.q8 = torch.zeros((T, C), dtype=torch.int8, device="cuda")
        self.e8 = torch.zeros((T, (C + 31) // 32), dtype=torch.uint8, device="cuda")
        self.rs0, self.rs1, self.logp, self.ent, self.lse = (f32(T) for _ in range(5))
        self.alse, self.top_logp = f32(heads, T), f32(T, 4)
        self.top = torch.zeros((T, 4), dtype=torch.int32, device="cuda")
        self.dlogp, self.dent = rand((1, T), "f32", seed + 8)[0], rand((1, T), "f32", seed + 9)[0]
        self.dz, self.dqkv = new(T, V), new(T, self.W)
        self.dy1, self.ds1, self.da, self.dy0, self.ds0, self.scratch = (new(T, C) for _ in range(6))
        self.dwv, self.dwo, self.dwqkv = new(C, V), new(C, C), new(C, self.W)
        self.dg0, self.dg1 = new(C), new(C)

    def outputs(self):
        return [self.s0, self.y0, self.rs0, self.qkv, self.a, self.alse, self.s1, self.y1, self.q8,
                self.e8, self.rs1, self.z, self.logp, self.ent, self.lse, self.top, self.top_logp,
                self.dz, self.dwv, self.ds1, self.dg1, self.dwo, self.dqkv, self.dwqkv, self.ds0,
                self.dg0]

    def parts(self, t):
        c, e = self.C, self.kv * self.D
        return t[:, :c], t[:, c:c + e], t[:, c + e:]

    def run(self):
        c, code, T, C, V, W = self.ctx, self.code, self.T, self.C, self.V, self.W
        shape = (self.qs, self.qs, len(self.starts) - 1, T, T, self.heads, self.kv, self.D)
        q, k, v = self.parts(self.qkv)
        c.rms_norm(self.x, C, T, C, self.y0, C, r=self.r, s=self.s0, gamma=self.g0, eps=EPS,
                   rstd=self.rs0, dtype=code)
        c.gemm_x16(code, 0, T, W, C, self.y0, C, self.wqkv, W, self.qkv, W)
        c.attention(q, W, k, W, v, W, *shape, self.a, C, lse=self.alse, dtype=code)
        c.gemm_x16(code, 0, T, C, C, self.a, C, self.wo, C, self.o, C)
        c.rms_norm(self.o, C, T, C, self.y1, C, r=self.s0, s=self.s1, gamma=self.g1, eps=EPS,
                   q=self.q8, e=self.e8, rstd=self.rs1, dtype=code)
        c.gemm_x16(code, 0, T, V, C, self.y1, C, self.wv, V, self.z, V)
        c.token_logprobs(self.z, V, self.tok, T, V, logp=self.logp, entropy=self.ent, lse=self.lse,
                         top=4, top_ids=self.top, top_logp=self.top_logp, dtype=code)
        c.token_logprobs_bwd(self.z, V, self.tok, T, V, self.lse, self.dz, V, entropy=self.ent,
                             dlogp=self.dlogp, dentropy=self.dent, dtype=code)
        c.matmul_bwd_ckpt8(T, V, C, self.q8, C, self.e8, (C + 31) // 32, self.wv, V, self.dz, V,
                           self.scratch, self.dy1, C, self.dwv, V, dtype=code)
        c.rms_norm_bwd(self.s1, C, self.dy1, C, self.rs1, T, C, gamma=self.g1, dx=self.ds1,
                       dgamma=self.dg1, dtype=code)
        c.matmul_bwd_x16(code, T, C, C, self.a, C, self.wo, C, self.ds1, C, self.da, C, self.dwo, C)
        dq, dk, dv = self.parts(self.dqkv)
        c.attention_bwd(q, W, k, W, v, W, self.a, C, self.da, C, self.alse, *shape, dq, W, dk, W, dv,
                        W, dtype=code)
        c.matmul_bwd_x16(code, T, W, C, self.y0, C, self.wqkv, W, self.dqkv, W, self.dy0, C,
                         self.dwqkv, W)
        c.rms_norm_bwd(self.s0, C, self.dy0, C, self.rs0, T, C, gamma=self.g0, ds=self.ds1,
                       dx=self.ds0, dgamma=self.dg0, dtype=code)

    def reference(self):
        p = [t.double().cpu().requires_grad_() for t in (self.x, self.g0, self.wqkv, self.wo, self.g1,
                                                        self.wv)]
        x, g0, wqkv, wo, g1, wv = p
        s0 = x + self.r.double().cpu()
        qkv = norm64(s0, g0) @ wqkv
        a = attention64(*self.parts(qkv), self.starts, self.starts, self.heads, self.kv,
                        self.D ** -0.5, True)
        y1 = norm64(s0 + a @ wo, g1)

        class Kept(torch.autograd.Function):
            """y.W whose weight's gradient reads y as its 8 bits restore it."""
            @staticmethod
            def forward(ctx, y, W):
                ctx.save_for_backward(W)
                return y @ W

            @staticmethod
            def backward(ctx, d):
                step = torch.exp2(self.e8.double().cpu() - 133)
                y8 = self.q8.double().cpu() * step.repeat_interleave(32, 1)[:, :self.C]
                return d @ ctx.saved_tensors[0].t(), y8.t() @ d

        z = torch.log_softmax(Kept.apply(y1, wv), 1)
        logp = z.gather(1, self.tok.long().cpu()[:, None])[:, 0]
        ent = -(z.exp() * z).sum(1)
        ((logp * self.dlogp.double().cpu()).sum() + (ent * self.dent.double().cpu()).sum()).backward()
        return logp.detach(), ent.detach(), [t.grad for t in p]


BLOCKS = [([0, 1], 1, 64, 2, 1, 33), ([0, 5, 70, 70, 128], 130, 96, 3, 1, 301),
          ([0, 333, 700], 700, 256, 4, 2, 1000)]


@pytest.mark.parametrize("case", BLOCKS, ids=lambda c: f"T{c[1]}xC{c[2]}")
@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_direct_calls_together(gpu_ctx, dt, case):
    note("block", dt, case)
    b = Block(gpu_ctx, dt, *case)
    b.run()
    torch.cuda.synchronize()
    logp, ent, ref = b.reference()
    got = [b.ds0, b.dg0, b.dwqkv, b.dwo, b.dg1, b.dwv]
    errs = [normwise_rel(g.double().cpu().numpy(), r.numpy()) for g, r in zip(got, ref)]
    print(errs, flush=True)
    assert max(errs) < TOL16[dt]
    # The most probable columns' log probabilities fall, and none is below the token's.
    assert (b.top_logp[:, :-1] >= b.top_logp[:, 1:]).all() and (b.top_logp[:, 0] >= b.logp).all()
    # logp is off by its logits' error twice, which is absolute: steps of the largest.
    big = float(b.z.abs().max())
    assert float((b.logp.double().cpu() - logp).abs().max()) < TOL16[dt] * big
    assert float((b.ent.double().cpu() - ent).abs().max()) < TOL16[dt] * big * math.log(case[-1])


@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_captured_calls_share_the_workspace_with_eager_ones(gpu_ctx, dt):
    """The calls on a context of their own, on its own stream, captured once and replayed
    between eager calls of other sizes in the same workspace: the eager bits every time."""
    import ferrograd_amd as fa

    s = torch.cuda.Stream()
    ctx = fa.Context(0, s.cuda_stream)
    try:
        ctx.reserve_workspace(256 << 20)
        b = Block(ctx, dt, *BLOCKS[2])
        other = Block(ctx, "bf16", *BLOCKS[1], seed=40)
        # A cache of one long sequence, whose keys are split, and long rows of few logits.
        kc = rand((9000, 128), dt, 50)
        starts = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
        kstart = torch.tensor([0, 9000], dtype=torch.int32, device="cuda")
        qrow, orow = rand((1, 512), dt, 51), torch.zeros((1, 512), dtype=DTS[dt][1], device="cuda")
        long = rand((2, 50000), dt, 52)
        ltok = torch.tensor([7, 49999], dtype=torch.int32, device="cuda")
        llogp, llse = torch.zeros(2, device="cuda"), torch.zeros(2, device="cuda")

        def calls():
            b.run()
            ctx.attention(qrow, 512, kc, 128, kc, 128, starts, kstart, 1, 1, 9000, 4, 1, 128, orow,
                          512, dtype=DTS[dt][0])
            ctx.token_logprobs(long, 50000, ltok, 2, 50000, logp=llogp, lse=llse, dtype=DTS[dt][0])

        outs = b.outputs() + [orow, llogp, llse]
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            calls()
        torch.cuda.synchronize()
        want = [t.clone() for t in outs]
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            calls()
        for rep in range(4):
            for t in outs:
                t.zero_()
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            for i, (t, w) in enumerate(zip(outs, want)):
                assert torch.equal(t, w), (rep, i)
            with torch.cuda.stream(s):
                other.run()
            if rep % 2:
                torch.cuda.synchronize()
    finally:
        ctx.sync()
        ctx.close()
