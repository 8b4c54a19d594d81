"""Attention over packed sequences against plain fp64 torch, through the C ABI.

Tolerances are error bounds, elementwise, with the terms of test_token_ops_gpu.py: u =
2^-24, h the storage type's rounding.  Products of 16-bit values are exact in fp32, a
score is a sum of D of them, off by at most (D + 4) u of the magnitudes' sum and 4 u of
itself; an exponential is off by its argument's error and 4 u; a sum over keys (or rows)
in any order by its count's u of the magnitudes' sum.  P and dS are rounded to the type
before their second product: h of each.  fp16's smallest steps: P carries 2^8 (2^-33 is
half a step of what it stands for), dS a power of two that brings the largest |dout| to 2^4
at least (half a step: 2^-28 of the largest).  Exponentials below fp32's smallest normal
number are 0: each is off by at most FLUSH = 2^-126 for that.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from test_token_ops_gpu import DTS, U, blank, ld, note, place, rand, within  # noqa: E402


FLUSH = 2.0 ** -126


class Batch:
    """Sequences [(lq, lk)] packed with `gap` rows of no sequence around them; room:
    rows of a cache past each sequence's keys."""

    def __init__(self, seqs, heads, kv, D, dt, causal=True, pad=0, start=0, gap=0, room=0, seed=1,
                 fused=False, std=1.0):
        self.seqs, self.heads, self.kv, self.D, self.dt, self.causal = seqs, heads, kv, D, dt, causal
        self.scale = float(np.float32(1.0 / math.sqrt(D)))
        lq, lk = [a for a, _ in seqs], [b for _, b in seqs]
        self.qs = [gap + sum(lq[:i]) for i in range(len(seqs) + 1)]
        self.ks = [gap + sum(lk[:i]) + room * i for i in range(len(seqs) + 1)]
        self.Tq, self.Tk = self.qs[-1] + gap, self.ks[-1] + gap
        wide, kvw = heads * D, kv * D
        if fused:
            x = rand((self.Tq, wide + 2 * kvw), dt, seed, std, 0.0, pad, start)
            self.q, self.k, self.v = x[:, :wide], x[:, wide:wide + kvw], x[:, wide + kvw:]
        else:
            self.q = rand((self.Tq, wide), dt, seed, std, 0.0, pad, start)
            self.k = rand((self.Tk, kvw), dt, seed + 1, std, 0.0, pad, start)
            self.v = rand((self.Tk, kvw), dt, seed + 2, 1.0, 0.0, pad, start)
        self.pad, self.start = pad, start
        for t in (self.k, self.v):  # what no sequence holds
            dead = torch.ones(self.Tk, dtype=torch.bool)
            for s, b in enumerate(lk):
                dead[self.ks[s]:self.ks[s] + b] = False
            if not fused:
                t[dead.cuda()] = math.nan
        if not fused and gap:
            self.q[:gap] = self.q[self.Tq - gap:] = math.nan
        self.d_qs = torch.tensor(self.qs, dtype=torch.int32, device="cuda")
        self.d_ks = torch.tensor(self.ks, dtype=torch.int32, device="cuda")
        self.d_kl = torch.tensor(lk, dtype=torch.int32, device="cuda") if room else None

    def shape(self):
        return (self.d_qs, self.d_ks, len(self.seqs), self.Tq, self.Tk, self.heads, self.kv, self.D)

    def qkv(self):
        return (self.q, ld(self.q), self.k, ld(self.k), self.v, ld(self.v))

    def forward(self, ctx):
        out, clean = blank((self.Tq, self.heads * self.D), self.dt, self.pad, self.start)
        lse = torch.full((self.heads, self.Tq), 7.0, device="cuda")
        ctx.attention(*self.qkv(), *self.shape(), out, ld(out), k_lens=self.d_kl, scale=self.scale,
                      causal=self.causal, lse=lse, dtype=DTS[self.dt][0])
        torch.cuda.synchronize()
        assert clean()
        return out, lse

    def parts(self, s, head):
        """q, k, v, visible, S of one sequence and head, fp64 on the host."""
        (a, b), D = self.seqs[s], self.D
        c = head // (self.heads // self.kv)
        q = self.q[self.qs[s]:self.qs[s] + a, head * D:head * D + D].double().cpu()
        k = self.k[self.ks[s]:self.ks[s] + b, c * D:c * D + D].double().cpu()
        v = self.v[self.ks[s]:self.ks[s] + b, c * D:c * D + D].double().cpu()
        see = torch.ones(a, b, dtype=torch.bool)
        if self.causal:
            see = see.tril(b - a)
        z = torch.where(see, (q @ k.t()) * self.scale, -math.inf)
        err = torch.where(see, U * ((self.D + 4) * self.scale * (q.abs() @ k.abs().t())
                                    + 4 * z.abs()), 0.0)
        return q, k, v, see, z, err

    def expected(self):
        """(rows, head, columns, out, its bound, lse, its bound, rows that see no key) of
        each sequence and head."""
        h = DTS[self.dt][2]
        tiny = 2.0 ** -33 if self.dt == "f16" else FLUSH
        for s, (a, b) in enumerate(self.seqs):
            for head in range(self.heads):
                _, _, v, see, z, err = self.parts(s, head)
                none = ~see.any(1)
                p = torch.where(none[:, None], 0.0, torch.softmax(z, 1)) if b else torch.zeros(a, 0)
                p = p.double()
                ls = torch.logsumexp(z, 1) if b else torch.full((a,), -math.inf).double()
                e = err.amax(1) if b else torch.zeros(a)
                rel = (h + 2 * e + U * (b + 64))[:, None]
                yield (slice(self.qs[s], self.qs[s] + a), head,
                       slice(head * self.D, head * self.D + self.D), p @ v,
                       rel * (p @ v.abs()) + tiny * v.abs().sum(0), ls,
                       e + U * (b + 24) + 4 * U * ls.abs(), none)

    def check_forward(self, out, lse):
        alive = torch.zeros(self.Tq, dtype=torch.bool)
        got, got_lse = out.cpu(), lse.cpu()
        for rq, head, cols, o, bound, ls, lbound, none in self.expected():
            alive[rq] = True
            within(got[rq, cols], o, bound, self.dt)
            gl = got_lse[head, rq]
            assert torch.equal(gl == -math.inf, none)
            within(gl[~none], ls[~none], lbound[~none])
        assert bool((out[~alive.cuda()] == 7.0).all()) and bool((lse[:, ~alive.cuda()] == 7.0).all())

    def backward(self, ctx, out, lse, dout, accumulate=None):
        made = [blank((self.Tq, self.heads * self.D), self.dt, self.pad, self.start)]
        made += [blank((self.Tk, self.kv * self.D), self.dt, self.pad, self.start) for _ in range(2)]
        g = [m[0] for m in made]
        if accumulate:
            for t, was in zip(g, accumulate):
                t.copy_(was)
        ctx.attention_bwd(*self.qkv(), out, ld(out), dout, ld(dout), lse, *self.shape(), g[0],
                          ld(g[0]), g[1], ld(g[1]), g[2], ld(g[2]), scale=self.scale,
                          causal=self.causal, accumulate=accumulate is not None,
                          dtype=DTS[self.dt][0])
        torch.cuda.synchronize()
        assert all(m[1]() for m in made)
        return g

    def check_backward(self, grads, out, lse, dout, was=None):
        h, D = DTS[self.dt][2], self.D
        G = self.heads // self.kv
        got = [g.cpu() for g in grads]
        old = [torch.zeros_like(g).double() for g in got] if was is None else [w.double().cpu() for w in was]
        alive = [torch.zeros(len(g), dtype=torch.bool) for g in got]
        for s, (a, b) in enumerate(self.seqs):
            rq, rk = slice(self.qs[s], self.qs[s] + a), slice(self.ks[s], self.ks[s] + b)
            alive[0][rq] = True
            alive[1][rk] = alive[2][rk] = True
            for c in range(self.kv):
                dk, dv, bk, bv = (torch.zeros(b, D).double() for _ in range(4))
                group = dout[rq, c * G * D:(c + 1) * G * D].double().abs().cpu()
                big = group.max() if a else 0.0
                for head in range(c * G, c * G + G):
                    cols = slice(head * D, head * D + D)
                    q, k, v, see, z, err = self.parts(s, head)
                    L = lse[head, rq].double().cpu()[:, None]
                    do, o = dout[rq, cols].double().cpu(), out[rq, cols].double().cpu()
                    none = ~see.any(1) if b else torch.ones(a, dtype=torch.bool)
                    p = torch.where(see, torch.exp(z - torch.where(none[:, None], 0.0, L)), 0.0)
                    ep = torch.where(see, 2 * err + U * (8 * torch.where(none[:, None], 0.0, L).abs()
                                                         + 16), 0.0)
                    delta = torch.where(none, 0.0, (do * o).sum(1))[:, None]
                    dp = do @ v.t()
                    ds = torch.where(see, p * (dp - delta), 0.0)
                    ed = U * (D + 8) * (do.abs() @ v.abs().t() + (do * o).abs().sum(1)[:, None])
                    es = torch.where(see, p * ((dp - delta).abs() * ep + ed)
                                     + FLUSH * (dp - delta).abs(), 0.0) + h * ds.abs()
                    tp = FLUSH
                    if self.dt == "f16":
                        es = es + torch.where(see, big * 2.0 ** -28, 0.0)
                        tp = 2.0 ** -33
                    dq = self.scale * (ds @ k)
                    bq = self.scale * (es @ k.abs() + U * (b + 64) * (ds.abs() @ k.abs()))
                    want = dq + old[0][rq, cols]
                    within(got[0][rq, cols], want, bq + 4 * U * (dq.abs() + want.abs()), self.dt)
                    dk += self.scale * (ds.t() @ q)
                    n = a * G
                    bk += self.scale * (es.t() @ q.abs() + U * (n + 64) * (ds.abs().t() @ q.abs()))
                    dv += p.t() @ do
                    bv += (p * (h + ep)).t() @ do.abs() + (U * (n + 64) * p + tp * see).t() @ do.abs()
                cols = slice(c * D, c * D + D)
                for i, (w, bound) in ((1, (dk, bk)), (2, (dv, bv))):
                    want = w + old[i][rk, cols]
                    within(got[i][rk, cols], want, bound + 4 * U * (w.abs() + want.abs()), self.dt)
        for g, al, w in zip(grads, alive, [7.0] * 3 if was is None else was):
            rest = g[~al.cuda()]
            assert torch.equal(rest, torch.full_like(rest, 7.0) if was is None else w[~al.cuda()])


SETS = [
    # seqs, heads, kv, D, causal, pad, start, gap
    ([(1, 1)], 1, 1, 1, True, 0, 0, 0),
    ([(3, 3), (1, 1), (0, 0), (40, 40)], 2, 1, 8, True, 0, 0, 2),
    ([(64, 64)], 2, 2, 64, True, 0, 0, 0),
    ([(130, 130), (7, 7)], 4, 2, 64, True, 8, 0, 1),
    ([(130, 300), (33, 33)], 2, 2, 64, False, 0, 0, 0),
    ([(70, 70), (200, 200), (1, 1)], 4, 1, 128, True, 0, 0, 0),
    ([(257, 257)], 2, 1, 128, False, 8, 0, 0),
    ([(50, 90), (129, 257)], 6, 2, 128, True, 0, 0, 3),
    ([(20, 5), (9, 0), (0, 9), (100, 60)], 2, 1, 64, True, 0, 0, 1),   # rows that see no key
    ([(20, 5), (9, 0), (0, 9)], 2, 2, 128, False, 0, 0, 0),
    ([(77, 77), (31, 95)], 3, 3, 72, True, 3, 1, 2),
    ([(77, 77), (65, 65)], 6, 2, 100, False, 1, 1, 0),
    ([(90, 90)], 7, 1, 33, True, 5, 3, 0),
    ([(150, 150)], 8, 1, 128, True, 3, 0, 0),
    ([(300, 700), (40, 1000)], 2, 1, 96, True, 8, 0, 1),
    ([(500, 500), (3, 3)], 4, 2, 90, False, 1, 0, 0),
    ([(1, 700), (1, 33), (2, 2), (1, 1)], 8, 2, 128, True, 0, 0, 0),   # single tokens
    ([(1, 129), (3, 64), (1, 0)], 5, 1, 80, True, 1, 1, 1),
]
IDS = [f"{i}-D{c[3]}" for i, c in enumerate(SETS)]


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("case", SETS, ids=IDS)
def test_forward(gpu_ctx, dt, case):
    note("attention", dt, case)
    seqs, heads, kv, D, causal, pad, start, gap = case
    b = Batch(seqs, heads, kv, D, dt, causal, pad, start, gap)
    b.check_forward(*b.forward(gpu_ctx))


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("case", SETS, ids=IDS)
def test_backward(gpu_ctx, dt, case):
    note("attention_bwd", dt, case)
    seqs, heads, kv, D, causal, pad, start, gap = case
    b = Batch(seqs, heads, kv, D, dt, causal, pad, start, gap)
    out, lse = b.forward(gpu_ctx)
    dout = rand((b.Tq, heads * D), dt, 9, 1.0, 0.0, pad, start)
    grads = b.backward(gpu_ctx, out, lse, dout)
    b.check_backward(grads, out, lse, dout)
    again = b.backward(gpu_ctx, out, lse, dout)
    assert all(torch.equal(x, y) for x, y in zip(grads, again))
    was = [rand(tuple(g.shape), dt, 10 + i) for i, g in enumerate(grads)]
    b.check_backward(b.backward(gpu_ctx, out, lse, dout, was), out, lse, dout, was)


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lq,lens,heads,kv,D,room", [
    (1, [5000], 8, 1, 128, 3), (1, [3000, 1, 0, 2047], 4, 4, 64, 40), (4, [6000, 900], 8, 2, 128, 0),
    (1, [4000], 3, 1, 48, 1), (40, [5000], 4, 2, 128, 0), (200, [9000], 2, 1, 64, 7)])
def test_tokens_over_a_cache(gpu_ctx, dt, lq, lens, heads, kv, D, room):
    """Few rows over many keys: keys shared out over waves and workgroups, a cache with
    room (NaN past each sequence's keys)."""
    note("cache", dt, lq, lens, heads, kv, D, room)
    b = Batch([(lq, n) for n in lens], heads, kv, D, dt, True, room=room)
    b.check_forward(*b.forward(gpu_ctx))


def test_many_sequences(gpu_ctx):
    """More sequences than a wave searches at once, most of them of no or few rows."""
    gen = np.random.default_rng(5)
    seqs = [(int(a), int(a + b)) for a, b in zip(gen.integers(0, 4, 300), gen.integers(0, 6, 300))]
    seqs[70] = (150, 150)
    for dt, D in (("bf16", 64), ("f32", 16)):
        b = Batch(seqs, 2, 1, D, dt, True, gap=1)
        out, lse = b.forward(gpu_ctx)
        b.check_forward(out, lse)
        dout = rand((b.Tq, 2 * D), dt, 9)
        b.check_backward(b.backward(gpu_ctx, out, lse, dout), out, lse, dout)


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_fused_projection_and_large_scores(gpu_ctx, dt):
    """q, k and v as columns of one matrix; scores far apart (one key takes all)."""
    b = Batch([(90, 90), (38, 38)], 4, 2, 64, dt, True, 8, fused=True, std=6.0)
    out, lse = b.forward(gpu_ctx)
    b.check_forward(out, lse)
    dout = rand((b.Tq, 4 * 64), dt, 9, 1.0, 0.0, 8)
    b.check_backward(b.backward(gpu_ctx, out, lse, dout), out, lse, dout)


def test_small_gradients_of_fp16(gpu_ctx):
    """dout near fp16's smallest normal numbers, rows of unlike size: dS keeps its bits."""
    for D in (64, 40):
        b = Batch([(300, 300)], 2, 1, D, "f16", True)
        out, lse = b.forward(gpu_ctx)
        dout = rand((b.Tq, 2 * D), "f16", 9)
        dout[:150] *= 2.0 ** -11
        grads = b.backward(gpu_ctx, out, lse, dout)
        b.check_backward(grads, out, lse, dout)


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D,lq,lk", [(64, 100, 100), (128, 70, 140), (40, 65, 65), (128, 1, 90), (96, 300, 300)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_keys_out_of_sight_do_not_reach_a_row(gpu_ctx, dt, D, lq, lk, bad):
    """The last key (causal: seen by the last row alone) holds NaN or infinity: the other
    rows, and the gradients that do not pass through it, are as with a number there."""
    note("out of sight", dt, D, lq, lk, bad)
    lk = max(lk, lq)
    b = Batch([(lq, lk + 1), (lq, lk)], 2, 1, D, dt, True)
    rows = slice(0, lq - 1)  # of the first sequence; and all of the second
    want, want_lse = b.forward(gpu_ctx)
    keep_k, keep_v = b.k.clone(), b.v.clone()
    exact = list(b.expected())
    b.k[lk], b.v[lk] = bad, bad
    out, lse = b.forward(gpu_ctx)
    for rq, head, cols, o, bound, ls, lbound, _ in exact:
        n = lq - 1 if rq.start == 0 else lq
        within(out[rq, cols][:n].cpu(), o[:n], bound[:n], dt)
        within(lse[head, rq][:n].cpu(), ls[:n], lbound[:n])
    assert torch.isnan(out[lq - 1].float()).any()
    # Gradients: the last row's query and dout are bad; earlier keys' sums hold them, the
    # last key's own alone do where every other row does not see it.
    b.k.copy_(keep_k)
    b.v.copy_(keep_v)
    dout = rand((b.Tq, 2 * D), dt, 9)
    ref = b.backward(gpu_ctx, want, want_lse, dout)
    if lq > 1:
        dout2, q0 = dout.clone(), b.q.clone()
        dout2[0] = bad  # the first row: seen keys 0 .. lk - lq + 1
        b.q[0] = bad
        got = b.backward(gpu_ctx, want, want_lse, dout2)
        b.q.copy_(q0)
        past = slice(lk - lq + 2, lk + 1)  # keys that the first row does not see
        for i in (1, 2):
            assert torch.isfinite(got[i][past].float()).all()
            assert torch.equal(got[i][lk + 1:], ref[i][lk + 1:])
        assert torch.equal(got[0][1:], ref[0][1:])
    b.k[lk] = bad
    got = b.backward(gpu_ctx, want, want_lse, dout)
    assert torch.isfinite(got[0][rows].float()).all()
    assert torch.equal(got[0][lq:], ref[0][lq:])


def test_gradient_by_differences(gpu_ctx):
    """dq, dk and dv against central differences of the forward, in fp32: each output is
    off by at most 400 u of order one, f''' h^2 / 6 of order one."""
    h = 2.0 ** -6
    b = Batch([(9, 12), (5, 5)], 4, 2, 16, "f32", True)
    w = rand((b.Tq, 64), "f32", 9, 0.3)

    def objective():
        return (b.forward(gpu_ctx)[0].double() * w.double()).sum().item()

    out, lse = b.forward(gpu_ctx)
    grads = b.backward(gpu_ctx, out, lse, w)
    for t, g in zip((b.q, b.k, b.v), grads):
        for i in (0, 37, t.numel() - 1):
            was = t.view(-1)[i].item()
            t.view(-1)[i] = was + h
            up = objective()
            t.view(-1)[i] = was - h
            down = objective()
            t.view(-1)[i] = was
            tol = 400 * U * w.double().abs().sum().item() / h + 4 * h * h
            assert abs((up - down) / (2 * h) - g.view(-1)[i].item()) <= tol
