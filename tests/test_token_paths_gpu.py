"""Layer norm and embedding on paths of their own: in place in every
layer norm kernel, every form of the token sort, table rows that the summing launch
zeroes, unused rows whatever the scale, captured gradients that use the workspace."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from test_token_ops_gpu import (DTS, U, blank, emb_grad, ld, ln_bwd_reference, note, place,  # noqa: E402
                                rand, tokens_of, within)

# -------------------------------------------------------------- layer norm
FWD_IN_PLACE = [  # rows held by 16, 64 and 256 lanes, by a workgroup, and read three times
    ("bf16", 9000, 72), ("f16", 3001, 1023), ("f32", 1100, 4096), ("bf16", 700, 2048),
    ("f32", 30, 4001), ("bf16", 300, 20001), ("f32", 300, 30000), ("f32", 3, 140000)]


@pytest.mark.parametrize("dt,R,C", FWD_IN_PLACE)
def test_layer_norm_in_place(gpu_ctx, dt, R, C):
    note("layer_norm in place", dt, R, C)
    x = rand((R, C), dt, 301, 2.0, -1.0, 3, 1)
    gamma, beta = rand((1, C), dt, 302, 0.2, 1.0)[0], rand((1, C), dt, 303)[0]
    y, untouched = blank((R, C), dt, 3, 1)
    args = dict(gamma=gamma, beta=beta, dtype=DTS[dt][0])
    gpu_ctx.layer_norm(x, ld(x), R, C, y, ld(y), **args)
    gpu_ctx.layer_norm(x, ld(x), R, C, x, ld(x), **args)
    torch.cuda.synchronize()
    assert torch.equal(x, y) and untouched()


BWD_IN_PLACE = [
    # Few rows in one launch; rows in registers, several to a workgroup, in turn ...
    ("bf16", 600, 1024), ("bf16", 9000, 72), ("f16", 2500, 1023), ("f32", 1500, 999),
    ("f32", 700, 4097), ("f16", 700, 8001),
    # ... with the weights' sums in LDS, and columns and rows in launches of their own,
    # rows in registers and read twice.
    ("bf16", 600, 16384), ("f32", 600, 9001), ("f32", 520, 16384), ("f16", 300, 17001),
    ("f32", 300, 20001), ("bf16", 300, 50000), ("f32", 300, 40000), ("bf16", 260, 70001)]


@pytest.mark.parametrize("dt,R,C", BWD_IN_PLACE)
def test_layer_norm_backward_in_place(gpu_ctx, dt, R, C):
    """dx over x or over dy: the bits of a dx of its own, and so the weights'."""
    note("layer_norm_bwd in place", dt, R, C)
    code = DTS[dt][0]
    x, dy = rand((R, C), dt, 311, 1.0, 0.5, 1), rand((R, C), dt, 312, 1.0, 0.1, 1)
    gamma = rand((1, C), dt, 313, 0.2, 1.0)[0]
    xd = x.double()
    mean = xd.mean(1).float()
    rstd = (1.0 / torch.sqrt(((xd - mean.double()[:, None]) ** 2).mean(1) + 1e-5)).float()
    del xd
    outs = []
    for weights in (True, False):
        for where in ("own", "dy", "x"):
            a, b = place(x.cpu(), 1), place(dy.cpu(), 1)
            dx = {"own": blank((R, C), dt, 1)[0], "dy": b, "x": a}[where]
            dg, db = (torch.empty(C, dtype=x.dtype, device="cuda") for _ in range(2))
            gpu_ctx.layer_norm_bwd(a, ld(a), b, ld(b), mean, rstd, R, C, gamma=gamma, dx=dx,
                                   lddx=ld(dx), dgamma=dg if weights else None,
                                   dbeta=db if weights else None, dtype=code)
            torch.cuda.synchronize()
            outs.append((dx, dg, db) if weights else (dx,))
    for o in outs[1:3]:
        assert all(torch.equal(p, q) for p, q in zip(outs[0], o))
    for o in outs[4:]:
        assert torch.equal(outs[3][0], o[0])
    rdx, bdx, rdg, bdg, rdb, bdb = ln_bwd_reference(x, dy, gamma, mean, rstd)
    for got, ref, bound in ((outs[0][0], rdx, bdx), (outs[3][0], rdx, bdx), (outs[0][1], rdg, bdg),
                            (outs[0][2], rdb, bdb)):
        within(got, ref, bound, dt)


# --------------------------------------------------------------- embedding
def gradient(tok, dout, V, scale):
    """fp64 sums, the bound of the computed ones and the rows with tokens.  A run of n
    positions is added in chains of at most 512 (a unit), at most n / (512 * 64) + 17 units
    and 64 of their sums one after the other: 700 + n / 2^15 additions at most."""
    inside = (tok >= 0) & (tok < V)
    t, d = tok[inside].long(), dout[inside].double()
    n = torch.bincount(t, minlength=V)
    if V <= 64:  # (index_add_ is slow where a row has millions)
        hot = (t[None] == torch.arange(V, device="cuda")[:, None]).double()
        s, a = hot @ d, hot @ d.abs()
    else:
        s = torch.zeros((V, d.shape[1]), dtype=torch.float64, device="cuda").index_add_(0, t, d)
        a = torch.zeros_like(s).index_add_(0, t, d.abs())
    scale = float(np.float32(scale))
    m = torch.minimum(n, 700 + n / 2 ** 15).double()[:, None]
    return s * scale, (m + 2) * U * a * abs(scale), n > 0


def check_gradient(ctx, dt, tok, V, C, pad=0, start=0, scale=-0.01):
    """Written over sevens, added to, and again: the rows of every token within their
    sums' bounds, every other row +0 (kept to the bit where the call adds), equal bits.
    (Rows of mean 1: a unit that a sum lacks shows.)"""
    T, code = tok.numel(), DTS[dt][0]
    dout = rand((T, C), dt, 322, 1.0, 1.0, pad, start)
    ref, bound, used = gradient(tok, dout, V, scale)
    ints = {"f32": torch.int32}.get(dt, torch.int16)
    outs = []
    for _ in range(2):
        d, untouched = blank((V, C), dt, pad, start)
        ctx.embedding_bwd(tok, T, V, C, dout, ld(dout), d, ld(d), scale=scale, dtype=code)
        torch.cuda.synchronize()
        assert untouched()
        outs.append(d)
    within(outs[0], ref, bound, dt)
    assert (outs[0].contiguous().view(ints)[~used] == 0).all()
    assert torch.equal(outs[0], outs[1])
    d, untouched = blank((V, C), dt, pad, start)
    d.copy_(rand((V, C), dt, 323))
    was = d.clone()
    ctx.embedding_bwd(tok, T, V, C, dout, ld(dout), d, ld(d), scale=scale, accumulate=True,
                      dtype=code)
    torch.cuda.synchronize()
    w = was[used].double()
    within(d[used], w + ref[used], bound[used] + U * (w.abs() + ref[used].abs()), dt)
    assert torch.equal(d[~used], was[~used]) and untouched()


SORTS = [  # T, V, C
    (65536, 1000, 24),              # radix sort: one pass of 10 bits
    (60001, 1500, 33),              # one of 11
    (3600000, 2, 4),                # one of 2, runs of thousands of units
    (12001, (1 << 20) + 5, 8),      # two of 11
    (70000, (1 << 22) + 3, 2),      # three of 8
    (131072, 50, 40), (9000, 1 << 20, 3)]  # workgroups that own tokens: few of them, many


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("kind", ["uniform", "hot", "outside"])
@pytest.mark.parametrize("shape", SORTS, ids=lambda s: "x".join(map(str, s)))
def test_embedding_backward_sorts(gpu_ctx, dt, kind, shape):
    T, V, C = shape
    note("embedding_bwd sort", dt, kind, shape)
    check_gradient(gpu_ctx, dt, tokens_of(kind, T, V, 321), V, C)


# Tables of more than 1.25 times what is zeroed beside the sort (20 MB and 30 for each 8192
# tokens), of fewer than 8 rows a token: the summing launch zeroes the last rows, a few to
# a workgroup, without those of tokens.
ZEROS = [("f32", 5000, 20000, 777, 3, 1), ("bf16", 5001, 20000, 1554, 0, 0),
         ("f16", 8000, 60000, 1025, 1, 0), ("f32", 8000, 60001, 512, 0, 0)]


@pytest.mark.parametrize("last", ["uniform", "frequent", "one", "none"])
@pytest.mark.parametrize("case", ZEROS, ids=lambda s: "x".join(map(str, s)))
def test_embedding_backward_zeroes_beside_the_sums(gpu_ctx, case, last):
    """Tokens in the last rows: some of them, one of them for almost half the batch (more
    positions than a workgroup has threads), only the last row, none at all."""
    dt, T, V, C, pad, start = case
    note("embedding_bwd zeros", case, last)
    tok = tokens_of("uniform", T, V // 16 if last in ("one", "none") else V, 331)
    if last == "frequent":
        tok[torch.rand(T, generator=torch.Generator().manual_seed(332)).cuda() < 0.45] = V - 9
    if last == "one":
        tok[T // 2] = V - 1
    check_gradient(gpu_ctx, dt, tok, V, C, pad, start)


def test_embedding_backward_zeroes_past_32_bits(gpu_ctx):
    """A table of more than 4 GiB, most of it zeroed beside the sums: every row."""
    T, V, C = 9000, 66000, 32768
    note("embedding_bwd zeros past 32 bits")
    tok = tokens_of("uniform", T, V, 341)
    dout = rand((T, C), "bf16", 342)
    d = torch.full((V, C), 7.0, dtype=torch.bfloat16, device="cuda")
    gpu_ctx.embedding_bwd(tok, T, V, C, dout, C, d, C, dtype=2)
    torch.cuda.synchronize()
    for v in range(0, V, 6000):
        mine = (tok >= v) & (tok < v + 6000)
        ref, bound, used = emb_grad(tok[mine] - v, dout[mine], min(6000, V - v), 1.0)
        got = d[v:v + 6000]
        within(got, ref, bound, "bf16")
        assert (got[~used].view(torch.int16) == 0).all()


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("scale", [-0.5, math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("T", [0, 1, 32, 33, 5000])
def test_rows_of_no_token_are_zero_whatever_the_scale(gpu_ctx, dt, scale, T):
    V, C = 700, 53
    note("embedding_bwd scale", dt, scale, T)
    tok = tokens_of("uniform", max(T, 1), V, 351)
    dout = rand((max(T, 1), C), dt, 352)
    d, untouched = blank((V, C), dt, 2)
    gpu_ctx.embedding_bwd(tok, T, V, C, dout, C, d, ld(d), scale=scale, dtype=DTS[dt][0])
    torch.cuda.synchronize()
    used = torch.zeros(V, dtype=torch.bool, device="cuda")
    used[tok[:T].long()] = True
    bits = d.contiguous().view({"f32": torch.int32}.get(dt, torch.int16))
    assert (bits[~used] == 0).all() and untouched()
    if not math.isfinite(scale):
        assert not torch.isfinite(d[used]).any()


# ------------------------------------------------------------------ graphs
def test_captured_gradients_share_the_workspace_with_eager_calls(gpu_ctx):
    """Batches whose sort, partial sums and joins are in the workspace, captured and
    replayed between eager calls of other sizes there: the eager bits every time."""
    import ferrograd_amd as fa

    s = torch.cuda.Stream()
    ctx = fa.Context(0, s.cuda_stream)
    try:
        ctx.reserve_workspace(256 << 20)
        new = lambda *sh: torch.empty(sh, dtype=torch.bfloat16, device="cuda")
        R, C = 5000, 520
        x, dy = rand((R, C), "bf16", 361), rand((R, C), "bf16", 362)
        mean, rstd = torch.zeros(R, device="cuda"), torch.ones(R, device="cuda")
        sizes = [(R, 300, "hot"), (R, 40000, "uniform"), (48000, 1000, "hot")]
        toks = [tokens_of(k, T, V, 363) for T, V, k in sizes]
        douts = [rand((T, C), "bf16", 364) for T, _, _ in sizes]
        tabs = [new(V, C) for _, V, _ in sizes]
        dx, dg, db = new(R, C), new(C), new(C)
        outs = [dx, dg, db] + tabs

        def calls():
            ctx.layer_norm_bwd(x, C, dy, C, mean, rstd, R, C, dx=dx, lddx=C, dgamma=dg, dbeta=db,
                               dtype=2)
            for (T, V, _), tok, dout, tab in zip(sizes, toks, douts, tabs):
                ctx.embedding_bwd(tok, T, V, C, dout, C, tab, C, dtype=2)

        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            calls()
        torch.cuda.synchronize()
        want = [t.clone() for t in outs]
        for (T, V, _), tok, dout, tab in zip(sizes, toks, douts, want[3:]):
            ref, bound, _ = emb_grad(tok, dout, V, 1.0)
            within(tab, ref, bound, "bf16")
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            calls()
        other = rand((6000, 1100), "f32", 365)
        om, orr = torch.zeros(6000, device="cuda"), torch.ones(6000, device="cuda")
        od, ot = torch.empty(1100, device="cuda"), torch.empty((90, 1100), device="cuda")
        otok = tokens_of("uniform", 6000, 90, 366)
        for rep in range(4):
            for t in outs:
                t.fill_(5.0)
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            for t, w in zip(outs, want):
                assert torch.equal(t, w), rep
            with torch.cuda.stream(s):
                ctx.layer_norm_bwd(other, 1100, other, 1100, om, orr, 6000, 1100, dgamma=od)
                ctx.embedding_bwd(otok, 6000, 90, 1100, other, 1100, ot, 1100)
            if rep % 2:
                torch.cuda.synchronize()
    finally:
        ctx.sync()
        ctx.close()
