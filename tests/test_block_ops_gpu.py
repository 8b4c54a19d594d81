"""RMS norm with the residual and token log probabilities against plain fp64 torch,
through the C ABI.

Tolerances are error bounds, elementwise, with the terms of test_token_ops_gpu.py: u =
2^-24, h the storage type's rounding, and N_ROW u for a row's fp32 sums.  A value
computed by k fp32 operations from exact ones is off by k u of the magnitudes that
enter.  An exponential 2^(x c - m), c = scale log2 e, takes an argument whose terms are
each off by at most 2 u of themselves (c, the product, m) and is itself off by 2 u.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from test_token_ops_gpu import DTS, N_ROW, TINY, U, blank, ld, note, place, rand, within  # noqa: E402

EPS = float(np.float32(1e-5))
SIZES = [(1, 1), (3, 7), (5, 8), (2, 31), (33, 100), (7, 512), (4, 1027), (3, 2048), (300, 515),
         (2, 4096), (5, 8200), (3, 16390), (2, 33000), (2, 70001)]


def f64(t):
    return t.double().cpu()


# ------------------------------------------------------------------ RMS norm
def rms_oracle(x, r, gamma, dt):
    s = x if r is None else (x.float() + r.float()).to(DTS[dt][1])
    z = f64(s)
    rstd = 1.0 / torch.sqrt((z * z).mean(1) + EPS)
    y = z * rstd[:, None] * (1.0 if gamma is None else f64(gamma))
    return s, rstd, y


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("R,C", SIZES)
@pytest.mark.parametrize("residual,pad,start", [(True, 0, 0), (False, 3, 1), (True, 5, 3)])
def test_rms_norm(gpu_ctx, dt, R, C, residual, pad, start):
    note("rms_norm", dt, R, C, residual, pad, start)
    code = DTS[dt][0]
    x = rand((R, C), dt, 1, 1.5, 0.3, pad, start)
    r = rand((R, C), dt, 2, 2.0, 0.0, pad + 1, start) if residual else None
    g = rand((1, C), dt, 3, 0.2, 1.0)[0] if start else None
    s, rstd, y = rms_oracle(x, r, g, dt)
    so, s_clean = blank((R, C), dt, pad, 0)
    yo, y_clean = blank((R, C), dt, pad + 2, start)
    ro = torch.empty(R, device="cuda")
    q = torch.full((R, C + pad), 7, dtype=torch.int8, device="cuda")
    e = torch.full((R, (C + 31) // 32 + pad), 7, dtype=torch.uint8, device="cuda")
    gpu_ctx.rms_norm(x, ld(x), R, C, yo, ld(yo), gamma=g, eps=EPS, rstd=ro, q=q, ldq=ld(q), e=e,
                     lde=ld(e), dtype=code,
                     **(dict(r=r, ldr=ld(r), s=so, lds=ld(so)) if residual else {}))
    torch.cuda.synchronize()
    if residual:
        assert torch.equal(so, s) and s_clean()
    # rstd: half the sum's relative error and a few roundings.
    rel = (N_ROW / 2 + 6) * U
    within(ro.cpu(), rstd, rstd * rel)
    within(yo.cpu(), y, y.abs() * (rel + 4 * U), dt)
    assert y_clean()
    # 8 bits: within half a step of y (a whole one where clamped), by a step that the
    # block's largest value asks for.
    nb = (C + 31) // 32
    b = e[:, :nb].cpu().double()
    pad_y = torch.nn.functional.pad(y, (0, nb * 32 - C)).reshape(R, nb, 32)
    top = pad_y.abs().amax(2)
    err = rel + 4 * U
    assert bool((top * (1 + err) >= torch.exp2(b - 127)).logical_or(b == 1).all())
    assert bool((top * (1 - err) < torch.exp2(b - 126)).all())
    step = torch.exp2(b - 133).repeat_interleave(32, 1)[:, :C]
    k = q[:, :C].cpu().double()
    half = torch.where(k.abs() == 127, 1.0, 0.5)
    within(k * step, y, step * half + y.abs() * err)
    assert bool((q[:, C:] == 7).all()) and bool((e[:, nb:] == 7).all())


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("R,C", [(5, 517), (3, 4103), (2, 33003), (2, 8193), (2, 65537)])
def test_rms_norm_in_place(gpu_ctx, dt, R, C):
    """s over r and y over x: a residual stream kept in one buffer."""
    code = DTS[dt][0]
    x, r = rand((R, C), dt, 4), rand((R, C), dt, 5, 3.0)
    s, _, y = rms_oracle(x, r, None, dt)
    gpu_ctx.rms_norm(x, ld(x), R, C, x, ld(x), r=r, ldr=ld(r), s=r, lds=ld(r), eps=EPS, dtype=code)
    torch.cuda.synchronize()
    assert torch.equal(r, s)
    within(x.cpu(), y, y.abs() * (N_ROW / 2 + 10) * U, dt)
    dy, rstd = rand((R, C), dt, 6), 1.0 / torch.sqrt(r.float().square().mean(1) + EPS)
    dx, dg = rms_bwd_oracle(r, dy, None, rstd, dy, dt)
    out, got = torch.empty(C, dtype=DTS[dt][1], device="cuda"), dy
    gpu_ctx.rms_norm_bwd(r, ld(r), dy, ld(dy), rstd, R, C, ds=dy, ldds=ld(dy), dx=dy, lddx=ld(dy),
                         dgamma=out, dtype=code)
    within(got.cpu(), *dx, dt)
    within(out.cpu(), *dg, dt)


def rms_bwd_oracle(s, dy, gamma, rstd, ds, dt):
    """(dx, its bound), (dgamma, its bound)."""
    s, d, k = f64(s), f64(dy), f64(rstd)[:, None]
    g = d * (1.0 if gamma is None else f64(gamma))
    R, C = s.shape
    xh = s * k
    m, mabs = (g * xh).mean(1, keepdim=True), (g * xh).abs().mean(1, keepdim=True)
    e = 0.0 if ds is None else f64(ds)
    dx = k * (g - xh * m) + e
    mag = k * (g.abs() + xh.abs() * mabs)
    bound = U * (8 * mag + k * xh.abs() * mabs * N_ROW + 2 * dx.abs())
    dg = (d * xh).sum(0)
    return (dx, bound), (dg, U * (R + 8) * (d * xh).abs().sum(0))


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("R,C", SIZES + [(700, 129), (2000, 70)])
@pytest.mark.parametrize("residual,pad,start", [(True, 0, 0), (False, 3, 1)])
def test_rms_norm_bwd(gpu_ctx, dt, R, C, residual, pad, start):
    note("rms_norm_bwd", dt, R, C, residual, pad, start)
    code = DTS[dt][0]
    s, dy = rand((R, C), dt, 7, 1.0, 0.2, pad, start), rand((R, C), dt, 8, 1.0, 0.0, pad + 1)
    ds = rand((R, C), dt, 9, 1.0, 0.0, pad, start) if residual else None
    g = rand((1, C), dt, 10, 0.2, 1.0)[0] if not start else None
    rstd = 1.0 / torch.sqrt(s.float().square().mean(1) + EPS)
    (dx, bx), (dg, bg) = rms_bwd_oracle(s, dy, g, rstd, ds, dt)
    out, clean = blank((R, C), dt, pad, start)
    for accumulate in (False, True):
        dgo = rand((1, C), dt, 11)[0]
        old = f64(dgo)
        gpu_ctx.rms_norm_bwd(s, ld(s), dy, ld(dy), rstd, R, C, gamma=g, ds=ds,
                             ldds=ld(ds) if residual else 0, dx=out, lddx=ld(out), dgamma=dgo,
                             dgamma_accumulate=accumulate, dtype=code)
        torch.cuda.synchronize()
        within(out.cpu(), dx, bx, dt)
        want = dg + old if accumulate else dg
        within(dgo.cpu(), want, bg + 2 * U * want.abs(), dt)
    assert clean()
    # Either output alone, the same bits.
    alone, dga = torch.empty_like(out), torch.empty_like(dgo)
    more = dict(ds=ds, ldds=ld(ds)) if residual else {}
    gpu_ctx.rms_norm_bwd(s, ld(s), dy, ld(dy), rstd, R, C, gamma=g, dx=alone, lddx=ld(alone),
                         dtype=code, **more)
    gpu_ctx.rms_norm_bwd(s, ld(s), dy, ld(dy), rstd, R, C, gamma=g, dgamma=dga, dtype=code)
    within(dga.cpu(), dg, bg, dt)
    assert torch.equal(alone, out)


def test_rms_norm_bwd_of_no_rows(gpu_ctx):
    """dgamma is written (or left), nothing is read."""
    for C in (40, 33000):
        dg = rand((1, C), "f32", 15)[0]
        was = dg.clone()
        any_ = torch.full((8,), math.nan, device="cuda")
        gpu_ctx.rms_norm_bwd(any_, C, any_, C, any_, 0, C, dgamma=dg, dgamma_accumulate=True)
        assert torch.equal(dg, was)
        gpu_ctx.rms_norm_bwd(any_, C, any_, C, any_, 0, C, dgamma=dg)
        assert bool((dg == 0).all())


def test_rms_norm_gradient_by_differences(gpu_ctx):
    """dx and dgamma against central differences of the forward itself, in fp32: the
    quotient's error is the rounding of y over the step and the third derivative."""
    R, C, h = 3, 40, 2.0 ** -6
    x, w = rand((R, C), "f32", 12), rand((R, C), "f32", 13)
    g = rand((1, C), "f32", 14, 0.2, 1.0)[0]
    y, rstd = torch.empty_like(x), torch.empty(R, device="cuda")

    def objective(x, g):
        gpu_ctx.rms_norm(x, C, R, C, y, C, gamma=g, eps=EPS, rstd=rstd)
        return (y.double() * w.double()).sum().item()

    objective(x, g)
    dx, dg = torch.empty_like(x), torch.empty_like(g)
    gpu_ctx.rms_norm_bwd(x, C, w, C, rstd, R, C, gamma=g, dx=dx, lddx=C, dgamma=dg)
    for t, d in ((x, dx), (g, dg)):
        for i in (0, 17, t.numel() - 1):
            was = t.view(-1)[i].item()
            t.view(-1)[i] = was + h
            up = objective(x, g)
            t.view(-1)[i] = was - h
            down = objective(x, g)
            t.view(-1)[i] = was
            # y is off by at most 40 u |y| each; f''' h^2 / 6 of values of order one.
            tol = 40 * U * (y.double() * w.double()).abs().sum().item() / h + 4 * h * h
            assert abs((up - down) / (2 * h) - d.view(-1)[i].item()) <= tol


# ------------------------------------------------------------ log probabilities
LP_SIZES = [(1, 1), (3, 5), (4, 33), (65, 64), (2, 700), (33, 1000), (2, 2049), (3, 32003),
            (1, 131072), (2, 200001)]


def lp_oracle(x, tok, scale):
    """(logp, entropy, lse) and the bound of each; a row of -inf where masked."""
    z = f64(x) * scale
    m = z.amax(1, keepdim=True)
    d = z - m
    e = torch.exp(d)
    s = e.sum(1)
    p = e / s[:, None]
    pd = torch.where(p > 0, p * d, 0.0)
    C = z.shape[1]
    ok = tok < C
    zt = z.gather(1, tok.clamp(max=C - 1)[:, None])[:, 0]
    lse = m[:, 0] + torch.log(s)
    logp = torch.where(ok, zt - lse, math.nan)
    h = torch.log(s) - pd.sum(1)
    big = torch.where(z > -math.inf, z, 0.0).abs().amax(1)
    arg = U * (6 * big + N_ROW + 10)  # of any exponential's argument, and of the sums
    spread = 1.0 - pd.sum(1)
    return ((logp, arg + U * (4 * logp.abs() + 8)), (h, arg * (2 * spread + 5)),
            (lse, arg + 4 * U * lse.abs()))


def tops_oracle(x, k):
    """Columns of the k largest, the lowest column first, NaN last."""
    v = f64(x).numpy() + 0.0
    v = np.where(np.isnan(v), -np.inf, v)  # (tests with NaN hold no -inf)
    return torch.from_numpy(np.argsort(-v, axis=1, kind="stable")[:, :k].copy())


def run_lp(ctx, x, tok, dt, top, scale):
    R, C = x.shape
    o = [torch.full((R,), 7.0, device="cuda") for _ in range(3)]
    ids = torch.full((R, max(top, 1)), 7, dtype=torch.int32, device="cuda")
    tops = torch.full((R, max(top, 1)), 7.0, device="cuda")
    ctx.token_logprobs(x, ld(x), tok.int().cuda(), R, C, logp=o[0], entropy=o[1], lse=o[2], top=top,
                       top_ids=ids if top else None, top_logp=tops if top else None, scale=scale,
                       dtype=DTS[dt][0])
    torch.cuda.synchronize()
    return o, ids.cpu(), tops.cpu()


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("R,C", LP_SIZES)
@pytest.mark.parametrize("scale,pad,start", [(1.0, 0, 0), (0.7, 3, 1)])
def test_logprobs(gpu_ctx, dt, R, C, scale, pad, start):
    note("token_logprobs", dt, R, C, scale, pad, start)
    scale = float(np.float32(scale))
    x = rand((R, C), dt, 20, 3.0, 1.0, pad, start)
    tok = torch.randint(0, C, (R,), generator=torch.Generator().manual_seed(21))
    top = min(C, 20 if start else 32)
    want = lp_oracle(x, tok, scale)
    got, ids, tops = run_lp(gpu_ctx, x, tok, dt, top, scale)
    for g, (w, b) in zip(got, want):
        within(g.cpu(), w, b)
    best = tops_oracle(x, top)
    assert torch.equal(ids.long(), best)
    (lse, b) = want[2]
    tl = f64(x).gather(1, best) * scale - lse[:, None]
    within(tops, tl, b[:, None] + U * (4 * tl.abs() + 8))


@pytest.mark.parametrize("C", [3001, 40003])
def test_logprobs_masked_ties_and_nan(gpu_ctx, C):
    """Masked logits (-inf, or the type's lowest number), rows of one value, tokens
    outside the vocabulary, NaN in one row alone."""
    for dt in ("bf16", "f32"):
        x = rand((8, C), dt, 22, 2.0)
        low = torch.finfo(DTS[dt][1]).min
        x[0, 5:] = -math.inf                       # five left
        x[1, ::2] = low
        x[2] = 0.25                                # every one an alternative
        x[3] = torch.where(x[3] > 0, 1.0, 0.0)     # two values
        x[4, 1:] = -math.inf                       # one left: certain
        x[5, C - 1] = 80.0
        x[6, :] = -math.inf
        x[6, C - 2:] = 0.0                          # the two past the last chunk's boundary
        tok = torch.tensor([3, 1, C - 1, 7, 0, C - 1, C - 1, C])
        want = lp_oracle(x, tok, 1.0)
        got, ids, tops = run_lp(gpu_ctx, x, tok, dt, 32, 1.0)
        for g, (w, b) in zip(got, want):
            g, w, b = g.cpu(), w, b
            assert torch.equal(torch.isnan(g), torch.isnan(w))
            within(g[~torch.isnan(w)], w[~torch.isnan(w)], b[~torch.isnan(w)])
        assert torch.equal(ids.long(), tops_oracle(x, 32))
        assert torch.isinf(tops[0, 5:]).all() and torch.isnan(got[0][7].cpu())
        y = x.clone()
        y[0], y[6], y[4] = 1.0, 2.0, 3.0
        y[3, 17] = math.nan
        got, ids, _ = run_lp(gpu_ctx, y, tok, dt, 5, 1.0)
        assert torch.isnan(got[2]).nonzero().flatten().tolist() == [3]
        assert torch.equal(ids.long(), tops_oracle(y, 5))
        y[:, :] = math.nan                         # alternatives by column alone
        _, ids, _ = run_lp(gpu_ctx, y, tok, dt, 5, 1.0)
        assert torch.equal(ids.long(), torch.arange(5).expand(8, 5))


def lp_bwd_oracle(x, tok, scale, lse, h, a, b):
    z = f64(x) * scale
    C = z.shape[1]
    lse, h, a, b = (f64(t)[:, None] for t in (lse, h, a, b))
    d = z - lse
    p = torch.exp(d)
    pd = torch.where(p > 0, p * (d + h), 0.0)
    hot = torch.nn.functional.one_hot(tok.clamp(max=C), C + 1)[:, :C].double()
    out = scale * (a * (hot - p) - b * pd)
    big = torch.where(z > -math.inf, z, 0.0).abs()
    rel = U * (8 * (big + lse.abs()) + 16)
    inner = torch.where(p > 0, p * (d.abs() + h.abs() + lse.abs() + big), 0.0)
    bound = scale * (a.abs() * (p * rel + 4 * U * hot) + b.abs() * (pd.abs() * rel + 8 * U * inner))
    return out, bound + 2 * U * out.abs()


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("R,C", LP_SIZES)
@pytest.mark.parametrize("scale,pad,start", [(1.0, 0, 0), (0.7, 3, 1)])
def test_logprobs_bwd(gpu_ctx, dt, R, C, scale, pad, start):
    note("token_logprobs_bwd", dt, R, C, scale, pad, start)
    scale = float(np.float32(scale))
    x = rand((R, C), dt, 23, 2.0, 0.5, pad, start)
    if C > 40:
        x[0, 3:30] = -math.inf
    gen = torch.Generator().manual_seed(24)
    tok = torch.randint(0, C, (R,), generator=gen)
    tok[R // 2] = C  # no column
    (_, _), (h, _), (lse, _) = lp_oracle(x, tok, scale)
    h, lse = h.float().cuda(), lse.float().cuda()
    a, b = torch.randn(R, generator=gen).cuda(), torch.randn(R, generator=gen).cuda()
    a[-1] = b[-1] = 0.0
    zero = torch.zeros_like(a)
    for ga, gb in ((a, b), (a, None), (None, b)):
        want, bound = lp_bwd_oracle(x, tok, scale, lse, h, zero if ga is None else ga,
                                    zero if gb is None else gb)
        out, clean = blank((R, C), dt, pad + 1, start)
        gpu_ctx.token_logprobs_bwd(x, ld(x), tok.int().cuda(), R, C, lse, out, ld(out), entropy=h,
                                   dlogp=ga, dentropy=gb, scale=scale, dtype=DTS[dt][0])
        torch.cuda.synchronize()
        within(out.cpu(), want, bound, dt)
        assert clean()
    assert bool((out[-1] == 0).all())
    same = place(x, pad, start)  # over the logits, the same bits
    gpu_ctx.token_logprobs_bwd(same, ld(same), tok.int().cuda(), R, C, lse, same, ld(same),
                               entropy=h, dentropy=b, scale=scale, dtype=DTS[dt][0])
    assert torch.equal(same, out)


def test_logprobs_padding_rows_are_not_read(gpu_ctx):
    """Rows without a gradient are zeros, NaN or not."""
    x = rand((4, 1001), "bf16", 25)
    x[1] = math.nan
    tok = torch.zeros(4, dtype=torch.int32, device="cuda")
    (_, _), (h, _), (lse, _) = lp_oracle(x, tok.long().cpu(), 1.0)
    a = torch.tensor([1.0, 0.0, -1.0, 0.0], device="cuda")
    out = torch.full_like(x, 7.0)
    gpu_ctx.token_logprobs_bwd(x, ld(x), tok, 4, 1001, lse.float().cuda(), out, ld(out), dlogp=a,
                               dtype=DTS["bf16"][0])
    assert bool((out[1] == 0).all()) and bool((out[3] == 0).all())
    assert bool(torch.isfinite(out[0].float()).all()) and bool((out[0] != 0).any())


def test_logprobs_gradient_by_differences(gpu_ctx):
    """a logp + b entropy against central differences of the forward, in fp32."""
    R, C, h = 2, 50, 2.0 ** -5
    x = rand((R, C), "f32", 26, 1.0)
    tok = torch.tensor([3, 49], dtype=torch.int32, device="cuda")
    a, b = torch.tensor([1.0, -0.5], device="cuda"), torch.tensor([0.25, 2.0], device="cuda")
    lp, en, lse = (torch.empty(R, device="cuda") for _ in range(3))

    def objective():
        gpu_ctx.token_logprobs(x, C, tok, R, C, logp=lp, entropy=en, lse=lse)
        return (a.double() * lp.double() + b.double() * en.double()).sum().item()

    objective()
    dx = torch.empty_like(x)
    gpu_ctx.token_logprobs_bwd(x, C, tok, R, C, lse, dx, C, entropy=en, dlogp=a, dentropy=b)
    grad = dx.clone()
    for i in (0, 3, 30, 2 * C - 1):
        was = x.view(-1)[i].item()
        x.view(-1)[i] = was + h
        up = objective()
        x.view(-1)[i] = was - h
        down = objective()
        x.view(-1)[i] = was
        # Each answer is off by less than 300 u; f''' h^2 / 6 of values of order one.
        assert abs((up - down) / (2 * h) - grad.view(-1)[i].item()) <= 4 * 300 * U / h + 2 * h * h
