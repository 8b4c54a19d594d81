"""Layer norm, embedding and 8-bit activation checkpoints against plain fp64
torch, through the C ABI.

Tolerances are error bounds, elementwise.  u = 2^-24 is fp32's rounding, h the
storage type's (2^-24, 2^-11, 2^-8).  A sum of n fp32 terms taken as chains of
at most m terms joined by a tree of at most 10 levels is off by at most
(m + 10) u times the sum of magnitudes; a row of up to 2^17 columns is summed
in chains of at most 128 (1024 threads; longer rows by chunks of at most 8, whose
sums' chains are shorter), so rows count N_ROW u.  Sums over rows
or tokens use the bound of any order, their count.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

U = 2.0 ** -24
N_ROW = 128 + 10 + 6
DTS = {"f32": (0, torch.float32, U), "f16": (1, torch.float16, 2.0 ** -11),
       "bf16": (2, torch.bfloat16, 2.0 ** -8)}
# Below these a type's step no longer shrinks with the value.
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -24, "bf16": 2.0 ** -133}
ACTS = {"none": 0, "relu": 1, "gelu": 2}
C0, C1 = float(np.float32(0.7978846)), float(np.float32(0.044715))


def note(*a):
    print(*a, flush=True)


def rand(shape, dt, seed, std=1.0, mean=0.0, pad=0, start=0):
    """A view of `shape` whose rows lie pad elements further apart and whose
    first element is `start` elements into its allocation."""
    g = torch.Generator().manual_seed(seed)
    R, C = shape
    x = (torch.randn(R, C, generator=g) * std + mean).to(DTS[dt][1])
    return place(x, pad, start)


def place(x, pad=0, start=0, fill=0.0):
    R, C = x.shape
    buf = torch.full((R * (C + pad) + start,), fill, dtype=x.dtype, device="cuda")
    v = buf[start:].view(R, C + pad)[:, :C]
    v.copy_(x)
    return v


def blank(shape, dt, pad=0, start=0):
    """An output view in a buffer of sevens, and the check that nothing else
    of the buffer was written."""
    R, C = shape
    buf = torch.full((R * (C + pad) + start + 16,), 7.0, dtype=DTS[dt][1], device="cuda")
    v = buf[start:start + R * (C + pad)].view(R, C + pad)[:, :C]

    def untouched():
        k = torch.ones_like(buf, dtype=torch.bool)
        k[start:start + R * (C + pad)].view(R, C + pad)[:, :C] = False
        return bool((buf[k] == 7.0).all())
    return v, untouched


def ld(t):
    return t.stride(0)


def within(got, ref, bound, dt=None):
    """|got - ref| <= bound (+ the rounding of the result to dt)."""
    ref = ref.double()
    if dt is not None:
        bound = bound + DTS[dt][2] * (ref.abs() + bound) + TINY[dt]
    bad = ~((got.double() - ref).abs() <= bound)
    if bad.any():
        i = bad.nonzero()[0].tolist()
        i = tuple(i)
        pytest.fail(f"{int(bad.sum())} of {bad.numel()} off, first at {i}: got "
                    f"{got[i].item()!r}, want {ref[i].item()!r}, bound "
                    f"{bound[i].item() if bound.dim() else bound.item()!r}")


# -------------------------------------------------------------- layer norm
LN_SHAPES = [  # R, C, pad, start
    (1, 1, 0, 0), (3, 2, 0, 1), (1, 7, 0, 0), (5, 33, 2, 0), (4, 64, 0, 0), (17, 255, 1, 3),
    (64, 256, 0, 0), (9, 777, 0, 0), (33, 1000, 8, 0), (130, 1531, 3, 1), (2, 2048, 0, 0),
    (257, 2048, 0, 0), (7, 4096, 0, 8), (12, 4100, 4, 0), (5, 8192, 0, 0), (3, 8200, 0, 2),
    (3, 16384, 0, 0), (2, 20001, 0, 0), (2, 32768, 0, 0), (2, 65537, 0, 1), (1, 131072, 0, 0),
    (300, 40000, 0, 0), (1, 140000, 0, 1)]


def ln_reference(x, gamma, beta, eps):
    x = x.double()
    mean = x.mean(1)
    xc = x - mean[:, None]
    rstd = 1.0 / torch.sqrt((xc * xc).mean(1) + eps)
    xh = xc * rstd[:, None]
    g = gamma.double() if gamma is not None else torch.ones_like(x[0])
    b = beta.double() if beta is not None else torch.zeros_like(x[0])
    return mean, rstd, xh, xh * g + b, g, b


def ln_bounds(x, mean, rstd, xh, g, b):
    """Bounds of the computed mean, rstd and y (before y's rounding): the mean's
    own error shifts x - mean, the variance's relative error is twice the
    row sums' (a shifted mean adds only its square)."""
    xa = x.double().abs().mean(1)
    d_mean = N_ROW * U * xa + U * mean.abs()
    r_rstd = (N_ROW + 4) * U + (d_mean * rstd) ** 2
    dx = d_mean * rstd
    y = g.abs() * (dx[:, None] + xh.abs() * (r_rstd[:, None] + 4 * U)) + 2 * U * b.abs()
    return d_mean, r_rstd * rstd, y


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("shape", LN_SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_layer_norm_forward(gpu_ctx, dt, shape):
    R, C, pad, start = shape
    note("layer_norm", dt, shape)
    code = DTS[dt][0]
    x = rand((R, C), dt, 1, 1.0, 0.5, pad, start)
    gamma = rand((1, C), dt, 2, 0.2, 1.0)[0]
    beta = rand((1, C), dt, 3, 0.3)[0]
    for affine in (True, False):
        y, untouched = blank((R, C), dt, pad, start)
        mean, rstd = (torch.full((R,), -1.0, device="cuda") for _ in range(2))
        gm, bt = (gamma, beta) if affine else (None, None)
        gpu_ctx.layer_norm(x, ld(x), R, C, y, ld(y), gamma=gm, beta=bt, eps=1e-5, mean=mean,
                           rstd=rstd, dtype=code)
        torch.cuda.synchronize()
        m, r, xh, yr, g, b = ln_reference(x, gm, bt, float(np.float32(1e-5)))
        dm, dr, dy = ln_bounds(x, m, r, xh, g, b)
        within(mean, m, dm)
        within(rstd, r, dr)
        within(y, yr, dy, dt)
        assert untouched()


def test_layer_norm_in_place_without_statistics_and_no_rows(gpu_ctx):
    for dt in DTS:
        x = rand((37, 1001), dt, 5, 2.0, -1.0, 3, 1)
        y = torch.empty_like(x)
        gpu_ctx.layer_norm(x, ld(x), 37, 1001, y, ld(y), dtype=DTS[dt][0])
        gpu_ctx.layer_norm(x, ld(x), 37, 1001, x, ld(x), dtype=DTS[dt][0])
        gpu_ctx.layer_norm(x, ld(x), 0, 1001, x, ld(x), dtype=DTS[dt][0])
        torch.cuda.synchronize()
        assert torch.equal(x, y)


@pytest.mark.parametrize("C", [96, 1531, 40000])
def test_layer_norm_rows_are_independent(gpu_ctx, C):
    """A row of NaN or infinity leaves the other rows as they are; a constant
    row gives beta (its variance is 0)."""
    x = rand((6, C), "f32", 7)
    x[3] = 1e10  # a mean that the sum rounds; x - mean is then not exactly 0
    x[5] = 2.0
    beta = rand((1, C), "f32", 8)[0]
    y0, y1 = torch.empty_like(x), torch.empty_like(x)
    gpu_ctx.layer_norm(x, C, 6, C, y0, C, beta=beta)
    z = x.clone()
    z[1, C // 2] = float("nan")
    z[2, 0] = float("inf")
    gpu_ctx.layer_norm(z, C, 6, C, y1, C, beta=beta)
    torch.cuda.synchronize()
    assert torch.isnan(y1[1]).all() and torch.isnan(y1[2]).all()
    for r in (0, 3, 4, 5):
        assert torch.equal(y0[r], y1[r])
    assert torch.isfinite(y0).all()
    # Sums of 2.0 are exact below 2^24 terms.
    assert torch.equal(y0[5], beta)


def test_layer_norm_keeps_digits_far_from_zero(gpu_ctx):
    """A row of mean 1000 and deviation 1/16: the variance comes from x - mean,
    not from a difference of squares (which would lose it in fp32)."""
    for C in (512, 8192, 50000):
        x = rand((4, C), "f32", 11, 2.0 ** -4, 1000.0)
        rstd = torch.empty(4, device="cuda")
        y = torch.empty_like(x)
        gpu_ctx.layer_norm(x, C, 4, C, y, C, rstd=rstd)
        torch.cuda.synchronize()
        m, r, xh, yr, g, b = ln_reference(x, None, None, float(np.float32(1e-5)))
        _, dr, dy = ln_bounds(x, m, r, xh, g, b)
        within(rstd, r, dr)
        within(y, yr, dy)


def ln_bwd_reference(x, dy, gamma, mean, rstd):
    x, dy, rs = x.double(), dy.double(), rstd.double()[:, None]
    xh = (x - mean.double()[:, None]) * rs
    g = dy * gamma.double() if gamma is not None else dy
    m1, m2 = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
    dx = rs * (g - m1 - xh * m2)
    # The row sums' errors, and the few operations after them.
    b = rs * (N_ROW * U * (g.abs().mean(1, keepdim=True) +
                           xh.abs() * (g * xh).abs().mean(1, keepdim=True)) +
              8 * U * (g.abs() + m1.abs() + (xh * m2).abs()))
    n = x.shape[0] + 8  # any order of the rows
    return dx, b, (dy * xh).sum(0), n * U * (dy * xh).abs().sum(0), dy.sum(0), n * U * dy.abs().sum(0)


LN_BWD_SHAPES = LN_SHAPES + [(300, 1, 0, 0), (1031, 72, 0, 0), (2048, 520, 0, 0),
                             (4099, 131, 5, 0), (515, 4096, 0, 0), (600, 9000, 0, 0),
                             (129, 1000, 0, 0), (256, 4100, 4, 1), (257, 6001, 1, 0),
                             (300, 16384, 0, 0), (1100, 17001, 0, 0), (600, 2048, 0, 0),
                             (640, 777, 3, 1), (641, 300, 0, 0), (257, 24, 0, 0)]


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("shape", LN_BWD_SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_layer_norm_backward(gpu_ctx, dt, shape):
    R, C, pad, start = shape
    note("layer_norm_bwd", dt, shape)
    code = DTS[dt][0]
    x = rand((R, C), dt, 21, 1.0, 0.5, pad, start)
    dy = rand((R, C), dt, 22, 1.0, 0.1, pad, start)
    gamma = rand((1, C), dt, 23, 0.2, 1.0)[0]
    xd = x.double()
    mean = xd.mean(1).float()
    rstd = (1.0 / torch.sqrt(((xd - mean.double()[:, None]) ** 2).mean(1) + 1e-5)).float()
    dx, untouched = blank((R, C), dt, pad, start)
    dg, ug = blank((1, C), dt)
    db, ub = blank((1, C), dt)
    gpu_ctx.layer_norm_bwd(x, ld(x), dy, ld(dy), mean, rstd, R, C, gamma=gamma, dx=dx, lddx=ld(dx),
                           dgamma=dg, dbeta=db, dtype=code)
    torch.cuda.synchronize()
    rdx, bdx, rdg, bdg, rdb, bdb = ln_bwd_reference(x, dy, gamma, mean, rstd)
    within(dx, rdx, bdx, dt)
    within(dg[0], rdg, bdg, dt)
    within(db[0], rdb, bdb, dt)
    assert untouched() and ug() and ub()
    # Without gamma; each output alone; then all of them added to.
    rdx, bdx, _, _, _, _ = ln_bwd_reference(x, dy, None, mean, rstd)
    d2, g2, b2 = torch.empty_like(dx), torch.empty_like(dg), torch.empty_like(db)
    args = (x, ld(x), dy, ld(dy), mean, rstd, R, C)
    gpu_ctx.layer_norm_bwd(*args, dx=d2, lddx=ld(d2), dtype=code)
    gpu_ctx.layer_norm_bwd(*args, dgamma=g2, dtype=code)
    gpu_ctx.layer_norm_bwd(*args, dbeta=b2, dtype=code)
    torch.cuda.synchronize()
    within(d2, rdx, bdx, dt)
    within(g2[0], rdg, bdg, dt)
    within(b2[0], rdb, bdb, dt)
    d3, g3, b3 = d2.clone(), g2.clone(), b2.clone()
    gpu_ctx.layer_norm_bwd(*args, dx=d3, lddx=ld(d3), dgamma=g3, dbeta=b3, accumulate=True,
                           dgamma_accumulate=True, dbeta_accumulate=True, dtype=code)
    torch.cuda.synchronize()
    for got, was, ref, bound in ((d3, d2, rdx, bdx), (g3[0], g2[0], rdg, bdg),
                                 (b3[0], b2[0], rdb, bdb)):
        within(got, was.double() + ref, bound + U * (was.double().abs() + ref.abs()), dt)


def test_layer_norm_backward_in_place_and_no_rows(gpu_ctx):
    for dt, C in (("bf16", 1024), ("f32", 999), ("f16", 30000)):
        code = DTS[dt][0]
        x, dy = rand((21, C), dt, 31), rand((21, C), dt, 32)
        mean, rstd = torch.zeros(21, device="cuda"), torch.ones(21, device="cuda")
        outs = []
        for where in ("own", "dy", "x"):
            a, b = x.clone(), dy.clone()
            dx = {"own": torch.empty_like(x), "dy": b, "x": a}[where]
            dg, db = (torch.empty(C, dtype=x.dtype, device="cuda") for _ in range(2))
            gpu_ctx.layer_norm_bwd(a, C, b, C, mean, rstd, 21, C, dx=dx, lddx=C, dgamma=dg,
                                   dbeta=db, dtype=code)
            torch.cuda.synchronize()
            outs.append((dx, dg, db))
        for o in outs[1:]:
            assert all(torch.equal(p, q) for p, q in zip(outs[0], o))
        dg.fill_(3.0)
        db.fill_(4.0)
        gpu_ctx.layer_norm_bwd(x, C, dy, C, mean, rstd, 0, C, dx=x, lddx=C, dgamma=dg, dbeta=db,
                               dgamma_accumulate=True, dtype=code)
        torch.cuda.synchronize()
        assert (dg == 3.0).all() and (db == 0.0).all()


def test_layer_norm_gradients_against_differences(gpu_ctx):
    """Central differences of sum(w * y) in fp64 at the operator's own inputs."""
    R, C = 5, 40
    x, w = rand((R, C), "f32", 41), rand((R, C), "f32", 42)
    gamma, beta = rand((1, C), "f32", 43, 0.2, 1.0)[0], rand((1, C), "f32", 44)[0]
    y, dx = torch.empty_like(x), torch.empty_like(x)
    mean, rstd = (torch.empty(R, device="cuda") for _ in range(2))
    dg, db = torch.empty_like(gamma), torch.empty_like(beta)
    gpu_ctx.layer_norm(x, C, R, C, y, C, gamma=gamma, beta=beta, mean=mean, rstd=rstd)
    gpu_ctx.layer_norm_bwd(x, C, w, C, mean, rstd, R, C, gamma=gamma, dx=dx, lddx=C, dgamma=dg,
                           dbeta=db)
    torch.cuda.synchronize()
    f = lambda x_, g_, b_: float((w.double() * ln_reference(x_, g_, b_, float(np.float32(1e-5)))[3]).sum())
    h = 2.0 ** -12
    for t, grad, at in ((x, dx, (3, 7)), (x, dx, (0, 39)), (gamma, dg, (11,)), (beta, db, (0,))):
        v = []
        for s in (h, -h):
            p = t.double().clone()
            p[at] += s
            v.append(f(*[p if q is t else q for q in (x, gamma, beta)]))
        # The differences' own error is about h^2 (6e-8) times third derivatives.
        assert abs((v[0] - v[1]) / (2 * h) - grad[at].item()) < 1e-4


# --------------------------------------------------------------- embedding
def tokens_of(kind, T, V, seed):
    g = torch.Generator().manual_seed(seed)
    if kind == "same":
        t = torch.full((T,), V - 1)
    elif kind == "hot":
        t = torch.randint(0, V, (T,), generator=g)
        t[torch.rand(T, generator=g) < 0.5] = V // 2
    elif kind == "sorted":
        t = torch.randint(0, V, (T,), generator=g).sort()[0]
    elif kind == "outside":
        t = torch.randint(0, 2 * V, (T,), generator=g)
        t[::5] = -1  # 2^32 - 1 as u32
    else:
        t = torch.randint(0, V, (T,), generator=g)
    return t.to(torch.int32).cuda()


EMB_SHAPES = [  # T, V, C, pad, start
    (1, 1, 1, 0, 0), (1, 5, 16, 0, 0), (7, 3, 33, 1, 1), (64, 10, 256, 0, 0), (64, 1000, 100, 4, 2),
    (255, 50, 777, 0, 0), (256, 4096, 64, 0, 0), (1000, 17, 1024, 0, 0), (1024, 70000, 8, 0, 0),
    (3001, 1009, 130, 3, 0), (4096, 64, 512, 8, 0), (4097, 300, 2051, 0, 1), (9000, 32000, 96, 0, 0),
    (20011, 257, 48, 0, 0), (40000, 5000, 24, 0, 0), (70000, 131072, 16, 0, 0),
    (131072, 3, 40, 0, 0), (300, 9, 8192, 0, 0), (50, 9, 20000, 0, 0), (257, 1, 24, 0, 0),
    (2000, 255, 16, 0, 0), (2000, 256, 16, 0, 0), (3000, 262144, 8, 0, 0),
    (32, 40, 72, 0, 0), (33, 40, 1100, 2, 1), (1025, 77, 600, 0, 0), (4096, 1000, 120, 1, 1)]


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("shape", EMB_SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_embedding_forward_is_one_rounded_product(gpu_ctx, dt, shape):
    T, V, C, pad, start = shape
    note("embedding", dt, shape)
    code, ty, _ = DTS[dt]
    table = rand((V, C), dt, 51, 0.02, 0.0, pad, start)
    for kind, scale in (("uniform", 1.0), ("outside", math.sqrt(C))):
        tok = tokens_of(kind, T, V, 52)
        out, untouched = blank((T, C), dt, pad, start)
        gpu_ctx.embedding(tok, T, V, C, table, ld(table), out, ld(out), scale=scale, dtype=code)
        torch.cuda.synchronize()
        inside = (tok >= 0) & (tok < V)
        ref = (table[tok.clamp(0, V - 1).long()].float() * float(np.float32(scale))).to(ty)
        assert torch.equal(out[inside], ref[inside])
        assert torch.isnan(out[~inside]).all()
        assert untouched()


def emb_grad(tok, dout, V, scale):
    inside = (tok >= 0) & (tok < V)
    s = torch.zeros((V, dout.shape[1]), dtype=torch.float64, device="cuda")
    a = torch.zeros_like(s)
    d = dout[inside].double()
    s.index_add_(0, tok[inside].long(), d)
    a.index_add_(0, tok[inside].long(), d.abs())
    n = torch.bincount(tok[inside].long(), minlength=V).double()[:, None]
    scale = float(np.float32(scale))
    return s * scale, (n + 2) * U * a * abs(scale), n[:, 0] > 0


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("kind", ["uniform", "hot", "same", "sorted", "outside"])
@pytest.mark.parametrize("shape", EMB_SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_embedding_backward(gpu_ctx, dt, kind, shape):
    T, V, C, pad, start = shape
    note("embedding_bwd", dt, kind, shape)
    code = DTS[dt][0]
    tok = tokens_of(kind, T, V, 61)
    dout = rand((T, C), dt, 62, 1.0, 0.0, pad, start)
    scale = 0.37
    ref, bound, used = emb_grad(tok, dout, V, scale)
    dt1, untouched = blank((V, C), dt, pad, start)
    gpu_ctx.embedding_bwd(tok, T, V, C, dout, ld(dout), dt1, ld(dt1), scale=scale, dtype=code)
    torch.cuda.synchronize()
    within(dt1, ref, bound, dt)
    assert (dt1[~used] == 0).all() and untouched()
    # Added to; rows of no token keep their bits (NaN and -0 among them).
    dt2, untouched = blank((V, C), dt, pad, start)
    dt2.copy_(rand((V, C), dt, 63))
    dt2[~used] = float("nan")
    was = dt2.clone()
    gpu_ctx.embedding_bwd(tok, T, V, C, dout, ld(dout), dt2, ld(dt2), scale=scale, accumulate=True,
                          dtype=code)
    torch.cuda.synchronize()
    w = was[used].double()
    within(dt2[used], w + ref[used], bound[used] + U * (w.abs() + ref[used].abs()), dt)
    assert torch.isnan(dt2[~used]).all() and untouched()
    # The same call again: the same bits.
    dt3, _ = blank((V, C), dt, pad, start)
    gpu_ctx.embedding_bwd(tok, T, V, C, dout, ld(dout), dt3, ld(dt3), scale=scale, dtype=code)
    torch.cuda.synchronize()
    assert torch.equal(dt1, dt3)


def test_embedding_backward_of_no_tokens_and_infinite_rows(gpu_ctx):
    d = torch.full((5, 12), 7.0, device="cuda")
    tok = torch.zeros(4, dtype=torch.int32, device="cuda")
    x = torch.ones((4, 12), device="cuda")
    gpu_ctx.embedding_bwd(tok, 0, 5, 12, x, 12, d, 12, accumulate=True)
    torch.cuda.synchronize()
    assert (d == 7.0).all()
    gpu_ctx.embedding_bwd(tok, 0, 5, 12, x, 12, d, 12)
    torch.cuda.synchronize()
    assert (d == 0.0).all()
    # Infinities stay in their rows and columns.
    tok[:] = torch.tensor([1, 3, 1, 2], dtype=torch.int32)
    x[1, 4] = float("inf")
    gpu_ctx.embedding_bwd(tok, 4, 5, 12, x, 12, d, 12)
    torch.cuda.synchronize()
    assert torch.isinf(d[3, 4]) and torch.isfinite(d).sum() == d.numel() - 1


# ------------------------------------------------------- 8-bit checkpoints
def quantise(x):
    """(q, e, z) by the format's definition, in fp64."""
    R, C = x.shape
    nb = (C + 31) // 32
    xb = torch.nn.functional.pad(x.double(), (0, nb * 32 - C)).view(R, nb, 32)
    top = xb.abs().amax(-1).float().contiguous()
    b = (top.view(torch.int32) >> 23).clamp(min=1).long()
    bad = ~torch.isfinite(xb).all(-1)
    b = torch.where(bad, torch.full_like(b, 255), b)
    pow2 = lambda e: ((e + 1023) << 52).view(torch.float64)
    q = torch.round(xb * pow2(133 - b)[..., None]).clamp(-127, 127)
    q = torch.where(bad[..., None], torch.zeros_like(q), q)
    z = torch.where(bad[..., None], torch.full_like(q, float("nan")), q * pow2(b - 133)[..., None])
    cut = lambda t: t.reshape(R, nb * 32)[:, :C]
    return cut(q).to(torch.int8), b.to(torch.uint8), cut(z)


def gelu_s(z):
    return 0.5 * (1.0 + torch.tanh(C0 * (z + C1 * z ** 3)))


def act_ref(act, z):
    """act(z), act'(z) in fp64 and the bounds of their fp32 evaluation: the
    logistic s's relative error is 4u times its argument's derivative (at most
    0.45) plus one unit each of exp2, add and reciprocal."""
    if act == "none":
        return z, torch.ones_like(z), 0 * z, 0 * z
    if act == "relu":
        return torch.where(z > 0, z, 0 * z), (z > 0).double(), 0 * z, 0 * z
    s = gelu_s(z)
    t = 2.0 * z * C0 * (1.0 + 3.0 * C1 * z * z)
    tb = t.abs().clamp(max=200.0)  # s (1 - s) is 0 past |z| = 8
    return z * s, s + t * s * (1 - s), 16 * U * z.abs(), 8 * U * (1 + tb)


def ckpt_values(R, C, dt, seed, pad=0, start=0):
    """Values over the type's whole range, block by block, zeros and
    borders among them."""
    g = torch.Generator().manual_seed(seed)
    nb = (C + 31) // 32
    lo, hi = {"f32": (-140, 120), "f16": (-20, 13), "bf16": (-120, 120)}[dt]
    e = torch.randint(lo, hi, (R, nb), generator=g).repeat_interleave(32, 1)[:, :C]
    x = torch.ldexp(torch.randn(R, C, generator=g, dtype=torch.float64), e)
    x[torch.rand(R, C, generator=g) < 0.05] = 0.0
    if R > 1:
        x[0] = torch.randn(C, generator=g).double()  # an ordinary row
    if R > 2:
        x[1] = 0.0
    if R > 3:  # steps and half steps of a block whose largest is 127.75 steps
        k = torch.arange(C, dtype=torch.float64) % 32
        x[2] = (k * 4.0 + 0.5) * 2.0 ** -3
        x[2][k == 31] = 127.75 * 2.0 ** -3
    m = torch.finfo(DTS[dt][1]).max
    return place(x.clamp(-m, m).to(DTS[dt][1]), pad, start)


CK_SHAPES = [(1, 1, 0, 0), (1, 31, 0, 0), (2, 32, 0, 0), (5, 33, 1, 1), (4, 100, 0, 0),
             (7, 256, 0, 0), (64, 784, 0, 0), (33, 1000, 8, 0), (50, 1531, 3, 3), (129, 4096, 0, 0),
             (6, 8200, 0, 4), (3, 20001, 0, 0), (2000, 64, 0, 0), (1, 131072, 0, 0)]


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("shape", CK_SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_ckpt8_save_and_load(gpu_ctx, dt, shape):
    R, C, pad, start = shape
    note("ckpt8", dt, shape)
    code, ty, _ = DTS[dt]
    x = ckpt_values(R, C, dt, 71, pad, start)
    nb = (C + 31) // 32
    qb = torch.full((R, C + pad + 5), 99, dtype=torch.int8, device="cuda")
    eb = torch.full((R, nb + pad), 99, dtype=torch.uint8, device="cuda")
    q, e = qb[:, start:start + C], eb[:, :nb]
    gpu_ctx.ckpt8_save(x, ld(x), R, C, q, ld(q), e, ld(e), dtype=code)
    torch.cuda.synchronize()
    rq, re, rz = quantise(x)
    assert torch.equal(q, rq) and torch.equal(e, re)
    q.zero_()
    e.zero_()
    assert (qb.sum() == 99 * R * (pad + 5)) and (eb.sum() == 99 * R * pad)
    q.copy_(rq)
    e.copy_(re)
    assert torch.equal(rz.to(ty).double(), rz)  # exact in its type
    step = torch.ldexp(torch.ones_like(rz), e.long().repeat_interleave(32, 1)[:, :C] - 133)
    assert ((rz - x.double()).abs() <= step).all()
    for act in ACTS:
        z, uz = blank((R, C), dt, pad, start)
        h, uh = blank((R, C), dt, pad + 1, start)
        gpu_ctx.ckpt8_load(q, ld(q), e, ld(e), R, C, z=z, ldz=ld(z), h=h, ldh=ld(h),
                           act=ACTS[act], dtype=code)
        h1, z1 = torch.empty_like(h), torch.empty_like(z)
        gpu_ctx.ckpt8_load(q, ld(q), e, ld(e), R, C, h=h1, ldh=ld(h1), act=ACTS[act], dtype=code)
        gpu_ctx.ckpt8_load(q, ld(q), e, ld(e), R, C, z=z1, ldz=ld(z1), act=ACTS[act], dtype=code)
        torch.cuda.synchronize()
        assert torch.equal(z.double(), rz) and torch.equal(z1, z) and uz() and uh()
        small = rz.abs() < 1e12  # gelu's z^3 stays in range
        f, _, bf, _ = act_ref(act, torch.where(small, rz, 0 * rz))
        within(torch.where(small, h.double(), f), f, bf, dt)
        assert torch.equal(h, h1)


@pytest.mark.parametrize("dt", DTS)
def test_ckpt8_blocks_with_infinities_and_nan(gpu_ctx, dt):
    code = DTS[dt][0]
    x = rand((3, 200), dt, 81)
    x[0, 40], x[1, 199], x[2, 0] = float("inf"), float("nan"), float("-inf")
    q = torch.empty((3, 200), dtype=torch.int8, device="cuda")
    e = torch.empty((3, 7), dtype=torch.uint8, device="cuda")
    z = torch.empty_like(x)
    gpu_ctx.ckpt8_save(x, 200, 3, 200, q, 200, e, 7, dtype=code)
    gpu_ctx.ckpt8_load(q, 200, e, 7, 3, 200, z=z, dtype=code)
    torch.cuda.synchronize()
    rq, re, rz = quantise(x)
    assert torch.equal(e, re) and int((e == 255).sum()) == 3
    nan = torch.isnan(rz)
    assert torch.equal(torch.isnan(z), nan) and torch.equal(z[~nan].double(), rz[~nan])
    assert torch.isnan(z[0, 32:64]).all() and torch.isnan(z[1, 192:]).all()


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("shape", CK_SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_act_bwd_ckpt8(gpu_ctx, dt, act, shape):
    R, C, pad, start = shape
    note("act_bwd_ckpt8", dt, act, shape)
    code = DTS[dt][0]
    q, e, z = quantise(rand((R, C), dt, 91, 2.0))
    q, e = q.contiguous(), e.contiguous()
    dh = rand((R, C), dt, 92, 1.0, 0.0, pad, start)
    dz, untouched = blank((R, C), dt, pad, start)
    gpu_ctx.act_bwd_ckpt8(ACTS[act], dh, ld(dh), q, C, e, e.shape[1], R, C, dz, ld(dz), dtype=code)
    torch.cuda.synchronize()
    _, d, _, bd = act_ref(act, z)
    within(dz, dh.double() * d, dh.double().abs() * (bd + U * d.abs()), dt)
    assert untouched()
    dh2 = dh.clone()
    gpu_ctx.act_bwd_ckpt8(ACTS[act], dh2, ld(dh2), q, C, e, e.shape[1], R, C, dh2, ld(dh2),
                          dtype=code)
    torch.cuda.synchronize()
    assert torch.equal(dh2, dz)


MM = [(1, 1, 1), (3, 5, 33), (64, 10, 256), (50, 101, 215), (256, 128, 512), (130, 1000, 260),
      (777, 333, 1029)]


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("shape", MM, ids=lambda s: "x".join(map(str, s)))
def test_matmul_bwd_ckpt8(gpu_ctx, dt, act, shape):
    M, N, K = shape
    note("matmul_bwd_ckpt8", dt, act, shape)
    code, ty, hu = DTS[dt]
    q, e, z = quantise(rand((M, K), dt, 101))
    q, e = q.contiguous(), e.contiguous()
    w = rand((K, N), dt, 102, math.sqrt(2.0 / K), 0.0, 1)
    dz = rand((M, N), dt, 103, 1.0, 0.0, 2)
    zr, xr = (torch.empty((M, K), dtype=ty, device="cuda") for _ in range(2))
    dx, ux = blank((M, K), dt, 3)
    dw, uw = blank((K, N), dt, 1)
    db, ub = blank((1, N), dt)

    def run(acc, dbias=True):
        gpu_ctx.matmul_bwd_ckpt8(M, N, K, q, K, e, e.shape[1], w, ld(w), dz, ld(dz), xr, dx, ld(dx),
                                 dw, ld(dw), Zr=zr if act != "none" else None,
                                 dbias=db if dbias else None, act=ACTS[act], accumulate=acc,
                                 dtype=code)
        torch.cuda.synchronize()

    run(False)
    f, d, bf, bd = act_ref(act, z)
    d64, w64 = dz.double().contiguous(), w.double().contiguous()
    # dW: the rounding of act(z) to its type, then any order of M terms.
    bx = bf + (hu if dt != "f32" else 0) * (f.abs() + bf) + TINY[dt]
    rdw = f.t().contiguous() @ d64
    bdw = bx.t().contiguous() @ d64.abs() + (M + 2) * U * (f.abs().t().contiguous() @ d64.abs())
    within(dw, rdw, bdw, dt)
    # dX: the product's own rounding to its type comes before act'.
    p = d64 @ w64.t().contiguous()
    pa = (N + 2) * U * (d64.abs() @ w64.abs().t().contiguous())
    pa = pa + (hu if dt != "f32" else 0) * (p.abs() + pa) + TINY[dt]
    bdx = pa * (d.abs() + bd) + p.abs() * (bd + U * d.abs())
    within(dx, p * d, bdx, dt)
    rdb, bdb = d64.sum(0), (M + 2) * U * d64.abs().sum(0)
    within(db[0], rdb, bdb, dt)
    assert ux() and uw() and ub()
    was = dx.double().clone(), dw.double().clone(), db.double().clone()
    run(True)
    hh = 0 if dt == "f32" else hu  # the sum is rounded before it is added
    for got, w0, ref, b in ((dx, was[0], p * d, bdx), (dw, was[1], rdw, bdw),
                            (db[0], was[2][0], rdb, bdb)):
        within(got, w0 + ref, b + (U + hh) * (w0.abs() + ref.abs() + b) + TINY[dt], dt)
    run(False, dbias=False)


# --------------------------------------- streams, graphs, far offsets, order
def test_calls_follow_their_contexts_stream_and_replay_in_graphs(gpu_ctx):
    """Each operator captured into a graph on a context of its own, replayed
    between eager calls of other sizes on the same context, gives the eager
    bits every time."""
    import ferrograd_amd as fa

    s = torch.cuda.Stream()
    ctx = fa.Context(0, s.cuda_stream)
    try:
        ctx.reserve_workspace(64 << 20)
        R, C, V = 700, 520, 300
        x, dy = rand((R, C), "bf16", 111), rand((R, C), "bf16", 112)
        tok = tokens_of("hot", R, V, 113)
        mean, rstd = (torch.empty(R, device="cuda") for _ in range(2))
        ty = torch.bfloat16
        new = lambda *sh: torch.empty(sh, dtype=ty, device="cuda")
        y, dx, dg, db, dtab, z, h = (new(R, C), new(R, C), new(C), new(C), new(V, C), new(R, C),
                                     new(R, C))
        q = torch.empty((R, C), dtype=torch.int8, device="cuda")
        e = torch.empty((R, 17), dtype=torch.uint8, device="cuda")
        outs = [y, mean, rstd, dx, dg, db, dtab, z, h]

        def calls():
            ctx.layer_norm(x, C, R, C, y, C, mean=mean, rstd=rstd, dtype=2)
            ctx.layer_norm_bwd(x, C, dy, C, mean, rstd, R, C, dx=dx, lddx=C, dgamma=dg, dbeta=db,
                               dtype=2)
            ctx.embedding_bwd(tok, R, V, C, dx, C, dtab, C, dtype=2)
            ctx.ckpt8_save(y, C, R, C, q, C, e, 17, dtype=2)
            ctx.ckpt8_load(q, C, e, 17, R, C, z=z, h=h, act=2, dtype=2)

        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            calls()
        torch.cuda.synchronize()
        want = [t.clone() for t in outs]
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            calls()
        other = rand((3000, 1100), "f32", 114)
        om, orr = torch.zeros(3000, device="cuda"), torch.ones(3000, device="cuda")
        od, ot = torch.empty(1100, device="cuda"), torch.empty((90, 1100), device="cuda")
        otok = tokens_of("uniform", 3000, 90, 115)
        for rep in range(4):
            for t in outs:
                t.zero_()
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            for t, w in zip(outs, want):
                assert torch.equal(t, w), rep
            with torch.cuda.stream(s):  # eager work in the same workspace
                ctx.layer_norm_bwd(other, 1100, other, 1100, om, orr, 3000, 1100, dgamma=od)
                ctx.embedding_bwd(otok, 3000, 90, 1100, other, 1100, ot, 1100)
            if rep % 2:
                torch.cuda.synchronize()
    finally:
        ctx.sync()
        ctx.close()


def test_offsets_past_32_bits(gpu_ctx):
    """2^31 + elements: the last rows of tensors of more than 4 GiB."""
    R, C = 66000, 32768
    code, ty, _ = DTS["bf16"]
    x = torch.zeros((R, C), dtype=ty, device="cuda")
    tail = rand((40, C), "bf16", 121)
    x[-40:] = tail
    y = torch.empty_like(x)
    gpu_ctx.layer_norm(x, C, R, C, y, C, dtype=code)
    y1 = torch.empty_like(tail)
    gpu_ctx.layer_norm(tail, C, 40, C, y1, C, dtype=code)
    torch.cuda.synchronize()
    assert torch.equal(y[-40:], y1) and (y[0] == 0).all()
    mean, rstd = torch.zeros(R, device="cuda"), torch.ones(R, device="cuda")
    dg, dg1 = (torch.empty(C, dtype=ty, device="cuda") for _ in range(2))
    gpu_ctx.layer_norm_bwd(x, C, x, C, mean, rstd, R, C, dx=y, lddx=C, dgamma=dg, dtype=code)
    gpu_ctx.layer_norm_bwd(tail, C, tail, C, mean, rstd, 40, C, dx=y1, lddx=C, dgamma=dg1,
                           dtype=code)
    torch.cuda.synchronize()
    assert torch.equal(y[-40:], y1)
    ref = (tail.double() ** 2).sum(0)
    within(dg, ref, 200 * U * ref, "bf16")
    # The lookup and its gradient, at the table's end and at the batch's.
    tok = torch.zeros(R, dtype=torch.int32, device="cuda")
    tok[-40:] = torch.arange(R - 40, R, dtype=torch.int32, device="cuda")
    gpu_ctx.embedding(tok, R, R, C, x, C, y, C, dtype=code)
    torch.cuda.synchronize()
    assert torch.equal(y[-40:], tail) and (y[0] == 0).all()
    y.fill_(9.0)
    gpu_ctx.embedding_bwd(tok, R, R, C, x, C, y, C, dtype=code)
    torch.cuda.synchronize()
    assert torch.equal(y[-40:], tail) and (y[1:100] == 0).all()
    q = torch.empty((R, C), dtype=torch.int8, device="cuda")
    e = torch.empty((R, C // 32), dtype=torch.uint8, device="cuda")
    gpu_ctx.ckpt8_save(x, C, R, C, q, C, e, C // 32, dtype=code)
    gpu_ctx.ckpt8_load(q, C, e, C // 32, R, C, z=y, dtype=code)
    torch.cuda.synchronize()
    assert torch.equal(y[-40:].double(), quantise(tail)[2]) and (y[0] == 0).all()
