"""Attention's backward over the range of its tensors' types: values far above order one,
gradients of any size.

Tolerances are the bounds of test_attention_gpu.py, and for fp16 one term more: dS carries a
power of two.  It brings the largest |dout| to 2^3 at least, unless something would pass 2^15 with
it, which it then brings to 2^14 at least: for dq the largest |dS|, for dk the largest |dout| times
the sum of the key's |V| and the largest |delta|, which bound dS.  fp16's half step below its
normal numbers, 2^-25, so stands for at most 2^-28 of the largest |dout| or 2^-39 of those.
"""
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from test_attention_gpu import FLUSH, Batch  # noqa: E402
from test_token_ops_gpu import DTS, U, note, rand, within  # noqa: E402


def check(b, grads, out, lse, dout):
    """dq, dk and dv of a batch against fp64."""
    h, D, G = DTS[b.dt][2], b.D, b.heads // b.kv
    got = [g.cpu() for g in grads]
    for s, (lq, lk) in enumerate(b.seqs):
        rq, rk = slice(b.qs[s], b.qs[s] + lq), slice(b.ks[s], b.ks[s] + lk)
        for c in range(b.kv):
            work, far = [], 0.0
            for head in range(c * G, c * G + G):
                cols = slice(head * D, head * D + D)
                q, k, v, see, z, err = b.parts(s, head)
                L = lse[head, rq].double().cpu()[:, None]
                do, o = dout[rq, cols].double().cpu(), out[rq, cols].double().cpu()
                p = torch.where(see, torch.exp(z - L), 0.0)
                ep = torch.where(see, 2 * err + U * (8 * L.abs() + 16), 0.0)
                delta = (do * o).sum(1)[:, None]
                part = do @ v.t() - delta
                ed = U * (D + 8) * (do.abs() @ v.abs().t() + (do * o).abs().sum(1)[:, None])
                work.append((head, cols, q, k, do, see, p, ep, p * part,
                             p * (part.abs() * ep + ed) + see * FLUSH * part.abs()))
                far = max(far, delta.abs().max().item())
            most = max((w[8].abs() + w[9]).max().item() for w in work)
            big = max(w[4].abs().max().item() for w in work)
            low, low_k = 0.0, 0.0
            if b.dt == "f16":
                low = 2.0 ** -28 * big + 2.0 ** -39 * most
                low_k = 2.0 ** -28 * big + 2.0 ** -39 * 1.001 * (big * v.abs().sum(1) + far)
            tp = 2.0 ** -33 if b.dt == "f16" else FLUSH
            dk, dv, bk, bv = (torch.zeros(lk, D).double() for _ in range(4))
            for head, cols, q, k, do, see, p, ep, ds, es in work:
                es = es + h * ds.abs()
                ek, es = es + low_k * see, es + low * see
                dq = b.scale * (ds @ k)
                bq = b.scale * (es @ k.abs() + U * (lk + 64) * (ds.abs() @ k.abs()))
                assert dq.abs().max() < 6e4
                within(got[0][rq, cols], dq, bq + 8 * U * dq.abs(), b.dt)
                dk += b.scale * (ds.t() @ q)
                n = lq * G
                bk += b.scale * (ek.t() @ q.abs() + U * (n + 64) * (ds.abs().t() @ q.abs()))
                dv += p.t() @ do
                bv += (p * (h + ep)).t() @ do.abs() + (U * (n + 64) * p + tp * see).t() @ do.abs()
            cols = slice(c * D, c * D + D)
            assert max(dk.abs().max(), dv.abs().max()) < 6e4
            within(got[1][rk, cols], dk, bk + 8 * U * dk.abs(), b.dt)
            within(got[2][rk, cols], dv, bv + 8 * U * dv.abs(), b.dt)


# Direct tiles; heads of other widths and rows off 16-byte boundaries, through registers; few
# tiles over long rows and keys, in splits; rows of unlike sight in one tile.
SHAPES = [
    ([(1, 2)], 1, 1, 128, False, 0), ([(100, 100), (40, 90)], 4, 2, 64, True, 0),
    ([(150, 150)], 2, 1, 128, True, 8), ([(90, 130)], 2, 1, 128, False, 3),
    ([(70, 70), (65, 33)], 2, 2, 40, False, 1), ([(77, 140)], 3, 1, 96, True, 0),
    ([(8, 3000)], 2, 1, 64, True, 0), ([(1500, 40)], 1, 1, 128, False, 0),
]


@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("dsize", [2.0 ** -14, 1.0, 2.0 ** 8])
@pytest.mark.parametrize("vsize,coherent", [(64.0, True), (130.0, True), (4000.0, True),
                                            (1000.0, False)])
@pytest.mark.parametrize("seqs,heads,kv,D,causal,pad", SHAPES,
                         ids=[f"{i}-D{c[3]}" for i, c in enumerate(SHAPES)])
def test_large_values(gpu_ctx, dt, dsize, vsize, coherent, seqs, heads, kv, D, causal, pad):
    """V far above order one: dS = P (dout . v - delta) has up to its size times D.  Coherent:
    all of a value's columns alike, its sign by the key, dout of one sign."""
    note("large values", dt, dsize, vsize, coherent, seqs, D)
    # (Keys and queries as small as keeps the gradients, dS's sums over them, in fp16.)
    b = Batch(seqs, heads, kv, D, dt, causal, pad)
    for t in (b.q, b.k):
        t.mul_(min(1.0, 20.0 / (dsize * vsize)))
    dout = rand((b.Tq, heads * D), dt, 9, 1.0, 0.0, pad)
    if coherent:
        sign = torch.where(torch.arange(b.Tk, device="cuda") % 2 == 0, 1.0, -1.0)
        b.v.copy_((sign * vsize)[:, None].expand(-1, kv * D))
        dout.abs_().clamp_(0.5, 2.0)
    else:
        b.v.mul_(vsize)
    dout.mul_(dsize)
    out, lse = b.forward(gpu_ctx)
    grads = b.backward(gpu_ctx, out, lse, dout)
    check(b, grads, out, lse, dout)
    assert all(torch.equal(x, y) for x, y in zip(grads, b.backward(gpu_ctx, out, lse, dout)))


@pytest.mark.parametrize("D,pad", [(64, 0), (128, 0), (100, 1)])
def test_fp16_power_falls_on_the_way(gpu_ctx, D, pad):
    """Values that grow along the keys, and gradients that grow along the rows: dS passes
    fp16's range only after sums were taken that carry another power."""
    note("power falls", D, pad)
    b = Batch([(260, 260)], 2, 1, D, "f16", False, pad)
    b.q.mul_(0.02)
    b.k.mul_(0.02)
    grow = 2.0 ** (torch.arange(260, device="cuda") // 26 - 1).float()
    b.v.mul_(grow[:, None])
    dout = rand((260, 2 * D), "f16", 9, 1.0, 0.0, pad)
    dout.mul_(2.0 ** (torch.arange(260, device="cuda") // 40 - 4).float()[:, None])
    out, lse = b.forward(gpu_ctx)
    check(b, b.backward(gpu_ctx, out, lse, dout), out, lse, dout)


@pytest.mark.parametrize("D", [64, 40])
def test_fp16_infinite_gradients_stay_their_rows(gpu_ctx, D):
    """A row whose dout is infinite or NaN has no finite dq; the other rows' are as without it."""
    note("infinite dout", D)
    b = Batch([(64, 64)], 1, 1, D, "f16", False)
    dout = rand((64, D), "f16", 9)
    out, lse = b.forward(gpu_ctx)
    want = b.backward(gpu_ctx, out, lse, dout)[0]
    dout[7, 3], dout[40, 0] = math.inf, math.nan
    got = b.backward(gpu_ctx, out, lse, dout)[0]
    rest = torch.ones(64, dtype=torch.bool, device="cuda")
    rest[[7, 40]] = False
    assert torch.equal(got[rest], want[rest]) and not torch.isfinite(got[~rest].float()).any()


@pytest.mark.parametrize("D,pad", [(128, 0), (128, 1), (64, 0), (80, 0)])
@pytest.mark.parametrize("value", [64.0, 100.0, 130.0, 4000.0])
def test_one_query_between_two_values(gpu_ctx, D, pad, value):
    """One query, two keys of equal score, values +v and -v, dout of one sign: out and delta are
    0, dS is dout . v / 2."""
    note("two values", D, pad, value)
    b = Batch([(1, 2)], 1, 1, D, "f16", True, pad)
    b.q.zero_()
    b.q[0, 0] = 1.0
    b.k.zero_()
    b.k[0, 1], b.k[1, 1] = 0.01, -0.01
    b.v[0], b.v[1] = value, -value
    dout = torch.full((1, D), 1.9, dtype=torch.float16, device="cuda")
    out, lse = b.forward(gpu_ctx)
    check(b, b.backward(gpu_ctx, out, lse, dout), out, lse, dout)


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D,pad", [(64, 0), (128, 0), (128, 1), (40, 0)])
@pytest.mark.parametrize("lq,lk,bad", [(2, 2, math.inf), (70, 90, math.nan), (70, 90, math.inf),
                                       (6, 3000, math.nan)])
def test_rows_of_minus_infinity_beside_keys_out_of_sight(gpu_ctx, dt, D, pad, lq, lk, bad):
    """Rows that see keys at scores of -inf alone have a dq of 0, whatever a key holds that
    they do not see."""
    note("-inf beside", dt, D, pad, lq, lk, bad)
    b = Batch([(lq, lk)], 2, 1, D, dt, True, pad)
    rows = list(range(0, lq - 1, 3))  # (the last row sees the last key)
    b.k[:, 0] = b.k[:, 0].abs() + 0.5
    for head in range(2):
        b.q[rows, head * D] = -math.inf
    dout = rand((b.Tq, 2 * D), dt, 9, 1.0, 0.0, pad)
    out, lse = b.forward(gpu_ctx)
    assert (out[rows] == 0).all() and (lse[:, rows] == -math.inf).all()
    want = b.backward(gpu_ctx, out, lse, dout)[0]
    assert (want[rows] == 0).all()
    for t in (b.k, b.v):
        t[lk - 1] = bad
    again, again_lse = b.forward(gpu_ctx)
    assert (again[rows] == 0).all() and (again_lse[:, rows] == -math.inf).all()
    got = b.backward(gpu_ctx, out, lse, dout)[0]
    assert (got[rows] == 0).all()
    assert torch.isfinite(got[:lq - 1].float()).all()


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D,pad", [(64, 0), (128, 0), (100, 1)])
@pytest.mark.parametrize("lq,lk", [(1, 40), (70, 90), (300, 300), (1, 5000), (40, 4000)])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_scores_that_fp32_rounds_by_more_than_one(gpu_ctx, dt, D, pad, lq, lk, sign):
    """Equal scores of some 1e9: every visible key counts alike.  And one key's a little larger:
    it takes all."""
    note("large scores", dt, D, pad, lq, lk, sign)
    b = Batch([(lq, lk)], 2, 1, D, dt, True, pad)
    b.q.fill_(19000.0)
    b.k.fill_(19000.0 * sign)
    h = DTS[dt][2]

    def rows(want):
        # Weights are equal to rounding: sums of as many terms, in any order, and P's rounding.
        out, lse = b.forward(gpu_ctx)
        bound = (h + U * (lk + 64)) * b.v.double().abs().cpu().max() * torch.ones(lq, D)
        for head in range(2):
            within(out[:, head * D:head * D + D].cpu(), want, bound, dt)
        z = b.scale * D * (b.q[0, 0].double() * b.k[:, 0].double().max()).item()
        assert (lse.double().cpu() - z).abs().max() <= 1e-4 * abs(z)

    v = b.v.double().cpu()
    seen = torch.arange(lk)[None] <= torch.arange(lq)[:, None] + lk - lq
    rows((seen.double() @ v) / seen.sum(1)[:, None])
    last = lk - lq  # (the last key that every row sees)
    b.k[last] += 1024.0
    rows(v[last].expand(lq, D))


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("scale", [2.0 ** -120, 1e-30, 1e-10])
@pytest.mark.parametrize("D,pad", [(64, 0), (100, 1)])
def test_small_scales(gpu_ctx, dt, scale, D, pad):
    """Scales that leave every visible key the same weight."""
    note("small scale", dt, scale, D, pad)
    b = Batch([(70, 90), (1, 300)], 2, 1, D, dt, True, pad)
    b.scale = float(scale)
    out, lse = b.forward(gpu_ctx)
    b.check_forward(out, lse)
    dout = rand((b.Tq, 2 * D), dt, 9, 1.0, 0.0, pad)
    grads = b.backward(gpu_ctx, out, lse, dout)
    b.check_backward(grads, out, lse, dout)
    assert bool((grads[2] != 0).any())


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D,pad", [(64, 0), (128, 0), (100, 1)])
@pytest.mark.parametrize("lq,lk", [(1, 40), (70, 90), (300, 300), (8, 3000)])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("one", [False, True])
def test_gradients_of_scores_that_fp32_rounds_by_more_than_one(gpu_ctx, dt, D, pad, lq, lk, sign, one):
    """lse alone no longer holds such rows' probabilities.  Equal scores: P is 1 / n; one key's
    larger: 1 and 0.  Beside a sequence of ordinary scores."""
    note("gradients of large scores", dt, D, pad, lq, lk, sign, one)
    b = Batch([(lq, lk), (40, 50)], 2, 1, D, dt, True, pad)
    far_q, far_k = slice(0, lq), slice(0, lk)
    b.q[far_q] = 19000.0
    b.k[far_k] = 19000.0 * sign
    see = torch.arange(lk)[None] <= torch.arange(lq)[:, None] + lk - lq
    p = see.double() / see.sum(1)[:, None]
    if one:
        last = lk - lq  # (the last key that every row sees)
        b.k[last] += 1024.0
        p = torch.zeros(lq, lk).double()
        p[:, last] = 1.0
    out, lse = b.forward(gpu_ctx)
    dout = rand((b.Tq, 2 * D), dt, 9, 2.0 ** -6, 0.0, pad)
    grads = b.backward(gpu_ctx, out, lse, dout)
    assert all(torch.equal(x, y) for x, y in zip(grads, b.backward(gpu_ctx, out, lse, dout)))
    # The ordinary sequence, as ever.
    near = [g.clone() for g in grads]
    seqs, qs, ks = b.seqs, b.qs, b.ks
    b.seqs, b.qs, b.ks = seqs[1:], qs[1:], ks[1:]
    check(b, near, out, lse, dout)
    b.seqs, b.qs, b.ks = seqs, qs, ks
    # The other: everything is fp32; P is off by its sum's rounding.
    k, v = b.k[far_k].double().cpu(), b.v[far_k].double().cpu()
    dk, dv, bk, bv = (torch.zeros(lk, D).double() for _ in range(4))
    for head in range(2):
        cols = slice(head * D, head * D + D)
        q, do, o = (t[far_q, cols].double().cpu() for t in (b.q, dout, out))
        part = do @ v.t() - (do * o).sum(1)[:, None]
        ds, rel = p * part, U * (lk + 64)
        es = p * (part.abs() * rel + U * (D + 8) * (do.abs() @ v.abs().t()
                                                    + (do * o).abs().sum(1)[:, None]))
        dq = b.scale * (ds @ k)
        within(grads[0][far_q, cols].cpu(), dq,
               b.scale * ((es + ds.abs() * U * (lk + 64)) @ k.abs()) + 8 * U * dq.abs(), dt)
        dk += b.scale * (ds.t() @ q)
        bk += b.scale * ((es + ds.abs() * U * (2 * lq + 64)).t() @ q.abs())
        dv += p.t() @ do
        bv += (p * (rel + U * (2 * lq + 64))).t() @ do.abs()
    within(grads[1][far_k].cpu(), dk, bk + 8 * U * dk.abs(), dt)
    within(grads[2][far_k].cpu(), dv, bv + 8 * U * dv.abs(), dt)


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D,pad", [(64, 0), (128, 0), (100, 1)])
@pytest.mark.parametrize("lq,lk,hidden", [(1, 40, False), (70, 90, False), (70, 90, True),
                                          (1, 5000, False), (200, 4000, False), (200, 4000, True)])
def test_rows_of_minus_infinity_are_0_whatever_the_values(gpu_ctx, dt, D, pad, lq, lk, hidden):
    """A row of none but scores of -inf is 0 also where a value that it sees is infinite (in
    splits and not, beside an infinite key out of sight and not)."""
    note("-inf and infinite values", dt, D, pad, lq, lk, hidden)
    b = Batch([(lq, lk)], 2, 1, D, dt, True, pad)
    rows = list(range(0, max(1, lq - 1), 2))
    b.k[:, 0] = b.k[:, 0].abs() + 0.5
    for head in range(2):
        b.q[rows, head * D] = -math.inf
    b.v[0] = math.inf
    if hidden:
        b.k[lk - 1], b.v[lk - 1] = math.inf, math.nan
    out, lse = b.forward(gpu_ctx)
    assert (out[rows] == 0).all() and (lse[:, rows] == -math.inf).all()
