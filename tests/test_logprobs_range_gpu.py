"""Token log probabilities and their gradient at large inverse temperatures and with logits at
the ends of their type, masked by -inf or by the type's lowest number."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from test_attention_gpu import FLUSH  # noqa: E402
from test_block_ops_gpu import lp_bwd_oracle, lp_oracle, run_lp, tops_oracle  # noqa: E402
from test_token_ops_gpu import DTS, U, blank, ld, note, rand, within  # noqa: E402


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("scale", [1e-9, 2e4, 1e5, 1e9, 1e30])
@pytest.mark.parametrize("C", [37, 1000, 20003])
def test_gradient_at_any_temperature(gpu_ctx, dt, scale, C):
    """Masked logits have no probability, whatever the scale: their gradients are 0, and the
    others' as the formula's."""
    note("temperature", dt, scale, C)
    scale = float(np.float32(scale))
    x = rand((6, C), dt, 31, min(2.0, 20.0 / scale) if scale > 1e-3 else 2.0)
    if dt == "f16" and scale > 1e4:  # what is left of these steps in fp16: a few equal numbers
        x.copy_(torch.where(x > 0, 0.0, -1.0))
    top = x.float().amax(1, keepdim=True)
    x[:, 2:5] = top.to(x.dtype)  # several columns share a row's probability
    low = torch.finfo(DTS[dt][1]).min
    x[0, 7:] = -math.inf
    x[1, 7:] = low
    x[2, 1::2] = -math.inf
    x[3, 20:] = low
    tok = torch.tensor([2, 3, 4, 25, C - 1, C])  # (row 3's is masked)
    (_, _), (h, _), (lse, _) = lp_oracle(x, tok, scale)
    h, lse = h.float().cuda(), lse.float().cuda()
    a, b = torch.tensor([1.0, -2.0, 0.5, 1.0, 3.0, 1.0]).cuda(), torch.tensor(
        [1.0, 0.25, -1.0, 1.0, 2.0, 1.0]).cuda()
    if dt == "f16" or scale < 1.0:  # (gradients of order one)
        a, b = a / scale, b / scale
    zero = torch.zeros_like(a)
    for ga, gb in ((a, b), (a, None), (None, b)):
        want, bound = lp_bwd_oracle(x, tok, scale, lse, h, zero if ga is None else ga,
                                    zero if gb is None else gb)
        out, clean = blank((6, C), dt, 1)
        gpu_ctx.token_logprobs_bwd(x, ld(x), tok.int().cuda(), 6, C, lse, out, ld(out), entropy=h,
                                   dlogp=ga, dentropy=gb, scale=scale, dtype=DTS[dt][0])
        torch.cuda.synchronize()
        assert torch.isfinite(out.float()).all() and clean()
        # Exponentials below fp32's smallest normal number, FLUSH, are 0: off by p < FLUSH of
        # a's term and, since p log(1 / p) grows with p there, by FLUSH (log(1 / FLUSH) + h) of b's.
        ga_, gb_ = (0.0 if t is None else t.abs().double().cpu()[:, None] for t in (ga, gb))
        flush = FLUSH * scale * (ga_ + gb_ * (88.0 + h.abs().double().cpu()[:, None]))
        within(out.cpu(), want, bound + flush, dt)
        assert (out[0, 7:] == 0).all() and (out[2, 1::2] == 0).all()


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_gradient_of_nan_logits_is_nan(gpu_ctx, dt):
    """A row that holds NaN has an lse of NaN, and so has every gradient of it."""
    x = rand((3, 700), dt, 32)
    x[1, 5] = math.nan
    tok = torch.tensor([3, 4, 699])
    (_, _), (h, _), (lse, _) = lp_oracle(x, tok, 1.0)
    one, out = torch.ones(3, device="cuda"), torch.zeros_like(x)
    for gb in (None, one):
        gpu_ctx.token_logprobs_bwd(x, ld(x), tok.int().cuda(), 3, 700, lse.float().cuda(), out,
                                   ld(out), entropy=h.float().cuda(), dlogp=one, dentropy=gb,
                                   dtype=DTS[dt][0])
        assert torch.isnan(out[1]).all() and torch.isfinite(out[[0, 2]].float()).all()


# A wave a row, four waves, rows in splits.
WIDTHS = [1, 5, 100, 3001, 40003, 131072]


def of_one_value(ctx, x, dt, scale, value, live, note_):
    """Rows whose `live` columns hold `value`, the largest there is: a uniform answer."""
    note(*note_)
    R, C = x.shape
    n = live.sum().item()
    cols = live.nonzero().flatten()
    tok = torch.stack([cols[0], cols[-1], cols[n // 2]]).cpu()
    top = min(C, 32)
    (logp, h, lse), ids, tops = run_lp(ctx, x, tok, dt, top, scale)
    # The sum is a whole number below 2^24; a logarithm and a subtraction.
    tol = torch.full((R,), 8 * U * (1.0 + math.log(n)))
    want = torch.full((R,), math.log(n)).double()
    within(logp.cpu(), -want, tol)
    within(h.cpu(), want, tol)
    z = value * scale
    within(lse.cpu(), z + want, tol + 4 * U * abs(z))
    assert torch.equal(ids.long(), tops_oracle(x, top))
    some = min(n, top)
    within(tops[:, :some], -want[:, None].expand(-1, some), tol[:, None])
    return tops


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("C", WIDTHS)
@pytest.mark.parametrize("scale", [1.0, 0.7])
def test_rows_of_the_types_lowest_number(gpu_ctx, dt, C, scale):
    """A mask of the type's lowest number that leaves nothing is a row of equal logits; among
    logits of -inf too, and at the type's largest."""
    scale = float(np.float32(scale))
    info = torch.finfo(DTS[dt][1])
    every = torch.ones(C, dtype=torch.bool, device="cuda")
    for value in (info.min, info.max):
        x = torch.full((3, C), value, dtype=DTS[dt][1], device="cuda")
        of_one_value(gpu_ctx, x, dt, scale, value, every, ("lowest", dt, C, value))
    if C < 5:
        return
    some = every.clone()
    some[1::2] = False
    x = torch.full((3, C), info.min, dtype=DTS[dt][1], device="cuda")
    x[:, 1::2] = -math.inf
    tops = of_one_value(gpu_ctx, x, dt, scale, info.min, some, ("lowest and -inf", dt, C))
    assert (tops[:, int(some.sum()):] == -math.inf).all()


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("C", [100, 3001, 40003, 131072])
def test_masked_tokens_of_the_lowest_number(gpu_ctx, dt, C):
    """Beside ordinary logits the lowest number is itself as a log probability, to rounding; a
    few large logits at one end of a row leave the rest without probability."""
    note("masked tokens", dt, C)
    low = torch.finfo(DTS[dt][1]).min
    x = torch.full((3, C), low, dtype=DTS[dt][1], device="cuda")
    x[0, 7:12] = 1.0
    x[1, C - 5:] = 2.0
    x[2, :] = low
    x[2, C // 2] = 3e38
    tok = torch.tensor([C - 1, 0, C // 2])
    (logp, h, lse), ids, tops = run_lp(gpu_ctx, x, tok, dt, 20, 1.0)
    five = math.log(5)
    within(logp.cpu(), torch.tensor([low, low, 0.0]).double(),
           torch.tensor([-low * U * 4, -low * U * 4, 1e-30]))
    within(h.cpu(), torch.tensor([five, five, 0.0]).double(), torch.tensor([1.0] * 3) * 32 * U)
    top = x[2, C // 2].item()
    within(lse.cpu(), torch.tensor([1.0 + five, 2.0 + five, top]).double(),
           torch.tensor([16 * U, 16 * U, 4 * U * top]))
    assert torch.equal(ids.long(), tops_oracle(x, 20))
    within(tops[:2, :5], torch.full((2, 5), -five).double(), torch.full((2, 5), 16 * U))
    within(tops[:2, 5:], torch.full((2, 15), low).double(), torch.full((2, 15), -low * U * 4))


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("value", [-1e10, -1e20, 3e20, "lowest"])
@pytest.mark.parametrize("scale", [1.0, 0.7, 0.37])
def test_gradient_of_rows_far_from_zero(gpu_ctx, dt, value, scale):
    """An lse so large that fp32 rounds it by more than the logits' spread: probabilities
    stay between 0 and 1."""
    note("far", dt, value, scale)
    ty, scale = DTS[dt][1], float(np.float32(scale))
    for C in (5, 1000):
        x = torch.full((2, C), torch.finfo(ty).min if value == "lowest" else value, dtype=ty,
                       device="cuda")
        tok = torch.tensor([1, C - 1])
        (_, h, lse), _, _ = run_lp(gpu_ctx, x, tok, dt, 0, scale)
        assert torch.isfinite(lse).all() and torch.isfinite(h).all()
        out, (a, b) = torch.zeros_like(x), (torch.tensor(t, device="cuda") for t in ([2.0, -1.0],
                                                                                     [0.5, 1.0]))
        gpu_ctx.token_logprobs_bwd(x, C, tok.int().cuda(), 2, C, lse, out, C, entropy=h, dlogp=a,
                                   dentropy=b, scale=scale, dtype=DTS[dt][0])
        # p (d + h), d <= 0, is at most h, and at least -1 / e.
        most = scale * (a.abs() + b.abs() * (h + 0.4)) * (1.0 + 2.0 ** -7)
        assert (out.float().abs() <= most[:, None]).all()


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("C", WIDTHS)
@pytest.mark.parametrize("value", [-1e4, -1e7, -1e10, 1e9])
def test_rows_of_one_large_number(gpu_ctx, dt, C, value):
    """A mask that leaves nothing, and a product with the scale that fp32 rounds by more than
    1: a row of equal logits all the same."""
    value = torch.tensor(value).to(DTS[dt][1]).item()
    x = torch.full((3, C), value, dtype=DTS[dt][1], device="cuda")
    every = torch.ones(C, dtype=torch.bool, device="cuda")
    of_one_value(gpu_ctx, x, dt, float(np.float32(0.7)), value, every, ("one", dt, C, value))


@pytest.mark.parametrize("C", [3000, 40003, 131072])
@pytest.mark.parametrize("at", [726817.0, -726817.0])
def test_rows_on_both_sides_of_the_large_numbers(gpu_ctx, C, at):
    """Parts of a row whose maximum counts as large, and parts whose does not, one row (2^20 over
    log2(e) is 726817)."""
    note("both sides", C, at)
    x = torch.full((2, C), at - 2.0, device="cuda")
    x[0, C // 2:] = at + 2.0
    x[1, :C // 2] = at + 2.0
    tok = torch.tensor([0, 0])
    (logp, h, lse), _, _ = run_lp(gpu_ctx, x, tok, "f32", 0, 1.0)
    want = lp_oracle(x, tok, 1.0)
    # The differences are exact; a product's rounding at 2^20 is up to 2^-4 in the exponent.
    for g, (w, _) in zip((logp, h, lse), want):
        within(g.cpu(), w, torch.full((2,), 0.1))


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("C", WIDTHS)
def test_rows_of_minus_infinity_alone(gpu_ctx, dt, C):
    """No log probabilities, and no gradients but of rows whose own are 0."""
    note("-inf alone", dt, C)
    x = torch.full((3, C), -math.inf, dtype=DTS[dt][1], device="cuda")
    x[1] = 0.5
    tok = torch.tensor([0, C - 1, C // 2])
    top = min(C, 5)
    (logp, h, lse), ids, tops = run_lp(gpu_ctx, x, tok, dt, top, 1.0)
    for t in (logp, h):
        assert torch.isnan(t).tolist() == [True, False, True]
    assert (lse == -math.inf).tolist() == [True, False, True]
    assert torch.equal(ids, torch.arange(top, dtype=torch.int32).expand(3, -1))
    assert torch.isnan(tops[0]).all() and torch.isfinite(tops[1]).all()
    out = torch.full_like(x, 7.0)
    gpu_ctx.token_logprobs_bwd(x, C, tok.int().cuda(), 3, C, lse, out, C, entropy=h,
                               dlogp=torch.tensor([1.0, 1.0, 0.0], device="cuda"),
                               dtype=DTS[dt][0])
    assert torch.isnan(out[0]).all() and torch.isfinite(out[1].float()).all()
    assert (out[2] == 0).all()
