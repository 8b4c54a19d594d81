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
