"""The 16-bit matmul backward from 8-bit activations: each output is rounded to its
type once, in every kernel that its products take."""
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from test_token_ops_gpu import (ACTS, DTS, TINY, U, act_ref, blank, ld, note, quantise, rand,  # noqa: E402
                                within)

# Few rows, 64 x 64 tiles, odd rows, K slices (workspace reserved below), and a layer whose
# two products are one launch.
SHAPES = [(16, 1000, 520), (64, 1001, 333), (50, 101, 215), (130, 1000, 260), (777, 333, 1029),
          (512, 1024, 2048), (2048, 4096, 4096)]


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_matmul_bwd_ckpt8_rounds_once(gpu_ctx, dt, act, shape):
    """dX is (dZ.W^T) act'(z) in fp32, rounded once; dW's operand act(z) is rounded to the
    type, its sum once; accumulated outputs are the fp32 sum with what was there, rounded
    once."""
    M, N, K = shape
    note("matmul_bwd_ckpt8 once", dt, act, shape)
    code, ty, hu = DTS[dt]
    gpu_ctx.reserve_workspace(64 << 20)
    q, e, z = quantise(rand((M, K), dt, 201))
    q, e = q.contiguous(), e.contiguous()
    w = rand((K, N), dt, 202, math.sqrt(2.0 / K))
    dz = rand((M, N), dt, 203)
    zr, xr = (torch.empty((M, K), dtype=ty, device="cuda") for _ in range(2))
    dx, ux = blank((M, K), dt)
    dw, uw = blank((K, N), dt)
    db, ub = blank((1, N), dt)

    def run(acc):
        gpu_ctx.matmul_bwd_ckpt8(M, N, K, q, K, e, e.shape[1], w, ld(w), dz, ld(dz), xr, dx, ld(dx),
                                 dw, ld(dw), Zr=zr, dbias=db, act=ACTS[act], accumulate=acc,
                                 dtype=code)
        torch.cuda.synchronize()

    run(False)
    f, d, bf, bd = act_ref(act, z)
    d64, w64 = dz.double().contiguous(), w.double().contiguous()
    p = d64 @ w64.t().contiguous()
    bp = (N + 2) * U * (d64.abs() @ w64.abs().t().contiguous())
    rdx, bdx = p * d, bp * (d.abs() + bd) + p.abs() * (bd + U * d.abs())
    bx = bf + hu * (f.abs() + bf) + TINY[dt]
    rdw = f.t().contiguous() @ d64
    bdw = bx.t().contiguous() @ d64.abs() + (M + 2) * U * (f.abs().t().contiguous() @ d64.abs())
    rdb, bdb = d64.sum(0), (M + 2) * U * d64.abs().sum(0)
    refs = ((dx, rdx, bdx), (dw, rdw, bdw), (db[0], rdb, bdb))
    for got, ref, b in refs:
        within(got, ref, b, dt)
    for k, (t, ref, _) in enumerate(refs):  # of the outputs' size
        t.copy_(rand((1, t.numel()), dt, 204 + k, float(ref.std(correction=0))).view(t.shape))
    was = [t.double().clone() for t, _, _ in refs]
    run(True)
    for (got, ref, b), w0 in zip(refs, was):
        within(got, w0 + ref, b + U * (w0.abs() + ref.abs() + b), dt)
    assert ux() and uw() and ub()
