"""RMS norm, token log probabilities and attention at the ends of what they take: offsets
past 32 bits, rows far apart, no rows or keys, starts past the tensors' ends, scores that
are all -inf."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from test_attention_gpu import Batch  # noqa: E402
from test_block_ops_gpu import EPS  # noqa: E402
from test_token_ops_gpu import DTS, U, blank, ld, note, rand, within  # noqa: E402


def test_rows_past_32_bits(gpu_ctx):
    """2^31 + elements: the last rows of tensors of more than 4 GiB give what they give by
    themselves."""
    R, C, n = 66000, 32768, 40
    code, ty, _ = DTS["bf16"]
    x = torch.zeros((R, C), dtype=ty, device="cuda")
    tail = rand((n, C), "bf16", 121)
    x[-n:] = tail
    y, s = torch.empty_like(x), torch.empty_like(x)
    q = torch.empty((R, C), dtype=torch.int8, device="cuda")
    e = torch.empty((R, C // 32), dtype=torch.uint8, device="cuda")
    k = torch.empty(R, device="cuda")
    note("rms_norm")
    gpu_ctx.rms_norm(x, C, R, C, y, C, r=x, s=s, eps=EPS, q=q, e=e, rstd=k, dtype=code)
    y1, s1, q1, e1 = (t[:n].clone() for t in (y, s, q, e))
    k1 = torch.empty(n, device="cuda")
    gpu_ctx.rms_norm(tail, C, n, C, y1, C, r=tail, s=s1, eps=EPS, q=q1, e=e1, rstd=k1, dtype=code)
    torch.cuda.synchronize()
    for a, b in ((y, y1), (s, s1), (q, q1), (e, e1), (k, k1)):
        assert torch.equal(a[-n:], b)
    assert (y[0] == 0).all() and torch.equal(s[-n:], tail + tail)
    note("rms_norm_bwd")
    dg, dg1 = (torch.empty(C, dtype=ty, device="cuda") for _ in range(2))
    gpu_ctx.rms_norm_bwd(s, C, x, C, k, R, C, ds=x, dx=y, dgamma=dg, dtype=code)
    gpu_ctx.rms_norm_bwd(s1, C, tail, C, k1, n, C, ds=tail, dx=y1, dgamma=dg1, dtype=code)
    torch.cuda.synchronize()
    assert torch.equal(y[-n:], y1)
    # Sums of n terms that are not 0, in any order, each product off by two roundings.
    terms = tail.double() * s1.double() * k1.double()[:, None]
    within(dg, terms.sum(0), (n + 10 + 2) * U * terms.abs().sum(0), "bf16")
    note("token_logprobs")
    tok = torch.arange(R, dtype=torch.int32, device="cuda") % C
    out = [torch.empty(R, device="cuda") for _ in range(3)]
    one = [torch.empty(n, device="cuda") for _ in range(3)]
    ids, vals = torch.empty((R, 5), dtype=torch.int32, device="cuda"), torch.empty((R, 5), device="cuda")
    ids1, vals1 = ids[:n].clone(), vals[:n].clone()
    run = lambda x, tok, R, o, i, v: gpu_ctx.token_logprobs(
        x, C, tok, R, C, logp=o[0], entropy=o[1], lse=o[2], top=5, top_ids=i, top_logp=v, dtype=code)
    run(x, tok, R, out, ids, vals)
    run(tail, tok[-n:], n, one, ids1, vals1)
    torch.cuda.synchronize()
    # (Few rows are split and joined: the statistics agree as sums in another order do.)
    assert torch.equal(ids[-n:], ids1)
    for a, b in zip(out, one):
        within(a[-n:].cpu(), b.cpu(), 600 * U * (1.0 + b.abs().cpu()))
    assert (out[0][0] + math.log(C)).abs() < 600 * U * math.log(C)
    note("token_logprobs_bwd")
    d = torch.ones(R, device="cuda")
    gpu_ctx.token_logprobs_bwd(x, C, tok, R, C, out[2], y, C, dlogp=d, dtype=code)
    gpu_ctx.token_logprobs_bwd(tail, C, tok[-n:], n, C, out[2][-n:], y1, C, dlogp=d[-n:], dtype=code)
    torch.cuda.synchronize()
    assert torch.equal(y[-n:], y1)


@pytest.mark.parametrize("wide", [2 ** 24 - 8, 2 ** 24 + 8, 2 ** 23 + 1])
def test_attention_of_rows_far_apart(gpu_ctx, wide):
    """Rows of 32 MiB and more: a tile's offsets need 32 bits, or more, of bytes."""
    note("attention", wide)
    heads, kv, D = 2, 1, 64
    b = Batch([(90, 130)], heads, kv, D, "bf16", pad=wide - heads * D)
    out, lse = b.forward(gpu_ctx)
    b.check_forward(out, lse)
    dout = rand((b.Tq, heads * D), "bf16", 9, pad=wide - heads * D)
    made = [torch.full((T, wide), 7.0, dtype=out.dtype, device="cuda") for T in (b.Tq, b.Tk, b.Tk)]
    grads = [t[:, :h * D] for t, h in zip(made, (heads, kv, kv))]
    gpu_ctx.attention_bwd(*b.qkv(), out, ld(out), dout, ld(dout), lse, *b.shape(), grads[0], wide,
                          grads[1], wide, grads[2], wide, scale=b.scale, dtype=DTS["bf16"][0])
    torch.cuda.synchronize()
    b.check_backward(grads, out, lse, dout)
    assert all(bool((t[:, g.shape[1]:g.shape[1] + 512] == 7.0).all()) for t, g in zip(made, grads))


@pytest.mark.parametrize("lq", [1, 40])
def test_attention_over_a_cache_past_32_bits(gpu_ctx, lq):
    """70000 keys, rows of 64 Ki elements, 2^32 + in all; heads 512 columns from the end."""
    note("long cache", lq)
    Tk, wide, D = 70000, 65536, 64
    code, ty, _ = DTS["bf16"]
    kc = torch.zeros((Tk, wide), dtype=ty, device="cuda")
    small = rand((Tk, 2 * D), "bf16", 5)
    k, v = kc[:, wide - 512:wide - 512 + D], kc[:, wide - D:]
    k.copy_(small[:, :D])
    v.copy_(small[:, D:])
    q = rand((lq, D), "bf16", 6)
    starts = [torch.tensor([0, t], dtype=torch.int32, device="cuda") for t in (lq, Tk)]
    outs = []
    for kk, vv in ((k, v), (small[:, :D].contiguous(), small[:, D:].contiguous())):
        out, lse = torch.zeros((lq, D), dtype=ty, device="cuda"), torch.zeros((1, lq), device="cuda")
        gpu_ctx.attention(q, D, kk, ld(kk), vv, ld(vv), *starts, 1, lq, Tk, 1, 1, D, out, D, lse=lse,
                          dtype=code)
        outs.append((out, lse))
    torch.cuda.synchronize()
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])
    dout, got = rand((lq, D), "bf16", 7), []
    for kk, vv in ((k, v), (small[:, :D].contiguous(), small[:, D:].contiguous())):
        dq = torch.zeros_like(q)
        dk, dv = torch.zeros_like(kc) if kk is k else torch.zeros_like(small), None
        n = dk.shape[1]
        dk, dv = dk[:, n - 2 * D:n - D], dk[:, n - D:]
        gpu_ctx.attention_bwd(q, D, kk, ld(kk), vv, ld(vv), out, D, dout, D, lse, *starts, 1, lq, Tk,
                              1, 1, D, dq, D, dk, n, dv, n, dtype=code)
        got.append((dq, dk, dv))
    torch.cuda.synchronize()
    for a, c in zip(*got):
        assert torch.equal(a, c) and bool(c.any())


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_attention_of_nothing(gpu_ctx, dt):
    """No sequences, no rows or no keys: tensors of none are NULL, and what there is of the
    others is written."""
    note("nothing", dt)
    code, ty, _ = DTS[dt]
    heads, kv, D = 4, 2, 64
    x = lambda T, h: rand((max(T, 1), h * D), dt, 3)[:T] if T else None
    for Tq, Tk in ((0, 0), (0, 70), (50, 0)):
        qs, ks = (torch.tensor([0, t], dtype=torch.int32, device="cuda") for t in (Tq, Tk))
        q, k, v = x(Tq, heads), x(Tk, kv), x(Tk, kv)
        seven = lambda t: None if t is None else torch.full_like(t, 7.0)
        out, lse = seven(q), torch.full((heads, Tq), 7.0, device="cuda") if Tq else None
        shape = (qs, ks, 1, Tq, Tk, heads, kv, D)
        gpu_ctx.attention(q, heads * D, k, kv * D, v, kv * D, *shape, out, heads * D, lse=lse,
                          dtype=code)
        dq, dk, dv = seven(q), seven(k), seven(v)
        gpu_ctx.attention_bwd(q, heads * D, k, kv * D, v, kv * D, out, heads * D, out, heads * D, lse,
                              *shape, dq, heads * D, dk, kv * D, dv, kv * D, dtype=code)
        torch.cuda.synchronize()
        for t in (out, dq, dk, dv):
            assert t is None or (t == 0).all()
        assert lse is None or (lse == -math.inf).all()
    # No sequence at all: everything is left as it is.
    q, k, v = x(50, heads), x(70, kv), x(70, kv)
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = seven(q)
    gpu_ctx.attention(q, heads * D, k, kv * D, v, kv * D, zero, zero, 0, 50, 70, heads, kv, D, out,
                      heads * D, dtype=code)
    torch.cuda.synchronize()
    assert (out == 7.0).all()


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_starts_past_the_ends_are_cut_off(gpu_ctx, dt):
    """Starts up to 2^32 - 1: the last sequence ends with the tensors, later ones are of
    nothing; nothing past the tensors is written."""
    note("starts", dt)
    b = Batch([(50, 60), (40, 30)], 4, 2, 64, dt, pad=8)
    big = lambda t: torch.cat([t[:2], torch.tensor([-1, -1, -1], dtype=torch.int32, device="cuda")])
    b.d_qs, b.d_ks = big(b.d_qs), big(b.d_ks)
    real = b.seqs
    b.seqs = real + [(0, 0), (0, 0)]
    b.qs, b.ks = b.qs + [b.Tq] * 2, b.ks + [b.Tk] * 2
    out, lse = b.forward(gpu_ctx)
    b.check_forward(out, lse)
    dout = rand((b.Tq, 256), dt, 9, pad=8)
    b.check_backward(b.backward(gpu_ctx, out, lse, dout), out, lse, dout)


@pytest.mark.parametrize("lq,lk", [(1, 700), (200, 200)])
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_scores_that_are_all_minus_infinity(gpu_ctx, dt, lq, lk):
    """A row all of whose scores are -inf has the sum 0 of a row that sees no key: 0, and
    the log of its sum -inf."""
    note("-inf", dt, lq, lk)
    b = Batch([(lq, lk)], 2, 1, 64, dt)
    b.q.abs_()
    b.q.add_(1.0)
    b.k.fill_(-math.inf)
    out, lse = b.forward(gpu_ctx)
    assert (out == 0).all() and (lse == -math.inf).all()


@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_one_tensor_as_q_k_and_v(gpu_ctx, dt):
    """Inputs may be one memory."""
    note("one tensor", dt)
    b = Batch([(100, 100), (29, 29)], 2, 2, 64, dt)
    b.k = b.v = b.q
    out, lse = b.forward(gpu_ctx)
    b.check_forward(out, lse)
    b.check_backward(b.backward(gpu_ctx, out, lse, out), out, lse, out)
