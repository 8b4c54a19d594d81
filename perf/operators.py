"""Measured cases of the token-model training operators, as a user's program
calls them through the package's public entry points.

Operators (case["op"]) and their passes (case["way"]):
  layer_norm  forward   y, mean and 1/sqrt(var + eps) of every row
              backward  dx, dgamma, dbeta from x, dy and the saved statistics
  embedding   forward   out[t] = scale * table[tokens[t]]
              backward  the table's gradient, sums over equal tokens
  ckpt8       round     a layer's pre-activation into 8 bits (the forward's
                        save) and back, with its activation (the backward's
                        load): int8 elements, one power-of-two exponent per
                        32 columns of a row
              act       dZ = dH * act'(Z) with Z held in 8 bits
              matmul    the gradients of act(Z).W from dZ with Z held in 8
                        bits: dX, dW, dbias

`own` false: elementary torch operations in fp32 (fp64 for the exact powers of
two of ckpt8).  `own` true: the library's calls.
"""
import math

import numpy as np
import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = float(np.float32(1e-5))
C0, C1 = float(np.float32(0.7978846)), float(np.float32(0.044715))  # the library's GELU
BLOCK = 32  # columns that share an exponent
WORKSPACE = 256 << 20  # reserved once per program, so that no call allocates


# ------------------------------------------------------------------- cases
def listed():
    return [
        # Serving a few sequences one token at a time: launch and latency.
        dict(name="ln_fwd_bf16_few", op="layer_norm", way="forward", dtype="bf16", rows=32,
             cols=2048, pad=0, affine=True),
        # A large training batch of wide rows: memory rate.
        dict(name="ln_fwd_bf16_large", op="layer_norm", way="forward", dtype="bf16", rows=16384,
             cols=8192, pad=0, affine=True),
        # The hidden layer of the 8-layer model (batch 2048, width 4096).
        dict(name="ln_bwd_bf16_4096", op="layer_norm", way="backward", dtype="bf16", rows=2048,
             cols=4096, pad=0, affine=True),
        # fp32 training, a large batch: the most bytes of the layer norm cases.
        dict(name="ln_bwd_f32_large", op="layer_norm", way="backward", dtype="f32", rows=16384,
             cols=4096, pad=0, affine=True),
        # Sizes that are no multiple of anything, rows that start on odd elements.
        dict(name="ln_bwd_f16_odd", op="layer_norm", way="backward", dtype="f16", rows=4099,
             cols=1531, pad=3, affine=True),
        # A batch of text looked up in a table of 32000 rows.
        dict(name="emb_fwd_bf16", op="embedding", way="forward", dtype="bf16", tokens=16384,
             vocab=32000, cols=4096, pad=0, spread="zipf"),
        # A small model's gradient over a small vocabulary: latency.
        dict(name="emb_bwd_bf16_few", op="embedding", way="backward", dtype="bf16", tokens=256,
             vocab=1000, cols=256, pad=0, spread="uniform"),
        # A training batch over a large vocabulary.
        dict(name="emb_bwd_bf16_large", op="embedding", way="backward", dtype="bf16",
             tokens=65536, vocab=131072, cols=2048, pad=0, spread="zipf"),
        # A padded batch: four tokens of ten are the same one; odd sizes.
        dict(name="emb_bwd_f32_hot", op="embedding", way="backward", dtype="f32", tokens=20011,
             vocab=50257, cols=777, pad=5, spread="hot"),
        # The hidden layer of the 8-layer model: kept in 8 bits and restored.
        dict(name="ckpt_round_bf16_4096", op="ckpt8", way="round", dtype="bf16", rows=2048,
             cols=4096, pad=0, act="gelu"),
        # An activation's gradient at odd sizes in fp32.
        dict(name="ckpt_act_f32_odd", op="ckpt8", way="act", dtype="f32", rows=3001, cols=2003,
             pad=3, act="gelu"),
        # The hidden layer's gradients from its 8-bit input: the most operations.
        dict(name="ckpt_matmul_bf16_4096", op="ckpt8", way="matmul", dtype="bf16", m=2048, n=4096,
             k=4096, act="gelu"),
    ]


MOST_BYTES = 805e6  # of the largest listed cases
MOST_MNK = 2048 * 4096 * 4096


def _size(rng, lo, hi):
    """Log-uniform in [lo, hi]; half of them rounded to a multiple of 64 (8 below 64)."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5:
        q = 64 if n >= 64 else 8
        n = max(q, n // q * q)
    return max(lo, min(hi, n))


def draw(rng):
    op = rng.choices(["layer_norm", "embedding", "ckpt8"], [40, 30, 30])[0]
    while True:
        case = dict(op=op, dtype=rng.choice(["bf16", "bf16", "f32", "f16"]),
                    pad=rng.choice([0, 0, 0, 8, rng.randint(1, 15)]))
        if op == "layer_norm":
            case.update(way=rng.choice(["forward", "backward", "backward"]),
                        rows=_size(rng, 1, 65536), cols=_size(rng, 16, 65536),
                        affine=rng.random() < 0.8)
        elif op == "embedding":
            case.update(way=rng.choice(["forward", "backward", "backward"]),
                        tokens=_size(rng, 1, 131072), vocab=_size(rng, 16, 262144),
                        cols=_size(rng, 16, 8192), spread=rng.choice(["uniform", "zipf", "hot"]))
        elif rng.random() < 0.6:
            case.update(way=rng.choice(["round", "act"]), rows=_size(rng, 1, 16384),
                        cols=_size(rng, 16, 32768), act=rng.choice(["none", "relu", "gelu"]))
        else:
            case.update(way="matmul", m=_size(rng, 16, 8192), n=_size(rng, 16, 8192),
                        k=_size(rng, 16, 8192), act=rng.choice(["none", "relu", "gelu"]), pad=0)
            # fp32 products take eight times a bf16 one's time.
            if case["m"] * case["n"] * case["k"] > MOST_MNK // (4 if case["dtype"] == "f32" else 1):
                continue
        if _bytes(case) <= MOST_BYTES:
            return case


# ------------------------------------------------------------------ inputs
class _Rand:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(int(seed))

    def normal(self, rows, cols, dtype, std=1.0, mean=0.0, pad=0):
        """A rows x cols view of rows that lie cols + pad elements apart."""
        t = torch.empty((rows, cols + pad), device="cuda").normal_(mean, std, generator=self.g)
        return t.to(DT[dtype])[:, :cols]

    def tokens(self, n, vocab, spread):
        p = torch.from_numpy(_token_cdf(vocab, spread)).cuda()
        u = torch.rand(n, device="cuda", generator=self.g, dtype=torch.float64)
        rank = torch.searchsorted(p, u).clamp_(max=vocab - 1)
        order = torch.randperm(vocab, device="cuda", generator=self.g)
        return order[rank].to(torch.int32)


def _token_p(vocab, spread):
    """Token probabilities by rank: uniform, 1 / (rank + 2.7) as in text, or
    that with four tenths of the batch on one (padding) token."""
    if spread == "uniform":
        return np.full(vocab, 1.0 / vocab)
    p = 1.0 / (np.arange(vocab) + 2.7)
    p /= p.sum()
    if spread == "hot":
        p *= 0.6
        p[0] += 0.4
    return p


def _token_cdf(vocab, spread):
    return np.cumsum(_token_p(vocab, spread))


def _empty(rows, cols, dtype, pad=0):
    return torch.empty((rows, cols + pad), device="cuda", dtype=DT[dtype])[:, :cols]


def _ld(t):
    return t.stride(0)


def _padded_blocks(x):
    """x as [rows, blocks, BLOCK], zeros past the last column."""
    rows, cols = x.shape
    nb = -(-cols // BLOCK)
    return torch.nn.functional.pad(x, (0, nb * BLOCK - cols)).reshape(rows, nb, BLOCK)


def _pow2(e):
    """2^e in fp64, exact, from int64 exponents."""
    return ((e + 1023) << 52).view(torch.float64)


def _quantise(x):
    """(int8 [rows, cols], exponent bytes [rows, blocks]) of x."""
    xb = _padded_blocks(x.float())
    bits = xb.abs().amax(-1).view(torch.int32).to(torch.int64)
    b = (bits >> 23).clamp_(min=1)
    q = torch.round(xb.double() * _pow2(133 - b)[..., None]).clamp_(-127, 127)
    return q.to(torch.int8).reshape(x.shape[0], -1)[:, :x.shape[1]], b.to(torch.uint8)


def _dequantise(q, b):
    """The values that q and b stand for, fp32 (every one is exact)."""
    z = _padded_blocks(q).double() * _pow2(b.to(torch.int64) - 133)[..., None]
    return z.reshape(q.shape[0], -1)[:, :q.shape[1]].float()


def _gelu_s(z):
    return 1.0 / (1.0 + torch.exp(-2.0 * (C0 * (z + C1 * z * z * z))))


def _act(act, z):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    return z * _gelu_s(z) if act == "gelu" else z


def _act_grad(act, z):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        s = _gelu_s(z)
        return s + 2.0 * z * s * (1.0 - s) * C0 * (1.0 + 3.0 * C1 * z * z)
    return torch.ones_like(z)


def _inputs(case, seed):
    r, d, pad = _Rand(seed), case["dtype"], case.get("pad", 0)
    if case["op"] == "layer_norm":
        R, C = case["rows"], case["cols"]
        # A residual stream: rows with a mean, columns of unlike size.
        t = dict(x=r.normal(R, C, d, 1.0, 0.5, pad))
        t["x"] *= r.normal(1, C, d, 0.3, 1.0)
        if case["affine"]:
            t["gamma"] = r.normal(1, C, d, 0.1, 1.0)[0]
            t["beta"] = r.normal(1, C, d, 0.1)[0]
        if case["way"] == "backward":
            t["dy"] = r.normal(R, C, d, 1.0, 0.0, pad)
            x = t["x"].float()
            t["mean"] = x.mean(1)
            t["rstd"] = 1.0 / torch.sqrt(
                (x - t["mean"][:, None]).square().mean(1) + EPS)
    elif case["op"] == "embedding":
        T, V, C = case["tokens"], case["vocab"], case["cols"]
        t = dict(tokens=r.tokens(T, V, case["spread"]), scale=float(np.float32(math.sqrt(C))))
        if case["way"] == "forward":
            t["table"] = r.normal(V, C, d, 0.02, 0.0, pad)
        else:
            t["dout"] = r.normal(T, C, d, 1.0, 0.0, pad)
    elif case["way"] == "round":
        t = dict(x=r.normal(case["rows"], case["cols"], d, 1.0, 0.0, pad))
    elif case["way"] == "act":
        q, b = _quantise(r.normal(case["rows"], case["cols"], d))
        t = dict(q=q.contiguous(), b=b, dh=r.normal(case["rows"], case["cols"], d, 1.0, 0.0, pad))
    else:
        m, n, k = case["m"], case["n"], case["k"]
        q, b = _quantise(r.normal(m, k, d))
        w = torch.empty((k, n), device="cuda").uniform_(-1.0, 1.0, generator=r.g)
        t = dict(q=q.contiguous(), b=b, w=(w * math.sqrt(6.0 / k)).to(DT[d]),
                 dz=r.normal(m, n, d))
    return t


_CTX = []


def _context():
    """The program's one context (its stream is torch's current one)."""
    if not _CTX:
        from ferrograd_amd import graph as G

        c = G.GpuContext.new(0).ctx
        c.reserve_workspace(WORKSPACE)
        _CTX.append(c)
    return _CTX[0]


def prepare(case, seed):
    if own:
        _context()  # first: it makes its stream torch's current one
    t = _inputs(case, seed)
    t["case"] = case
    if not own:
        return t
    import ferrograd_amd as fa

    d, pad = case["dtype"], case.get("pad", 0)
    t["ctx"] = _context()
    t["code"] = {"f32": fa.DTYPE_F32, "f16": fa.DTYPE_F16, "bf16": fa.DTYPE_BF16}[d]
    if "act" in case:
        t["act"] = {"none": fa.ACT_NONE, "relu": fa.ACT_RELU, "gelu": fa.ACT_GELU}[case["act"]]
    if case["op"] == "layer_norm":
        R, C = case["rows"], case["cols"]
        if case["way"] == "forward":
            t["y"] = _empty(R, C, d, pad)
            t["mean"], t["rstd"] = (torch.empty(R, device="cuda") for _ in range(2))
        else:
            t["dx"] = _empty(R, C, d, pad)
            if case["affine"]:
                t["dgamma"], t["dbeta"] = (_empty(1, C, d)[0] for _ in range(2))
    elif case["op"] == "embedding":
        if case["way"] == "forward":
            t["out"] = _empty(case["tokens"], case["cols"], d, pad)
        else:
            t["dtable"] = _empty(case["vocab"], case["cols"], d, pad)
    elif case["way"] == "round":
        R, C = case["rows"], case["cols"]
        t["q"] = torch.empty((R, C), device="cuda", dtype=torch.int8)
        t["b"] = torch.empty((R, -(-C // BLOCK)), device="cuda", dtype=torch.uint8)
        t["z"], t["h"] = _empty(R, C, d, pad), _empty(R, C, d, pad)
    elif case["way"] == "act":
        t["dz"] = _empty(case["rows"], case["cols"], d, pad)
    else:
        m, n, k = case["m"], case["n"], case["k"]
        t["zr"], t["xr"], t["dx"] = (_empty(m, k, d) for _ in range(3))
        t["dw"], t["db"] = _empty(k, n, d), _empty(1, n, d)[0]
    return t


# --------------------------------------------------------------------- run
def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    c, ctx, dt = s["case"], s["ctx"], s["code"]
    if c["op"] == "layer_norm":
        R, C = c["rows"], c["cols"]
        if c["way"] == "forward":
            ctx.layer_norm(s["x"], _ld(s["x"]), R, C, s["y"], _ld(s["y"]), gamma=s.get("gamma"),
                           beta=s.get("beta"), eps=EPS, mean=s["mean"], rstd=s["rstd"], dtype=dt)
            return s["y"], s["mean"], s["rstd"]
        ctx.layer_norm_bwd(s["x"], _ld(s["x"]), s["dy"], _ld(s["dy"]), s["mean"], s["rstd"], R, C,
                           gamma=s.get("gamma"), dx=s["dx"], lddx=_ld(s["dx"]),
                           dgamma=s.get("dgamma"), dbeta=s.get("dbeta"), dtype=dt)
        return (s["dx"], s["dgamma"], s["dbeta"]) if c["affine"] else (s["dx"],)
    if c["op"] == "embedding":
        T, V, C = c["tokens"], c["vocab"], c["cols"]
        if c["way"] == "forward":
            ctx.embedding(s["tokens"], T, V, C, s["table"], _ld(s["table"]), s["out"],
                          _ld(s["out"]), scale=s["scale"], dtype=dt)
            return s["out"]
        ctx.embedding_bwd(s["tokens"], T, V, C, s["dout"], _ld(s["dout"]), s["dtable"],
                          _ld(s["dtable"]), scale=s["scale"], dtype=dt)
        return s["dtable"]
    q, b = s["q"], s["b"]
    if c["way"] == "round":
        R, C = c["rows"], c["cols"]
        ctx.ckpt8_save(s["x"], _ld(s["x"]), R, C, q, _ld(q), b, _ld(b), dtype=dt)
        ctx.ckpt8_load(q, _ld(q), b, _ld(b), R, C, z=s["z"], ldz=_ld(s["z"]), h=s["h"],
                       ldh=_ld(s["h"]), act=s["act"], dtype=dt)
        return s["z"], s["h"]
    if c["way"] == "act":
        ctx.act_bwd_ckpt8(s["act"], s["dh"], _ld(s["dh"]), q, _ld(q), b, _ld(b), c["rows"],
                          c["cols"], s["dz"], _ld(s["dz"]), dtype=dt)
        return s["dz"]
    m, n, k = c["m"], c["n"], c["k"]
    ctx.matmul_bwd_ckpt8(m, n, k, q, _ld(q), b, _ld(b), s["w"], n, s["dz"], n, s["xr"], s["dx"], k,
                         s["dw"], n, Zr=s["zr"], dbias=s["db"], act=s["act"], dtype=dt)
    return s["dx"], s["dw"], s["db"]


def _run_plain(s):
    c = s["case"]
    d = DT[c["dtype"]]
    if c["op"] == "layer_norm":
        x = s["x"].float()
        if c["way"] == "forward":
            mean = x.mean(1)
            xc = x - mean[:, None]
            rstd = 1.0 / torch.sqrt(xc.square().mean(1) + EPS)
            y = xc * rstd[:, None]
            if c["affine"]:
                y = y * s["gamma"].float() + s["beta"].float()
            return y.to(d), mean, rstd
        rstd = s["rstd"][:, None]
        xh = (x - s["mean"][:, None]) * rstd
        dy = s["dy"].float()
        g = dy * s["gamma"].float() if c["affine"] else dy
        dx = rstd * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
        if not c["affine"]:
            return (dx.to(d),)
        return dx.to(d), (dy * xh).sum(0).to(d), dy.sum(0).to(d)
    if c["op"] == "embedding":
        tok = s["tokens"].long()
        if c["way"] == "forward":
            return (s["table"][tok].float() * s["scale"]).to(d)
        g = torch.zeros((c["vocab"], c["cols"]), device="cuda")
        g.index_add_(0, tok, s["dout"].float())
        return (g * s["scale"]).to(d)
    if c["way"] == "round":
        z = _dequantise(*_quantise(s["x"]))
        return z.to(d), _act(c["act"], z).to(d)
    z = _dequantise(s["q"], s["b"])
    if c["way"] == "act":
        return (s["dh"].float() * _act_grad(c["act"], z)).to(d)
    dz = s["dz"].float()
    dx = (dz @ s["w"].float().t()) * _act_grad(c["act"], z)
    dw = _act(c["act"], z).t() @ dz
    return dx.to(d), dw.to(d), dz.sum(0).to(d)


# -------------------------------------------------------------------- work
def _distinct(case):
    """Expected number of distinct tokens of the batch."""
    p = _token_p(case["vocab"], case["spread"])
    return float(-np.expm1(case["tokens"] * np.log1p(-np.minimum(p, 1 - 1e-12))).sum())


def _bytes(case):
    e = SIZE[case["dtype"]]
    if case["op"] == "layer_norm":
        R, C = case["rows"], case["cols"]
        if case["way"] == "forward":
            return 2 * R * C * e + 8 * R + (2 * C * e if case["affine"] else 0)
        return 3 * R * C * e + 8 * R + (3 * C * e if case["affine"] else 0)
    if case["op"] == "embedding":
        T, V, C = case["tokens"], case["vocab"], case["cols"]
        if case["way"] == "forward":
            return 4 * T + T * C * e + int(_distinct(case)) * C * e
        return 4 * T + T * C * e + V * C * e
    if case["way"] == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        return m * k * (1 + 1 / BLOCK) + (m * k + 2 * k * n + m * n + n) * e
    held = 1 + 1 / BLOCK
    R, C = case["rows"], case["cols"]
    return R * C * (3 * e + 2 * held if case["way"] == "round" else 2 * e + held)


def work(case):
    if case["op"] == "layer_norm":
        flops = case["rows"] * case["cols"] * (7 if case["way"] == "forward" else 14)
    elif case["op"] == "embedding":
        flops = case["tokens"] * case["cols"]
    elif case["way"] == "matmul":
        flops = 4 * case["m"] * case["n"] * case["k"]
    else:
        flops = 4 * case["rows"] * case["cols"]
    return {"bytes": _bytes(case), "flops": flops}


# ------------------------------------------------------------------- exact
def exact(case, seed):
    t = _inputs(case, seed)
    f = torch.float64
    if case["op"] == "layer_norm":
        x = t["x"].to(f)
        C = x.shape[1]
        if case["way"] == "forward":
            mean = x.sum(1) / C
            x = x - mean[:, None]
            rstd = torch.rsqrt((x * x).sum(1) / C + EPS)
            y = x * rstd[:, None]
            if case["affine"]:
                y = torch.addcmul(t["beta"].to(f), y, t["gamma"].to(f))
            return y, mean, rstd
        rstd = t["rstd"].to(f)[:, None]
        xh = (x - t["mean"].to(f)[:, None]) * rstd
        dy = t["dy"].to(f)
        g = dy * t["gamma"].to(f) if case["affine"] else dy
        dx = rstd * (g - (g.sum(1)[:, None] + xh * (g * xh).sum(1)[:, None]) / C)
        if not case["affine"]:
            return (dx,)
        return dx, (dy * xh).sum(0), dy.sum(0)
    if case["op"] == "embedding":
        tok = t["tokens"].long()
        if case["way"] == "forward":
            return torch.index_select(t["table"], 0, tok).to(f) * t["scale"]
        out = torch.zeros((case["vocab"], case["cols"]), device="cuda", dtype=f)
        for k in range(0, case["tokens"], 16384):
            out.index_add_(0, tok[k:k + 16384], t["dout"][k:k + 16384].to(f), alpha=t["scale"])
        return out

    def gelu(z):
        return 0.5 * z * (1.0 + torch.tanh(C0 * (z + C1 * z ** 3)))

    def gelu_grad(z):
        th = torch.tanh(C0 * (z + C1 * z ** 3))
        return 0.5 * (1.0 + th) + 0.5 * z * (1.0 - th * th) * C0 * (1.0 + 3.0 * C1 * z * z)

    def values(q, e):
        e = e.double().repeat_interleave(BLOCK, 1)[:, :q.shape[1]]
        return q.double() * torch.exp2(e - 133.0)

    act = case["act"]
    if case["way"] == "round":
        x = t["x"].to(f)
        z = torch.empty_like(x)
        for k in range(0, x.shape[1], BLOCK):
            xb = x[:, k:k + BLOCK]
            top = xb.abs().amax(1)
            m = torch.frexp(top)[0]  # top / m is the power of two above top, exactly
            step = torch.where(m > 0, top / m, 0.0).clamp(min=2.0 ** -125)[:, None] * 2.0 ** -7
            z[:, k:k + BLOCK] = (xb / step).round().clamp(-127, 127) * step
    else:
        z = values(t["q"], t["b"])
    if act == "gelu":
        h, dh = (gelu(z) if case["way"] != "act" else None), gelu_grad(z)
    elif act == "relu":
        h, dh = z.clamp(min=0.0), (z > 0).to(f)
    else:
        h, dh = z, torch.ones_like(z)
    if case["way"] == "round":
        return z, h
    if case["way"] == "act":
        return t["dh"].to(f) * dh
    dz = t["dz"].to(f)
    return torch.mm(dz, t["w"].to(f).t().contiguous()) * dh, torch.mm(h.t().contiguous(), dz), dz.sum(0)
