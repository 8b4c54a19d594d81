"""Measured cases of a transformer block's operators, as a user's program calls
them through the package's public entry points.

Operators (case["op"]) and their passes (case["way"]):
  attention  forward   packed sequences of different lengths, grouped heads,
                       causal or not; out and the log of each row's sum.  Single
                       tokens over a cache with room are the same call
             backward  dq, dk, dv from out, dout and those logs
  rms_norm   forward   s = x + r (the residual), y = s * rstd * gamma, and y in
                       8 bits where asked (int8 elements, one power-of-two
                       exponent per 32 columns of a row), returned as its values
             backward  dx (with the residual's own gradient added) and dgamma
  logprobs   forward   log probability of each row's token, entropy, log of the
                       row's sum, the most probable tokens in order
             backward  dlogits from the gradients of log probability and entropy

`own` false: elementary torch operations in fp32.  `own` true: the library's calls.
"""
import math
import random

import numpy as np
import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = float(np.float32(1e-5))
BLOCK = 32  # columns that share an exponent
WORKSPACE = 512 << 20  # reserved once per program, so that no call allocates


# ------------------------------------------------------------------- cases
def _att(way, dtype, n, lq, past, heads, kv, dim, **more):
    """n sequences of at most lq new tokens after at most `past` earlier ones;
    spread "mixed": lengths from 1 up, the first the longest; room: keys lie in a
    cache with as many rows for every sequence; pad: elements between rows."""
    case = dict(op="attention", way=way, dtype=dtype, n=n, lq=lq, past=past, heads=heads, kv=kv,
                dim=dim, causal=True, spread="mixed", room=False, pad=0)
    case.update(more)
    return case


def listed():
    return [
        # A short prompt on a small model: latency.
        dict(name="att_fwd_bf16_small", **_att("forward", "bf16", 1, 64, 0, 8, 8, 64)),
        # Serving 64 sequences one token at a time over a cache of up to 8192: memory rate.
        dict(name="att_token_bf16", **_att("forward", "bf16", 64, 1, 8191, 32, 8, 128, room=True)),
        # Prompts of up to 4096 tokens packed into one batch, 4096 wide: the matrix units.
        dict(name="att_fwd_bf16_packed", **_att("forward", "bf16", 8, 4096, 0, 32, 8, 128)),
        # Its training pass: the most operations.
        dict(name="att_bwd_bf16_packed", **_att("backward", "bf16", 8, 4096, 0, 32, 8, 128)),
        # Odd heads and lengths, bidirectional, rows off every boundary, fp32.
        dict(name="att_bwd_f32_odd", **_att("backward", "f32", 5, 777, 0, 6, 3, 72, causal=False,
                                            pad=3)),
        # A decoder layer's norm while serving a few sequences: latency.
        dict(name="rms_fwd_bf16_few", op="rms_norm", way="forward", dtype="bf16", rows=32, cols=4096,
             pad=0, residual=True, bits8=False),
        # A training batch's norm, kept in 8 bits for the backward of the product after it.
        dict(name="rms_fwd_bf16_8bit", op="rms_norm", way="forward", dtype="bf16", rows=16384,
             cols=4096, pad=0, residual=True, bits8=True),
        # The backward of such a batch in fp32, odd sizes.
        dict(name="rms_bwd_f32_odd", op="rms_norm", way="backward", dtype="f32", rows=4099,
             cols=2051, pad=1, residual=True, bits8=False),
        # The same in 16 bits over whole rows: memory rate.
        dict(name="rms_bwd_bf16", op="rms_norm", way="backward", dtype="bf16", rows=16384,
             cols=4096, pad=0, residual=True, bits8=False),
        # Serving: 64 tokens' log probabilities with 20 alternatives over 131072.
        dict(name="lp_fwd_bf16_token", op="logprobs", way="forward", dtype="bf16", rows=64,
             cols=131072, pad=0, top=20, scale=1.25),
        # Scoring a batch of text over an odd vocabulary.
        dict(name="lp_fwd_f32_batch", op="logprobs", way="forward", dtype="f32", rows=4096,
             cols=50257, pad=0, top=5, scale=1.0),
        # The gradient of a policy's objective with an entropy bonus; a quarter of the rows padded.
        dict(name="lp_bwd_bf16_batch", op="logprobs", way="backward", dtype="bf16", rows=8192,
             cols=32000, pad=0, top=0, scale=1.0),
    ]


MOST_SCORES = 1.1e9  # of a padded batch's scores: one head's rows times keys, all heads
MOST_FLOPS = {"bf16": 8e11, "f16": 8e11, "f32": 1e11}
MOST_BYTES = 840e6


def _size(rng, lo, hi):
    """Log-uniform in [lo, hi]; half of them rounded to a multiple of 64 (8 below 64)."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5:
        q = 64 if n >= 64 else 8
        n = max(q, n // q * q)
    return max(lo, min(hi, n))


def draw(rng):
    op = rng.choices(["attention", "rms_norm", "logprobs"], [50, 25, 25])[0]
    while True:
        dtype = rng.choice(["bf16", "bf16", "f32", "f16"])
        way = rng.choice(["forward", "backward"])
        pad = rng.choice([0, 0, 0, 8, rng.randint(1, 15)])
        if op == "attention":
            kv = rng.randint(1, 8)
            token = way == "forward" and rng.random() < 0.4
            case = _att(way, dtype, _size(rng, 1, 64), rng.choice([1, 1, 1, 4]) if token
                        else _size(rng, 1, 4096),
                        _size(rng, 1, 16384) if token else rng.choice([0, 0, _size(rng, 1, 4096)]),
                        kv * rng.choice([1, 2, 3, 4, 8]), kv,
                        rng.choice([64, 128, 128, 32, 80, 96, rng.randint(1, 128)]),
                        causal=rng.random() < 0.75, spread=rng.choice(["mixed", "equal"]),
                        room=token and rng.random() < 0.7, pad=pad)
            scores = case["n"] * case["heads"] * case["lq"] * (case["lq"] + case["past"])
            if scores > MOST_SCORES or work(case)["flops"] > MOST_FLOPS[dtype]:
                continue
        elif op == "rms_norm":
            bits8 = way == "forward" and dtype != "f32" and rng.random() < 0.5
            case = dict(op=op, way=way, dtype=dtype, rows=_size(rng, 1, 65536),
                        cols=_size(rng, 16, 32768), pad=pad, residual=rng.random() < 0.7,
                        bits8=bits8)
        else:
            case = dict(op=op, way=way, dtype=dtype, rows=_size(rng, 1, 16384),
                        cols=_size(rng, 32, 262144), pad=pad,
                        top=rng.choice([0, 1, 5, 20, 32]) if way == "forward" else 0,
                        scale=rng.choice([1.0, 1.25, 0.5]))
        if work(case)["bytes"] <= MOST_BYTES:
            return case


def _lengths(case):
    """(queries, keys) of each sequence, from the case alone."""
    n, lq, past = case["n"], case["lq"], case["past"]
    rng = random.Random(n * 7919 + lq * 31 + past)
    mixed = case["spread"] == "mixed"
    q = [rng.randint(1, lq) if mixed and k else lq for k in range(n)]
    return q, [a + (rng.randint(0, past) if mixed and k else past) for k, a in enumerate(q)]


def _starts(lens):
    return [0] + list(np.cumsum(lens).tolist())


# ------------------------------------------------------------------ inputs
class _Rand:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(int(seed))

    def normal(self, rows, cols, dtype, std=1.0, mean=0.0, pad=0):
        """A rows x cols view of rows that lie cols + pad elements apart."""
        t = torch.empty((rows, cols + pad), device="cuda").normal_(mean, std, generator=self.g)
        return t.to(DT[dtype])[:, :cols]

    def tokens(self, logits):
        """A token of each row, drawn with the row's probabilities."""
        u = torch.rand(logits.shape, device="cuda", generator=self.g).clamp_(1e-20, 1.0)
        return (logits.float() - torch.log(-torch.log(u))).argmax(1).to(torch.int32)


def _empty(rows, cols, dtype, pad=0):
    return torch.empty((rows, cols + pad), device="cuda", dtype=DT[dtype])[:, :cols]


def _ld(t):
    return t.stride(0)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _attention_inputs(case, r):
    d, pad, D = case["dtype"], case["pad"], case["dim"]
    wide, kvw = case["heads"] * D, case["kv"] * D
    lq, lk = _lengths(case)
    Tq = sum(lq)
    t = dict(qs=_ints(_starts(lq)), Tq=Tq, lens=None, maxq=max(lq), maxk=max(lk))
    if case["room"]:  # a cache of as many rows for each, uninitialised past a sequence's keys
        cap = max(lk) + 5
        t["Tk"] = cap * case["n"]
        t["ks"], t["lens"] = _ints([cap * k for k in range(case["n"] + 1)]), _ints(lk)
        dead = torch.arange(t["Tk"], device="cuda") % cap >= t["lens"].repeat_interleave(cap)
        t["q"] = r.normal(Tq, wide, d, pad=pad)
        t["k"], t["v"] = (r.normal(t["Tk"], kvw, d, pad=pad) for _ in range(2))
        t["k"][dead], t["v"][dead] = float("nan"), float("nan")
    elif case["past"]:
        t["Tk"], t["ks"] = sum(lk), _ints(_starts(lk))
        t["q"] = r.normal(Tq, wide, d, pad=pad)
        t["k"], t["v"] = (r.normal(t["Tk"], kvw, d, pad=pad) for _ in range(2))
    else:  # one projection's output holds all three
        t["Tk"], t["ks"] = Tq, t["qs"]
        x = r.normal(Tq, wide + 2 * kvw, d, pad=pad)
        t["q"], t["k"], t["v"] = x[:, :wide], x[:, wide:wide + kvw], x[:, wide + kvw:]
    t["scale"] = float(np.float32(1.0 / math.sqrt(D)))
    if case["way"] == "backward":
        t["case"] = case
        out, t["lse"] = _attention_plain(t)
        t["out"] = _empty(Tq, wide, d, pad)
        t["out"].copy_(out)
        t["dout"] = r.normal(Tq, wide, d, pad=pad)
    return t


def _inputs(case, seed):
    r, d, pad = _Rand(seed), case["dtype"], case["pad"]
    if case["op"] == "attention":
        return _attention_inputs(case, r)
    R, C = case["rows"], case["cols"]
    if case["op"] == "rms_norm":
        t = dict(x=r.normal(R, C, d, 1.0, 0.0, pad), gamma=r.normal(1, C, d, 0.1, 1.0)[0])
        if case["way"] == "forward":
            if case["residual"]:
                t["r"] = r.normal(R, C, d, 2.0, 0.0, pad)
            return t
        t["dy"] = r.normal(R, C, d, 1.0, 0.0, pad)
        t["rstd"] = 1.0 / torch.sqrt(t["x"].float().square().mean(1) + EPS)
        if case["residual"]:
            t["ds"] = r.normal(R, C, d, 1.0, 0.0, pad)
        return t
    t = dict(x=r.normal(R, C, d, 3.0, 0.0, pad))
    t["tokens"] = r.tokens(t["x"])
    if case["way"] == "backward":
        _, t["entropy"], t["lse"] = _row_stats(t["x"].float() * case["scale"], t["tokens"])
        live = torch.rand(R, device="cuda", generator=r.g) < 0.75
        t["dlogp"] = torch.randn(R, device="cuda", generator=r.g) * live
        t["dentropy"] = 0.01 * live.float()
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

    d, pad = case["dtype"], case["pad"]
    t["ctx"] = _context()
    t["code"] = {"f32": fa.DTYPE_F32, "f16": fa.DTYPE_F16, "bf16": fa.DTYPE_BF16}[d]
    if case["op"] == "attention":
        wide, kvw = case["heads"] * case["dim"], case["kv"] * case["dim"]
        if case["way"] == "forward":
            t["out"] = _empty(t["Tq"], wide, d, pad)
            t["lse"] = torch.empty((case["heads"], t["Tq"]), device="cuda")
        else:
            t["dq"] = _empty(t["Tq"], wide, d, pad)
            t["dk"], t["dv"] = (_empty(t["Tk"], kvw, d, pad) for _ in range(2))
        return t
    R, C = case["rows"], case["cols"]
    if case["op"] == "rms_norm":
        if case["way"] == "forward":
            t["y"], t["rstd"] = _empty(R, C, d, pad), torch.empty(R, device="cuda")
            if case["residual"]:
                t["s"] = _empty(R, C, d, pad)
            if case["bits8"]:
                t["q"] = torch.empty((R, C), device="cuda", dtype=torch.int8)
                t["e"] = torch.empty((R, -(-C // BLOCK)), device="cuda", dtype=torch.uint8)
                t["z"] = _empty(R, C, d, pad)
        else:
            t["dx"], t["dgamma"] = _empty(R, C, d, pad), _empty(1, C, d)[0]
    elif case["way"] == "forward":
        t["logp"], t["entropy"], t["lse"] = (torch.empty(R, device="cuda") for _ in range(3))
        if case["top"]:
            t["ids"] = torch.empty((R, case["top"]), device="cuda", dtype=torch.int32)
            t["tops"] = torch.empty((R, case["top"]), device="cuda")
    else:
        t["dx"] = _empty(R, C, d, pad)
    return t


# --------------------------------------------------------------------- run
def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    c, ctx, dt = s["case"], s["ctx"], s["code"]
    if c["op"] == "attention":
        shape = (s["qs"], s["ks"], c["n"], s["Tq"], s["Tk"], c["heads"], c["kv"], c["dim"])
        qkv = (s["q"], _ld(s["q"]), s["k"], _ld(s["k"]), s["v"], _ld(s["v"]))
        if c["way"] == "forward":
            ctx.attention(*qkv, *shape, s["out"], _ld(s["out"]), k_lens=s["lens"],
                          scale=s["scale"], causal=c["causal"], lse=s["lse"], dtype=dt)
            return s["out"], s["lse"]
        ctx.attention_bwd(*qkv, s["out"], _ld(s["out"]), s["dout"], _ld(s["dout"]), s["lse"],
                          *shape, s["dq"], _ld(s["dq"]), s["dk"], _ld(s["dk"]), s["dv"],
                          _ld(s["dv"]), scale=s["scale"], causal=c["causal"], dtype=dt)
        return s["dq"], s["dk"], s["dv"]
    R, C, x = c["rows"], c["cols"], s["x"]
    if c["op"] == "rms_norm":
        if c["way"] == "backward":
            ds = s.get("ds")
            ctx.rms_norm_bwd(x, _ld(x), s["dy"], _ld(s["dy"]), s["rstd"], R, C, gamma=s["gamma"],
                             ds=ds, ldds=_ld(ds) if c["residual"] else 0, dx=s["dx"],
                             lddx=_ld(s["dx"]), dgamma=s["dgamma"], dtype=dt)
            return s["dx"], s["dgamma"]
        add = dict(r=s["r"], ldr=_ld(s["r"]), s=s["s"], lds=_ld(s["s"])) if c["residual"] else {}
        held = dict(q=s["q"], ldq=C, e=s["e"], lde=_ld(s["e"])) if c["bits8"] else {}
        ctx.rms_norm(x, _ld(x), R, C, s["y"], _ld(s["y"]), gamma=s["gamma"], eps=EPS,
                     rstd=s["rstd"], dtype=dt, **add, **held)
        if c["bits8"]:
            ctx.ckpt8_load(s["q"], C, s["e"], _ld(s["e"]), R, C, z=s["z"], ldz=_ld(s["z"]),
                           dtype=dt)
        return s["y"], s["rstd"], s.get("s"), s.get("z")
    if c["way"] == "forward":
        ctx.token_logprobs(x, _ld(x), s["tokens"], R, C, logp=s["logp"], entropy=s["entropy"],
                           lse=s["lse"], top=c["top"], top_ids=s.get("ids"),
                           top_logp=s.get("tops"), scale=c["scale"], dtype=dt)
        return s["logp"], s["entropy"], s["lse"], s.get("ids"), s.get("tops")
    ctx.token_logprobs_bwd(x, _ld(x), s["tokens"], R, C, s["lse"], s["dx"], _ld(s["dx"]),
                           entropy=s["entropy"], dlogp=s["dlogp"], dentropy=s["dentropy"],
                           scale=c["scale"], dtype=dt)
    return s["dx"]


def _padded(x, starts, lens, longest, heads, group):
    """Rows of the sequences as [n, heads, longest * group, D], fp32, zeros past each."""
    at = torch.arange(longest, device="cuda")
    alive = at < lens[:, None]
    idx = torch.where(alive, starts[:, None] + at, 0)
    y = torch.where(alive[..., None], x[idx].float(), 0.0)
    n, D = len(lens), x.shape[1] // (heads * group)
    y = y.view(n, longest, heads, group, D).permute(0, 2, 1, 3, 4)
    return y.reshape(n, heads, longest * group, D)


def _packed(y, starts, rows, group):
    """_padded's inverse: one row per token of `rows`."""
    n, heads, m, D = y.shape
    y = y.view(n, heads, m // group, group, D).permute(0, 2, 1, 3, 4)
    y = y.reshape(n * (m // group), heads * group * D)
    row = torch.arange(rows, device="cuda")
    seq = torch.searchsorted(starts[1:].contiguous(), row, right=True)
    return y[seq * (m // group) + row - starts[seq]]


def _attention_parts(s):
    c = s["case"]
    G = c["heads"] // c["kv"]
    qs, ks = s["qs"].long(), s["ks"].long()
    lq = qs[1:] - qs[:-1]
    lk = s["lens"].long() if s["lens"] is not None else ks[1:] - ks[:-1]
    q = _padded(s["q"], qs[:-1], lq, s["maxq"], c["kv"], G)
    k = _padded(s["k"], ks[:-1], lk, s["maxk"], c["kv"], 1)
    v = _padded(s["v"], ks[:-1], lk, s["maxk"], c["kv"], 1)
    i, j = torch.arange(s["maxq"], device="cuda")[:, None], torch.arange(s["maxk"], device="cuda")
    see = (i < lq[:, None, None]) & (j < lk[:, None, None])
    if c["causal"]:
        see = see & (j <= i + (lk - lq)[:, None, None])
    see = see.repeat_interleave(G, 1)[:, None]
    sc = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(s["scale"])
    return G, qs, ks, lq, lk, q, k, v, see, sc.masked_fill_(~see, -math.inf)


def _attention_plain(s):
    c = s["case"]
    G, qs, _, _, _, _, _, v, _, sc = _attention_parts(s)
    m = sc.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    p = sc.sub_(m).exp_()
    l = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / torch.where(l == 0, 1.0, l)
    lse = _packed(m + torch.log(l), qs, s["Tq"], G)
    return _packed(out, qs, s["Tq"], G).to(DT[c["dtype"]]), lse.t().contiguous()


def _attention_bwd_plain(s):
    d = DT[s["case"]["dtype"]]
    kv = s["case"]["kv"]
    G, qs, ks, lq, lk, q, k, v, see, p = _attention_parts(s)
    lse = _padded(s["lse"].t(), qs[:-1], lq, s["maxq"], kv, G)
    p = p.sub_(torch.where(lse == -math.inf, 0.0, lse)).exp_()
    do = _padded(s["dout"], qs[:-1], lq, s["maxq"], kv, G)
    o = _padded(s["out"], qs[:-1], lq, s["maxq"], kv, G)
    dv = torch.matmul(p.transpose(-1, -2).contiguous(), do)
    dp = torch.matmul(do, v.transpose(-1, -2).contiguous())
    ds = dp.sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(s["scale"])
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(-1, -2).contiguous(), q)
    return (_packed(dq, qs, s["Tq"], G).to(d), _packed(dk, ks, s["Tk"], 1).to(d),
            _packed(dv, ks, s["Tk"], 1).to(d))


def _row_stats(z, tokens):
    """Log probability of each row's token, entropy, log of the sum of exponentials."""
    m = z.amax(1, keepdim=True)
    z = z - m
    e = torch.exp(z)
    total = e.sum(1)
    log = torch.log(total)
    at = torch.gather(z, 1, tokens.long()[:, None])[:, 0]
    return at - log, log - (e * z).sum(1) / total, m[:, 0] + log


def _top(x, k):
    """Columns of the k largest of each row, the lowest column first among equals."""
    bits = (x + 0.0).view(torch.int32)
    key = torch.where(bits < 0, bits ^ 0x7fffffff, bits).long()
    key = (key << 32) - torch.arange(x.shape[1], device="cuda")
    return torch.topk(key, k, dim=1, sorted=True)[1]


def _exponents(y):
    """The exponent bytes of y's blocks and y as [rows, blocks, BLOCK], zeros past the last column."""
    rows, cols = y.shape
    nb = -(-cols // BLOCK)
    yb = torch.nn.functional.pad(y, (0, nb * BLOCK - cols)).reshape(rows, nb, BLOCK)
    return (yb.abs().amax(-1).float().view(torch.int32) >> 23).clamp_(min=1).long(), yb


def _run_plain(s):
    c = s["case"]
    d = DT[c["dtype"]]
    if c["op"] == "attention":
        return _attention_plain(s) if c["way"] == "forward" else _attention_bwd_plain(s)
    x = s["x"].float()
    if c["op"] == "rms_norm":
        if c["way"] == "backward":
            rstd = s["rstd"][:, None]
            xh = x * rstd
            dy = s["dy"].float()
            g = dy * s["gamma"].float()
            dx = rstd * (g - xh * (g * xh).mean(1, keepdim=True))
            if c["residual"]:
                dx = dx + s["ds"].float()
            return dx.to(d), (dy * xh).sum(0).to(d)
        kept = None
        if c["residual"]:
            kept = (x + s["r"].float()).to(d)
            x = kept.float()
        rstd = 1.0 / torch.sqrt(x.square().mean(1) + EPS)
        y = x * rstd[:, None] * s["gamma"].float()
        z = None
        if c["bits8"]:
            b, yb = _exponents(y)
            step = ((b + (1023 - 133)) << 52).view(torch.float64)[..., None]
            z = torch.round(yb.double() / step).clamp_(-127, 127) * step
            z = z.reshape(len(y), -1)[:, :c["cols"]].to(d)
        return y.to(d), rstd, kept, z
    z = x * c["scale"]
    if c["way"] == "forward":
        logp, entropy, lse = _row_stats(z, s["tokens"])
        if not c["top"]:
            return logp, entropy, lse, None, None
        ids = _top(x, c["top"])
        return logp, entropy, lse, ids.to(torch.int32), torch.gather(z, 1, ids) - lse[:, None]
    z = z - s["lse"][:, None]
    p = torch.exp(z)
    a, b = s["dlogp"][:, None] * c["scale"], s["dentropy"][:, None] * c["scale"]
    dx = -p * (a + b * (z + s["entropy"][:, None]))
    return dx.scatter_add_(1, s["tokens"].long()[:, None], a).to(d)


# -------------------------------------------------------------------- work
def _pairs(case):
    """(query, key) pairs that attention looks at, of one head."""
    n = 0
    for a, b in zip(*_lengths(case)):
        n += a * b - a * (a - 1) // 2 if case["causal"] else a * b
    return n


def work(case):
    e = SIZE[case["dtype"]]
    fwd = case["way"] == "forward"
    if case["op"] == "attention":
        lq, lk = _lengths(case)
        D = case["dim"]
        rows, keys = sum(lq) * case["heads"], sum(lk) * case["kv"]
        return {"bytes": (2 if fwd else 4) * (rows + keys) * D * e + 4 * rows,
                "flops": (4 if fwd else 10) * D * case["heads"] * _pairs(case)}
    R, C = case["rows"], case["cols"]
    if case["op"] == "rms_norm":
        if not fwd:
            return {"bytes": R * C * (3 + case["residual"]) * e + 4 * R + 2 * C * e,
                    "flops": 9 * R * C}
        held = 2 * (1 + 1 / BLOCK) + e if case["bits8"] else 0  # written, read, its values written
        return {"bytes": R * C * ((4 if case["residual"] else 2) * e + held) + 4 * R + C * e,
                "flops": (5 + 3 * case["bits8"]) * R * C}
    if fwd:
        return {"bytes": R * C * e + R * (16 + 8 * case["top"]), "flops": 6 * R * C}
    return {"bytes": 2 * R * C * e + 20 * R, "flops": 7 * R * C}


# ------------------------------------------------------------------- exact
def _attention_exact(case, t):
    f = torch.float64
    D, H, KV = case["dim"], case["heads"], case["kv"]
    G = H // KV
    lq, lk = _lengths(case)
    qs, ks = t["qs"].tolist(), t["ks"].tolist()
    fwd = case["way"] == "forward"
    out = [torch.zeros((t["Tq"], H * D), device="cuda", dtype=f)]
    if fwd:
        out.append(torch.zeros((H, t["Tq"]), device="cuda", dtype=f))
    else:
        out += [torch.zeros((t["Tk"], KV * D), device="cuda", dtype=f) for _ in range(2)]
    for n, (a, b) in enumerate(zip(lq, lk)):
        rq, rk = slice(qs[n], qs[n] + a), slice(ks[n], ks[n] + b)
        see = None
        if case["causal"]:
            see = torch.ones((a, b), device="cuda", dtype=torch.bool).tril(b - a)
        for h in range(H):
            ch, ck = slice(h * D, h * D + D), slice(h // G * D, h // G * D + D)
            q, k, v = t["q"][rq, ch].to(f), t["k"][rk, ck].to(f), t["v"][rk, ck].to(f)
            z = (q @ k.t().contiguous()) * t["scale"]
            if see is not None:
                z = torch.where(see, z, -math.inf)
            if fwd:
                out[0][rq, ch] = torch.softmax(z, 1) @ v
                out[1][h, rq] = torch.logsumexp(z, 1)
                continue
            p = torch.exp(z - t["lse"][h, rq].to(f)[:, None])
            do, o = t["dout"][rq, ch].to(f), t["out"][rq, ch].to(f)
            ds = p * (do @ v.t().contiguous() - (do * o).sum(1, keepdim=True)) * t["scale"]
            out[0][rq, ch] = ds @ k
            out[1][rk, ck] += ds.t().contiguous() @ q
            out[2][rk, ck] += p.t().contiguous() @ do
    return tuple(out)


def exact(case, seed):
    t = _inputs(case, seed)
    f = torch.float64
    if case["op"] == "attention":
        return _attention_exact(case, t)
    x = t["x"].to(f)
    if case["op"] == "rms_norm":
        gamma, C = t["gamma"].to(f), x.shape[1]
        if case["way"] == "backward":
            rs, dy = t["rstd"].to(f)[:, None], t["dy"].to(f)
            dot = (dy * gamma * x).sum(1, keepdim=True) * rs / C
            dx = rs * (dy * gamma - rs * x * dot)
            if case["residual"]:
                dx += t["ds"].to(f)
            return dx, (dy * x * rs).sum(0)
        kept = None
        if case["residual"]:
            kept = x + t["r"].to(f)
            x = kept.to(DT[case["dtype"]]).to(f)  # (the norm is of the sum as it is kept)
        rs = torch.rsqrt((x * x).sum(1) / C + EPS)
        y = x * rs[:, None] * gamma
        z = None
        if case["bits8"]:
            z = torch.empty_like(y)
            for k in range(0, C, BLOCK):
                yb = y[:, k:k + BLOCK]
                top = yb.abs().amax(1)
                m = torch.frexp(top)[0]  # top / m is the power of two above top, exactly
                step = torch.where(m > 0, top / m, 0.0).clamp(min=2.0 ** -125)[:, None] * 2.0 ** -7
                z[:, k:k + BLOCK] = (yb / step).round().clamp(-127, 127) * step
        return y, rs, kept, z
    x *= case["scale"]
    tok = t["tokens"].long()[:, None]
    if case["way"] == "forward":
        lse = torch.logsumexp(x, 1)
        p = torch.softmax(x, 1)
        logp = x.gather(1, tok)[:, 0] - lse
        tops = None
        if case["top"]:
            tops = torch.sort(x, 1, descending=True)[0][:, :case["top"]] - lse[:, None]
        return logp, (p * (lse[:, None] - x)).sum(1), lse, None, tops
    lp = x - t["lse"].to(f)[:, None]
    p = torch.exp(lp)
    a, b = t["dlogp"].to(f)[:, None], t["dentropy"].to(f)[:, None]
    hot = torch.zeros_like(p).scatter_(1, tok, 1.0)
    return case["scale"] * (a * (hot - p) - b * p * (lp + t["entropy"].to(f)[:, None]))
