"""The operators on 8-bit floating point weights, as cases that can be timed and compared.

Weights are e4m3 codes (4 exponent bits, 3 mantissa bits, largest value 448, no infinities) with one f32
scale for each block of 128 x 128 values: w[i, j] = code[i, j] * scale[i // 128, j // 128].

  linear  y = q(x) w^T: each row of x is cut into blocks of 128 along k and put in the same 8 bits,
            s = max(max|x| / 448, 2^-126), code = e4m3(x / s)   (both quotients held in f32, to nearest even)
          so that y[i, j] = sum over blocks b of s[i, b] scale[j // 128, b] sum_k code_x[i, k] code_w[j, k].
          x and y are f32, f16 or bf16, each by its own choice.
  moe     a whole mixture-of-experts layer for a few tokens, the activations kept as they come:
            l = x router^T, p = softmax(l), E(x) = the top_k experts of largest l (ties to the lower index)
            y = sum over e in E(x) of c_e down_e (silu(gate_e x) * up_e x)
          with c_e = p_e, or p_e / (sum of the chosen p) where `renormalize` is set. y has x's type.

`own` picks the side: the plain form in elementary torch operations, or the framework's entry points.
"""
import math

import torch

own = False

BLOCK = 128
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODE = {"f32": 0, "f16": 1, "bf16": 2}  # the framework's dtype numbers

# (k, n) of the configurations' projections: the decider's, the encoder's and the benchmark's
SHAPES = [(1024, 1024), (1024, 4096), (4096, 1024), (4096, 4096), (4096, 14336), (2560, 9216), (9216, 2560),
          (2560, 8192), (2560, 1024), (4096, 2560), (1024, 32000)]
FLOP_MOST = 2 * 16384 * 4096 * 14336
EXPERTS_MOST = 32 * 4096 * 1536  # values of one of the largest layer's three projections


def listed():
    return [
        # one request's token through one projection: the smallest call, latency counts
        dict(name="linear_m1_4096x4096", kind="linear", m=1, k=4096, n=4096, x="bf16", y="bf16"),
        # four requests' tokens through the decider's widest projection of its MLP
        dict(name="linear_m4_2560x9216", kind="linear", m=4, k=2560, n=9216, x="f16", y="f16"),
        # sixteen rows against a whole vocabulary, scores kept in f32
        dict(name="linear_m16_1024x32000", kind="linear", m=16, k=1024, n=32000, x="f32", y="f32"),
        # a short question to the decider (229 tokens), on its f32 residual stream
        dict(name="linear_m229_9216x2560", kind="linear", m=229, k=9216, n=2560, x="f32", y="f32"),
        # four short texts in the encoder (77 tokens each): its FFN's first projection
        dict(name="linear_m308_1024x4096", kind="linear", m=308, k=1024, n=4096, x="f16", y="f16"),
        # nothing a multiple of anything: rows, columns and blocks that end inside a tile
        dict(name="linear_m1001_1111x1777", kind="linear", m=1001, k=1111, n=1777, x="bf16", y="bf16"),
        # the benchmark's 8-bit product, a large batch
        dict(name="linear_m8192_4096x4096", kind="linear", m=8192, k=4096, n=4096, x="bf16", y="bf16"),
        # bulk prefill: the largest product of the benchmark
        dict(name="linear_m16384_4096x14336", kind="linear", m=16384, k=4096, n=14336, x="bf16", y="bf16"),
        # one token of one request: 8 of 64 experts are read
        dict(name="moe_t1_e64k8_2560x1024", kind="moe", t=1, e=64, top=8, d=2560, ff=1024, x="bf16", norm=True),
        # eight requests on a small layer
        dict(name="moe_t8_e16k2_1024x512", kind="moe", t=8, e=16, top=2, d=1024, ff=512, x="f16", norm=False),
        # odd sizes throughout, experts with a row or none
        dict(name="moe_t13_e24k3_1000x700", kind="moe", t=13, e=24, top=3, d=1000, ff=700, x="bf16", norm=True),
        # sixty-four requests, in f32: every expert is read, by eight tokens each
        dict(name="moe_t64_e32k4_4096x1536", kind="moe", t=64, e=32, top=4, d=4096, ff=1536, x="f32", norm=True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    if rng.random() < 0.6:
        k, n = rng.choice(SHAPES) if rng.random() < 0.5 else (_log_int(rng, 100, 9600), _log_int(rng, 40, 14400))
        m = _log_int(rng, 1, max(1, min(16384, FLOP_MOST // (2 * k * n))))
        return dict(kind="linear", m=m, k=k, n=n, x=rng.choice(list(DTYPES)), y=rng.choice(list(DTYPES)))
    d, ff = _log_int(rng, 200, 4096), _log_int(rng, 100, 2048)
    e = _log_int(rng, 4, max(4, min(128, EXPERTS_MOST // (d * ff))))
    return dict(kind="moe", t=_log_int(rng, 1, 64), e=e, top=rng.randint(1, min(8, e)), d=d, ff=ff,
                x=rng.choice(list(DTYPES)), norm=rng.random() < 0.5)


# ---- what a program sets up once --------------------------------------------------

_shared = {}


def _context():
    """The program's one context, on the stream the program works on."""
    if not _shared:
        from decisive_amd import rocm
        stream = torch.cuda.Stream()
        torch.cuda.set_stream(stream)
        ctx = rocm.Context(0)
        ctx.set_stream(stream.cuda_stream)
        _shared.update(ctx=ctx, stream=stream, rocm=rocm)
    torch.cuda.set_stream(_shared["stream"])
    return _shared["ctx"], _shared["rocm"]


def _rng(seed):
    return torch.Generator(device="cuda").manual_seed(seed * 7919 + 11)


def _activations(g, rows, width, dtype):
    """Rows of a residual stream: normal values, a few channels many times the others."""
    channel = torch.exp(0.6 * torch.randn(width, generator=g, device="cuda"))
    return (torch.randn(rows, width, generator=g, device="cuda") * channel).to(DTYPES[dtype])


def _weights(g, experts, rows, cols):
    """Codes [experts, rows, cols] (bytes) and block scales of normal weights of variance 1 / cols, whose rows
    differ in size as trained ones do."""
    codes = torch.empty(experts, rows, cols, dtype=torch.uint8, device="cuda")
    rb, cb = -(-rows // BLOCK), -(-cols // BLOCK)
    scales = torch.empty(experts, rb, cb, device="cuda")
    for e in range(experts):
        w = torch.randn(rows, cols, generator=g, device="cuda") * (cols ** -0.5)
        w *= torch.exp(0.3 * torch.randn(rows, 1, generator=g, device="cuda"))
        padded = torch.zeros(rb * BLOCK, cb * BLOCK, device="cuda")
        padded[:rows, :cols] = w
        s = padded.abs().view(rb, BLOCK, cb, BLOCK).amax((1, 3)) / 448
        codes[e] = (w / _spread(s, rows, cols)).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        scales[e] = s
    return codes, scales


def _spread(s, rows, cols):
    """Block scales [..., rows / 128, cols / 128] as one scale for each value."""
    return s.repeat_interleave(BLOCK, -2)[..., :rows, :].repeat_interleave(BLOCK, -1)[..., :cols]


def prepare(case, seed):
    g = _rng(seed)
    st = dict(case=dict(case))
    if case["kind"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        st["x"] = _activations(g, m, k, case["x"])
        codes, scales = _weights(g, 1, n, k)
        st["codes"], st["scales"] = codes[0], scales[0]
        if own:
            ctx, _ = _context()
            st["ctx"] = ctx
            st["y"] = torch.empty(m, n, dtype=DTYPES[case["y"]], device="cuda")
            torch.cuda.synchronize()
            st["w"] = ctx.fp8_weight(st["codes"], st["scales"], n, k)
    else:
        t, e, d, ff = case["t"], case["e"], case["d"], case["ff"]
        st["x"] = _activations(g, t, d, case["x"])
        st["router"] = torch.randn(e, d, generator=g, device="cuda") * (d ** -0.5)
        st["gate"], st["up"], st["down"] = _weights(g, e, ff, d), _weights(g, e, ff, d), _weights(g, e, d, ff)
        if own:
            ctx, rocm = _context()
            st["y"] = torch.empty(t, d, dtype=DTYPES[case["x"]], device="cuda")
            torch.cuda.synchronize()
            cfg = rocm.MoeConfig(experts=e, top_k=case["top"], hidden=d, ff=ff, renormalize=int(case["norm"]))
            st["moe"] = ctx.moe(cfg, st["router"], rocm.F32, st["gate"], st["up"], st["down"])
    return st


# ---- the plain forms -----------------------------------------------------------------


def _values(codes, scales):
    """The weights that codes and block scales stand for, in f32."""
    return codes.view(torch.float8_e4m3fn).float() * _spread(scales, codes.shape[-2], codes.shape[-1])


def _linear(st):
    case, x = st["case"], st["x"].float()
    m, k = x.shape
    blocks = -(-k // BLOCK)
    xb = torch.nn.functional.pad(x, (0, blocks * BLOCK - k)).view(m, blocks, BLOCK)
    most = xb.abs().amax(-1, keepdim=True)
    s = (most / torch.full_like(most, 448)).clamp_min(2.0 ** -126)  # by a number alone it would be a product with 1 / 448
    xq = ((xb / s).clamp(-448, 448).to(torch.float8_e4m3fn).float() * s).view(m, -1)[:, :k]
    return (xq @ _values(st["codes"], st["scales"]).t()).to(DTYPES[case["y"]])


def _moe(st):
    case, x = st["case"], st["x"].float()
    t, e, top = case["t"], case["e"], case["top"]
    logits = x @ st["router"].t()
    ids = torch.sort(logits, dim=-1, descending=True, stable=True).indices[:, :top]
    c = torch.softmax(logits, -1).gather(1, ids)
    if case["norm"]:
        c = c / c.sum(-1, keepdim=True)
    if t * top <= e:  # fewer choices than experts: the chosen experts' weights alone
        pick = ids.flatten()
        gate, up, down = (_values(st[p][0][pick], st[p][1][pick]) for p in ("gate", "up", "down"))
        rows = x.repeat_interleave(top, 0).unsqueeze(-1)
        h = torch.nn.functional.silu(gate @ rows) * (up @ rows)
        y = ((down @ h).view(t, top, -1) * c.unsqueeze(-1)).sum(1)
    else:  # every expert on every token, those not chosen with a share of nothing
        gate, up, down = (_values(*st[p]) for p in ("gate", "up", "down"))
        h = torch.nn.functional.silu(x @ gate.transpose(1, 2)) * (x @ up.transpose(1, 2))
        share = torch.zeros(t, e, device=x.device).scatter_(1, ids, c)
        y = ((h @ down.transpose(1, 2)) * share.t().unsqueeze(-1)).sum(0)
    return y.to(DTYPES[case["x"]])


def run(st):
    case = st["case"]
    if own:
        if case["kind"] == "linear":
            st["ctx"].fp8_linear(st["w"], st["x"], CODE[case["x"]], case["m"], st["y"], CODE[case["y"]])
        else:
            st["moe"].forward(st["x"], CODE[case["x"]], case["t"], st["y"])
        return st["y"]
    return _linear(st) if case["kind"] == "linear" else _moe(st)


# ---- what the operators cannot do without -----------------------------------------------

_SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def work(case):
    if case["kind"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        scales = 4 * -(-k // BLOCK) * -(-n // BLOCK)
        return {"bytes": m * k * _SIZE[case["x"]] + n * k + scales + m * n * _SIZE[case["y"]], "flops": 2 * m * n * k}
    t, e, top, d, ff = case["t"], case["e"], case["top"], case["d"], case["ff"]
    chosen = e * (1 - (1 - top / e) ** t)  # experts that t tokens choose, on average
    scales = 4 * -(-d // BLOCK) * -(-ff // BLOCK)
    return {"bytes": chosen * 3 * (d * ff + scales) + 4 * e * d + 2 * t * d * _SIZE[case["x"]],
            "flops": 2 * t * top * 3 * d * ff + 2 * t * e * d}


# ---- the definitions in 64 bits -----------------------------------------------------------


def _e4m3_table():
    """The 256 values of e4m3 by their bits: sign, 4 exponent bits of bias 7, 3 mantissa bits."""
    out = []
    for b in range(256):
        exponent, mantissa = b >> 3 & 15, b & 7
        v = math.ldexp(mantissa, -9) if exponent == 0 else math.ldexp(8 + mantissa, exponent - 10)
        out.append(math.nan if b & 127 == 127 else -v if b & 128 else v)
    return torch.tensor(out, dtype=torch.float64, device="cuda")


def _wide(codes, scales):
    """The weights of one matrix in 64 bits."""
    w = _e4m3_table()[codes.int()]
    i, j = (torch.arange(size, device="cuda") // BLOCK for size in w.shape)
    return w * scales.double()[i][:, j]


def _to_e4m3(v):
    """v (64 bits, |v| <= 464) rounded to the nearest e4m3 value, ties to the even one."""
    exponent = torch.frexp(v.abs()).exponent - 1
    step = torch.ldexp(torch.ones_like(v), exponent.clamp_min(-6) - 3)
    return (torch.round(v / step) * step).clamp(-448, 448)


def exact(case, seed):
    st = prepare(case, seed)
    x = st["x"].double()
    if case["kind"] == "linear":
        q = torch.zeros_like(x)
        for b in range(0, case["k"], BLOCK):
            part = x[:, b:b + BLOCK]
            s = (part.abs().max(1, keepdim=True).values / 448).float().double().clamp_min(2.0 ** -126)
            q[:, b:b + BLOCK] = _to_e4m3((part / s).float().double()) * s
        return q @ _wide(st["codes"], st["scales"]).t()
    t, top = case["t"], case["top"]
    logits = x @ st["router"].double().t()
    p = torch.exp(logits - logits.max(1, keepdim=True).values)
    p = p / p.sum(1, keepdim=True)
    order = torch.argsort(-logits, dim=1, stable=True)[:, :top]
    chosen = torch.zeros_like(p).scatter_(1, order, 1.0)
    p = p * chosen
    if case["norm"]:
        p = p / p.sum(1, keepdim=True)
    y = torch.zeros(t, case["d"], dtype=torch.float64, device="cuda")
    for e in range(case["e"]):
        rows = chosen[:, e].nonzero().flatten()
        if rows.numel() == 0:
            continue
        a = x[rows] @ _wide(st["gate"][0][e], st["gate"][1][e]).t()
        h = a / (1 + torch.exp(-a)) * (x[rows] @ _wide(st["up"][0][e], st["up"][1][e]).t())
        y[rows] += (h @ _wide(st["down"][0][e], st["down"][1][e]).t()) * p[rows, e:e + 1]
    return y
