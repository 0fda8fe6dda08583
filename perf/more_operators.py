"""What stands between two layers of a decoder on low-precision weights, as cases that can be timed and compared.

  norm    the residual's addition, the root-mean-square norm, and its output in 8 bits with scales:
            h = T(f32(x + r)), i = f32(1 / sqrt(mean(h^2) + eps)) with the mean in 64 bits, y = f32(f32(h i) g)
            a block of 128 values of a row: s = max(f32(max|y| / 448), 2^-126), code = e4m3(f32(y / s))
          h replaces r, T is the type of x and r; y itself is kept in T where `keep` is set.
  linear  y = q(x) q(w)^T on microscaled 4-bit floating point: a block of 32 values along k has the scale 2^e,
            e = floor(log2 max|v|) - 2 (-127 at least), and codes e2m1(v / 2^e), to nearest even, at most 6
          x and y are f32, f16 or bf16, each by its own choice; w is kept in that form.
  enter   a layer's entry: norm whose output goes to the 4-bit form, and two products (gate and up) of its codes.
  select  the experts of a token from its logits l:
            s = softmax(l) or 1 / (1 + exp(-l)), c = s + bias
            groups: the `keep_groups` groups of experts whose one or two largest c have the largest sum
            the `top` experts of largest c in them, ties to the lower index; shares s (times `scale`), over their sum
            where `renorm` is set
          The choice is made in 64 bits: scores next to each other are no rarity among many tokens.

`own` picks the side: the plain form in elementary torch operations, or the framework's entry points.
"""
import math

import torch

own = False

BLOCK = 128  # values with one scale in 8 bits
MICRO = 32   # values with one scale in 4 bits
EPS = 1e-6
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODE = {"f32": 0, "f16": 1, "bf16": 2}  # the framework's dtype numbers

# (k, n) of the configurations' projections: the decider's, the encoder's and the benchmark's
SHAPES = [(1024, 1024), (1024, 4096), (4096, 1024), (4096, 4096), (4096, 14336), (2560, 9216), (9216, 2560),
          (2560, 8192), (2560, 1024), (4096, 2560), (1024, 32000)]
FLOP_MOST = 2 * 16384 * 4096 * 14336


def listed():
    return [
        # one request's token: latency alone
        dict(name="norm_r1_2560", kind="norm", m=1, d=2560, x="bf16", keep=False),
        # rows of an odd length, the normed row kept beside its codes (for a router)
        dict(name="norm_r1001_1111", kind="norm", m=1001, d=1111, x="f16", keep=True),
        # bulk prefill at the benchmark's width
        dict(name="norm_r16384_4096", kind="norm", m=16384, d=4096, x="bf16", keep=False),
        # one request's token through one projection: the smallest call
        dict(name="linear_m1_4096x4096", kind="linear", m=1, k=4096, n=4096, x="bf16", y="bf16"),
        # sixteen rows against a whole vocabulary, scores kept in f32
        dict(name="linear_m16_1024x32000", kind="linear", m=16, k=1024, n=32000, x="f32", y="f32"),
        # nothing a multiple of anything: rows, columns and blocks that end inside a tile
        dict(name="linear_m1001_1111x1777", kind="linear", m=1001, k=1111, n=1777, x="f16", y="f16"),
        # bulk prefill: the largest product of the benchmark
        dict(name="linear_m16384_4096x14336", kind="linear", m=16384, k=4096, n=14336, x="bf16", y="bf16"),
        # eight requests' tokens at the entry of the decider's MLP
        dict(name="enter_m8_2560x9216", kind="enter", m=8, k=2560, n=9216, x="bf16", y="bf16"),
        # a short question to the decider (229 tokens), on its f32 residual stream
        dict(name="enter_m229_2560x9216", kind="enter", m=229, k=2560, n=9216, x="f32", y="f32"),
        # one token of one request among 64 experts, plain softmax shares
        dict(name="select_t1_e64k8", kind="select", t=1, e=64, top=8, score="softmax", bias=False, groups=1,
             keep_groups=1, best=1, renorm=True, scale=1.0, x="f32"),
        # requests in flight on a layer of few experts, ties among 16-bit logits
        dict(name="select_t100_e24k3", kind="select", t=100, e=24, top=3, score="softmax", bias=False, groups=3,
             keep_groups=2, best=1, renorm=False, scale=1.0, x="bf16"),
        # a whole batch's tokens: balanced sigmoid scores, half of eight groups kept
        dict(name="select_t16384_e256k8", kind="select", t=16384, e=256, top=8, score="sigmoid", bias=True, groups=8,
             keep_groups=4, best=2, renorm=True, scale=2.5, x="f32"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    at, types = rng.random(), list(DTYPES)
    if at < 0.25:
        d = rng.choice(SHAPES)[0] if rng.random() < 0.3 else _log_int(rng, 64, 9600)
        return dict(kind="norm", m=_log_int(rng, 1, min(16384, 16384 * 4096 // d)), d=d, x=rng.choice(types),
                    keep=rng.random() < 0.5)
    if at < 0.75:
        k, n = rng.choice(SHAPES) if rng.random() < 0.5 else (_log_int(rng, 100, 9600), _log_int(rng, 40, 14400))
        kind, most = ("linear", 16384) if at < 0.6 else ("enter", 4096)
        m = _log_int(rng, 1, max(1, min(most, FLOP_MOST // (4 * k * n))))
        return dict(kind=kind, m=m, k=k, n=n, x=rng.choice(types), y=rng.choice(types))
    groups = rng.choice([1, 1, 2, 3, 4, 8])
    e = groups * _log_int(rng, 2, 256 // groups)
    keep = rng.randint(1, groups)
    return dict(kind="select", t=_log_int(rng, 1, 16384), e=e, top=rng.randint(1, min(16, e // groups * keep)),
                score=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.5, groups=groups, keep_groups=keep,
                best=rng.randint(1, 2), renorm=rng.random() < 0.5, scale=rng.choice([1.0, 2.5]), x=rng.choice(types))


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
    return torch.Generator(device="cuda").manual_seed(seed * 6007 + 17)


def _activations(g, rows, width, dtype):
    """Rows of a residual stream: normal values, a few channels many times the others."""
    channel = torch.exp(0.6 * torch.randn(width, generator=g, device="cuda"))
    return (torch.randn(rows, width, generator=g, device="cuda") * channel).to(DTYPES[dtype])


def _weights(g, n, k):
    """Codes [n, ceil(k / 2)] (two a byte, the even k in the low half) and scale bytes [n, ceil(k / 32)] of normal
    weights of variance 1 / k, whose rows differ in size as trained ones do."""
    w = torch.randn(n, k, generator=g, device="cuda") * (k ** -0.5)
    w *= torch.exp(0.3 * torch.randn(n, 1, generator=g, device="cuda"))
    blocks = -(-k // MICRO)
    w = torch.nn.functional.pad(w, (0, blocks * MICRO - k)).view(n, blocks, MICRO)
    e = torch.frexp(w.abs().amax(2, keepdim=True)).exponent - 3
    a = torch.ldexp(w.abs(), -e)
    code = sum((a > edge).to(torch.uint8) for edge in (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0))
    code = (code | (w < 0).to(torch.uint8) << 3).view(n, -1)[:, :k + k % 2]
    return code[:, 0::2] | code[:, 1::2] << 4, (e + 127).to(torch.uint8).view(n, blocks)


def _outputs(case):
    """Where the framework's calls write."""
    empty = lambda *shape, **kw: torch.empty(*shape, device="cuda", **kw)  # noqa: E731
    if case["kind"] == "select":
        return dict(ids=empty(case["t"], case["top"], dtype=torch.int32), shares=empty(case["t"], case["top"]))
    m, out = case["m"], {}
    d = case["d"] if case["kind"] == "norm" else case["k"]
    if case["kind"] != "linear":
        out["h"] = empty(m, d, dtype=DTYPES[case["x"]])
    if case["kind"] == "norm":
        blocks = -(-d // BLOCK)
        out.update(codes=empty(m, blocks * BLOCK, dtype=torch.uint8), scales=empty(blocks, m))
        if case["keep"]:
            out["y"] = empty(m, d, dtype=DTYPES[case["x"]])
    elif case["kind"] == "linear":
        out["y"] = empty(m, case["n"], dtype=DTYPES[case["y"]])
    else:
        out.update({p: empty(m, case["n"], dtype=DTYPES[case["y"]]) for p in ("gate", "up")})
    return out


def prepare(case, seed):
    g, kind = _rng(seed), case["kind"]
    st = dict(case=dict(case))
    if kind == "select":
        st["logits"] = (1.5 * torch.randn(case["t"], case["e"], generator=g, device="cuda")).to(DTYPES[case["x"]])
        st["bias"] = 0.1 * torch.randn(case["e"], generator=g, device="cuda") if case["bias"] else None
    else:
        d = case["d"] if kind == "norm" else case["k"]
        st["x"] = _activations(g, case["m"], d, case["x"])
        if kind != "linear":
            st["r"] = _activations(g, case["m"], d, case["x"])
            st["g"] = torch.exp(0.3 * torch.randn(d, generator=g, device="cuda"))
        if kind != "norm":
            st["weights"] = [_weights(g, case["n"], d) for _ in range(2 if kind == "enter" else 1)]
    if own:
        st["ctx"], rocm = _context()
        st["out"] = _outputs(case)
        torch.cuda.synchronize()
        if "weights" in st:
            st["w"] = [st["ctx"].mx4_weight(codes, scales, case["n"], case["k"]) for codes, scales in st["weights"]]
        if kind == "enter":
            codes, scales = rocm.mx4_bytes(case["m"], case["k"])
            st["q"], st["s"] = (torch.empty(b, dtype=torch.uint8, device="cuda") for b in (codes, scales))
        if kind == "select":
            st["rule"] = rocm.MoeSelection(experts=case["e"], top_k=case["top"], sigmoid=int(case["score"] == "sigmoid"),
                                           groups=case["groups"], top_groups=case["keep_groups"],
                                           group_best=case["best"], renormalize=int(case["renorm"]), scale=case["scale"])
    return st


# ---- the plain forms -----------------------------------------------------------------


def _micro(x):
    """f32 rows as the values of their 4-bit form."""
    m, k = x.shape
    blocks = -(-k // MICRO)
    v = torch.nn.functional.pad(x, (0, blocks * MICRO - k)).view(m, blocks, MICRO)
    most = v.abs().amax(2, keepdim=True)
    e = torch.where(most > 0, torch.frexp(most).exponent - 3, -127).clamp_min(-127)
    v = torch.ldexp(v, -e)
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    v = torch.copysign((torch.round(a / step) * step).clamp_max(6), v)
    return torch.ldexp(v, e).view(m, -1)[:, :k]


def _weight_values(codes, scales, k):
    """The weight that codes and scale bytes stand for, in f32."""
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    v = torch.stack((table[(codes & 15).int()], table[(codes >> 4).int()]), -1).view(codes.shape[0], -1)[:, :k]
    return torch.ldexp(v, scales.int().repeat_interleave(MICRO, 1)[:, :k] - 127)


def _normed(st):
    """h in its type and y in f32."""
    h = (st["x"].float() + st["r"].float()).to(st["x"].dtype)
    wide = h.double()
    i = (1 / torch.sqrt((wide * wide).mean(1, keepdim=True) + EPS)).float()
    return h, h.float() * i * st["g"]


def _norm(st):
    h, y = _normed(st)
    m, d = y.shape
    blocks = -(-d // BLOCK)
    v = torch.nn.functional.pad(y, (0, blocks * BLOCK - d)).view(m, blocks, BLOCK)
    most = v.abs().amax(2, keepdim=True)
    s = (most / torch.full_like(most, 448)).clamp_min(2.0 ** -126)  # by a number alone it would be a product with 1 / 448
    codes = (v / s).clamp(-448, 448).to(torch.float8_e4m3fn).view(m, -1)
    out = dict(h=h, codes=codes, scales=s.view(m, blocks).t().contiguous())
    if st["case"]["keep"]:
        out["y"] = y.to(h.dtype)
    return out


def _linear(st):
    case = st["case"]
    codes, scales = st["weights"][0]
    return dict(y=(_micro(st["x"].float()) @ _weight_values(codes, scales, case["k"]).t()).to(DTYPES[case["y"]]))


def _enter(st):
    case = st["case"]
    h, y = _normed(st)
    q = _micro(y)
    gate, up = ((q @ _weight_values(c, s, case["k"]).t()).to(DTYPES[case["y"]]) for c, s in st["weights"])
    return dict(h=h, gate=gate, up=up)


def _select(st):
    case, l = st["case"], st["logits"].double()
    t, e, groups = case["t"], case["e"], case["groups"]
    s = torch.softmax(l, 1) if case["score"] == "softmax" else torch.sigmoid(l)
    c = s if st["bias"] is None else s + st["bias"].double()
    if groups > 1:
        part = torch.sort(c.view(t, groups, -1), dim=2, descending=True).values
        order = torch.sort(part[:, :, :case["best"]].sum(2), dim=1, descending=True, stable=True).indices
        stays = torch.zeros(t, groups, dtype=torch.bool, device=l.device).scatter_(1, order[:, :case["keep_groups"]], True)
        c = c.masked_fill(~stays.repeat_interleave(e // groups, 1), -math.inf)
    ids = torch.sort(c, dim=1, descending=True, stable=True).indices[:, :case["top"]]
    share = s.gather(1, ids)
    if case["renorm"]:
        share = share / share.sum(1, keepdim=True)
    return dict(ids=ids.int(), shares=(share * case["scale"]).float())


def run(st):
    case, kind = st["case"], st["case"]["kind"]
    if not own:
        return {"norm": _norm, "linear": _linear, "enter": _enter, "select": _select}[kind](st)
    ctx, out, x = st["ctx"], st["out"], CODE[case["x"]]
    if kind == "norm":
        ctx.add_rmsnorm_fp8(st["x"], st["r"], x, case["m"], case["d"], st["g"], EPS, out["h"], out["codes"],
                            out["scales"], y=out.get("y"), zero_centered=False)
        return {**out, "codes": out["codes"].view(torch.float8_e4m3fn)}
    if kind == "linear":
        ctx.mx4_linear(st["w"][0], st["x"], x, case["m"], out["y"], CODE[case["y"]])
    elif kind == "enter":
        ctx.add_rmsnorm_mx4(st["x"], st["r"], x, case["m"], case["k"], st["g"], EPS, out["h"], st["q"], st["s"],
                            zero_centered=False)
        for w, y in zip(st["w"], (out["gate"], out["up"])):
            ctx.mx4_linear_q4(w, st["q"], st["s"], case["m"], y, CODE[case["y"]])
    else:
        ctx.moe_select(st["rule"], st["logits"], x, case["t"], st["bias"], out["ids"], out["shares"])
    return out


# ---- what the operators cannot do without -----------------------------------------------

_SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def work(case):
    kind, size = case["kind"], _SIZE[case["x"]]
    if kind == "select":
        t, e = case["t"], case["e"]
        return {"bytes": t * e * size + 8 * t * case["top"] + 4 * e * case["bias"], "flops": t * e}
    m = case["m"]
    if kind == "norm":
        d = case["d"]
        return {"bytes": m * d * (size * (3 + case["keep"]) + 1) + 4 * m * -(-d // BLOCK) + 4 * d, "flops": 4 * m * d}
    k, n, products = case["k"], case["n"], 1 + (kind == "enter")
    weight = n * -(-k // 2) + n * -(-k // MICRO)
    rows = m * k * size if kind == "linear" else 3 * m * k * size + 4 * k
    return {"bytes": rows + products * (weight + m * n * _SIZE[case["y"]]), "flops": 2 * products * m * n * k}


# ---- the definitions in 64 bits -----------------------------------------------------------


def _to_grid(v, mantissa, least, most):
    """v (64 bits) rounded to the nearest number of `mantissa` bits behind the point, exponents from `least` on, ties
    to the even one, at most `most`."""
    exponent = torch.frexp(v.abs()).exponent - 1
    step = torch.exp2((exponent.clamp_min(least) - mantissa).double())
    return (torch.round(v / step) * step).clamp(-most, most)


def _exact_micro(v):
    """The values of the 4-bit form of f32 rows held in 64 bits."""
    q = torch.empty_like(v)
    for b in range(0, v.shape[1], MICRO):
        part = v[:, b:b + MICRO]
        most = part.abs().amax(1, keepdim=True)
        scale = torch.exp2(torch.floor(torch.log2(most.clamp_min(2.0 ** -125))) - 2)
        scale = torch.where(scale * 4 > most.clamp_min(2.0 ** -125), scale / 2, scale)  # a logarithm rounded upwards
        q[:, b:b + MICRO] = _to_grid(part / scale, 1, 0, 6.0) * scale
    return q


def _exact_weight(codes, scales, k):
    pairs = torch.zeros(codes.shape[0], 2 * codes.shape[1], dtype=torch.float64, device=codes.device)
    for half in (0, 1):
        c = (codes >> (4 * half) & 15).double()
        size, sign = c % 8, 1 - 2 * (c >= 8).double()
        exponent, odd = torch.div(size, 2, rounding_mode="floor"), size % 2
        value = torch.where(exponent == 0, odd / 2, (1 + odd / 2) * torch.exp2(exponent - 1))
        pairs[:, half::2] = sign * value
    block = torch.arange(k, device=codes.device) // MICRO
    return pairs[:, :k] * torch.exp2(scales.double() - 127)[:, block]


def _exact_normed(st):
    h = (st["x"].double() + st["r"].double()).float().to(st["x"].dtype).double()
    i = torch.rsqrt(h.square().sum(1, keepdim=True) / h.shape[1] + EPS).float().double()
    return h, ((h * i).float().double() * st["g"].double()).float().double()


def exact(case, seed):
    st, kind = prepare(case, seed), case["kind"]
    if kind == "linear":
        return dict(y=_exact_micro(st["x"].double()) @ _exact_weight(*st["weights"][0], case["k"]).t())
    if kind == "enter":
        h, y = _exact_normed(st)
        q = _exact_micro(y)
        gate, up = (q @ _exact_weight(codes, scales, case["k"]).t() for codes, scales in st["weights"])
        return dict(h=h, gate=gate, up=up)
    if kind == "norm":
        h, y = _exact_normed(st)
        m, d = y.shape
        blocks = -(-d // BLOCK)
        codes = torch.zeros(m, blocks * BLOCK, dtype=torch.float64, device="cuda")
        scales = torch.zeros(blocks, m, dtype=torch.float64, device="cuda")
        for b in range(blocks):
            part = y[:, b * BLOCK:(b + 1) * BLOCK]
            s = (part.abs().amax(1) / 448).float().double().clamp_min(2.0 ** -126)
            scales[b] = s
            codes[:, b * BLOCK:b * BLOCK + part.shape[1]] = _to_grid((part / s[:, None]).float().double(), 3, -6, 448.0)
        return dict(h=h, codes=codes, scales=scales, **(dict(y=y) if case["keep"] else {}))
    l = st["logits"].double()
    if case["score"] == "softmax":
        s = torch.exp(l - l.amax(1, keepdim=True))
        s = s / s.sum(1, keepdim=True)
    else:
        s = 1 / (1 + torch.exp(-l))
    c = s.clone() if st["bias"] is None else s + st["bias"].double()
    width = case["e"] // case["groups"]
    if case["groups"] > 1:
        best = torch.stack([c[:, a:a + width].topk(min(case["best"], width), 1).values.sum(1)
                            for a in range(0, case["e"], width)], 1)
        kept = torch.argsort(-best, dim=1, stable=True)[:, :case["keep_groups"]]
        group = torch.arange(case["e"], device="cuda") // width
        c[~(group[None, :, None] == kept[:, None, :]).any(2)] = -math.inf
    chosen = torch.argsort(-c, dim=1, stable=True)[:, :case["top"]]
    share = torch.gather(s, 1, chosen)
    if case["renorm"]:
        share = share / share.sum(1, keepdim=True)
    return dict(ids=None, shares=share * case["scale"])
