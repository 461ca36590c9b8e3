"""The 8-bit decode/prefill MLP operators, case by case: rows quantised to 8 bits with a scale each (plain rows, the
RMS norm with the residual's addition, SwiGLU) and matrix products with bias, activation and residual in the epilogue
(16-bit operands, or 8-bit operands with scales).

``run`` computes a case either in plain torch operations (fp32, one rounding at the end) or, where ``own`` is true, by
the package's operators.  ``exact`` gives the same values in 64 bits.
"""

import math

import torch

own = False

E4M3 = torch.float8_e4m3fn
MAX8 = 448.0            # largest finite e4m3 value
FLOOR = 2.0 ** -64      # smallest row maximum a scale is made from
EPS = 1e-5
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one token's attention output on its way into an 8-bit output projection
        {"name": "quantize_1x4096", "op": "quantize", "dtype": "bf16", "m": 1, "n": 4096},
        # a ragged prefill batch, or a weight being laid out in 8 bits
        {"name": "quantize_4099x8192", "op": "quantize", "dtype": "fp16", "m": 4099, "n": 8192},
        # the norm before the MLP of one decoded token
        {"name": "add_rms_1x4096", "op": "rms", "dtype": "bf16", "m": 1, "n": 4096, "res": True},
        # the same norm over a long prefill
        {"name": "add_rms_8192x4096", "op": "rms", "dtype": "bf16", "m": 8192, "n": 4096, "res": True},
        # gate and up of a small decode batch, as halves of one [M, 2I] product
        {"name": "swiglu_8x14336", "op": "swiglu", "dtype": "bf16", "m": 8, "n": 14336},
        # and of a prefill
        {"name": "swiglu_2048x14336", "op": "swiglu", "dtype": "fp16", "m": 2048, "n": 14336},
        # output projection of one token onto the residual stream
        {"name": "linear_1x4096x4096", "op": "linear", "dtype": "bf16", "m": 1, "n": 4096, "k": 4096, "bias": False,
         "act": "none", "res": True},
        # a prefill's up projection with bias and activation
        {"name": "linear_4096x14336x4096", "op": "linear", "dtype": "fp16", "m": 4096, "n": 14336, "k": 4096,
         "bias": True, "act": "gelu_tanh", "res": False},
        # gate/up product of a small decode batch with 8-bit weights
        {"name": "linear8_5x28672x4096", "op": "linear8", "dtype": "bf16", "m": 5, "n": 28672, "k": 4096, "bias": False,
         "act": "none", "res": False},
        # down projection of a ragged prefill onto the residual stream
        {"name": "linear8_2050x4096x14336", "op": "linear8", "dtype": "bf16", "m": 2050, "n": 4096, "k": 14336,
         "bias": True, "act": "none", "res": True},
        # the whole MLP block of one token, and of a ragged prefill
        {"name": "mlp8_1x4096x14336", "op": "mlp8", "dtype": "bf16", "m": 1, "h": 4096, "i": 14336},
        {"name": "mlp8_1031x4096x14336", "op": "mlp8", "dtype": "bf16", "m": 1031, "h": 4096, "i": 14336},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _width(rng, low, high):
    """A row width: mostly a multiple of 16, one in five any number."""
    w = _log_int(rng, low, high)
    return w if rng.random() < 0.2 else max(16, w // 16 * 16)


def draw(rng):
    op = rng.choice(["quantize", "rms", "swiglu", "linear", "linear8", "mlp8"])
    case = {"op": op, "dtype": rng.choice(["bf16", "fp16"]), "m": _log_int(rng, 1, 8192)}
    if op in ("quantize", "rms", "swiglu"):
        case["n"] = _width(rng, 64, 28672)
        case["m"] = min(case["m"], (8192 * 4096) // case["n"])
        if op == "rms":
            case["res"] = rng.random() < 0.7
    elif op in ("linear", "linear8"):
        # outputs of any number (a vocabulary has odd ones), inner widths as models have them
        case["n"] = rng.choice([_log_int(rng, 64, 32768), 16 * _log_int(rng, 4, 2048)])
        case["k"] = 16 * _log_int(rng, 4, 1024)
        case["m"] = max(1, min(case["m"], (4096 * 14336 * 4096) // (case["n"] * case["k"])))
        case["bias"] = rng.random() < 0.5
        case["act"] = rng.choice(["none", "none", "relu", "silu", "gelu", "gelu_tanh"])
        case["res"] = rng.random() < 0.5
    else:
        case["h"] = 128 * rng.randint(2, 64)
        case["i"] = 128 * rng.randint(4, 160)
        case["m"] = max(1, min(case["m"], (1031 * 4096 * 14336) // (case["h"] * case["i"])))
    return case


# ------------------------------------------------------------------ inputs
def _rows8(y):
    """fp32 rows -> (e4m3 values, fp32 scale per row)."""
    a = y.abs().amax(dim=-1, keepdim=True).clamp_min(FLOOR)
    q = (y * (MAX8 / a)).clamp(-MAX8, MAX8).to(E4M3)
    return q, (a / MAX8).squeeze(-1)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    t = TYPES[case["dtype"]]

    def rn(*shape, scale=1.0):
        return torch.randn(*shape, device=dev, generator=g).mul_(scale)

    def hidden(m, n):
        # activations: a few columns are an order of magnitude larger than the rest
        column = 1.0 + 12.0 * (torch.rand(n, device=dev, generator=g) < 0.01)
        return (rn(m, n) * column).to(t)

    def weight8(n, k):
        return _rows8(rn(n, k, scale=k ** -0.5))

    op, m = case["op"], case["m"]
    s = {"case": dict(case)}
    if op == "quantize":
        s["x"] = hidden(m, case["n"])
    elif op == "rms":
        n = case["n"]
        s["x"] = hidden(m, n)
        s["res"] = rn(m, n, scale=2.0).to(t) if case["res"] else None
        s["w"] = (1.0 + rn(n, scale=0.1)).to(t)
    elif op == "swiglu":
        s["gu"] = rn(m, 2 * case["n"], scale=1.5).to(t)
    elif op in ("linear", "linear8"):
        n, k = case["n"], case["k"]
        if op == "linear":
            s["x"], s["w"] = hidden(m, k), rn(n, k, scale=k ** -0.5).to(t)
        else:
            s["x"], s["xs"] = _rows8(hidden(m, k).float())
            s["w"], s["ws"] = weight8(n, k)
        s["bias"] = rn(n, scale=0.5).to(t) if case["bias"] else None
        s["res"] = rn(m, n, scale=2.0).to(t) if case["res"] else None
    else:
        h, i = case["h"], case["i"]
        s["x"] = hidden(m, h)
        s["w"] = (1.0 + rn(h, scale=0.1)).to(t)
        s["wgu"], s["sgu"] = weight8(2 * i, h)
        s["wd"], s["sd"] = weight8(h, i)
    return s


# ------------------------------------------------------------------ plain form
def _act(v, name):
    if name == "relu":
        return v.clamp_min(0.0)
    if name == "silu":
        return v / (1.0 + torch.exp(-v))
    if name == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))
    return v


def _norm(v, w):
    return v * torch.rsqrt((v * v).mean(dim=-1, keepdim=True) + EPS) * w


def _product8(x, xs, w, ws):
    return (x.float() @ w.float().T) * xs[:, None] * ws


def _plain(s):
    case = s["case"]
    op, t = case["op"], TYPES[case["dtype"]]
    if op == "quantize":
        return _rows8(s["x"].float())
    if op == "rms":
        v = s["x"].float()
        if s["res"] is None:
            return _rows8(_norm(v, s["w"].float()))
        v = v + s["res"].float()
        return (*_rows8(_norm(v, s["w"].float())), v.to(t))
    if op == "swiglu":
        gate, up = s["gu"].float().split(case["n"], dim=-1)
        return _rows8(_act(gate, "silu") * up)
    if op in ("linear", "linear8"):
        v = s["x"].float() @ s["w"].float().T if op == "linear" else _product8(s["x"], s["xs"], s["w"], s["ws"])
        if s["bias"] is not None:
            v = v + s["bias"].float()
        v = _act(v, case["act"])
        if s["res"] is not None:
            v = v + s["res"].float()
        return v.to(t)
    q, qs = _rows8(_norm(s["x"].float(), s["w"].float()))
    gate, up = _product8(q, qs, s["wgu"], s["sgu"]).to(t).float().split(case["i"], dim=-1)
    q, qs = _rows8(_act(gate, "silu") * up)
    return (_product8(q, qs, s["wd"], s["sd"]) + s["x"].float()).to(t)


def run(state):
    if not own:
        return _plain(state)
    import fused_decode_b200 as fd

    s, case = state, state["case"]
    op, t = case["op"], TYPES[case["dtype"]]
    act = None if case.get("act", "none") == "none" else case["act"]
    if op == "quantize":
        return fd.quantize_fp8(s["x"])
    if op == "rms":
        if s["res"] is None:
            return fd.rms_norm_fp8(s["x"], s["w"], EPS)
        return fd.add_rms_norm_fp8(s["x"], s["res"], s["w"], EPS)
    if op == "swiglu":
        gate, up = s["gu"].split(case["n"], dim=-1)
        return fd.swiglu_fp8(gate, up)
    if op == "linear":
        return fd.linear_act(s["x"], s["w"], s["bias"], activation=act, row_add=s["res"])
    if op == "linear8":
        return fd.linear_fp8(s["x"], s["xs"], s["w"], s["ws"], s["bias"], activation=act, row_add=s["res"],
                             out_dtype=t)
    return fd.post_attn_mlp_fp8(s["x"], s["w"], s["wgu"], s["sgu"], s["wd"], s["sd"], EPS)


# ------------------------------------------------------------------ 64 bits
def _grid8(v):
    """64-bit values rounded to the e4m3 grid: 3 fraction bits, exponents from -6, ties to even."""
    v = v.clamp(-MAX8, MAX8)
    exponent = torch.frexp(v)[1] - 1
    step = torch.ldexp(torch.ones_like(v), exponent.clamp_min(-6) - 3)
    return torch.round(v / step) * step


def _scaled64(y):
    """(value over scale before its rounding to 8 bits, scale)."""
    scale = y.abs().amax(dim=-1, keepdim=True).clamp_min(FLOOR) / MAX8
    return y / scale, scale.squeeze(-1)


def _act64(v, name):
    if name == "relu":
        return torch.where(v > 0, v, torch.zeros_like(v))
    if name == "silu":
        return v * torch.special.expit(v)
    if name == "gelu":
        return v * 0.5 * torch.special.erfc(-v / math.sqrt(2.0))
    if name == "gelu_tanh":
        return v * torch.special.expit(2.0 * math.sqrt(2.0 / math.pi) * (v + 0.044715 * v ** 3))
    return v


def exact(case, seed):
    """What ``run`` returns, in 64 bits.  Values held in 8 bits are given before that last rounding, so that what is
    said of either side is its distance from the true quantity, the rounding included."""
    s = prepare(case, seed)
    op = case["op"]
    d = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor)}
    if op == "quantize":
        return _scaled64(d["x"])
    if op == "rms":
        v = d["x"] + d["res"] if case["res"] else d["x"]
        y = v / (v.square().sum(dim=-1, keepdim=True) / case["n"] + EPS).sqrt() * d["w"]
        return (*_scaled64(y), v) if case["res"] else _scaled64(y)
    if op == "swiglu":
        return _scaled64(_act64(d["gu"][:, :case["n"]], "silu") * d["gu"][:, case["n"]:])
    if op in ("linear", "linear8"):
        x, w = (d["x"], d["w"]) if op == "linear" else (d["x"] * d["xs"][:, None], d["w"] * d["ws"][:, None])
        v = torch.mm(x, w.t())
        if case["bias"]:
            v = v + d["bias"]
        v = _act64(v, case["act"])
        return v + d["res"] if case["res"] else v
    i = case["i"]
    y = d["x"] / (d["x"].square().sum(dim=-1, keepdim=True) / case["h"] + EPS).sqrt() * d["w"]
    q, scale = _scaled64(y)
    gu = torch.mm(_grid8(q) * scale[:, None], (d["wgu"] * d["sgu"][:, None]).t())
    gu = gu.to(TYPES[case["dtype"]]).double()  # the products between the stages are kept in 16 bits
    q, scale = _scaled64(_act64(gu[:, :i], "silu") * gu[:, i:])
    return torch.mm(_grid8(q) * scale[:, None], (d["wd"] * d["sd"][:, None]).t()) + d["x"]


# ------------------------------------------------------------------ work
def work(case):
    op, m = case["op"], case["m"]
    if op == "quantize":
        n = case["n"]
        return {"bytes": 3 * m * n + 4 * m, "flops": 2 * m * n}
    if op == "rms":
        n = case["n"]
        return {"bytes": (7 if case["res"] else 3) * m * n + 2 * n + 4 * m, "flops": 6 * m * n}
    if op == "swiglu":
        n = case["n"]
        return {"bytes": 5 * m * n + 4 * m, "flops": 8 * m * n}
    if op in ("linear", "linear8"):
        n, k = case["n"], case["k"]
        size = (2 if op == "linear" else 1) * (m * k + n * k) + (4 * (m + n) if op == "linear8" else 0)
        out = 2 * m * n * (2 if case["res"] else 1) + (2 * n if case["bias"] else 0)
        return {"bytes": size + out, "flops": 2 * m * n * k}
    h, i = case["h"], case["i"]
    return {"bytes": 3 * h * i + 4 * (2 * i + h) + 2 * h + 4 * m * h, "flops": 6 * m * h * i}
