"""The token and pixel operators of the library as they are measured: the linear layer (matrix product with bias,
activation and residual in its epilogue, binary16 or 8 bit operands) and the root-mean-square norm (with the residual's
addition, binary16 or 8 bit output with a scale per row).

`run` computes a case in plain torch operations, in 32 bits and rounded once at the end, or, with `own` set, through the
library's own entry points on the same inputs.  `exact` restates the definitions in 64 bits.
"""
import math

import torch

own = False

E4M3_MAX = 448.0
EPS = 1e-5
LEAKY_ALPHA = 0.125
FRAME = 1088 * 1920  # pixels of the benchmark's frame: a pointwise layer has one row per pixel


def _linear(name, rows, c_in, c_out, dtype="f16", act="none", bias=True, residual=False):
    case = {"op": "linear", "rows": rows, "c_in": c_in, "c_out": c_out, "dtype": dtype, "act": act, "bias": bias,
            "residual": residual}
    return {"name": name, **case} if name else case


def _norm(name, rows, channels, dtype="f16", residual=False):
    case = {"op": "rmsnorm", "rows": rows, "channels": channels, "dtype": dtype, "residual": residual}
    return {"name": name, **case} if name else case


def listed():
    return [
        # one token through a square layer of a residual block: the call is bound by latency and the weights' bytes
        _linear("linear one row 4096 to 4096 +residual", 1, 4096, 4096, residual=True),
        # a small batch of single tokens through the widening layer of a feed-forward block, weights held in 8 bits
        _linear("linear 16 rows 4096 to 12288 e4m3 silu", 16, 4096, 12288, "e4m3", "silu", bias=False),
        # a short prompt, or the bottleneck level of a small picture (10 x 10 positions)
        _linear("linear 100 rows 2048 to 8192 gelu", 100, 2048, 8192, act="gelu"),
        # the 1x1 convolution that brings a decoder level's 96 channels down to 64 on the benchmark's whole frame
        _linear("linear frame 96 to 64 relu", FRAME, 96, 64, act="relu"),
        # the network's nine input channels (colour, albedo, normal) lifted on a half resolution frame: rows of 18 bytes
        _linear("linear half frame 9 to 32 leaky", FRAME // 4, 9, 32, act="leaky"),
        # sizes off every tile border: 999 columns have rows that no 16 byte store can write
        _linear("linear ragged 1001 rows 1000 to 999", 1001, 1000, 999, residual=True),
        # a long prompt through a feed-forward block: binary16 operands, and 8 bit operands
        _linear("linear 8192 rows 4096 to 16384 gelu tanh", 8192, 4096, 16384, act="gelu_tanh"),
        _linear("linear 8192 rows 8192 to 8192 e4m3 +residual", 8192, 8192, 8192, "e4m3", residual=True),
        # the norm in front of a layer for one token, of a residual stream, in the 8 bits the layer reads
        _norm("rmsnorm one row 4096 +residual e4m3", 1, 4096, "e4m3", residual=True),
        # the norm over the 32 channels of every pixel of the benchmark's frame
        _norm("rmsnorm frame 32", FRAME, 32),
        # rows of an odd number of channels: every other row starts off a 4 byte boundary
        _norm("rmsnorm ragged 1001 rows of 5001 +residual", 1001, 5001, residual=True),
        # a long prompt's residual stream
        _norm("rmsnorm 16384 rows of 4096 +residual e4m3", 16384, 4096, "e4m3", residual=True),
    ]


_MOST_FLOPS = 2 * 8192 ** 3
_MOST_BYTES = 600e6


def _size(rng, lo, hi):
    """A size in lo .. hi, spread over its logarithm; two in three are multiples of 8, 16 or 64, the others are as drawn."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    step = rng.choice([8, 16, 64, 64, 1, 1])
    return min(hi, max(lo, n // step * step)) if n >= step else n


def draw(rng):
    while True:
        dtype = rng.choice(["f16", "e4m3"])
        if rng.random() < 0.6:
            kind = rng.random()
            if kind < 0.35:  # single tokens
                rows, c_in, c_out = rng.randint(1, 64), _size(rng, 64, 16384), _size(rng, 64, 16384)
            elif kind < 0.8:  # prompts
                rows, c_in, c_out = _size(rng, 65, 16384), _size(rng, 64, 16384), _size(rng, 64, 16384)
            else:  # pixels
                rows, c_in, c_out = _size(rng, 4096, FRAME), _size(rng, 3, 256), _size(rng, 3, 256)
            case = _linear(None, rows, c_in, c_out, dtype, rng.choice(["none", "relu", "leaky", "gelu", "gelu_tanh", "silu"]),
                           rng.random() < 0.5, rng.random() < 0.5)
        elif rng.random() < 0.7:
            case = _norm(None, _size(rng, 1, 32768), _size(rng, 64, 32768), dtype, rng.random() < 0.5)
        else:  # pixels
            case = _norm(None, _size(rng, 4096, FRAME), _size(rng, 3, 256), dtype, rng.random() < 0.5)
        w = work(case)
        if w["flops"] <= _MOST_FLOPS and w["bytes"] <= _MOST_BYTES:
            return case


def work(case):
    m = case["rows"]
    if case["op"] == "linear":
        k, n, f16 = case["c_in"], case["c_out"], case["dtype"] == "f16"
        b = (m * k + n * k) * (2 if f16 else 1) + 2 * m * n * (2 if case["residual"] else 1)
        b += (2 * n if case["bias"] else 0) + (0 if f16 else 4 * (m + n))
        return {"bytes": b, "flops": 2 * m * n * k}
    c, f16 = case["channels"], case["dtype"] == "f16"
    b = 2 * m * c * (3 if case["residual"] else 1) + m * c * (2 if f16 else 1) + 2 * c + (0 if f16 else 4 * m)
    return {"bytes": b, "flops": 4 * m * c}


def _e4m3_rows(t):
    """Rows quantised as a program keeps them: 8 bit values and what one unit of them stands for, per row."""
    scale = t.abs().amax(1).clamp_min(1e-12) / E4M3_MAX
    return (t / scale[:, None]).to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    half = dict(device="cuda", dtype=torch.float16)

    def normal(*shape):
        return torch.randn(*shape, generator=g, **half)

    m, s = case["rows"], {"case": case}
    if case["op"] == "linear":
        k, n = case["c_in"], case["c_out"]
        x, w = normal(m, k), normal(n, k) * (1.0 / math.sqrt(k))
        if case["dtype"] == "e4m3":
            s["x"], s["x_scale"] = _e4m3_rows(x.float())
            s["w"], s["w_scale"] = _e4m3_rows(w.float())
        else:
            s["x"], s["w"], s["x_scale"], s["w_scale"] = x, w, None, None
        s["bias"] = normal(n) * 0.1 if case["bias"] else None
        s["residual"] = normal(m, n) if case["residual"] else None
        s["out"] = torch.empty(m, n, **half)
    else:
        c = case["channels"]
        s["x"] = normal(m, c)
        s["residual"] = normal(m, c) * 2.0 if case["residual"] else None
        s["weight"] = 1.0 + 0.2 * normal(c)
        s["sum"] = torch.empty(m, c, **half) if case["residual"] else None
        f16 = case["dtype"] == "f16"
        s["out"] = torch.empty(m, c, device="cuda", dtype=torch.float16 if f16 else torch.float8_e4m3fn)
        s["scale"] = None if f16 else torch.empty(m, device="cuda", dtype=torch.float32)
    if own:
        s["call"] = _own_call(s)
    return s


def _own_call(s):
    """What a program keeps of a layer beside its buffers: the linear layer's plan, the norm's descriptor."""
    from denox_b200 import lib

    def ptr(t):
        return None if t is None else t.data_ptr()

    case = s["case"]
    dtype = {"f16": lib.DT_F16, "e4m3": lib.DT_E4M3}[case["dtype"]]
    if case["op"] == "rmsnorm":
        return lib.rmsnorm_desc(case["rows"], case["channels"], ptr(s["x"]), ptr(s["out"]), out_dtype=dtype, eps=EPS,
                                residual=ptr(s["residual"]), weight=ptr(s["weight"]), sum_out=ptr(s["sum"]),
                                out_scale=ptr(s["scale"]))
    act = {"none": lib.ACT_NONE, "relu": lib.ACT_RELU, "leaky": lib.ACT_LEAKY, "gelu": lib.ACT_GELU,
           "gelu_tanh": lib.ACT_GELU_TANH, "silu": lib.ACT_SILU}[case["act"]]
    return lib.LinearPlan(lib.linear_desc(case["rows"], case["c_in"], case["c_out"], ptr(s["x"]), ptr(s["w"]),
                                          ptr(s["out"]), dtype=dtype, activation=act, leaky_alpha=LEAKY_ALPHA,
                                          x_scale=ptr(s["x_scale"]), w_scale=ptr(s["w_scale"]), bias=ptr(s["bias"]),
                                          residual=ptr(s["residual"])))


def _run_own(s):
    from denox_b200 import lib
    stream = torch.cuda.current_stream().cuda_stream
    if s["case"]["op"] == "linear":
        s["call"].launch(stream)
        return s["out"]
    lib.rmsnorm(s["call"], stream)
    return [t for t in (s["out"], s["scale"], s["sum"]) if t is not None]


def _act(t, kind):
    if kind == "relu":
        return t.clamp_min(0.0)
    if kind == "leaky":
        return torch.maximum(t, LEAKY_ALPHA * t)
    if kind == "gelu":
        return 0.5 * t * (1.0 + torch.erf(t * math.sqrt(0.5)))
    if kind == "gelu_tanh":
        return 0.5 * t * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (t + 0.044715 * t * t * t)))
    if kind == "silu":
        return t / (1.0 + torch.exp(-t))
    return t


def run(s):
    if own:
        return _run_own(s)
    case = s["case"]
    if case["op"] == "linear":
        y = s["x"].float() @ s["w"].float().t()
        if s["x_scale"] is not None:
            y = y * s["x_scale"][:, None] * s["w_scale"]
        if s["bias"] is not None:
            y = y + s["bias"].float()
        y = _act(y, case["act"])
        if s["residual"] is not None:
            y = y + s["residual"].float()
        return y.half()
    h = s["x"].float()
    if s["residual"] is not None:
        h = h + s["residual"].float()
    y = h * torch.rsqrt((h * h).mean(1, keepdim=True) + EPS) * s["weight"].float()
    if case["dtype"] == "f16":
        out = [y.half()]
    else:
        top = y.abs().amax(1)
        scale = torch.where(top > 0, top / E4M3_MAX, torch.ones_like(top))
        out = [(y / scale[:, None]).to(torch.float8_e4m3fn), scale]
    return out + ([h.half()] if s["residual"] is not None else [])


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        y = torch.empty(case["rows"], case["c_out"], device="cuda", dtype=torch.float64)
        wt = s["w"].to(torch.float64).t().contiguous()
        if s["w_scale"] is not None:
            wt.mul_(s["w_scale"].to(torch.float64))
        step = max(1, (1 << 28) // (case["c_in"] + case["c_out"]))
        for r in range(0, case["rows"], step):
            rows = slice(r, min(case["rows"], r + step))
            a = s["x"][rows].to(torch.float64)
            if s["x_scale"] is not None:
                a.mul_(s["x_scale"][rows, None].to(torch.float64))
            z = torch.mm(a, wt)
            if s["bias"] is not None:
                z.add_(s["bias"].to(torch.float64))
            if case["act"] == "relu":
                z = torch.where(z > 0, z, torch.zeros_like(z))
            elif case["act"] == "leaky":
                z = torch.where(z > 0, z, z * LEAKY_ALPHA)
            elif case["act"] == "gelu":
                z = z * torch.special.ndtr(z)
            elif case["act"] == "gelu_tanh":  # (1 + tanh u) / 2 is the logistic function of 2 u
                z = z * torch.special.expit(z * (1.0 + 0.044715 * z.square()) * math.sqrt(8.0 / math.pi))
            elif case["act"] == "silu":
                z = z * torch.special.expit(z)
            if s["residual"] is not None:
                z.add_(s["residual"][rows].to(torch.float64))
            y[rows] = z
        return y
    h = s["x"].to(torch.float64)
    if s["residual"] is not None:
        h += s["residual"].to(torch.float64)
    rms = torch.sqrt(torch.linalg.vector_norm(h, dim=1) ** 2 / case["channels"] + EPS)
    y = h * s["weight"].to(torch.float64) / rms[:, None]
    if case["dtype"] == "f16":
        out = [y]
    else:
        scale = torch.linalg.vector_norm(y, ord=math.inf, dim=1) / E4M3_MAX
        scale[scale == 0] = 1.0
        out = [y / scale[:, None], scale]
    return out + ([h] if s["residual"] is not None else [])
