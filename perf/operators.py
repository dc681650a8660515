"""The operators of the 8-bit linear path and of the gated feed-forward projection: their cases and plain forms.

Four operators of a transformer's feed-forward half: the root-mean-square norm with the residual's addition
and an 8-bit output with a scale for each row, the row-wise quantisation alone, the int8 matrix product with
scales for each token and channel, and the gated projection ``act(x Wg) * (x Wu)`` (16-bit with its gradients,
8-bit with scales).  ``own = False`` computes them with elementary torch operations in 32 bits.
"""
import math

import torch

own = False

E4M3 = torch.float8_e4m3fn
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "e4m3": E4M3, "int8": torch.int8}
TOP = {"e4m3": 448.0, "int8": 127.0}
TINY = torch.finfo(torch.float32).tiny
EPS = 1e-6


def listed():
    return [
        # the norm before a layer's feed-forward block when one token is generated: latency alone
        {"name": "norm_one_token", "op": "norm", "m": 1, "n": 4096, "in": "bf16", "out": "e4m3"},
        # the same norm over a prompt's tokens: memory traffic alone
        {"name": "norm_prompt", "op": "norm", "m": 8192, "n": 4096, "in": "bf16", "out": "e4m3"},
        # an odd batch with rows that no vector width divides
        {"name": "norm_odd", "op": "norm", "m": 1237, "n": 5003, "in": "fp16", "out": "e4m3"},
        # the activation between the projections of a feed-forward block, for a batch of single tokens
        {"name": "quantize_tokens", "op": "quantize", "m": 16, "n": 14336, "in": "bf16", "out": "e4m3"},
        # and for a prompt
        {"name": "quantize_prompt", "op": "quantize", "m": 4096, "n": 14336, "in": "bf16", "out": "e4m3"},
        # the down projection in int8 for a batch of single tokens, its 16-bit input quantised in the call
        {"name": "int8_linear_tokens", "op": "int8_linear", "m": 16, "n": 4096, "k": 14336, "in": "bf16"},
        # the up projection in int8 for a ragged batch of prompts
        {"name": "int8_gemm_prompt", "op": "int8_gemm", "m": 2005, "n": 14336, "k": 4096, "out": "bf16"},
        # the square product at which the fp8 GEMM is quoted
        {"name": "int8_gemm_8192", "op": "int8_gemm", "m": 8192, "n": 8192, "k": 8192, "out": "bf16"},
        # both projections of the feed-forward block for a few single tokens: the weights' stream
        {"name": "gated_tokens", "op": "gated8", "m": 8, "k": 4096, "f": 14336, "in": "e4m3", "act": "silu", "out": "bf16"},
        # and for a prompt
        {"name": "gated_prompt", "op": "gated8", "m": 4096, "k": 4096, "f": 14336, "in": "e4m3", "act": "silu", "out": "bf16"},
        # a training step's forward and backward pass through the gated projection
        {"name": "gated_train", "op": "gated_train", "m": 2048, "k": 4096, "f": 14336, "in": "bf16", "act": "silu"},
        # a small odd one in half precision, with the other activation
        {"name": "gated_train_small", "op": "gated_train", "m": 333, "k": 1000, "f": 2728, "in": "fp16", "act": "gelu"},
    ]


def _spread(rng, low, high, step=1):
    """A size between low and high, even in its logarithm, a multiple of step."""
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    return max(step, int(round(v / step)) * step)


def draw(rng):
    op = rng.choice(["norm", "quantize", "int8_linear", "int8_gemm", "gated8", "gated_train"])
    tokens = _spread(rng, 1, 8192)
    if op in ("norm", "quantize"):
        n = _spread(rng, 64, 16384, rng.choice([1, 8, 64]))
        return {"op": op, "m": tokens, "n": n, "in": rng.choice(["bf16", "fp16", "fp32"]), "out": "e4m3"}
    if op == "int8_linear":
        return {"op": op, "m": min(tokens, 4096), "n": _spread(rng, 256, 8192, 8), "k": _spread(rng, 256, 14336, 16), "in": rng.choice(["bf16", "fp16"])}
    if op == "int8_gemm":
        return {"op": op, "m": tokens, "n": _spread(rng, 256, 8192, 8), "k": _spread(rng, 256, 8192, 16), "out": rng.choice(["bf16", "fp16"])}
    act = rng.choice(["silu", "gelu", "gelu_tanh"])
    if op == "gated8":
        return {"op": op, "m": min(tokens, 4096), "k": _spread(rng, 256, 4096, 16), "f": _spread(rng, 256, 14336, 8), "in": rng.choice(["e4m3", "int8"]), "act": act, "out": rng.choice(["bf16", "fp16"])}
    return {"op": op, "m": min(tokens, 2048), "k": _spread(rng, 256, 4096, 8), "f": _spread(rng, 256, 14336, 8), "in": rng.choice(["bf16", "fp16"]), "act": act}


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _codes(g, rows, cols, kind):
    """Rows of 8-bit codes as a quantiser leaves them, and the scales that go with them."""
    if kind == "int8":
        codes = (_randn(g, rows, cols) * 32.0).round_().clamp_(-127, 127).to(torch.int8)
    else:
        codes = (_randn(g, rows, cols) * 100.0).clamp_(-448, 448).to(E4M3)
    scales = torch.rand(rows, generator=g, device="cuda").mul_(0.5).add_(0.75)
    return codes, scales


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c, m = case, case["m"]
    s = {"case": c}
    if c["op"] in ("norm", "quantize"):
        dt = DTYPES[c["in"]]
        s["x"] = _randn(g, m, c["n"]).to(dt)
        if c["op"] == "norm":
            s["residual"] = (_randn(g, m, c["n"]) * 3.0).to(dt)
            s["weight"] = (1.0 + 0.2 * _randn(g, c["n"])).to(dt)
        return s
    k = c["k"]
    if c["op"] in ("int8_linear", "int8_gemm"):
        w, sw = _codes(g, c["n"], k, "int8")  # a weight is stored with its inputs contiguous
        s["w"], s["scale_w"] = w.t(), (sw * (0.02 / 32.0)).reshape(1, -1)
        if c["op"] == "int8_linear":
            s["x"] = _randn(g, m, k).to(DTYPES[c["in"]])
        else:
            x, sx = _codes(g, m, k, "int8")
            s["x"], s["scale_x"] = x, (sx / 32.0).reshape(-1, 1)
        return s
    f = c["f"]
    if c["op"] == "gated8":
        top = 32.0 if c["in"] == "int8" else 100.0
        x, sx = _codes(g, m, k, c["in"])
        s["x"], s["scale_x"] = x, (sx / top).reshape(-1, 1)
        for name in ("gate", "up"):
            w, sw = _codes(g, f, k, c["in"])
            s["w_" + name], s["scale_" + name] = w.t(), (sw * (1.0 / (math.sqrt(k) * top))).reshape(1, -1)
        return s
    dt = DTYPES[c["in"]]
    s["x"] = _randn(g, m, k).to(dt).requires_grad_()
    for name in ("gate", "up"):
        s["w_" + name] = (_randn(g, f, k) / math.sqrt(k)).to(dt).t().requires_grad_()
    s["dh"] = _randn(g, m, f).to(dt)
    return s


def _quantized(y, out):
    scale = (y.abs().amax(dim=1, keepdim=True) / TOP[out]).clamp_min(TINY)
    q = y / scale
    return q.to(E4M3) if out == "e4m3" else q.round().clamp(-127, 127), scale


def _act(g, kind):
    """The activation and its derivative."""
    if kind == "silu":
        s = 1.0 / (1.0 + torch.exp(-g))
        return g * s, s * (1.0 + g * (1.0 - s))
    if kind == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))
    a, b = math.sqrt(2.0 / math.pi), 0.044715
    t = torch.tanh(a * (g + b * g * g * g))
    return 0.5 * g * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * a * (1.0 + 3.0 * b * g * g)


def _plain(s):
    c = s["case"]
    with torch.no_grad():
        if c["op"] == "norm":
            h = s["x"].float() + s["residual"].float()
            y = h * (1.0 / torch.sqrt((h * h).mean(dim=1, keepdim=True) + EPS)) * s["weight"].float()
            return (*_quantized(y, c["out"]), h.to(s["x"].dtype))
        if c["op"] == "quantize":
            return _quantized(s["x"].float(), c["out"])
        if c["op"] == "int8_linear":
            q, scale = _quantized(s["x"].float(), "int8")
            return ((q @ s["w"].float()) * scale * s["scale_w"]).to(s["x"].dtype)
        if c["op"] == "int8_gemm":
            return ((s["x"].float() @ s["w"].float()) * s["scale_x"] * s["scale_w"]).to(DTYPES[c["out"]])
        x, wg, wu = s["x"].float(), s["w_gate"].float(), s["w_up"].float()
        if c["op"] == "gated8":
            g = (x @ wg) * s["scale_x"] * s["scale_gate"]
            u = (x @ wu) * s["scale_x"] * s["scale_up"]
            return (_act(g, c["act"])[0] * u).to(DTYPES[c["out"]])
        g, u, dh = x @ wg, x @ wu, s["dh"].float()
        a, da = _act(g, c["act"])
        dg, du = dh * u * da, dh * a
        got = a * u, dg @ wg.t() + du @ wu.t(), (dg.t() @ x).t(), (du.t() @ x).t()
        return tuple(t.to(s["x"].dtype) for t in got)


def _framework(s):
    import helion_b200 as hb

    c = s["case"]
    if c["op"] == "norm":
        return hb.rms_norm_quantize(s["x"], s["weight"], residual=s["residual"], eps=EPS, out_dtype=DTYPES[c["out"]])
    if c["op"] == "quantize":
        return hb.quantize_rows(s["x"], out_dtype=DTYPES[c["out"]])
    if c["op"] == "int8_linear":
        q, scale = hb.quantize_rows(s["x"], out_dtype=torch.int8)
        return hb.int8_gemm(q, s["w"], scale_a=scale, scale_b=s["scale_w"], out_dtype=s["x"].dtype)
    if c["op"] == "int8_gemm":
        return hb.int8_gemm(s["x"], s["w"], scale_a=s["scale_x"], scale_b=s["scale_w"], out_dtype=DTYPES[c["out"]])
    if c["op"] == "gated8":
        return hb.gated_gemm(
            s["x"], s["w_gate"], s["w_up"], scale_x=s["scale_x"], scale_gate=s["scale_gate"], scale_up=s["scale_up"],
            activation=c["act"], out_dtype=DTYPES[c["out"]],
        )
    h = hb.gated_matmul(s["x"], s["w_gate"], s["w_up"], activation=c["act"])
    return (h.detach(), *torch.autograd.grad(h, (s["x"], s["w_gate"], s["w_up"]), s["dh"]))


def run(state):
    return _framework(state) if own else _plain(state)


def work(case):
    c, m = case, case["m"]
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    if c["op"] == "norm":
        e = size[c["in"]]
        return {"bytes": m * c["n"] * (3 * e + 1) + c["n"] * e + 4 * m, "flops": 8 * m * c["n"]}
    if c["op"] == "quantize":
        return {"bytes": m * c["n"] * (size[c["in"]] + 1) + 4 * m, "flops": 3 * m * c["n"]}
    k = c["k"]
    if c["op"] == "int8_linear":
        return {"bytes": 2 * m * k + k * c["n"] + 4 * c["n"] + 2 * m * c["n"], "flops": 2 * m * k * c["n"]}
    if c["op"] == "int8_gemm":
        return {"bytes": m * k + k * c["n"] + 4 * (m + c["n"]) + 2 * m * c["n"], "flops": 2 * m * k * c["n"]}
    f = c["f"]
    if c["op"] == "gated8":
        return {"bytes": m * k + 2 * k * f + 4 * (m + 2 * f) + 2 * m * f, "flops": 4 * m * k * f}
    # x, dh and both weights in; h, dx and both weights' gradients out
    return {"bytes": 2 * (2 * m * k + 2 * m * f + 4 * k * f), "flops": 12 * m * k * f}


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    d = {k: v.detach().double() for k, v in s.items() if isinstance(v, torch.Tensor)}
    if c["op"] in ("norm", "quantize"):
        h = y = d["x"]
        if c["op"] == "norm":
            h = h + d["residual"]
            y = h / (h.pow(2).mean(1, keepdim=True) + EPS).sqrt() * d["weight"]
        scale = y.abs().max(dim=1, keepdim=True).values / TOP[c["out"]]
        q = (y / scale).to(E4M3).double()
        return (q, scale, h) if c["op"] == "norm" else (q, scale)
    if c["op"] == "int8_linear":
        scale = d["x"].abs().max(dim=1, keepdim=True).values / 127.0
        return torch.matmul(torch.round(d["x"] / scale), d["w"]) * (scale * d["scale_w"])
    if c["op"] == "int8_gemm":
        return torch.matmul(d["x"], d["w"]) * (d["scale_x"] * d["scale_w"])
    if c["op"] == "gated8":
        x = d["x"] * d["scale_x"]
        g, u = x @ (d["w_gate"] * d["scale_gate"]), x @ (d["w_up"] * d["scale_up"])
    else:
        g, u = d["x"] @ d["w_gate"], d["x"] @ d["w_up"]
    if c["act"] == "silu":
        a = g * torch.sigmoid(g)
        da = torch.sigmoid(g) + a * torch.sigmoid(-g)
    elif c["act"] == "gelu":
        cdf = 0.5 * torch.erfc(-g / math.sqrt(2.0))
        a, da = g * cdf, cdf + g * torch.exp(-g.square() / 2.0) / math.sqrt(2.0 * math.pi)
    else:
        # 0.5 (1 + tanh z) is the logistic function of 2 z
        z2 = 2.0 * math.sqrt(2.0 / math.pi) * (g + 0.044715 * g.pow(3))
        p = torch.sigmoid(z2)
        a, da = g * p, p + g * p * torch.sigmoid(-z2) * (2.0 * math.sqrt(2.0 / math.pi) * (1.0 + 3.0 * 0.044715 * g.square()))
    if c["op"] == "gated8":
        return a * u
    dg, du = d["dh"] * u * da, d["dh"] * a
    return a * u, torch.matmul(dg, d["w_gate"].T) + torch.matmul(du, d["w_up"].T), d["x"].T @ dg, d["x"].T @ du
