"""Performance cases of the 8-bit projections of the decoder, through their public entry points.

Every case is one pass through operators of nanokv_amd.q8:

  norm    RMSNorm with the residual's addition, its output held in 8 bits with a
          scale a row (rmsnorm_q8), read back (dequantize_q8);
  quant   rows to 8 bits with a scale and back (quantize_q8, dequantize_q8);
  linear  the product of rows with 8-bit weights: rows are quantised, the product
          is taken in integers and scaled by token and channel (linear_q8);
  gated   the same for a gate|up weight, with SiLU(gate) * up (linear_silu_mul_q8);
  token   the norm in front of a gated product (norm_linear_silu_mul_q8);
  mlp     a decoder layer's second half: norm, gated product, quantised rows,
          product (rmsnorm_q8, linear_silu_mul_q8, linear_q8).

With `own` false `run` computes them in elementary torch operations, in 32 bits;
the sums of a product's integers, which pass 24 bits, in 64.  `exact` restates
each of them in 64 bits.
"""

import math
import os
import sys

import torch

own = False

EPS = 1e-6
TINY = 2.0 ** -119    # rows whose largest magnitude is below are zero
MOST = 4096 * 19456 * 2560    # rows * channels * depth of the largest listed case


def listed():
    return [
        # the norm in front of a projection, one decode token: the smallest call
        {"name": "norm_token", "op": "norm", "m": 1, "k": 2560, "residual": True},
        # the same for a default prompt chunk
        {"name": "norm_chunk", "op": "norm", "m": 4096, "k": 2560, "residual": True},
        # the MLP's hidden rows of a ragged chunk
        {"name": "quant_hidden_1001", "op": "quant", "m": 1001, "k": 9728},
        # q|k|v of one decode token
        {"name": "linear_token_qkv", "op": "linear", "m": 1, "k": 2560, "n": 6144, "bias": False},
        # a norm and the gate|up projection of one decode token
        {"name": "token_gate_up", "op": "token", "m": 1, "k": 2560, "n": 9728, "residual": True},
        # the LM head of one decode token
        {"name": "linear_token_head", "op": "linear", "m": 1, "k": 2560, "n": 151936, "bias": False},
        # gate|up of a speculative round's draft tokens
        {"name": "gated_draft_6", "op": "gated", "m": 6, "k": 2560, "n": 9728},
        # down projection of a prompt's short tail
        {"name": "linear_tail_37", "op": "linear", "m": 37, "k": 9728, "n": 2560, "bias": False},
        # q|k|v with its bias (attention_bias), a short prompt of odd length
        {"name": "linear_301_bias", "op": "linear", "m": 301, "k": 2560, "n": 6144, "bias": True},
        # output projection of a default prompt chunk
        {"name": "linear_chunk_o", "op": "linear", "m": 4096, "k": 4096, "n": 2560, "bias": False},
        # gate|up of a default prompt chunk: the largest call
        {"name": "gated_chunk", "op": "gated", "m": 4096, "k": 2560, "n": 9728},
        # a layer's whole second half on a ragged chunk
        {"name": "mlp_2777", "op": "mlp", "m": 2777, "k": 2560, "n": 9728, "residual": True},
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["norm", "quant", "linear", "linear", "linear", "gated", "gated", "token", "mlp"])
    m = rng.choice([1, rng.randint(2, 16), log_int(17, 4096), log_int(17, 4096)])
    k = 16 * log_int(8, 768)           # 128 .. 12288
    if op == "norm":
        return {"op": op, "m": m, "k": min(k, 8192), "residual": rng.random() < 0.7}
    if op == "quant":
        return {"op": op, "m": m, "k": k}
    if op == "linear":
        n = log_int(100, 32768)
        while m * n * k > MOST:
            n = n // 2
        return {"op": op, "m": m, "k": k, "n": n, "bias": rng.random() < 0.3}
    k = min(k, 8192)
    n = 16 * log_int(16, 768)          # 256 .. 12288 of gate and as many of up
    while 2 * m * n * k > MOST // (2 if op == "mlp" else 1):
        n = n // 32 * 16
    case = {"op": op, "m": min(m, 4) if op == "token" else m, "k": k, "n": n}
    if op != "gated":
        case["residual"] = rng.random() < 0.7
    return case


# -- inputs ------------------------------------------------------------------
def _hidden(g, m, k):
    """Rows of a decoder's residual stream: channels of unequal size, a few of them large."""
    x = torch.randn(m, k, generator=g, device="cuda")
    ch = torch.randn(k, generator=g, device="cuda").mul_(0.6).exp_()
    ch[torch.randint(0, k, (max(1, k // 512),), generator=g, device="cuda")] *= 12.0
    return x.mul_(ch).to(torch.bfloat16)


def _weight(g, n, k):
    """An [n, k] weight as a checkpoint's N(0, 0.02), quantised once as the model does on load."""
    q = torch.empty(n, k, dtype=torch.int8, device="cuda")
    s = torch.empty(n, device="cuda")
    step = max(1, (1 << 26) // k)
    for i in range(0, n, step):
        w = torch.randn(min(step, n - i), k, generator=g, device="cuda").mul_(0.02).to(torch.bfloat16)
        q[i:i + step], s[i:i + step] = _quantize(w.float())
    return q, s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + 17)
    m, k, op = case["m"], case["k"], case["op"]
    s = {"op": op, "x": _hidden(g, m, k), "residual": None, "bias": None}
    if case.get("residual"):
        s["residual"] = (torch.randn(m, k, generator=g, device="cuda") * 2).to(torch.bfloat16)
    if op in ("norm", "token", "mlp"):
        s["norm"] = (1 + 0.2 * torch.randn(k, generator=g, device="cuda")).to(torch.bfloat16)
    if op in ("gated", "token", "mlp"):
        s["w"] = _weight(g, 2 * case["n"], k)
    if op == "linear":
        s["w"] = _weight(g, case["n"], k)
        if case["bias"]:
            s["bias"] = torch.randn(case["n"], generator=g, device="cuda").to(torch.bfloat16)
    if op == "mlp":
        s["down"] = _weight(g, k, case["n"])
    return s


# -- the plain form ----------------------------------------------------------
def _quantize(y):
    """Rows of fp32 -> (int8 codes, fp32 scales)."""
    top = y.abs().amax(dim=-1)
    zero = top < TINY
    inv = torch.where(zero, torch.zeros_like(top), 127.0 / top)
    return torch.round(y * inv[:, None]).to(torch.int8), torch.where(zero, torch.zeros_like(top), top / 127.0)


def _norm(x, weight, residual):
    t = x.float()
    if residual is not None:
        t = t + residual.float()
    y = t * torch.rsqrt((t * t).mean(dim=-1, keepdim=True) + EPS) * weight.float()
    return y, t.to(torch.bfloat16)


def _read_back(q, s):
    return (q.float() * s[:, None]).to(torch.bfloat16)


def _product(q, s, w):
    """fp32 product of quantised rows with a quantised weight; the integers are summed in 64 bits."""
    return (q.double() @ w[0].double().T).float() * s[:, None] * w[1]


def _gated(q, s, w):
    gate, up = _product(q, s, w).chunk(2, dim=-1)
    return (gate / (1.0 + torch.exp(-gate)) * up).to(torch.bfloat16)


def _plain(s):
    op = s["op"]
    if op == "quant":
        q, c = _quantize(s["x"].float())
        return {"values": _read_back(q, c), "scale": c}
    if op == "linear":
        y = _product(*_quantize(s["x"].float()), s["w"])
        if s["bias"] is not None:
            y = y + s["bias"].float()
        return y.to(torch.bfloat16)
    if op == "gated":
        return _gated(*_quantize(s["x"].float()), s["w"])
    y, res = _norm(s["x"], s["norm"], s["residual"])
    q, c = _quantize(y)
    if op == "norm":
        return {"values": _read_back(q, c), "scale": c, "residual": res}
    h = _gated(q, c, s["w"])
    if op == "mlp":
        h = _product(*_quantize(h.float()), s["down"]).to(torch.bfloat16)
    return {"y": h, "residual": res}


def _framework():
    """nanokv_amd.q8, imported once as a program does, not in every pass."""
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nano-vllm-kv-optimizer_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from nanokv_amd import q8
    return q8


def _own(s):
    op, x, res = s["op"], s["x"], s["residual"]
    q8 = sys.modules.get("nanokv_amd.q8") or _framework()
    if op == "quant":
        t = q8.quantize_q8(x)
        return {"values": q8.dequantize_q8(t), "scale": t.scale}
    if op == "linear":
        return q8.linear_q8(x, q8.Q8(*s["w"]), s["bias"])
    if op == "gated":
        return q8.linear_silu_mul_q8(x, q8.Q8(*s["w"]))
    if op == "token":
        y, res = q8.norm_linear_silu_mul_q8(x, s["norm"], EPS, q8.Q8(*s["w"]), residual=res)
        return {"y": y, "residual": res}
    t, res = q8.rmsnorm_q8(x, s["norm"], EPS, residual=res)
    if op == "norm":
        return {"values": q8.dequantize_q8(t), "scale": t.scale, "residual": res}
    h = q8.linear_silu_mul_q8(t, q8.Q8(*s["w"]))
    return {"y": q8.linear_q8(h, q8.Q8(*s["down"])), "residual": res}


def run(state):
    if own:
        return _own(state)
    return _plain(state)


# -- what a pass cannot do without -------------------------------------------
def work(case):
    m, k, op = case["m"], case["k"], case["op"]
    row = 2 * m * k
    rows = row * (2 if case.get("residual") else 1)
    if op == "quant":
        return {"bytes": 2 * row + 4 * m, "flops": 4 * m * k}
    if op == "norm":
        return {"bytes": rows + 2 * k + 2 * row + 4 * m, "flops": 9 * m * k}
    n = case["n"]
    if op == "linear":
        return {"bytes": row + n * k + 4 * n + 2 * m * n + (2 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    if op == "gated":
        return {"bytes": row + 2 * n * k + 8 * n + 2 * m * n, "flops": 4 * m * n * k}
    if op == "token":
        return {"bytes": rows + 2 * k + 2 * n * k + 8 * n + 2 * m * n + row, "flops": 4 * m * n * k}
    return {"bytes": rows + 2 * k + 3 * n * k + 8 * n + 4 * k + 2 * row, "flops": 6 * m * n * k}


# -- in 64 bits --------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]

    def codes(v):      # integers in [-127, 127] and the size of one step, of every row
        peak = v.abs().max(dim=1, keepdim=True).values
        step = torch.where(peak < TINY, 1.0, peak / 127.0)
        return (v / step).round(), torch.where(peak < TINY, 0.0, step)

    def values(v):
        c, step = codes(v)
        return c * step

    def times(v, w):
        return values(v) @ (w[0].double() * w[1].double()[:, None]).t()

    v = s["x"].double()
    res = v
    if s["residual"] is not None:
        res = v = v + s["residual"].double()
    if op in ("norm", "token", "mlp"):
        v = v / (v.square().sum(dim=1, keepdim=True) / case["k"] + EPS).sqrt() * s["norm"].double()
    if op == "quant":
        return {"values": values(v), "scale": codes(v)[1][:, 0]}
    if op == "norm":
        return {"values": values(v), "scale": codes(v)[1][:, 0], "residual": res}
    y = times(v, s["w"])
    if op == "linear":
        return y if s["bias"] is None else y + s["bias"].double()
    n = case["n"]
    y = y[:, :n] * torch.sigmoid(y[:, :n]) * y[:, n:]
    if op == "gated":
        return y
    if op == "mlp":    # its hidden rows are bf16, as a product returns them
        y = times(y.to(torch.bfloat16).double(), s["down"])
    return {"y": y, "residual": res}
