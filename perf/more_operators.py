"""Products whose activations stay in bf16, as timed cases.

Three operators belong together: the projection on bf16 weights with bias,
activation and residual in its epilogue; the gated pair of such projections
(a bf16 MLP, a shared expert); and a whole mixture-of-experts layer for up to
16 tokens on block-scaled FP8 experts (e4m3 codes, one scale per 128 x 128
block): route, gate/up, SwiGLU, down, combine, residual. Widths are those of
the repository's benchmark and tests (4096 / 12288, 5120 / 17408, experts of
hidden 2048 and width 768) and generic ones that end inside every tile.

The plain form is elementary torch in 32 bits, rounded once at the end;
exact() is the definition in 64 bits on the same inputs.
"""
import math
import os
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F8 = torch.float8_e4m3fn
BF16 = torch.bfloat16
BLOCK = 128


def _clef():
    package = os.path.join(_ROOT, "clef-hrx_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import clef_i4

    return clef_i4


def _linear(name, m, k, n, bias=None, act=None, residual=False, out="bf16"):
    return {"name": name, "kind": "linear", "m": m, "k": k, "n": n, "bias": bias, "act": act, "residual": residual,
            "out": out}


def _gate_up(name, m, k, n, act="silu", bias=None):
    return {"name": name, "kind": "gate_up", "m": m, "k": k, "n": n, "act": act, "bias": bias}


def _moe(name, t, hidden, inter, experts, topk, scales, router, residual):
    return {"name": name, "kind": "moe", "t": t, "hidden": hidden, "inter": inter, "experts": experts, "topk": topk,
            "scales": scales, "router": router, "residual": residual}


def listed():
    return [
        # The router gate of one decoded token, logits kept in f32: the smallest call.
        _linear("linear_m1_router", 1, 2048, 128, out="f32"),
        # One decoded token through the MLP's first projection: the weight stream.
        _linear("linear_m1", 1, 4096, 12288, bias="bf16", act="gelu"),
        # 37 decode streams, output projection with its residual; a width and a
        # depth that end inside a tile.
        _linear("linear_m37_ragged_res", 37, 4160, 1353, bias="f32", residual=True),
        # Rows of an odd width, which start at any even byte.
        _linear("linear_m235_odd", 235, 1001, 333, bias="bf16", act="relu"),
        # The MLP's down projection over a 620-token prompt.
        _linear("linear_m620_res", 620, 17408, 5120, residual=True),
        # A full prefill chunk through the benchmark's projection.
        _linear("linear_m4096", 4096, 4096, 12288, bias="bf16", act="gelu_tanh"),
        # The shared expert of one decoded token.
        _gate_up("gate_up_m1", 1, 2048, 768),
        # Gate and up projections over a prompt of 1711 tokens, GeGLU with biases.
        _gate_up("gate_up_m1711", 1711, 5120, 17408, act="gelu_tanh", bias="bf16"),
        # The experts of one decoded token, the router's logits in hand.
        _moe("moe_t1", 1, 2048, 768, 128, 8, "e8m0", False, False),
        # The whole block of one decoded token: router projection, experts, residual.
        _moe("moe_t1_router_res", 1, 2048, 768, 128, 8, "f32", True, True),
        # Five streams through fewer experts of widths that end inside a block.
        _moe("moe_t5_ragged", 5, 1000, 520, 60, 4, "f32", True, True),
        # Sixteen streams: most experts are named, many by several tokens.
        _moe("moe_t16", 16, 2048, 768, 128, 8, "e8m0", False, True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _by8(rng, lo, hi):
    """A multiple of 8, log-uniform in [lo, hi]."""
    return max(lo, min(hi, _log(rng, lo, hi) // 8 * 8))


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear", "gate_up", "moe", "moe"])
    if kind == "moe":
        experts = rng.choice([8, 32, 60, 64, 128])
        c = _moe(None, rng.randint(1, 16), _by8(rng, 256, 4096), _by8(rng, 256, 2048), experts,
                 rng.choice([1, 2, 4, 6, 8]), rng.choice(["f32", "e8m0"]), rng.random() < 0.5, rng.random() < 0.5)
        while c["experts"] * c["hidden"] * c["inter"] > 128 * 2048 * 768:
            big = "hidden" if c["hidden"] > c["inter"] else "inter"
            c[big] = max(256, c[big] // 2 // 8 * 8)
    else:
        m, k, n = _log(rng, 1, 8192), _by8(rng, 64, 17408), _log(rng, 32, 17408)
        odd = rng.random() < 0.15
        if odd:  # rows that start at any even byte: the unusual layout, at moderate sizes
            m, k = min(m, 512), min(k, 2048) + 1
        bias = rng.choice([None, "bf16", "f32"])
        if kind == "linear":
            c = _linear(None, m, k, n, bias, rng.choice([None, None, "relu", "gelu", "gelu_tanh", "silu"]),
                        rng.random() < 0.5, rng.choice(["bf16", "bf16", "f32"]))
        else:
            c = _gate_up(None, m, k, n, rng.choice(["silu", "silu", "gelu", "gelu_tanh", "sigmoid"]), bias)
        most = 4096 * 4096 * 12288 if kind == "linear" else 1711 * 5120 * 17408
        while c["m"] * c["k"] * c["n"] > most:
            c["m"] = (c["m"] + 1) // 2
    del c["name"]
    return c


# ---------------------------------------------------------------- inputs

def _blocks(width):
    return (width + BLOCK - 1) // BLOCK


def _rows(rows, width, gen):
    """bf16 rows as a model has them behind a norm: normal, each row with its
    own size, and a few columns many times larger."""
    x = torch.randn(rows, width, generator=gen, device="cuda")
    x *= torch.exp(0.5 * torch.randn(rows, 1, generator=gen, device="cuda"))
    big = torch.rand(width, generator=gen, device="cuda") < 0.004
    return (x * torch.where(big, 20.0, 1.0)).to(BF16)


def _dense(rows, cols, gen):
    return (torch.randn(rows, cols, generator=gen, device="cuda") * 0.02).to(BF16)


def _bias(n, kind, gen):
    b = torch.randn(n, generator=gen, device="cuda") * 0.5
    return b.to(BF16) if kind == "bf16" else b


def _experts(count, rows, cols, scales, gen):
    """e4m3 codes [count][rows][cols] of normal weights, and their scales
    [count][ceil(rows / 128)][ceil(cols / 128)]: amax / 448 of each block in
    f32, or the power of two at or above it as e8m0."""
    codes = torch.empty(count, rows, cols, dtype=F8, device="cuda")
    nb, kb = _blocks(rows), _blocks(cols)
    scale = torch.empty(count, nb, kb, device="cuda")
    for first in range(0, count, 16):
        part = min(16, count - first)
        w = torch.zeros(part, nb * BLOCK, kb * BLOCK, device="cuda")
        w[:, :rows, :cols] = torch.randn(part, rows, cols, generator=gen, device="cuda") * 0.02
        w = w.view(part, nb, BLOCK, kb, BLOCK)
        s = w.abs().amax((2, 4)) / 448.0
        if scales == "e8m0":
            s = torch.exp2(torch.ceil(torch.log2(s)))
        q = (w / s[:, :, None, :, None]).clamp(-448.0, 448.0).to(F8)
        codes[first:first + part] = q.view(part, nb * BLOCK, kb * BLOCK)[:, :rows, :cols]
        scale[first:first + part] = s
    return codes, scale.to(torch.float8_e8m0fnu) if scales == "e8m0" else scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    if case["kind"] == "moe":
        t, hidden, inter, experts = (case[i] for i in ("t", "hidden", "inter", "experts"))
        s["x"] = _rows(t, hidden, gen)
        if case["router"]:
            s["router_w"] = _dense(experts, hidden, gen)
        else:
            s["logits"] = torch.randn(t, experts, generator=gen, device="cuda")
        s["weights"] = [_experts(experts, r, c, case["scales"], gen)
                        for r, c in ((inter, hidden), (inter, hidden), (hidden, inter))]
        if case["residual"]:
            s["res"] = torch.randn(t, hidden, generator=gen, device="cuda").to(BF16)
        if own:
            # what a loader keeps: the experts in the kernels' layout
            clef = _clef()
            s["layer"] = clef.MoeLayerF8(*[clef.f8_weight(c, w) for c, w in s["weights"]], topk=case["topk"],
                                         router=s.get("router_w"))
        return s
    s["x"] = _rows(case["m"], case["k"], gen)
    count = 2 if case["kind"] == "gate_up" else 1
    s["weights"] = [_dense(case["n"], case["k"], gen) for _ in range(count)]
    s["biases"] = [_bias(case["n"], case["bias"], gen) if case["bias"] else None for _ in range(count)]
    if case.get("residual"):
        s["res"] = torch.randn(case["m"], case["n"], generator=gen, device="cuda").to(BF16)
    return s


# ---------------------------------------------------------------- the passes

def run(s):
    kind = s["kind"]
    if own:
        clef = _clef()
        if kind == "linear":
            return clef.linear(s["x"], s["weights"][0], bias=s["biases"][0], activation=s["act"],
                               residual=s.get("res"), dtype=torch.float32 if s["out"] == "f32" else BF16)
        if kind == "gate_up":
            return clef.linear_gate_up(s["x"], s["weights"][0], s["weights"][1], activation=s["act"],
                                       gate_bias=s["biases"][0], up_bias=s["biases"][1])
        return s["layer"].decode(s["x"], s.get("logits"), residual=s.get("res"))
    if kind == "moe":
        return _moe_plain(s)
    x = s["x"].float()
    sums = []
    for w, b in zip(s["weights"], s["biases"]):
        y = x @ w.float().t()
        sums.append(y if b is None else y + b.float())
    y = _act(sums[0], s["act"])
    if kind == "gate_up":
        return (y * sums[1]).to(BF16)
    if "res" in s:
        y = y + s["res"].float()
    return y if s["out"] == "f32" else y.to(BF16)


def _act(v, name):
    if name == "relu":
        return torch.where(v > 0, v, torch.zeros_like(v))
    if name == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))
    if name == "silu":
        return v / (1.0 + torch.exp(-v))
    if name == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-v))
    return v


def _named(codes, scale, ids):
    """The weights of the experts `ids`, f32 [len(ids)][rows][cols]."""
    _, rows, cols = codes.shape
    wide = scale[ids].float().repeat_interleave(BLOCK, 1)[:, :rows].repeat_interleave(BLOCK, 2)[:, :, :cols]
    return codes.view(torch.uint8)[ids].view(F8).float() * wide


def _moe_plain(s):
    x, k = s["x"].float(), s["topk"]
    logits = x @ s["router_w"].float().t() if s["router"] else s["logits"]
    top, ids = torch.sort(logits, dim=1, descending=True, stable=True)  # ties: the lower id
    p = torch.exp(top[:, :k] - top[:, :1])
    p = p / p.sum(1, keepdim=True)
    rows = []
    for t in range(s["t"]):
        gate, up, down = (_named(*w, ids[t, :k]) for w in s["weights"])
        g, u = (gate * x[t]).sum(-1), (up * x[t]).sum(-1)
        h = g / (1.0 + torch.exp(-g)) * u
        rows.append(((down * h[:, None, :]).sum(-1) * p[t, :, None]).sum(0))
    y = torch.stack(rows)
    return (y + s["res"].float() if "res" in s else y).to(BF16)


# ---------------------------------------------------------------- bounds and the definition

def work(case):
    if case["kind"] == "moe":
        t, hidden, inter, experts, topk = (case[i] for i in ("t", "hidden", "inter", "experts", "topk"))
        # the experts that a token names, taken as evenly chosen
        named = experts * (1.0 - (1.0 - topk / experts) ** t)
        scales = 3 * _blocks(hidden) * _blocks(inter) * (1 if case["scales"] == "e8m0" else 4)
        nbytes = named * (3 * hidden * inter + scales) + 2 * t * hidden * (3 if case["residual"] else 2)
        nbytes += 2 * experts * hidden if case["router"] else 4 * t * experts
        flops = 6 * t * topk * hidden * inter + (2 * t * experts * hidden if case["router"] else 0)
        return {"bytes": nbytes, "flops": flops}
    m, k, n = case["m"], case["k"], case["n"]
    mats = 2 if case["kind"] == "gate_up" else 1
    nbytes = 2 * m * k + mats * 2 * n * k + m * n * (4 if case.get("out") == "f32" else 2)
    nbytes += mats * n * {None: 0, "bf16": 2, "f32": 4}[case["bias"]]
    return {"bytes": nbytes + (2 * m * n if case.get("residual") else 0), "flops": 2 * m * n * k * mats}


def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].double()

    def phi(v, name):
        if name == "relu":
            return v.clamp(min=0.0)
        if name == "gelu":
            return v * torch.special.ndtr(v)
        if name == "gelu_tanh":
            return v * torch.sigmoid(math.sqrt(8.0 / math.pi) * (v + 0.044715 * v ** 3))
        if name == "silu":
            return v * torch.sigmoid(v)
        return torch.sigmoid(v) if name == "sigmoid" else v

    if case["kind"] != "moe":
        y = [x @ w.double().T + (0.0 if b is None else b.double()) for w, b in zip(s["weights"], s["biases"])]
        out = phi(y[0], case["act"])
        if len(y) == 2:
            return out * y[1]
        return out + s["res"].double() if "res" in s else out

    def weight64(codes, scale, e):
        c = codes[e].double()
        r = torch.arange(c.shape[0], device="cuda") // BLOCK
        q = torch.arange(c.shape[1], device="cuda") // BLOCK
        return c * scale[e].double()[r[:, None], q[None, :]]

    logits = x @ s["router_w"].double().T if case["router"] else s["logits"].double()
    out = s["res"].double() if "res" in s else torch.zeros_like(x)
    for t, row in enumerate(logits.tolist()):
        best = sorted(range(len(row)), key=lambda e: (-row[e], e))[:case["topk"]]
        p = [math.exp(row[e] - row[best[0]]) for e in best]
        for e, pe in zip(best, p):
            gate, up, down = (weight64(*w, e) for w in s["weights"])
            g = gate @ x[t]
            out[t] += pe / sum(p) * (down @ (g * torch.sigmoid(g) * (up @ x[t])))
    return out
