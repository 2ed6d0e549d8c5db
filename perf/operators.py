"""The block-scaled FP8 operators as timed cases.

Values are e4m3 with one scale for each block of 128 along k: an activation
row has a scale for every 128 columns, a weight one for every 128 x 128 block
(f32, or a power of two held as e8m0). Four operators belong together: the
quantizer of activation rows, the projection (plain, with a residual, gate/up
with SwiGLU; the activation comes in as bf16 and is quantized by the call),
the listing of a router's choices by expert, and the experts' products over
those lists. Widths are those of the repository's benchmark and tests (4096 /
12288, 5120 / 17408, experts of hidden 2048 and width 768) and generic ones
that end inside a block.

The plain form is elementary torch in 32 bits; exact() is the definition in 64
bits on the same inputs: y = sum over blocks of (sum of code products) times
both scales, SwiGLU silu(gate) * up of the unrounded sums, a bf16 residual
added, one rounding at the end.
"""
import math
import os
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F8 = torch.float8_e4m3fn
BLOCK = 128


def _clef():
    package = os.path.join(_ROOT, "clef-hrx_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import clef_i4

    return clef_i4


def listed():
    return [
        # The router's input of one decoded token: the smallest quantizer call.
        {"name": "quantize_m1", "kind": "quantize", "m": 1, "k": 2048},
        # Hidden rows of a prefill chunk in front of the MLP's down projection.
        {"name": "quantize_m4096", "kind": "quantize", "m": 4096, "k": 12288},
        # One decoded token through a projection: latency and the weight stream.
        {"name": "linear_m1", "kind": "linear", "m": 1, "k": 4096, "n": 12288, "residual": False, "scales": "e8m0"},
        # 37 decode streams, output projection with its residual, a width and a
        # depth that end inside a block; a checkpoint's f32 scales.
        {"name": "linear_m37_ragged_res", "kind": "linear", "m": 37, "k": 4160, "n": 1352, "residual": True,
         "scales": "f32"},
        # The MLP's down projection over a 620-token prompt.
        {"name": "linear_m620_res", "kind": "linear", "m": 620, "k": 17408, "n": 5120, "residual": True,
         "scales": "f32"},
        # A full prefill chunk through the benchmark's projection.
        {"name": "linear_m4096", "kind": "linear", "m": 4096, "k": 4096, "n": 12288, "residual": False,
         "scales": "e8m0"},
        # Gate and up projections with SwiGLU of the same model as m620, a
        # prompt of 1711 tokens.
        {"name": "gate_up_m1711", "kind": "gate_up", "m": 1711, "k": 5120, "n": 17408, "scales": "f32"},
        # The router's choices of a 235-token prompt listed by expert.
        {"name": "group_t235", "kind": "group", "t": 235, "experts": 128, "topk": 8, "skew": 0.0},
        # A packed batch of long prompts with uneven routing.
        {"name": "group_t65536_skewed", "kind": "group", "t": 65536, "experts": 128, "topk": 8, "skew": 1.0},
        # The experts of one decoded token: gate/up with SwiGLU.
        {"name": "experts_gate_up_t1", "kind": "experts_gate_up", "t": 1, "k": 2048, "n": 768, "experts": 128,
         "topk": 8, "skew": 0.0, "scales": "e8m0"},
        # Uneven routing of a 700-token prompt, the experts' down products.
        {"name": "experts_down_t700_skewed", "kind": "experts_down", "t": 700, "k": 768, "n": 2048, "experts": 128,
         "topk": 8, "skew": 1.0, "scales": "f32"},
        # A full prefill chunk through the experts' gate/up.
        {"name": "experts_gate_up_t4096", "kind": "experts_gate_up", "t": 4096, "k": 2048, "n": 768, "experts": 128,
         "topk": 8, "skew": 0.0, "scales": "e8m0"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _by8(rng, lo, hi):
    """A multiple of 8, log-uniform in [lo, hi]."""
    return max(lo, min(hi, _log(rng, lo, hi) // 8 * 8))


def draw(rng):
    kind = rng.choice(["quantize", "linear", "linear", "linear", "gate_up", "group", "experts_gate_up",
                       "experts_gate_up", "experts_down", "experts_down"])
    if kind == "quantize":
        c = {"kind": kind, "m": _log(rng, 1, 16384), "k": _by8(rng, 256, 17408)}
        while c["m"] * c["k"] > 4096 * 12288:
            c["m"] = (c["m"] + 1) // 2
        return c
    if kind in ("linear", "gate_up"):
        c = {"kind": kind, "m": _log(rng, 1, 8192), "k": _by8(rng, 256, 17408), "n": _by8(rng, 256, 17408),
             "scales": rng.choice(["f32", "e8m0"])}
        if kind == "linear":
            c["residual"] = rng.random() < 0.5
        most = 4096 * 4096 * 12288 if kind == "linear" else 1711 * 5120 * 17408
        while c["m"] * c["k"] * c["n"] > most:
            c["m"] = (c["m"] + 1) // 2
        return c
    experts = rng.choice([8, 32, 60, 64, 128])
    topk = rng.choice([1, 2, 4, 6, 8])
    skew = rng.choice([0.0, 0.5, 1.0])
    if kind == "group":
        return {"kind": kind, "t": _log(rng, 1, 65536), "experts": experts, "topk": topk, "skew": skew}
    c = {"kind": kind, "t": _log(rng, 1, 4096), "k": _by8(rng, 256, 4096), "n": _by8(rng, 256, 4096),
         "experts": experts, "topk": topk, "skew": skew, "scales": rng.choice(["f32", "e8m0"])}
    gu = 2 if kind == "experts_gate_up" else 1
    while c["experts"] * c["k"] * c["n"] * gu > 128 * 2048 * 1536:
        c["n"] = max(256, c["n"] // 2 // 8 * 8)
        c["k"] = c["k"] if c["n"] > 256 else max(256, c["k"] // 2 // 8 * 8)
    while c["t"] * c["topk"] * c["k"] * c["n"] * gu > 32768 * 2048 * 1536:
        c["t"] = (c["t"] + 1) // 2
    return c


# ---------------------------------------------------------------- inputs

def _blocks(width):
    return (width + BLOCK - 1) // BLOCK


def _activation(rows, width, gen):
    """bf16 rows as a model has them behind a norm: normal, each row with its
    own size, and a few columns many times larger."""
    x = torch.randn(rows, width, generator=gen, device="cuda")
    x *= torch.exp(0.5 * torch.randn(rows, 1, generator=gen, device="cuda"))
    big = torch.rand(width, generator=gen, device="cuda") < 0.004
    return (x * torch.where(big, 20.0, 1.0)).to(torch.bfloat16)


def _weight(count, rows, cols, scales, gen):
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


def _routes(t, experts, topk, skew, gen):
    """A router's answer [t][2 * topk]: distinct expert ids as f32, then their
    probabilities."""
    logits = torch.randn(t, experts, generator=gen, device="cuda")
    logits += 2.0 * skew * torch.randn(experts, generator=gen, device="cuda")
    top, ids = logits.topk(topk, dim=1)
    return torch.cat([ids.float(), torch.softmax(top, 1)], 1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    kind = case["kind"]
    if kind in ("quantize", "linear", "gate_up"):
        s["x"] = _activation(case["m"], case["k"], gen)
    if kind == "group":
        s["routes"] = _routes(case["t"], case["experts"], case["topk"], case["skew"], gen)
    if kind in ("linear", "gate_up"):
        s["weights"] = [_weight(1, case["n"], case["k"], case["scales"], gen)
                        for _ in range(2 if kind == "gate_up" else 1)]
        if case.get("residual"):
            s["res"] = torch.randn(case["m"], case["n"], generator=gen, device="cuda").to(torch.bfloat16)
    if kind.startswith("experts"):
        routes = _routes(case["t"], case["experts"], case["topk"], case["skew"], gen)
        s["offsets"], s["slots"] = _lists(routes, case["experts"])
        s["longest"] = int((s["offsets"][1:] - s["offsets"][:-1]).max())  # the plain form's padding
        s["x"] = _activation(case["t"] * (case["topk"] if kind == "experts_down" else 1), case["k"], gen)
        s["a"] = _quantize(s["x"])
        s["weights"] = [_weight(case["experts"], case["n"], case["k"], case["scales"], gen)
                        for _ in range(2 if kind == "experts_gate_up" else 1)]
    if own:
        # what a loader keeps: the weights in the kernels' layout; the experts'
        # activations as the quantizer left them
        clef = _clef()
        if "weights" in s:
            s["packed"] = [clef.f8_weight(c, w) for c, w in s["weights"]]
        if kind.startswith("experts"):
            s["prepared"] = clef.prepare_f8(s["x"])
    return s


# ---------------------------------------------------------------- the passes

def run(s):
    kind = s["kind"]
    if own:
        clef = _clef()
        if kind == "quantize":
            a = clef.prepare_f8(s["x"])
            return {"codes": a.codes, "scales": a.scales}
        if kind == "linear":
            return clef.project_quantized_f8(s["x"], s["packed"][0], residual=s.get("res"))
        if kind == "gate_up":
            return clef.project_gate_up_f8(clef.prepare_f8(s["x"]), s["packed"][0], s["packed"][1])
        if kind == "group":
            offsets, slots = clef.omni_group_slots(s["routes"], s["experts"])
            return {"offsets": offsets, "slots": slots}
        if kind == "experts_gate_up":
            return clef.expert_gate_up_f8(s["prepared"], s["packed"][0], s["packed"][1], s["offsets"], s["slots"],
                                          s["topk"])
        return clef.expert_f8(s["prepared"], s["packed"][0], s["offsets"], s["slots"], s["topk"], input_routed=True)
    if kind == "quantize":
        codes, scales = _quantize(s["x"])
        return {"codes": codes, "scales": scales}
    if kind == "linear":
        y = _spread(*_quantize(s["x"])) @ _weight_f32(*s["weights"][0])[0].t()
        return (y + s["res"].float() if "res" in s else y).to(torch.bfloat16)
    if kind == "gate_up":
        a = _spread(*_quantize(s["x"]))
        g, u = a @ _weight_f32(*s["weights"][0])[0].t(), a @ _weight_f32(*s["weights"][1])[0].t()
        return (g / (1.0 + torch.exp(-g)) * u).to(torch.bfloat16)
    if kind == "group":
        offsets, slots = _lists(s["routes"], s["experts"])
        return {"offsets": offsets, "slots": slots}
    gu = kind == "experts_gate_up"
    offsets, slots = s["offsets"].long(), s["slots"].long()
    place = offsets[:-1, None] + torch.arange(s["longest"], device="cuda")
    listed_here = place < offsets[1:, None]
    slot = slots[place.clamp(max=slots.numel() - 1)]
    a = _spread(*s["a"])[slot // s["topk"] if gu else slot] * listed_here[..., None]
    y = [torch.bmm(a, _weight_f32(*w).transpose(1, 2).contiguous()) for w in s["weights"]]
    y = (y[0] / (1.0 + torch.exp(-y[0])) * y[1] if gu else y[0]).to(torch.bfloat16)
    total = slots.numel()
    out = torch.empty(total + 1, s["n"], dtype=torch.bfloat16, device="cuda")
    out[torch.where(listed_here, slot, total).view(-1)] = y.view(-1, s["n"])
    return out[:total]


def _quantize(x):
    """e4m3 codes [rows][width] and f32 scales [rows][ceil(width / 128)]: the
    scale is the power of two at or above amax / 448 of the block (blocks
    below 2^-118 count as that), so x / scale is exact and the only rounding
    is e4m3's."""
    rows, width = x.shape
    v = torch.zeros(rows, _blocks(width) * BLOCK, device="cuda")
    v[:, :width] = x
    v = v.view(rows, -1, BLOCK)
    part, exponent = torch.frexp(v.abs().amax(-1).clamp(min=2.0 ** -118))
    exponent = exponent - 9 + (part > 0.875)  # amax = part * 2^exponent, part in [0.5, 1); 448 = 0.875 * 2^9
    scale, inverse = (((127 + e) << 23).to(torch.int32).view(torch.float32) for e in (exponent, -exponent))
    return (v * inverse[..., None]).view(rows, -1)[:, :width].to(F8), scale


def _spread(codes, scale):
    """The rows that codes and block scales stand for, f32."""
    rows, width = codes.shape
    return codes.float() * scale.float().repeat_interleave(BLOCK, 1)[:, :width]


def _weight_f32(codes, scale):
    """The weights that codes and block scales stand for, f32 [count][rows][cols]."""
    _, rows, cols = codes.shape
    wide = scale.float().repeat_interleave(BLOCK, 1)[:, :rows].repeat_interleave(BLOCK, 2)[:, :, :cols]
    return codes.float() * wide


def _lists(routes, experts):
    """The route ordinals t * topk + r by expert, ascending in each, and the
    places where the experts' lists begin."""
    ids = routes[:, :routes.shape[1] // 2].to(torch.int32).reshape(-1)
    counts = (ids[:, None] == torch.arange(experts, dtype=torch.int32, device="cuda")).sum(0)
    offsets = torch.zeros(experts + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = counts.cumsum(0)
    return offsets, torch.sort(ids, stable=True)[1].to(torch.int32)


# ---------------------------------------------------------------- bounds and the definition

def work(case):
    kind = case["kind"]
    if kind == "group":
        routed = case["t"] * case["topk"]
        return {"bytes": 8 * routed + 4 * (case["experts"] + 1), "flops": 0}
    if kind == "quantize":
        m, k = case["m"], case["k"]
        return {"bytes": 3 * m * k + 4 * m * _blocks(k), "flops": 2 * m * k}
    k, n = case["k"], case["n"]
    if kind in ("linear", "gate_up"):
        m, mats = case["m"], 2 if kind == "gate_up" else 1
        nbytes = 2 * m * k + mats * (n * k + 4 * _blocks(n) * _blocks(k)) + 2 * m * n
        return {"bytes": nbytes + (2 * m * n if case.get("residual") else 0), "flops": 2 * m * n * k * mats}
    # experts: the weights of those that a token names (taken as evenly chosen)
    t, e, mats = case["t"], case["experts"], 2 if kind == "experts_gate_up" else 1
    routed = t * case["topk"]
    named = e * (1.0 - (1.0 - case["topk"] / e) ** t)
    rows = t if mats == 2 else routed
    nbytes = rows * (k + 4 * _blocks(k)) + named * mats * n * k + 4 * (routed + e + 1) + 2 * routed * n
    return {"bytes": nbytes, "flops": 2 * routed * n * k * mats}


def _codes64(x):
    """The quantizer by its definition, in 64 bits: (values, scales)."""
    def two_to(e):
        return ((e.long() + 1023) << 52).view(torch.float64)

    rows, width = x.shape
    v = torch.nn.functional.pad(x.double(), (0, -width % BLOCK)).unflatten(1, (-1, BLOCK))
    part, e = torch.frexp(v.abs().max(-1).values.clamp(min=2.0 ** -118) / 448.0)
    e = torch.where(part == 0.5, e - 1, e)  # the least e with 2^e >= amax / 448
    q = v * two_to(-e)[..., None]
    step = two_to(torch.frexp(q.abs().clamp(min=2.0 ** -6))[1] - 4)  # e4m3: 4 bits, least exponent -6
    return (torch.round(q / step) * step).flatten(1)[:, :width], two_to(e)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "group":
        routes = s["routes"].cpu()
        ids = routes[:, :case["topk"]].reshape(-1).long()
        lists = [torch.nonzero(ids == e).reshape(-1) for e in range(case["experts"])]
        ends = torch.tensor([0] + [len(x) for x in lists]).cumsum(0)
        return {"offsets": ends.int(), "slots": torch.cat(lists).int()}
    if kind == "quantize":
        codes, scale = _codes64(s["x"])
        return {"codes": codes, "scales": scale}

    def rows64(x):
        v, scale = _codes64(x)
        return v * torch.repeat_interleave(scale, BLOCK, dim=1)[:, :v.shape[1]]

    def weight64(codes, scale, e):
        c = codes[e].double()
        r = torch.arange(c.shape[0], device="cuda") // BLOCK
        q = torch.arange(c.shape[1], device="cuda") // BLOCK
        return c * scale[e].double()[r[:, None], q[None, :]]

    x = rows64(s["x"])
    if kind == "linear":
        y = x @ weight64(*s["weights"][0], 0).T
        return y + s["res"].double() if "res" in s else y
    if kind == "gate_up":
        g, u = (x @ weight64(*w, 0).T for w in s["weights"])
        return g * torch.sigmoid(g) * u
    out = torch.zeros(s["slots"].numel(), case["n"], dtype=torch.float64, device="cuda")
    ends = s["offsets"].tolist()
    for e in range(case["experts"]):
        mine = s["slots"][ends[e]:ends[e + 1]].long()
        if len(mine):
            y = [x[mine // case["topk"] if kind == "experts_gate_up" else mine] @ weight64(*w, e).T
                 for w in s["weights"]]
            out[mine] = y[0] * torch.sigmoid(y[0]) * y[1] if len(y) == 2 else y[0]
    return out
