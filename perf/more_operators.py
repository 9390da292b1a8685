"""Performance cases of what a decoder layer does around its products: the operators between a block's output and the next block's input.

Every case is a dict of plain values; "op" says which operator one pass goes through:

  norm         a block's output, normed, gated and scaled, added to the residual stream, and the norm of the sum (launch_add_norm)
  rope         norms and rotary positions of a step's queries and keys (launch_rope_qk)
  route        experts of each token and their weights from the router's logits (launch_moe_route)
  linear       rows quantized to 8 bits with one scale each, times 8-bit weights with one scale for each output channel (linear_w8a8)
  norm_linear  the way into a block: launch_add_norm, which quantizes the rows that it norms, and their product (launch_gemm_w8a8)

Values follow from the seed, everything else from the case alone.  The path is inference only: it has no backward.
"""
import importlib
import math

import torch

DEV = "cuda"
own = False
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
FLT_MAX = torch.finfo(torch.float32).max
INF = float("inf")
MOST_FLOPS = 3.66e11                # of a drawn product: what the largest listed one has


def listed():
    return [
        # one decode token between two blocks: the smallest call, latency only
        {"name": "norm_1", "op": "norm", "S": 1, "K": 5120, "dtype": "fp32", "y_dtype": "fp32", "variant": 0, "post": -1, "gate": "", "alpha": 1.0},
        # batched decode of a layer that norms the block's output too, 16-bit stream, fp32 products
        {"name": "norm_post_33", "op": "norm", "S": 33, "K": 3840, "dtype": "bf16", "y_dtype": "fp32", "variant": 1, "post": 1, "gate": "", "alpha": 1.0},
        # a prefill chunk, a gate for each channel and a residual scale: memory traffic only
        {"name": "norm_gate_8192", "op": "norm", "S": 8192, "K": 5120, "dtype": "fp32", "y_dtype": "fp32", "variant": 0, "post": -1, "gate": "channel", "alpha": 0.22},
        # decode of 64 requests deep in long contexts, queries and keys normed first
        {"name": "rope_64", "op": "rope", "T": 64, "pad": 3, "far": 131072, "Hq": 32, "Hkv": 8, "D": 128, "rotary": 128, "interleaved": 0, "variant": 0, "scaling": "bands", "dtype": "fp32"},
        # a prompt, half of each head rotated, interleaved pairs, positions stretched for a long context
        {"name": "rope_8000", "op": "rope", "T": 8000, "pad": 0, "far": 8000, "Hq": 32, "Hkv": 8, "D": 128, "rotary": 64, "interleaved": 1, "variant": -1, "scaling": "yarn", "dtype": "bf16"},
        # batched decode in front of the routed-expert block
        {"name": "route_8", "op": "route", "S": 8, "E": 128, "topk": 8, "scoring": "softmax", "bias": 0, "groups": 1, "topk_groups": 1, "group_score": "max", "renormalise": 1,
         "scale": 1.0, "masked": 0, "dtype": "fp32"},
        # a prefill chunk, experts in groups, balanced by a bias, some of them switched off
        {"name": "route_4096", "op": "route", "S": 4096, "E": 256, "topk": 8, "scoring": "sigmoid", "bias": 1, "groups": 8, "topk_groups": 4, "group_score": "sum2", "renormalise": 1,
         "scale": 2.5, "masked": 1, "dtype": "fp32"},
        # single-stream decode of a layer that is kept at 8 bits
        {"name": "linear_1", "op": "linear", "M": 1, "N": 17408, "K": 5120, "bias": 0, "x_dtype": "fp32", "y_dtype": "fp32"},
        # batched decode, few outputs from long rows
        {"name": "linear_16", "op": "linear", "M": 16, "N": 3840, "K": 15360, "bias": 0, "x_dtype": "bf16", "y_dtype": "bf16"},
        # a short prompt of ragged length, ragged outputs, a bias
        {"name": "linear_333", "op": "linear", "M": 333, "N": 4091, "K": 3840, "bias": 1, "x_dtype": "fp16", "y_dtype": "fp32"},
        # a prefill chunk
        {"name": "linear_2048", "op": "linear", "M": 2048, "N": 17408, "K": 5120, "bias": 0, "x_dtype": "fp32", "y_dtype": "fp32"},
        # verify step of speculative decoding entering a layer: the QKV product of the normed rows
        {"name": "norm_linear_64", "op": "norm_linear", "S": 64, "K": 5120, "N": 6144, "dtype": "fp32", "y_dtype": "fp32", "variant": 0, "post": -1, "gate": "", "alpha": 1.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _k(rng, lo, hi):
    return max(lo, 32 * (_log(rng, lo, hi) // 32))


def _type(rng):
    return rng.choice(("fp32", "fp32", "fp16", "bf16"))


def draw(rng):
    for _ in range(1000):
        c = _draw(rng)
        w = work(c)
        if w["flops"] <= MOST_FLOPS and w["bytes"] <= 6.8e8:
            return c
    raise RuntimeError("no case in the range")


def _norm_of(rng):
    dt = _type(rng)
    return {"dtype": dt, "y_dtype": rng.choice((dt, dt, "fp32")), "variant": rng.choice((0, 0, 1, 2)), "post": rng.choice((-1, -1, 0, 1, 2)),
            "gate": rng.choice(("", "", "channel", "token")), "alpha": rng.choice((1.0, 1.0, 0.22, 0.5))}


def _draw(rng):
    op = rng.choice(("norm", "norm", "rope", "rope", "route", "route", "linear", "linear", "linear", "norm_linear"))
    if op == "norm":
        return {"op": op, "S": _log(rng, 1, 8192), "K": _k(rng, 256, 16384)} | _norm_of(rng)
    if op == "rope":
        D = rng.choice((64, 80, 96, 128, 128, 128, 256))
        Hkv = rng.choice((1, 2, 4, 8))
        T = _log(rng, 1, 8192)
        return {"op": op, "T": T, "pad": rng.choice((0, 0, 3)), "far": T + _log(rng, 1, 1000000), "Hq": Hkv * rng.choice((1, 3, 4, 5, 7, 8)), "Hkv": Hkv, "D": D,
                "rotary": rng.choice((D, D, 8 * rng.randint(1, D // 8))), "interleaved": rng.choice((0, 0, 1)), "variant": rng.choice((-1, 0, 1, 2)),
                "scaling": rng.choice(("none", "linear", "ntk", "yarn", "bands")), "dtype": _type(rng)}
    if op == "route":
        E = rng.choice((8, 16, 60, 64, 96, 128, 160, 256, 384, 512))
        groups = rng.choice([g for g in (1, 1, 2, 4, 8) if E % g == 0 and E // g >= 2])
        topk_groups = rng.randint(1, groups)
        return {"op": op, "S": _log(rng, 1, 8192), "E": E, "topk": rng.randint(1, min(16, E // groups * topk_groups)), "scoring": rng.choice(("softmax", "sigmoid")), "bias": rng.choice((0, 1)),
                "groups": groups, "topk_groups": topk_groups, "group_score": rng.choice(("max", "sum2")), "renormalise": rng.choice((0, 1, 1)), "scale": rng.choice((1.0, 2.5)),
                "masked": rng.choice((0, 0, 1)), "dtype": _type(rng)}
    if op == "linear":
        return {"op": op, "M": _log(rng, 1, 4096), "N": _log(rng, 256, 20000), "K": _k(rng, 256, 16384), "bias": rng.choice((0, 1)), "x_dtype": _type(rng), "y_dtype": _type(rng)}
    return {"op": op, "S": _log(rng, 1, 2048), "K": _k(rng, 2048, 8192), "N": _log(rng, 1024, 17408)} | _norm_of(rng)


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) % (1 << 62))
    return g


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV)


def _scaling(c):
    """Base and parameters of the rotary frequencies: a context of 8192 tokens stretched eight times."""
    return 10000.0 if c["scaling"] == "yarn" else 500000.0, {"none": {}, "linear": {"factor": 8.0}, "ntk": {"factor": 8.0}, "yarn": {"factor": 8.0, "original": 8192.0},
                                                          "bands": {"factor": 8.0, "original": 8192.0}}[c["scaling"]]


def _norm_state(c, g):
    S, K = c["S"], c["K"]
    s = {"h": (_randn(g, S, K) * torch.exp(0.5 * _randn(g, S, 1))).to(DTYPES[c["dtype"]]), "y": (0.7 * _randn(g, S, K)).to(DTYPES[c["y_dtype"]])}
    weight = lambda variant: None if variant in (-1, 2) else (0.2 * _randn(g, K) + (1.0 if variant == 0 else 0.0))
    s["w"], s["post_w"] = weight(c["variant"]), weight(c["post"])
    s["gate"] = {"": None, "channel": _randn(g, K), "token": _randn(g, S, K)}[c["gate"]] if c["gate"] else None
    s["h_out"] = torch.empty_like(s["h"])
    if own:
        s["norm"] = importlib.import_module("dgx-serving_b200").Norm.of(K, s["w"], c["variant"], 1e-6, s["post_w"], c["post"], s["gate"], c["alpha"], c["dtype"], c["y_dtype"])
    return s


def _weights(c, g):
    """8-bit weights of N channels as a file holds them, and room for the rows' codes."""
    N, K, M = c["N"], c["K"], c.get("M", c.get("S"))
    return {"wq": (40.0 * _randn(g, N, K)).round_().clamp_(-127, 127).to(torch.int8), "ws": 5e-4 * torch.exp(0.3 * _randn(g, N)),
            "xq": torch.empty((M, K), dtype=torch.int8, device=DEV), "xs": torch.empty(M, device=DEV), "out": torch.empty((M, N), dtype=DTYPES[c["y_dtype"]], device=DEV)}


def prepare(case, seed):
    c, g = case, _gen(seed)
    s = {"case": c}
    if c["op"] == "norm":
        s |= _norm_state(c, g)
        s["n"] = torch.empty_like(s["h"])
    elif c["op"] == "rope":
        T, D, cols = c["T"] + c["pad"], c["D"], (c["Hq"] + 2 * c["Hkv"]) * c["D"]
        s["rows"] = _randn(g, T, cols).to(DTYPES[c["dtype"]])                        # queries, keys and values of a token side by side
        if c["far"] == c["T"]:
            s["position"] = torch.arange(T, dtype=torch.int32, device=DEV)
        else:                                                                        # requests anywhere in their contexts
            s["position"] = torch.randint(0, c["far"], (T,), generator=g, device=DEV, dtype=torch.int32)
        s["position"][c["T"]:] = -1                                                  # rows of a padded step that no request owns
        for n in ("q_w", "k_w"):
            s[n] = None if c["variant"] in (-1, 2) else 0.2 * _randn(g, D) + (1.0 if c["variant"] == 0 else 0.0)
        s["q_out"] = torch.zeros((T, c["Hq"] * D), dtype=s["rows"].dtype, device=DEV)
        s["k_out"] = torch.zeros((T, c["Hkv"] * D), dtype=s["rows"].dtype, device=DEV)
        if own:
            w = importlib.import_module("dgx-serving_b200")
            base, more = _scaling(c)
            s["rope"] = w.Rope.of(D, c["rotary"], base, c["scaling"], bool(c["interleaved"]), s["q_w"], s["k_w"], c["variant"], 1e-6, device=DEV, **more)
    elif c["op"] == "route":
        s["logits"] = (1.5 * _randn(g, c["S"], c["E"])).to(DTYPES[c["dtype"]])
        if c["masked"]:
            s["logits"][:, torch.randperm(c["E"], generator=g, device=DEV)[: c["E"] // 8]] = -INF
        s["bias"] = 0.1 * _randn(g, c["E"]) if c["bias"] else None
        s["idx"] = torch.empty((c["S"], c["topk"]), dtype=torch.int32, device=DEV)
        s["weight"] = torch.empty((c["S"], c["topk"]), device=DEV)
        if own:
            s["router"] = importlib.import_module("dgx-serving_b200").Router.of(c["E"], c["topk"], c["scoring"], s["bias"], c["groups"], c["topk_groups"], c["group_score"],
                                                                                bool(c["renormalise"]), c["scale"])
    elif c["op"] == "linear":
        s["x"] = (_randn(g, c["M"], c["K"]) * torch.exp(0.5 * _randn(g, c["M"], 1))).to(DTYPES[c["x_dtype"]])
        s["b"] = _randn(g, c["N"]) if c["bias"] else None
        s |= _weights(c, g)
    else:
        s |= _norm_state(c, g)
        s |= _weights(c, g)
    return s


def run(s):
    c = s["case"]
    if own:
        return _own(s, c, importlib.import_module("dgx-serving_b200"))
    return {"norm": _norm, "rope": _rope, "route": _route, "linear": _linear, "norm_linear": _norm_linear}[c["op"]](s, c)


def _own(s, c, w):
    if c["op"] == "norm":
        w.launch_add_norm(s["norm"], s["h"], s["y"], c["S"], H_out=s["h_out"], N=s["n"])
        return {"h": s["h_out"], "n": s["n"]}
    if c["op"] == "rope":
        rows, Hq, Hkv, D = s["rows"], c["Hq"], c["Hkv"], c["D"]
        cols = (Hq + 2 * Hkv) * D
        w.launch_rope_qk(s["rope"], rows, cols, Hq, rows[:, Hq * D:], cols, Hkv, s["position"], c["T"] + c["pad"], s["q_out"], Hq * D, s["k_out"], Hkv * D, c["dtype"])
        return {"q": s["q_out"], "k": s["k_out"]}
    if c["op"] == "route":
        w.launch_moe_route(s["router"], s["logits"], c["E"], c["S"], s["idx"], s["weight"], c["dtype"])
        return {"idx": s["idx"], "weight": s["weight"]}
    if c["op"] == "linear":
        w.linear_w8a8(s["x"], c["K"], s["xq"], s["xs"], s["wq"], s["ws"], s["out"], c["N"], c["M"], c["N"], c["K"], c["x_dtype"], c["y_dtype"], bias=s["b"])
        return s["out"]
    w.launch_add_norm(s["norm"], s["h"], s["y"], c["S"], H_out=s["h_out"], xq=s["xq"], xs=s["xs"], group=0)
    w.launch_gemm_w8a8(s["xq"], s["xs"], s["wq"], s["ws"], s["out"], c["N"], c["S"], c["N"], c["K"], c["y_dtype"])
    return {"h": s["h_out"], "y": s["out"]}


def _normed(x, weight, variant):
    """x * r * weight; the sum of squares, which is long, and r in 64 bits, and r rounded once."""
    if variant == -1:
        return x
    r = (1.0 / torch.sqrt(x.double().square().mean(-1, keepdim=True) + 1e-6)).float()
    x = x * r
    return x if variant == 2 else x * (weight if variant == 0 else 1.0 + weight)


def _add_norm(s, c):
    p = _normed(s["y"].float(), s["post_w"], c["post"])
    p = (p if s["gate"] is None else p * s["gate"]) * c["alpha"]
    h = s["h"].float() + p
    return h, _normed(h, s["w"], c["variant"])


def _norm(s, c):
    h, n = _add_norm(s, c)
    return {"h": h.to(s["h"].dtype), "n": n.to(s["h"].dtype)}


def _frequencies(c):
    """Radians a token of each pair, in 64 bits, and what cosine and sine are multiplied by."""
    base, p = _scaling(c)
    R, kind = c["rotary"], c["scaling"]
    if kind == "ntk":                                      # the base that stretches the longest wave by the factor
        base = base * p["factor"] ** (R / max(1, R - 2))
    f = base ** (-torch.arange(0, R, 2, dtype=torch.float64, device=DEV) / R)
    if kind == "linear":
        f = f / p["factor"]
    if kind == "yarn":                                     # pairs of more than 32 turns in the original context as they are, of less than one interpolated
        at = lambda turns: R * math.log(p["original"] / (turns * 2 * math.pi)) / (2 * math.log(base))
        lo, hi = max(0, math.floor(at(32.0))), min(R - 1, math.ceil(at(1.0)))
        ramp = ((torch.arange(R // 2, dtype=torch.float64, device=DEV) - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        f = f / p["factor"] * ramp + f * (1 - ramp)
    if kind == "bands":                                    # the same by wave lengths: one and four waves in the original context
        ramp = ((p["original"] * f / (2 * math.pi) - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        f = f / p["factor"] * (1 - ramp) + f * ramp
    return f, 0.1 * math.log(p["factor"]) + 1.0 if kind == "yarn" else 1.0


def _turned(x, cos, sin, c):
    """x [T, H, D] with the first `rotary` elements of each head turned by the angles cos, sin [T, rotary / 2]."""
    R = c["rotary"]
    cos, sin = cos[:, None], sin[:, None]
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if c["interleaved"] else (x[..., : R // 2], x[..., R // 2: R])
    u, v = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((u, v), -1).flatten(-2) if c["interleaved"] else torch.cat((u, v), -1)
    return torch.cat((turned, x[..., R:]), -1)


def _rope(s, c):
    T, Hq, Hkv, D = s["rows"].shape[0], c["Hq"], c["Hkv"], c["D"]
    f, magnitude = _frequencies(c)
    angle = s["position"].double()[:, None] * f            # far positions: an angle in 32 bits has no digits left behind the point
    cos, sin = (torch.cos(angle) * magnitude).float(), (torch.sin(angle) * magnitude).float()
    x = s["rows"].float().view(T, Hq + 2 * Hkv, D)
    q = _turned(_normed(x[:, :Hq], s["q_w"], c["variant"]), cos, sin, c)
    k = _turned(_normed(x[:, Hq:Hq + Hkv], s["k_w"], c["variant"]), cos, sin, c)
    there = (s["position"] >= 0)[:, None]
    return {"q": torch.where(there, q.reshape(T, -1).to(s["rows"].dtype), s["q_out"]), "k": torch.where(there, k.reshape(T, -1).to(s["rows"].dtype), s["k_out"])}


def _route(s, c):
    x = s["logits"].double().nan_to_num(nan=-INF, posinf=FLT_MAX, neginf=-INF)
    S, E, G = c["S"], c["E"], c["groups"]
    # choices are made between values that may lie next to one another: in 64 bits
    if c["scoring"] == "softmax":
        top = x.amax(1, keepdim=True)
        e = torch.exp(x - torch.where(top == -INF, torch.zeros_like(top), top))
        total = e.sum(1, keepdim=True)
        score = torch.where(total > 0, e / total, e)
    else:
        score = 1.0 / (1.0 + torch.exp(-x))
    by_logit = c["scoring"] == "softmax" and s["bias"] is None and c["group_score"] == "max"
    choice = x if by_logit else score if s["bias"] is None else score + s["bias"].double()
    if c["topk_groups"] < G:
        members = choice.view(S, G, E // G)
        group = members.amax(2) if c["group_score"] == "max" else members.topk(2, 2).values.sum(2)
        best = torch.sort(group, dim=1, descending=True, stable=True).indices[:, : c["topk_groups"]]
        open_ = torch.zeros_like(group, dtype=torch.bool).scatter_(1, best, True).repeat_interleave(E // G, 1)
        order = torch.sort(choice, dim=1, descending=True, stable=True).indices
        order = order.gather(1, torch.sort((~open_.gather(1, order)).to(torch.int32), dim=1, stable=True).indices)
    else:
        order = torch.sort(choice, dim=1, descending=True, stable=True).indices
    idx = order[:, : c["topk"]]
    weight = score.gather(1, idx)
    if c["renormalise"]:
        total = weight.sum(1, keepdim=True)
        weight = torch.where(total > 0, weight / total, weight)
    return {"idx": idx.to(torch.int32), "weight": (weight * c["scale"]).float()}


def _codes(x):
    """Rows as whole numbers in units of a row's scale, the largest magnitude / 127; a row of zeros has the scale 0."""
    scale = x.abs().amax(1, keepdim=True) / torch.full_like(x[:, :1], 127.0)
    return torch.where(scale > 0, torch.round(x / scale), torch.zeros_like(x)).clamp(-127, 127), scale


def _product(s, x):
    q, scale = _codes(x)
    return q @ s["wq"].float().T * scale * s["ws"]


def _linear(s, c):
    y = _product(s, s["x"].float())
    return (y if s["b"] is None else y + s["b"]).to(s["out"].dtype)


def _norm_linear(s, c):
    h, n = _add_norm(s, c)
    return {"h": h.to(s["h"].dtype), "y": _product(s, n).to(s["out"].dtype)}


def work(case):
    c = case
    size = {"fp32": 4, "fp16": 2, "bf16": 2}
    if c["op"] in ("norm", "norm_linear"):
        S, K = c["S"], c["K"]
        vectors = 4 * K * ((c["variant"] in (0, 1)) + (c["post"] in (0, 1)) + (c["gate"] == "channel"))
        rows = S * K * (2 * size[c["dtype"]] + size[c["y_dtype"]] + (4 if c["gate"] == "token" else 0))
        if c["op"] == "norm":
            return {"bytes": float(rows + S * K * size[c["dtype"]] + vectors), "flops": 0.0}
        return {"bytes": float(rows + vectors + c["N"] * (K + 4) + S * c["N"] * size[c["y_dtype"]]), "flops": 2.0 * S * c["N"] * K}
    if c["op"] == "rope":
        return {"bytes": 2.0 * c["T"] * (c["Hq"] + c["Hkv"]) * c["D"] * size[c["dtype"]] + 4.0 * (c["T"] + c["pad"]), "flops": 0.0}
    if c["op"] == "route":
        return {"bytes": float(c["S"] * (c["E"] * size[c["dtype"]] + 8 * c["topk"]) + 4 * c["E"] * c["bias"]), "flops": 0.0}
    return {"bytes": float(c["M"] * c["K"] * size[c["x_dtype"]] + c["N"] * (c["K"] + 4 + 4 * c["bias"]) + c["M"] * c["N"] * size[c["y_dtype"]]), "flops": 2.0 * c["M"] * c["N"] * c["K"]}


def _exact_norm(x, weight, variant, rounded):
    """The norm of x in 64 bits.  rounded: with the roundings to fp32 that belong to the definition where codes are made of the result."""
    if variant == -1:
        return x
    at = (lambda v: v.float().double()) if rounded else (lambda v: v)
    factor = at(torch.rsqrt((x * x).sum(1, keepdim=True) / x.shape[1] + 1e-6))
    x = at(x * factor)
    if variant == 2:
        return x
    return at(x * at(weight.double() + (1.0 if variant == 1 else 0.0)))


def _exact_sum(s, c, rounded):
    at = (lambda v: v.float().double()) if rounded else (lambda v: v)
    add = _exact_norm(s["y"].double(), s["post_w"], c["post"], rounded)
    if s["gate"] is not None:
        add = at(add * s["gate"].double())
    add = at(add * float(torch.tensor(c["alpha"], dtype=torch.float32)))
    return at(s["h"].double() + add)


def _exact_product(s, x, bias):
    scale = (x.abs().amax(1) / 127).float().double()
    unit = torch.where(scale > 0, scale, torch.ones_like(scale))[:, None]
    codes = (x / unit).float().double().round().clamp(-127, 127)      # the quotient that is rounded to a code is an fp32 number, as the scale is
    y = (codes @ s["wq"].double().T) * scale[:, None] * s["ws"].double()[None, :]
    return y if bias is None else y + bias.double()


def exact(case, seed):
    c = case
    s = prepare(c, seed)
    if c["op"] == "norm":
        h = _exact_sum(s, c, False)
        return {"h": h, "n": _exact_norm(h, s["w"], c["variant"], False)}
    if c["op"] == "linear":
        return _exact_product(s, s["x"].double(), s["b"])
    if c["op"] == "norm_linear":
        h = _exact_sum(s, c, True)
        return {"h": _exact_sum(s, c, False), "y": _exact_product(s, _exact_norm(h, s["w"], c["variant"], True), None)}
    if c["op"] == "route":
        x = s["logits"].double()
        idx = _route(s, c)["idx"].long()                               # whole numbers have no exact form of their own; the weights follow from them
        p = torch.softmax(x, 1) if c["scoring"] == "softmax" else torch.sigmoid(x)
        w = torch.gather(p, 1, idx)
        if c["renormalise"]:
            w = w / w.sum(1, keepdim=True)
        return {"idx": None, "weight": w * c["scale"]}
    T, D, R, p = s["rows"].shape[0], c["D"], c["rotary"], _scaling(c)
    f = torch.empty(R // 2, dtype=torch.float64)
    for i in range(R // 2):
        base = p[0] * p[1]["factor"] ** (R / max(1, R - 2)) if c["scaling"] == "ntk" else p[0]
        f[i] = math.exp(-2 * i / R * math.log(base))
        if c["scaling"] == "linear":
            f[i] /= p[1]["factor"]
        elif c["scaling"] == "yarn":
            first, last = (R * math.log(p[1]["original"] / (2 * math.pi * t)) / (2 * math.log(base)) for t in (32, 1))
            first, last = max(0, math.floor(first)), min(R - 1, math.ceil(last))
            part = min(1.0, max(0.0, (i - first) / max(last - first, 1e-3)))
            f[i] *= 1 - part + part / p[1]["factor"]
        elif c["scaling"] == "bands":
            waves = p[1]["original"] * float(f[i]) / (2 * math.pi)
            part = min(1.0, max(0.0, (waves - 1) / 3))
            f[i] *= part + (1 - part) / p[1]["factor"]
    z = torch.polar(torch.full((T, R // 2), 0.1 * math.log(p[1]["factor"]) + 1 if c["scaling"] == "yarn" else 1.0, dtype=torch.float64, device=DEV),
                    s["position"].double()[:, None] * f.to(DEV)[None, :])[:, None, :]
    out = {}
    for name, lo, n, w in (("q", 0, c["Hq"], s["q_w"]), ("k", c["Hq"], c["Hkv"], s["k_w"])):
        x = s["rows"][:, lo * D:(lo + n) * D].double().reshape(T * n, D)
        x = _exact_norm(x, w, c["variant"], False).view(T, n, D).clone()
        pair = (slice(0, R, 2), slice(1, R, 2)) if c["interleaved"] else (slice(0, R // 2), slice(R // 2, R))
        t = torch.complex(x[..., pair[0]].contiguous(), x[..., pair[1]].contiguous()) * z
        x[..., pair[0]], x[..., pair[1]] = t.real, t.imag
        x[s["position"] < 0] = 0.0
        out[name] = x.reshape(T, n * D)
    return out
