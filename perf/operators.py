"""Performance cases of the 8-bit KV cache: the operators that a serving program calls around the products of a layer.

Every case is a dict of plain values; "op" says which operator one pass goes through:

  plan        block tables and slot maps of a step, built on the GPU from the requests' lengths (kv_plan)
  cache       a step's keys and values written to the 8-bit blocks, and the blocks' tokens that this may have changed read back as
              numbers (launch_kv_append_q8, launch_kv_read_q8): int8 codes with one fp32 scale for each block of tokens and head
  attention   attention of a step's queries over those blocks (launch_attention_q8)

Lengths follow from the case alone (spread over [kv_lo, kv_hi] and [q_lo, q_hi]), values from the seed.  The path is inference only:
it has no backward.
"""
import importlib
import math

import torch

DEV = "cuda"
own = False
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one decode step of a small batch: the next token of 24 requests
        {"name": "plan_decode_24", "op": "plan", "R": 24, "kv_lo": 0, "kv_hi": 4000, "q_lo": 1, "q_hi": 1, "block": 16, "short": 0},
        # a full scheduler step of a large server, prompts and decodes mixed, the free list running out before the last requests
        {"name": "plan_mixed_2048", "op": "plan", "R": 2048, "kv_lo": 0, "kv_hi": 8000, "q_lo": 1, "q_hi": 160, "block": 32, "short": 1},
        # decode: one new token for each of 64 requests, most of them into a partly filled block
        {"name": "cache_decode_64", "op": "cache", "R": 64, "kv_lo": 1, "kv_hi": 4000, "q_lo": 1, "q_hi": 1, "Hkv": 8, "D": 128, "block": 16, "dtype": "fp32"},
        # prefill: the prompts' keys and values, ragged, starting anywhere in a block
        {"name": "cache_prefill_8192", "op": "cache", "R": 5, "kv_lo": 0, "kv_hi": 999, "q_lo": 700, "q_hi": 3000, "Hkv": 8, "D": 128, "block": 16, "dtype": "bf16"},
        # wide heads, larger blocks, chunks of a few dozen tokens
        {"name": "cache_chunks_256", "op": "cache", "R": 33, "kv_lo": 0, "kv_hi": 2000, "q_lo": 7, "q_hi": 130, "Hkv": 2, "D": 256, "block": 64, "dtype": "fp16"},
        # single-stream decode with a short history: the smallest call, latency only
        {"name": "decode_1", "op": "attention", "R": 1, "kv_lo": 413, "kv_hi": 413, "q_lo": 1, "q_hi": 1, "Hq": 32, "Hkv": 8, "D": 128, "block": 16,
         "dtype": "fp32", "causal": 1, "window": 0, "softcap": 0.0},
        # two long documents: few rows, the keys' axis split over the whole GPU
        {"name": "decode_long_2", "op": "attention", "R": 2, "kv_lo": 98001, "kv_hi": 131072, "q_lo": 1, "q_hi": 1, "Hq": 32, "Hkv": 8, "D": 128, "block": 64,
         "dtype": "bf16", "causal": 1, "window": 0, "softcap": 0.0},
        # batched decode, ragged histories
        {"name": "decode_64", "op": "attention", "R": 64, "kv_lo": 200, "kv_hi": 8192, "q_lo": 1, "q_hi": 1, "Hq": 32, "Hkv": 8, "D": 128, "block": 16,
         "dtype": "fp32", "causal": 1, "window": 0, "softcap": 0.0},
        # a sliding-window layer with capped logits and wide heads, large batch
        {"name": "decode_window_128", "op": "attention", "R": 128, "kv_lo": 30, "kv_hi": 4096, "q_lo": 1, "q_hi": 1, "Hq": 16, "Hkv": 2, "D": 256, "block": 32,
         "dtype": "fp16", "causal": 1, "window": 1024, "softcap": 50.0},
        # verify step of speculative decoding: one to eight queries a request, an odd number of heads to a group
        {"name": "verify_16", "op": "attention", "R": 16, "kv_lo": 900, "kv_hi": 6000, "q_lo": 1, "q_hi": 8, "Hq": 28, "Hkv": 4, "D": 128, "block": 16,
         "dtype": "fp32", "causal": 1, "window": 0, "softcap": 0.0},
        # a long prompt in one go
        {"name": "prefill_4096", "op": "attention", "R": 1, "kv_lo": 4096, "kv_hi": 4096, "q_lo": 4096, "q_hi": 4096, "Hq": 32, "Hkv": 8, "D": 128, "block": 64,
         "dtype": "bf16", "causal": 1, "window": 0, "softcap": 0.0},
        # a mixed step: prompt chunks over longer histories next to single tokens
        {"name": "prefill_mixed_9", "op": "attention", "R": 9, "kv_lo": 800, "kv_hi": 5000, "q_lo": 1, "q_hi": 1000, "Hq": 32, "Hkv": 8, "D": 128, "block": 16,
         "dtype": "fp32", "causal": 1, "window": 0, "softcap": 0.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    for _ in range(1000):
        c = _draw(rng)
        if c["op"] != "attention":
            return c
        seq, q = _lengths(c)
        w = work(c)
        pad = len(q) * max(seq)
        if (w["bytes"] <= 7e8 and w["flops"] <= 1.37e11 and pad * c["Hkv"] * c["D"] <= 5.4e8 and pad * max(q) * c["Hq"] <= 1.6e9):
            return c
    raise RuntimeError("no case in the range")


def _draw(rng):
    op = rng.choice(("plan", "cache", "cache", "attention", "attention", "attention", "attention"))
    if op == "plan":
        lo = rng.choice((0, 0, 1, 100))
        return {"op": op, "R": _log(rng, 1, 2048), "kv_lo": lo, "kv_hi": lo + _log(rng, 1, 8000), "q_lo": rng.choice((0, 1)), "q_hi": rng.choice((1, 1, _log(rng, 2, 160))),
                "block": rng.choice((16, 32, 64, 128)), "short": rng.choice((0, 0, 1))}
    D = rng.choice((64, 128, 128, 256))
    Hkv = rng.choice((1, 2, 4, 8))
    c = {"op": op, "D": D, "Hkv": Hkv, "block": rng.choice((16, 32, 64, 128)), "dtype": rng.choice(("fp32", "fp32", "fp16", "bf16"))}
    if op == "cache":
        q_hi = rng.choice((1, 1, _log(rng, 2, 3000)))
        c |= {"R": _log(rng, 1, max(2, min(256, 9000 // q_hi))), "kv_lo": 0, "kv_hi": _log(rng, 1, 4000), "q_lo": min(q_hi, rng.choice((0, 1, 7))), "q_hi": q_hi}
        return c
    kind = rng.choice(("decode", "decode", "few", "prefill"))
    q_hi = {"decode": 1, "few": rng.randint(2, 16), "prefill": _log(rng, 33, 4096)}[kind]
    lo = _log(rng, 1, 4000)
    c |= {"R": _log(rng, 1, {"decode": 128, "few": 32, "prefill": 10}[kind]), "kv_lo": lo, "kv_hi": lo + _log(rng, 1, 131072 - 4000 if rng.random() < 0.2 else 6000),
          "q_lo": rng.choice((1, q_hi)), "q_hi": q_hi, "Hq": Hkv * rng.choice((1, 2, 3, 4, 5, 7, 8)), "causal": rng.choice((1, 1, 1, 0)),
          "window": rng.choice((0, 0, 0, _log(rng, 1, 4096))), "softcap": rng.choice((0.0, 0.0, 30.0))}
    return c


def _lengths(c):
    """Tokens that a request has after the step, and those of them that the step brings: spread over the case's ranges, in no order."""
    seq, new = [], []
    for i in range(c["R"]):
        u, v = (i * 0.6180339887 + 0.37) % 1.0, (i * 0.4142135623 + 0.61) % 1.0
        kv = c["kv_lo"] + int((c["kv_hi"] - c["kv_lo"] + 1) * u)
        q = c["q_hi"] if c["q_lo"] == c["q_hi"] else int(round(max(c["q_lo"], 0.5) * (c["q_hi"] / max(c["q_lo"], 0.5)) ** v))
        seq.append(max(kv, q) if c["op"] == "attention" else kv + q)
        new.append(q)
    return seq, new


def _ceil(a, b):
    return -(-a // b)


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) % (1 << 62))
    return g


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _starts(counts):
    at = [0]
    for n in counts:
        at.append(at[-1] + n)
    return at


def _tables(c, lengths, spare, g):
    """Block tables of requests that hold `lengths` tokens, over a pool in random order; entries past a request's blocks name none (-1).
    Returns the table, the pool's size and the pool's order (the blocks behind the used ones are free)."""
    need = [_ceil(n, c["block"]) for n in lengths]
    width = max(1, max(_ceil(s, c["block"]) for s in _lengths(c)[0]))
    used = sum(need)
    order = torch.randperm(used + spare, generator=g, device=DEV).to(torch.int32)
    need_t, start_t = _ints(need)[:, None], _ints(_starts(need)[:-1])[:, None]
    col = torch.arange(width, device=DEV, dtype=torch.int32)[None, :]
    table = torch.where(col < need_t, order[(start_t + col).clamp(max=max(0, used + spare - 1)).long()], torch.full_like(col, -1))
    return table.contiguous(), used + spare, order


def _pool(c, blocks, used, g):
    """Codes and scales of a pool: what quantizing normal values gives, each block and head with a magnitude of its own.  The scales of
    blocks that no request holds are not numbers."""
    out = []
    for _ in range(2):
        x = torch.randn((blocks, c["Hkv"], c["block"], c["D"]), generator=g, device=DEV, dtype=torch.float16)
        amax = x.abs().amax(dim=(2, 3)).float()
        codes = (x * (127.0 / amax).to(torch.float16)[:, :, None, None]).round_().clamp_(-127, 127).to(torch.int8)
        scale = amax / 127 * torch.exp(0.3 * torch.randn(amax.shape, generator=g, device=DEV))
        out.append((codes, torch.where(used[:, None], scale, torch.full_like(scale, float("nan")))))
    return {"k": out[0][0], "v": out[1][0], "k_scale": out[0][1], "v_scale": out[1][1]}


def prepare(case, seed):
    c, g = case, _gen(seed)
    seq, new = _lengths(c)
    old = [s - n for s, n in zip(seq, new)]
    T = sum(new)
    s = {"case": c, "T": T, "max_q": max(new), "new_len": _ints(new), "kv_len": _ints(old), "cu": _ints(_starts(new))}
    if c["op"] == "plan":
        need = sum(_ceil(a, c["block"]) - _ceil(b, c["block"]) for a, b in zip(seq, old))
        free = max(1, need * 9 // 10) if c["short"] else need + 7
        s["table"], _, order = _tables(c, old, free + 5, g)
        s["free"], s["first"] = order[len(order) - free - 2:].contiguous(), _ints([2])     # the list's first two are taken already
        s["rows"] = T + 3                                                                  # a step padded by three rows
        s |= {"seq_len": torch.empty_like(s["kv_len"]), "cu_new": torch.empty_like(s["cu"]), "status": torch.empty(4, dtype=torch.int32, device=DEV),
              "slot": torch.empty(s["rows"], dtype=torch.int32, device=DEV), "position": torch.empty(s["rows"], dtype=torch.int32, device=DEV)}
        return s
    dt = DTYPES[c["dtype"]]
    s["table"], blocks, order = _tables(c, seq, 9, g)
    used = torch.zeros(blocks, dtype=torch.bool, device=DEV)
    used[order[: blocks - 9].long()] = True
    s |= _pool(c, blocks, used, g)
    if c["op"] == "cache":
        # keys and values as one row of the projections' output holds them: behind the queries' columns
        width = c["Hkv"] * c["D"]
        rows = torch.randn((T, 3 * width), generator=g, device=DEV) * torch.exp(0.5 * torch.randn((T, 1), generator=g, device=DEV))
        s["kv_rows"] = rows.to(dt)
        t = torch.arange(T, device=DEV)
        r = torch.searchsorted(s["cu"][1:].long().contiguous(), t, right=True)
        pos = s["kv_len"][r].long() + t - s["cu"][r].long()
        s["slot"] = (s["table"][r, pos // c["block"]].long() * c["block"] + pos % c["block"]).to(torch.int32)
        s["begin"] = s["kv_len"] // c["block"] * c["block"]
        span = [b - a // c["block"] * c["block"] if b > a else 0 for a, b in zip(old, seq)]
        s["cu_read"], s["n_read"] = _ints(_starts(span)), sum(span)
        s["k_out"] = torch.empty((s["n_read"], c["Hkv"], c["D"]), dtype=dt, device=DEV)
        s["v_out"] = torch.empty_like(s["k_out"])
    else:
        s["seq_len"] = _ints(seq)
        s["q"] = (1.5 * torch.randn((T, c["Hq"], c["D"]), generator=g, device=DEV)).to(dt)
        s["scale"] = c["D"] ** -0.5
        s["out"] = torch.empty_like(s["q"])
    if own:
        w = importlib.import_module("dgx-serving_b200")
        s["cache"] = w.KVCache.of(s["k"], s["v"], s["k_scale"], s["v_scale"])
        if c["op"] == "attention":                        # a program keeps one workspace for all layers; the calls leave it zeroed
            s["workspace"] = torch.zeros(w.attention_q8_workspace_bytes(c["Hq"], s["cache"], T, s["max_q"]), dtype=torch.uint8, device=DEV)
    return s


def run(s):
    c = s["case"]
    if own:
        return _own(s, c, importlib.import_module("dgx-serving_b200"))
    return {"plan": _plan, "cache": _cache, "attention": _attention}[c["op"]](s, c)


def _own(s, c, w):
    if c["op"] == "plan":
        w.kv_plan(s["kv_len"], s["new_len"], c["R"], c["block"], s["table"], s["table"].shape[1], s["free"], s["free"].numel(), s["first"],
                  s["seq_len"], s["cu_new"], s["slot"], s["position"], s["rows"], s["status"])
        return {"table": s["table"], "seq_len": s["seq_len"], "cu": s["cu_new"], "slot": s["slot"], "position": s["position"], "status": s["status"]}
    dt = c["dtype"]
    if c["op"] == "cache":
        width = c["Hkv"] * c["D"]
        rows = s["kv_rows"]
        w.launch_kv_append_q8(rows[:, width:], rows[:, 2 * width:], 3 * width, s["slot"], s["T"], s["cache"], dt)
        w.launch_kv_read_q8(s["cache"], s["table"], s["table"].shape[1], s["begin"], s["cu_read"], c["R"], s["n_read"], s["k_out"], s["v_out"], width, dt)
        return {"k": s["k_out"], "v": s["v_out"]}
    w.launch_attention_q8(s["q"], c["Hq"] * c["D"], s["cache"], s["table"], s["table"].shape[1], s["cu"], s["seq_len"], c["R"], s["T"], c["Hq"],
                          s["out"], c["Hq"] * c["D"], s["scale"], dt, s["workspace"], causal=c["causal"], window=c["window"], softcap=c["softcap"], max_q=s["max_q"])
    return s["out"]


def _plan(s, c):
    B, R, width = c["block"], c["R"], s["table"].shape[1]
    kv, new = s["kv_len"].long(), s["new_len"].long()
    seq = kv + new
    have, want = (kv + B - 1) // B, (seq + B - 1) // B
    need = torch.where(want <= width, want - have, torch.zeros_like(have))
    first = s["first"].long()
    upto = need.cumsum(0)
    served = (want <= width) & ((need == 0) | (upto <= s["free"].numel() - first))
    begin = first + upto - need                                        # a request's first block in the free list
    take = torch.where(served, need, torch.zeros_like(need))
    end = torch.where(take > 0, begin + take, first.expand(R)).amax().clamp(min=first[0])
    col = torch.arange(width, device=DEV)[None, :]
    fresh = (col >= have[:, None]) & (col < (have + take)[:, None])
    src = (begin[:, None] + col - have[:, None]).clamp(0, s["free"].numel() - 1)
    table = torch.where(fresh, s["free"][src], s["table"])
    cu = torch.cat([torch.zeros_like(kv[:1]), new.cumsum(0)])
    t = torch.arange(s["rows"], device=DEV)
    r = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    inside = r < R
    r = r.clamp(max=R - 1)
    inside = inside & served[r]
    pos = kv[r] + t - cu[r]
    slot = table[r, (pos // B).clamp(0, width - 1)].long() * B + pos % B
    none = torch.full_like(slot, -1)
    slot, pos = torch.where(inside, slot, none), torch.where(inside, pos, none)
    status = torch.stack([end, (~served).sum(), take.sum(), torch.where(served, new, torch.zeros_like(new)).sum()])
    return {k: v.to(torch.int32) for k, v in {"table": table, "seq_len": torch.where(served, seq, torch.zeros_like(seq)), "cu": cu, "slot": slot,
                                             "position": pos, "status": status}.items()}


def _quotient(a, b):
    """a / b, 0 where b is 0; both tensors, so that the division is a division."""
    return torch.where(b > 0, a / b, torch.zeros_like(a))


def _write(x, slot, codes, scale, B):
    """The rows x[T, H, D] into their slots.  A block's scale becomes the larger of what it was, if it held tokens before, and its new rows'
    largest magnitude / 127; codes that were there are rounded to the new scale."""
    x = x.float()
    block, off = slot // B, slot % B
    head = torch.ones_like(block, dtype=torch.bool)
    head[1:] = block[1:] != block[:-1]
    group = head.cumsum(0) - 1
    ids, filled = block[head], off[head]
    amax = torch.zeros((ids.numel(), x.shape[1]), device=DEV).index_reduce(0, group, x.abs().amax(2), "amax")
    before = torch.where(filled[:, None] > 0, scale[ids], torch.zeros_like(amax))
    now = torch.maximum(before, amax / torch.full_like(amax, 127.0))
    held = codes[ids].float()
    again = torch.round(held * _quotient(before, now)[:, :, None, None])
    kept = (torch.arange(B, device=DEV)[None, :] < filled[:, None])[:, None, :, None]
    codes[ids] = torch.where(kept, again, held).to(torch.int8)
    scale[ids] = now
    q = torch.round(_quotient(x, now[group][:, :, None].expand_as(x))).clamp(-127, 127)
    codes[block, :, off] = q.to(torch.int8)


def _cache(s, c):
    B, H, D = c["block"], c["Hkv"], c["D"]
    rows, slot = s["kv_rows"].view(s["T"], 3, H, D), s["slot"].long()
    _write(rows[:, 1], slot, s["k"], s["k_scale"], B)
    _write(rows[:, 2], slot, s["v"], s["v_scale"], B)
    t = torch.arange(s["n_read"], device=DEV)
    r = torch.searchsorted(s["cu_read"][1:].contiguous(), t.to(torch.int32), right=True)
    pos = s["begin"][r].long() + t - s["cu_read"][r].long()
    block, off = s["table"][r, pos // B].long(), pos % B
    return {n: (s[n][block, :, off].float() * s[n + "_scale"][block][:, :, None]).to(DTYPES[c["dtype"]]) for n in ("k", "v")}


def _attention(s, c):
    B, R, Hq, H, D = c["block"], c["R"], c["Hq"], c["Hkv"], c["D"]
    n, L = s["max_q"], int(s["table"].shape[1]) * B
    table = s["table"].clamp(min=0).long()
    new, seq, cu = s["new_len"].long(), s["seq_len"].long(), s["cu"].long()

    def rows(codes, scale):                               # [R, H, L, D]; what lies past a request's tokens is 0
        there = (torch.arange(L, device=DEV)[None, :] < seq[:, None]).view(R, -1, 1, B, 1)
        x = torch.where(there, codes[table].float() * scale[table][..., None, None], torch.zeros((), device=DEV))
        return x.transpose(1, 2).reshape(R, H, L, D)

    i = torch.arange(n, device=DEV)[None, :]
    q = s["q"][(cu[:-1, None] + i).clamp(max=max(0, s["T"] - 1))].float()                         # [R, n, Hq, D]
    q = q.transpose(1, 2).reshape(R, H, Hq // H * n, D)
    score = (q @ rows(s["k"], s["k_scale"]).transpose(2, 3)).view(R, Hq, n, L) * s["scale"]
    if c["softcap"]:
        score = torch.tanh(score / c["softcap"]) * c["softcap"]
    j, p = torch.arange(L, device=DEV), (seq - new)[:, None] + i
    seen = (j[None, None, :] < seq[:, None, None]) & (i < new[:, None])[:, :, None]
    if c["causal"]:
        seen = seen & (j <= p[:, :, None])
    if c["window"]:
        seen = seen & (j > p[:, :, None] - c["window"])
    score = score.masked_fill_(~seen[:, None], float("-inf"))
    top = score.amax(3, keepdim=True)
    score = torch.exp(score.sub_(torch.where(top == float("-inf"), torch.zeros_like(top), top)))
    total = score.sum(3, keepdim=True)
    out = score.view(R, H, -1, L) @ rows(s["v"], s["v_scale"])
    out = _quotient(out.view(R, Hq, n, D), total.expand(R, Hq, n, D))
    t = torch.arange(s["T"], device=DEV)
    r = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    return out[r, :, t - cu[r]].to(s["q"].dtype)


def work(case):
    c = case
    seq, new = _lengths(c)
    B = c["block"]
    if c["op"] == "plan":
        fresh = sum(_ceil(a, B) - _ceil(a - n, B) for a, n in zip(seq, new))
        return {"bytes": 4.0 * (4 * c["R"] + 2 * sum(new) + 2 * fresh), "flops": 0.0}
    size, T = 4 if c["dtype"] == "fp32" else 2, sum(new)
    if c["op"] == "cache":
        # rows in; codes out, those of a block's earlier tokens read and written too; the touched blocks' codes read, their numbers out
        held = sum((a - n) % B for a, n in zip(seq, new) if n)
        return {"bytes": 2.0 * c["Hkv"] * c["D"] * (T * (size + 1) + 2 * held + (T + held) * (1 + size)), "flops": 0.0}
    keys = pairs = blocks = 0
    for L, n in zip(seq, new):
        lo = [max(0, L - n + i - c["window"] + 1) if c["window"] else 0 for i in range(n)]
        hi = [L - n + i + 1 if c["causal"] else L for i in range(n)]
        pairs += sum(h - l for l, h in zip(lo, hi))
        if n:
            keys += max(hi) - min(lo)
            blocks += _ceil(max(hi), B) - min(lo) // B
    return {"bytes": 2.0 * c["Hkv"] * (keys * c["D"] + 4 * blocks) + 2.0 * T * c["Hq"] * c["D"] * size, "flops": 4.0 * c["Hq"] * c["D"] * pairs}


def exact(case, seed):
    c = case
    if c["op"] == "plan":
        return None
    s = prepare(c, seed)
    seq, new = _lengths(c)
    B, D, H = c["block"], c["D"], c["Hkv"]
    where = s["table"].cpu().tolist()
    if c["op"] == "cache":
        at, out = _starts(new), {"k": [], "v": []}
        x = s["kv_rows"].double().view(s["T"], 3, H, D)
        for r in range(c["R"]):
            pos, row, end = seq[r] - new[r], at[r], seq[r]
            for name, part in (("k", 1), ("v", 2)):
                p, t = pos, row
                while p < end:
                    b, o = where[r][p // B], p % B
                    m = min(B - o, end - p)
                    fresh = x[t:t + m, part].transpose(0, 1)                                        # [H, m, D]
                    # the scale is an fp32 number, and so is each quotient that is rounded to a code: those roundings are the definition
                    scale = (fresh.abs().amax((1, 2)) / 127).float().double()
                    old = s[name][b, :, :o].double()
                    if o:
                        before = s[name + "_scale"][b].double()
                        scale = torch.maximum(scale, before)
                        ratio = torch.where(scale > 0, before / scale, scale).float().double()
                        old = (old * ratio[:, None, None]).float().double().round()
                    unit = torch.where(scale > 0, scale, torch.ones_like(scale))[:, None, None]
                    codes = torch.cat([old, (fresh / unit).float().double().round().clamp(-127, 127)], 1)
                    out[name].append((codes * scale[:, None, None]).transpose(0, 1))
                    p, t = p + m, t + m
        return {n: torch.cat(v) if v else torch.zeros((0, H, D), dtype=torch.float64, device=DEV) for n, v in out.items()}
    G, outs, at = c["Hq"] // H, [], _starts(new)
    for r in range(c["R"]):
        L, n = seq[r], new[r]
        ids = s["table"][r, : _ceil(L, B)].long()
        q = s["q"][at[r]:at[r + 1]].double()
        k, v = ((s[m][ids].double() * s[m + "_scale"][ids].double()[:, :, None, None]).transpose(0, 1).reshape(H, -1, D)[:, :L] for m in ("k", "v"))
        i, j = torch.arange(L - n, L, device=DEV)[:, None], torch.arange(L, device=DEV)[None, :]
        hidden = torch.zeros((n, L), dtype=torch.bool, device=DEV)
        if c["causal"]:
            hidden |= j > i
        if c["window"]:
            hidden |= j <= i - c["window"]
        o = torch.empty((n, c["Hq"], D), dtype=torch.float64, device=DEV)
        for h in range(c["Hq"]):
            z = q[:, h] @ k[h // G].T * s["scale"]
            z = c["softcap"] * torch.tanh(z / c["softcap"]) if c["softcap"] else z
            o[:, h] = torch.softmax(z.masked_fill(hidden, -math.inf), 1) @ v[h // G]
        outs.append(o)
    return torch.cat(outs)
