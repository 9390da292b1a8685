"""The 8-bit KV cache's operators in numpy, in 64 bits, one request and one head at a time: what the GPU tests compare with."""
import numpy as np


def plan(kv_len, new_len, block, table, free, first, rows):
    """Outputs of kv_plan; `table` is not changed."""
    table, R, at = table.copy(), len(kv_len), first
    before = 0
    seq, cu = np.zeros(R, np.int32), np.zeros(R + 1, np.int32)
    slot, position = np.full(rows, -1, np.int32), np.full(rows, -1, np.int32)
    unserved = tokens = 0
    for r in range(R):
        kv, new = max(0, int(kv_len[r])), max(0, int(new_len[r]))
        cu[r + 1] = cu[r] + new
        have, want = -(-kv // block), -(-(kv + new) // block)
        need = want - have if want <= table.shape[1] else 0
        ok = want <= table.shape[1] and (need == 0 or before + need <= len(free) - first)
        for j in range(need if ok else 0):
            table[r, have + j] = free[first + before + j]
        if ok and need:
            at = first + before + need
        before += need
        if not ok:
            unserved += 1
            continue
        seq[r] = kv + new
        tokens += new
        for i in range(new):
            if cu[r] + i < rows:
                position[cu[r] + i] = kv + i
                slot[cu[r] + i] = table[r, (kv + i) // block] * block + (kv + i) % block
    return {"table": table, "seq_len": seq, "cu": cu, "slot": slot, "position": position, "status": np.array([at, unserved, at - first, tokens], np.int32)}


def append(x, slot, codes, scale):
    """Rows x[T, heads, dim] (fp32 values) into codes [blocks, heads, block, dim] and scale [blocks, heads], in place.  The scale, the
    quotients that are rounded to codes and the products of held codes are fp32 numbers by definition."""
    block, t = codes.shape[2], 0
    f32 = np.float32
    while t < len(slot):
        if slot[t] < 0:
            t += 1
            continue
        b, o, m = slot[t] // block, slot[t] % block, 1
        while t + m < len(slot) and slot[t + m] == slot[t] + m and o + m < block:
            m += 1
        for h in range(codes.shape[1]):
            new = x[t:t + m, h].astype(np.float64)
            amax = np.nanmax(np.abs(np.where(np.isnan(new), 0.0, new)))
            was = float(scale[b, h]) if o else 0.0
            now = max(was, float(f32(amax / 127.0)))
            if o and now > was:
                ratio = float(f32(was / now))
                codes[b, h, :o] = np.rint(f32(codes[b, h, :o].astype(np.float64) * ratio)).astype(np.int8)
            with np.errstate(invalid="ignore"):
                q = np.rint(f32(new / now)) if now > 0 else np.zeros_like(new)
            codes[b, h, o:o + m] = np.clip(np.nan_to_num(q, nan=0.0), -127, 127).astype(np.int8)
            scale[b, h] = f32(now)
        t += m


def rows_of(codes, scale, table_row, tokens):
    """[tokens, heads, dim] numbers of one request."""
    block = codes.shape[2]
    out = np.zeros((tokens, codes.shape[1], codes.shape[3]))
    for p in range(0, tokens, block):
        b, m = table_row[p // block], min(block, tokens - p)
        with np.errstate(invalid="ignore"):
            out[p:p + m] = (codes[b, :, :m].astype(np.float64) * scale[b].astype(np.float64)[:, None, None]).transpose(1, 0, 2)
    return out


def attention(q, cu, seq_len, k, v, scale, causal=1, window=0, softcap=0.0):
    """q [T, heads_q, dim] fp64; k[r], v[r] [tokens, heads, dim] fp64.  (out, lse, reach): reach bounds the sum of |q k| scale of a row's scores."""
    out, lse, reach = np.zeros(q.shape), np.full(q.shape[:2], -np.inf), 0.0
    for r in range(len(seq_len)):
        n, L = cu[r + 1] - cu[r], int(seq_len[r])
        for i in range(n):
            p = L - n + i
            lo = max(0, p - window + 1) if window else 0
            hi = p + 1 if causal else L
            if hi <= lo:
                continue
            for h in range(q.shape[1]):
                kk, vv = k[r][lo:hi, h * k[r].shape[1] // q.shape[1]], v[r][lo:hi, h * k[r].shape[1] // q.shape[1]]
                z = kk @ q[cu[r] + i, h] * scale
                reach = max(reach, float((np.abs(kk) @ np.abs(q[cu[r] + i, h])).max() * abs(scale)))
                if softcap:
                    z = softcap * np.tanh(z / softcap)
                w = np.exp(z - z.max())
                out[cu[r] + i, h] = w @ vv / w.sum()
                lse[cu[r] + i, h] = z.max() + np.log(w.sum())
    return out, lse, reach
