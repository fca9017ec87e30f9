"""The paged-cache operators in 64 bits and plain loops, from their definitions: what tests/test_gpu_cache.py compares the
kernels with."""
import math

import numpy as np

MIN_EXP, MAX_EXP = -64, 120


def e4m3_values():
    c = np.arange(256)
    e, m = (c >> 3) & 15, (c & 7).astype(np.float64)
    v = np.where(e > 0, (1 + m / 8) * 2.0 ** (e - 7), m / 8 * 2.0 ** -6)
    v = np.where((c & 127) == 127, np.nan, v)
    return np.where(c > 127, -v, v)


VALUES = e4m3_values()


def e4m3_round(x):
    """Codes of the nearest E4M3 values of float64 `x`: ties to even, saturating, NaN as 0x7F."""
    x = np.asarray(x, dtype=np.float64)
    size = np.minimum(np.abs(np.nan_to_num(x, nan=0.0, posinf=1e300, neginf=-1e300)), 448.0)
    exp = np.floor(np.log2(np.maximum(size, 2.0 ** -6)))
    step = 2.0 ** (exp - 3)
    size = np.round(size / step) * step                     # numpy rounds halves to even
    exp = np.floor(np.log2(np.maximum(size, 2.0 ** -6)))
    normal = size >= 2.0 ** -6
    code = np.where(normal, ((exp + 7).astype(np.int64) << 3) + np.round((size / 2.0 ** exp - 1) * 8).astype(np.int64),
                    np.round(size / 2.0 ** -9).astype(np.int64))
    code = code + np.where(np.signbit(x), 128, 0)
    return np.where(np.isnan(x), 127, code).astype(np.uint8)


def scale_for(amax):
    e = MIN_EXP
    while e < MAX_EXP and 448.0 * 2.0 ** e < amax:
        e += 1
    return 2.0 ** e


def store(codes, scales, rows, slots):
    """`codes` [blocks, heads, block, dim] and `scales` [blocks, heads] after the rows [tokens, heads, dim] (float64)."""
    codes, scales = codes.copy(), scales.astype(np.float64).copy()
    bs = codes.shape[2]
    count = codes.shape[0] * bs
    t = 0
    while t < len(slots):
        if not 0 <= slots[t] < count:
            t += 1
            continue
        block, end = slots[t] // bs, t
        while end < len(slots) and 0 <= slots[end] < count and slots[end] // bs == block:
            end += 1
        low = min(slots[t:end]) % bs
        for h in range(codes.shape[1]):
            x = rows[t:end, h]
            fin = np.abs(x[np.isfinite(x)])
            need = scale_for(fin.max() if fin.size else 0.0)
            old = scales[block, h] if low > 0 else 0.0
            now = max(old, need)
            if low > 0 and now != old:
                codes[block, h, :low] = e4m3_round(VALUES[codes[block, h, :low]] * (old / now))
            scales[block, h] = now
            for i in range(t, end):
                codes[block, h, slots[i] % bs] = e4m3_round(rows[i, h] / now)
        t = end
    return codes, scales


def attention(q, k, v, k_scale, v_scale, row_offsets, kv_len, table, scale, causal, window):
    """(out, lse) in float64, NaN where a row belongs to no request.  q [tokens, heads, dim] float64; k, v codes."""
    tokens, heads, dim = q.shape
    kv_heads, bs = k.shape[1], k.shape[2]
    group = heads // kv_heads
    out, lse = np.full(q.shape, np.nan), np.full((tokens, heads), np.nan)
    for r in range(len(kv_len)):
        a, b, n = row_offsets[r], row_offsets[r + 1], kv_len[r]
        blocks = [table[r][j // bs] for j in range(n)]
        ok = np.array([0 <= x < k.shape[0] for x in blocks], dtype=bool).reshape(n)
        for h in range(kv_heads):
            kk, vv = np.zeros((n, dim)), np.zeros((n, dim))
            for j in range(n):
                if ok[j]:
                    kk[j] = VALUES[k[blocks[j], h, j % bs]] * float(k_scale[blocks[j], h])
                    vv[j] = VALUES[v[blocks[j], h, j % bs]] * float(v_scale[blocks[j], h])
            for t in range(a, b):
                pos = n - (b - a) + (t - a)
                j = np.arange(n)
                see = ok & ((j <= pos) if causal else True) & ((j > pos - window) if window else True)
                for g in range(h * group, (h + 1) * group):
                    if not see.any():
                        out[t, g], lse[t, g] = 0.0, -math.inf
                        continue
                    s = kk[see] @ q[t, g] * scale
                    m = s.max()
                    p = np.exp(s - m)
                    out[t, g], lse[t, g] = (p / p.sum()) @ vv[see], m + math.log(p.sum())
    return out, lse


def assign(cached, new, table, free, count, block, max_tokens):
    """dict of what cache_assign writes; `table` and `free` are copied."""
    table, free = table.copy(), free.copy()
    columns = table.shape[1]
    have = [-(-c // block) for c in cached]
    stack = list(free[:count])
    for r, n in enumerate(new):
        if n < 0:
            stack += [table[r, i] for i in range(have[r])]
    row, rows_end, offsets, want = 0, [], [0], 0
    slots, positions = np.full(max_tokens, -1, np.int64), np.full(max_tokens, -1, np.int32)
    kv, denied, height = [], 0, len(stack)
    for r, n in enumerate(new):
        grow = max(n, 0)
        start, row = row, row + grow
        offsets.append(min(row, max_tokens))
        if n < 0:
            kv.append(0)
            continue
        need = -(-(cached[r] + grow) // block) - have[r]
        fits = cached[r] + grow <= columns * block and (grow == 0 or row <= max_tokens)
        if fits:
            want += need
        served = fits and (need == 0 or want <= height)
        kv.append(cached[r] + grow if served else cached[r])
        denied += not served
        if served:
            for i in range(need):
                table[r, have[r] + i] = stack.pop()
        for i in range(grow):
            if start + i < max_tokens:
                pos = cached[r] + i
                positions[start + i] = pos
                if served:
                    slots[start + i] = int(table[r, pos // block]) * block + pos % block
    for i in range(min(count, len(stack)), min(len(stack), len(free))):
        free[i] = stack[i]
    return {"block_table": table, "free_blocks": free, "free_count": len(stack), "row_offsets": np.array(offsets),
            "kv_len": np.array(kv), "slots": slots, "positions": positions, "denied": denied}
