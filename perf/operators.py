"""The operators around a paged key / value cache held in 8 bits, as cases to be measured.

  assign     block tables, slot maps, row offsets and cached lengths of the next step, made on the GPU from the lengths
             of the requests; finished requests give their blocks back, growing ones take blocks from the free stack
  store      the step's keys and values go into the cache as E4M3 codes with one power-of-two scale per block of tokens
             and head; where a new token raises a block's scale, the codes that are in the block already are re-scaled
  attention  softmax(scale * Q K^T) V over the cache, for single tokens, short runs of tokens and whole prompts

`run` computes them with elementary torch operations in 32 bits, or, where `own` is set, with this repository's kernels.
The cache is [blocks][kv heads][tokens of a block][head size], one (block, head) page being one contiguous run.
"""
import math
import random

import torch

own = False

DEVICE = "cuda"
E4M3_MAX = 448.0
MIN_EXP, MAX_EXP = -64, 120          # exponents that a scale may have
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
MAX_WORK = 1.1e9                     # bytes (or flops / 250) that a drawn case may cost at most


# ---------------------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # one user, one token, a short context: nothing but latency
        {"name": "attn_one_token", "op": "attention", "requests": 1, "q": "1-1", "kv": "1000-1000", "heads": 32,
         "kv_heads": 8, "dim": 128, "block": 16, "type": "bf16", "causal": True, "window": 0},
        # a decode step of a serving batch with ragged contexts
        {"name": "attn_decode_batch", "op": "attention", "requests": 64, "q": "1-1", "kv": "200-8192", "heads": 32,
         "kv_heads": 8, "dim": 128, "block": 64, "type": "bf16", "causal": True, "window": 0},
        # a decode step of a few very long contexts, many query heads per kv head
        {"name": "attn_decode_long", "op": "attention", "requests": 4, "q": "1-1", "kv": "90001-131072", "heads": 64,
         "kv_heads": 8, "dim": 128, "block": 128, "type": "bf16", "causal": True, "window": 0},
        # verification of drafted tokens under a sliding window, small heads
        {"name": "attn_verify_window", "op": "attention", "requests": 48, "q": "4-4", "kv": "700-6000", "heads": 16,
         "kv_heads": 4, "dim": 64, "block": 32, "type": "f16", "causal": True, "window": 1024},
        # prompts of a batch, nothing cached before
        {"name": "attn_prompts", "op": "attention", "requests": 4, "q": "1201-4096", "kv": "0-0", "heads": 32,
         "kv_heads": 8, "dim": 128, "block": 64, "type": "bf16", "causal": True, "window": 0},
        # a chunk of a long prompt behind what is cached of it: few rows, a long axis
        {"name": "attn_chunk", "op": "attention", "requests": 2, "q": "257-512", "kv": "15000-30000", "heads": 16,
         "kv_heads": 2, "dim": 128, "block": 64, "type": "bf16", "causal": True, "window": 0},
        # decoding requests and chunks of prompts in one step, and every query sees the whole cache (an encoder's states)
        {"name": "attn_mixed_full", "op": "attention", "requests": 21, "q": "1-300", "kv": "0-2500", "heads": 14,
         "kv_heads": 2, "dim": 64, "block": 16, "type": "f16", "causal": False, "window": 0},
        # one new token for each request of a decode step
        {"name": "store_decode", "op": "store", "requests": 128, "new": "1-1", "kv_heads": 8, "dim": 128, "block": 64,
         "type": "bf16"},
        # the tokens of a batch of prompts
        {"name": "store_prompts", "op": "store", "requests": 6, "new": "1000-8191", "kv_heads": 8, "dim": 128,
         "block": 64, "type": "bf16"},
        # short ragged chunks, small heads, an odd number of kv heads
        {"name": "store_ragged", "op": "store", "requests": 37, "new": "1-150", "kv_heads": 5, "dim": 64, "block": 16,
         "type": "f16"},
        # a decode step: every request grows by one token, a few finish
        {"name": "assign_decode", "op": "assign", "requests": 256, "new": "1-1", "kv": "1-4000", "finished": 9,
         "block": 64, "columns": 128, "lack": 0},
        # a step with many prompts, for which the pool does not reach: the last ones have to wait
        {"name": "assign_prompts", "op": "assign", "requests": 1000, "new": "1-1500", "kv": "0-9000", "finished": 150,
         "block": 16, "columns": 1024, "lack": 10},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        op = rng.choice(["attention", "attention", "store", "assign"])
        if op == "attention":
            kv_heads = rng.choice([1, 2, 3, 4, 8])
            form = rng.choice(["decode", "decode", "verify", "prompt", "chunk", "mixed"])
            kv = sorted(_log(rng, 1, 40000) for _ in range(2))
            q, requests = [1, 1], _log(rng, 1, 200)
            if form == "verify":
                q = [rng.randint(1, 3), rng.randint(4, 9)]
            elif form == "prompt":
                q, kv, requests = sorted(_log(rng, 16, 4096) for _ in range(2)), [0, 0], _log(rng, 1, 8)
            elif form == "chunk":
                q, requests = sorted(_log(rng, 32, 700) for _ in range(2)), _log(rng, 1, 6)
            elif form == "mixed":
                q, requests = [1, _log(rng, 20, 500)], _log(rng, 2, 24)
            case = {"op": op, "requests": requests, "q": q, "kv": kv, "heads": kv_heads * rng.choice([1, 2, 4, 5, 7, 8]),
                    "kv_heads": kv_heads, "dim": rng.choice([64, 128]), "block": rng.choice([16, 32, 64, 128]),
                    "type": rng.choice(["bf16", "f16"]), "causal": rng.random() < 0.8,
                    "window": rng.choice([0, 0, 0, _log(rng, 20, 4000)])}
        elif op == "store":
            case = {"op": op, "requests": _log(rng, 1, 300), "new": rng.choice([[1, 1], [1, _log(rng, 2, 20)],
                    sorted(_log(rng, 20, 6000) for _ in range(2))]), "kv_heads": rng.choice([1, 2, 5, 8, 16]),
                    "dim": rng.choice([64, 128]), "block": rng.choice([16, 32, 64, 128]),
                    "type": rng.choice(["bf16", "f16"])}
        else:
            block = rng.choice([16, 32, 64, 128])
            kv = sorted(rng.choice([0, _log(rng, 1, 12000)]) for _ in range(2))
            new = rng.choice([[1, 1], [0, _log(rng, 2, 2000)]])
            requests = _log(rng, 1, 2000)
            case = {"op": op, "requests": requests, "new": new, "kv": kv, "finished": rng.randint(0, requests // 4),
                    "block": block, "columns": -(-(kv[1] + new[1]) // block) + rng.randint(0, 9),
                    "lack": rng.choice([0, 0, 0, rng.randint(5, 50)])}
        case = {k: "%d-%d" % tuple(v) if isinstance(v, list) else v for k, v in case.items()}
        w = work(case)
        if max(w["bytes"], w["flops"] / 250) < MAX_WORK and _plain_bytes(case) < 24e9:
            return case


def _pair(v):
    return tuple(int(x) for x in v.split("-")) if isinstance(v, str) else tuple(v)


def _spread(lo_hi, n, salt):
    """n lengths between lo and hi, both of them among these where n > 1; the same ones whatever the seed."""
    lo, hi = _pair(lo_hi)
    r = random.Random(1000003 * salt + 7919 * lo + hi + n)
    got = [r.randint(lo, hi) for _ in range(n)]
    got[0] = hi
    if n > 1:
        got[-1] = lo
    return got


def _lengths(case):
    """(rows of each request, cached tokens of each request with these rows among them)."""
    n = case["requests"]
    q = _spread(case["q"], n, 1)
    return q, [a + b for a, b in zip(q, _spread(case["kv"], n, 2))]


def _seen(case):
    """Per request (pairs of a row and a token it sees, tokens that any of its rows sees)."""
    w = case["window"]
    for q, kv in zip(*_lengths(case)):
        pairs, first = 0, kv
        for pos in range(kv - q, kv):
            last = pos + 1 if case["causal"] else kv
            lo = max(0, pos - w + 1) if w else 0
            pairs += max(0, last - lo)
            first = min(first, lo)
        yield pairs, kv - first if q else 0


def _plain_bytes(case):
    """What the plain form holds at its largest."""
    if case["op"] != "attention":
        return 0
    q, kv = _lengths(case)
    n, q, kv = case["requests"], max(q), max(kv)
    return 4 * n * kv * (4 * case["kv_heads"] * case["dim"] + 3 * case["heads"] * q)


def work(case):
    if case["op"] == "attention":
        q, kv = _lengths(case)
        seen = list(_seen(case))
        tokens, h, d = sum(s for _, s in seen), case["kv_heads"], case["dim"]
        pages = sum(-(-s // case["block"]) for _, s in seen)
        bytes_ = (2 * tokens * h * d + pages * (8 * h + 4)               # codes, scales, table entries
                  + 2 * sum(q) * case["heads"] * d * 2                   # queries and outputs
                  + 4 * sum(q) * case["heads"] + 8 * len(q))             # log-sum-exp, lengths
        return {"bytes": bytes_, "flops": 4.0 * case["heads"] * d * sum(p for p, _ in seen)}
    if case["op"] == "store":
        new, (h, d) = _spread(case["new"], case["requests"], 3), (case["kv_heads"], case["dim"])
        runs = sum(-(-n // case["block"]) for n in new)
        return {"bytes": sum(new) * (2 * h * d * 3 + 8) + runs * 2 * h * 8, "flops": 4.0 * sum(new) * h * d}
    new, kv, grown = _assign_lengths(case)               # a lack of blocks is left out of account
    taken = sum(-(-(n + k) // case["block"]) - -(-k // case["block"]) for n, k in zip(new, kv) if n > 0)
    given = sum(-(-k // case["block"]) for n, k in zip(new, kv) if n < 0)
    return {"bytes": 20 * len(new) + 12 * grown + 8 * (taken + given), "flops": 10.0 * (len(new) + grown)}


# -------------------------------------------------------------------------------------------------------- inputs

def _int32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEVICE)


def _values(g, shape, spread):
    """Activations: per-channel gains and a few loud tokens. shape [..., tokens, dim]."""
    x = torch.randn(shape, generator=g, device=DEVICE)
    x *= torch.exp(0.4 * torch.randn(shape[-1:], generator=g, device=DEVICE))
    x *= spread * torch.exp2(torch.randn(shape[:-1] + (1,), generator=g, device=DEVICE))
    return x


def _random_cache(g, blocks, case):
    """Codes and scales as a cache has them after use: pages quantised with a power-of-two scale each."""
    h, bs, d = case["kv_heads"], case["block"], case["dim"]
    out = []
    for spread in (0.7, 0.3):
        codes = torch.empty((blocks, h, bs, d), dtype=torch.uint8, device=DEVICE)
        scales = torch.empty((blocks, h), dtype=torch.float32, device=DEVICE)
        step = max(1, (1 << 28) // (h * bs * d))
        for b in range(0, blocks, step):
            x = _values(g, (min(step, blocks - b), h, bs, d), spread)
            s = torch.exp2(_exponent(x.abs().amax((2, 3))))
            codes[b:b + step] = (x / s[:, :, None, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(torch.uint8)
            scales[b:b + step] = s
        out += [codes, scales]
    return out


def _tables(g, kv, block, spare=3, columns=None):
    """A table of blocks dealt at random, and the number of blocks in the pool."""
    need = [-(-k // block) for k in kv]
    pool = sum(need) + spare
    deal = torch.randperm(pool, generator=g, device=DEVICE).to(torch.int32)
    columns = columns or max(1, max(need))
    table = torch.full((len(kv), columns), -1, dtype=torch.int32, device=DEVICE)
    n = torch.tensor(need, device=DEVICE)
    col = torch.arange(columns, device=DEVICE)[None]
    first = torch.cumsum(n, 0) - n
    there = col < n[:, None]
    table[there] = deal[(first[:, None] + col)[there]]
    return table, pool, deal


def _offsets(n):
    c = [0]
    for x in n:
        c.append(c[-1] + x)
    return c


def _assign_lengths(case):
    n = case["requests"]
    new, kv = _spread(case["new"], n, 4), _spread(case["kv"], n, 5)
    for r in random.Random(n).sample(range(n), case["finished"]):
        new[r] = -1
    return new, kv, sum(x for x in new if x > 0)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    state = dict(case)
    if case["op"] == "attention":
        q, kv = _lengths(case)
        state["block_table"], pool, _ = _tables(g, kv, case["block"])
        state["k"], state["k_scale"], state["v"], state["v_scale"] = _random_cache(g, pool, case)
        _stale_tails(g, state, kv)
        shape = (sum(q), case["heads"], case["dim"])
        t = TYPES[case["type"]]
        state["q_rows"] = _values(g, shape, 1.0).to(t)
        state["row_offsets"], state["kv_len"] = _int32(_offsets(q)), _int32(kv)
        state["max_q"], state["max_kv"], state["min_q"] = max(q), max(kv), min(q)
        state["scale"] = case["dim"] ** -0.5
        state["out"] = torch.zeros(shape, dtype=t, device=DEVICE)
        state["lse"] = torch.zeros(shape[:2], dtype=torch.float32, device=DEVICE)
    elif case["op"] == "store":
        new = _spread(case["new"], case["requests"], 3)
        kv = [n + c for n, c in zip(new, _spread((0, 500), len(new), 6))]
        table, pool, _ = _tables(g, kv, case["block"])
        state["k"], state["k_scale"], state["v"], state["v_scale"] = _random_cache(g, pool, case)
        shape = (sum(new), case["kv_heads"], case["dim"])
        t = TYPES[case["type"]]
        state["k_rows"], state["v_rows"] = _values(g, shape, 0.7).to(t), _values(g, shape, 0.3).to(t)
        state["slots"] = _plain_slots(_int32(_offsets(new)), _int32(kv), table, case["block"], sum(new))[0]
    else:
        new, kv, grown = _assign_lengths(case)
        order = torch.randperm(len(new), generator=g, device=DEVICE)        # other seeds: other requests have these lengths
        state["new_len"], state["cached_len"] = _int32(new)[order].contiguous(), _int32(kv)[order].contiguous()
        state["block_table"], pool, deal = _tables(g, state["cached_len"].tolist(), case["block"], 0, case["columns"])
        spare = sum(-(-(n + k) // case["block"]) - -(-k // case["block"]) for n, k in zip(new, kv) if n > 0)
        back = sum(-(-k // case["block"]) for n, k in zip(new, kv) if n < 0)
        spare = max(0, spare * (100 - case["lack"]) // 100 + 5 - back)
        # ids of the free blocks in the order in which they came back; room behind them for those that come back now
        state["free_blocks"] = torch.full((pool + spare,), -1, dtype=torch.int32, device=DEVICE)
        state["free_blocks"][:spare] = pool + torch.randperm(spare, generator=g, device=DEVICE).to(torch.int32)
        state["free_count"] = _int32([spare])
        n = len(new)
        state["rows"] = grown + 7                                            # a padded batch
        state["free_count_out"], state["denied"] = _int32([0]), _int32([0])
        state["row_offsets"], state["kv_len"] = _int32([0] * (n + 1)), _int32([0] * n)
        state["slots"] = torch.zeros(grown + 7, dtype=torch.int64, device=DEVICE)
        state["positions"] = torch.zeros(grown + 7, dtype=torch.int32, device=DEVICE)
    return state


def _stale_tails(g, state, kv):
    """The rows behind a request's last token hold whatever a former owner of the block left there."""
    bs = state["block"]
    last = torch.tensor([(k - 1) // bs for k in kv], device=DEVICE).clamp(min=0)
    block = state["block_table"][torch.arange(len(kv), device=DEVICE), last].long()
    used = torch.tensor([(k - 1) % bs + 1 for k in kv], device=DEVICE)
    keep = torch.tensor([k > 0 for k in kv], device=DEVICE)
    block, used = block[keep], used[keep]
    row = torch.arange(bs, device=DEVICE)[None, None, :, None]
    for codes in (state["k"], state["v"]):
        page = codes[block]
        junk = torch.randint(0, 256, page.shape, generator=g, device=DEVICE, dtype=torch.uint8)
        codes[block] = torch.where(row < used[:, None, None, None], page, junk)


# ---------------------------------------------------------------------------------------------------- plain forms

def _exponent(amax):
    """The smallest whole e with amax <= 448 * 2^e, within the range that a scale may have."""
    m, e = torch.frexp(amax)                                  # amax = m * 2^e, m in [0.5, 1): 448 = 0.875 * 2^9
    e = torch.where(m <= 0.875, e - 9, e - 8)
    e = torch.where(amax > 0, e, torch.full_like(e, MIN_EXP))
    return e.clamp(MIN_EXP, MAX_EXP).float()


def _plain_slots(row_offsets, kv_len, table, block, rows):
    """(slot, position, request) of each row of a packed batch; -1 behind the last request's rows."""
    offs = row_offsets.long()
    t = torch.arange(rows, device=DEVICE)
    r = torch.searchsorted(offs[1:].contiguous(), t, right=True)
    there = r < kv_len.numel()
    r = r.clamp(max=kv_len.numel() - 1)
    pos = kv_len.long()[r] - offs[r + 1] + t
    page = table[r, (pos // block).clamp(0, table.shape[1] - 1)].long()
    return torch.where(there, page * block + pos % block, -1), torch.where(there, pos, -1), r


def _plain_assign(s):
    bs = s["block"]
    new, old = s["new_len"].long(), s["cached_len"].long()
    grow, done = new.clamp(min=0), new < 0
    have = (old + bs - 1) // bs
    need = torch.where(done, 0, (old + grow + bs - 1) // bs - have)
    fits = have + need <= s["block_table"].shape[1]
    need = torch.where(fits, need, 0)
    back = torch.where(done, have, 0)
    count = s["free_count"].long()
    back_to = torch.cumsum(back, 0)
    need_to = torch.cumsum(need, 0)
    top = count + back_to[-1]
    served = fits & ((need == 0) | (need_to <= top))
    stack = s["free_blocks"].clone()
    col = torch.arange(s["block_table"].shape[1], device=DEVICE)[None]
    given = col < back[:, None]
    at = (count + (back_to - back)[:, None] + col)[given]
    stack[at] = s["block_table"][given]
    taken = (col >= have[:, None]) & (col < (have + need)[:, None]) & served[:, None]
    nth = ((need_to - need)[:, None] + col - have[:, None])[taken]
    s["block_table"][taken] = stack[top - 1 - nth]
    popped = torch.where(served, need_to, 0).max()
    s["free_count_out"][:] = (top - popped).int()
    keep = torch.arange(stack.numel(), device=DEVICE)
    s["free_blocks"][:] = torch.where((keep >= count) & (keep < top - popped), stack, s["free_blocks"])
    s["denied"][:] = (~served).sum().int()
    s["row_offsets"][1:] = torch.cumsum(grow, 0).int()
    s["kv_len"][:] = torch.where(done, 0, torch.where(served, old + grow, old)).int()
    slots, pos, r = _plain_slots(s["row_offsets"], torch.where(done, 0, old + grow), s["block_table"], bs, s["rows"])
    s["slots"][:] = torch.where(served[r], slots, -1)
    s["positions"][:] = pos.int()
    return _assign_out(s)


def _assign_out(s):
    return {k: s[k] for k in ("block_table", "row_offsets", "kv_len", "slots", "positions", "free_blocks",
                              "free_count_out", "denied")}


def _plain_store(s):
    bs, slots = s["block"], s["slots"]
    there = slots >= 0
    block, off = (slots // bs)[there], (slots % bs)[there]
    pages = s["k"].shape[0]
    first = torch.full((pages,), bs, device=DEVICE).scatter_reduce(0, block, off, "amin")
    touched = torch.unique(block)
    old_rows = torch.arange(bs, device=DEVICE)[None, None, :, None] < first[touched][:, None, None, None]
    for codes, scale, rows in ((s["k"], s["k_scale"], s["k_rows"]), (s["v"], s["v_scale"], s["v_rows"])):
        x = rows.float()[there]
        size = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(2)
        amax = torch.zeros_like(scale).scatter_reduce(0, block[:, None].expand_as(size), size, "amax")
        want = torch.exp2(_exponent(amax[touched]))
        was = scale[touched]
        kept = (first[touched] > 0)[:, None]
        now = torch.where(kept & (was >= want), was, want)
        page = codes[touched].view(torch.float8_e4m3fn).float()
        moved = (page * (was / now)[:, :, None, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(torch.uint8)
        codes[touched] = torch.where(old_rows & (now != was)[:, :, None, None], moved, codes[touched])
        scale[touched] = now
        y = (x / scale[block][:, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(torch.uint8)
        codes[block, :, off] = y
    return _store_out(s)


def _store_out(s):
    return {"k": s["k"].view(torch.float8_e4m3fn), "v": s["v"].view(torch.float8_e4m3fn), "k_scale": s["k_scale"],
            "v_scale": s["v_scale"]}


def _plain_pages(codes, scale, table, kv, there):
    """The cache of each request in 32 bits, [request][kv head][token][dim]; tokens that it has not are zero."""
    n, cols = table.shape
    table = table.long().clamp(min=0)
    x = codes[table].view(torch.float8_e4m3fn).float() * scale[table][..., None, None]      # [n][cols][h][bs][d]
    h, bs, d = x.shape[2:]
    x = x.permute(0, 2, 1, 3, 4).reshape(n, h, cols * bs, d)[:, :, :kv]
    return torch.where(there[:, None, :, None], x, 0.0)


def _plain_attention(s):
    n, h, d = s["requests"], s["kv_heads"], s["dim"]
    group, mq, mk = s["heads"] // h, s["max_q"], s["max_kv"]
    offs, kv = s["row_offsets"].long(), s["kv_len"].long()
    q_len = offs[1:] - offs[:-1]
    tok = torch.arange(mk, device=DEVICE)[None]
    there = tok < kv[:, None]
    k = _plain_pages(s["k"], s["k_scale"], s["block_table"], mk, there)
    v = _plain_pages(s["v"], s["v_scale"], s["block_table"], mk, there)
    rows = s["q_rows"].shape[0]
    t = torch.arange(rows, device=DEVICE)
    r = torch.searchsorted(offs[1:].contiguous(), t, right=True)
    i = t - offs[r]
    q = torch.zeros((n, mq, s["heads"], d), device=DEVICE)
    q[r, i] = s["q_rows"].float()
    q = q.reshape(n, mq, h, group, d).permute(0, 2, 3, 1, 4).reshape(n, h, group * mq, d)
    pos = (kv - q_len)[:, None] + torch.arange(mq, device=DEVICE)[None]                       # [n][mq]
    see = there[:, None, :].expand(n, mq, mk)
    if s["causal"]:
        see = see & (tok[:, None] <= pos[:, :, None])
    if s["window"]:
        see = see & (tok[:, None] > pos[:, :, None] - s["window"])
    a = torch.matmul(q, k.transpose(2, 3)).reshape(n, h, group, mq, mk)
    a *= s["scale"]
    a.masked_fill_(~see[:, None, None], -math.inf)
    m = a.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    a = a.sub_(m).exp_()
    total = a.sum(-1)
    o = torch.matmul(a.reshape(n, h, group * mq, mk), v).reshape(n, h, group, mq, d)
    o = torch.where(total[..., None] > 0, o / total[..., None], 0.0)
    lse = torch.log(total) + m[..., 0]
    o = o.permute(0, 3, 1, 2, 4).reshape(n, mq, s["heads"], d)
    lse = lse.permute(0, 3, 1, 2).reshape(n, mq, s["heads"])
    s["out"][:] = o[r, i].to(s["out"].dtype)
    s["lse"][:] = lse[r, i]
    return {"out": s["out"], "lse": s["lse"]}


# ------------------------------------------------------------------------------------------------------------ run

def run(state):
    if own:
        return _own(state)
    return {"attention": _plain_attention, "store": _plain_store, "assign": _plain_assign}[state["op"]](state)


def _own(s):
    from ops_tensor_b200 import native
    if s["op"] == "assign":
        native.cache_assign(s["cached_len"], s["new_len"], s["block_table"], s["free_blocks"], s["free_count"],
                            block_size=s["block"], row_offsets=s["row_offsets"], kv_len=s["kv_len"], slots=s["slots"],
                            positions=s["positions"], free_count_out=s["free_count_out"], denied=s["denied"])
        return _assign_out(s)
    if "cache" not in s:
        s["cache"] = native.PagedCache(s["k"], s["v"], s["k_scale"], s["v_scale"])
    if s["op"] == "store":
        native.cache_store(s["cache"], s["k_rows"], s["v_rows"], s["slots"])
        return _store_out(s)
    if "workspace" not in s:      # kept by a program beside its output buffers
        s["workspace"] = native.cache_attention_workspace(s["cache"], s["q_rows"], requests=s["requests"],
                                                          max_q=s["max_q"], max_kv=s["max_kv"])
    native.cache_attention(s["cache"], s["q_rows"], s["row_offsets"], s["kv_len"], s["block_table"], scale=s["scale"],
                           max_q=s["max_q"], max_kv=s["max_kv"], min_q=s["min_q"], causal=s["causal"],
                           window=s["window"], out=s["out"], lse=s["lse"], workspace=s["workspace"])
    return {"out": s["out"], "lse": s["lse"]}


# ---------------------------------------------------------------------------------------------------------- exact

def _exact_codes(codes):
    """The value of each E4M3 code in 64 bits, by the format's definition."""
    c = torch.arange(256, device=DEVICE)
    e, m = (c >> 3) & 15, (c & 7).double()
    v = torch.where(e > 0, (1 + m / 8) * torch.exp2((e - 7).double()), m / 8 * 2.0 ** -6)
    v = torch.where((c & 127) == 127, math.nan, v) * torch.where(c > 127, -1.0, 1.0)
    return v[codes.long()]


def _exact_round(x):
    """x to the nearest E4M3 value, ties to even, in 64 bits."""
    size = x.abs().clamp(max=E4M3_MAX)
    step = torch.exp2(torch.floor(torch.log2(size.clamp(min=2.0 ** -6))) - 3)
    return torch.copysign(torch.round(size / step) * step, x)


def _exact_attention(s):
    h, group, bs = s["kv_heads"], s["heads"] // s["kv_heads"], s["block"]
    offs, kv = s["row_offsets"].tolist(), s["kv_len"].tolist()
    out = torch.zeros(s["q_rows"].shape, dtype=torch.float64, device=DEVICE)
    lse = torch.full(s["q_rows"].shape[:2], -math.inf, dtype=torch.float64, device=DEVICE)
    for r in range(s["requests"]):
        n, kv_r = offs[r + 1] - offs[r], kv[r]
        if n == 0 or kv_r == 0:
            continue
        pages = s["block_table"][r, :-(-kv_r // bs)].long()
        first = torch.arange(kv_r - n, kv_r, device=DEVICE)
        tok = torch.arange(kv_r, device=DEVICE)
        hide = torch.zeros((n, kv_r), dtype=torch.bool, device=DEVICE)
        if s["causal"]:
            hide |= tok[None] > first[:, None]
        if s["window"]:
            hide |= tok[None] <= first[:, None] - s["window"]
        for j in range(h):
            k, v = (_exact_codes(c[pages, j].reshape(-1, s["dim"])[:kv_r])
                    * w[pages, j].double().repeat_interleave(bs)[:kv_r, None]
                    for c, w in ((s["k"], s["k_scale"]), (s["v"], s["v_scale"])))
            for i in range(j * group, (j + 1) * group):
                a = s["q_rows"][offs[r]:offs[r + 1], i].double() @ k.T * s["scale"]
                a = a.masked_fill(hide, -math.inf)
                z = torch.logsumexp(a, 1, keepdim=True)
                p = torch.where(z == -math.inf, 0.0, torch.exp(a - z))
                out[offs[r]:offs[r + 1], i], lse[offs[r]:offs[r + 1], i] = p @ v, z[:, 0]
    return {"out": out, "lse": lse}


def _exact_store(s):
    bs = s["block"]
    got = {}
    slots = s["slots"].tolist()
    runs, start = [], 0
    for t in range(1, len(slots) + 1):
        if t == len(slots) or slots[t] // bs != slots[start] // bs:
            runs.append((start, t, slots[start] // bs, slots[start] % bs))
            start = t
    if len(runs) > 4000:
        return None
    for name, rows in (("k", s["k_rows"]), ("v", s["v_rows"])):
        codes, scale = _exact_codes(s[name]), s[name + "_scale"].double()
        for a, b, block, off in runs:
            x = rows[a:b].double()
            amax = x.abs().amax((0, 2))
            want = torch.exp2(torch.round(torch.log2((amax / E4M3_MAX).clamp(min=2.0 ** MIN_EXP))))
            want = torch.where(want * E4M3_MAX < amax, 2 * want, want)
            now = torch.maximum(want, scale[block]) if off else want
            if off:
                codes[block, :, :off] = _exact_round(codes[block, :, :off] * (scale[block] / now)[:, None, None])
            scale[block] = now
            codes[block, :, off:off + b - a] = _exact_round(x / now[None, :, None]).transpose(0, 1)
        got[name], got[name + "_scale"] = codes, scale
    return got


def exact(case, seed):
    if case["op"] == "assign":
        return None                   # whole numbers: they have to be equal
    state = prepare(case, seed)
    return _exact_attention(state) if case["op"] == "attention" else _exact_store(state)
