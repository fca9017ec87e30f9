"""GPU parity of the paged 8-bit cache: block tables and slot maps, the quantising store, the attention, and a serving
loop of the three, against tests/cache_reference.py (64 bits, plain loops).

Tolerances.  assign: equal.  store: equal bits; every step of the rule (a power-of-two scale, one division, one rounding)
is exact or correctly rounded in float32 for 8- and 11-bit inputs.  attention, with u = finfo(type).eps / 2 the output's
half step: the output rounding is at most u |out|; the probabilities are rounded to half, 2^-11 of each at most (half of
its eps of 2^-10), which moves out by at most 2^-11 sum p |v| / sum p; a score is off by at most d * 2^-23 * scale * |q| |k|
(float32 sums of d exact products) and the exponential by 2^-21, which with e = exp(error) - 1 moves out by at most
2 e sum p |v| / sum p and lse by the error itself plus float32 rounding of lse.
"""
import numpy as np
import pytest

import cache_reference as ref
from ops_tensor_b200 import native

pytestmark = pytest.mark.gpu
U = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}              # eps / 2


def torch_type(name):
    import torch
    return {"bf16": torch.bfloat16, "f16": torch.float16}[name]


def i32(x, device):
    import torch
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=device)


# ------------------------------------------------------------------------------------------------ assign

def run_assign(device, cached, new, table, free, count, block, max_tokens, in_place=False):
    import torch
    n = len(cached)
    t = {"cached": i32(cached, device).reshape(n), "new": i32(new, device).reshape(n), "table": i32(table, device),
         "free": i32(free, device).reshape(-1), "count": i32([count], device)}
    kv = t["cached"] if in_place else torch.full((n,), -7, dtype=torch.int32, device=device)
    count_out = t["count"] if in_place else i32([-7], device)
    offsets = torch.full((n + 1,), -7, dtype=torch.int32, device=device)
    slots = torch.full((max_tokens,), -7, dtype=torch.int64, device=device)
    positions = torch.full((max_tokens,), -7, dtype=torch.int32, device=device)
    denied = i32([-7], device)
    for _ in range(1 if in_place else 2):                  # twice: the same answer
        native.cache_assign(t["cached"], t["new"], t["table"], t["free"], t["count"], block_size=block,
                            row_offsets=offsets, kv_len=kv, slots=slots, positions=positions, free_count_out=count_out,
                            denied=denied)
    return {"block_table": t["table"].cpu().numpy(), "free_blocks": t["free"].cpu().numpy(),
            "free_count": int(count_out.item()), "row_offsets": offsets.cpu().numpy(), "kv_len": kv.cpu().numpy(),
            "slots": slots.cpu().numpy(), "positions": positions.cpu().numpy(), "denied": int(denied.item())}


def assign_inputs(seed, n, block, lens, news, ended, slack, columns, room=None):
    rng = np.random.default_rng(seed)
    cached = rng.integers(lens[0], lens[1] + 1, n)
    new = rng.integers(news[0], news[1] + 1, n)
    new[rng.permutation(n)[:ended]] = -1
    have = -(-cached // block)
    need = np.where(new > 0, -(-(cached + new) // block) - have, 0)
    ids = rng.permutation(int(have.sum() + need.sum()) + 50)
    table = np.full((n, columns), -1)
    at = 0
    for r in range(n):
        table[r, :have[r]] = ids[at:at + have[r]]
        at += have[r]
    spare = max(0, int(need.sum()) - int(have[new < 0].sum()) + slack)
    free = np.full(spare + int(have.sum()) + 3 if room is None else room, -5)
    free[:spare] = rng.permutation(1000000)[:spare] + 1000
    return cached, new, table, free, spare


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("seed,n,block,lens,news,ended,slack,pad", [
    (1, 1, 16, (0, 0), (1, 1), 0, 0, 0), (2, 1, 16, (16, 16), (1, 1), 0, 0, 3), (3, 1, 64, (100, 100), (-1, -1), 1, 0, 2),
    (4, 7, 32, (0, 200), (0, 3), 2, 5, 1), (5, 33, 16, (0, 100), (0, 90), 9, -7, 40), (6, 300, 128, (0, 700), (1, 1), 30, 0, 5),
    (7, 1500, 16, (0, 60), (0, 40), 400, -900, 100), (8, 8192, 16, (0, 30), (1, 2), 100, 0, 17),
    (9, 3, 64, (5, 5), (30000, 40000), 0, 0, 0), (10, 40, 16, (0, 90), (0, 0), 0, 0, 9),
    (11, 65, 16, (0, 300), (-1, -1), 65, 0, 4), (12, 12, 16, (64, 64), (16, 16), 4, -100, 0)])
def test_assign(cuda_device, seed, n, block, lens, news, ended, slack, pad, in_place):
    """One block and many, stacks that reach, that do not and that are empty, ended requests whose blocks are handed out in
    the same call, padding rows, in place and not."""
    columns = -(-(lens[1] + max(news[1], 0)) // block) + 2
    cached, new, table, free, count = assign_inputs(seed, n, block, lens, news, ended, slack, columns)
    max_tokens = int(np.maximum(new, 0).sum()) + pad
    got = run_assign(cuda_device, cached, new, table, free, count, block, max_tokens, in_place)
    want = ref.assign(cached.tolist(), new.tolist(), table, free, count, block, max_tokens)
    for key in want:
        assert np.array_equal(got[key], want[key]), key


def test_assign_limits(cuda_device):
    """Rows of the table that are too short, rows behind max_tokens, a stack with no room for what comes back, lengths that
    make no sense: bounded, and the others are served."""
    table = np.arange(4 * 6).reshape(4, 6)
    # request 1 needs a seventh column; the others get their blocks
    args = ([10, 90, 17, 32], [20, 10, 1, 1], table, np.arange(100, 140), 40, 16, 40)
    got, want = run_assign(cuda_device, *args), ref.assign(*args)
    assert want["denied"] == 1
    for key in want:
        assert np.array_equal(got[key], want[key]), key
    # max_tokens cuts request 2 off
    args = ([10, 20, 17, 32], [5, 5, 9, 0], table, np.arange(100, 140), 40, 16, 12)
    got, want = run_assign(cuda_device, *args), ref.assign(*args)
    assert want["denied"] == 1 and want["row_offsets"].tolist() == [0, 5, 10, 12, 12]
    for key in want:
        assert np.array_equal(got[key], want[key]), key
    # five blocks come back to a stack with room for two: two are kept, the count says two
    args = ([80], [-1], table[:1], np.array([7, -5, -5]), 1, 16, 4)
    got = run_assign(cuda_device, *args)
    assert got["free_blocks"].tolist() == [7, 0, 1] and got["free_count"] == 3
    # nonsense lengths are clamped to the table
    got = run_assign(cuda_device, [-9, 2000000000], [-1, 2000000000], table[:2], np.arange(9), 9, 16, 8)
    assert got["kv_len"].tolist() == [0, 96] and got["denied"] == 1 and (got["slots"] == -1).all()
    # no requests at all
    got = run_assign(cuda_device, [], [], np.zeros((0, 4)), np.arange(9), 9, 16, 8)
    assert got["free_count"] == 9 and got["denied"] == 0 and (got["slots"] == -1).all() and got["row_offsets"].tolist() == [0]


# ------------------------------------------------------------------------------------------------ store

def random_cache(rng, blocks, heads, bs, dim, device, order="hnd", spread=1.0):
    """(PagedCache, numpy codes k, v, scales k, v); every byte value occurs but NaN."""
    import torch
    np_codes, np_scales, tensors = [], [], []
    for _ in range(2):
        c = rng.integers(0, 256, (blocks, heads, bs, dim)).astype(np.uint8)
        c[(c & 127) == 127] = 0x35
        s = np.exp2(rng.integers(-12, -6, (blocks, heads))).astype(np.float32) * np.float32(spread)
        t = torch.from_numpy(c).to(device)
        if order == "nhd":                                 # tokens outside heads in memory
            t = t.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
        elif order == "wide":                              # rows of a larger allocation
            big = torch.zeros((blocks, heads + 1, bs + 2, dim + 16), dtype=torch.uint8, device=device)
            big[:, :heads, :bs, :dim] = t
            t = big[:, :heads, :bs, :dim]
        np_codes.append(c)
        np_scales.append(s)
        tensors += [t, torch.from_numpy(s).to(device)]
    return native.PagedCache(tensors[0], tensors[2], tensors[1], tensors[3]), np_codes, np_scales


def check_store(cache, codes, scales, k, v, slots):
    for got_c, got_s, c, s, x in ((cache.k, cache.k_scale, codes[0], scales[0], k), (cache.v, cache.v_scale, codes[1], scales[1], v)):
        want_c, want_s = ref.store(c, s, x.double().cpu().numpy(), slots)
        assert np.array_equal(got_s.cpu().numpy().astype(np.float64), want_s)
        assert np.array_equal(got_c.cpu().numpy(), want_c)


@pytest.mark.parametrize("order", ["hnd", "nhd", "wide"])
@pytest.mark.parametrize("kind,heads,bs,dim", [("bf16", 1, 16, 128), ("f16", 3, 32, 64), ("bf16", 8, 64, 64), ("f16", 2, 128, 128)])
def test_store(cuda_device, kind, heads, bs, dim, order):
    """Runs that fill a block, start inside one, end inside one, single rows, skipped rows; scales that rise and that do
    not."""
    import torch
    rng = np.random.default_rng(heads * bs + dim)
    blocks = 23
    cache, codes, scales = random_cache(rng, blocks, heads, bs, dim, cuda_device, order)
    ids = rng.permutation(blocks)
    slots = []
    for i, b in enumerate(ids[:15]):
        first = [0, 0, bs - 1, 5, bs // 2][i % 5]
        count = [bs, 3, 1, bs - 5, 1][i % 5]
        slots += [int(b) * bs + first + j for j in range(count)]
        if i % 4 == 0:
            slots += [-1, blocks * bs, -(1 << 40), 1 << 40][:1 + i % 4 + 1]
    n = len(slots)
    g = torch.Generator(device=cuda_device)
    g.manual_seed(heads)
    k, v = (torch.randn((n, heads, dim), generator=g, device=cuda_device) *
            torch.exp2(torch.randint(-9, 6, (n, heads, 1), generator=g, device=cuda_device).float()) for _ in range(2))
    k, v = k.to(torch_type(kind)), v.to(torch_type(kind))
    if order == "wide":                                    # rows inside a wider tensor, as a QKV product leaves them
        both = torch.cat([k, v], dim=1)
        k, v = both[:, :heads], both[:, heads:]
    native.cache_store(cache, k, v, torch.tensor(slots, dtype=torch.int64, device=cuda_device))
    check_store(cache, codes, scales, k, v, slots)


@pytest.mark.parametrize("n", [1, 3, 511, 512, 4095, 4097])
def test_store_window_borders(cuda_device, n):
    """Calls of every window size, runs across the windows' borders."""
    import torch
    rng = np.random.default_rng(n)
    bs, heads, dim = 16, 1, 64
    cache, codes, scales = random_cache(rng, n // bs + 3, heads, bs, dim, cuda_device)
    slots = [5 + i for i in range(n)]
    k, v = (torch.from_numpy(rng.standard_normal((n, heads, dim))).to(cuda_device).to(torch.bfloat16) for _ in range(2))
    native.cache_store(cache, k, v, torch.tensor(slots, dtype=torch.int64, device=cuda_device))
    check_store(cache, codes, scales, k, v, slots)


def test_store_special_values(cuda_device):
    """NaN, infinities, zeros, the largest and smallest magnitudes, exact powers, ties, and slots named twice."""
    import torch
    rng = np.random.default_rng(4)
    for kind, big, tiny in (("bf16", 3.3e38, 1e-40), ("f16", 65504.0, 6e-8)):
        cache, codes, scales = random_cache(rng, 12, 2, 16, 64, cuda_device)
        rows = rng.standard_normal((12, 2, 64))
        rows[0, 0, 3], rows[0, 1, 5] = np.nan, np.inf
        rows[1] = 0.0
        rows[2, 0] = big
        rows[3, 0] = -big
        rows[4] = tiny
        rows[5, 0] = 448.0 * np.exp2(np.arange(64) % 6)
        rows[6, 0] = np.nan
        rows[7, 0], rows[7, 1] = -np.inf, 0.0
        rows[8, 0, :32] = np.arange(32) / 16 + 1 / 32      # halves between codes
        k = torch.from_numpy(rows).to(cuda_device).to(torch_type(kind))
        v = k.flip(0).contiguous()
        # fresh blocks, rows behind older ones, and (at the end) one slot three times
        slots = [0, 16, 32, 48 + 7, 64 + 1, 80, 96 + 15, 112, 128 + 2, 144 + 4, 144 + 4, 144 + 4]
        native.cache_store(cache, k, v, torch.tensor(slots, dtype=torch.int64, device=cuda_device))
        check_store(cache, codes, scales, k, v, slots)


def test_store_foreign_scales(cuda_device):
    """A cache whose scales are no powers of two: kept while they suffice, codes divided by them."""
    import torch
    rng = np.random.default_rng(5)
    cache, codes, scales = random_cache(rng, 6, 2, 32, 128, cuda_device, spread=1.37)
    k, v = (torch.from_numpy(rng.standard_normal((6, 2, 128)) * 0.01).to(cuda_device).to(torch.float16) for _ in range(2))
    slots = [32 * b + 9 for b in range(6)]
    native.cache_store(cache, k, v, torch.tensor(slots, dtype=torch.int64, device=cuda_device))
    for got_c, got_s, c, s, x in ((cache.k, cache.k_scale, codes[0], scales[0], k), (cache.v, cache.v_scale, codes[1], scales[1], v)):
        want_c, want_s = ref.store(c, s, x.double().cpu().numpy(), slots)
        assert np.array_equal(got_s.cpu().numpy(), want_s.astype(np.float32))
        # x / scale and code * (old / new) round to float32 before the code: where the 64-bit quotient is within 2^-23 of a
        # border between two codes the code may be the neighbour's; nowhere else
        diff = got_c.cpu().numpy() != want_c
        assert diff.mean() <= 1e-4
        assert np.abs(got_c.cpu().numpy().astype(int) - want_c.astype(int)).max() <= 1


# ------------------------------------------------------------------------------------------------ attention

def attention_case(device, seed, q_lens, kv_lens, heads, kv_heads, dim, bs, kind="bf16", causal=True, window=0, order="hnd",
                   scale=None, pad=0, table=None, change=None, max_q=None, min_q=0, loud=1.0, sm_limit=0):
    """Runs one call and holds it against the reference."""
    import torch
    rng = np.random.default_rng(seed)
    n = len(kv_lens)
    columns = max(1, max(-(-k // bs) for k in kv_lens))
    blocks = sum(-(-k // bs) for k in kv_lens) + 2
    cache, codes, scales = random_cache(rng, blocks, kv_heads, bs, dim, device, order)
    # values of a magnitude that gives scores of a few units: codes reach 448, so scales of about 2^-9
    ids = rng.permutation(blocks)
    tab = np.full((n, columns), -1)
    at = 0
    for r, kv in enumerate(kv_lens):
        c = -(-kv // bs)
        tab[r, :c] = ids[at:at + c]
        at += c
    if table is not None:
        table(tab)
    offsets = np.concatenate([[0], np.cumsum(q_lens)])
    tokens = int(offsets[-1]) + pad
    q = rng.standard_normal((tokens, heads, dim)) * loud
    scale = dim ** -0.5 if scale is None else scale
    q_t = torch.from_numpy(q).to(device).to(torch_type(kind))
    # unused rows of the blocks, and blocks of nobody, hold anything: NaN codes and huge scales among it
    used = np.zeros((blocks, bs), dtype=bool)
    for r, kv in enumerate(kv_lens):
        for j in range(kv):
            if 0 <= tab[r, j // bs] < blocks:
                used[tab[r, j // bs], j % bs] = True
    for c, t in zip(codes, (cache.k, cache.v)):
        c[np.broadcast_to(~used[:, None, :, None], c.shape)] = 0x7F
    for s, t in zip(scales, (cache.k_scale, cache.v_scale)):
        s[~used.any(1)] = np.nan
        t.copy_(torch.from_numpy(s))
    if change is not None:
        change(codes, scales, tab, q_t)
        for s, t in zip(scales, (cache.k_scale, cache.v_scale)):
            t.copy_(torch.from_numpy(s))
    for c, t in zip(codes, (cache.k, cache.v)):
        t.copy_(torch.from_numpy(c))
    args = (cache, q_t, i32(offsets, device), i32(kv_lens, device), i32(tab, device))
    results = []
    for limit in (sm_limit, 1):                            # on few SMs a small call's long requests take the other kernel
        out = torch.full(q_t.shape, 7.0, dtype=q_t.dtype, device=device)
        lse = torch.full(q_t.shape[:2], 7.0, dtype=torch.float32, device=device)
        workspace = native.cache_attention_workspace(cache, q_t, requests=n, max_q=max_q or max(q_lens),
                                                     max_kv=max(kv_lens), sm_limit=limit)
        workspace.fill_(0xFF)
        kw = dict(scale=scale, max_q=max_q or max(q_lens), max_kv=max(kv_lens), min_q=min_q, causal=causal, window=window,
                  sm_limit=limit)
        native.cache_attention(*args, **kw, out=out, lse=lse, workspace=workspace)
        results.append((out, lse, kw))
    qd = q_t.double().cpu().numpy()
    want, want_lse = ref.attention(qd, codes[0], codes[1], scales[0], scales[1], offsets, kv_lens, tab, scale, causal, window)
    # sum p |v| / sum p, and the largest |q| |k| of a row
    mass, _ = ref.attention(qd, codes[0], np.where((codes[1] & 127) == 127, 0, codes[1] & 127).astype(np.uint8), scales[0],
                            scales[1], offsets, kv_lens, tab, scale, causal, window)
    inside = np.arange(tokens) < offsets[-1]
    qn = np.sqrt((np.nan_to_num(qd) ** 2).sum(2))
    kn = max((np.sqrt((np.nan_to_num(ref.VALUES[codes[0][b]]) ** 2).sum(-1)) * scales[0][b][:, None]).max()
             for b in range(blocks) if used[b].any()) if used.any() else 0.0
    err = dim * 2.0 ** -23 * abs(scale) * qn * kn + 2.0 ** -21
    grow = np.expm1(err)[..., None]
    bound = U[kind] * np.abs(want) + (2.0 ** -11 + 2 * grow) * mass + 1e-7
    if kind == "f16":
        bound = bound + 2.0 ** -25                         # half's subnormal step
    for out, lse, kw in results:
        got, got_lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
        assert (got[~inside] == 7.0).all() and (got_lse[~inside] == 7.0).all(), "rows outside every request were written"
        bad = inside[:, None, None] & ~((np.abs(got - want) <= bound) | (np.isnan(got) & np.isnan(want)))
        assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], want[bad][:5])
        fin = np.isfinite(want_lse) & inside[:, None]
        off = np.abs(np.where(fin, got_lse, 0.0) - np.where(fin, want_lse, 0.0))
        assert (off[fin] <= (err + 4 * 2.0 ** -23 * (np.abs(want_lse) + 30))[fin]).all()
        rest = inside[:, None] & ~np.isfinite(want_lse)
        assert np.array_equal(got_lse[rest], want_lse[rest], equal_nan=True)
        again = torch.full_like(out, 7.0)
        native.cache_attention(*args, **kw, out=again)     # without lse, with a workspace of its own
        assert torch.equal(out.view(torch.int16), again.view(torch.int16))
    return out, cache, args, kw


@pytest.mark.parametrize("bs", [16, 32, 64, 128])
@pytest.mark.parametrize("dim,kind", [(128, "bf16"), (64, "f16"), (128, "f16"), (64, "bf16")])
def test_attention_single_tokens(cuda_device, bs, dim, kind):
    """One token per request: lengths around a tile's and a page's end, one token, none."""
    attention_case(cuda_device, bs + dim, [1] * 9, [1, 2, 15, 16, 17, 63, 64, 65, 300], 8, 2, dim, bs, kind)
    attention_case(cuda_device, bs + dim, [1, 1, 1], [0, 129, 0], 5, 5, dim, bs, kind)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 3), (14, 2), (16, 1), (17, 1), (40, 1), (32, 8), (71, 1)])
def test_attention_head_groups(cuda_device, heads, kv_heads):
    """Groups of one head, odd groups, groups that pass a row tile."""
    attention_case(cuda_device, heads, [1, 2], [70, 130], heads, kv_heads, 64, 32)


@pytest.mark.parametrize("order", ["nhd", "wide"])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_cache_orders(cuda_device, order, dim):
    attention_case(cuda_device, 3, [1, 3, 40], [200, 77, 150], 8, 4, dim, 32, order=order)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window", [0, 1, 7, 64, 1000])
def test_attention_masks(cuda_device, causal, window):
    """Runs of tokens, prompts, queries before the first key (rows that see nothing), sliding windows."""
    attention_case(cuda_device, window, [1, 5, 70, 20, 130, 3], [200, 5, 70, 9, 330, 0], 4, 2, 64, 16, "f16", causal, window, pad=3)
    attention_case(cuda_device, window, [9, 0, 33], [150, 40, 33], 6, 2, 128, 64, "bf16", causal, window, pad=1)


@pytest.mark.parametrize("q_len", [1, 2, 4, 8, 9, 16, 17, 31, 64, 65, 127, 128, 129, 200])
def test_attention_row_counts(cuda_device, q_len):
    attention_case(cuda_device, q_len, [q_len, 1, q_len], [q_len + 100, 40, q_len], 4, 2, 64, 32)
    attention_case(cuda_device, q_len, [q_len], [q_len + 13], 2, 1, 128, 64, "f16", min_q=q_len)


def test_attention_long(cuda_device):
    """A context cut into many pieces, beside short ones, joined again."""
    attention_case(cuda_device, 8, [1, 1, 2], [9000, 3, 4100], 4, 1, 128, 64)
    attention_case(cuda_device, 9, [1], [20000], 2, 1, 64, 16, "f16")
    attention_case(cuda_device, 10, [40], [5000], 4, 1, 128, 128)


@pytest.mark.parametrize("sm_limit", [1, 3, 40])
def test_attention_on_a_share_of_the_sms(cuda_device, sm_limit):
    """Other cuts of the work, down to blocks that each take many items and items in many blocks."""
    attention_case(cuda_device, 51, [1, 1, 30, 2], [700, 3, 400, 64], 6, 2, 64, 16, "f16", sm_limit=sm_limit)
    attention_case(cuda_device, 52, [70, 300], [900, 310], 4, 1, 128, 64, min_q=70, sm_limit=sm_limit)


def test_attention_hints_are_only_hints(cuda_device):
    """min_q above what the requests have, max_q and max_kv far above it."""
    import torch
    attention_case(cuda_device, 53, [1, 40, 3], [90, 60, 200], 8, 2, 64, 32, min_q=40)
    attention_case(cuda_device, 54, [1, 2], [90, 60], 4, 2, 128, 32, max_q=500)
    # nothing cached at all, and a table without columns
    cache = native.PagedCache.empty(2, 2, 16, 64, cuda_device)
    for n, heads in ((1, 2), (40, 4)):
        q = torch.ones((n, heads, 64), dtype=torch.bfloat16, device=cuda_device)
        lse = torch.zeros((n, heads), device=cuda_device)
        out = native.cache_attention(cache, q, i32([0, n], cuda_device), i32([0], cuda_device),
                                     torch.zeros((1, 0), dtype=torch.int32, device=cuda_device), max_q=n, max_kv=0, lse=lse)
        assert bool((out == 0).all()) and bool(torch.isneginf(lse).all())
    # windows as wide as an int goes, of more rows than there are keys
    attention_case(cuda_device, 58, [1, 30], [90, 7], 4, 2, 64, 32, window=(1 << 31) - 1)
    attention_case(cuda_device, 59, [1, 30], [90, 7], 4, 2, 128, 32, window=89)


def test_attention_many_requests(cuda_device):
    """More requests than a block has threads, most of them empty or short."""
    rng = np.random.default_rng(55)
    q = rng.integers(0, 2, 1100).tolist()
    kv = [int(x) for x in rng.integers(0, 40, 1100)]
    attention_case(cuda_device, 55, q, kv, 1, 1, 64, 16)
    q[17] = 150
    attention_case(cuda_device, 56, q, kv, 1, 1, 64, 16, "f16")


def test_offsets_beyond_32_bits(cuda_device):
    """A cache of more than 2^32 bytes for K alone, its last blocks in use: store, decode step and prompt."""
    import torch
    bs, heads, dim = 128, 8, 128
    blocks = (1 << 32) // (bs * heads * dim) + 40
    k, v = (torch.empty((blocks, heads, bs, dim), dtype=torch.uint8, device=cuda_device) for _ in range(2))
    ks, vs = (torch.ones((blocks, heads), dtype=torch.float32, device=cuda_device) for _ in range(2))
    big = native.PagedCache(k, v, ks, vs)
    small = native.PagedCache.empty(4, heads, bs, dim, cuda_device)
    ids = [blocks - 1, blocks - 17, 3]
    g = torch.Generator(device=cuda_device)
    g.manual_seed(1)
    rows = 300
    x, y, q = (torch.randn((rows, heads, dim), generator=g, device=cuda_device).to(torch.bfloat16) for _ in range(3))
    for cache, table in ((big, ids), (small, [2, 0, 1])):
        slots = torch.tensor([table[t // bs] * bs + t % bs for t in range(rows)], dtype=torch.int64, device=cuda_device)
        native.cache_store(cache, x, y, slots)
    for n in (1, rows):
        args = (q[:n], i32([0, n], cuda_device), i32([rows], cuda_device))
        a = native.cache_attention(big, *args, i32([ids], cuda_device), max_q=n, max_kv=rows)
        b = native.cache_attention(small, *args, i32([[2, 0, 1]], cuda_device), max_q=n, max_kv=rows)
        assert torch.equal(a, b) and torch.isfinite(a.float()).all() and bool((a != 0).any())


def test_other_streams_and_wide_strides(cuda_device):
    """Inputs made on another stream than the call's, a block table and lengths inside larger tensors."""
    import torch
    rng = np.random.default_rng(57)
    cache, _, _ = random_cache(rng, 20, 2, 16, 64, cuda_device)
    q = torch.randn((6, 4, 64), device=cuda_device).to(torch.float16)
    table = i32(rng.permutation(20)[:15].reshape(3, 5), cuda_device)
    want = native.cache_attention(cache, q, i32([0, 1, 4, 6], cuda_device), i32([80, 50, 33], cuda_device), table, max_q=3, max_kv=80)
    wide = i32(np.full((3, 9), -1), cuda_device)
    wide[:, 2:7] = table
    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream(cuda_device))
    with torch.cuda.stream(side):
        qq = torch.zeros((6, 9, 72), dtype=torch.float16, device=cuda_device)
        qq[:, 3:7, :64] = q
        out = torch.full((6, 5, 64), 3.0, dtype=torch.float16, device=cuda_device)
        native.cache_attention(cache, qq[:, 3:7, :64], i32([0, 1, 4, 6], cuda_device), i32([80, 50, 33], cuda_device),
                               wide[:, 2:7], max_q=3, max_kv=80, out=out[:, 1:])
    torch.cuda.current_stream(cuda_device).wait_stream(side)
    assert torch.equal(out[:, 1:], want) and bool((out[:, 0] == 3.0).all())


def test_attention_nan_where_it_is_not_seen(cuda_device):
    """NaN codes and scores in tokens that a row does not see never reach it; where it sees them it is NaN, as in the
    formula."""
    def future(codes, scales, tab, q):
        # token 60 of request 0 (page 3 at 16 tokens a page): dim 5 of V; token 63: all of K
        codes[1][tab[0, 3], 0, 12, 5] = 0x7F
        codes[0][tab[0, 3], 0, 15, :] = 0xFF
        codes[1][tab[1, 0], 1, 0, 7] = 0x7F                # behind request 1's window for its last rows
    attention_case(cuda_device, 21, [8, 30], [64, 30], 4, 2, 64, 16, "f16", True, 20, change=future)
    attention_case(cuda_device, 22, [3, 2], [64, 30], 4, 2, 128, 16, "bf16", True, 0, change=future)
    attention_case(cuda_device, 23, [64, 30], [64, 30], 4, 2, 128, 16, "bf16", True, 9, change=future)

    def query(codes, scales, tab, q):
        q[1, 2, 3] = float("nan")
        q[2, 0, 9] = float("inf")
    import torch
    rng = np.random.default_rng(0)
    for q_lens, kv in (([4], [50]), ([40], [50])):
        cache, codes, scales = random_cache(rng, 9, 2, 16, 64, cuda_device)
        q = torch.randn((q_lens[0], 4, 64), device=cuda_device).to(torch.bfloat16)
        args = (i32([0, q_lens[0]], cuda_device), i32(kv, cuda_device), i32(np.arange(8)[None], cuda_device))
        clean = native.cache_attention(cache, q, *args, max_q=q_lens[0], max_kv=50)
        query(None, None, None, q)
        out = native.cache_attention(cache, q, *args, max_q=q_lens[0], max_kv=50)
        assert torch.isnan(out[1, 2]).all() and torch.isnan(out[2, 0]).all()
        out[1, 2], out[2, 0] = clean[1, 2], clean[2, 0]
        assert torch.equal(out, clean)


def test_attention_extremes(cuda_device):
    """Loud scores, tiny and huge scales, a block of zeros beside loud ones, queries of zero and of the type's extremes."""
    attention_case(cuda_device, 31, [1, 3], [200, 90], 4, 2, 128, 32, loud=40.0)
    attention_case(cuda_device, 32, [1, 40], [200, 90], 4, 2, 64, 32, "f16", loud=0.0)
    attention_case(cuda_device, 33, [2, 40], [200, 90], 4, 2, 64, 32, scale=0.0)
    attention_case(cuda_device, 34, [2, 40], [200, 90], 4, 2, 64, 32, scale=-0.11)

    def scales_apart(codes, scales, tab, q):
        scales[1][tab[0, 0]] = 2.0 ** -64                   # a block whose V is as good as nothing
        scales[1][tab[0, 1]] = 2.0 ** 20
        scales[0][tab[0, 2]] = 2.0 ** -60
    attention_case(cuda_device, 35, [1, 1], [200, 90], 4, 2, 64, 32, change=scales_apart)
    attention_case(cuda_device, 36, [50, 1], [200, 90], 4, 2, 128, 32, change=scales_apart)

    def tiny_queries(codes, scales, tab, q):
        q *= 2.0 ** -100
        q[0] *= 2.0 ** 60
        q[1] *= 2.0 ** 100
    attention_case(cuda_device, 37, [3, 20], [100, 90], 4, 2, 64, 32, change=tiny_queries)


def test_attention_blocks_that_do_not_exist(cuda_device):
    """Such tokens count as not seen, the status word says 8, and pages that no row sees are not looked at."""
    def damage(tab):
        tab[0, 1], tab[0, 2], tab[1, 0] = -1, 1 << 30, -(1 << 31)
    assert native.device_status() == 0
    attention_case(cuda_device, 41, [1, 1, 1], [100, 16, 40], 4, 2, 64, 16, table=damage)
    assert native.device_status() == 8
    attention_case(cuda_device, 42, [40, 20, 1], [100, 40, 40], 4, 2, 128, 16, table=damage)
    assert native.device_status() == 8
    # a window keeps pages in front of it out of use: their entries may be anything
    attention_case(cuda_device, 43, [1, 1, 1], [100, 48, 40], 4, 2, 64, 16, window=30, table=lambda t: t.__setitem__((0, 1), -1))
    assert native.device_status() == 0


def test_attention_broken_bounds(cuda_device):
    """Offsets and lengths outside their bounds are cut to them: nothing out of range is read or written."""
    import torch
    rng = np.random.default_rng(6)
    cache, _, _ = random_cache(rng, 8, 2, 16, 64, cuda_device)
    q = torch.randn((12, 4, 64), device=cuda_device).to(torch.bfloat16)
    table = i32(np.arange(8).reshape(2, 4), cuda_device)
    for offsets, kv in (([-5, 3, 400], [30, 20]), ([0, 9, 4], [64, 1 << 30]), ([0, 4, 12], [-7, 64])):
        out = native.cache_attention(cache, q, i32(offsets, cuda_device), i32(kv, cuda_device), table, max_q=5, max_kv=40)
        assert torch.isfinite(out.float()).all()
    assert native.device_status() == 0


# ------------------------------------------------------------------------------------------------ together

def serving_loop(device, steps, heads, kv_heads, dim, bs, graph=False, seed=0):
    """Prompts, then decode steps, one request ending and its blocks going to others; every step's attention against the
    reference over the cache's own codes, and the codes against the rows that were stored."""
    import torch
    rng = np.random.default_rng(seed)
    n, blocks, columns = 3, 24, 12
    cache = native.PagedCache.empty(blocks, kv_heads, bs, dim, device)
    table = torch.full((n, columns), -1, dtype=torch.int32, device=device)
    free, count = torch.arange(blocks, dtype=torch.int32, device=device), i32([blocks], device)
    kv = torch.zeros(n, dtype=torch.int32, device=device)
    denied = i32([0], device)
    codes = [cache.k.cpu().numpy(), cache.v.cpu().numpy()]
    scales = [cache.k_scale.cpu().numpy(), cache.v_scale.cpu().numpy()]
    plan = [[37, 5, 20], [1, 1, 1], [1, 0, 3], [1, -1, 1], [2, 30, 1]] + [[1, 1, 1]] * max(0, steps - 5)
    for new in plan[:steps]:
        tokens = sum(max(x, 0) for x in new) + 2            # a padded batch
        offsets = torch.zeros(n + 1, dtype=torch.int32, device=device)
        slots = torch.zeros(tokens, dtype=torch.int64, device=device)
        native.cache_assign(kv, i32(new, device), table, free, count, block_size=bs, row_offsets=offsets, kv_len=kv,
                            slots=slots, denied=denied)
        k, v = (torch.from_numpy(rng.standard_normal((tokens, kv_heads, dim))).to(device).to(torch.bfloat16) for _ in range(2))
        native.cache_store(cache, k, v, slots)
        q = torch.from_numpy(rng.standard_normal((tokens, heads, dim))).to(device).to(torch.bfloat16)
        out = native.cache_attention(cache, q, offsets, kv, table, max_q=max(max(new), 1), max_kv=columns * bs)
        assert int(denied.item()) == 0
        slots_h = slots.cpu().numpy().tolist()
        for i, (x, c, s) in enumerate(((k, cache.k, cache.k_scale), (v, cache.v, cache.v_scale))):
            codes[i], scales[i] = ref.store(codes[i], scales[i], x.double().cpu().numpy(), slots_h)
            assert np.array_equal(c.cpu().numpy(), codes[i]) and np.array_equal(s.cpu().numpy().astype(np.float64), scales[i])
        lens = kv.cpu().numpy()
        off = offsets.cpu().numpy()
        want, _ = ref.attention(q.double().cpu().numpy(), codes[0], codes[1], scales[0], scales[1], off, lens.tolist(),
                                table.cpu().numpy(), dim ** -0.5, True, 0)
        mass, _ = ref.attention(q.double().cpu().numpy(), codes[0], codes[1] & 127, scales[0], scales[1], off, lens.tolist(),
                                table.cpu().numpy(), dim ** -0.5, True, 0)
        used = off[-1]
        err = np.abs(out.double().cpu().numpy() - want)[:used]
        assert (err <= 2.0 ** -8 * np.abs(want[:used]) + 2.0 ** -10 * mass[:used] + 1e-6).all()
        assert (out[used:] == 0).all()
    live = sum(-(-int(x) // bs) for x in kv.cpu().numpy())
    assert int(count.item()) == blocks - live
    held = set(free.cpu().numpy()[:blocks - live].tolist())
    rows = table.cpu().numpy()
    for r, x in enumerate(kv.cpu().numpy()):
        held |= set(rows[r, :-(-int(x) // bs)].tolist())
    assert held == set(range(blocks))                       # no block lost, none twice


@pytest.mark.parametrize("dim,bs,heads,kv_heads", [(128, 16, 8, 2), (64, 32, 6, 3)])
def test_serving_loop(cuda_device, dim, bs, heads, kv_heads):
    serving_loop(cuda_device, 8, heads, kv_heads, dim, bs)


def test_between_the_gemms(cuda_device):
    """As a layer uses them: the QKV product's rows go to the store and the attention as views, the attention's output
    through the FP8 quantiser into the output product."""
    import torch
    heads, kv_heads, dim, bs, rows, width = 8, 2, 128, 64, 96, 512
    g = torch.Generator(device=cuda_device)
    g.manual_seed(3)
    x = torch.randn((rows, width), generator=g, device=cuda_device).to(torch.bfloat16)
    w = (torch.randn(((heads + 2 * kv_heads) * dim, width), generator=g, device=cuda_device) * width ** -0.5).to(torch.bfloat16)
    qkv = native.dense_gemm(x, w).view(rows, heads + 2 * kv_heads, dim)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
    cache = native.PagedCache.empty(8, kv_heads, bs, dim, cuda_device)
    table = torch.full((2, 4), -1, dtype=torch.int32, device=cuda_device)
    free, count = torch.arange(8, dtype=torch.int32, device=cuda_device), i32([8], cuda_device)
    kv, offsets = i32([0, 0], cuda_device), i32([0, 0, 0], cuda_device)
    slots = torch.zeros(rows, dtype=torch.int64, device=cuda_device)
    native.cache_assign(kv, i32([90, 6], cuda_device), table, free, count, block_size=bs, row_offsets=offsets, kv_len=kv, slots=slots)
    native.cache_store(cache, k, v, slots)
    out = native.cache_attention(cache, q, offsets, kv, table, max_q=90, max_kv=256)
    codes, scale = native.quantize_fp8_row_groups(out.reshape(rows, heads * dim).float())
    wo, so = native.quantize_fp8_blocks(torch.randn((256, heads * dim), generator=g, device=cuda_device) * 0.03)
    y = native.fp8_gemm(codes, scale, wo, so)
    # the same attention from the unquantised rows: K and V lose at most 2^-4 of each element in the cache
    for a, b in ((0, 90), (90, 96)):
        kk, vv = (t[a:b].double().repeat_interleave(heads // kv_heads, 1).transpose(0, 1) for t in (k, v))
        s = q[a:b].double().transpose(0, 1) @ kk.transpose(1, 2) * dim ** -0.5
        s = s.masked_fill(torch.triu(torch.ones(b - a, b - a, dtype=torch.bool, device=cuda_device), 1), -float("inf"))
        want = (torch.softmax(s, -1) @ vv).transpose(0, 1)
        rel = (out[a:b].double() - want).norm() / want.norm()
        assert rel < 2.0 ** -4
    assert torch.isfinite(y.float()).all() and native.device_status() == 0


def test_graphs_streams_and_two_calls_at_once(cuda_device):
    """A captured step replayed on other lengths gives what the calls give; two graphs of different shapes share a
    workspace in turn; two streams with a workspace each run at once."""
    import torch
    rng = np.random.default_rng(12)
    bs, dim, heads, kv_heads = 16, 64, 4, 2

    def problem(n, longest, q_len):
        cache, _, _ = random_cache(rng, n * (-(-longest // bs)), kv_heads, bs, dim, cuda_device)
        table = i32(rng.permutation(cache.num_blocks).reshape(n, -1), cuda_device)
        q = torch.randn((n * q_len, heads, dim), device=cuda_device).to(torch.bfloat16)
        offsets = i32(np.arange(n + 1) * q_len, cuda_device)
        kv = i32(rng.integers(q_len, longest + 1, n), cuda_device)
        out = torch.zeros_like(q)
        return cache, q, offsets, kv, table, out, dict(max_q=q_len, max_kv=longest)

    a, b = problem(5, 600, 1), problem(2, 3000, 40)
    need = max(native.cache_attention_workspace_bytes(x[0], x[1], requests=x[3].numel(), **x[6]) for x in (a, b))
    shared = torch.empty(need, dtype=torch.uint8, device=cuda_device)
    graphs = []
    for x in (a, b):
        native.cache_attention(*x[:5], **x[6], out=x[5], workspace=shared)          # first use outside the capture
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            native.cache_attention(*x[:5], **x[6], out=x[5], workspace=shared)
        graphs.append(g)
    for round_ in range(3):
        for x in (a, b):
            x[3].copy_(i32(rng.integers(x[6]["max_q"], x[6]["max_kv"] + 1, x[3].numel()), cuda_device))
            x[5].zero_()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for x in (a, b):
            assert torch.equal(x[5], native.cache_attention(*x[:5], **x[6]))
    streams = [torch.cuda.Stream(cuda_device) for _ in range(2)]
    outs = [[], []]
    torch.cuda.synchronize()
    for _ in range(4):
        for s, x, o in zip(streams, (a, b), outs):
            with torch.cuda.stream(s):
                o.append(native.cache_attention(*x[:5], **x[6]))
    torch.cuda.synchronize()
    for x, o in zip((a, b), outs):
        assert all(torch.equal(y, x[5]) for y in o)
    assert native.device_status() == 0
