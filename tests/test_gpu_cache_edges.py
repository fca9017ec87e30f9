"""GPU: the paged-cache operators at the edges of their buffers (every kind of slot outside the cache, guards around all that
is written, lengths and offsets that make no sense) and a whole step captured once and replayed."""
import numpy as np
import pytest

import cache_reference as ref
from ops_tensor_b200 import native
from test_gpu_cache import check_store, i32, random_cache

pytestmark = pytest.mark.gpu
INT_MIN, INT_MAX = -(1 << 31), (1 << 31) - 1


@pytest.mark.parametrize("kind,heads,bs,dim", [("bf16", 2, 16, 128), ("f16", 3, 64, 64)])
def test_store_skips_every_slot_outside_the_cache(cuda_device, kind, heads, bs, dim):
    """Slots below, just behind and far outside the cache, up to the ends of 64 bits and at values whose low 32 bits would
    be inside, before, between and behind runs of several lengths."""
    import torch
    rng = np.random.default_rng(bs)
    blocks = 21
    cache, codes, scales = random_cache(rng, blocks, heads, bs, dim, cuda_device)
    outside = [-1, blocks * bs, -(1 << 40), 1 << 40, -(1 << 63), (1 << 63) - 1, (1 << 32) + 3, -(1 << 32) + 5, INT_MIN,
               1 << 31, -blocks * bs, blocks * bs + 1]
    slots, ids = [outside[0]], rng.permutation(blocks)
    for i, b in enumerate(ids[:18]):
        first, count = [(0, bs), (3, 2), (bs - 1, 1), (5, bs - 5), (1, 7)][i % 5]
        slots += [int(b) * bs + first + j for j in range(count)]
        slots += [outside[(i + j) % len(outside)] for j in range(1 + i % 4)]
    slots += outside
    assert all(slots.count(x) >= 2 for x in outside)
    k, v = (torch.from_numpy(rng.standard_normal((len(slots), heads, dim))).to(cuda_device)
            .to({"bf16": torch.bfloat16, "f16": torch.float16}[kind]) for _ in range(2))
    native.cache_store(cache, k, v, torch.tensor(slots, dtype=torch.int64, device=cuda_device))
    check_store(cache, codes, scales, k, v, slots)


@pytest.mark.parametrize("kind,bs,dim", [("bf16", 16, 128), ("f16", 128, 64), ("bf16", 128, 128)])
def test_store_runs_in_any_order(cuda_device, kind, bs, dim):
    """Rows of one block in reverse, shuffled, with holes, and slots named again near by and far off, in runs of up to twice a
    block: the last row of a slot stays, all of them count for the scale."""
    import torch
    rng = np.random.default_rng(bs + dim)
    blocks, heads = 9, 2
    cache, codes, scales = random_cache(rng, blocks, heads, bs, dim, cuda_device)
    rows = [np.arange(bs)[::-1], rng.permutation(bs), rng.permutation(bs)[:bs // 2 + 1], rng.integers(0, bs, 2 * bs),
            rng.integers(bs // 2, bs, bs), np.r_[np.arange(3, bs), np.arange(bs - 4)], np.repeat(np.arange(1, bs), 2),
            np.array([7, 5, 7]), np.full(9, bs - 1)]
    slots = [int(b) * bs + int(x) for b, r in zip(rng.permutation(blocks), rows) for x in r]
    k, v = (torch.from_numpy(rng.standard_normal((len(slots), heads, dim)) * np.exp2(rng.integers(-6, 7, (len(slots), heads, 1))))
            .to(cuda_device).to({"bf16": torch.bfloat16, "f16": torch.float16}[kind]) for _ in range(2))
    native.cache_store(cache, k, v, torch.tensor(slots, dtype=torch.int64, device=cuda_device))
    check_store(cache, codes, scales, k, v, slots)


class Guarded:
    """A tensor inside a larger one whose borders have to stay as they are."""

    def __init__(self, shape, dtype, device, value, guard=64):
        import torch
        self.n, self.guard, self.value = int(np.prod(shape)), guard, value
        self.all = torch.full((self.n + 2 * guard,), value, dtype=dtype, device=device)
        self.inside = self.all[guard:guard + self.n].view(shape)

    def intact(self):
        return bool((self.all[:self.guard] == self.value).all()) and bool((self.all[self.guard + self.n:] == self.value).all())


@pytest.mark.parametrize("sm_limit", [0, 1])
@pytest.mark.parametrize("q_off,kv,rows,lens", [
    ([-5, 3, 400], [30, 20], [(0, 3), (3, 33)], [30, 20]),            # behind the last row, before the first
    ([0, 50, 4], [64, 1 << 30], [(0, 30), (50, 50)], [40, 40]),       # falling
    ([0, 4, 60], [-7, 64], [(0, 4), (4, 34)], [0, 40]),               # more rows than max_q, longer than max_kv
    ([INT_MIN, 2, INT_MAX], [INT_MAX, INT_MIN], [(0, 2), (2, 32)], [40, 0]),
    ([INT_MAX, INT_MIN, INT_MIN], [5, 5], [(60, 60), (0, 0)], [5, 5]),
    ([60, 60, 60], [40, 40], [(60, 60), (60, 60)], [40, 40])])
def test_attention_cuts_offsets_and_lengths(cuda_device, q_off, kv, rows, lens, sm_limit):
    """60 rows, max_q 30, max_kv 40: `rows` and `lens` are what is left of the offsets and lengths.  The rows that a request
    has are the reference's, all others, and what lies around out, lse and the workspace, stay as they were (up to 60
    packed rows a request: on one SM the many-rows kernel, else the few-rows kernel)."""
    import torch
    rng = np.random.default_rng(6)
    heads, kv_heads, dim, tokens = 4, 2, 64, 60
    cache, codes, scales = random_cache(rng, 8, kv_heads, 16, dim, cuda_device)
    q = torch.from_numpy(rng.standard_normal((tokens, heads, dim))).to(cuda_device).to(torch.bfloat16)
    tab = np.arange(8).reshape(2, 4)
    out = Guarded((tokens, heads, dim), torch.bfloat16, cuda_device, 7.0)
    lse = Guarded((tokens, heads), torch.float32, cuda_device, 7.0)
    need = native.cache_attention_workspace_bytes(cache, q, requests=2, max_q=30, max_kv=40, sm_limit=sm_limit)
    space = Guarded((need,), torch.uint8, cuda_device, 0xA5, guard=4096)
    native.cache_attention(cache, q, i32(q_off, cuda_device), i32(kv, cuda_device), i32(tab, cuda_device), max_q=30, max_kv=40,
                           out=out.inside, lse=lse.inside, workspace=space.inside, sm_limit=sm_limit)
    assert out.intact() and lse.intact() and space.intact() and native.device_status() == 0
    got, got_lse = out.inside.double().cpu().numpy(), lse.inside.double().cpu().numpy()
    qd = q.double().cpu().numpy()
    written = np.zeros(tokens, dtype=bool)
    for r, ((a, b), n) in enumerate(zip(rows, lens)):
        written[a:b] = True
        args = ([0, b - a], [n], tab[r:r + 1], dim ** -0.5, True, 0)
        want, want_lse = ref.attention(qd[a:b], codes[0], codes[1], scales[0], scales[1], *args)
        mass, _ = ref.attention(qd[a:b], codes[0], codes[1] & 127, scales[0], scales[1], *args)
        # output 2^-8, probabilities 2^-11, scores dim * 2^-23 * scale |q| |k| with |q| |k| below 12 * 64^0.5 * 448 * 2^-7
        err = dim * 2.0 ** -23 * dim ** -0.5 * 12 * 8 * 448 * 2.0 ** -7 + 2.0 ** -21
        assert (np.abs(got[a:b] - want) <= 2.0 ** -8 * np.abs(want) + (2.0 ** -11 + 2 * np.expm1(err)) * mass + 1e-7).all()
        empty = np.isneginf(want_lse)
        assert np.array_equal(np.isneginf(got_lse[a:b]), empty)
        assert (np.abs(got_lse[a:b][~empty] - want_lse[~empty]) <= err + 4 * 2.0 ** -23 * (np.abs(want_lse[~empty]) + 30)).all()
    assert (got[~written] == 7.0).all() and (got_lse[~written] == 7.0).all()


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("seed", range(6))
def test_assign_stays_in_its_buffers(cuda_device, seed, in_place):
    """Lengths of any value, a count of free blocks below zero and above the stack, on one block and many: what lies around
    every output stays as it was, and the lists agree with the loop on the cut values."""
    import torch
    rng = np.random.default_rng(seed)
    n, block, columns, capacity = [1, 5, 40, 300, 37, 2][seed], [16, 128, 32, 64, 16, 64][seed], 7, [30, 90, 60, 700, 0, 5][seed]
    max_tokens = [9, 40, 3000, 20000, 60, 0][seed]
    odd = np.array([INT_MIN, -1, 0, 1, 2, block, columns * block, columns * block + 1, INT_MAX], dtype=np.int64)
    cached = np.where(rng.random(n) < 0.3, rng.choice(odd, n), rng.integers(0, columns * block + 1, n))
    new = np.where(rng.random(n) < 0.3, rng.choice(odd, n), rng.integers(-1, 2 * block, n))
    count = [INT_MAX, -9, 60, 350, 3, INT_MIN][seed]
    guarded = {"table": Guarded((n, columns), torch.int32, cuda_device, -5), "free": Guarded((capacity,), torch.int32, cuda_device, -5),
               "count": Guarded((1,), torch.int32, cuda_device, -5), "cached": Guarded((n,), torch.int32, cuda_device, -5),
               "offsets": Guarded((n + 1,), torch.int32, cuda_device, -5), "slots": Guarded((max_tokens,), torch.int64, cuda_device, -5),
               "positions": Guarded((max_tokens,), torch.int32, cuda_device, -5), "denied": Guarded((1,), torch.int32, cuda_device, -5),
               "kv": Guarded((n,), torch.int32, cuda_device, -5), "left": Guarded((1,), torch.int32, cuda_device, -5)}
    t = {k: g.inside for k, g in guarded.items()}
    table, free = rng.permutation(n * columns).reshape(n, columns), rng.permutation(capacity) + 5000
    for key, x in (("table", table), ("free", free), ("count", [count]), ("cached", cached)):
        t[key].copy_(i32(x, cuda_device).reshape(t[key].shape))
    kv, left = (t["cached"], t["count"]) if in_place else (t["kv"], t["left"])
    native.cache_assign(t["cached"], i32(new, cuda_device), t["table"], t["free"], t["count"], block_size=block,
                        row_offsets=t["offsets"], kv_len=kv, slots=t["slots"], positions=t["positions"], free_count_out=left,
                        denied=t["denied"])
    assert all(g.intact() for g in guarded.values())
    cut = np.clip(cached, 0, columns * block)
    # (the loop walks a request's rows one by one: as many as pass every limit stand for 2^31)
    some = np.minimum(new, columns * block + max_tokens + 1)
    want = ref.assign(cut.tolist(), some.tolist(), table, free, min(max(count, 0), capacity), block, max_tokens)
    got = {"block_table": t["table"], "free_blocks": t["free"], "row_offsets": t["offsets"], "kv_len": kv, "slots": t["slots"],
           "positions": t["positions"]}
    for key, x in got.items():
        assert np.array_equal(x.cpu().numpy(), want[key]), key
    assert int(left.item()) == min(want["free_count"], capacity) and int(t["denied"].item()) == want["denied"]


@pytest.mark.parametrize("dim,bs,heads,kv_heads,rows", [(64, 16, 6, 3, 60), (128, 32, 8, 2, 1100)])
def test_captured_step(cuda_device, dim, bs, heads, kv_heads, rows):
    """Assign, store and attention of a padded batch captured once, lengths updated in place, and replayed on other lengths:
    prompts, decode steps, drafted tokens, requests that wait, end and start again.  1100 rows take assign's second launch.
    Codes, scales, tables and lists have to be the loop's; the attention's bound is 2^-8 of the output, 2^-11 for its
    probabilities and less than 2^-11 for the scores: |q| |k| <= dim (1 + 2^-4), twice dim^0.5 * 2^-23 times that."""
    import torch
    rng = np.random.default_rng(dim)
    n, blocks, columns = 4, 30, 9
    torch_rows = lambda h: torch.zeros((rows, h, dim), dtype=torch.bfloat16, device=cuda_device)

    def state():
        return dict(cache=native.PagedCache.empty(blocks, kv_heads, bs, dim, cuda_device), kv=i32([0] * n, cuda_device),
                    table=torch.full((n, columns), -1, dtype=torch.int32, device=cuda_device),
                    free=torch.arange(blocks, dtype=torch.int32, device=cuda_device), count=i32([blocks], cuda_device),
                    denied=i32([0], cuda_device), new=i32([0] * n, cuda_device), offsets=i32([0] * (n + 1), cuda_device),
                    slots=torch.zeros(rows, dtype=torch.int64, device=cuda_device), k=torch_rows(kv_heads), v=torch_rows(kv_heads),
                    q=torch_rows(heads), out=torch_rows(heads), lse=torch.zeros((rows, heads), device=cuda_device))

    def step(s, space):
        native.cache_assign(s["kv"], s["new"], s["table"], s["free"], s["count"], block_size=bs, row_offsets=s["offsets"],
                            kv_len=s["kv"], slots=s["slots"], denied=s["denied"])
        native.cache_store(s["cache"], s["k"], s["v"], s["slots"])
        native.cache_attention(s["cache"], s["q"], s["offsets"], s["kv"], s["table"], max_q=50, max_kv=columns * bs, out=s["out"],
                               lse=s["lse"], workspace=space)

    s = state()
    space = native.cache_attention_workspace(s["cache"], s["q"], requests=n, max_q=50, max_kv=columns * bs)
    step(state(), space)                                              # first calls outside the capture, on other tensors
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(s, space)
    codes = [np.zeros((blocks, kv_heads, bs, dim), np.uint8) for _ in range(2)]
    scales = [np.ones((blocks, kv_heads)) for _ in range(2)]
    table, free, count, kv = s["table"].cpu().numpy(), np.arange(blocks), blocks, [0] * n
    for new in ([20, 0, 7, 1], [1, 33, 1, 1], [4, 1, -1, 1], [1, 1, 9, 0], [-1, 2, 1, 30], [5, 1, 1, -1], [1, 1, 1, 1]):
        data = {"k": kv_heads, "v": kv_heads, "q": heads}
        for key, h in data.items():
            s[key].copy_(torch.from_numpy(rng.standard_normal((rows, h, dim))).to(cuda_device).clamp(-1, 1))
        s["new"].copy_(i32(new, cuda_device))
        s["out"].fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        a = ref.assign(kv, new, table, free, count, bs, rows)
        for key, x in (("block_table", s["table"]), ("free_blocks", s["free"]), ("row_offsets", s["offsets"]), ("kv_len", s["kv"]),
                       ("slots", s["slots"])):
            assert np.array_equal(x.cpu().numpy(), a[key]), key
        assert int(s["count"].item()) == a["free_count"] and int(s["denied"].item()) == a["denied"] == 0
        table, free, count, kv = a["block_table"], a["free_blocks"], a["free_count"], a["kv_len"].tolist()
        for i, (x, c, w) in enumerate(((s["k"], s["cache"].k, s["cache"].k_scale), (s["v"], s["cache"].v, s["cache"].v_scale))):
            codes[i], scales[i] = ref.store(codes[i], scales[i], x.double().cpu().numpy(), a["slots"].tolist())
            assert np.array_equal(c.cpu().numpy(), codes[i]) and np.array_equal(w.cpu().numpy().astype(np.float64), scales[i])
        used = a["row_offsets"][-1]
        args = (scales[0], scales[1], a["row_offsets"], kv, table, dim ** -0.5, True, 0)
        q = s["q"].double().cpu().numpy()[:used]
        want, want_lse = ref.attention(q, codes[0], codes[1], *args)
        mass, _ = ref.attention(q, codes[0], codes[1] & 127, *args)
        got = s["out"].double().cpu().numpy()
        assert (np.abs(got[:used] - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -10 * mass + 1e-7).all()
        assert (np.abs(s["lse"].double().cpu().numpy()[:used] - want_lse) <= 2.0 ** -11).all()
        assert (got[used:] == 7.0).all()
    assert native.device_status() == 0


def test_layers_without_waiting(cuda_device):
    """Steps of a layer (QKV product, assign, store, attention, quantiser, output product) issued without waiting for anything,
    with buffers used again at once, against the same steps with a wait behind every call: equal bit for bit.  The kernels
    start before the one in front of them has ended (programmatic stream serialisation) and may touch nothing until it
    has."""
    import torch
    heads, kv_heads, dim, bs, width, steps = 8, 2, 128, 64, 512, 12
    g = torch.Generator(device=cuda_device)
    g.manual_seed(9)
    w = (torch.randn(((heads + 2 * kv_heads) * dim, width), generator=g, device=cuda_device) * width ** -0.5).to(torch.bfloat16)
    wo, so = native.quantize_fp8_blocks(torch.randn((width, heads * dim), generator=g, device=cuda_device) * 0.03)
    news = [[200, 3, 70]] + [[1, 1, 1], [4, 0, 90], [1, 30, 1], [-1, 1, 1], [130, 1, 2]] * 3
    inputs = [(torch.randn((240, width), generator=g, device=cuda_device).to(torch.bfloat16), i32(n, cuda_device))
              for n in news[:steps]]

    def run(wait):
        cache = native.PagedCache.empty(40, kv_heads, bs, dim, cuda_device)
        table = torch.full((3, 16), -1, dtype=torch.int32, device=cuda_device)
        free, count = torch.arange(40, dtype=torch.int32, device=cuda_device), i32([40], cuda_device)
        kv, offsets = i32([0] * 3, cuda_device), i32([0] * 4, cuda_device)
        slots = torch.zeros(280, dtype=torch.int64, device=cuda_device)[:240]
        out = torch.zeros((240, heads, dim), dtype=torch.bfloat16, device=cuda_device)
        results, space = [], None
        pause = torch.cuda.synchronize if wait else (lambda: None)
        for x, new in inputs:
            qkv = native.dense_gemm(x, w).view(240, heads + 2 * kv_heads, dim)
            pause()
            q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
            native.cache_assign(kv, new, table, free, count, block_size=bs, row_offsets=offsets, kv_len=kv, slots=slots)
            pause()
            native.cache_store(cache, k, v, slots)
            pause()
            if space is None:
                space = native.cache_attention_workspace(cache, q, requests=3, max_q=200, max_kv=1024)
            out.zero_()
            native.cache_attention(cache, q, offsets, kv, table, max_q=200, max_kv=1024, out=out, workspace=space)
            pause()
            codes, scale = native.quantize_fp8_row_groups(out.view(240, heads * dim).float())
            pause()
            results += [out.clone(), native.fp8_gemm(codes, scale, wo, so)]
            pause()
        torch.cuda.synchronize()
        return results + [cache.k, cache.v, cache.k_scale, cache.v_scale, table, kv, count, slots]

    want = run(True)
    for _ in range(4):
        for a, b in zip(run(False), want):
            assert torch.equal(a, b)
    assert all(bool((x != 0).any()) for x in want) and native.device_status() == 0
