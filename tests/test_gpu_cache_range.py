"""GPU: the cache attention where weights and scales lie far apart, against tests/cache_reference.py (64 bits)."""
import numpy as np
import pytest

import cache_reference as ref
from ops_tensor_b200 import native
from test_gpu_cache import attention_case, i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("code,at", [(0x62, 5), (0x63, 5), (0x64, 5), (0x64, 1500)])
def test_attention_sink_without_a_value(cuda_device, kind, code, at):
    """One token outweighs every other by 20 to 25 bits and has no value, as an attention sink: the output is made by the
    small weights alone, which have to keep their 11 bits in both kernels (attention_case's second run, on one SM, takes
    the 40 packed rows through the many-rows kernel).  Query elements are about one, so the sink's score is
    128^-0.5 * 128 * its key's value (40, 44, 48 / 32) = 14.1, 15.6, 17.0 against scores of 0: weights of 2^-20.4 to 2^-24.5
    of the largest, 2^-26 being where the many-rows kernel's halves become subnormal.  The small weights of a row are
    equal, so their roundings do not cancel.  Outputs are 0.04 to 1, far above the 1e-7 that the bound has for zeros."""
    def sink(codes, scales, tab, q):
        rng = np.random.default_rng(code + at)
        codes[0][:] = 0
        codes[1][:] = rng.integers(0x60, 0x7F, codes[1].shape)                     # 32 to 448, times 2
        scales[0][:], scales[1][:] = 2.0 ** -5, 2.0
        block, row = tab[0, at // 32], at % 32
        codes[0][block, :, row], codes[1][block, :, row] = code, 0
        q *= 0.02
        q += 1.0
    attention_case(cuda_device, 61, [20], [3000], 2, 1, 128, 32, kind, change=sink)


@pytest.mark.parametrize("dim,kind", [(128, "bf16"), (64, "f16")])
def test_attention_loud_scores_in_many_rows(cuda_device, dim, kind):
    """Scores of hundreds in rows of the many-rows kernel: references that grow from tile to tile."""
    attention_case(cuda_device, 62, [30, 3], [900, 90], 4, 2, dim, 32, kind, loud=40.0)


def scales_case(device, q_lens, kv_lens, dim, v_scale_of, counts_as, sm_limit):
    """A call on V scales that `v_scale_of(tab)` gives, held against the reference on `counts_as` of them, relative to the
    values that a row sums.  A score with log2 of the V scale is up to 2^8, so it, the reference taken from it and that log2
    (approximated to 2^-22 of its value) are off by at most 2^-16 each, an exponential by 2^-21; lse, (m + log2 l) ln 2 with
    both up to 2^8, by as much again."""
    import torch
    rng = np.random.default_rng(71)
    bs, heads, kv_heads, n = 16, 4, 2, len(kv_lens)
    columns = max(-(-k // bs) for k in kv_lens)
    blocks = n * columns
    tab = rng.permutation(blocks).reshape(n, columns)
    codes = [rng.integers(0, 0x30, (blocks, kv_heads, bs, dim)).astype(np.uint8) for _ in range(2)]       # up to 0.5
    codes[0] |= rng.integers(0, 2, codes[0].shape).astype(np.uint8) << 7
    k_scale = np.ones((blocks, kv_heads), np.float32)
    v_scale = v_scale_of(tab, np.ones((blocks, kv_heads), np.float64)).astype(np.float32)
    cache = native.PagedCache(*(torch.from_numpy(x).to(device) for x in (codes[0], codes[1], k_scale, v_scale)))
    offsets = np.concatenate([[0], np.cumsum(q_lens)])
    q = torch.from_numpy(rng.standard_normal((offsets[-1], heads, dim))).to(device).to(torch.bfloat16)
    lse = torch.empty((offsets[-1], heads), dtype=torch.float32, device=device)
    out = native.cache_attention(cache, q, i32(offsets, device), i32(kv_lens, device), i32(tab, device), max_q=max(q_lens),
                                 max_kv=max(kv_lens), lse=lse, sm_limit=sm_limit)
    args = (q.double().cpu().numpy(), codes[0], codes[1], k_scale, counts_as(v_scale.astype(np.float64)), offsets, kv_lens, tab,
            dim ** -0.5, True, 0)
    want, want_lse = ref.attention(*args)                  # (V is not negative: `want` is what the row sums)
    size = np.linalg.norm(args[0], axis=2) * np.linalg.norm(ref.VALUES[codes[0]], axis=3).max()
    err = dim * 2.0 ** -23 * dim ** -0.5 * size + 2.0 ** -21 + 3 * 2.0 ** -16
    got, got_lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
    big = np.abs(want) > 3.38e38                           # bf16's end
    ok = np.abs(got - want) <= (2.0 ** -8 + 2.0 ** -11 + 2 * np.expm1(err)[..., None]) * want
    assert (ok | big & np.isinf(got)).all(), (got[~ok][:5], want[~ok][:5])
    assert (np.abs(got_lse - want_lse) <= err + 2.0 ** -14 + 2.0 ** -22 * np.abs(want_lse)).all()


@pytest.mark.parametrize("sm_limit", [0, 1])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("exponent", [-64, -70, 20, 118, 120, 125.7, 126.5, 127.9])
def test_attention_v_scale_ends(cuda_device, dim, exponent, sm_limit):
    """Every V scale at the ends of what the store writes, behind them, and at float32's own upper end."""
    scales_case(cuda_device, [1, 30], [200, 300], dim, lambda tab, s: s * 2.0 ** exponent, lambda s: np.maximum(s, 2.0 ** -64),
                sm_limit)


@pytest.mark.parametrize("sm_limit", [0, 1])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_v_scales_far_apart(cuda_device, dim, sm_limit):
    """V scales 2^96 apart in one row: the tokens of the small ones add nothing to the output but their weights count."""
    def apart(tab, s):
        s[tab[0, ::2]], s[tab[1, 3:]] = 2.0 ** -64, 2.0 ** -64
        s[tab[0, 1::2]], s[tab[1, :3]] = 2.0 ** 32, 2.0 ** 32
        return s
    scales_case(cuda_device, [1, 30], [200, 300], dim, apart, lambda s: s, sm_limit)
