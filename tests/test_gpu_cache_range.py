"""GPU: the cache attention where weights and scales lie far apart, against tests/cache_reference.py (64 bits)."""
import numpy as np
import pytest

from test_gpu_cache import attention_case

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
