"""Calls of the cache attention that cannot give what its formula says, refused before anything is launched (no GPU needed;
pointers are made-up numbers)."""
import ctypes as C

import pytest

from ops_tensor_b200 import native
from test_cache_boundary import INVALID, NO_SPACE, OK, P, attention, cache, lib  # noqa: F401


@pytest.mark.parametrize("scale,status", [
    (3.0e38, INVALID), (-2.4e38, INVALID), (3.4028234e38, INVALID), (2.3e38, OK), (-2.3e38, OK), (0.0, OK), (1e-45, OK)])
def test_scales_that_powers_of_two_cannot_hold(lib, scale, status):
    """Scores are taken as powers of two: scale * log2(e) has to be a finite float32."""
    n = C.c_size_t(5)
    assert lib.blazeCacheAttentionWorkspaceSize(C.byref(cache()), C.byref(attention(scale=scale)), C.byref(n)) == status
    # (a call that is right otherwise ends at its workspace)
    got = lib.blazeCacheAttention(C.byref(cache()), C.byref(attention(scale=scale, out=2 * P, workspace=None)), None)
    assert got == (NO_SPACE if status == OK else status)


def test_output_over_the_queries(lib):
    """A query row is read by every block that has a part of its work, so the output cannot take its place."""
    assert lib.blazeCacheAttention(C.byref(cache()), C.byref(attention(q=P, out=P)), None) == INVALID
