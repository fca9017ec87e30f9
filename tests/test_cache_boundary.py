"""Argument checks of the paged-cache entry points: every refusal comes before anything is launched, so they run on a
machine without a GPU.  Pointers are made-up numbers; no call here is a valid one."""
import ctypes as C

import pytest

from ops_tensor_b200 import native

OK, INVALID, UNSUPPORTED, NO_SPACE = (native.STATUS_SUCCESS, native.STATUS_INVALID_VALUE, native.STATUS_NOT_SUPPORTED,
                                      native.STATUS_INSUFFICIENT_WORKSPACE)
P = 1 << 20                                                # a pointer that nobody follows


@pytest.fixture(scope="module")
def lib(built_library):
    return native.lib()


def filled(struct, **kw):
    s = struct()
    s.struct_size = C.sizeof(struct)
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def cache(**kw):
    d = dict(elem=0, num_blocks=8, block_size=16, kv_heads=2, head_dim=64, k=P, v=P, block_stride=2048, head_stride=1024,
             token_stride=64, k_scale=P, v_scale=P, scale_stride=2)
    d.update(kw)
    return filled(native.KvCacheDesc, **d)


def assign(**kw):
    d = dict(requests=4, block_size=16, max_blocks=8, max_tokens=10, cached_len=P, new_len=P, block_table=P, table_stride=8,
             free_blocks=P, free_capacity=8, free_count=P, free_count_out=P, row_offsets=P, kv_len=P, slots=P)
    d.update(kw)
    return filled(native.CacheAssignArgs, **d)


def store(**kw):
    d = dict(tokens=3, in_type=native.OUT_BF16, k=P, v=P, k_token_stride=128, k_head_stride=64, v_token_stride=128,
             v_head_stride=64, slots=P)
    d.update(kw)
    return filled(native.CacheStoreArgs, **d)


def attention(**kw):
    d = dict(requests=2, tokens=3, heads=4, q_type=native.OUT_BF16, q=P, q_token_stride=256, q_head_stride=64, out=P,
             out_token_stride=256, out_head_stride=64, row_offsets=P, kv_len=P, block_table=P, table_stride=8, max_blocks=8,
             max_q=2, max_kv=128, scale=0.125, causal=1, workspace=P, workspace_bytes=1 << 40)
    d.update(kw)
    return filled(native.CacheAttentionArgs, **d)


CACHE_FAULTS = [
    (dict(struct_size=8), INVALID), (dict(num_blocks=0), INVALID), (dict(kv_heads=0), INVALID), (dict(k=None), INVALID),
    (dict(v=None), INVALID), (dict(k_scale=None), INVALID), (dict(v_scale=None), INVALID), (dict(elem=1), UNSUPPORTED),
    (dict(elem=2), UNSUPPORTED), (dict(block_size=8), UNSUPPORTED), (dict(block_size=48), UNSUPPORTED),
    (dict(block_size=256), UNSUPPORTED), (dict(head_dim=80), UNSUPPORTED), (dict(head_dim=256), UNSUPPORTED),
    (dict(k=P + 8), UNSUPPORTED), (dict(v=P + 1), UNSUPPORTED), (dict(k_scale=P + 2), UNSUPPORTED),
    (dict(token_stride=48), INVALID), (dict(token_stride=72), UNSUPPORTED), (dict(head_stride=0), INVALID),
    (dict(head_stride=1032), UNSUPPORTED), (dict(block_stride=-2048), INVALID), (dict(block_stride=2056), UNSUPPORTED),
    (dict(block_stride=1 << 40), UNSUPPORTED), (dict(scale_stride=1), INVALID),
]


@pytest.mark.parametrize("fault,status", CACHE_FAULTS)
def test_cache_descriptor(lib, fault, status):
    assert lib.blazeCacheStore(C.byref(cache(**fault)), C.byref(store()), None) == status
    n = C.c_size_t(5)
    assert lib.blazeCacheAttentionWorkspaceSize(C.byref(cache(**fault)), C.byref(attention()), C.byref(n)) == status
    assert n.value == 5
    assert lib.blazeCacheAttention(C.byref(cache(**fault)), C.byref(attention()), None) == status


@pytest.mark.parametrize("fault,status", [
    (dict(struct_size=100), INVALID), (dict(requests=-1), INVALID), (dict(max_blocks=-1), INVALID), (dict(max_tokens=-1), INVALID),
    (dict(free_capacity=-1), INVALID), (dict(table_stride=7), INVALID), (dict(block_size=24), UNSUPPORTED),
    (dict(block_size=0), UNSUPPORTED), (dict(requests=8193), UNSUPPORTED),
    (dict(max_blocks=1 << 28, table_stride=1 << 28), UNSUPPORTED),
    (dict(requests=8192, max_blocks=1 << 20, table_stride=1 << 20), UNSUPPORTED),
    (dict(cached_len=None), INVALID), (dict(new_len=None), INVALID), (dict(block_table=None), INVALID),
    (dict(free_blocks=None), INVALID), (dict(free_count=None), INVALID), (dict(free_count_out=None), INVALID),
    (dict(row_offsets=None), INVALID), (dict(kv_len=None), INVALID), (dict(slots=None), INVALID), (dict(slots=P + 4), INVALID),
    (dict(positions=P + 1), INVALID), (dict(denied=P + 2), INVALID), (dict(cached_len=P + 2), INVALID)])
def test_assign_arguments(lib, fault, status):
    assert lib.blazeCacheAssign(C.byref(assign(**fault)), None) == status


@pytest.mark.parametrize("fault,status", [
    (dict(struct_size=0), INVALID), (dict(tokens=-1), INVALID), (dict(tokens=0), OK), (dict(in_type=native.OUT_F32), UNSUPPORTED),
    (dict(k=None), INVALID), (dict(v=None), INVALID), (dict(slots=None), INVALID), (dict(slots=P + 4), INVALID),
    (dict(k=P + 8), UNSUPPORTED), (dict(v=P + 2), UNSUPPORTED), (dict(k_token_stride=130), UNSUPPORTED),
    (dict(v_token_stride=4), UNSUPPORTED), (dict(k_head_stride=65), UNSUPPORTED), (dict(v_head_stride=2), UNSUPPORTED)])
def test_store_arguments(lib, fault, status):
    assert lib.blazeCacheStore(C.byref(cache()), C.byref(store(**fault)), None) == status


@pytest.mark.parametrize("fault,status", [
    (dict(struct_size=1), INVALID), (dict(requests=-1), INVALID), (dict(tokens=-1), INVALID), (dict(heads=0), INVALID),
    (dict(heads=3), INVALID), (dict(max_q=-1), INVALID), (dict(min_q=-1), INVALID), (dict(max_kv=-1), INVALID),
    (dict(max_kv=129), INVALID), (dict(table_stride=7), INVALID), (dict(window=-1), INVALID), (dict(causal=2), INVALID),
    (dict(sm_limit=-1), INVALID), (dict(scale=float("inf")), INVALID), (dict(scale=float("nan")), INVALID),
    (dict(requests=8193), UNSUPPORTED), (dict(q_type=native.OUT_F32), UNSUPPORTED), (dict(max_q=1 << 30), UNSUPPORTED),
    (dict(max_kv=(1 << 30) + 1, max_blocks=1 << 27, table_stride=1 << 27), UNSUPPORTED),
    (dict(requests=8000, max_kv=1 << 29, max_blocks=1 << 25, table_stride=1 << 25), UNSUPPORTED)])
def test_attention_bounds(lib, fault, status):
    n = C.c_size_t(5)
    assert lib.blazeCacheAttentionWorkspaceSize(C.byref(cache()), C.byref(attention(**fault)), C.byref(n)) == status
    assert lib.blazeCacheAttention(C.byref(cache()), C.byref(attention(**fault)), None) == status


@pytest.mark.parametrize("fault,status", [
    (dict(requests=0), OK), (dict(tokens=0), OK), (dict(max_q=0), OK),
    (dict(q=None), INVALID), (dict(out=None), INVALID), (dict(row_offsets=None), INVALID), (dict(kv_len=None), INVALID),
    (dict(block_table=None), INVALID), (dict(q=P + 2), UNSUPPORTED), (dict(out=P + 8), UNSUPPORTED), (dict(lse=P + 1), UNSUPPORTED),
    (dict(kv_len=P + 1), UNSUPPORTED), (dict(q_token_stride=258), UNSUPPORTED), (dict(out_head_stride=60), UNSUPPORTED),
    (dict(workspace=None), NO_SPACE), (dict(workspace_bytes=100), NO_SPACE), (dict(workspace=P + 64), INVALID)])
def test_attention_arguments(lib, fault, status):
    assert lib.blazeCacheAttention(C.byref(cache()), C.byref(attention(**fault)), None) == status


def test_workspace_follows_the_bounds_and_the_share_of_sms(lib):
    def need(**kw):
        n = C.c_size_t(0)
        assert lib.blazeCacheAttentionWorkspaceSize(C.byref(cache()), C.byref(attention(**kw)), C.byref(n)) == OK
        return n.value
    assert need() > 0 and need(sm_limit=10) < need()
    # larger bounds never need less
    wide = dict(max_blocks=4096, table_stride=4096)
    for fixed in (dict(), dict(tokens=400, max_q=300), dict(tokens=30000, max_q=9000, heads=16)):
        for name, steps in (("tokens", (1, 30, 3000, 100000)), ("requests", (1, 200, 3000, 8192)),
                            ("max_q", (1, 4, 5, 300, 9000)), ("max_kv", (0, 64, 3000, 65536))):
            sizes = [need(**{**wide, **fixed, name: v}) for v in steps]
            assert sizes == sorted(sizes) and sizes[0] > 0, (fixed, name, sizes)
    assert lib.blazeCacheAttentionWorkspaceSize(C.byref(cache()), C.byref(attention()), None) == INVALID


def test_python_wrappers_refuse_host_tensors():
    torch = pytest.importorskip("torch")
    c = torch.zeros((4, 2, 16, 64), dtype=torch.uint8)
    s = torch.ones((4, 2))
    with pytest.raises(ValueError):
        native.PagedCache(c, c, s, s)
    z = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError):
        native.cache_assign(z, z, z.view(1, 4), z, z, block_size=16, row_offsets=z, kv_len=z, slots=z)
