"""ctypes binding of libops_tensor_b200.so.

Loading fails loudly when the library has not been built: there is no CPU or PyTorch fallback for any operation of
this package.  torch tensors are used only as owners of device memory; every computation happens inside the shared
library.
"""
from __future__ import annotations

import ctypes as C
import struct
from pathlib import Path

_LIB_PATH = Path(__file__).resolve().parent / "libops_tensor_b200.so"

STATUS_SUCCESS = 0
STATUS_NOT_INITIALIZED = 1
STATUS_ALLOC_FAILED = 3
STATUS_INVALID_VALUE = 7
STATUS_ARCH_MISMATCH = 8
STATUS_EXECUTION_FAILED = 13
STATUS_INTERNAL_ERROR = 14
STATUS_NOT_SUPPORTED = 15
STATUS_INSUFFICIENT_WORKSPACE = 19

ELEM_E4M3, ELEM_E2M1, ELEM_E5M2 = 0, 1, 2
ACT_IDENTITY, ACT_RELU, ACT_GELU_TANH, ACT_SILU, ACT_SIGMOID, ACT_TANH = 0, 1, 2, 3, 4, 5
SCHED_AUTO, SCHED_DATA_PARALLEL, SCHED_STREAM_K = 0, 1, 2
OUT_BF16, OUT_F16, OUT_F32, OUT_MX_E4M3, OUT_FP8_128 = 0, 1, 2, 3, 4


def out_type_of(tensor) -> int:
    """blazeOutType_t of a torch output tensor (bf16, half or float32)."""
    import torch
    return {torch.bfloat16: OUT_BF16, torch.float16: OUT_F16, torch.float32: OUT_F32,
            torch.uint8: OUT_MX_E4M3}[tensor.dtype]


class MxGemmArgs(C.Structure):
    _fields_ = [
        ("struct_size", C.c_size_t),
        ("M", C.c_int32), ("N", C.c_int32), ("K", C.c_int32),
        ("b_elem", C.c_int32),
        ("A", C.c_void_p), ("lda", C.c_int64),
        ("B", C.c_void_p), ("ldb", C.c_int64),
        ("scaleA", C.c_void_p), ("scaleB", C.c_void_p),
        ("bias", C.c_void_p),
        ("residual", C.c_void_p), ("ldr", C.c_int64),
        ("D", C.c_void_p), ("ldd", C.c_int64),
        ("activation", C.c_int32),
        ("tile_n", C.c_int32),
        ("reuse_b_prepass", C.c_int32),
        ("sm_limit", C.c_int32),
        ("cta_pair", C.c_int32),
        ("a_elem", C.c_int32),
        ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t),
        ("d_type", C.c_int32), ("b_layout", C.c_int32),
        ("scaleD", C.c_void_p),
        ("sched", C.c_int32), ("n_peers", C.c_int32),
        ("peerD", C.c_void_p * 7),
    ]


class BatchDims(C.Structure):
    """blazeBatchDims: batch extents of D, A and B (outermost first, 1 = unused or broadcast)."""
    _fields_ = [("c", C.c_int32 * 4), ("a", C.c_int32 * 4), ("b", C.c_int32 * 4), ("bias_per_batch", C.c_int32),
                ("reserved", C.c_int32)]


class Fp8GemmArgs(C.Structure):
    _fields_ = [
        ("struct_size", C.c_size_t),
        ("M", C.c_int32), ("N", C.c_int32), ("K", C.c_int32),
        ("groups", C.c_int32),
        ("group_rows", C.c_void_p),
        ("A", C.c_void_p), ("lda", C.c_int64),
        ("B", C.c_void_p), ("ldb", C.c_int64),
        ("scaleA", C.c_void_p), ("scaleB", C.c_void_p),
        ("bias", C.c_void_p),
        ("residual", C.c_void_p), ("ldr", C.c_int64),
        ("D", C.c_void_p), ("ldd", C.c_int64),
        ("activation", C.c_int32),
        ("sched", C.c_int32),
        ("sm_limit", C.c_int32),
        ("d_type", C.c_int32),
        ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t),
        ("scaleD", C.c_void_p),
        ("n_peers", C.c_int32), ("b_is_static", C.c_int32),
        ("peerD", C.c_void_p * 7),
    ]


class DenseGemmArgs(C.Structure):
    """blazeDenseGemmArgs: INT8 (A8W8) and fp16 / bf16 GEMMs without block scales."""
    _fields_ = [
        ("struct_size", C.c_size_t),
        ("M", C.c_int32), ("N", C.c_int32), ("K", C.c_int32),
        ("kind", C.c_int32),
        ("A", C.c_void_p), ("lda", C.c_int64),
        ("B", C.c_void_p), ("ldb", C.c_int64),
        ("scale_mode", C.c_int32), ("activation", C.c_int32),
        ("scaleA", C.c_void_p), ("scaleB", C.c_void_p), ("scaleN", C.c_void_p),
        ("bias", C.c_void_p),
        ("residual", C.c_void_p), ("ldr", C.c_int64),
        ("D", C.c_void_p), ("ldd", C.c_int64),
        ("d_type", C.c_int32), ("sm_limit", C.c_int32),
    ]


DENSE_S8, DENSE_F16, DENSE_BF16 = 0, 1, 2
DENSE_SCALE_NONE, DENSE_SCALE_PER_TENSOR, DENSE_SCALE_PER_CHANNEL = 0, 1, 2
OUT_S32 = 5


class KvCacheDesc(C.Structure):
    """blazeKvCache: the paged 8-bit key / value cache."""
    _fields_ = [
        ("struct_size", C.c_size_t),
        ("elem", C.c_int32),
        ("num_blocks", C.c_int32), ("block_size", C.c_int32), ("kv_heads", C.c_int32), ("head_dim", C.c_int32),
        ("reserved", C.c_int32),
        ("k", C.c_void_p), ("v", C.c_void_p),
        ("block_stride", C.c_int64), ("head_stride", C.c_int64), ("token_stride", C.c_int64),
        ("k_scale", C.c_void_p), ("v_scale", C.c_void_p),
        ("scale_stride", C.c_int64),
    ]


class CacheAssignArgs(C.Structure):
    _fields_ = [
        ("struct_size", C.c_size_t),
        ("requests", C.c_int32), ("block_size", C.c_int32), ("max_blocks", C.c_int32), ("max_tokens", C.c_int32),
        ("cached_len", C.c_void_p), ("new_len", C.c_void_p),
        ("block_table", C.c_void_p), ("table_stride", C.c_int64),
        ("free_blocks", C.c_void_p), ("free_capacity", C.c_int32), ("reserved", C.c_int32),
        ("free_count", C.c_void_p), ("free_count_out", C.c_void_p),
        ("row_offsets", C.c_void_p), ("kv_len", C.c_void_p),
        ("slots", C.c_void_p), ("positions", C.c_void_p), ("denied", C.c_void_p),
    ]


class CacheStoreArgs(C.Structure):
    _fields_ = [
        ("struct_size", C.c_size_t),
        ("tokens", C.c_int32), ("in_type", C.c_int32),
        ("k", C.c_void_p), ("v", C.c_void_p),
        ("k_token_stride", C.c_int64), ("k_head_stride", C.c_int64),
        ("v_token_stride", C.c_int64), ("v_head_stride", C.c_int64),
        ("slots", C.c_void_p),
    ]


class CacheAttentionArgs(C.Structure):
    _fields_ = [
        ("struct_size", C.c_size_t),
        ("requests", C.c_int32), ("tokens", C.c_int32), ("heads", C.c_int32), ("q_type", C.c_int32),
        ("q", C.c_void_p), ("q_token_stride", C.c_int64), ("q_head_stride", C.c_int64),
        ("out", C.c_void_p), ("out_token_stride", C.c_int64), ("out_head_stride", C.c_int64),
        ("lse", C.c_void_p),
        ("row_offsets", C.c_void_p), ("kv_len", C.c_void_p),
        ("block_table", C.c_void_p), ("table_stride", C.c_int64),
        ("max_blocks", C.c_int32),
        ("max_q", C.c_int32), ("min_q", C.c_int32), ("max_kv", C.c_int32),
        ("scale", C.c_float), ("causal", C.c_int32), ("window", C.c_int32), ("sm_limit", C.c_int32),
        ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t),
    ]


class BlazeError(RuntimeError):
    def __init__(self, status: int, where: str):
        self.status = status
        super().__init__(f"{where} failed with acltensorStatus_t {status}")


_lib = None


def lib() -> C.CDLL:
    """The loaded shared library; raises if it is missing (build it with `python -m ops_tensor_b200.build`)."""
    global _lib
    if _lib is None:
        if not _LIB_PATH.exists():
            raise RuntimeError(
                f"{_LIB_PATH} is missing: the CUDA library has not been built. Run `python -m ops_tensor_b200.build`. "
                "There is no fallback path.")
        _lib = C.CDLL(str(_LIB_PATH))
        _declare(_lib)
    return _lib


def _declare(l: C.CDLL) -> None:
    l.blazeMxGemmWorkspaceSize.argtypes = [C.POINTER(MxGemmArgs), C.POINTER(C.c_size_t)]
    l.blazeMxGemm.argtypes = [C.POINTER(MxGemmArgs), C.c_void_p]
    l.blazeMxGemmNoAlloc.argtypes = [C.POINTER(MxGemmArgs), C.c_void_p, C.c_void_p]
    l.blazeMxGemmNoAlloc.restype = C.c_int
    l.blazeMxGemmBatchedWorkspaceSize.argtypes = [C.POINTER(MxGemmArgs), C.POINTER(BatchDims), C.POINTER(C.c_size_t)]
    l.blazeMxGemmBatchedWorkspaceSize.restype = C.c_int
    l.blazeMxGemmBatched.argtypes = [C.POINTER(MxGemmArgs), C.POINTER(BatchDims), C.c_void_p]
    l.blazeMxGemmBatched.restype = C.c_int
    l.blazeDenseGemm.argtypes = [C.POINTER(DenseGemmArgs), C.c_void_p]
    l.blazeDenseGemm.restype = C.c_int
    l.blazeFp8GemmWorkspaceSize.argtypes = [C.POINTER(Fp8GemmArgs), C.POINTER(C.c_size_t)]
    l.blazeFp8Gemm.argtypes = [C.POINTER(Fp8GemmArgs), C.c_void_p]
    l.blazeQuantizeMx.argtypes = [C.c_void_p, C.c_int64, C.c_int32, C.c_int32, C.c_int32, C.c_void_p, C.c_int64,
                                  C.c_void_p, C.c_void_p]
    l.blazeQuantizeFp8RowGroups.argtypes = [C.c_void_p, C.c_int64, C.c_int32, C.c_int32, C.c_void_p, C.c_int64,
                                            C.c_void_p, C.c_void_p]
    l.blazeQuantizeFp8Blocks.argtypes = [C.c_void_p, C.c_int64, C.c_int32, C.c_int32, C.c_void_p, C.c_int64,
                                         C.c_void_p, C.c_void_p]
    # (void pointers: a byref() of the structure or its bytes)
    l.blazeCacheAssign.argtypes = [C.c_void_p, C.c_void_p]
    l.blazeCacheStore.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p]
    l.blazeCacheAttentionWorkspaceSize.argtypes = [C.c_void_p, C.c_void_p, C.POINTER(C.c_size_t)]
    l.blazeCacheAttention.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p]
    l.blazeAddF32.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p, C.c_int64, C.c_void_p]
    l.blazeSelfTestWaitTimeout.argtypes = [C.c_int64, C.c_void_p]
    l.blazeSelfTestWaitTimeout.restype = C.c_int
    l.blazeDeviceStatus.argtypes = [C.POINTER(C.c_int32), C.c_int32]
    l.blazeDeviceInfo.argtypes = [C.POINTER(C.c_int32), C.POINTER(C.c_int32), C.POINTER(C.c_int32)]
    for name in ("blazeMxGemmWorkspaceSize", "blazeMxGemm", "blazeFp8GemmWorkspaceSize", "blazeFp8Gemm",
                 "blazeQuantizeMx", "blazeQuantizeFp8RowGroups", "blazeQuantizeFp8Blocks", "blazeAddF32",
                 "blazeDeviceStatus", "blazeDeviceInfo", "blazeCacheAssign", "blazeCacheStore",
                 "blazeCacheAttentionWorkspaceSize", "blazeCacheAttention"):
        getattr(l, name).restype = C.c_int


def check(status: int, where: str) -> None:
    if status != STATUS_SUCCESS:
        raise BlazeError(status, where)


def _ptr(t):
    return None if t is None else C.c_void_p(t.data_ptr())


def _stream():
    import torch
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def device_status(reset: bool = True) -> int:
    v = C.c_int32(0)
    check(lib().blazeDeviceStatus(C.byref(v), 1 if reset else 0), "blazeDeviceStatus")
    return v.value


def device_info():
    a, b, c = C.c_int32(), C.c_int32(), C.c_int32()
    check(lib().blazeDeviceInfo(C.byref(a), C.byref(b), C.byref(c)), "blazeDeviceInfo")
    return a.value, b.value, c.value


# ------------------------------------------------------------------------------------------------ quantisers

def mx_scale_cols(K: int) -> int:
    return -(-K // 64) * 2


def quantize_mx(x, elem: int = ELEM_E4M3):
    """x: float32 CUDA tensor [rows, K] -> (codes uint8 [rows, K] or [rows, K/2], scales uint8 [rows, ceil(K/64)*2])."""
    import torch
    assert x.is_cuda and x.dtype == torch.float32 and x.dim() == 2 and x.stride(1) == 1
    rows, K = x.shape
    codes = torch.empty((rows, K // 2 if elem == ELEM_E2M1 else K), dtype=torch.uint8, device=x.device)
    scales = torch.empty((rows, mx_scale_cols(K)), dtype=torch.uint8, device=x.device)
    check(lib().blazeQuantizeMx(_ptr(x), x.stride(0), rows, K, elem, _ptr(codes), codes.stride(0), _ptr(scales),
                                _stream()), "blazeQuantizeMx")
    return codes, scales


def quantize_fp8_row_groups(x):
    import torch
    assert x.is_cuda and x.dtype == torch.float32 and x.dim() == 2 and x.stride(1) == 1
    rows, K = x.shape
    codes = torch.empty((rows, K), dtype=torch.uint8, device=x.device)
    scales = torch.empty((rows, -(-K // 128)), dtype=torch.float32, device=x.device)
    check(lib().blazeQuantizeFp8RowGroups(_ptr(x), x.stride(0), rows, K, _ptr(codes), codes.stride(0), _ptr(scales),
                                          _stream()), "blazeQuantizeFp8RowGroups")
    return codes, scales


def quantize_fp8_blocks(w):
    import torch
    assert w.is_cuda and w.dtype == torch.float32 and w.dim() == 2 and w.stride(1) == 1
    N, K = w.shape
    codes = torch.empty((N, K), dtype=torch.uint8, device=w.device)
    scales = torch.empty((-(-K // 128), -(-N // 128)), dtype=torch.float32, device=w.device)
    check(lib().blazeQuantizeFp8Blocks(_ptr(w), w.stride(0), N, K, _ptr(codes), codes.stride(0), _ptr(scales),
                                       _stream()), "blazeQuantizeFp8Blocks")
    return codes, scales


# ------------------------------------------------------------------------------------------------ GEMMs

def mx_gemm_args(a, sa, b, sb, out, *, b_elem=ELEM_E4M3, bias=None, residual=None, activation=ACT_IDENTITY,
                 tile_n=0, reuse_b_prepass=False, sm_limit=0, cta_pair=0, workspace=None, a_elem=ELEM_E4M3,
                 scale_out=None, b_n_major=False, sched=SCHED_AUTO, peer_outs=None) -> MxGemmArgs:
    M, K = a.shape
    if a_elem == ELEM_E2M1:
        K *= 2                       # two codes per byte
    N = b.shape[1] if b_n_major else b.shape[0]
    args = MxGemmArgs()
    args.struct_size = C.sizeof(MxGemmArgs)
    args.M, args.N, args.K = M, N, K
    args.b_elem = b_elem
    args.A, args.lda = a.data_ptr(), a.stride(0)
    args.B, args.ldb = b.data_ptr(), b.stride(0)
    args.scaleA, args.scaleB = sa.data_ptr(), sb.data_ptr()
    args.bias = bias.data_ptr() if bias is not None else None
    args.residual = residual.data_ptr() if residual is not None else None
    args.ldr = residual.stride(0) if residual is not None else 0
    args.D, args.ldd = out.data_ptr(), out.stride(0)
    args.d_type = out_type_of(out)
    args.activation = activation
    args.tile_n = tile_n
    args.reuse_b_prepass = 1 if reuse_b_prepass else 0
    args.sm_limit = sm_limit
    args.cta_pair = cta_pair
    args.a_elem = a_elem
    args.scaleD = scale_out.data_ptr() if scale_out is not None else None
    args.b_layout = 1 if b_n_major else 0
    args.sched = sched
    if peer_outs:
        # further copies of `out` (same shape, pitch and dtype) that the epilogue stores every tile to as well
        if len(peer_outs) > 7 or any(t.shape != out.shape or t.stride(0) != out.stride(0) or t.dtype != out.dtype
                                     for t in peer_outs):
            raise ValueError("peer outputs must match the output's shape, pitch and dtype (at most 7)")
        args.n_peers = len(peer_outs)
        for i, t in enumerate(peer_outs):
            args.peerD[i] = t.data_ptr()
    if workspace is not None:
        args.workspace, args.workspace_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    return args


def mx_gemm_workspace_bytes(args: MxGemmArgs) -> int:
    n = C.c_size_t(0)
    check(lib().blazeMxGemmWorkspaceSize(C.byref(args), C.byref(n)), "blazeMxGemmWorkspaceSize")
    return n.value


def mx_gemm(a, sa, b, sb, *, out=None, workspace=None, **kw):
    """D = act(A x B^T + bias) + residual for MX operands; allocates `out` / `workspace` when not given."""
    import torch
    M = a.shape[0]
    N = b.shape[1] if kw.get("b_n_major") else b.shape[0]
    if out is None:
        out = torch.empty((M, N), dtype=torch.bfloat16, device=a.device)
    args = mx_gemm_args(a, sa, b, sb, out, workspace=workspace, **kw)
    if workspace is None:
        need = mx_gemm_workspace_bytes(args)
        workspace = torch.empty(max(need, 256), dtype=torch.uint8, device=a.device)
        args.workspace, args.workspace_bytes = workspace.data_ptr(), workspace.numel()
    check(lib().blazeMxGemm(C.byref(args), _stream()), "blazeMxGemm")
    return out


def fp8_gemm_args(a, sa, b, sb, out, *, group_rows=None, bias=None, residual=None, activation=ACT_IDENTITY,
                  sched=SCHED_AUTO, sm_limit=0, workspace=None, scale_out=None, peer_outs=None,
                  b_is_static=False) -> Fp8GemmArgs:
    M, K = a.shape
    if b.dim() == 3:
        G, N, _ = b.shape
        ldb = b.stride(1)
    else:
        G, (N, _) = 0, b.shape
        ldb = b.stride(0)
    args = Fp8GemmArgs()
    args.struct_size = C.sizeof(Fp8GemmArgs)
    args.M, args.N, args.K = M, N, K
    args.groups = G
    args.group_rows = group_rows.data_ptr() if group_rows is not None else None
    args.A, args.lda = a.data_ptr(), a.stride(0)
    args.B, args.ldb = b.data_ptr(), ldb
    args.scaleA, args.scaleB = sa.data_ptr(), sb.data_ptr()
    args.bias = bias.data_ptr() if bias is not None else None
    args.residual = residual.data_ptr() if residual is not None else None
    args.ldr = residual.stride(0) if residual is not None else 0
    args.D, args.ldd = out.data_ptr(), out.stride(0)
    args.d_type = OUT_FP8_128 if scale_out is not None else out_type_of(out)
    args.scaleD = scale_out.data_ptr() if scale_out is not None else None
    args.activation = activation
    args.sched = sched
    args.sm_limit = sm_limit
    args.b_is_static = 1 if b_is_static else 0
    if peer_outs:
        if len(peer_outs) > 7 or any(t.shape != out.shape or t.stride(0) != out.stride(0) or t.dtype != out.dtype
                                     for t in peer_outs):
            raise ValueError("peer outputs must match the output's shape, pitch and dtype (at most 7)")
        args.n_peers = len(peer_outs)
        for i, t in enumerate(peer_outs):
            args.peerD[i] = t.data_ptr()
    if workspace is not None:
        args.workspace, args.workspace_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    return args


def fp8_gemm_workspace_bytes(args: Fp8GemmArgs) -> int:
    n = C.c_size_t(0)
    check(lib().blazeFp8GemmWorkspaceSize(C.byref(args), C.byref(n)), "blazeFp8GemmWorkspaceSize")
    return n.value


def fp8_gemm(a, sa, b, sb, *, out=None, workspace=None, **kw):
    import torch
    M = a.shape[0]
    N = b.shape[-2]
    if out is None:
        out = torch.empty((M, N), dtype=torch.bfloat16, device=a.device)
    args = fp8_gemm_args(a, sa, b, sb, out, workspace=workspace, **kw)
    if workspace is None:
        need = fp8_gemm_workspace_bytes(args)
        if need:
            workspace = torch.empty(need, dtype=torch.uint8, device=a.device)
            args.workspace, args.workspace_bytes = workspace.data_ptr(), workspace.numel()
    check(lib().blazeFp8Gemm(C.byref(args), _stream()), "blazeFp8Gemm")
    return out


def dense_gemm(a, b, *, out=None, out_dtype=None, scale_a=None, scale_b=None, scale_n=None, bias=None, residual=None,
               activation=ACT_IDENTITY, sm_limit=0):
    """D = act(A x B^T + bias) + residual for int8, half or bf16 operands (A [M, K], B [N, K], K contiguous).
    int8: `scale_a` and `scale_b` (one float32 each) or `scale_n` (uint64 per column) de-quantise on store, `bias` is
    int32; with no scale and an int32 `out` the raw sums are stored."""
    import torch
    M, K = a.shape
    N = b.shape[0]
    kind = {torch.int8: DENSE_S8, torch.float16: DENSE_F16, torch.bfloat16: DENSE_BF16}[a.dtype]
    if out is None:
        out = torch.empty((M, N), dtype=out_dtype or (torch.float16 if kind != DENSE_BF16 else torch.bfloat16),
                          device=a.device)
    args = DenseGemmArgs()
    args.struct_size = C.sizeof(DenseGemmArgs)
    args.M, args.N, args.K = M, N, K
    args.kind = kind
    args.A, args.lda = a.data_ptr(), a.stride(0)
    args.B, args.ldb = b.data_ptr(), b.stride(0)
    args.scale_mode = DENSE_SCALE_PER_CHANNEL if scale_n is not None else (
        DENSE_SCALE_PER_TENSOR if scale_a is not None else DENSE_SCALE_NONE)
    args.activation = activation
    args.scaleA = scale_a.data_ptr() if scale_a is not None else None
    args.scaleB = scale_b.data_ptr() if scale_b is not None else None
    args.scaleN = scale_n.data_ptr() if scale_n is not None else None
    args.bias = bias.data_ptr() if bias is not None else None
    args.residual = residual.data_ptr() if residual is not None else None
    args.ldr = residual.stride(0) if residual is not None else 0
    args.D, args.ldd = out.data_ptr(), out.stride(0)
    args.d_type = OUT_S32 if out.dtype == torch.int32 else out_type_of(out)
    args.sm_limit = sm_limit
    check(lib().blazeDenseGemm(C.byref(args), _stream()), "blazeDenseGemm")
    return out


MAX_PEERS = 7          # BLAZE_MAX_PEERS


class PeerSignalArgs(C.Structure):
    _fields_ = [
        ("struct_size", C.c_size_t),
        ("my_rank", C.c_int32),
        ("n_peers", C.c_int32),
        ("peer_ranks", C.c_int32 * MAX_PEERS),
        ("local_flags", C.c_void_p),
        ("peer_flags", C.c_void_p * MAX_PEERS),
        ("value", C.c_uint64),
        ("limit_cycles", C.c_int64),
    ]


def peer_signal(local_flags, peer_flags, my_rank: int, peer_ranks, value: int, limit_cycles: int = 0) -> None:
    """Closing signal of a fused gather (`blazePeerSignal`): stores `value` into slot `my_rank` of every peer's flag
    array and waits, bounded, until this GPU's own array shows `value` from every peer.  `local_flags`: this rank's
    int64 tensor [ranks]; `peer_flags`: the peers' arrays as mapped into this process, in the order of `peer_ranks`."""
    args = PeerSignalArgs()
    args.struct_size = C.sizeof(PeerSignalArgs)
    args.my_rank = my_rank
    args.n_peers = len(peer_flags)
    for q, (t, r) in enumerate(zip(peer_flags, peer_ranks)):
        args.peer_flags[q] = t.data_ptr()
        args.peer_ranks[q] = r
    args.local_flags = local_flags.data_ptr()
    args.value = value
    args.limit_cycles = limit_cycles
    l = lib()
    l.blazePeerSignal.restype = C.c_int
    check(l.blazePeerSignal(C.byref(args), _stream()), "blazePeerSignal")


# ------------------------------------------------------------------------------------------------ paged 8-bit cache

torch = None          # imported when the first of these calls is made


def _import_torch():
    global torch
    import torch


# The arguments' layouts, for the calls of every step: packing them costs a fifth of filling the ctypes structures in.
_ASSIGN = struct.Struct("@Niiii PP Pq Pii PP PP PPP")
_STORE = struct.Struct("@Nii PP qqqq P")
_ATTENTION = struct.Struct("@Niiii Pqq Pqq P PP Pq iiii fiii PN")


def _launch(name, device: int, *args) -> None:
    """Calls a C entry point on the current stream of the GPU that its tensors live on, with that GPU current."""
    fn = getattr(lib(), name)
    if device == torch.cuda.current_device():
        status = fn(*args, torch._C._cuda_getCurrentRawStream(device))
    else:
        with torch.cuda.device(device):
            status = fn(*args, torch._C._cuda_getCurrentRawStream(device))
    if status != STATUS_SUCCESS:
        raise BlazeError(status, name)


def _same_device(first, *others) -> int:
    """The GPU of all these tensors (None among them is left out)."""
    device = first.get_device()
    if device < 0:
        raise ValueError("the cache operators take CUDA tensors")
    for t in others:
        if t is not None and t.get_device() != device:
            raise ValueError(f"a tensor is on {t.device}, the others on {first.device}")
    return device


def _vector(t, name, dtype, at_least) -> int:
    """The address of a contiguous vector."""
    if t.dtype is not dtype or t.dim() != 1 or t.numel() < at_least or not t.is_contiguous():
        raise ValueError(f"{name}: a contiguous {dtype} vector of at least {at_least} elements is wanted")
    return t.data_ptr()


def _table(t):
    """(rows, columns, pitch) of a block table."""
    if t.dtype is not torch.int32 or t.dim() != 2:
        raise ValueError("block_table: an int32 [requests, blocks] tensor is wanted")
    rows, columns = t.shape
    if rows == 0 or columns == 0 or t.is_contiguous():
        return rows, columns, columns
    if columns > 1 and t.stride(1) != 1:
        raise ValueError("block_table: rows of contiguous elements are wanted")
    return rows, columns, t.stride(0) if rows > 1 else columns


class PagedCache:
    """A paged key / value cache in E4M3 with one float32 scale per (block, kv head): `k`, `v` [blocks, kv heads, block
    size, head size] of uint8 or float8_e4m3fn with equal strides (any order of the first three dimensions in memory;
    `k.permute(0, 2, 1, 3)` of a [blocks, tokens, heads, size] tensor is one), `k_scale`, `v_scale` float32
    [blocks, kv heads].  Keeps the tensors; `desc` is the C ABI's view of them."""

    def __init__(self, k, v, k_scale, v_scale):
        if torch is None:
            _import_torch()
        _same_device(k, v, k_scale, v_scale)
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.dtype not in (torch.uint8, torch.float8_e4m3fn):
            raise ValueError("k and v: two [blocks, heads, block size, head size] tensors of uint8 or float8_e4m3fn")
        n, h, bs, d = k.shape
        strides = [s for s, size in zip(k.stride(), k.shape) if size > 1]
        if strides != [s for s, size in zip(v.stride(), v.shape) if size > 1] or k.stride(3) != 1 or v.stride(3) != 1:
            raise ValueError("k and v must have the same strides, the last dimension contiguous")
        for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
            if t.dtype != torch.float32 or tuple(t.shape) != (n, h) or (h > 1 and t.stride(1) != 1):
                raise ValueError(f"{name}: a float32 [blocks, heads] tensor with contiguous rows is wanted")
        if n > 1 and k_scale.stride(0) != v_scale.stride(0):
            raise ValueError("k_scale and v_scale must have the same row stride")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.device = k.device
        self.num_blocks, self.kv_heads, self.block_size, self.head_dim = n, h, bs, d
        c = self.desc = KvCacheDesc()
        c.struct_size = C.sizeof(KvCacheDesc)
        c.elem = ELEM_E4M3
        c.num_blocks, c.kv_heads, c.block_size, c.head_dim = n, h, bs, d
        c.k, c.v = k.data_ptr(), v.data_ptr()
        c.block_stride, c.head_stride, c.token_stride = k.stride()[:3]
        c.k_scale, c.v_scale = k_scale.data_ptr(), v_scale.data_ptr()
        c.scale_stride = k_scale.stride(0) if n > 1 else h
        self._desc_at = C.addressof(c)

    @classmethod
    def empty(cls, num_blocks, kv_heads, block_size, head_dim, device="cuda"):
        """A new cache: codes of zero, scales of one."""
        if torch is None:
            _import_torch()
        shape = (num_blocks, kv_heads, block_size, head_dim)
        k, v = (torch.zeros(shape, dtype=torch.uint8, device=device) for _ in range(2))
        ks, vs = (torch.ones((num_blocks, kv_heads), dtype=torch.float32, device=device) for _ in range(2))
        return cls(k, v, ks, vs)


def cache_assign(cached_len, new_len, block_table, free_blocks, free_count, *, block_size, row_offsets, kv_len, slots,
                 positions=None, free_count_out=None, denied=None):
    """The bookkeeping of a serving step on the GPU (blazeCacheAssign): blocks for the requests that grow, the blocks of
    the ended ones (`new_len` < 0) back on the stack, and the packed batch's `row_offsets`, `slots` and `positions`.
    `kv_len` may be `cached_len`; `free_count_out` defaults to `free_count` (in place)."""
    if torch is None:
        _import_torch()
    if free_count_out is None:
        free_count_out = free_count
    device = _same_device(cached_len, new_len, block_table, free_blocks, free_count, row_offsets, kv_len, slots,
                          positions, free_count_out, denied)
    n, tokens, i32 = cached_len.numel(), slots.numel(), torch.int32
    rows, columns, pitch = _table(block_table)
    if rows < n:
        raise ValueError("block_table has fewer rows than there are requests")
    a = _ASSIGN.pack(
        _ASSIGN.size, n, block_size, columns, tokens,
        _vector(cached_len, "cached_len", i32, n), _vector(new_len, "new_len", i32, n),
        block_table.data_ptr(), pitch,
        _vector(free_blocks, "free_blocks", i32, 0), free_blocks.numel(), 0,
        _vector(free_count, "free_count", i32, 1), _vector(free_count_out, "free_count_out", i32, 1),
        _vector(row_offsets, "row_offsets", i32, n + 1), _vector(kv_len, "kv_len", i32, n),
        _vector(slots, "slots", torch.int64, 0),
        0 if positions is None else _vector(positions, "positions", i32, tokens),
        0 if denied is None else _vector(denied, "denied", i32, 1))
    _launch("blazeCacheAssign", device, a)


def _rows(t, name):
    """(address, token stride, head stride) of bf16 or half rows [tokens, heads, head size]; the stride of a dimension
    of one, which never counts, as 0."""
    if (t.dtype is not torch.bfloat16 and t.dtype is not torch.float16) or t.dim() != 3:
        raise ValueError(f"{name}: a bf16 or half [tokens, heads, head size] tensor is wanted")
    st, sh, sd = t.stride()
    if sd != 1 and t.shape[2] > 1:
        raise ValueError(f"{name}: the last dimension must be contiguous")
    return t.data_ptr(), st if t.shape[0] > 1 else 0, sh if t.shape[1] > 1 else 0


def cache_store(cache: PagedCache, k, v, slots):
    """Quantises the rows of `k` and `v` [tokens, kv heads, head size] into the cache's slots (blazeCacheStore)."""
    if torch is None:
        _import_torch()
    device = _same_device(cache.k, k, v, slots)
    at = _vector(slots, "slots", torch.int64, 0)
    n = slots.numel()
    pk, k_token, k_head = _rows(k, "k")
    pv, v_token, v_head = _rows(v, "v")
    rows = (cache.kv_heads, cache.head_dim)
    if k.dtype is not v.dtype or k.shape[0] < n or v.shape[0] < n or k.shape[1:] != rows or v.shape[1:] != rows:
        raise ValueError(f"k and v: [at least {n}, {cache.kv_heads}, {cache.head_dim}] is wanted, of one type")
    a = _STORE.pack(_STORE.size, n, out_type_of(k), pk, pv, k_token, k_head, v_token, v_head, at)
    _launch("blazeCacheStore", device, cache._desc_at, a)


def _attention_bounds(cache, q, requests, max_q, max_kv, sm_limit) -> CacheAttentionArgs:
    """Arguments as far as the workspace's size depends on them."""
    blocks = -(-max_kv // cache.block_size)
    return CacheAttentionArgs(struct_size=C.sizeof(CacheAttentionArgs), requests=requests, tokens=q.shape[0],
                              heads=q.shape[1], q_type=out_type_of(q), table_stride=blocks, max_blocks=blocks,
                              max_q=max_q, max_kv=max_kv, scale=1.0, sm_limit=sm_limit)


def cache_attention_workspace_bytes(cache: PagedCache, q, *, requests, max_q, max_kv, sm_limit=0) -> int:
    if torch is None:
        _import_torch()
    n = C.c_size_t(0)
    _rows(q, "q")
    with torch.cuda.device(cache.device):
        check(lib().blazeCacheAttentionWorkspaceSize(
            cache._desc_at, C.byref(_attention_bounds(cache, q, requests, max_q, max_kv, sm_limit)), C.byref(n)),
            "blazeCacheAttentionWorkspaceSize")
    return n.value


def cache_attention_workspace(cache: PagedCache, q, *, requests, max_q, max_kv, sm_limit=0):
    """A workspace for cache_attention calls of at most these bounds and as many rows as `q` has; needs no initialisation,
    keeps nothing between calls."""
    if torch is None:
        _import_torch()
    need = cache_attention_workspace_bytes(cache, q, requests=requests, max_q=max_q, max_kv=max_kv, sm_limit=sm_limit)
    return torch.empty(max(need, 256), dtype=torch.uint8, device=cache.device)


def cache_attention(cache: PagedCache, q, row_offsets, kv_len, block_table, *, scale=None, max_q, max_kv, min_q=0,
                    causal=True, window=0, out=None, lse=None, workspace=None, sm_limit=0):
    """Attention of the packed queries `q` [tokens, heads, head size] over the cache (blazeCacheAttention); `scale`
    defaults to head size ** -0.5.  `max_q`, `max_kv` bound the requests' rows and lengths, `min_q` is a hint.
    Allocates `out` (zeros: rows outside every request are not written) and `workspace` when not given; fills `lse`
    [tokens, heads] float32 when given."""
    if torch is None:
        _import_torch()
    if out is None:
        out = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    if workspace is None:
        workspace = cache_attention_workspace(cache, q, requests=kv_len.numel(), max_q=max_q, max_kv=max_kv,
                                              sm_limit=sm_limit)
    device = _same_device(cache.k, q, row_offsets, kv_len, block_table, out, lse, workspace)
    n = kv_len.numel()
    offsets, lens = _vector(row_offsets, "row_offsets", torch.int32, n + 1), _vector(kv_len, "kv_len", torch.int32, 0)
    table_rows, columns, pitch = _table(block_table)
    if table_rows < n:
        raise ValueError("block_table has fewer rows than there are requests")
    pq, q_token, q_head = _rows(q, "q")
    po, out_token, out_head = _rows(out, "out")
    tokens, heads, dim = q.shape
    if dim != cache.head_dim:
        raise ValueError(f"q has heads of {dim}, the cache of {cache.head_dim}")
    if out.shape != q.shape or out.dtype is not q.dtype:
        raise ValueError("out must have q's shape and type")
    if lse is not None and (lse.dtype is not torch.float32 or lse.shape != (tokens, heads) or not lse.is_contiguous()):
        raise ValueError("lse: a contiguous float32 [tokens, heads] tensor is wanted")
    if not workspace.is_contiguous():
        raise ValueError("workspace: a contiguous tensor is wanted")
    a = _ATTENTION.pack(
        _ATTENTION.size, n, tokens, heads, out_type_of(q), pq, q_token, q_head, po, out_token, out_head,
        0 if lse is None else lse.data_ptr(), offsets, lens, block_table.data_ptr(), pitch, columns,
        max_q, min_q, max_kv, dim ** -0.5 if scale is None else scale, 1 if causal else 0, window, sm_limit,
        workspace.data_ptr(), workspace.numel() * workspace.element_size())
    _launch("blazeCacheAttention", device, cache._desc_at, a)
    return out


def add_f32(a, c, out=None):
    import torch
    if out is None:
        out = torch.empty_like(a)
    check(lib().blazeAddF32(_ptr(a), _ptr(c), _ptr(out), a.numel(), _stream()), "blazeAddF32")
    return out
