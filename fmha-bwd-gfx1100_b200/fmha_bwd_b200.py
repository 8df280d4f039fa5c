"""Host-side mirror of the reference's Python/ctypes interface for the
attention-backward path, backed by the sm_100a libraries in build/.

Reference interface (benchmark_pytorch_final.py):
  * ``lib = ctypes.CDLL('./build/libfmha_bwd_bf16.so')`` with argtypes of
    8 x c_void_p + 4 x c_int (:30-37)
  * ``custom_flash_attn_backward(Q, K, V, P, dO)`` (:39-53): zero-fills the
    outputs and calls ``fmha_bwd_full_py`` with device pointers
  * ``pytorch_naive_backward`` (:58-70): einsum reference (no scale)
  * ``benchmark_size(batch, heads, M, N, K_dim, ...)`` (:82-136)

This module keeps those names, argument meanings and return values. It
differs from the reference script in three deliberate ways:
  * ``total_heads`` is ``batch * heads`` (the reference passes ``heads``,
    :51, which only covers batch 1);
  * the library is chosen by dtype (bf16 -> libfmha_bwd_bf16.so, fp16 ->
    libfmha_bwd_fp16.so) instead of always loading the bf16 one;
  * a call the library rejects raises ``FmhaBwdError`` with the library's
    error code and message instead of silently returning zeros.

There is no fallback: if the CUDA library is missing or the device is not an
sm_100 GPU, calls raise.
"""
from __future__ import annotations

import ctypes
import functools
import math
import os
import struct

import torch

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
ROOT_DIR = os.path.dirname(PKG_DIR)
BUILD_DIR = os.path.join(ROOT_DIR, "build")

LIB_NAMES = {
    torch.bfloat16: ("libfmha_bwd_bf16.so", "fmha_bwd_full_py", "fmha_bwd_full_stream"),
    torch.float16: ("libfmha_bwd_fp16.so", "fmha_bwd_full_fp16", "fmha_bwd_full_fp16_stream"),
}
# precomputed-rowsum entries (additive to the reference's ABI)
DELTA_NAMES = {
    torch.bfloat16: "fmha_bwd_full_delta",
    torch.float16: "fmha_bwd_full_fp16_delta",
}

# recompute-P entries: P = exp(scale Q K^T - LSE) formed on chip
LSE_NAMES = {
    torch.bfloat16: "fmha_bwd_full_lse",
    torch.float16: "fmha_bwd_full_fp16_lse",
}

# attention entries: forward and backward against an encoder's states, and
# attention behind a shared prefix (argument block fmha_attn_t)
ATTN_NAMES = {
    torch.bfloat16: ("fmha_cross_fwd", "fmha_cross_bwd", "fmha_prefix_attn"),
    torch.float16: ("fmha_cross_fp16_fwd", "fmha_cross_fp16_bwd", "fmha_prefix_fp16_attn"),
}
_CROSS_FWD, _CROSS_BWD, _PREFIX = range(3)

ERROR_NAMES = {
    0: "OK",
    1: "INVALID_ARGUMENT",
    2: "MISALIGNED",
    3: "UNSUPPORTED_DEVICE",
    4: "OUT_OF_MEMORY",
    5: "LAUNCH",
    6: "DEVICE_TIMEOUT",
    7: "NO_DRIVER",
}


class FmhaBwdError(RuntimeError):
    def __init__(self, code: int, message: str):
        super().__init__(f"fmha_bwd error {code} ({ERROR_NAMES.get(code, '?')}): {message}")
        self.code = code


_LIBS: dict[str, ctypes.CDLL] = {}

_PTR_ARGS = [ctypes.c_void_p] * 8
_INT_ARGS = [ctypes.c_int] * 4


def library_path(dtype: torch.dtype) -> str:
    if dtype not in LIB_NAMES:
        raise TypeError(f"unsupported dtype {dtype}; use torch.bfloat16 or torch.float16")
    return os.path.join(BUILD_DIR, LIB_NAMES[dtype][0])


def load_library(dtype: torch.dtype = torch.bfloat16) -> ctypes.CDLL:
    """Load (once) and return the ctypes handle for ``dtype``'s library, with
    the same argtypes the reference script declares (:32-37)."""
    path = library_path(dtype)
    lib = _LIBS.get(path)
    if lib is not None:
        return lib
    if not os.path.exists(path):
        raise FileNotFoundError(
            f"{path} is missing: build it with python fmha-bwd-gfx1100_b200/build_libs.py")
    lib = ctypes.CDLL(path)
    _, full, stream = LIB_NAMES[dtype]
    getattr(lib, full).argtypes = _PTR_ARGS + _INT_ARGS
    getattr(lib, full).restype = None
    getattr(lib, stream).argtypes = _PTR_ARGS + _INT_ARGS + [ctypes.c_void_p]
    getattr(lib, stream).restype = ctypes.c_int
    delta = DELTA_NAMES[dtype]
    getattr(lib, delta).argtypes = _PTR_ARGS + [ctypes.c_void_p] + _INT_ARGS + [ctypes.c_void_p]
    getattr(lib, delta).restype = ctypes.c_int
    lse = LSE_NAMES[dtype]
    getattr(lib, lse).argtypes = (_PTR_ARGS + [ctypes.c_void_p] + _INT_ARGS +
                                  [ctypes.c_float, ctypes.c_void_p])
    getattr(lib, lse).restype = ctypes.c_int
    for name in ATTN_NAMES[dtype]:
        getattr(lib, name).argtypes = [ctypes.c_char_p, ctypes.c_void_p]
        getattr(lib, name).restype = ctypes.c_int
    lib.fmha_attn_workspace.argtypes = [ctypes.c_char_p, ctypes.c_int, ctypes.c_void_p]
    lib.fmha_attn_workspace.restype = ctypes.c_int
    lib.fmha_bwd_last_error.argtypes = []
    lib.fmha_bwd_last_error.restype = ctypes.c_int
    lib.fmha_bwd_last_error_message.argtypes = []
    lib.fmha_bwd_last_error_message.restype = ctypes.c_char_p
    lib.fmha_bwd_poll_device_status.argtypes = []
    lib.fmha_bwd_poll_device_status.restype = ctypes.c_int
    lib.fmha_bwd_set_wait_timeout_ms.argtypes = [ctypes.c_int]
    lib.fmha_bwd_set_wait_timeout_ms.restype = None
    _LIBS[path] = lib
    return lib


def rowsum_delta(P, dO, V):
    """D = rowsum(P * (dO V^T)) in fp32, [H, M] (reference formula,
    cpu_reference.hpp:32-35), computed with torch for callers and tests of
    the precomputed-rowsum entry."""
    dP = torch.einsum("...mk,...nk->...mn", dO.float(), V.float())
    return (dP * P.float()).sum(dim=-1).contiguous()


def last_error(dtype: torch.dtype = torch.bfloat16) -> tuple[int, str]:
    lib = load_library(dtype)
    return lib.fmha_bwd_last_error(), (lib.fmha_bwd_last_error_message() or b"").decode()


def _raise_if_error(lib: ctypes.CDLL, rc: int | None = None) -> None:
    code = lib.fmha_bwd_last_error() if rc is None else rc
    if code != 0:
        msg = (lib.fmha_bwd_last_error_message() or b"").decode()
        raise FmhaBwdError(code, msg)


def _check_inputs(Q, K, V, P, dO):
    for name, t in (("Q", Q), ("K", K), ("V", V), ("P", P), ("dO", dO)):
        if not t.is_cuda:
            raise ValueError(f"{name} must be a CUDA tensor")
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
        if t.dtype != Q.dtype:
            raise TypeError(f"{name} has dtype {t.dtype}, expected {Q.dtype}")


def fmha_bwd(Q, K, V, P, dO, *, out=None, stream=None, sync: bool = True, delta=None):
    """Backward of attention for head-flattened tensors.

    Q, dO: [H, M, d]; K, V: [H, N, d]; P: [H, M, N] (any leading shape that
    flattens to these, contiguous). Returns (dQ, dK, dV) with the shapes of
    Q, K, V. ``out`` may supply preallocated (dQ, dK, dV) tensors, which are
    fully overwritten. With ``sync=True`` the call uses the reference entry
    (``fmha_bwd_full_py`` / ``fmha_bwd_full_fp16``), which returns after the
    work has finished; with ``sync=False`` it uses the stream-ordered entry
    on ``stream`` (default: torch's current stream) and returns at once.
    ``delta``, when given, is D = rowsum(P * dP) (equivalently rowsum(dO * O)
    for the forward output O), an fp32 CUDA tensor of H*M elements; the
    precomputed-rowsum entry then skips the rowsum and one GEMM-sized pass
    (stream-ordered; synchronised afterwards when ``sync`` is set).
    """
    _check_inputs(Q, K, V, P, dO)
    d = Q.shape[-1]
    M = Q.shape[-2]
    N = K.shape[-2]
    H = Q.numel() // (M * d)
    if K.numel() != H * N * d or V.numel() != H * N * d or dO.numel() != H * M * d \
            or P.numel() != H * M * N:
        raise ValueError("inconsistent shapes for Q, K, V, P, dO")
    lib = load_library(Q.dtype)
    if out is None:
        dQ, dK, dV = torch.empty_like(Q), torch.empty_like(K), torch.empty_like(V)
    else:
        dQ, dK, dV = out
    args = (dQ.data_ptr(), dK.data_ptr(), dV.data_ptr(), Q.data_ptr(), K.data_ptr(),
            V.data_ptr(), P.data_ptr(), dO.data_ptr(), M, N, d, H)
    _, full, stream_fn = LIB_NAMES[Q.dtype]
    if delta is not None:
        if not delta.is_cuda or delta.dtype != torch.float32 or not delta.is_contiguous() \
                or delta.numel() != H * M:
            raise ValueError("delta must be a contiguous fp32 CUDA tensor of H*M elements")
        s = stream if stream is not None else torch.cuda.current_stream(Q.device)
        rc = getattr(lib, DELTA_NAMES[Q.dtype])(*args[:8], delta.data_ptr(), *args[8:],
                                               ctypes.c_void_p(s.cuda_stream))
        _raise_if_error(lib, rc)
        if sync:
            s.synchronize()
        return dQ, dK, dV
    if sync:
        getattr(lib, full)(*args)
        _raise_if_error(lib)
    else:
        s = stream if stream is not None else torch.cuda.current_stream(Q.device)
        rc = getattr(lib, stream_fn)(*args, ctypes.c_void_p(s.cuda_stream))
        _raise_if_error(lib, rc)
    return dQ, dK, dV


def fmha_bwd_lse(Q, K, V, O, dO, LSE, scale: float, *, out=None, stream=None,
                 sync: bool = True):
    """Backward that recomputes P = exp(scale Q K^T - LSE) on chip instead of
    reading it (the FlashAttention form). Q, O, dO: [H, M, d]; K, V: [H, N, d];
    LSE: fp32 [H, M] (natural log of the row sums of exp(scale Q K^T)).
    Returns (dQ, dK, dV) = (scale dS K, scale dS^T Q, P^T dO) with
    dS = P (dO V^T - rowsum(dO * O)). Stream-ordered on ``stream`` (default:
    torch's current stream); with ``sync`` the call waits and raises on an
    in-kernel wait timeout."""
    for name, t in (("Q", Q), ("K", K), ("V", V), ("O", O), ("dO", dO)):
        if not t.is_cuda or not t.is_contiguous() or t.dtype != Q.dtype:
            raise ValueError(f"{name} must be a contiguous CUDA tensor of {Q.dtype}")
    d = Q.shape[-1]
    M, N = Q.shape[-2], K.shape[-2]
    H = Q.shape[:-2].numel()
    if K.shape[-1] != d or V.shape != K.shape or O.shape != Q.shape or dO.shape != Q.shape:
        raise ValueError("shape mismatch among Q, K, V, O, dO")
    if not LSE.is_cuda or LSE.dtype != torch.float32 or not LSE.is_contiguous() or LSE.numel() != H * M:
        raise ValueError("LSE must be a contiguous fp32 CUDA tensor of H*M elements")
    lib = load_library(Q.dtype)
    if out is None:
        out = (torch.empty_like(Q), torch.empty_like(K), torch.empty_like(V))
    dQ, dK, dV = out
    s = stream if stream is not None else torch.cuda.current_stream(Q.device)
    rc = getattr(lib, LSE_NAMES[Q.dtype])(
        dQ.data_ptr(), dK.data_ptr(), dV.data_ptr(), Q.data_ptr(), K.data_ptr(), V.data_ptr(),
        O.data_ptr(), dO.data_ptr(), LSE.data_ptr(), M, N, d, H, float(scale),
        ctypes.c_void_p(s.cuda_stream))
    _raise_if_error(lib, rc)
    if sync:
        s.synchronize()
        if lib.fmha_bwd_poll_device_status() != 0:
            raise FmhaBwdError(6, "fmha_bwd_lse: an in-kernel wait gave up")
    return dQ, dK, dV


# ------------------------------------------------- attention: encoder states
# fmha_attn_t of include/fmha_bwd.h: ten tensors (pointer, batch, head and row
# stride), LSE, kv_lens, prefix_lens, workspace, its bytes, eight sizes, scale.
_ATTN = struct.Struct("=40q5q8ifi")
_NO_TENSOR = (0, 0, 0, 0)


def _tensor_arg(t):
    sb, sh, sr, _ = t.stride()
    return t.data_ptr(), sb, sh, sr


def _check_attn_tensor(name, t, dev, dtype, shape):
    if t.get_device() != dev:
        raise ValueError(f"{name} must be a CUDA tensor on device {dev}")
    if t.dtype != dtype:
        raise TypeError(f"{name} has dtype {t.dtype}, expected {dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.stride(3) != 1:
        raise ValueError(f"{name} must have unit stride along its last axis")


def _check_lens(name, t, dev, count):
    if t is not None and (t.get_device() != dev or t.dtype != torch.int32 or t.dim() != 1 or t.numel() != count
                          or not t.is_contiguous()):
        raise ValueError(f"{name} must be a contiguous int32 tensor of {count} elements on device {dev}")


def _check_lse(LSE, dev, shape):
    if LSE.get_device() != dev or LSE.dtype != torch.float32 or LSE.shape != shape[:3] or not LSE.is_contiguous():
        raise ValueError(f"LSE must be a contiguous fp32 tensor of shape {tuple(shape[:3])} on device {dev}")


def _check_qkv(Q, shape, K, V, names=("K", "V")):
    """Checks Q (whose shape is `shape`) against K and V; returns K's shape and the device index."""
    dev, dtype = Q.get_device(), Q.dtype
    if dev < 0:
        raise ValueError("Q must be a CUDA tensor")
    if dtype not in LIB_NAMES:
        raise TypeError(f"unsupported dtype {dtype}; use torch.bfloat16 or torch.float16")
    kshape = K.shape
    if len(shape) != 4 or len(kshape) != 4:
        raise ValueError(f"Q and {names[0]} must be [batch, heads, rows, d]")
    if kshape[1] == 0 or shape[1] % kshape[1] != 0:
        raise ValueError(f"{shape[1]} query heads do not divide among {kshape[1]} kv heads")
    if kshape[3] != shape[3]:
        raise ValueError(f"{names[0]} has {kshape[3]} columns, Q has {shape[3]}")
    if Q.stride(3) != 1:
        raise ValueError("Q must have unit stride along its last axis")
    _check_attn_tensor(names[0], K, dev, dtype, kshape)
    _check_attn_tensor(names[1], V, dev, dtype, kshape)
    return kshape, dev


@functools.lru_cache(maxsize=4096)
def _attn_entry(dtype, op, sizes):
    """The entry of `op` for `dtype`, its library, and the workspace bytes of these sizes."""
    lib = load_library(dtype)
    need = ctypes.c_uint64()
    rc = lib.fmha_attn_workspace(_ATTN.pack(*_NO_TENSOR * 10, 0, 0, 0, 0, 0, *sizes, 1.0, 0), op, ctypes.byref(need))
    _raise_if_error(lib, rc)
    return getattr(lib, ATTN_NAMES[dtype][op]), lib, need.value


def _run_attn(op, Q, dev, tensors, make_out, out, LSE, kv_lens, prefix_lens, sizes, scale, stream, sync):
    """One call of an attention entry on `stream`. `tensors` are the ten of
    fmha_attn_t, with ... in the place of each output (an LSE that is one comes
    last among them) and None for those that the entry does not take; outputs
    and workspace come from torch's allocator, for the stream that the call
    runs on."""
    if not 0 < scale < math.inf:
        raise ValueError(f"scale must be positive and finite, not {scale}")
    if torch.cuda.current_device() != dev:
        with torch.cuda.device(dev):
            return _run_attn(op, Q, dev, tensors, make_out, out, LSE, kv_lens, prefix_lens, sizes, scale, stream, sync)
    if stream is not None:
        current = torch.cuda.current_stream(dev)
        if stream.device.index != dev:
            raise ValueError(f"stream is on {stream.device}, the tensors on device {dev}")
        if stream != current:
            with torch.cuda.stream(stream):
                res = _run_attn(op, Q, dev, tensors, make_out, out, LSE, kv_lens, prefix_lens, sizes, scale, None, sync)
            # memory used on a stream other than the one it was allocated for
            for t in (*tensors, LSE, kv_lens, prefix_lens):
                if isinstance(t, torch.Tensor):
                    t.record_stream(stream)
            for t in res:
                t.record_stream(stream if out is not None else current)
            return res
    entry, lib, need = _attn_entry(Q.dtype, op, sizes)
    res = made = make_out() if out is None else out
    ws = torch.empty(need, dtype=torch.uint8, device=Q.device).data_ptr() if need else 0
    args = []
    k = 0
    for t in tensors:
        if t is None:
            args += _NO_TENSOR
        elif t is Ellipsis:
            args += _tensor_arg(made[k])
            k += 1
        else:
            args += _tensor_arg(t)
    rc = entry(
        _ATTN.pack(*args, (made[k] if LSE is Ellipsis else LSE).data_ptr(),
                   0 if kv_lens is None else kv_lens.data_ptr(), 0 if prefix_lens is None else prefix_lens.data_ptr(),
                   ws, need, *sizes, scale, 0), torch._C._cuda_getCurrentRawStream(dev))
    if rc != 0:
        _raise_if_error(lib, rc)
    if sync:
        torch.cuda.current_stream(dev).synchronize()
        if lib.fmha_bwd_poll_device_status() != 0:
            raise FmhaBwdError(6, f"{ATTN_NAMES[Q.dtype][op]}: an in-kernel wait gave up")
    return tuple(res)


def cross_attn_fwd(Q, K, V, kv_lens=None, scale=None, *, out=None, stream=None, sync: bool = True):
    """Attention to an encoder's states of another length: returns (O, LSE)
    with O = softmax(scale Q K^T) V over each batch entry's valid keys and LSE
    the fp32 row log-sum-exp that fmha_bwd_lse and cross_attn_bwd take.

    Q: [B, Hq, M, d]; K, V: [B, Hkv, N, d], Hq a multiple of Hkv (query head h
    reads kv head h // (Hq // Hkv)). Any strides above 0 that are multiples of
    8 elements, with unit stride along d, so the transposed views of [B, rows,
    H, d] projections need no copy (broadcast views, with stride 0, do). ``kv_lens``: int32 [B] on the device, the
    valid rows of K and V (None: all); what lies behind them is never used. A
    row without valid keys gets O = 0 and LSE = -inf. ``scale`` defaults to
    1/sqrt(d). M = 1 is the form for single tokens: each K and V is then read
    once, by as many SMs as it takes.

    ``out`` may supply (O, LSE). Runs on ``stream`` (default: torch's current
    stream); with ``sync`` the call waits and raises on an in-kernel wait
    timeout. With sync=False it can be captured into a CUDA graph."""
    shape = B, Hq, M, d = Q.shape
    kshape, dev = _check_qkv(Q, shape, K, V)
    if kshape[0] != B:
        raise ValueError(f"K has batch {kshape[0]}, expected {B}")
    _check_lens("kv_lens", kv_lens, dev, B)
    if out is not None:
        _check_attn_tensor("O", out[0], dev, Q.dtype, shape)
        _check_lse(out[1], dev, shape)
    return _run_attn(
        _CROSS_FWD, Q, dev, (Q, ..., K, V, None, None, None, None, None, None),
        lambda: (torch.empty_like(Q), Q.new_empty((B, Hq, M), dtype=torch.float32)), out, ..., kv_lens,
        None, (B, Hq, kshape[1], M, kshape[2], d, 0, 0), d ** -0.5 if scale is None else float(scale), stream, sync)


def cross_attn_bwd(Q, K, V, O, LSE, dO, kv_lens=None, scale=None, *, out=None, stream=None, sync: bool = True):
    """Backward of cross_attn_fwd: returns (dQ, dK, dV) from the forward's O
    and LSE and from dO, with the same kv_lens and scale. dK and dV sum over
    the query heads of their kv head and are zero at and past kv_lens. There
    are no atomics: two calls give the same bits. ``out`` may supply (dQ, dK,
    dV), which are fully overwritten; ``stream`` and ``sync`` as there."""
    shape = B, Hq, M, d = Q.shape
    kshape, dev = _check_qkv(Q, shape, K, V)
    if kshape[0] != B:
        raise ValueError(f"K has batch {kshape[0]}, expected {B}")
    _check_attn_tensor("O", O, dev, Q.dtype, shape)
    _check_attn_tensor("dO", dO, dev, Q.dtype, shape)
    _check_lse(LSE, dev, shape)
    _check_lens("kv_lens", kv_lens, dev, B)
    if out is not None:
        for name, t, like in zip(("dQ", "dK", "dV"), out, (shape, kshape, kshape)):
            _check_attn_tensor(name, t, dev, Q.dtype, like)
    return _run_attn(
        _CROSS_BWD, Q, dev, (Q, O, K, V, dO, ..., ..., ..., None, None),
        lambda: (torch.empty_like(Q), torch.empty_like(K), torch.empty_like(V)), out, LSE, kv_lens, None,
        (B, Hq, kshape[1], M, kshape[2], d, 0, 0), d ** -0.5 if scale is None else float(scale), stream, sync)


def prefix_attn(Q, Kp, Vp, K, V, prefix_lens=None, kv_lens=None, scale=None, *, out=None, stream=None,
                sync: bool = True):
    """Attention of the newest tokens of a batch whose entries share long
    prefixes: returns (O, LSE) as cross_attn_fwd does.

    Q: [B, Hq, M, d], the M newest tokens of each entry (M = 1 when decoding,
    more when several drafted tokens are checked at once). Kp, Vp: [P, Hkv,
    Np, d], shared by B / P consecutive entries each (entry b reads prefix
    b // (B // P)), of which prefix_lens[p] rows count. K, V: [B, Hkv, N, d],
    each entry's own cache behind the prefix, of which kv_lens[b] rows count,
    the M newest tokens' own rows last: row m sees all but the M - 1 - m
    newest, and nothing of those reaches it. The softmax runs over both. The
    prefix is read once for all of its entries, or once for each where that is
    little. Strides, ``out``, ``stream`` and ``sync`` as cross_attn_fwd."""
    shape = B, Hq, M, d = Q.shape
    kshape, dev = _check_qkv(Q, shape, K, V)
    pshape, _ = _check_qkv(Q, shape, Kp, Vp, ("Kp", "Vp"))
    P, Hkv = pshape[:2]
    if kshape[0] != B or kshape[1] != Hkv:
        raise ValueError(f"K has batch and heads {tuple(kshape[:2])}, expected {(B, Hkv)}")
    if P == 0 or B % P != 0:
        raise ValueError(f"{B} batch entries do not divide among {P} prefixes")
    _check_lens("prefix_lens", prefix_lens, dev, P)
    _check_lens("kv_lens", kv_lens, dev, B)
    if out is not None:
        _check_attn_tensor("O", out[0], dev, Q.dtype, shape)
        _check_lse(out[1], dev, shape)
    return _run_attn(
        _PREFIX, Q, dev, (Q, ..., K, V, None, None, None, None, Kp, Vp),
        lambda: (torch.empty_like(Q), Q.new_empty((B, Hq, M), dtype=torch.float32)), out, ..., kv_lens,
        prefix_lens, (B, Hq, Hkv, M, kshape[2], d, P, pshape[2]), d ** -0.5 if scale is None else float(scale), stream,
        sync)


# ---------------------------------------------------------------- stage hooks
# The reference's test_* wrappers (src/fmha_bwd_kernels.hip:525-560,
# src/fmha_bwd_kernels_fp16.hip:284-314), one stage per launch with its
# 16-bit intermediate in global memory. bf16 names have no suffix, fp16
# names end in _fp16.
STAGE_NAMES = ("dp", "softmax_bwd", "dq", "dk", "dv")


def _stage_fn(lib: ctypes.CDLL, dtype: torch.dtype, stage: str):
    name = f"test_{stage}_kernel" + ("_fp16" if dtype == torch.float16 else "")
    f = getattr(lib, name)
    if stage == "softmax_bwd":
        f.argtypes = [ctypes.c_void_p] * 3 + [ctypes.c_int] * 3
    else:
        f.argtypes = [ctypes.c_void_p] * 3 + [ctypes.c_int] * 4
    f.restype = None
    return f


def run_stage(stage: str, a, b, *, sync: bool = True):
    """Run one stage hook on [H, rows, cols] inputs in the reference's
    argument order and return its output:
      dp (dO, V) -> dP [H,M,N];  softmax_bwd (P, dP) -> dS [H,M,N];
      dq (dS, K) -> dQ [H,M,d];  dk (dS, Q) -> dK [H,N,d];
      dv (P, dO) -> dV [H,N,d].
    The hook launches on the legacy default stream; with ``sync`` the call
    waits for it and raises on an error or an in-kernel wait timeout."""
    if stage not in STAGE_NAMES:
        raise ValueError(f"unknown stage {stage!r}; one of {STAGE_NAMES}")
    for name, t in (("a", a), ("b", b)):
        if not t.is_cuda or not t.is_contiguous() or t.dtype != a.dtype or t.dim() < 3:
            raise ValueError(f"{name} must be a contiguous CUDA tensor [H, rows, cols] of {a.dtype}")
    lib = load_library(a.dtype)
    H = a.shape[:-2].numel()
    if stage == "dp":  # dO [H,M,d], V [H,N,d]
        M, d = a.shape[-2:]
        N = b.shape[-2]
        out = torch.empty(*a.shape[:-1], N, dtype=a.dtype, device=a.device)
        ints = (M, N, d, H)
    elif stage == "softmax_bwd":  # P, dP [H,M,N]
        M, N = a.shape[-2:]
        out = torch.empty_like(a)
        ints = (M, N, H)
    elif stage == "dq":  # dS [H,M,N], K [H,N,d]
        M, N = a.shape[-2:]
        d = b.shape[-1]
        out = torch.empty(*a.shape[:-1], d, dtype=a.dtype, device=a.device)
        ints = (M, N, d, H)
    else:  # dk: dS [H,M,N], Q [H,M,d]; dv: P [H,M,N], dO [H,M,d]
        M, N = a.shape[-2:]
        d = b.shape[-1]
        out = torch.empty(*a.shape[:-2], N, d, dtype=a.dtype, device=a.device)
        ints = (M, N, d, H)
    _stage_fn(lib, a.dtype, stage)(a.data_ptr(), b.data_ptr(), out.data_ptr(), *ints)
    _raise_if_error(lib)
    if sync:
        torch.cuda.synchronize(a.device)
        if lib.fmha_bwd_poll_device_status() != 0:
            raise FmhaBwdError(6, f"stage {stage}: an in-kernel wait gave up")
    return out


def custom_flash_attn_backward(Q, K, V, P, dO):
    """Mirror of the reference's custom_flash_attn_backward
    (benchmark_pytorch_final.py:39-53) for [batch, heads, M, d] inputs.
    Outputs are zero-filled first, as the reference does (:43-45), then fully
    overwritten by the library."""
    batch, heads, M, K_dim = Q.shape
    dQ = torch.zeros_like(Q)
    dK = torch.zeros_like(K)
    dV = torch.zeros_like(V)
    return fmha_bwd(Q, K, V, P, dO, out=(dQ, dK, dV))


def pytorch_naive_backward(Q, K, V, P, dO):
    """The reference script's einsum formula (benchmark_pytorch_final.py:58-70),
    computed here in fp32 on the inputs' device. Test/benchmark reference only."""
    Qf, Kf, Vf, Pf, dOf = (t.float() for t in (Q, K, V, P, dO))
    dP = torch.einsum("...mk,...nk->...mn", dOf, Vf)
    rowsum = (dP * Pf).sum(dim=-1, keepdim=True)
    dS = Pf * (dP - rowsum)
    dQ = torch.einsum("...mn,...nk->...mk", dS, Kf)
    dK = torch.einsum("...mn,...mk->...nk", dS, Qf)
    dV = torch.einsum("...mn,...mk->...nk", Pf, dOf)
    return dQ, dK, dV


def _einsum_backward_native(Q, K, V, P, dO):
    """The reference script's einsum backward (benchmark_pytorch_final.py:58-70)
    in the inputs' own dtype, as that script times it (:110-115)."""
    dP = torch.einsum("...mk,...nk->...mn", dO, V)
    rowsum = (dP * P).sum(dim=-1, keepdim=True)
    dS = P * (dP - rowsum)
    dQ = torch.einsum("...mn,...nk->...mk", dS, K)
    dK = torch.einsum("...mn,...mk->...nk", dS, Q)
    dV = torch.einsum("...mn,...mk->...nk", P, dO)
    return dQ, dK, dV


def benchmark_size(batch, heads, M, N, K_dim, dtype=torch.bfloat16, warmup=5, reps=20):
    """Mirror of the reference's benchmark_size (benchmark_pytorch_final.py:82-136):
    seeded inputs, warmup, CUDA-event timing of ``reps`` synchronous calls and
    of ``reps`` einsum backwards in the inputs' dtype (the PyTorch baseline),
    FLOPs = 4 * 2*M*N*d per head (:125-127, here summed over batch*heads),
    and the max difference against the einsum reference (computed here in
    fp32). Returns the reference's keys: M, N, K, custom_time_ms,
    pytorch_time_ms, speedup, max_diff, custom_tflops."""
    device = torch.device("cuda")
    torch.manual_seed(42)
    Q = torch.randn(batch, heads, M, K_dim, dtype=dtype, device=device)
    K = torch.randn(batch, heads, N, K_dim, dtype=dtype, device=device)
    V = torch.randn(batch, heads, N, K_dim, dtype=dtype, device=device)
    dO = torch.randn(batch, heads, M, K_dim, dtype=dtype, device=device)
    P = torch.softmax(torch.randn(batch, heads, M, N, dtype=dtype, device=device), dim=-1)
    for _ in range(warmup):
        custom_flash_attn_backward(Q, K, V, P, dO)
    torch.cuda.synchronize()
    start = torch.cuda.Event(enable_timing=True)
    end = torch.cuda.Event(enable_timing=True)
    start.record()
    for _ in range(reps):
        dQ, dK, dV = custom_flash_attn_backward(Q, K, V, P, dO)
    end.record()
    torch.cuda.synchronize()
    custom_ms = start.elapsed_time(end) / reps
    for _ in range(warmup):
        _einsum_backward_native(Q, K, V, P, dO)
    torch.cuda.synchronize()
    start.record()
    for _ in range(reps):
        _einsum_backward_native(Q, K, V, P, dO)
    end.record()
    torch.cuda.synchronize()
    pt_ms = start.elapsed_time(end) / reps
    rQ, rK, rV = pytorch_naive_backward(Q, K, V, P, dO)
    max_diff = max((dQ.float() - rQ).abs().max().item(), (dK.float() - rK).abs().max().item(),
                   (dV.float() - rV).abs().max().item())
    flops = 4 * 2.0 * M * N * K_dim * batch * heads
    return {
        "M": M, "N": N, "K": K_dim,
        "custom_time_ms": custom_ms,
        "pytorch_time_ms": pt_ms,
        "speedup": pt_ms / custom_ms if custom_ms > 0 else 0.0,
        "max_diff": max_diff,
        "custom_tflops": flops / (custom_ms * 1e-3) / 1e12 if custom_ms > 0 else 0.0,
    }
