"""CPU checks of the attention entries: the C-ABI refuses bad argument blocks
on the host, the Python entries refuse bad tensors, and the 64-bit reference
of the GPU tests agrees with autograd and notices planted mistakes."""
from __future__ import annotations

import ctypes

import pytest
import torch

import attn_reference as R
from test_abi import LIBS, _ensure_built

ENTRIES = {"bf16": ("fmha_cross_fwd", "fmha_cross_bwd", "fmha_prefix_attn"),
           "fp16": ("fmha_cross_fp16_fwd", "fmha_cross_fp16_bwd", "fmha_prefix_fp16_attn")}


class Tensor(ctypes.Structure):
    _fields_ = [("ptr", ctypes.c_void_p), ("batch", ctypes.c_int64), ("head", ctypes.c_int64), ("row", ctypes.c_int64)]


class Attn(ctypes.Structure):
    _fields_ = ([(n, Tensor) for n in ("Q", "O", "K", "V", "dO", "dQ", "dK", "dV", "Kp", "Vp")] +
                [(n, ctypes.c_void_p) for n in ("LSE", "kv_lens", "prefix_lens", "workspace")] +
                [("workspace_bytes", ctypes.c_uint64)] +
                [(n, ctypes.c_int) for n in ("batch", "q_heads", "kv_heads", "M", "N", "K_dim", "prefixes", "N_prefix")] +
                [("softmax_scale", ctypes.c_float), ("reserved", ctypes.c_int)])


def good():
    """A right argument block whose pointers are never followed."""
    a = Attn(batch=2, q_heads=4, kv_heads=2, M=100, N=50, K_dim=64, prefixes=1, N_prefix=70, softmax_scale=0.125,
             LSE=0x900000, workspace=0xA00000, workspace_bytes=1 << 40)
    for i, (name, _) in enumerate(Attn._fields_[:10]):
        rows = {"K": 50, "V": 50, "dK": 50, "dV": 50, "Kp": 70, "Vp": 70}.get(name, 100)
        heads = 2 if rows != 100 else 4
        setattr(a, name, Tensor(0x10000000 * (i + 1), heads * rows * 64, rows * 64, 64))
    return a


def entry(kind, i):
    _ensure_built()
    lib = ctypes.CDLL(LIBS[kind])
    f = getattr(lib, ENTRIES[kind][i])
    f.argtypes, f.restype = [ctypes.c_void_p, ctypes.c_void_p], ctypes.c_int
    lib.fmha_bwd_last_error_message.restype = ctypes.c_char_p
    return lambda a: (f(ctypes.byref(a) if a is not None else None, None), lib.fmha_bwd_last_error_message().decode())


def change(**kw):
    a = good()
    for k, v in kw.items():
        name, _, part = k.partition("__")
        setattr(getattr(a, name) if part else a, part or name, v)
    return a


BAD = [
    (1, "positive", dict(batch=0)), (1, "positive", dict(M=-1)), (1, "positive", dict(N=0)),
    (1, "K_dim", dict(K_dim=96)), (1, "multiple", dict(q_heads=3)), (1, "2^30", dict(M=1 << 29)),
    (1, "Q", dict(Q__ptr=None)), (1, "V", dict(V__ptr=None)), (2, "K", dict(K__ptr=0x1008)),
    (2, "O", dict(O__ptr=0x1002)), (2, "multiple of 8", dict(K__row=68)), (1, "stride", dict(K__batch=0)),
    (1, "stride", dict(V__head=-64)), (1, "rows overlap", dict(Q__row=32)), (1, "LSE", dict(LSE=None)),
    (2, "LSE", dict(LSE=0x1002)), (2, "kv_lens", dict(kv_lens=0x1001)), (1, "scale", dict(softmax_scale=0.0)),
    (1, "scale", dict(softmax_scale=float("nan"))), (1, "scale", dict(softmax_scale=float("inf"))),
]
BAD_OF = {
    0: [(1, "overlap", dict(O__head=64)), (1, "input", dict(O__ptr=0x10000000)),
        (1, "input", dict(LSE=0x10000000)), (1, "another", dict(LSE=0x20000000))],
    1: [(1, "dO", dict(dO__ptr=None)), (1, "overlap", dict(dK__batch=64)), (2, "dV", dict(dV__ptr=0x1004)),
        (1, "input", dict(dQ__ptr=0x10000000)), (1, "another", dict(dK__ptr=0x80000000)),
        (1, "another", dict(dQ__ptr=0x70000000))],
    2: [(1, "Kp", dict(Kp__ptr=None)), (1, "prefixes", dict(prefixes=0)), (1, "multiple", dict(prefixes=3)),
        (1, "N_prefix", dict(N_prefix=0)), (2, "prefix_lens", dict(prefix_lens=0x1002)),
        (2, "Vp", dict(Vp__row=66))],
}


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("i", [0, 1, 2])
def test_entries_refuse_bad_blocks(kind, i):
    call = entry(kind, i)
    assert call(None)[0] == 1
    for code, word, kw in BAD + BAD_OF[i]:
        got, message = call(change(**kw))
        assert (got, word in message) == (code, True), (kw, got, message)


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
def test_a_right_block_gets_as_far_as_the_device(kind):
    """No GPU here: the checks pass and the device is what is missing."""
    if torch.cuda.is_available():
        pytest.skip("the pointers lead nowhere")
    for i in range(3):
        assert entry(kind, i)(good())[0] in (3, 5)


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
def test_workspace_query(kind):
    _ensure_built()
    lib = ctypes.CDLL(LIBS[kind])
    need = ctypes.c_uint64()
    for op in range(3):
        assert lib.fmha_attn_workspace(ctypes.byref(good()), op, ctypes.byref(need)) == 0
    assert lib.fmha_attn_workspace(ctypes.byref(good()), 3, ctypes.byref(need)) == 1
    assert lib.fmha_attn_workspace(None, 0, ctypes.byref(need)) == 1
    assert lib.fmha_attn_workspace(ctypes.byref(change(K_dim=80)), 0, ctypes.byref(need)) == 1


def test_python_entries_refuse_cpu_tensors():
    import fmha_bwd_b200 as F

    x = torch.zeros(1, 2, 8, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        F.cross_attn_fwd(x, x, x)
    with pytest.raises(ValueError):
        F.cross_attn_bwd(x, x, x, x, torch.zeros(1, 2, 8), x)
    with pytest.raises(ValueError):
        F.prefix_attn(x, x, x, x, x)


def test_argument_block_layout():
    import fmha_bwd_b200 as F

    assert F._ATTN.size == ctypes.sizeof(Attn)


# ------------------------------------------------- the reference, on the CPU
def _case(dtype=torch.float64):
    g = torch.Generator().manual_seed(1)
    Q, K, V, dO = (torch.randn(2, h, n, 64, generator=g).to(dtype) for h, n in ((4, 9), (2, 13), (2, 13), (4, 9)))
    return Q, K, V, dO, torch.tensor([13, 6])


def test_reference_backward_is_the_gradient_of_its_forward():
    Q, K, V, dO, n = _case()
    leaves = [t.clone().requires_grad_() for t in (Q, K, V)]
    O = R.forward(*leaves, n, 0.125)[0]
    want = torch.autograd.grad((O * dO).sum(), leaves)
    O, LSE, _, _ = R.forward(Q, K, V, n, 0.125)
    got, _ = R.backward(Q, K, V, O, LSE, dO, n, 0.125)
    for a, b in zip(got, want):
        assert torch.allclose(a, b, rtol=1e-10, atol=1e-12)


def test_reference_prefix_is_the_forward_over_both():
    Q, K, V, _, n = _case()
    O, LSE, _, _ = R.prefix(Q[:, :, :1], K[:1, :, :5], V[:1, :, :5], K[:, :, 5:], V[:, :, 5:], None, n - 5, 0.125)
    k, v = (torch.cat([t[:1, :, :5].expand(2, -1, -1, -1), t[:, :, 5:]], 2) for t in (K, V))
    want, lse, _, _ = R.forward(Q[:, :, :1], k, v, n, 0.125)
    assert torch.allclose(O, want) and torch.allclose(LSE, lse)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_bounds_notice_planted_mistakes(dtype):
    """A right answer, rounded, passes; one key too many, a head read from its
    neighbour and a forgotten scale do not."""
    Q, K, V, dO, n = _case(dtype)
    O, LSE, bound, _ = R.forward(Q, K, V, n, 0.125)
    R.check("O", O.to(dtype), O, bound)
    for wrong in (R.forward(Q, K, V, n + torch.tensor([0, 1]), 0.125)[0],
                  R.forward(Q, K.flip(1), V.flip(1), n, 0.125)[0], R.forward(Q, K, V, n, 0.126)[0]):
        with pytest.raises(AssertionError):
            R.check("O", wrong.to(dtype), O, bound)
    outs, bounds = R.backward(Q, K, V, O.to(dtype), LSE.float(), dO, n, 0.125)
    for x, b in zip(outs, bounds):
        R.check("gradient", x.to(dtype), x, b)
        with pytest.raises(AssertionError):
            R.check("gradient", (x * 1.05).to(dtype), x, b)
