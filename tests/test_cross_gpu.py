"""Cross attention to an encoder's states (forward, backward, single tokens)
and attention behind a shared prefix on the GPU, through the public Python
entries, against 64-bit forms with counted roundings (attn_reference.py)."""
from __future__ import annotations

import math

import pytest
import torch

import attn_reference as R

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
NAN = float("nan")


@pytest.fixture(scope="module")
def F():
    import fmha_bwd_b200 as F

    F.load_library(torch.bfloat16)
    F.load_library(torch.float16)
    return F


def tensor(g, B, H, n, d, dtype, layout="bnhd", std=1.0):
    x = (torch.randn(B, H, n, d, generator=g, device="cuda") * std).to(dtype)
    if layout == "bhnd":
        return x
    if layout == "bnhd":  # as a projection leaves it
        return x.transpose(1, 2).contiguous().transpose(1, 2)
    # rows, heads and batches apart from one another
    big = torch.full((B, H + 1, n + 3, d + 24), NAN, device="cuda", dtype=dtype)
    big[:, :H, :n, 8:8 + d] = x
    return big[:, :H, :n, 8:8 + d]


def spoil(t, lens):
    """NaN and infinities in the rows that do not count, as an allocator leaves them."""
    if lens is None:
        return
    for b, n in enumerate(lens.tolist()):
        t[b, :, max(0, n):] = NAN
        t[b, :, max(0, n)::2, ::2] = float("inf")


def make(B, Hq, Hkv, M, N, d, name, lens=None, layout="bnhd", std=1.0, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    Q = tensor(g, B, Hq, M, d, DT[name], layout, std)
    K = tensor(g, B, Hkv, N, d, DT[name], layout, std)
    V = tensor(g, B, Hkv, N, d, DT[name], layout)
    n = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    spoil(K, n)
    spoil(V, n)
    return Q, K, V, n


# (B, Hq, Hkv, M, N, d, dtype, lens, layout, std of Q and K)
SHAPES = [
    (1, 1, 1, 1, 1, 64, "bf16", None, "bhnd", 1),
    (1, 1, 1, 1, 1, 128, "fp16", [0], "bhnd", 1),
    (2, 2, 1, 1, 7, 64, "fp16", [3, 7], "bnhd", 1),
    (3, 4, 4, 5, 33, 128, "bf16", [0, 33, 1], "bnhd", 1),
    (1, 3, 3, 127, 64, 64, "bf16", None, "bnhd", 1),
    (2, 2, 2, 128, 128, 128, "bf16", None, "bhnd", 1),
    (2, 2, 2, 129, 129, 128, "fp16", [128, 129], "bnhd", 1),
    (2, 6, 2, 300, 200, 64, "fp16", [17, 200], "apart", 1),
    (1, 8, 2, 16, 520, 128, "bf16", [511], "bnhd", 1),
    (2, 4, 1, 257, 385, 128, "bf16", [256, 384], "apart", 1),
    (4, 4, 2, 70, 777, 64, "bf16", [0, 777, 640, -5], "bnhd", 1),
    (1, 2, 2, 640, 1024, 64, "fp16", [1000], "bnhd", 1),
    (1, 2, 2, 200, 300, 128, "bf16", None, "bnhd", 3),       # sharp: scores in the tens
    (2, 2, 2, 130, 400, 64, "fp16", [399, 400], "bnhd", 4),
    (1, 32, 4, 3, 100, 128, "fp16", None, "bnhd", 1),        # 24 rows a kv head
    (1, 1, 1, 1100, 40, 128, "bf16", [40], "bhnd", 1),
    (5, 40, 8, 1, 1500, 128, "bf16", [1, 1500, 700, 16, 0], "bnhd", 1),
    (2, 71, 1, 1, 130, 64, "fp16", [129, 5], "bnhd", 1),
    (1, 2, 1, 1, 20000, 64, "bf16", [19999], "bhnd", 1),
    (300, 1, 1, 1, 20, 64, "fp16", None, "bnhd", 1),
    (1, 6, 3, 64, 4000, 128, "fp16", [3999], "bnhd", 1),     # few rows, many keys
    (2, 6, 3, 40, 2100, 64, "fp16", [2100, 0], "bnhd", 1),
    (1, 2, 2, 130, 4200, 128, "bf16", [4199], "bnhd", 1),
    (1, 4, 1, 700, 1000, 64, "bf16", None, "bnhd", 1),       # few items of many steps, both ways round
    (1, 16, 2, 600, 77, 128, "bf16", [70], "bnhd", 1),
    (3, 8, 8, 200, 900, 64, "fp16", [900, 3, 0], "apart", 1),
    (1, 32, 4, 300, 900, 128, "bf16", None, "bnhd", 1),
]


@pytest.mark.parametrize("B,Hq,Hkv,M,N,d,name,lens,layout,std", SHAPES)
def test_forward(F, B, Hq, Hkv, M, N, d, name, lens, layout, std):
    Q, K, V, n = make(B, Hq, Hkv, M, N, d, name, lens, layout, std)
    O, LSE = F.cross_attn_fwd(Q, K, V, n)
    ref, lse, bound, lse_bound = R.forward(Q, K, V, n, d ** -0.5)
    R.check("O", O, ref, bound)
    R.check("LSE", LSE, lse, lse_bound)
    assert O.dtype == Q.dtype and LSE.dtype == torch.float32


# single tokens over caches large enough to be read as one stream: items that do
# and do not divide among a block's warps, 8 and 16 rows, empty and short entries
# between long ones, several entries to a block and several blocks to an entry
LONG = [
    (3, 20, 4, 1, 16400, 128, "bf16", [16400, 0, 9000]),
    (5, 10, 10, 1, 8200, 64, "fp16", [8200, 1, 0, 4097, 8191]),
    (2, 55, 5, 1, 25000, 128, "fp16", [24999, 16]),
    (1, 13, 13, 1, 40000, 64, "bf16", None),
    (40, 7, 1, 2, 5000, 128, "bf16", [5000 - 131 * i for i in range(38)] + [0, 5000]),
    (2, 11, 11, 1, 9000, 128, "fp16", [3, 17]),
    (1, 1, 1, 1, 200000, 128, "bf16", [199999]),
]


@pytest.mark.parametrize("B,Hq,Hkv,M,N,d,name,lens", LONG)
def test_long_caches(F, B, Hq, Hkv, M, N, d, name, lens):
    Q, K, V, n = make(B, Hq, Hkv, M, N, d, name, lens, seed=18)
    O, LSE = F.cross_attn_fwd(Q, K, V, n)
    ref, lse, bound, lse_bound = R.forward(Q, K, V, n, d ** -0.5)
    R.check("O", O, ref, bound)
    R.check("LSE", LSE, lse, lse_bound)
    again = F.cross_attn_fwd(Q, K, V, n)
    assert torch.equal(O, again[0]) and torch.equal(LSE, again[1])


def saved(Q, K, V, n, scale):
    """O and LSE of a right forward, rounded to their types."""
    ref, lse, _, _ = R.forward(Q, K, V, n, scale)
    return ref.to(Q.dtype), lse.float()


@pytest.mark.parametrize("B,Hq,Hkv,M,N,d,name,lens,layout,std", SHAPES)
def test_backward(F, B, Hq, Hkv, M, N, d, name, lens, layout, std):
    Q, K, V, n = make(B, Hq, Hkv, M, N, d, name, lens, layout, std, seed=2)
    dO = tensor(torch.Generator(device="cuda").manual_seed(3), B, Hq, M, d, DT[name], layout, 0.1)
    O, LSE = saved(Q, K, V, n, d ** -0.5)
    got = F.cross_attn_bwd(Q, K, V, O, LSE, dO, n)
    outs, bounds = R.backward(Q, K, V, O, LSE, dO, n, d ** -0.5)
    for label, x, ref, bound in zip(("dQ", "dK", "dV"), got, outs, bounds):
        R.check(label, x, ref, bound)
    if n is not None:
        for b, count in enumerate(n.clamp(0, N).tolist()):
            assert not got[1][b, :, count:].any() and not got[2][b, :, count:].any()


@pytest.mark.parametrize("std", [1e-4, 300.0])
def test_backward_of_small_and_large_gradients(F, std):
    """fp16 gradients near the ends of the type's range keep their relative accuracy."""
    Q, K, V, n = make(2, 4, 2, 150, 260, 64, "fp16", [260, 130], seed=4)
    dO = tensor(torch.Generator(device="cuda").manual_seed(5), 2, 4, 150, 64, torch.float16, std=std)
    O, LSE = saved(Q, K, V, n, 0.125)
    got = F.cross_attn_bwd(Q, K, V, O, LSE, dO, n)
    outs, bounds = R.backward(Q, K, V, O, LSE, dO, n, 0.125)
    for label, x, ref, bound in zip(("dQ", "dK", "dV"), got, outs, bounds):
        R.check(label, x, ref, bound)


@pytest.mark.parametrize("name,d", [("bf16", 128), ("fp16", 64)])
def test_backward_against_differences(F, name, d):
    """dQ, dK, dV against central differences of the 64-bit loss sum(O * dO)."""
    scale, h = d ** -0.5, 1e-4
    Q, K, V, n = make(1, 2, 1, 40, 70, d, name, [65], "bhnd", seed=6)
    K[:, :, 65:] = 0  # the differences below go through the plain form's masks as well
    V[:, :, 65:] = 0
    dO = tensor(torch.Generator(device="cuda").manual_seed(7), 1, 2, 40, d, DT[name])
    O, LSE = saved(Q, K, V, n, scale)
    got = F.cross_attn_bwd(Q, K, V, O, LSE, dO, n, scale)
    _, bounds = R.backward(Q, K, V, O, LSE, dO, n, scale, delta_err=R.roundings(DT[name])[0])

    def loss(q, k, v):
        return (R.forward(q, k, v, n, scale)[0] * dO.double()).sum()

    x = [t.double() for t in (Q, K, V)]
    for i, label in enumerate(("dQ", "dK", "dV")):
        for seed in range(3):
            U = torch.randn(x[i].shape, dtype=torch.float64, device="cuda",
                            generator=torch.Generator(device="cuda").manual_seed(seed))
            up, down = ([t + sign * h * U if j == i else t for j, t in enumerate(x)] for sign in (1, -1))
            slope = (loss(*up) - loss(*down)) / (2 * h)
            # the bounds along U, LSE's rounding (2^-24 |LSE| on every weight), and
            # h^2 / 6 times a third derivative, which scores of size 1 keep under 1e3 |slope terms|
            tol = (bounds[i] * U.abs()).sum() + 1e-5 * (got[i].double() * U).abs().sum()
            assert abs((got[i].double() * U).sum() - slope) <= tol, label


@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("M", [1, 130])
def test_nan_is_not_lost(F, name, M):
    """A NaN in one query row: that row of O, LSE and dQ, and what sums over it."""
    Q, K, V, n = make(1, 2, 1, M, 150, 64, name, [140], seed=15)
    dO = tensor(torch.Generator(device="cuda").manual_seed(16), 1, 2, M, 64, Q.dtype)
    Q[0, 0, M // 2, 3] = math.nan
    O, LSE = F.cross_attn_fwd(Q, K, V, n)
    dQ, dK, dV = F.cross_attn_bwd(Q, K, V, O, LSE, dO, n)
    hit = torch.zeros(1, 2, M, dtype=torch.bool, device="cuda")
    hit[0, 0, M // 2] = True
    assert torch.equal(LSE.isnan(), hit)
    for x in (O, dQ):
        assert torch.equal(x.isfinite().all(-1), ~hit) and torch.equal(x.isfinite().any(-1), ~hit)
    for x in (dK, dV):
        assert not x[:, :, :140].isfinite().any() and (x[:, :, 140:] == 0).all()


@pytest.mark.parametrize("d,name", [(64, "fp16"), (128, "bf16")])
def test_runs_of_entries_without_keys(F, d, name):
    """More in a row than a CTA holds units of work ahead, between others."""
    B, H, M, N = 120, 8, 20, 140
    Q, K, V, n = make(B, H, H, M, N, d, name, [140] * 19 + [0] * 82 + [77] * 19, seed=17)
    O, LSE = F.cross_attn_fwd(Q, K, V, n)
    ref, lse, bound, lse_bound = R.forward(Q, K, V, n, d ** -0.5)
    R.check("O", O, ref, bound)
    R.check("LSE", LSE, lse, lse_bound)
    dO = tensor(torch.Generator(device="cuda").manual_seed(18), B, H, M, d, Q.dtype)
    grads = F.cross_attn_bwd(Q, K, V, O, LSE, dO, n)
    for label, x, ref, bound in zip(("dQ", "dK", "dV"), grads, *R.backward(Q, K, V, O, LSE, dO, n, d ** -0.5)):
        R.check(label, x, ref, bound)
    _, Kp, Vp, np_ = make(B, H, H, 1, 130, d, name, [0] * 30 + [130] + [0] * 85 + [9] * 4, seed=19)
    O, LSE = F.prefix_attn(Q, Kp, Vp, K, V, np_, n)
    ref, lse, bound, lse_bound = R.prefix(Q, Kp, Vp, K, V, np_, n, d ** -0.5)
    R.check("O", O, ref, bound)
    R.check("LSE", LSE, lse, lse_bound)


PREFIXES = [
    # (P, S, Hq, Hkv, M, N, Np, d, dtype, lens, prefix_lens, layout)
    (1, 1, 1, 1, 1, 1, 1, 64, "bf16", None, None, "bhnd"),
    (1, 4, 2, 2, 1, 20, 100, 64, "fp16", [0, 1, 20, 7], None, "bnhd"),
    (2, 3, 8, 2, 1, 33, 257, 128, "bf16", [33, 0, 5, 16, 17, 32], [129, 0], "bnhd"),
    (1, 2, 6, 1, 3, 40, 300, 64, "fp16", [2, 40], [299], "apart"),    # the first token of row 0 has no own key
    (1, 70, 4, 2, 1, 9, 500, 128, "bf16", None, None, "bnhd"),        # 140 rows a kv head: over one tile
    (3, 5, 16, 4, 5, 64, 130, 128, "fp16", None, [128, 1, 130], "bnhd"),
    (1, 1, 48, 1, 4, 50, 700, 64, "bf16", [50], None, "bnhd"),        # 192 rows of one entry
    (1, 2, 2, 1, 130, 150, 200, 128, "bf16", [130, 150], None, "bnhd"),
    (2, 1, 4, 4, 1, 2000, 3000, 64, "fp16", [2000, 3], [2999, 64], "bnhd"),
    (1, 2, 2, 2, 1, 30, 20, 64, "bf16", [0, 30], [0], "bhnd"),        # entry 0 has no key at all
    (1, 2, 4, 2, 300, 700, 260, 128, "bf16", [700, 120], None, "bnhd"),       # own tokens over several tiles
    (2, 1, 3, 1, 150, 1000, 1100, 64, "fp16", [1000, 149], [0, 1100], "bnhd"),
    (1, 2, 1, 1, 1, 20, 20000, 64, "bf16", None, None, "bnhd"),
    (1, 2, 1, 1, 1, 20, 30000, 64, "bf16", None, None, "bnhd"),       # 117 parts of the prefix
    (1, 3, 4, 2, 2, 40, 20500, 128, "fp16", [40, 0, 1], None, "bnhd"),        # parts, and own keys or none
    (2, 40, 8, 4, 1, 100, 513, 128, "bf16", None, [513, 100], "bnhd"),
    (8, 1, 16, 4, 2, 300, 500, 64, "fp16", [300, 1, 2, 0, 17, 16, 299, 100], None, "bnhd"),   # nothing shared
    (3, 2, 4, 4, 1, 17, 33, 128, "fp16", [0, 17, 16, 1, 0, 3], [33, 0, 16], "apart"),
    (2, 40, 32, 4, 3, 100, 513, 128, "bf16", None, [513, 200], "bnhd"),       # more items than SMs
]


@pytest.mark.parametrize("P,S,Hq,Hkv,M,N,Np,d,name,lens,prefix_lens,layout", PREFIXES)
def test_prefix(F, P, S, Hq, Hkv, M, N, Np, d, name, lens, prefix_lens, layout):
    Q, K, V, n = make(P * S, Hq, Hkv, M, N, d, name, lens, layout, seed=8)
    _, Kp, Vp, np_ = make(P, Hkv, Hkv, 1, Np, d, name, prefix_lens, layout, seed=9)
    O, LSE = F.prefix_attn(Q, Kp, Vp, K, V, np_, n)
    ref, lse, bound, lse_bound = R.prefix(Q, Kp, Vp, K, V, np_, n, d ** -0.5)
    R.check("O", O, ref, bound)
    R.check("LSE", LSE, lse, lse_bound)


def test_prefix_of_different_size_scores(F):
    """Prefix and own cache whose largest scores lie far apart, both ways round."""
    for own, ahead in ((6.0, 0.1), (0.1, 6.0)):
        g = torch.Generator(device="cuda").manual_seed(10)
        Q = tensor(g, 4, 4, 1, 64, torch.bfloat16)
        K, V = tensor(g, 4, 2, 50, 64, torch.bfloat16, std=own), tensor(g, 4, 2, 50, 64, torch.bfloat16)
        Kp, Vp = tensor(g, 1, 2, 400, 64, torch.bfloat16, std=ahead), tensor(g, 1, 2, 400, 64, torch.bfloat16)
        O, LSE = F.prefix_attn(Q, Kp, Vp, K, V)
        ref, lse, bound, lse_bound = R.prefix(Q, Kp, Vp, K, V, None, None, 0.125)
        R.check("O", O, ref, bound)
        R.check("LSE", LSE, lse, lse_bound)


def test_training_step_and_generation_together(F):
    """A run as it would be used: forward and backward of one step feed each
    other, the trained states are then read token by token, and samples of the
    same prompt share it."""
    B, Hq, Hkv, M, N, d = 2, 4, 2, 200, 333, 128
    Q, K, V, n = make(B, Hq, Hkv, M, N, d, "bf16", [333, 100], seed=11)
    dO = tensor(torch.Generator(device="cuda").manual_seed(12), B, Hq, M, d, torch.bfloat16)
    O, LSE = F.cross_attn_fwd(Q, K, V, n, sync=False)
    grads = F.cross_attn_bwd(Q, K, V, O, LSE, dO, n, sync=False)
    outs, bounds = R.backward(Q, K, V, O, LSE, dO, n, d ** -0.5)
    for label, x, ref, bound in zip(("dQ", "dK", "dV"), grads, outs, bounds):
        R.check(label, x, ref, bound)
    # each token alone gives its row of the whole
    ref, lse, bound, lse_bound = R.forward(Q, K, V, n, d ** -0.5)
    for m in (0, 57, 199):
        o, l = F.cross_attn_fwd(Q[:, :, m:m + 1], K, V, n)
        R.check("O", o, ref[:, :, m:m + 1], bound[:, :, m:m + 1])
        R.check("LSE", l, lse[:, :, m:m + 1], lse_bound[:, :, m:m + 1])
    # a prompt of 300 states shared by three samples with 33 of their own
    k1, v1 = K[:1, :, :300], V[:1, :, :300]
    k2, v2 = K[:1, :, 300:].repeat(3, 1, 1, 1), V[:1, :, 300:].repeat(3, 1, 1, 1)
    q = Q[:1, :, :1].repeat(3, 1, 1, 1)
    o, l = F.prefix_attn(q, k1, v1, k2, v2)
    for s in range(3):
        R.check("O", o[s:s + 1], ref[:1, :, :1], bound[:1, :, :1])
        R.check("LSE", l[s:s + 1], lse[:1, :, :1], lse_bound[:1, :, :1])


def test_gradient_feeds_the_existing_backward(F):
    """cross_attn_fwd's O and LSE are what fmha_bwd_lse takes."""
    H, M, N, d = 3, 200, 264, 64
    Q, K, V, _ = make(1, H, H, M, N, d, "bf16", None, "bhnd", seed=13)
    dO = tensor(torch.Generator(device="cuda").manual_seed(14), 1, H, M, d, torch.bfloat16, "bhnd")
    O, LSE = F.cross_attn_fwd(Q, K, V)
    a = F.fmha_bwd_lse(Q[0], K[0], V[0], O[0].contiguous(), dO[0], LSE[0], d ** -0.5)
    outs, bounds = R.backward(Q, K, V, O, LSE, dO, None, d ** -0.5)
    for label, x, ref, bound in zip(("dQ", "dK", "dV"), a, outs, bounds):
        R.check(label, x[None], ref, bound)


def all_calls(F, seed=15):
    """Each entry once at a shape that takes each of its kernels: (call, out shapes)."""
    Q, K, V, n = make(2, 4, 2, 200, 300, 64, "bf16", [300, 77], seed=seed)
    dO = tensor(torch.Generator(device="cuda").manual_seed(seed), 2, 4, 200, 64, torch.bfloat16)
    O, LSE = saved(Q, K, V, n, 0.125)
    q = Q[:, :, :1].contiguous()
    Kp, Vp = K[:1, :, :77], V[:1, :, :77]
    kn = torch.tensor([10, 33], dtype=torch.int32, device="cuda")
    return {
        "fwd": lambda **kw: F.cross_attn_fwd(Q, K, V, n, **kw),
        "few": lambda **kw: F.cross_attn_fwd(Q[:, :, :30], K, V, n, **kw),
        "decode": lambda **kw: F.cross_attn_fwd(q, K, V, n, **kw),
        "bwd": lambda **kw: F.cross_attn_bwd(Q, K, V, O, LSE, dO, n, **kw),
        "prefix": lambda **kw: F.prefix_attn(q, Kp, Vp, K, V, None, kn, **kw),
    }, (Q, K, V, dO)


@pytest.mark.parametrize("which", ["fwd", "few", "decode", "bwd", "prefix"])
def test_same_bits_again(F, which):
    calls, _ = all_calls(F)
    a, b = calls[which](), calls[which]()
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("which", ["fwd", "few", "decode", "bwd", "prefix"])
def test_given_outputs_and_what_lies_around_them(F, which):
    """Strided outputs inside a larger buffer: the elements between stay as they were."""
    calls, _ = all_calls(F)
    want = calls[which]()
    outs, bigs = [], []
    for t in want:
        if t.dim() == 3:
            outs.append(torch.full_like(t, 7.0))
            continue
        B, H, n, d = t.shape
        big = torch.full((B + 1, n + 2, H + 1, d + 8), 7.0, dtype=t.dtype, device="cuda")
        bigs.append((big, (slice(0, B), slice(1, n + 1), slice(0, H), slice(8, 8 + d))))
        outs.append(big[bigs[-1][1]].transpose(1, 2))
    got = calls[which](out=tuple(outs))
    for x, y, o in zip(got, want, outs):
        assert x.data_ptr() == o.data_ptr() and torch.equal(x, y)
    for big, inner in bigs:
        big[inner] = 7.0
        assert bool((big == 7.0).all())


@pytest.mark.parametrize("which", ["fwd", "few", "decode", "bwd", "prefix"])
def test_on_another_stream(F, which):
    calls, _ = all_calls(F)
    want = calls[which]()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = calls[which](stream=side, sync=False)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_two_streams_at_once(F):
    """Calls that overlap on the GPU share nothing."""
    calls, _ = all_calls(F)
    want = {k: f() for k, f in calls.items()}
    sides = [torch.cuda.Stream() for _ in range(3)]
    for s in sides:
        s.wait_stream(torch.cuda.current_stream())
    got = [(k, f(stream=s, sync=False)) for _ in range(4) for s in sides for k, f in calls.items()]
    torch.cuda.synchronize()
    for k, outs in got:
        assert all(torch.equal(x, y) for x, y in zip(outs, want[k])), k


def test_captured_graphs_replay_with_new_inputs(F):
    """Two graphs, one of them holding every entry, replayed alternately after
    the inputs change in place; an eager call between them disturbs neither."""
    calls, inputs = all_calls(F, seed=16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, held = [], []
    with torch.cuda.stream(side):
        for f in calls.values():
            f(sync=False)
        for which in (list(calls), ["bwd", "prefix"]):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                held.append({k: calls[k](sync=False) for k in which})
            graphs.append(g)
    torch.cuda.synchronize()
    for step in range(2):
        for t in inputs:
            t.mul_(1.0 if step == 0 else 0.5)
        want = {k: [x.clone() for x in f()] for k, f in calls.items()}
        for g in graphs:
            g.replay()
        calls["bwd"]()
        for g in reversed(graphs):
            g.replay()
        torch.cuda.synchronize()
        for outs in held:
            for k, xs in outs.items():
                assert all(torch.equal(x, y) for x, y in zip(xs, want[k])), k


@pytest.mark.parametrize("M,Np", [(1, 20600), (20, 700)])
def test_prefix_in_parts_on_streams_and_in_graphs(F, M, Np):
    """The form of three launches that overlap, for single tokens and for more."""
    Q, K, V, n = make(6, 8, 2, M, 70, 64, "bf16", [70, 0, 33, 1, 70, 16], seed=20)
    _, Kp, Vp, np_ = make(2, 2, 2, 1, Np, 64, "bf16", [Np, 500], seed=21)
    call = lambda **kw: F.prefix_attn(Q, Kp, Vp, K, V, np_, n, **kw)  # noqa: E731
    want = call()
    ref, lse, bound, lse_bound = R.prefix(Q, Kp, Vp, K, V, np_, n, 0.125)
    R.check("O", want[0], ref, bound)
    R.check("LSE", want[1], lse, lse_bound)
    sides = [torch.cuda.Stream() for _ in range(3)]
    for s in sides:
        s.wait_stream(torch.cuda.current_stream())
    got = [call(stream=s, sync=False) for _ in range(8) for s in sides]
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for outs in got for x, y in zip(outs, want))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=sides[0]):
        held = [call(sync=False) for _ in range(3)]
    for factor in (1.0, 0.5):
        for t in (Q, K, Vp):
            t.mul_(factor)
        want = call()
        g.replay()
        other = call(sync=False)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for outs in (*held, other) for x, y in zip(outs, want))


def test_refusals_on_the_device(F):
    Q, K, V, n = make(2, 4, 2, 8, 16, 64, "bf16", [16, 3])
    dO, (O, LSE) = torch.ones_like(Q), saved(Q, K, V, n, 0.125)
    fwd = F.cross_attn_fwd
    with pytest.raises(TypeError):
        fwd(Q.float(), K.float(), V.float())
    with pytest.raises(TypeError):
        fwd(Q, K.half(), V)
    with pytest.raises(ValueError):
        fwd(Q, K[:1], V[:1])                          # another batch
    with pytest.raises(ValueError):
        fwd(Q, K, V[:, :, :8])                        # another length
    with pytest.raises(ValueError):
        fwd(Q[:, :3], K, V)                           # 3 heads on 2
    with pytest.raises(ValueError):
        fwd(Q.transpose(2, 3).contiguous().transpose(2, 3), K, V)  # stride along d
    with pytest.raises(ValueError):
        fwd(Q, K, V, n.long())
    with pytest.raises(ValueError):
        fwd(Q, K, V, n.cpu())
    with pytest.raises(ValueError):
        fwd(Q, K, V, n[:1])
    for scale in (0.0, -1.0, NAN, math.inf):
        with pytest.raises(ValueError):
            fwd(Q, K, V, n, scale)
    with pytest.raises(ValueError):
        F.cross_attn_bwd(Q, K, V, O, LSE.double(), dO)
    with pytest.raises(ValueError):
        F.cross_attn_bwd(Q, K, V, O[:, :, :4], LSE, dO)
    with pytest.raises(ValueError):
        F.prefix_attn(Q, K[:, :1], V[:, :1], K, V)
    with pytest.raises(ValueError):
        F.prefix_attn(Q[:1], K, V, K[:1], V[:1])      # one entry, two prefixes
    with pytest.raises(F.FmhaBwdError):
        fwd(Q[..., :32].contiguous(), K[..., :32].contiguous(), V[..., :32].contiguous())
    with pytest.raises(F.FmhaBwdError):
        fwd(Q, K[:1].expand(2, -1, -1, -1), V)        # expanded
    with pytest.raises(F.FmhaBwdError):
        fwd(Q, K, V, out=(O[:1].expand(2, -1, -1, -1), LSE))
    with pytest.raises(F.FmhaBwdError):
        fwd(Q, K, V, out=(Q, LSE))                    # over an input
    buf = torch.zeros(2 * 4 * 8 * 64 + 8, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(F.FmhaBwdError):
        fwd(buf[4:-4].view(2, 4, 8, 64), K, V)        # 8-byte aligned
    with pytest.raises(F.FmhaBwdError):
        fwd(torch.zeros(2, 4, 8, 68, dtype=torch.bfloat16, device="cuda")[..., :64], K, V)  # rows 136 bytes apart
    # and the next right call is not disturbed
    R.check("O", fwd(Q, K, V, n)[0], *R.forward(Q, K, V, n, 0.125)[0::2])


def test_an_offset_past_32_bits(F):
    """A batch entry whose states start over 2^32 elements into the cache."""
    rows = (1 << 32) // (8 * 64) + 64
    big = torch.empty(2, rows, 8, 64, dtype=torch.bfloat16, device="cuda")  # 8.6 GB
    g = torch.Generator(device="cuda").manual_seed(17)
    K, V = (big[:, o:o + 150].transpose(1, 2) for o in (0, 200))
    for t in (K, V):
        t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
    n = torch.tensor([150, 140], dtype=torch.int32, device="cuda")
    for M in (1, 40):
        Q = tensor(g, 2, 8, M, 64, torch.bfloat16)
        O, LSE = F.cross_attn_fwd(Q, K, V, n)
        ref, lse, bound, lse_bound = R.forward(Q, K, V, n, 0.125)
        R.check("O", O, ref, bound)
        R.check("LSE", LSE, lse, lse_bound)
        dO = tensor(g, 2, 8, M, 64, torch.bfloat16)
        got = F.cross_attn_bwd(Q, K, V, O, LSE, dO, n, out=(torch.empty_like(Q), torch.empty(2, 8, 150, 64, dtype=Q.dtype, device="cuda"), torch.empty(2, 8, 150, 64, dtype=Q.dtype, device="cuda")))
        outs, bounds = R.backward(Q, K, V, O, LSE, dO, n, 0.125)
        for label, x, r, b in zip(("dQ", "dK", "dV"), got, outs, bounds):
            R.check(label, x, r, b)
