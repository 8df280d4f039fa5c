"""Edges of the attention entries on the GPU: inputs at which a kernel of this
kind goes wrong without its ordinary cases showing it. References and bounds as
in test_cross_gpu.py."""
from __future__ import annotations

import math

import pytest
import torch

import attn_reference as R
from test_cross_gpu import DT, F, NAN, make, saved, tensor  # noqa: F401 (F is a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name,d", [("bf16", 128), ("fp16", 64)])
def test_many_ends_of_entries_in_one_stream(F, name, d):
    """Every entry ends inside a tile of 16 keys, with NaN behind, and the same
    shared memory takes further tiles."""
    B, N = 24, 8200
    lens = [N - 1 - 16 * 13 * b if b % 3 else 16 * b + 5 for b in range(B)]
    assert all(n % 16 for n in lens)
    Q, K, V, n = make(B, 8, 4, 1, N, d, name, lens, seed=31)
    O, LSE = F.cross_attn_fwd(Q, K, V, n)
    ref, lse, bound, lse_bound = R.forward(Q, K, V, n, d ** -0.5)
    R.check("O", O, ref, bound)
    R.check("LSE", LSE, lse, lse_bound)
    for _ in range(20):
        again = F.cross_attn_fwd(Q, K, V, n)
        assert torch.equal(O, again[0]) and torch.equal(LSE, again[1])


# ----------------------------------------------------- gradients of unlike sizes
def group_gradients(Q, K, V, O, LSE, dO, n, scale):
    """R.backward's gradients and bounds of one entry's kv head ([G, M, d], [n, d]
    of its valid keys), with fp16's dS held times the power of two that this
    head's largest finite |dO| and |V| allow: below 2^e and 2^e' they leave
    2^(14 - log2 d - e - e') or more, so a half-step of 2^-25 stands for at most
    2^-25 2^-14 d (2 max|dO|) (2 max|V|) = d 2^-37 max|dO| max|V|."""
    G, M, d = Q.shape
    u, sub = R.roundings(Q.dtype)
    q, k, v, o, do = Q.double(), K[:n].double(), V[:n].double(), O.double(), dO.double()
    S = scale * q @ k.T
    err = (d + 4) * R.E * scale * (q.abs() @ k.abs().T) + 4 * R.E * S.abs()
    lse = LSE.double()[..., None]
    P = torch.exp(S - lse)
    rel_p = 1.01 * err + 2.0 ** -21 + 4 * R.E * lse.abs()
    dP, D = do @ v.T, (do * o).sum(-1, keepdim=True)
    dS = P * (dP - D)
    acc = (d + 4) * R.E
    e_s = P * acc * (do.abs() @ v.abs().T + (do.abs() * o.abs()).sum(-1, keepdim=True)) + (u + rel_p + 4 * R.E) * dS.abs()
    if Q.dtype == torch.float16:
        e_s = e_s + d * 2.0 ** -37 * float(do[do.isfinite()].abs().max()) * float(v.abs().max())
    many = (G * M + 8) * R.E
    dQ, bQ = scale * dS @ k, scale * (e_s + (n + 8) * R.E * dS.abs()) @ k.abs()
    dK = (scale * dS.mT @ q).sum(0)
    bK = (scale * (e_s + many * dS.abs()).mT @ q.abs()).sum(0)
    dV = (P.mT @ do).sum(0)
    bV = (((u + rel_p + many) * P + sub * 2.0 ** -10).mT @ do.abs()).sum(0)
    return (dQ, dK, dV), tuple((1 + u) * b + u * x.abs() + sub for b, x in zip((bQ, bK, bV), (dQ, dK, dV)))


# sizes of dO and of V, for each entry and each of its two kv heads
UNLIKE = {
    "entries": ([[300, 300], [0.02, 0.02], [300, 300]], [[16, 16], [1, 1], [16, 16]]),
    "heads": ([[300, 0.02], [0.02, 300], [1e-3, 1]], [[16, 1], [0.05, 16], [1, 1]]),
    "tiny": ([[1, 1e-4], [1e-4, 1e-4], [1, 1]], [[1, 1], [1, 0.02], [1, 1]]),
}


@pytest.mark.parametrize("M,N", [(40, 77), (300, 777)])
@pytest.mark.parametrize("sizes", sorted(UNLIKE))
@pytest.mark.parametrize("name,d", [("fp16", 64), ("fp16", 128), ("bf16", 64)])
@pytest.mark.parametrize("wild", [None, "entry without keys", "one row"])
def test_gradients_of_entries_and_heads_of_unlike_sizes(F, M, N, sizes, name, d, wild):
    """Each head's gradients keep their own precision whatever the others hold:
    sizes 1e4 and more apart, an entry without keys whose dO is infinite, and one
    row of dO that is (its own head's dQ is right in the other rows)."""
    lens = [N, N - 20, 0]
    Q, K, V, n = make(3, 4, 2, M, N, d, name, lens, seed=41)
    dO = tensor(torch.Generator(device="cuda").manual_seed(42), 3, 4, M, d, DT[name])
    of_do, of_v = (torch.tensor(x, device="cuda")[:, :, None, None] for x in UNLIKE[sizes])
    dO = (dO.float() * of_do.repeat_interleave(2, 1)).to(dO.dtype)
    V = (V.float() * of_v).to(V.dtype)
    O, LSE = saved(Q, K, V, n, d ** -0.5)
    odd = None
    if wild == "entry without keys":
        dO[2] = float("inf")
    if wild == "one row":
        odd = (1, 2, M // 2)
        dO[odd] = float("inf")
    got = F.cross_attn_bwd(Q, K, V, O, LSE, dO, n)
    for b in range(2):
        for h in range(2):
            hs = slice(2 * h, 2 * h + 2)
            do = dO[b, hs].clone()
            alone = odd is None or (b, h) != (odd[0], odd[1] // 2)
            if not alone:  # its row's sums are not finite; the other rows do not know of it
                do[odd[1] % 2, odd[2]] = 0
            outs, bounds = group_gradients(Q[b, hs], K[b, h], V[b, h], O[b, hs], LSE[b, hs], do, lens[b], d ** -0.5)
            x = got[0][b, hs].clone()
            if not alone:
                x[odd[1] % 2, odd[2]] = 0
            R.check(f"dQ of {b}, {h}", x, outs[0], bounds[0])
            if alone:
                R.check(f"dK of {b}, {h}", got[1][b, h, :lens[b]], outs[1], bounds[1])
                R.check(f"dV of {b}, {h}", got[2][b, h, :lens[b]], outs[2], bounds[2])
            assert not got[1][b, h, lens[b]:].any() and not got[2][b, h, lens[b]:].any()
    assert not any(x[2].any() for x in got)


# ------------------------------------------------------------ weights at their ends
@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("M,N,front", [(40, 300, 128), (40, 300, 130), (300, 4200, 2000), (1, 300, 130)])
def test_scores_of_minus_infinity_before_small_ones(F, name, M, N, front):
    """Keys that no weight falls on, whole tiles of them, ahead of others whose
    scores lie near -100: the same as without them."""
    Q, K, V, _ = make(2, 2, 1, M, N, 64, name, seed=51)
    Q[..., 0] = 1
    Q[..., 1] = 4
    K[..., 1] = -200
    K[:, :, :front, 0] = float("-inf")
    O, LSE = F.cross_attn_fwd(Q, K, V, scale=0.125)
    ref, lse, bound, lse_bound = R.forward(Q, K[:, :, front:], V[:, :, front:], None, 0.125)
    assert float(lse.max()) < -80
    R.check("O", O, ref, bound)
    R.check("LSE", LSE, lse, lse_bound)


@pytest.mark.parametrize("name", ["bf16", "fp16"])
def test_weights_of_the_backward_over_their_whole_range(F, name):
    """dV is the weight itself where one row counts, whose LSE the test chooses:
    in every place of a tile, from weights that vanish to those that overflow
    (of an LSE that is not the scores'), and NaN."""
    powers = [-1e30, -200, -128, -127, -126, -125.5, -60.25, -24, -14.5, -3.7, -1, -0.5, -0.25, 0, 0.3, 0.5, 2.5, 5.5]
    # in fp16 weights are held times 2^10: from 2^6 on they are infinite
    powers += [6.5, 40, 126.75, 129, 140, 300, 1e30, NAN] if name == "bf16" else [140, 300, 1e30, NAN]
    M, N, d = 16, 8, 64
    B = M * len(powers)
    Q = torch.zeros(B, 1, M, d, dtype=DT[name], device="cuda")
    K = torch.zeros(B, 1, N, d, dtype=DT[name], device="cuda")
    dO = torch.ones_like(Q)
    LSE = torch.full((B, 1, M), float("inf"), device="cuda")
    want = torch.empty(B, dtype=torch.float64, device="cuda")
    for i, x in enumerate(powers):
        for r in range(M):
            LSE[i * M + r, 0, r] = -x * math.log(2)
            want[i * M + r] = 2.0 ** x if x < 128 else (float("inf") if x == x else NAN)
    dV = F.cross_attn_bwd(Q, K, torch.ones_like(K), torch.zeros_like(Q), LSE, dO)[2].double()
    u, sub = R.roundings(DT[name])
    # LSE is rounded, and multiplied by log2 e and rounded once more
    arg = 4 * R.E * torch.tensor(powers, dtype=torch.float64, device="cuda").abs().nan_to_num(0).repeat_interleave(M)
    bound = (2 * u + 2.0 ** -21 + arg.clamp(max=1)) * want + sub * 2.0 ** -10 + sub + 2.0 ** -126
    for key in range(N):
        for col in (0, 7, d - 1):
            x = dV[:, 0, key, col]
            assert torch.equal(x.isnan(), want.isnan())
            R.check("weight", x[~want.isnan()], want[~want.isnan()], bound[~want.isnan()])


# ------------------------------------------------- what a newer token's row holds
MASKED = [
    # P, S, Hq, Hkv, M, N, Np, d, dtype, kv_lens
    (1, 2, 4, 4, 2, 40, 100, 64, "fp16", [40, 7]),
    (2, 1, 8, 2, 3, 300, 70, 128, "bf16", [300, 18]),
    (1, 3, 2, 1, 5, 33, 129, 64, "bf16", [33, 17, 5]),
    (1, 1, 1, 1, 16, 4000, 30000, 128, "fp16", [3999]),       # few rows, split among blocks
    (1, 2, 4, 1, 4, 200, 30000, 64, "bf16", [200, 131]),      # few rows, parts and a join
    (2, 2, 6, 2, 7, 150, 90, 64, "fp16", [150, 130, 7, 129]),  # 21 rows a kv head
    (1, 2, 2, 2, 130, 400, 64, 128, "bf16", [400, 131]),
    (1, 1, 3, 1, 300, 700, 200, 64, "fp16", [700]),
    (1, 4, 8, 8, 257, 1300, 100, 128, "fp16", [1300, 257, 258, 1281]),
    (2, 40, 32, 4, 3, 300, 200, 128, "bf16", [3 + (61 * b) % 298 for b in range(80)]),  # several items to a block
    (2, 40, 32, 4, 3, 300, 200, 64, "fp16", [300] * 80),
]


@pytest.mark.parametrize("what", ["V", "K"])
@pytest.mark.parametrize("P,S,Hq,Hkv,M,N,Np,d,name,lens", MASKED)
def test_a_newer_token_does_not_reach_older_ones(F, what, P, S, Hq, Hkv, M, N, Np, d, name, lens):
    """NaN and infinities in the row of one of the newest tokens: the tokens
    before it do not see them, it and those behind it do, in their columns."""
    B = P * S
    Q, K, V, n = make(B, Hq, Hkv, M, N, d, name, lens, seed=61)
    _, Kp, Vp, _ = make(P, Hkv, Hkv, 1, Np, d, name, None, seed=62)
    for tok in sorted({1, M // 2, M - 1} - {0}):
        k, v, clean = K.clone(), V.clone(), V.clone()
        for b in range(B):
            key = lens[b] - M + tok
            if what == "K":
                k[b, :, key] = NAN
            else:
                v[b, :, key, 3], v[b, :, key, d - 1], v[b, :, key, d // 2] = NAN, float("inf"), float("-inf")
                clean[b, :, key, [3, d - 1, d // 2]] = 0
        got, lse = F.prefix_attn(Q, Kp, Vp, k, v, None, n)
        ref, want_lse, bound, lse_bound = R.prefix(Q, Kp, Vp, K, clean if what == "V" else V, None, n, d ** -0.5)
        if what == "K":
            R.check("O", got[:, :, :tok], ref[:, :, :tok], bound[:, :, :tok])
            R.check("LSE", lse[:, :, :tok], want_lse[:, :, :tok], lse_bound[:, :, :tok])
            assert got[:, :, tok:].isnan().all() and lse[:, :, tok:].isnan().all()
            continue
        R.check("LSE", lse, want_lse, lse_bound)
        assert got[:, :, tok:, 3].isnan().all()
        assert (got[:, :, tok:, d - 1] == float("inf")).all() and (got[:, :, tok:, d // 2] == float("-inf")).all()
        got = got.clone()
        for c in (3, d - 1, d // 2):
            got[:, :, tok:, c] = ref[:, :, tok:, c].to(got.dtype)
        R.check("O", got, ref, bound)
