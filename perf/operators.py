"""Measured cases of the attention operators around an encoder's states and a
shared prefix, with their plain forms.

Operators (Q [B, Hq, M, d]; every kv head serves Hq / Hkv query heads):

  cross_fwd   O and LSE of attention to an encoder's states K, V
              [B, Hkv, N, d], of which batch entry b has kv_lens[b] valid rows
  cross_bwd   dQ, dK, dV of the same, from O, LSE and dO
  decode      cross_fwd for single tokens (M = 1): the states are read once
  prefix      attention of new tokens to a prefix that S consecutive batch
              entries share, and to each entry's own cache behind it

`own` selects what run() does: the plain torch form (False) or the calls a
user makes of the library (True).
"""
import functools
import math
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------- cases
def listed():
    return [
        # image tokens attending to a padded batch of text-encoder states (the
        # cross-attention workload of the benchmark, with ragged lengths)
        dict(name="cross_fwd_image", op="cross_fwd", dtype="bf16", B=2, Hq=24, Hkv=24, M=4096, N=512, d=128, lens="ragged"),
        # the long video latent against a long conditioning sequence
        dict(name="cross_fwd_video", op="cross_fwd", dtype="bf16", B=1, Hq=40, Hkv=40, M=16384, N=1024, d=128, lens="full"),
        # a small ragged batch of prompts, shared kv heads, one entry without any state
        dict(name="cross_fwd_ragged", op="cross_fwd", dtype="fp16", B=3, Hq=12, Hkv=4, M=333, N=777, d=64, lens="empty"),
        # the training steps of the same three
        dict(name="cross_bwd_image", op="cross_bwd", dtype="bf16", B=2, Hq=24, Hkv=24, M=4096, N=512, d=128, lens="ragged"),
        dict(name="cross_bwd_video", op="cross_bwd", dtype="bf16", B=1, Hq=40, Hkv=40, M=16384, N=1024, d=128, lens="full"),
        dict(name="cross_bwd_ragged", op="cross_bwd", dtype="fp16", B=3, Hq=12, Hkv=4, M=333, N=777, d=64, lens="empty"),
        # one token of a batch of transcripts, each against its own audio states
        dict(name="decode_batch", op="decode", dtype="fp16", B=64, Hq=16, Hkv=16, M=1, N=1500, d=64, lens="full"),
        # one token of one sequence: latency
        dict(name="decode_single", op="decode", dtype="bf16", B=1, Hq=32, Hkv=8, M=1, N=4096, d=128, lens="full"),
        # one token against long documents of different lengths
        dict(name="decode_long", op="decode", dtype="bf16", B=4, Hq=64, Hkv=8, M=1, N=32768, d=128, lens="ragged"),
        # a few samples of one short prompt: latency
        dict(name="prefix_few", op="prefix", dtype="fp16", B=4, S=4, Hq=16, Hkv=16, M=1, N=64, Np=1000, d=64, lens="ragged"),
        # a large batch behind one long system prompt
        dict(name="prefix_batch", op="prefix", dtype="bf16", B=64, S=64, Hq=32, Hkv=8, M=1, N=512, Np=8192, d=128, lens="ragged"),
        # several prompts of different lengths, 16 samples each, three new tokens a sample
        dict(name="prefix_samples", op="prefix", dtype="bf16", B=128, S=16, Hq=32, Hkv=4, M=3, N=300, Np=4097, d=128, lens="ragged"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        op = rng.choice(["cross_fwd", "cross_bwd", "decode", "prefix"])
        hkv = rng.choice([1, 2, 3, 4, 8, 12, 16, 24])
        case = dict(op=op, dtype=rng.choice(["bf16", "fp16"]), d=rng.choice([64, 128]),
                    Hkv=hkv, Hq=hkv * rng.choice([1, 1, 2, 3, 4, 8]), lens=rng.choice(["full", "ragged", "empty"]))
        if op in ("cross_fwd", "cross_bwd"):
            case.update(B=rng.randint(1, 8), M=_log(rng, 1, 16384), N=_log(rng, 1, 8192))
            cap = dict(listed()[4 if op == "cross_bwd" else 1])
        elif op == "decode":
            case.update(B=_log(rng, 1, 128), M=1, N=_log(rng, 1, 65536))
            cap = dict(listed()[8])
        else:
            p, s = _log(rng, 1, 8), _log(rng, 1, 64)
            case.update(B=p * s, S=s, M=rng.choice([1, 1, 1, 2, 3, 5]), N=_log(rng, 5, 2048), Np=_log(rng, 1, 32768))
            cap = dict(listed()[10])
        # no dearer than the largest listed case of the operator, and of a size
        # at which the plain form's scores fit the card
        w, c = work(case), work(cap)
        if w["bytes"] <= c["bytes"] and w["flops"] <= c["flops"]:
            return case


def _lengths(kind, count, most):
    """`count` lengths up to `most`, spread evenly; "empty" has a zero first."""
    if kind == "full":
        return [most] * count
    lens = [max(1, -(-most * (2 * i + 1) // (2 * count))) for i in range(count)]
    lens[-1] = most
    if kind == "empty" and count > 1:
        lens[0] = 0
    return lens


def work(case):
    B, Hq, Hkv, M, d = (case[k] for k in ("B", "Hq", "Hkv", "M", "d"))
    keys = _lengths(case["lens"], B, case["N"])
    total = sum(keys)
    rows = B * Hq * M
    q, kv, lse = 2 * rows * d, 2 * 2 * Hkv * total * d, 4 * rows
    pairs = Hq * M * total
    if case["op"] == "prefix":
        prefix = _lengths("full" if case["lens"] == "full" else "ragged", B // case["S"], case["Np"])
        kv += 2 * 2 * Hkv * sum(prefix) * d
        pairs += Hq * M * case["S"] * sum(prefix)
    if case["op"] == "cross_bwd":  # Q, O, dO, LSE, K, V in; dQ, and dK, dV whole, out
        return {"bytes": 4 * q + lse + kv + 2 * 2 * B * Hkv * case["N"] * d, "flops": 10 * pairs * d}
    return {"bytes": 2 * q + lse + kv, "flops": 4 * pairs * d}


# ------------------------------------------------------------------ inputs
def _states(g, *shape, dtype, std=1.0):
    """[B, H, rows, d] as a projection leaves it: a transposed view of [B, rows, H, d]."""
    b, h, n, d = shape
    return (torch.randn(b, n, h, d, generator=g, device="cuda") * std).to(dtype).transpose(1, 2)


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(1_000_003 * seed + 17)
    dt = DTYPES[case["dtype"]]
    B, Hq, Hkv, M, N, d = (case[k] for k in ("B", "Hq", "Hkv", "M", "N", "d"))
    s = {"op": case["op"], "scale": 1.0 / math.sqrt(d)}
    s["Q"] = _states(g, B, Hq, M, d, dtype=dt)
    s["K"] = _states(g, B, Hkv, N, d, dtype=dt)
    s["V"] = _states(g, B, Hkv, N, d, dtype=dt)
    order = torch.randperm(B, generator=g, device="cuda")
    s["lens"] = torch.tensor(_lengths(case["lens"], B, N), dtype=torch.int32, device="cuda")[order].contiguous()
    if case["op"] == "prefix":
        P = B // case["S"]
        s["Kp"] = _states(g, P, Hkv, case["Np"], d, dtype=dt)
        s["Vp"] = _states(g, P, Hkv, case["Np"], d, dtype=dt)
        lens = _lengths("full" if case["lens"] == "full" else "ragged", P, case["Np"])
        s["lens_p"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    if case["op"] == "cross_bwd":
        s["dO"] = _states(g, B, Hq, M, d, dtype=dt, std=0.1)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if s["op"] == "cross_bwd":  # what the forward pass of the same step has left
        s["O"], s["LSE"] = _plain_forward(s["Q"], s["K"], s["V"], s["lens"], s["scale"])
    return s


# -------------------------------------------------------------- plain form
def _scores(Q, K, keys, scale):
    """Scaled scores [B, Hkv, G, M, N] in 32 bits, -inf where `keys` is false."""
    B, Hq, M, d = Q.shape
    q = Q.float().reshape(B, K.shape[1], Hq // K.shape[1] * M, d)
    s = (q @ K.float().transpose(-1, -2) * scale).reshape(B, K.shape[1], -1, M, K.shape[2])
    return s.masked_fill(~keys, float("-inf"))


def _weights(S):
    """exp(S - max), its row sums and the row log-sum-exp; zeros and -inf for a row without keys."""
    top = S.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
    e = torch.exp(S - top)
    total = e.sum(-1, keepdim=True)
    return e, total, torch.log(total) + top


def _plain_forward(Q, K, V, lens, scale):
    keys = (torch.arange(K.shape[2], device=K.device) < lens[:, None])[:, None, None, None, :]
    e, total, lse = _weights(_scores(Q, K, keys, scale))
    o = (e.flatten(2, 3) @ V.float()).reshape(*e.shape[:-1], V.shape[-1])
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    return o.reshape(Q.shape).to(Q.dtype), lse.reshape(Q.shape[:-1])


def _plain_backward(Q, K, V, O, LSE, dO, lens, scale):
    B, Hq, M, d = Q.shape
    Hkv, N = K.shape[1:3]
    keys = (torch.arange(N, device=K.device) < lens[:, None])[:, None, None, None, :]
    lse = LSE.reshape(B, Hkv, -1, M, 1)
    P = torch.exp(_scores(Q, K, keys, scale) - torch.where(lse == float("-inf"), torch.zeros_like(lse), lse)).flatten(2, 3)
    q, o, do = (t.float().reshape(B, Hkv, -1, d) for t in (Q, O, dO))
    dS = P * (do @ V.float().transpose(-1, -2) - (do * o).sum(-1, keepdim=True))
    dQ = (scale * (dS @ K.float())).reshape(Q.shape)
    dK = scale * (dS.transpose(-1, -2) @ q)
    dV = P.transpose(-1, -2) @ do
    return dQ.to(Q.dtype), dK.to(K.dtype), dV.to(V.dtype)


def _plain_prefix(Q, Kp, Vp, K, V, lens_p, lens, scale):
    B, Hq, M, d = Q.shape
    P, Hkv = Kp.shape[:2]
    S = B // P
    # scores against the prefix: the samples of a prompt are rows of one product
    q = Q.float().reshape(P, S, Hkv, -1, d).transpose(1, 2).reshape(P, Hkv, -1, d)
    ahead = (q @ Kp.float().transpose(-1, -2) * scale).reshape(P, Hkv, S, -1, M, Kp.shape[2])
    keys = torch.arange(Kp.shape[2], device=Q.device) < lens_p[:, None]
    ahead = ahead.masked_fill(~keys[:, None, None, None, None, :], float("-inf"))
    ahead = ahead.transpose(1, 2).reshape(B, Hkv, -1, M, Kp.shape[2])
    # scores against the entry's own cache: new token m sees all but the M - 1 - m newest
    last = lens[:, None] - (M - 1 - torch.arange(M, device=Q.device))
    keys = (torch.arange(K.shape[2], device=Q.device) < last[..., None])[:, None, None, :, :]
    e, total, lse = _weights(torch.cat([ahead, _scores(Q, K, keys, scale)], -1))
    e_p, e_s = e[..., :Kp.shape[2]], e[..., Kp.shape[2]:]
    e_p = e_p.reshape(P, S, Hkv, -1, Kp.shape[2]).transpose(1, 2).reshape(P, Hkv, -1, Kp.shape[2])
    o = (e_p @ Vp.float()).reshape(P, Hkv, S, -1, d).transpose(1, 2).reshape(B, Hkv, -1, d)
    o = o + e_s.flatten(2, 3) @ V.float()
    o = o.reshape(B, Hkv, -1, M, d) / total
    return o.reshape(Q.shape).to(Q.dtype), lse.reshape(Q.shape[:-1])


@functools.cache
def _library():
    sys.path.append("fmha-bwd-gfx1100_b200")  # the package's folder, whose name is no module's
    import fmha_bwd_b200

    return fmha_bwd_b200


def run(state):
    s = state
    if own:
        F = _library()
        if s["op"] == "cross_bwd":
            return F.cross_attn_bwd(s["Q"], s["K"], s["V"], s["O"], s["LSE"], s["dO"], s["lens"], s["scale"], sync=False)
        if s["op"] == "prefix":
            return F.prefix_attn(s["Q"], s["Kp"], s["Vp"], s["K"], s["V"], s["lens_p"], s["lens"], s["scale"], sync=False)
        return F.cross_attn_fwd(s["Q"], s["K"], s["V"], s["lens"], s["scale"], sync=False)
    if s["op"] == "cross_bwd":
        return _plain_backward(s["Q"], s["K"], s["V"], s["O"], s["LSE"], s["dO"], s["lens"], s["scale"])
    if s["op"] == "prefix":
        return _plain_prefix(s["Q"], s["Kp"], s["Vp"], s["K"], s["V"], s["lens_p"], s["lens"], s["scale"])
    return _plain_forward(s["Q"], s["K"], s["V"], s["lens"], s["scale"])


# ------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    """The definition in float64, one kv head of one batch entry at a time."""
    s = prepare(case, seed)
    B, Hq, M, d = s["Q"].shape
    Hkv, scale = s["K"].shape[1], s["scale"]
    G = Hq // Hkv
    f = dict(dtype=torch.float64, device="cuda")
    lens = s["lens"].tolist()
    if s["op"] == "cross_bwd":
        out = [torch.zeros(t.shape, **f) for t in (s["Q"], s["K"], s["V"])]
    else:
        out = [torch.zeros(B, Hq, M, d, **f), torch.full((B, Hq, M), float("-inf"), **f)]
    for b in range(B):
        for h in range(Hkv):
            hs = slice(h * G, (h + 1) * G)
            q = s["Q"][b, hs].double()
            k, v = (s[t][b, h, :lens[b]].double() for t in ("K", "V"))
            if s["op"] == "cross_bwd":
                if lens[b] == 0:
                    continue
                do, o = s["dO"][b, hs].double(), s["O"][b, hs].double()
                for g in range(G):
                    p = torch.exp(torch.einsum("md,nd->mn", q[g], k) * scale - s["LSE"][b, h * G + g].double()[:, None])
                    ds = torch.einsum("md,nd->mn", do[g], v) - torch.einsum("md,md->m", do[g], o[g])[:, None]
                    ds *= p
                    out[0][b, h * G + g] = scale * torch.einsum("mn,nd->md", ds, k)
                    out[1][b, h, :lens[b]] += scale * torch.einsum("mn,md->nd", ds, q[g])
                    out[2][b, h, :lens[b]] += torch.einsum("mn,md->nd", p, do[g])
                continue
            allowed = torch.ones(M, lens[b], dtype=torch.bool, device="cuda")
            if s["op"] == "prefix":
                p = b // (B // s["Kp"].shape[0])
                n = int(s["lens_p"][p])
                k, v = (torch.cat([s[t][p, h, :n].double(), w]) for t, w in (("Kp", k), ("Vp", v)))
                # token m of the M new ones does not see the tokens after it
                behind = torch.arange(M, device="cuda")[:, None] + (lens[b] - M) >= torch.arange(lens[b], device="cuda")
                allowed = torch.cat([torch.ones(M, n, dtype=torch.bool, device="cuda"), behind], 1)
            if k.shape[0] == 0:
                continue
            a = torch.einsum("gmd,nd->gmn", q, k).mul_(scale).masked_fill_(~allowed, float("-inf"))
            out[1][b, hs] = torch.logsumexp(a, -1)
            out[0][b, hs] = torch.einsum("gmn,nd->gmd", torch.softmax(a, -1), v)
    return tuple(out)
