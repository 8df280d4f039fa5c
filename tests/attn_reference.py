"""Plain 64-bit forms of the attention operators, each with a bound on how far
a right 16-bit kernel may be from it, element by element.

The bounds count roundings. u = eps/2 is the relative error of one rounding to
the outputs' type. The kernels round in this order (everything else is fp32,
relative error e = 2^-24 an operation):

  score  s = scale q.k: d products and sums                       -> ds below
  weight p = exp(s - m), rounded to 16 bits to be multiplied      -> u + 2^-21
         (2^-22 for the exponential, as much for its argument's scaling);
         fp16 holds p times 2^6 in the forward, 2^10 in the backward, so its
         subnormal half-step 2^-25 stands for 2^-31 and 2^-35
  ds     p (dP - D), rounded to 16 bits likewise; fp16 holds it with dO scaled
         so that its largest magnitude lies in [8, 16): half-step 2^-25 / 8
         times that magnitude
  output one rounding, u relative, and in fp16 2^-25 absolute.

A score's own error ds moves its weight by the factor exp(ds), ds <= 0.01 here,
so |dp| <= 1.01 ds p.
"""
from __future__ import annotations

import torch

E = 2.0 ** -24


def roundings(dtype):
    """u, and fp16's subnormal half-step (bf16 has fp32's range)."""
    return torch.finfo(dtype).eps / 2, 2.0 ** -25 if dtype == torch.float16 else 0.0


def _expand(t, G):
    return t.double().repeat_interleave(G, dim=1)


def _masked(t, keys):
    """Rows that are not keys as zeros, whatever they hold."""
    return torch.where(keys[:, None, :, None], t, torch.zeros((), dtype=t.dtype, device=t.device))


def key_mask(lens, N, B, device):
    n = torch.full((B,), N, device=device) if lens is None else lens.clamp(0, N)
    return torch.arange(N, device=device) < n[:, None]


def _scores(Q, K, scale):
    q, k = Q.double(), _expand(K, Q.shape[1] // K.shape[1])
    d = Q.shape[-1]
    S = scale * q @ k.transpose(-1, -2)
    # d products summed, the scaling, and the subtraction of a maximum of this size
    err = (d + 4) * E * scale * (q.abs() @ k.abs().transpose(-1, -2)) + 4 * E * S.abs()
    return S, err


def _softmax(S, err, V, allowed, dtype):
    u, sub = roundings(dtype)
    S = S.masked_fill(~allowed, float("-inf"))
    any_key = allowed.any(-1, keepdim=True).expand(*S.shape[:-1], 1)
    LSE = torch.where(any_key[..., 0], torch.logsumexp(S, -1), float("-inf"))
    P = torch.where(any_key, torch.exp(S - torch.where(any_key, LSE[..., None], 0.0)), 0.0)
    n = S.shape[-1]
    O = P @ V
    err = torch.where(allowed, err, 0.0)
    worst = err.amax(-1, keepdim=True)
    # weights and their sum share the score errors; both sums have n terms
    rel = u + 2.0 ** -21 + 2.02 * worst + (2 * n + 64) * E
    bound = rel * (P @ V.abs()) + sub * 2.0 ** -6 * (V.abs().sum(-2, keepdim=True) * any_key)
    bound = (1 + u) * bound + u * O.abs() + sub
    lse_bound = 1.01 * worst[..., 0] + (n + 64) * E + 2.0 ** -21 + 8 * E * torch.where(any_key[..., 0], LSE, 0.0).abs()
    return O, LSE, bound, lse_bound


def forward(Q, K, V, lens, scale):
    """O, LSE and their bounds."""
    B, Hq, M, _ = Q.shape
    keys = key_mask(lens, K.shape[2], B, Q.device)
    S, err = _scores(Q, _masked(K, keys), scale)
    v = _expand(_masked(V, keys), Hq // K.shape[1])
    return _softmax(S, err, v, keys[:, None, None, :].expand_as(S), Q.dtype)


def prefix(Q, Kp, Vp, K, V, prefix_lens, lens, scale):
    B, Hq, M, _ = Q.shape
    P = Kp.shape[0]
    kp = key_mask(prefix_lens, Kp.shape[2], P, Q.device).repeat_interleave(B // P, 0)
    ko = key_mask(lens, K.shape[2], B, Q.device)
    k = torch.cat([_masked(Kp.repeat_interleave(B // P, 0), kp), _masked(K, ko)], 2)
    v = torch.cat([_masked(Vp.repeat_interleave(B // P, 0), kp), _masked(V, ko)], 2)
    n = ko.sum(-1)[:, None] - (M - 1 - torch.arange(M, device=Q.device))
    own = torch.arange(K.shape[2], device=Q.device) < n[..., None]
    allowed = torch.cat([kp[:, None].expand(-1, M, -1), own], -1)[:, None]
    S, err = _scores(Q, k, scale)
    return _softmax(S, err, _expand(v, Hq // K.shape[1]), allowed.expand_as(S), Q.dtype)


def backward(Q, K, V, O, LSE, dO, lens, scale, delta_err=0.0):
    """(dQ, dK, dV) of the operator as a function of its inputs, O and LSE
    among them, and their bounds. `delta_err`: relative error of O that the
    comparison has on top (u where O was rounded and the other side's was not)."""
    B, Hq, M, d = Q.shape
    Hkv, N = K.shape[1:3]
    G = Hq // Hkv
    u, sub = roundings(Q.dtype)
    keys = key_mask(lens, N, B, Q.device)
    Km, Vm = _masked(K, keys), _masked(V, keys)
    S, err = _scores(Q, Km, scale)
    q, k, v, o, do = Q.double(), _expand(Km, G), _expand(Vm, G), O.double(), dO.double()
    live = keys[:, None, None, :]
    lse = torch.where(LSE == float("-inf"), torch.zeros_like(LSE), LSE).double()[..., None]
    P = torch.where(live, torch.exp(S - lse), 0.0)
    relP = 1.01 * torch.where(live, err, 0.0) + 2.0 ** -21 + 4 * E * lse.abs()
    dP = do @ v.transpose(-1, -2)
    D = (do * o).sum(-1, keepdim=True)
    dS = P * (dP - D)
    acc = (d + 4) * E
    eD = (acc + delta_err) * (do.abs() * o.abs()).sum(-1, keepdim=True)
    eS = P * (acc * (do.abs() @ v.abs().transpose(-1, -2)) + eD) + (u + relP + 4 * E) * dS.abs()
    half = sub / 8 * float(do.abs().max()) if do.numel() else 0.0
    eS = torch.where(live, eS + half, 0.0)

    def group(t):
        return t.reshape(B, Hkv, G, N, d).sum(2)

    dQ = scale * dS @ k
    bQ = scale * (eS + (N + 8) * E * dS.abs()) @ k.abs()
    dK = group(scale * dS.transpose(-1, -2) @ q)
    bK = group(scale * (eS + (G * M + 8) * E * dS.abs()).transpose(-1, -2) @ q.abs())
    dV = group(P.transpose(-1, -2) @ do)
    eP = torch.where(live, (u + relP + (G * M + 8) * E) * P + sub * 2.0 ** -10, 0.0)
    bV = group(eP.transpose(-1, -2) @ do.abs())
    outs = (dQ, dK, dV)
    return outs, tuple((1 + u) * b + u * x.abs() + sub for b, x in zip((bQ, bK, bV), outs))


def check(name, got, ref, bound):
    """Every element within its bound; infinities have to be equal."""
    got = got.double()
    assert got.shape == ref.shape, f"{name}: shape {tuple(got.shape)}, expected {tuple(ref.shape)}"
    inf = torch.isinf(ref)
    assert torch.equal(got[inf], ref[inf]), f"{name}: infinities differ"
    off = (got[~inf] - ref[~inf]).abs() - bound.expand_as(ref)[~inf]
    bad = ~(off <= 0)  # NaN counts
    assert not bool(bad.any()), (f"{name}: {int(bad.sum())} of {bad.numel()} elements outside their bound, the worst by "
                                 f"{float(off[bad].nan_to_num(float('inf')).max()):.3g}")
