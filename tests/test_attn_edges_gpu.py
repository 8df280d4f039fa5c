"""Edges of the attention entries on the GPU: inputs at which a kernel of this
kind goes wrong without its ordinary cases showing it. References and bounds as
in test_cross_gpu.py."""
from __future__ import annotations

import pytest
import torch

import attn_reference as R
from test_cross_gpu import DT, F, make  # noqa: F401 (F is a fixture)

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
