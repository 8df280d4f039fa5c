"""CPU checks that the attention entries refuse outputs and workspaces that lie
over what the call reads or writes, byte for byte, and take tensors that only
interleave. The pointers are never followed."""
from __future__ import annotations

import ctypes
import random

import pytest
import torch

from test_attn_cpu import Tensor, change, entry, good

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="the pointers lead nowhere")
MISSING = (3, 5)  # the device is what is missing: every check has passed

# good()'s tensors: 2 x 4 heads (2 kv heads), 100 x 50 rows of 64, 2 bytes each
Q, O, K, V, DO, DQ, DK, DV, KP, VP = (0x10000000 * (i + 1) for i in range(10))
Q_BYTES, K_BYTES = 2 * 4 * 100 * 64 * 2, 2 * 2 * 50 * 64 * 2


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("i,kw,word", [
    (0, dict(O__ptr=Q + 128), "input"), (0, dict(O__ptr=Q - Q_BYTES + 16), "input"),
    (0, dict(O__ptr=K + K_BYTES - 16), "input"), (0, dict(LSE=V + 4), "input"),
    (0, dict(LSE=O + Q_BYTES - 4), "another"), (0, dict(kv_lens=O + 4), "input"),
    (1, dict(LSE=DQ + 64), "input"), (1, dict(dQ__ptr=0x900000), "input"), (1, dict(dK__ptr=O + 1024), "input"),
    (1, dict(dV__ptr=DK + K_BYTES - 16), "another"), (1, dict(kv_lens=DV), "input"),
    (1, dict(dQ__ptr=DO - 16), "input"),
    (2, dict(O__ptr=KP + 128), "input"), (2, dict(prefix_lens=O), "input"), (2, dict(LSE=VP + 400), "input"),
    (1, dict(workspace=Q + 16), "workspace"), (1, dict(workspace=DV + 16), "workspace"),
    (2, dict(workspace=KP), "workspace"), (1, dict(workspace=0x900000 - 16), "workspace"),
])
def test_overlaps_are_refused(kind, i, kw, word):
    if i == 2:  # long enough for parts, hence a workspace
        kw = dict(kw, N_prefix=60000)
    code, message = entry(kind, i)(change(**kw))
    assert (code, word in message) == (1, True), (code, message)


@pytest.mark.parametrize("i", [0, 1, 2])
@pytest.mark.parametrize("kw", [dict(K__batch=(1 << 38) - 8, batch=1 << 20), dict(V__row=1 << 37, N=1 << 12)])
def test_strides_past_any_memory_are_refused(i, kw):
    code, message = entry("bf16", i)(change(**kw))
    assert (code, "past any memory" in message) == (1, True), message


@pytest.mark.parametrize("i,kw", [
    (0, dict(O__ptr=Q + Q_BYTES)), (0, dict(O__ptr=Q - Q_BYTES)), (0, dict(LSE=O + Q_BYTES)),
    (1, dict(dV__ptr=DK + K_BYTES)), (1, dict(LSE=DQ - 4 * 2 * 4 * 100)), (1, dict(kv_lens=DQ - 8)),
    (0, dict(workspace=Q)),  # not needed at these sizes, so not looked at
])
def test_neighbours_are_taken(i, kw):
    assert entry("bf16", i)(change(**kw))[0] in MISSING


def packed(base, slot, slots, heads, rows, d=64, batch_rows=None):
    """Slot of a [batch][rows][slots][heads][d] buffer."""
    row = slots * heads * d
    return Tensor(base + 2 * slot * heads * d, (batch_rows or rows) * row, d, row)


def test_interleaved_tensors_are_taken():
    a = good()
    a.q_heads = a.kv_heads = 2
    a.M = a.N = 100
    a.Q, a.K, a.V = (packed(Q, s, 3, 2, 100) for s in range(3))
    a.O, a.dO = (packed(O, s, 2, 2, 100) for s in range(2))
    a.dQ, a.dK, a.dV = (packed(DQ, s, 3, 2, 100) for s in range(3))
    assert entry("bf16", 1)(a)[0] in MISSING
    # an output among the inputs' rows, in a buffer with rows to spare
    a.Q, a.K, a.V, a.O = (packed(Q, s, 4, 2, 100, batch_rows=107) for s in range(4))
    assert entry("bf16", 0)(a)[0] in MISSING
    a.O.ptr -= 16
    assert entry("bf16", 0)(a) == (1, "an output lies over an input")
    # every other row of a long buffer, of many heads
    a.M = a.N = 20000
    a.Q, a.O = Tensor(Q, 1 << 30, 64, 512), Tensor(Q + 512, 1 << 30, 64, 512)
    a.K = a.V = Tensor(V, 1 << 30, 64, 128)
    assert entry("bf16", 0)(a)[0] in MISSING
    a.O = Tensor(Q + 256, 1 << 30, 64, 1024)  # every fourth: 128 elements on, among rows of 512
    assert entry("bf16", 0)(a)[0] in MISSING


def test_random_strides_against_every_byte():
    """Refused if and only if some element of O is one of Q's."""
    rng = random.Random(7)
    call = entry("bf16", 0)

    def elements(t, n):
        at = (t.ptr - Q) // 2
        return {at + i * t.batch + j * t.head + k * t.row for i in range(n[0]) for j in range(n[1]) for k in range(n[2])}

    met = apart = 0
    for _ in range(4000):
        n = rng.randint(1, 3), rng.randint(1, 3), rng.randint(1, 5)
        a = good()
        a.batch, a.q_heads, a.M = n
        a.kv_heads = 1
        steps = [8 * rng.choice([8, 9, 16, 17, 24, 32, 48, 72, 96, 200, 216]) for _ in range(6)]
        a.Q = Tensor(Q, *steps[:3])
        a.O = Tensor(Q + 16 * rng.randint(-200, 400), *(steps[:3] if rng.random() < 0.4 else steps[3:]))
        code, message = call(a)
        if "overlapping strides" in message:
            continue
        # runs of 64 elements from starts that are multiples of 8: they meet where starts are less than 64 apart
        q, o = elements(a.Q, n), elements(a.O, n)
        want = any(x + y in q for x in o for y in range(-56, 57, 8))
        assert (code == 1 and "input" in message) == want and (want or code in MISSING), (n, steps, a.O.ptr - Q, message)
        met, apart = met + want, apart + (not want)
    assert met > 300 and apart > 300
