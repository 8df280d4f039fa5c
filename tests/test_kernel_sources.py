"""Orderings that no run can show to be missing, read from the kernels' source."""
from __future__ import annotations

import os
import re

from conftest import PKG

CSRC = os.path.join(PKG, "csrc")


def source(name):
    with open(os.path.join(CSRC, name)) as f:
        return f.read()


def body(text, name):
    """The braces' text of the function `name`."""
    at = text.index("{", text.index(f" {name}("))
    depth = 0
    for i in range(at, len(text)):
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        if depth == 0:
            return text[at:i + 1]
    raise AssertionError(f"{name} does not end")


def test_zeroes_in_a_landed_tile_come_before_the_next_copy_into_it():
    """Ordinary stores to shared memory and a later TMA copy to the same bytes
    need a proxy fence between them, by the threads that stored."""
    zero = r"reinterpret_cast<uint4\*>\((?:src|tile)[^;]*=\s*make_uint4\(0, 0, 0, 0\);"
    for file, name, copies in (("fmha_attn_decode.cuh", "attn_decode_stream_kernel", r"\bload\(stage\);"),
                               ("fmha_attn_fwd.cuh", "clear_tail", r"$")):
        text = body(source(file), name)
        stores = list(re.finditer(zero, text))
        assert stores
        for m in stores:
            between = text[m.end():m.end() + re.search(copies, text[m.end():]).start()]
            assert "fence_proxy_async_smem();" in between, f"{name}: no proxy fence behind {m.group()!r}"


def test_every_tmem_load_waits_in_its_own_statement():
    """tcgen05.ld writes its registers some time after it was issued: between it
    and a wait in another statement the compiler may copy or spill them."""
    text = source("sm100_ptx.cuh")
    loads = [m.group() for m in re.finditer(r"asm volatile\(.*?\);\n", text, re.S) if "tcgen05.ld." in m.group()]
    assert len(loads) >= 5
    for statement in loads:
        assert "tcgen05.wait::ld.sync.aligned;" in statement, statement[:120]
    for name in sorted(os.listdir(CSRC)):
        assert name == "sm100_ptx.cuh" or "tcgen05.ld." not in source(name), name
