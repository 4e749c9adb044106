"""CPU: what the 4-bit kernels and calls promise and no device run can show."""

from __future__ import annotations

import ctypes as C
import re
from pathlib import Path

import pytest
import torch

from evspark_b200 import _native as N
from evspark_b200 import q4
from tests.test_q4 import cache, weight

CSRC = Path(__file__).resolve().parents[1] / "evspark_b200" / "csrc"


def kernels(source: str):
    """(name, parameters, body) of the kernels of a source file."""
    for m in re.finditer(r"__global__ void\s*(?:__launch_bounds__\([^{;]*?\)\s*)?(\w+)\(", source):
        depth, at = 1, m.end()
        while depth:
            depth += {"(": 1, ")": -1}.get(source[at], 0)
            at += 1
        end = source.index("\n}\n", at)
        yield m.group(1), source[m.end():at - 1], source[at:end]


def test_kernels_that_start_early_read_by_ordinary_loads():
    """A kernel that waits for its predecessor while it runs must not ask for data that stay unwritten for its whole
    life: no read-only loads, no restrict on an input, and no load that the compiler may move above the wait."""
    early = 0
    for path in sorted(CSRC.glob("q4*")):
        source = re.sub(r"//[^\n]*", "", path.read_text())
        assert "__ldg" not in source and ".nc." not in source, path.name
        for asm in re.findall(r"asm(?: volatile)?\(\s*\"ld\.global.*?\);", source, re.S):
            assert asm.startswith("asm volatile") and '"memory"' in asm, (path.name, asm)
        for name, params, body in kernels(source):
            if "pdl_wait" in body:
                early += 1
                assert not re.search(r"const\s+\w+\s*\*\s*__restrict__", params), (path.name, name)
    assert early >= 8


@pytest.mark.parametrize("n,k", [(2 ** 31, 1), (2 ** 32 + 5, 1), (1, 2 ** 24 + 1), (1, 2 ** 32 + 5), (2 ** 20, 2 ** 16)])
def test_sizes_beyond_32_bits_are_refused(n, k):
    """Sizes go to the library as 32-bit integers: 2^32 + 5 rows must not come out as five."""
    with pytest.raises(ValueError, match="at most"):
        q4.quantize_weight(torch.zeros(1, 1).expand(n, k), 32)
    with pytest.raises(ValueError, match="at most"):
        q4.Q4Weight(torch.zeros(1, dtype=torch.uint8), torch.zeros(1, dtype=torch.bfloat16), (n, k), 32)


def test_calls_beyond_32_bits_are_refused():
    with pytest.raises(ValueError, match="rows"):
        q4.q4_linear(torch.zeros(1, 100).expand(2 ** 32 + 5, 100), weight())
    c, one = cache(), torch.zeros(1, dtype=torch.int32)
    table, k = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, 1, 2, 64)
    q = torch.zeros(1, 1, 1, 64).expand(1, 1, 2 ** 32 + 4, 64)
    with pytest.raises(ValueError, match="heads"):
        q4.q4_attention(q, c, table, one, out=q)
    with pytest.raises(ValueError, match="heads"):
        q4.q4_kv_append(c, table, one, k, k, q=q, q_out=q)


def test_check_says_what_was_met(monkeypatch):
    waited = []
    monkeypatch.setattr(torch.cuda, "synchronize", lambda device=None: waited.append(device))
    c = cache()
    c._err = torch.tensor([N.EVS_ETIMEOUT, 9, 3], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="wait.*row 3"):
        c.check()
    c._err = torch.tensor([N.EVS_ERANGE, 9, 5], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="row 5 has a length"):
        c.check()
    c.check()  # read once
    assert waited == [c._index] * 3


def test_workspace_holds_the_rows_of_the_call_alone():
    """One token of one query head a kv head: a row a head, not a tile of 16."""
    d = N.Q4CacheDesc(256, None, 1 << 20, 64, 32, 128)
    for batch, tokens, heads in ((64, 1, 32), (1, 13, 32), (3, 5, 96)):
        r = N.Q4RowsDesc(256, 256, None, 2048, 2048, batch, tokens)
        rows, slots = tokens * heads // 32, 2048 * 64 // 1024
        need = N.lib().evs_q4_attention_workspace(C.byref(d), C.byref(r), heads, 0)
        assert need == batch * 32 * rows * slots * (128 + 2) * 4


def test_tensors_whose_addresses_are_kept_cannot_be_replaced():
    """A replaced tensor would be freed while calls go on reading its memory."""
    w, c = weight(), cache()
    for obj, names in ((w, ("codes", "scales")), (c, ("pool",))):
        for name in names:
            before = getattr(obj, name)
            with pytest.raises(AttributeError, match="replaced"):
                setattr(obj, name, before.clone())
            assert getattr(obj, name) is before
    for obj, name in ((w, "shape"), (w, "group"), (c, "page_size"), (c, "head_dim"), (c, "num_pages"), (c, "kv_heads")):
        with pytest.raises(AttributeError, match="replaced"):
            setattr(obj, name, 32)
