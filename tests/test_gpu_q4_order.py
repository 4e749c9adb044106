"""Calls behind each other on one stream with no wait between them: every call sees what the one before wrote."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_q4 import BF, F32, i32, make_rows, q4, randn  # noqa: F401  (q4: the module's fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,k,group,dtype", [(64, 128, 64, BF), (4096, 1024, 128, BF), (200, 300, 32, F32)])
def test_linear_behind_the_quantisation_into_its_own_buffers(q4, n, k, group, dtype):  # noqa: F811
    """The weight is quantised anew into the same codes and scales before each call."""
    rounds = 40
    ws = randn(rounds, n, k, seed=1, dtype=dtype)
    x = randn(5, k, seed=2, dtype=dtype)
    want = torch.stack([q4.q4_linear(x, q4.quantize_weight(ws[i], group)) for i in range(rounds)])
    w = q4.quantize_weight(ws[0], group)
    got = torch.empty_like(want)
    torch.cuda.synchronize()
    for i in range(rounds):
        q4._call(0, "evs_q4_quantize", ws[i].data_ptr(), q4._DT[dtype], k, n, k, group, w.codes.data_ptr(),
                 w.scales.data_ptr())
        q4.q4_linear(x, w, out=got[i])
    assert torch.equal(got, want)
    # a call behind a call whose result it reads
    back = q4.quantize_weight(randn(k, n, seed=3), group)
    torch.cuda.synchronize()
    chain = [q4.q4_linear(q4.q4_linear(x, w), back) for _ in range(rounds)]
    torch.cuda.synchronize()
    assert all(torch.equal(c, q4.q4_linear(want[-1], back)) for c in chain)


@pytest.mark.parametrize("start,H,G,D,dtype", [(5, 4, 2, 64, BF), (2040, 2, 2, 128, BF), (4080, 4, 1, 32, F32)])
def test_decode_steps_behind_each_other(q4, start, H, G, D, dtype):  # noqa: F811
    """Each token appended and attended at once: neighbours share the lines of a page's codes and scales."""
    steps = 60
    end = start + steps
    cache, table = make_rows(q4, [end], 16, G, D)
    k, v = randn(1, end, G, D, seed=1, dtype=dtype), randn(1, end, G, D, seed=2, dtype=dtype)
    q = randn(1, steps, H, D, seed=3, dtype=dtype)
    at = [i32([start + t]) for t in range(steps)]
    q4.q4_kv_append(cache, table, i32([0]), k[:, :start], v[:, :start])
    torch.cuda.synchronize()
    got, read = [], []
    for t in range(steps):
        s = slice(start + t, start + t + 1)
        rot = q4.q4_kv_append(cache, table, at[t], k[:, s], v[:, s], q=q[:, t:t + 1])
        got.append(q4.q4_attention(rot, cache, table, at[t]))
        read.append(q4.q4_kv_read(cache, table, at[t], 1))
    torch.cuda.synchronize()
    rot = q4.q4_kv_append(cache, table, at[0], k[:, start:], v[:, start:], q=q)
    assert torch.equal(torch.cat(got, 1), torch.cat([q4.q4_attention(rot[:, t:t + 1], cache, table, at[t])
                                                     for t in range(steps)], 1))
    kk, vv = q4.q4_kv_read(cache, table, at[0], steps)
    assert torch.equal(torch.cat([r[0] for r in read], 1), kk) and torch.equal(torch.cat([r[1] for r in read], 1), vv)
    cache.check()


def test_check_sees_calls_of_other_streams(q4):  # noqa: F811
    """A bad page met on another stream, behind work that is still running when check is called."""
    cache, table = make_rows(q4, [40], 16, 1, 64)
    q, at = randn(1, 1, 1, 64, seed=1), i32([20])
    bad = torch.full_like(table, cache.num_pages)
    side = torch.cuda.Stream()
    q4.q4_attention(q, cache, table, at)  # the kernel is loaded: its first call may wait for the device
    torch.cuda._sleep(1000)
    cache.check()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)  # about 0.1 s
        q4.q4_attention(q, cache, bad, at)
    with pytest.raises(RuntimeError, match="page table|pool"):
        cache.check()
    cache.check()  # read once
