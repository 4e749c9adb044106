"""CPU: the 4-bit operators refuse what they do not take, before any device call; the format's claims."""

from __future__ import annotations

import ctypes as C

import pytest
import torch

from evspark_b200 import _native as N
from evspark_b200 import q4
from tests import _q4_ref as R


def test_held_values_are_exact_in_bf16_and_within_half_a_step():
    x = torch.randn(64, 256, generator=torch.Generator().manual_seed(1), dtype=torch.float64) * \
        torch.exp(4 * torch.randn(64, 1, generator=torch.Generator().manual_seed(2), dtype=torch.float64))
    c, s = R.quantize(x, 32)
    h = R.held(x, 32)
    assert torch.equal(h.to(torch.bfloat16).double(), h)
    assert int(c.min()) >= 1 and int(c.max()) <= 15
    assert bool(((h - x).abs() <= 0.5 * s.repeat_interleave(32, -1)).all())


def weight(n=8, k=100, group=32):
    w = q4.Q4Weight.__new__(q4.Q4Weight)  # host tensors: only the checks before the device call run
    kp = q4.padded_features(k)
    w.codes, w.scales = torch.zeros(n, kp // 2, dtype=torch.uint8), torch.zeros(kp // group, n, dtype=torch.bfloat16)
    w.shape, w.group = (n, k), group
    w._args, w._index = (0, 0, n, k, group), -1
    return w


def cache(pages=4, G=2, D=64, page=16):
    c = q4.Q4Cache.__new__(q4.Q4Cache)
    c.pool = torch.zeros(pages, G, q4.Q4Cache.block_bytes(D, page), dtype=torch.uint8)
    c.num_pages, c.kv_heads, c.head_dim, c.page_size, c._index = pages, G, D, page, -1
    return c


def test_weight_refusals():
    codes, scales = torch.zeros(8, 64, dtype=torch.uint8), torch.zeros(4, 8, dtype=torch.bfloat16)
    for args in [(codes, scales, (8, 100), 48), (codes, scales, (8, 129), 32), (codes, scales, (0, 100), 32),
                 (codes.int(), scales, (8, 100), 32), (codes, scales.float(), (8, 100), 32),
                 (codes, scales.t(), (8, 100), 32), (codes, scales, (8, 100), 64),
                 (torch.zeros(64, 8, dtype=torch.uint8).t(), scales, (8, 100), 32)]:
        with pytest.raises(ValueError):
            q4.Q4Weight(*args)
    for w, group in [(torch.zeros(8), 32), (torch.zeros(0, 4), 32), (torch.zeros(8, 8), 16),
                     (torch.zeros(8, 8, dtype=torch.float16), 32)]:
        with pytest.raises(ValueError):
            q4.quantize_weight(w, group)


def test_linear_refusals():
    w = weight()
    for x, kw in [(torch.zeros(2, 99), {}), (torch.zeros(2, 100, dtype=torch.float16), {}), (torch.zeros(()), {}),
                  (torch.zeros(2, 100), dict(out_dtype=torch.float16)), (torch.zeros(2, 100), dict(out=torch.zeros(2, 9))),
                  (torch.zeros(2, 100), dict(out=torch.zeros(8, 2).t())),
                  (torch.zeros(2, 100), dict(out=torch.zeros(2, 8, dtype=torch.int32)))]:
        with pytest.raises(ValueError):
            q4.q4_linear(x, w, **kw)


def test_cache_refusals():
    for kw in [dict(head_dim=48), dict(head_dim=256), dict(page_size=8), dict(page_size=40), dict(page_size=8192),
               dict(num_pages=0), dict(kv_heads=0)]:
        with pytest.raises(ValueError):
            q4.Q4Cache(**{**dict(num_pages=2, kv_heads=1, head_dim=64), **kw})
    with pytest.raises(ValueError):
        q4.Q4Cache.from_pool(torch.zeros(2, 1, 100, dtype=torch.uint8), head_dim=64, page_size=16)
    with pytest.raises(ValueError):
        q4.Q4Cache.from_pool(torch.zeros(2, 1, 1152), head_dim=64, page_size=16)


def test_append_read_attention_refusals():
    c = cache()
    table, lengths = torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    k, q = torch.zeros(3, 5, 2, 64), torch.zeros(3, 5, 4, 64)
    bad_rows = [dict(page_table=table.long()), dict(page_table=table[:2]), dict(page_table=torch.zeros(2, 3, dtype=torch.int32).t()),
                dict(lengths=lengths.long()), dict(lengths=lengths[:2]), dict(counts=lengths[:1]), dict(counts=lengths.long()),
                dict(lengths=torch.zeros(6, dtype=torch.int32)[::2])]
    for bad in bad_rows:
        kw = {**dict(page_table=table, lengths=lengths), **bad}
        with pytest.raises(ValueError):
            q4.q4_kv_append(c, k=k, v=k, **kw)
        with pytest.raises(ValueError):
            q4.q4_attention(q, c, **kw)
    for args in [dict(k=k.half(), v=k.half()), dict(k=k, v=k.bfloat16()), dict(k=k[:, :, :1], v=k), dict(k=k, v=k[..., :32]),
                 dict(k=k, v=k, q=q.bfloat16()), dict(k=k, v=k, q_out=q), dict(k=k, v=k, q=q, q_out=q[:, :4]),
                 dict(k=k.transpose(-1, -2).contiguous().transpose(-1, -2), v=k), dict(k=k[0], v=k[0])]:
        with pytest.raises(ValueError):
            q4.q4_kv_append(c, table, lengths, **args)
    for args in [dict(q=q[:, :, :3]), dict(q=q.half()), dict(q=q[0]), dict(q=q, max_length=0), dict(q=q, out=q[:, :3]),
                 dict(q=q, out=q.bfloat16()), dict(q=q[..., :32])]:
        with pytest.raises(ValueError):
            q4.q4_attention(cache=c, page_table=table, lengths=lengths, **args)
    with pytest.raises(ValueError):
        q4.q4_kv_read(c, table, lengths, 4, dtype=torch.float16)
    with pytest.raises(ValueError):
        q4.q4_kv_read(c, table, lengths, 4, out=(k, k))


def test_entry_points_refuse_bad_arguments():
    """The C entry points check sizes, types and pointers before any device call (addresses never followed)."""
    lib, one = N.lib(), 256
    bad = [(one, 7, 100, 1, one, one, 8, 100, 32, one, 0, 8), (one, 0, 99, 1, one, one, 8, 100, 32, one, 0, 8),
           (one, 0, 100, 0, one, one, 8, 100, 32, one, 0, 8), (one, 0, 100, 1, one + 8, one, 8, 100, 32, one, 0, 8),
           (one, 0, 100, 1, one, one, 8, 100, 48, one, 0, 8), (one, 0, 100, 1, one, one, 8, 0, 32, one, 0, 8),
           (one, 0, 100, 1, one, one, 8, 100, 32, one, 0, 7), (None, 0, 100, 1, one, one, 8, 100, 32, one, 0, 8),
           (one + 2, 0, 100, 1, one, one, 8, 100, 32, one, 0, 8)]
    for a in bad:
        assert lib.evs_q4_linear(*a, None) == N.EVS_EINVAL, a
    good = dict(pool=one, err=None, num_pages=4, page_size=16, kv_heads=2, head_dim=64)
    rows = dict(page_table=one, lengths=one, counts=None, table_stride=3, max_pages=3, batch=2, tokens=5)
    st = (C.c_int64 * 3)(640, 128, 64)

    def run(c, r, H=4, dtype=0, ws=one, ml=0):
        c, r = N.Q4CacheDesc(**c), N.Q4RowsDesc(**r)
        return (lib.evs_q4_attention(C.byref(c), C.byref(r), one, st, H, 1.0, ml, one, st, dtype, ws, 1 << 30, None),
                lib.evs_q4_attention_workspace(C.byref(c), C.byref(r), H, ml),
                lib.evs_q4_kv_append(C.byref(c), C.byref(r), one, st, one, st, one, st, one, st, H, dtype, 1e4, None))

    for c in [dict(head_dim=48), dict(page_size=24), dict(num_pages=0), dict(kv_heads=0), dict(pool=None), dict(pool=one + 4)]:
        a, w, p = run({**good, **c}, rows)
        assert a == p == N.EVS_EINVAL and w == -1, c
    for r in [dict(page_table=None), dict(lengths=None), dict(table_stride=2), dict(max_pages=0), dict(batch=0), dict(tokens=0)]:
        a, w, p = run(good, {**rows, **r})
        assert a == p == N.EVS_EINVAL and w == -1, r
    a, w, p = run(good, {**rows, "max_pages": 1 << 27, "table_stride": 1 << 27})
    assert a == p == N.EVS_ERANGE and w == -1
    assert run(good, rows, H=3)[0] == run(good, rows, H=1)[0] == run(good, rows, dtype=5)[0] == N.EVS_EINVAL
    assert run(good, rows, ws=None)[0] == run(good, rows, ws=one + 4)[0] == run(good, rows, ml=-1)[0] == N.EVS_EINVAL
    d, r = N.Q4CacheDesc(**good), N.Q4RowsDesc(**rows)
    assert lib.evs_q4_kv_append(C.byref(d), C.byref(r), one, st, one, st, one, st, None, None, 4, 0, 1e4, None) == N.EVS_EINVAL
    assert lib.evs_q4_kv_append(C.byref(d), C.byref(r), one, st, one, st, None, None, None, None, 0, 0, 0.0, None) == N.EVS_EINVAL


def test_workspace_is_bounded_and_covers_a_token():
    d = N.Q4CacheDesc(256, None, 1 << 20, 64, 32, 128)
    lib = N.lib()
    r = N.Q4RowsDesc(256, 256, None, 4096, 4096, 1, 13)
    assert lib.evs_q4_attention_workspace(C.byref(d), C.byref(r), 32, 2048) == 0  # one cluster folds it
    for tokens, H, ml in [(1, 32, 3000), (13, 32, 65549), (1024, 32, 262144), (4096, 256, 262144)]:
        r = N.Q4RowsDesc(256, 256, None, 4096, 4096, 1, tokens)
        w = lib.evs_q4_attention_workspace(C.byref(d), C.byref(r), H, ml)
        assert 0 < w <= 320 << 20


@pytest.mark.skipif(torch.cuda.is_available(), reason="a GPU is present")
def test_fails_loudly_without_gpu():
    with pytest.raises(RuntimeError, match="CUDA|device"):
        q4.quantize_weight(torch.zeros(8, 8), 32)
    with pytest.raises(RuntimeError, match="CUDA|device"):
        q4.Q4Cache(2, 1, 64)
