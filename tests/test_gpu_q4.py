"""The 4-bit operators on the device against their definitions in 64 bits (tests/_q4_ref.py)."""

from __future__ import annotations

import math

import pytest
import torch

from tests import _q4_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def q4():
    from evspark_b200 import q4 as m

    return m


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def randn(*shape, seed=0, dtype=F32):
    return torch.randn(*shape, generator=gen(seed), device=DEV).to(dtype)


# ---- weights -------------------------------------------------------------------------------
@pytest.mark.parametrize("n,k,group,dtype", [(1, 1, 32, F32), (5, 31, 32, BF), (33, 128, 64, BF), (16, 129, 128, F32),
                                             (130, 704, 32, BF), (64, 1000, 64, F32)])
def test_quantize_matches_the_format(q4, n, k, group, dtype):
    w = randn(n, k, seed=n + k, dtype=dtype) * torch.exp(randn(n, 1, seed=1) * 3).to(dtype)
    w[0, :] = 0
    qw = q4.quantize_weight(w, group)
    kp = q4.padded_features(k)
    padded = torch.zeros(n, kp, dtype=torch.float64, device=DEV)
    padded[:, :k] = w.double()
    codes, scales = R.quantize(padded, group)
    assert torch.equal(qw.codes, R.pack(codes))
    assert torch.equal(qw.scales.double(), scales.t())
    want = R.held(padded, group)[:, :k]
    assert torch.equal(qw.dequantize(F32).double(), want)
    assert torch.equal(qw.dequantize(BF).double(), want)  # held values are exact in bf16


def test_quantize_special_groups(q4):
    w = torch.ones(8, 128, device=DEV)
    w[1, 3] = math.nan
    w[2, 40] = math.inf
    w[3, 70] = -math.inf
    w[4] *= 2.0 ** -121
    w[5, :32] = 3e38
    w[6, 5] = 2.5 * 2 ** -7  # ties go to even
    d = q4.quantize_weight(w, 32).dequantize(F32)
    assert d[1, :32].isnan().all() and d[2, 32:64].isnan().all() and d[3, 64:96].isnan().all()
    assert d[5, :32].isnan().all() and (d[4] == 0).all()
    assert torch.equal(d[0].double(), R.held(w[0].double(), 32))
    assert int(d.isnan().sum()) == 4 * 32


LINEAR = [(1, 128, 128, 128, BF), (1, 4096, 4096, 128, BF), (8, 33, 65, 32, BF), (9, 1, 1, 32, F32), (13, 704, 256, 64, F32),
          (16, 257, 1408, 64, BF), (17, 130, 2816, 128, BF), (33, 1003, 717, 32, F32), (64, 384, 4096, 64, BF),
          (65, 200, 512, 128, BF), (200, 129, 300, 32, F32), (3, 128, 22528, 128, BF)]


@pytest.mark.parametrize("m,n,k,group,dtype", LINEAR)
def test_linear(q4, m, n, k, group, dtype):
    w = q4.quantize_weight(randn(n, k, seed=3) * k ** -0.5, group)
    x = randn(m, k, seed=4, dtype=dtype)
    held = w.dequantize(F32).double()
    want = x.double() @ held.t()
    bound = R.linear_bound(x, held)
    got = q4.q4_linear(x, w)
    assert got.dtype == F32 and got.shape == (m, n)
    err = (got.double() - want).abs()
    assert bool((err <= bound).all()), float((err / bound).max())
    got16 = q4.q4_linear(x, w, out_dtype=BF)
    assert bool(((got16.double() - want).abs() <= bound + 2.0 ** -8 * (want.abs() + bound)).all())
    # a row's bits do not depend on the other rows
    for r in {0, m // 2, m - 1}:
        assert torch.equal(q4.q4_linear(x[r:r + 1], w), got[r:r + 1])


def test_linear_strides_and_outputs(q4):
    w = q4.quantize_weight(randn(96, 200, seed=5), 64)
    big = randn(12, 433, seed=6, dtype=BF)
    want = q4.q4_linear(big[:, 1:201].contiguous(), w)
    assert torch.equal(q4.q4_linear(big[:, 1:201], w), want)  # rows at odd offsets
    assert torch.equal(q4.q4_linear(big[::3, 1:201], w), want[::3])
    assert torch.equal(q4.q4_linear(big[:, 1:201].unflatten(0, (3, 4)), w), want.unflatten(0, (3, 4)))
    assert torch.equal(q4.q4_linear(big[0, 1:201], w), want[0])
    t = randn(200, 12, seed=6, dtype=BF)
    assert torch.equal(q4.q4_linear(t.t(), w), q4.q4_linear(t.t().contiguous(), w))
    out = torch.full((14, 96), 7.0, device=DEV)
    assert q4.q4_linear(big[:, 1:201], w, out=out[1:13]) is not None
    assert torch.equal(out[1:13], want) and bool((out[0] == 7).all()) and bool((out[13] == 7).all())
    assert q4.q4_linear(big[:0, 1:201], w).shape == (0, 96)


def test_linear_non_finite_rows_stay_in_their_rows(q4):
    w = q4.quantize_weight(randn(40, 128, seed=7), 128)
    x = randn(5, 128, seed=8)
    clean = q4.q4_linear(x, w)
    x[1, 0], x[3, 127] = math.nan, math.inf
    got = q4.q4_linear(x, w)
    assert torch.equal(got[[0, 2, 4]], clean[[0, 2, 4]])
    assert bool(got[1].isnan().all()) and not bool(got[3].isfinite().all())


# ---- cache ---------------------------------------------------------------------------------
def make_rows(q4, ends, page, G, D, seed=0, extra=2, fill=0xFF):
    """A pool of garbage (codes of 15, NaN scales) and scattered pages for rows that reach ``ends`` tokens."""
    need = [max(1, -(-e // page)) for e in ends]
    total = sum(need) + extra
    cache = q4.Q4Cache(total, G, D, page_size=page, device=DEV)
    cache.pool.fill_(fill)
    perm = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(ends), max(need)), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor([perm.pop() for _ in range(n)], dtype=torch.int32)
    return cache, table.to(DEV)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def fill_cache(q4, cache, table, starts, ends, G, D, seed=0, dtype=BF):
    """Append random keys and values for positions [0, ends[b]); returns the held values per row."""
    T = max(ends)
    k, v = randn(len(ends), T, G, D, seed=seed + 1, dtype=dtype), randn(len(ends), T, G, D, seed=seed + 2, dtype=dtype)
    q4.q4_kv_append(cache, table, i32([0] * len(ends)), k, v, counts=i32(ends))
    kk, vv = q4.q4_kv_read(cache, table, i32([0] * len(ends)), T, counts=i32(ends))
    return kk, vv


@pytest.mark.parametrize("D,G,H,page,dtype", [(128, 4, 4, 64, BF), (128, 2, 6, 16, F32), (64, 3, 15, 48, BF),
                                              (64, 1, 8, 128, F32), (32, 8, 8, 32, F32), (32, 5, 5, 16, BF)])
def test_append_rotates_quantises_and_pages(q4, D, G, H, page, dtype):
    starts, counts, T = [0, 1, page - 1, 777, 262000, 5], [7, 3, 7, 5, 6, 0], 7
    ends = [s + c for s, c in zip(starts, counts)]
    cache, table = make_rows(q4, ends, page, G, D)
    before = cache.pool.clone()
    qkv = randn(6, T, (H + 2 * G) * D, seed=11, dtype=dtype)
    q = qkv[..., :H * D].unflatten(-1, (H, D))
    k = qkv[..., H * D:(H + G) * D].unflatten(-1, (G, D))
    v = qkv[..., (H + G) * D:].unflatten(-1, (G, D))
    q_out = torch.full((6, T, H, D), 7.0, dtype=dtype, device=DEV)
    q4.q4_kv_append(cache, table, i32(starts), k, v, q=q, counts=i32(counts), q_out=q_out)
    cache.check()
    codes = page * D // 2
    touched = torch.zeros_like(before, dtype=torch.bool)
    for b, (s, c) in enumerate(zip(starts, counts)):
        assert bool((q_out[b, c:] == 7).all())  # padding is left as it was
        if c == 0:
            continue
        pos = torch.arange(s, s + c, device=DEV)
        want_q = R.rotate(q[b, :c], pos)
        # one rounding to the type (by way of fp32)
        assert bool(((q_out[b, :c].double() - want_q).abs() <= (torch.finfo(dtype).eps / 2 + 2.0 ** -23) * want_q.abs()
                     + 2.0 ** -40).all())
        for what, x in enumerate((R.rotate(k[b, :c], pos), v[b, :c].double())):
            cc, ss = R.quantize(x, 32)
            for i in range(c):
                p, slot = int(table[b, (s + i) // page]), (s + i) % page
                blk = cache.pool[p]
                at = what * codes + slot * D // 2
                assert torch.equal(blk[:, at:at + D // 2], R.pack(cc[i]))
                touched[p, :, at:at + D // 2] = True
                sc = blk[:, 2 * codes + what * (page * D // 16):][:, :page * D // 16].contiguous().view(BF)
                assert torch.equal(sc.view(G, D // 32, page)[:, :, slot].double(), ss[i])
                for grp in range(D // 32):
                    o = 2 * codes + what * (page * D // 16) + 2 * (grp * page + slot)
                    touched[p, :, o:o + 2] = True
    assert torch.equal(cache.pool[~touched], before[~touched])  # nothing else was written


def test_append_special_values(q4):
    cache, table = make_rows(q4, [8], 16, 1, 64)
    k, v = randn(1, 8, 1, 64, seed=1), randn(1, 8, 1, 64, seed=2)
    v[0, 1, 0, 5], v[0, 2, 0, 40], v[0, 3] = math.nan, math.inf, 0
    k[0, 4, 0, 0], v[0, 5, 0, :32], v[0, 6, 0, 32:] = math.nan, 3e38, 2.0 ** -130
    q4.q4_kv_append(cache, table, i32([0]), k, v)
    kk, vv = q4.q4_kv_read(cache, table, i32([0]), 8, dtype=F32)
    assert bool(vv[0, 1, 0, :32].isnan().all()) and bool(vv[0, 1, 0, 32:].isfinite().all())
    assert bool(vv[0, 2, 0, 32:].isnan().all()) and bool((vv[0, 3] == 0).all())
    assert bool(kk[0, 4].isnan().all())  # the rotation carries the NaN into the pair's other half
    assert bool(vv[0, 5, 0, :32].isnan().all()) and bool((vv[0, 6, 0, 32:] == 0).all())


def test_append_unaligned_views_and_default_q_out(q4):
    cache, table = make_rows(q4, [20], 16, 2, 64)
    big = randn(1, 5, 2, 67, seed=3, dtype=BF)
    k, v, q = big[..., 1:65], big[..., 2:66], big[..., 3:67]
    a = q4.q4_kv_append(cache, table, i32([13]), k, v, q=q)
    pool = cache.pool.clone()
    cache.pool.fill_(0xFF)
    qq = q.contiguous()
    b = q4.q4_kv_append(cache, table, i32([13]), k.contiguous(), v.contiguous(), q=qq, q_out=qq)  # in place
    assert torch.equal(a, b) and torch.equal(pool, cache.pool)


ATTEND = [  # starts, T, counts, H, G, D, page, dtype
    ([0], 1, None, 1, 1, 32, 16, F32),
    ([0, 1, 15, 16, 17], 1, None, 4, 4, 64, 16, BF),
    ([0, 3, 62, 63, 64, 250, 255, 256], 13, None, 2, 2, 128, 64, BF),
    ([5, 100, 31, 700], 7, [7, 0, 3, 1], 10, 2, 64, 48, F32),
    ([1023, 2], 13, [13, 4], 16, 2, 128, 32, BF),
    ([300], 5, None, 20, 1, 32, 16, BF),
    ([40], 3, None, 34, 2, 128, 128, F32),
    ([4090], 13, None, 3, 1, 32, 64, BF),
    ([4095, 4096, 10], 2, None, 2, 1, 32, 64, F32),
    ([65530], 13, None, 1, 1, 32, 128, F32),
    ([70000, 20], 2, None, 2, 1, 32, 128, BF),
    # many rows a kv head beyond the fused lengths: warps share the decoding of the keys
    ([2500, 60, 4090], 13, [13, 5, 13], 16, 2, 128, 64, BF),
    ([2300], 7, None, 20, 2, 64, 48, F32),
    ([3001, 0], 16, [16, 9], 12, 3, 32, 16, BF),
    ([5000], 40, None, 2, 2, 128, 32, F32),
]


@pytest.mark.parametrize("starts,T,counts,H,G,D,page,dtype", ATTEND)
def test_attention(q4, starts, T, counts, H, G, D, page, dtype):
    counts = counts or [T] * len(starts)
    ends = [s + c for s, c in zip(starts, counts)]
    cache, table = make_rows(q4, ends, page, G, D, seed=H)
    k, v = fill_cache(q4, cache, table, starts, ends, G, D, seed=T, dtype=dtype)
    q = randn(len(starts), T, H, D, seed=9, dtype=dtype) * 2
    out = torch.full((len(starts), T, H, D), 7.0, dtype=dtype, device=DEV)
    q4.q4_attention(q, cache, table, i32(starts), counts=i32(counts), out=out)
    cache.check()
    for b, (s, c) in enumerate(zip(starts, counts)):
        assert bool((out[b, c:] == 7).all())
        if c == 0:
            continue
        want, av, mag = R.attend(q[b, :c], k[b, :s + c].double(), v[b, :s + c].double(), s, D ** -0.5)
        bound = R.attend_bound(want, av, mag, s + c, D, dtype)
        err = (out[b, :c].double() - want).abs()
        assert bool((err <= bound).all()), (b, float((err / bound).max()))


@pytest.mark.parametrize("start,T,H,G,D,dtype", [(250, 13, 8, 2, 64, BF), (4088, 16, 3, 1, 32, BF), (1000, 9, 6, 2, 128, F32),
                                                 (65529, 13, 1, 1, 32, BF), (3500, 13, 16, 2, 128, BF),
                                                 (1020, 12, 20, 2, 32, F32), (131070, 5, 16, 1, 32, BF)])
def test_attention_bits_depend_on_the_token_alone(q4, start, T, H, G, D, dtype):
    """A verify block, single steps, another batch, page size, bound and strides give the same bits."""
    end = start + T
    cache, table = make_rows(q4, [end, 40, end], 64, G, D)
    k, v = randn(3, end, G, D, seed=1, dtype=dtype), randn(3, end, G, D, seed=2, dtype=dtype)
    k[2], v[2] = k[0], v[0]
    q4.q4_kv_append(cache, table, i32([0, 0, 0]), k, v, counts=i32([end, 40, end]))
    q = randn(3, T, H, D, seed=3, dtype=dtype) * 2
    q[2] = q[0]
    block = q4.q4_attention(q, cache, table, i32([start, 20, start]), counts=i32([T, 5, T]))
    assert torch.equal(block[0], block[2])
    for t in (0, 1, T // 2, T - 1):
        step = q4.q4_attention(q[:1, t:t + 1], cache, table[:1], i32([start + t]), max_length=start + t + 1)
        assert torch.equal(step[0, 0], block[0, t]), t
    # a table with room for more (its empty entries are never read) takes the two-kernel path at any length
    roomy = torch.full((1, 64 + table.shape[1]), -1, dtype=torch.int32, device=DEV)
    roomy[:, :table.shape[1]] = table[:1]
    assert torch.equal(q4.q4_attention(q[:1], cache, roomy, i32([start]))[0], block[0])
    cache.check()
    other, ot = make_rows(q4, [end], 16, G, D, seed=5)
    q4.q4_kv_append(other, ot, i32([0]), k[:1], v[:1])
    wide = torch.zeros(1, T, H, D + 3, dtype=dtype, device=DEV)
    wide[..., 1:D + 1] = q[0]
    got = q4.q4_attention(wide[..., 1:D + 1], other, ot, i32([start]), out=wide[..., 2:D + 2].clone()[..., :D])
    assert torch.equal(got[0], block[0])


@pytest.mark.parametrize("H,room", [(2, 0), (2, 200), (12, 200)])  # one cluster; two kernels; shared decoding
def test_attention_nan_keys_and_values_reach_only_who_sees_them(q4, H, room):
    D, G, T, start = 64, 1, 6, 60
    cache, table = make_rows(q4, [start + T], 16, G, D)
    table = torch.cat([table, torch.full((1, room), -1, dtype=torch.int32, device=DEV)], 1)
    k, v = randn(1, start + T, G, D, seed=1), randn(1, start + T, G, D, seed=2)
    q4.q4_kv_append(cache, table, i32([0]), k, v)
    q = randn(1, T, H, D, seed=3)
    clean = q4.q4_attention(q, cache, table, i32([start]))
    vb, kb = v.clone(), k.clone()
    vb[0, start + 2, 0, 40] = math.nan  # the token at start + 2, second group of features
    kb[0, start + 4, 0, 1] = math.inf
    q4.q4_kv_append(cache, table, i32([0]), kb, vb)
    got = q4.q4_attention(q, cache, table, i32([start]))
    assert torch.equal(got[0, :2], clean[0, :2])
    assert bool(got[0, 2:4, :, 32:].isnan().all()) and torch.equal(got[0, 2:4, :, :32], clean[0, 2:4, :, :32])
    assert bool(got[0, 4:].isnan().all())


def test_attention_scale_and_sharp_scores(q4):
    """Scores far apart (one key takes all the weight) and a scale of the caller's."""
    D, end = 128, 600
    cache, table = make_rows(q4, [end], 64, 2, D)
    k, v = fill_cache(q4, cache, table, [end - 4], [end], 2, D)
    q = randn(1, 4, 4, D, seed=5) * 30
    out = q4.q4_attention(q, cache, table, i32([end - 4]), scale=0.7)
    want, av, mag = R.attend(q[0], k[0].double(), v[0].double(), end - 4, 0.7)
    bound = R.attend_bound(want, av, mag, end, D, F32)
    assert bool(((out[0].double() - want).abs() <= bound).all())


def test_bad_pages_and_lengths_are_reported_not_followed(q4):
    cache, table = make_rows(q4, [40, 40, 40, 40], 16, 1, 64, fill=0)
    k, v = randn(4, 40, 1, 64, seed=1), randn(4, 40, 1, 64, seed=2)
    q4.q4_kv_append(cache, table, i32([0] * 4), k, v)
    q = randn(4, 2, 1, 64, seed=3)
    good = q4.q4_attention(q, cache, table, i32([38] * 4))
    cache.check()
    bad = table.clone()
    bad[1, 1] = cache.num_pages
    bad[2, 0] = -7
    lengths = i32([38, 38, 38, 47])
    got = q4.q4_attention(q, cache, bad, lengths)
    assert torch.equal(got[0], good[0]) and bool(got[1:].isnan().all())
    with pytest.raises(RuntimeError, match="page table|pool"):
        cache.check()
    cache.check()  # read once
    before = cache.pool.clone()
    q4.q4_kv_append(cache, bad, i32([0, 16, 0, -1]), k[:, :1], v[:, :1], counts=i32([0, 1, 1, 1]))
    assert torch.equal(before, cache.pool)
    with pytest.raises(RuntimeError):
        cache.check()
    assert bool(q4.q4_attention(q, cache, table, lengths, counts=i32([2, 3, 2, 2]))[1].isnan().all())
    with pytest.raises(RuntimeError):
        cache.check()
    # the same with many rows a head and room in the table (shared decoding, two kernels)
    many = randn(4, 12, 6, 64, seed=4)
    room = torch.cat([bad, torch.full((4, 200), -1, dtype=torch.int32, device=DEV)], 1)
    got = q4.q4_attention(many, cache, room, i32([28, 28, 28, -2]))
    fine = q4.q4_attention(many[:1], cache, table[:1], i32([28]))
    # row 1 misses its second page (positions 16 .. 31), which every token from 28 on sees
    assert torch.equal(got[0], fine[0]) and bool(got[1:].isnan().all())
    with pytest.raises(RuntimeError):
        cache.check()
    # a bound below the true length is noted, and that row's result is NaN
    long, lt = make_rows(q4, [600], 16, 1, 32)
    q4.q4_kv_append(long, lt, i32([0]), randn(1, 600, 1, 32), randn(1, 600, 1, 32))
    assert bool(q4.q4_attention(randn(1, 1, 1, 32), long, lt, i32([599]), max_length=256).isnan().all())
    with pytest.raises(RuntimeError):
        long.check()


def test_together_in_a_captured_graph_on_another_stream(q4):
    """A decode step of projection, append, attention and projection, captured and replayed with new inputs."""
    d, H, G, D, T = 256, 4, 2, 64, 3
    w_qkv = q4.quantize_weight(randn((H + 2 * G) * D, d, seed=1) * d ** -0.5, 64)
    w_o = q4.quantize_weight(randn(d, H * D, seed=2) * d ** -0.5, 64)
    cache, table = make_rows(q4, [200, 200], 16, G, D)
    lengths = i32([90, 0])

    def step(x):
        qkv = q4.q4_linear(x, w_qkv, out_dtype=BF).unflatten(-1, (H + 2 * G, D))
        q = q4.q4_kv_append(cache, table, lengths, qkv[:, :, H:H + G], qkv[:, :, H + G:], q=qkv[:, :, :H])
        a = q4.q4_attention(q, cache, table, lengths)
        return q4.q4_linear(a.flatten(2), w_o)

    q4.q4_kv_append(cache, table, i32([0, 0]), randn(2, 90, G, D, seed=4, dtype=BF), randn(2, 90, G, D, seed=5, dtype=BF))
    xs = [randn(2, T, d, seed=10 + i, dtype=BF) for i in range(4)]
    want = []
    for i, x in enumerate(xs):
        lengths.copy_(i32([90 + T * i, T * i]))
        want.append(step(x).clone())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    x = xs[0].clone()
    with torch.cuda.stream(side):
        step(x)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            y = step(x)
        for i in range(4):
            x.copy_(xs[i])
            lengths.copy_(i32([90 + T * i, T * i]))
            g.replay()
            assert torch.equal(y, want[i]), i
    torch.cuda.current_stream().wait_stream(side)
    cache.check()
    # and in 64 bits, from what the cache holds: the attention's inputs are the kernel's own
    assert bool(want[-1].isfinite().all())


def test_large_pool_offsets(q4):
    """Pages beyond 2^31 bytes of the pool."""
    page, G, D = 128, 8, 128
    block = q4.Q4Cache.block_bytes(D, page)
    pages = (2 ** 32) // (G * block) + 3
    cache = q4.Q4Cache(pages, G, D, page_size=page, device=DEV)
    k, v = randn(1, 130, G, D, seed=1, dtype=BF), randn(1, 130, G, D, seed=2, dtype=BF)
    far, near = i32([[pages - 1, pages - 2]]), i32([[0, 1]])
    for t in (far, near):
        q4.q4_kv_append(cache, t, i32([0]), k, v)
    q = randn(1, 2, G, D, seed=3, dtype=BF)
    assert torch.equal(q4.q4_attention(q, cache, far, i32([128])), q4.q4_attention(q, cache, near, i32([128])))
    a, b = (q4.q4_kv_read(cache, t, i32([0]), 130) for t in (far, near))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    cache.check()


# positions from 4,096 on, more than 64 rows a kv head, bf16 queries, heads of 128: the tcgen05 kernel
LONG = [  # starts, T, counts, H, G, page
    ([4096], 65, None, 1, 1, 64),
    ([4090], 13, None, 12, 2, 16),
    ([5000, 100, 4095, 7000, 0], 70, [70, 4, 2, 0, 1], 4, 4, 48),
    ([6143, 4223, 4200], 9, [9, 1, 8], 8, 1, 128),
    ([8191, 5119], 21, [21, 20], 28, 2, 32),
    ([4500], 130, None, 2, 1, 64),
    ([131070], 33, None, 2, 1, 4096),
]


@pytest.mark.parametrize("starts,T,counts,H,G,page", LONG)
def test_attention_long(q4, starts, T, counts, H, G, page):
    test_attention(q4, starts, T, counts, H, G, 128, page, BF)


@pytest.mark.parametrize("start,T,H,G", [(4088, 13, 2, 2), (7000, 13, 8, 2), (4090, 64, 1, 1)])
def test_attention_long_blocks_equal_steps(q4, start, T, H, G):
    test_attention_bits_depend_on_the_token_alone(q4, start, T, H, G, 128, BF)


@pytest.mark.parametrize("start,T,H,G", [(4088, 40, 4, 2), (7000, 13, 16, 2), (131066, 12, 8, 1)])
def test_attention_long_bits_depend_on_the_token_alone(q4, start, T, H, G):
    """Other rows, other blocks, a padded batch, another page size, bound and strides give the same bits."""
    D, end = 128, start + T
    cache, table = make_rows(q4, [end, end, 4100], 64, G, D)
    k, v = randn(3, end, G, D, seed=1, dtype=BF), randn(3, end, G, D, seed=2, dtype=BF)
    k[1], v[1] = k[0], v[0]
    q4.q4_kv_append(cache, table, i32([0, 0, 0]), k, v, counts=i32([end, end, 4100]))
    q = randn(3, T, H, D, seed=3, dtype=BF) * 2
    q[1] = q[0]
    block = q4.q4_attention(q, cache, table, i32([start, start, 4090]), counts=i32([T, T, 5]))
    assert torch.equal(block[0], block[1])
    alone = q4.q4_attention(q[:1], cache, table[:1], i32([start]), max_length=end)
    assert torch.equal(alone[0], block[0])
    # the same token at another place of a block, behind more padding
    rows = 65 * G // H + 1  # more than 64 rows a kv head
    for first in (1, T // 2):
        part = torch.zeros(1, max(rows, T + 7), H, D, dtype=BF, device=DEV)
        part[0, :T - first] = q[0, first:]
        got = q4.q4_attention(part, cache, table[:1], i32([start + first]), counts=i32([T - first]))
        assert torch.equal(got[0, :T - first], block[0, first:]), first
    other, ot = make_rows(q4, [end], 16, G, D, seed=5)
    q4.q4_kv_append(other, ot, i32([0]), k[:1], v[:1])
    wide = torch.zeros(1, T, H, D + 3, dtype=BF, device=DEV)
    wide[..., 1:D + 1] = q[0]
    assert torch.equal(q4.q4_attention(wide[..., 1:D + 1], other, ot, i32([start]))[0], block[0])
    cache.check()


def test_attention_long_unaligned_queries_and_growing_scores(q4):
    """Queries that cannot be read as words, and keys that grow along the row: the reference of the sums moves."""
    D, G, H, T, start = 128, 1, 3, 25, 4600
    cache, table = make_rows(q4, [start + T], 32, G, D)
    k, v = randn(1, start + T, G, D, seed=1, dtype=BF), randn(1, start + T, G, D, seed=2, dtype=BF)
    k *= torch.linspace(0.01, 6, start + T, device=DEV)[None, :, None, None].to(BF)
    q4.q4_kv_append(cache, table, i32([0]), k, v)
    kk, vv = q4.q4_kv_read(cache, table, i32([0]), start + T)
    wide = randn(1, T, H, D + 3, seed=3, dtype=BF)
    q = wide[..., 1:D + 1]
    out = q4.q4_attention(q, cache, table, i32([start]))
    want, av, mag = R.attend(q[0], kk[0].double(), vv[0].double(), start, D ** -0.5)
    assert bool(((out[0].double() - want).abs() <= R.attend_bound(want, av, mag, start + T, D, BF)).all())
    assert torch.equal(out, q4.q4_attention(q.contiguous(), cache, table, i32([start])))


def test_attention_long_sharp_scores(q4):
    """One key takes nearly all the weight, at every place of a step."""
    D, G, H, T, start = 128, 1, 4, 20, 4700
    cache, table = make_rows(q4, [start + T], 64, G, D)
    k, v = fill_cache(q4, cache, table, [start], [start + T], G, D)
    q = randn(1, T, H, D, seed=5, dtype=BF) * 20
    out = q4.q4_attention(q, cache, table, i32([start]), scale=0.5)
    want, av, mag = R.attend(q[0], k[0].double(), v[0].double(), start, 0.5)
    assert bool(((out[0].double() - want).abs() <= R.attend_bound(want, av, mag, start + T, D, BF)).all())


def test_attention_long_nan_groups_and_bad_pages(q4):
    D, G, H, T, start = 128, 2, 24, 7, 4400
    cache, table = make_rows(q4, [start + T, start + T], 16, G, D)
    k, v = randn(2, start + T, G, D, seed=1, dtype=BF), randn(2, start + T, G, D, seed=2, dtype=BF)
    q4.q4_kv_append(cache, table, i32([0, 0]), k, v)
    q = randn(2, T, H, D, seed=3, dtype=BF)
    clean = q4.q4_attention(q, cache, table, i32([start, start]))
    cache.check()
    vb, kb = v.clone(), k.clone()
    vb[0, start + 2, 0, 70] = math.nan  # the token at start + 2, third group of features of kv head 0
    kb[0, start + 5, 1, 1] = math.inf  # ... at start + 5, kv head 1
    q4.q4_kv_append(cache, table, i32([0, 0]), kb, vb)
    got = q4.q4_attention(q, cache, table, i32([start, start]))
    assert torch.equal(got[1], clean[1]) and torch.equal(got[0, :2], clean[0, :2])
    assert bool(got[0, 2:, :12, 64:96].isnan().all())
    keep = [i for i in range(D) if not 64 <= i < 96]
    assert torch.equal(got[0, 2:, :12][..., keep], clean[0, 2:, :12][..., keep])
    assert torch.equal(got[0, :5, 12:], clean[0, :5, 12:]) and bool(got[0, 5:, 12:].isnan().all())
    q4.q4_kv_append(cache, table, i32([0, 0]), k, v)
    bad = table.clone()
    bad[0, 200] = cache.num_pages
    got = q4.q4_attention(q, cache, bad, i32([start, start]))
    assert bool(got[0].isnan().all()) and torch.equal(got[1], clean[1])
    with pytest.raises(RuntimeError):
        cache.check()
    got = q4.q4_attention(q, cache, table, i32([start, -3]))
    assert torch.equal(got[0], clean[0]) and bool(got[1].isnan().all())
    with pytest.raises(RuntimeError):
        cache.check()


def test_outputs_that_overlap_are_refused(q4):
    D, G, H, T, B = 64, 2, 4, 3, 2
    cache, table = make_rows(q4, [40, 40], 16, G, D)
    buf = randn(B, T, (H + 2 * G + 1) * D, seed=1, dtype=BF)
    q, k, v = (buf[..., a * D:b * D].unflatten(-1, (-1, D)) for a, b in ((0, H), (H, H + G), (H + G, H + 2 * G)))
    at = i32([5, 9])
    pool = cache.pool.clone()
    for bad in (buf[..., D:(H + 1) * D], buf[..., (H + G - 2) * D:(2 * H + G - 2) * D],
                buf[0, 0, :H * D].clone().expand(B, T, H * D)):
        with pytest.raises(ValueError, match="overlap"):
            q4.q4_kv_append(cache, table, at, k, v, q=q, q_out=bad.unflatten(-1, (-1, D)))
    assert torch.equal(pool, cache.pool)
    # apart from each other: a column of the same buffer that no input holds, or q itself
    want = q4.q4_kv_append(cache, table, at, k, v, q=q)
    assert torch.equal(q4.q4_kv_append(cache, table, at, k, v, q=q, q_out=q), want) and torch.equal(q, want)
    heads_first = torch.cat([t.transpose(1, 2) for t in (randn(B, T, H, D, seed=8, dtype=BF), k, v)], 1)
    qt, kt, vt = (heads_first[:, a:b].transpose(1, 2) for a, b in ((0, H), (H, H + G), (H + G, H + 2 * G)))
    rotated = q4.q4_kv_append(cache, table, at, kt, vt, q=qt)
    assert torch.equal(q4.q4_kv_append(cache, table, at, kt, vt, q=qt, q_out=qt), rotated)
    with pytest.raises(ValueError, match="overlap"):
        q4.q4_kv_append(cache, table, at, kt, vt, q=qt, q_out=heads_first[:, 1:H + 1].transpose(1, 2))
    # attention in place equals the one into another tensor, on both launch paths
    for room in (0, 300):
        wide = torch.cat([table, torch.full((B, room), -1, dtype=torch.int32, device=DEV)], 1)
        q4.q4_kv_append(cache, wide, i32([0, 0]), *(randn(B, 12, G, D, seed=s, dtype=BF) for s in (2, 3)))
        ref = q4.q4_attention(want, cache, wide, at)
        mine = want.clone()
        assert torch.equal(q4.q4_attention(mine, cache, wide, at, out=mine), ref)
    flat = randn(B * T * H * D + 64, seed=4, dtype=BF)
    with pytest.raises(ValueError, match="overlap"):
        q4.q4_attention(flat[:-64].view(B, T, H, D), cache, table, at, out=flat[64:].view(B, T, H, D))
    with pytest.raises(ValueError, match="overlap"):
        q4.q4_attention(want, cache, table, at, out=want[:, :1].clone().expand(B, T, H, D))
    kk = torch.empty(B, T, G, D, dtype=BF, device=DEV)
    with pytest.raises(ValueError, match="overlap"):
        q4.q4_kv_read(cache, table, at, T, out=(kk, kk))
    w = q4.quantize_weight(randn(128, 128, seed=5), 64)
    x = randn(4, 128, seed=6)
    with pytest.raises(ValueError, match="overlap"):
        q4.q4_linear(x, w, out=x)
    with pytest.raises(ValueError, match="scale"):
        q4.q4_attention(want, cache, table, at, scale=2e38)


def test_workspace_follows_the_table_not_the_bound_alone(q4):
    """The same max_length with a short and then a long page table."""
    D, G, end = 32, 1, 3000
    cache, table = make_rows(q4, [end], 16, G, D)
    k, v = randn(1, end, G, D, seed=1), randn(1, end, G, D, seed=2)
    q4.q4_kv_append(cache, table, i32([0]), k, v)
    q = randn(1, 2, G, D, seed=3)
    want = q4.q4_attention(q, cache, table, i32([end - 2]))
    fresh = q4.Q4Cache.from_pool(cache.pool, head_dim=D, page_size=16)
    q4.q4_attention(q, fresh, table[:, :10].contiguous(), i32([100]), max_length=end)
    assert torch.equal(q4.q4_attention(q, fresh, table, i32([end - 2]), max_length=end), want)
    fresh.check()


@pytest.mark.parametrize("D,H,G,T,start,dtype", [(32, 4, 2, 40, 2500, F32), (128, 3, 1, 50, 2300, BF), (128, 2, 1, 130, 4000, BF),
                                                 (128, 6, 1, 50, 6000, BF)])
def test_small_workspace_takes_several_passes(q4, D, H, G, T, start, dtype):
    """The C entry with less scratch than it asks for: the same bits in more passes, and a refusal below a token."""
    import ctypes as C

    from evspark_b200 import _native as N

    end = start + T
    cache, table = make_rows(q4, [end, 7], 32, G, D)
    fill_cache(q4, cache, table, [0, 0], [end, 7], G, D, dtype=dtype)
    lengths, counts = i32([start, 2]), i32([T, 5])
    q = randn(2, T, H, D, seed=7, dtype=dtype)
    want = q4.q4_attention(q, cache, table, lengths, counts=counts)
    rows = N.Q4RowsDesc(table.data_ptr(), lengths.data_ptr(), counts.data_ptr(), table.stride(0), table.shape[1], 2, T)
    need = N.lib().evs_q4_attention_workspace(cache._ref, C.addressof(rows), H, 0)
    per_row = need // (-(-T * H // G // 16) * 16)
    strides = (C.c_int64 * 3)(*q.stride()[:3])
    for scratch in (16 * per_row, 48 * per_row, need):
        out = torch.zeros_like(q)
        ws = torch.empty(scratch, dtype=torch.uint8, device=DEV)
        q4._call(0, "evs_q4_attention", cache._ref, C.addressof(rows), q.data_ptr(), strides, H, D ** -0.5, 0,
                 out.data_ptr(), strides, q4._DT[dtype], ws.data_ptr(), scratch)
        assert torch.equal(out[0], want[0]) and torch.equal(out[1, :5], want[1, :5]) and not bool(out[1, 5:].any())
    with pytest.raises(ValueError, match="workspace"):
        q4._call(0, "evs_q4_attention", cache._ref, C.addressof(rows), q.data_ptr(), strides, H, D ** -0.5, 0,
                 out.data_ptr(), strides, q4._DT[dtype], ws.data_ptr(), 8 * per_row // 16)
    cache.check()


def test_attention_long_in_graphs_and_on_two_streams_at_once(q4):
    """The tcgen05 kernel captured, replayed with other lengths and queries, and two calls at the same time."""
    D, G, H, T, room = 128, 4, 8, 40, 9000
    cache, table = make_rows(q4, [room, room], 64, G, D)
    fill_cache(q4, cache, table, [0, 0], [room, room], G, D)
    q, lengths = randn(2, T, H, D, seed=5, dtype=BF), i32([4090, 8000])
    out = torch.zeros_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        q4.q4_attention(q, cache, table, lengths, out=out)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            q4.q4_attention(q, cache, table, lengths, out=out)
    torch.cuda.current_stream().wait_stream(side)
    for seed, starts in ((6, (8900, 5000)), (7, (100, 4500)), (8, (4096, 0))):
        q.copy_(randn(2, T, H, D, seed=seed, dtype=BF))
        lengths.copy_(i32(starts))
        graph.replay()
        assert torch.equal(out, q4.q4_attention(q, cache, table, lengths)), starts
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    qs = [randn(2, T, H, D, seed=20 + i, dtype=BF) for i in range(2)]
    at = [i32([8000, 6000]), i32([5000, 8500])]
    want = [q4.q4_attention(qs[i], cache, table, at[i]) for i in range(2)]
    got = [[], []]
    torch.cuda.synchronize()
    for _ in range(6):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(q4.q4_attention(qs[i], cache, table, at[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i])
    cache.check()


def test_captured_behind_copies_memsets_and_another_stream(q4):
    """Every call of the module in one graph, each behind another kind of work: its inputs come from a copy, a
    memset, a kernel of another stream, a kernel of its own stream and a call of the module."""
    n, k, D, G, H = 512, 256, 64, 2, 4
    w = q4.quantize_weight(randn(n, k, seed=1), 64)
    host = torch.zeros(3, k).pin_memory()
    x, y = torch.empty(3, k, device=DEV), torch.empty(3, n, device=DEV)
    cache, table = make_rows(q4, [60], 16, G, D)
    lengths = i32([50])
    qkv = torch.empty(1, 4, (H + 2 * G) * D, device=DEV)
    qkv_in = randn(1, 4, (H + 2 * G) * D, seed=2)
    fill_cache(q4, cache, table, [0], [50], G, D, dtype=F32)
    outs = [torch.zeros_like(y) for _ in range(3)]
    main, side = torch.cuda.Stream(), torch.cuda.Stream()

    def run():
        x.copy_(host, non_blocking=True)  # a copy
        q4.q4_linear(x, w, out=outs[0])
        x.zero_()  # a memset or a kernel
        q4.q4_linear(x, w, out=outs[1])
        side.wait_stream(main)
        with torch.cuda.stream(side):
            x.fill_(0.5)
            qkv.copy_(qkv_in * 2)
        main.wait_stream(side)  # a join of two streams
        q4.q4_linear(x, w, out=outs[2])
        q, kk, v = (qkv[..., a * D:b * D].unflatten(-1, (-1, D)) for a, b in ((0, H), (H, H + G), (H + G, H + 2 * G)))
        rot = q4.q4_kv_append(cache, table, lengths, kk, v, q=q)
        att = q4.q4_attention(rot, cache, table, lengths)
        with torch.cuda.stream(side):
            side.wait_stream(main)
            back = q4.q4_kv_read(cache, table, lengths, 4)
        main.wait_stream(side)
        return rot, att, *back

    main.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(main):
        host.copy_(torch.randn(3, k, generator=torch.Generator().manual_seed(0)))
        run()
        main.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=main):
            captured = run()
        for seed in (1, 2, 3):
            host.copy_(torch.randn(3, k, generator=torch.Generator().manual_seed(seed)))
            qkv_in.copy_(randn(1, 4, (H + 2 * G) * D, seed=40 + seed))
            graph.replay()
            main.synchronize()
            got = [t.clone() for t in (*outs, *captured)]
            main.synchronize()
            want = [*outs, *run()]
            main.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want)), seed
            assert torch.equal(got[0], q4.q4_linear(host.to(DEV), w)) and not bool(got[1].any())
    cache.check()
