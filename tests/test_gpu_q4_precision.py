"""Attention over the 4-bit cache where a loose bound would hide a fault: weights that nearly cancel, one key that
carries the weight at every border of the split, outputs inside larger tensors."""

from __future__ import annotations

import pytest
import torch

from tests import _q4_ref as R
from tests.test_gpu_q4 import DEV, fill_cache, i32, make_rows, q4, randn  # noqa: F401  (q4: the module's fixture)

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def tight_bound(out, av, mag, keys: int, D: int, dtype: torch.dtype) -> torch.Tensor:
    """A score: D / 16 product steps (three times as many for the three parts of fp32 queries) and the fold of their
    parts cut at most 2^-22 of its sum of magnitudes each, the rounded scale and the fma of its exponent add
    2 2^-23 + 2^-24 of it.  The exponentials (one of the weight, at most seven of moved references and folds) add
    2^-22 each.  These move numerator and denominator alike: twice.  The sums over the keys are cut in each product
    step (three parts at most) and in at most 40 folds: twice 2^-22 of the sum of magnitudes.  A weight as a product
    operand is two bf16 parts, 2^-18 of it (fp32: three, 2^-24), in the numerator alone.  One rounding to the type.
    What fp32 and bf16 do not hold below 2^-126: as in R.attend_bound."""
    bf = dtype == BF
    score = ((1 if bf else 3) * D / 16 + 4) * 2.0 ** -22 * mag + 8 * 2.0 ** -22
    rel = 2 * score + 2 * (3 * keys / 16 + 40) * 2.0 ** -22 + (2.0 ** -18 if bf else 2.0 ** -24)
    return (1 + 2.0 ** -8) * rel[..., None] * av + torch.finfo(dtype).eps / 2 * out.abs() + keys * 2.0 ** -112


def check(q4, cache, table, q, kk, vv, start, D, scale=None):
    out = q4.q4_attention(q, cache, table, i32([start]), scale=scale)
    cache.check()
    want, av, mag = R.attend(q[0], kk[0].double(), vv[0].double(), start, scale or D ** -0.5)
    bound = tight_bound(want, av, mag, start + q.shape[1], D, q.dtype)
    err = (out[0].double() - want).abs()
    assert bool((err <= bound).all()), float((err / bound).max())
    return out


# one cluster, two kernels (16-row tiles), the tcgen05 kernel, fp32
CANCEL = [(2, 13, 8, 2, 128, BF), (0, 6, 4, 4, 64, BF), (2600, 13, 4, 1, 128, BF), (2600, 9, 4, 2, 32, BF),
          (5000, 13, 4, 4, 128, BF), (4700, 40, 4, 2, 128, BF), (20, 5, 2, 1, 64, F32)]


@pytest.mark.parametrize("start,T,H,G,D,dtype", CANCEL)
def test_weights_that_nearly_cancel(q4, start, T, H, G, D, dtype):  # noqa: F811
    """Two keys alone have values, opposite ones: the output is the difference of two weights, far below their sum."""
    end = start + T
    cache, table = make_rows(q4, [end], 32, G, D)
    k, v = randn(1, end, G, D, seed=1, dtype=dtype), torch.zeros(1, end, G, D, dtype=dtype, device=DEV)
    at = start // 2
    v[0, 0] = randn(G, D, seed=2, dtype=dtype)
    v[0, at + 1] = -v[0, 0]
    q4.q4_kv_append(cache, table, i32([0]), k, v)
    kk, vv = q4.q4_kv_read(cache, table, i32([0]), end, dtype=F32)
    check(q4, cache, table, randn(1, T, H, D, seed=3, dtype=dtype), kk, vv, start, D)


BORDERS = [0, 15, 16, 127, 128, 1023, 1024, 1151, 2047, 2048, 4095, 4096, 5119, 5120, 8191, 8192, 16383, 16384, 16447,
           16448, 18431, 18432]


@pytest.mark.parametrize("rows", [1, 80])  # 16-row tiles; more than 64 rows a kv head: tcgen05 from 4,096 on
@pytest.mark.parametrize("start", [2040, 4094, 18440])
def test_one_key_carries_the_weight_at_every_border(q4, start, rows):  # noqa: F811
    """Token t's query is a multiple of the key at a border of units, slots, classes or pages."""
    D, T = 128, 12
    end = start + T
    cache, table = make_rows(q4, [end], 48, 1, D)
    kk, vv = fill_cache(q4, cache, table, [start], [end], 1, D)
    H = -(-rows // T)
    places = [p for p in BORDERS if p <= start] + [start]
    for at in range(0, len(places), T):
        some = (places[at:at + T] * T)[:T]
        q = (4 * kk[:, some].float()).to(BF).expand(1, T, H, D)
        out = check(q4, cache, table, q, kk, vv, start, D)
        # the other keys' weights are below e^-10 in sum
        assert float((out[0, :, 0].float() - vv[0, some, 0].float()).abs().max()) < 0.05


@pytest.mark.parametrize("start,T,H,G,D,dtype", [(40, 5, 4, 2, 64, BF), (2500, 5, 4, 2, 64, F32), (5000, 40, 4, 2, 128, BF)])
def test_output_inside_a_larger_tensor(q4, start, T, H, G, D, dtype):  # noqa: F811
    """Rows at odd offsets, heads before tokens: the same bits, and nothing around them is written."""
    cache, table = make_rows(q4, [start + T], 32, G, D)
    fill_cache(q4, cache, table, [start], [start + T], G, D, dtype=dtype)
    q = randn(1, T, H, D, seed=4, dtype=dtype)
    want = q4.q4_attention(q, cache, table, i32([start]))
    wide = torch.full((1, H + 2, T + 1, D + 5), 7.0, dtype=dtype, device=DEV)
    out = wide[:, 1:H + 1, :T, 3:D + 3].transpose(1, 2)
    assert q4.q4_attention(q, cache, table, i32([start]), out=out).data_ptr() == out.data_ptr()
    assert torch.equal(out, want)
    out.fill_(7.0)
    assert bool((wide == 7).all())


@pytest.mark.parametrize("dtype", [BF, F32])
def test_rotated_queries_and_read_back_inside_larger_tensors(q4, dtype):  # noqa: F811
    D, G, H, T, start = 64, 2, 4, 9, 30
    cache, table = make_rows(q4, [start + T], 16, G, D)
    k, v, q = (randn(1, T, n, D, seed=s, dtype=dtype) for n, s in ((G, 1), (G, 2), (H, 3)))
    want = q4.q4_kv_append(cache, table, i32([start]), k, v, q=q)
    kk, vv = q4.q4_kv_read(cache, table, i32([start]), T, dtype=dtype)
    wide = torch.full((3, 1, H + 1, T + 2, D + 3), 7.0, dtype=dtype, device=DEV)
    q_out, k_out, v_out = (wide[i, :, 1:1 + n, 1:T + 1, 1:D + 1].transpose(1, 2) for i, n in enumerate((H, G, G)))
    q4.q4_kv_append(cache, table, i32([start]), k, v, q=q, q_out=q_out)
    q4.q4_kv_read(cache, table, i32([start]), T, out=(k_out, v_out))
    assert torch.equal(q_out, want) and torch.equal(k_out, kk) and torch.equal(v_out, vv)
    for t in (q_out, k_out, v_out):
        t.fill_(7.0)
    assert bool((wide == 7).all())
    cache.check()
