"""The 4-bit format at its borders: scales at and around a tie of the five-bit rounding, values at and around the
halves between two codes, sizes at which a scale becomes zero or NaN."""

from __future__ import annotations

import math

import pytest
import torch

from tests import _q4_ref as R
from tests.test_gpu_q4 import BF, DEV, F32, i32, make_rows, q4, randn  # noqa: F401  (q4: the module's fixture)

pytestmark = pytest.mark.gpu


def near(x: float, dtype) -> list[float]:
    """x and its neighbours in the type."""
    t = torch.tensor(x, dtype=dtype)
    step = torch.finfo(dtype).eps * 2.0 ** math.floor(math.log2(x))
    return [float((t.double() + d * step).to(dtype)) for d in (-2, -1, 0, 1, 2)]


def border_groups(dtype) -> torch.Tensor:
    """Groups of 32: absmax around every tie of the scale's rounding, values around every half of the scale."""
    rows = []
    for m in range(16):  # ties of five bits: 1 + m / 16 + 1 / 32
        for absmax in near(7 * (1 + m / 16 + 1 / 32), dtype):
            _, s = R.quantize(torch.full((32,), absmax, dtype=torch.float64), 32)
            halves = [v for n in range(7) for v in near((n + 0.5) * float(s), dtype)[1:4]]
            row = (torch.tensor([absmax] + halves, dtype=torch.float64)[:32]).to(dtype)
            row = torch.cat([row, torch.full((32 - row.numel(),), absmax, dtype=dtype)]).clamp(max=absmax)
            rows.append(row * torch.where(torch.arange(32) % 3 == 1, -1, 1).to(dtype))
    g = torch.stack(rows)
    return torch.cat([g, g * 2.0 ** -100, g * 2.0 ** 90]).to(DEV)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_weight_borders(q4, dtype):  # noqa: F811
    g = border_groups(dtype)
    for group in (32, 64, 128):
        w = g[:g.shape[0] // 4 * 4].reshape(-1, 128) if group > 32 else g.reshape(-1, 32)
        qw = q4.quantize_weight(w, group)
        padded = torch.zeros(w.shape[0], 128, dtype=torch.float64, device=DEV)
        padded[:, :w.shape[1]] = w.double()
        codes, scales = R.quantize(padded, group)
        assert torch.equal(qw.codes, R.pack(codes)) and torch.equal(qw.scales.double(), scales.t())


@pytest.mark.parametrize("D,dtype", [(32, BF), (64, F32), (128, BF), (128, F32)])
def test_cache_borders(q4, D, dtype):  # noqa: F811
    """Values as they are, and keys at position 0 (which the rotation leaves as they are)."""
    g = border_groups(dtype)
    x = g[:g.shape[0] // (D // 32) * (D // 32)].reshape(1, -1, 1, D)
    T = x.shape[1]
    cache, table = make_rows(q4, [T], 16, 1, D)
    k = randn(1, T, 1, D, seed=1, dtype=dtype)
    q4.q4_kv_append(cache, table, i32([0]), k, x)
    _, vv = q4.q4_kv_read(cache, table, i32([0]), T, dtype=F32)
    assert torch.equal(vv[0, :, 0].double(), R.held(x[0, :, 0].double(), 32))
    rows, tables = x[0, :, 0].reshape(T, 1, 1, D), torch.arange(T, dtype=torch.int32, device=DEV)[:, None]
    each = q4.Q4Cache(T, 1, D, page_size=16, device=DEV)
    zero = torch.zeros(T, dtype=torch.int32, device=DEV)
    q4.q4_kv_append(each, tables, zero, rows, rows)
    kk, vv = q4.q4_kv_read(each, tables, zero, 1, dtype=F32)
    want = R.held(rows.double(), 32)
    assert torch.equal(kk.double(), want) and torch.equal(vv.double(), want)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_smallest_and_largest_scales(q4, dtype):  # noqa: F811
    """absmax / 7 around 2^-120 (below: zeros) and 2^120 (above: NaN)."""
    edges = [a * sign for e in (2.0 ** -120, 2.0 ** 120) for a in near(7 * e, dtype) for sign in (1, -1)]
    x = torch.tensor(edges, dtype=dtype, device=DEV)[:, None] * torch.linspace(0, 1, 32, device=DEV).to(dtype)
    want = R.held(x.double(), 32)
    got = q4.quantize_weight(x, 32).dequantize(F32).double()
    assert torch.equal(got.nan_to_num(nan=7.0), want.nan_to_num(nan=7.0)) and 0 < int(want.isnan().sum()) < want.numel()
    T = x.shape[0]
    cache, table = make_rows(q4, [T], 16, 1, 32)
    v = x.reshape(1, T, 1, 32)
    q4.q4_kv_append(cache, table, i32([0]), torch.zeros_like(v), v)
    _, vv = q4.q4_kv_read(cache, table, i32([0]), T, dtype=F32)
    assert torch.equal(vv[0, :, 0].double().nan_to_num(nan=7.0), want.nan_to_num(nan=7.0))
