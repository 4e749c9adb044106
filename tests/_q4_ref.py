"""The 4-bit format and its operators written from their definitions in 64 bits (numpy / torch, any device)."""

from __future__ import annotations

import math

import torch

F64 = torch.float64


def round5(t: torch.Tensor) -> torch.Tensor:
    m, e = torch.frexp(t)
    return torch.ldexp(torch.round(m * 32) / 32, e)


def quantize(x: torch.Tensor, group: int):
    """x [..., n], n a multiple of group -> (codes int64 [..., n], scales float64 [..., n / group])."""
    g = x.to(F64).unflatten(-1, (-1, group))
    t = g.abs().amax(-1) / 7
    t = torch.where(g.isnan().any(-1), torch.full_like(t, math.nan), t)
    s = torch.where(t < 2.0 ** -120, torch.zeros_like(t), round5(t))
    s = torch.where(t <= 2.0 ** 120, s, torch.full_like(t, math.nan))
    live = (s > 0)[..., None]
    c = torch.where(live, torch.round(g / torch.where(live, s[..., None], torch.ones_like(g))).clamp(-7, 7),
                    torch.zeros_like(g))
    return (c.to(torch.int64) + 8).flatten(-2), s


def held(x: torch.Tensor, group: int) -> torch.Tensor:
    """The values that a quantised x stands for."""
    c, s = quantize(x, group)
    return (c - 8).to(F64) * s.repeat_interleave(group, -1)


def pack(codes: torch.Tensor) -> torch.Tensor:
    return (codes[..., 0::2] | (codes[..., 1::2] << 4)).to(torch.uint8)


def rotate(x: torch.Tensor, pos: torch.Tensor, base: float = 10000.0) -> torch.Tensor:
    """x [T, heads, D] at positions pos [T]."""
    half = x.shape[-1] // 2
    ang = pos.to(F64)[:, None, None] * base ** (-torch.arange(half, dtype=F64, device=x.device) / half)
    a, b = x[..., :half].to(F64), x[..., half:].to(F64)
    return torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()], -1)


def attend(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, start: int, scale: float):
    """q [T, H, D] at positions start.., k and v [keys, G, D] in 64 bits -> (out [T, H, D], sum p |v| / sum p,
    largest scale * sum |q k| of a row)."""
    T, H, D = q.shape
    G = k.shape[1]
    kk, vv = k.repeat_interleave(H // G, 1), v.repeat_interleave(H // G, 1)
    s = torch.einsum("thd,khd->thk", q.to(F64), kk) * scale
    mag = torch.einsum("thd,khd->thk", q.to(F64).abs(), kk.abs().nan_to_num()) * abs(scale)
    hidden = torch.arange(k.shape[0], device=q.device)[None, :] > start + torch.arange(T, device=q.device)[:, None]
    s = s.masked_fill(hidden[:, None], -math.inf)
    mag = mag.masked_fill(hidden[:, None], 0).amax(-1)
    p = torch.softmax(s, -1)
    out = torch.zeros(T, H, D, dtype=F64, device=q.device)
    av = torch.zeros_like(out)
    for t in range(T):  # a hidden key must not enter the sum, not even as 0 NaN
        n = start + t + 1
        out[t] = torch.einsum("hk,khd->hd", p[t, :, :n], vv[:n])
        av[t] = torch.einsum("hk,khd->hd", p[t, :, :n], vv[:n].abs())
    return out, av, mag


def linear_bound(x: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    """How far fp32 sums of exact products may be off: every product step of 16 features cuts at most 2^-22 of
    the sum of magnitudes (operand alignment and the add, both by truncation), as does each of the at most
    20 adds of partial sums; three-part fp32 rows run three product steps per 16 features."""
    steps = 3 * -(-x.shape[-1] // 16) + 20
    return steps * 2.0 ** -22 * (x.to(F64).abs() @ w.to(F64).abs().t())


def attend_bound(out, av, mag, keys: int, D: int, dtype: torch.dtype) -> torch.Tensor:
    """A score is off by at most (3 D / 16 + 2) 2^-22 of its sum of magnitudes (fp32 product steps, the scale)
    and one rounding of its base-2 exponent (2^-23 of it); a weight exp2(s - m) by that (times ln 2 < 1,
    both s and m), by 2^-22 of the exponential and by its rounding as a product operand (bf16 queries: one
    bf16 part, half a step of at most 2^-8 of the weight; fp32: three parts, 2^-24).  Sums over n keys add
    (n / 16 + 40) 2^-22 (product steps, folds).  Numerator and denominator each move by that relative
    error: twice it, times sum p |v| / sum p; then one rounding to the type.
    fp32 and bf16 hold nothing below 2^-126 at full precision: the second part of a weight under 2^-110
    of the largest (2^-8 of it, so under 2^-118) may be lost, and with it 2^-118 |v| of each of the n
    keys, |v| being at most 2^6 in these tests: the sum of the weights is at least the largest."""
    parts = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
    rel = 2 * ((3 * D / 16 + 4) * 2.0 ** -22 * 1.5 * mag) + 2.0 ** -22 + parts + (3 * keys / 16 + 40) * 2.0 ** -22
    return 2 * rel[..., None] * av + torch.finfo(dtype).eps / 2 * out.abs() + keys * 2.0 ** -112
