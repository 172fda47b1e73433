"""The 8-bit cache written out: e4m3 numbers with a power of two a row, in 64 bits, and attention over what it holds."""

from __future__ import annotations

import math

import torch

LOW, HIGH, TOP = -64, 119, 448.0


def exponent_of(row: torch.Tensor) -> torch.Tensor:
    """The smallest e with max |x| <= 448 * 2^e over a row's finite numbers, kept within LOW .. HIGH."""
    x = row.double().abs()
    top = torch.where(torch.isfinite(x), x, torch.zeros_like(x)).amax(-1)
    out = torch.full(top.shape, LOW, dtype=torch.int64)
    for e in range(HIGH - 1, LOW - 1, -1):  # the last power that is too small, plus one
        out = torch.maximum(out, torch.where(top > TOP * 2.0**e, torch.full_like(out, e + 1), out))
    return out


def nearest8(y: torch.Tensor) -> torch.Tensor:
    """The nearest e4m3 number of each y, ties to the even one: steps of an eighth of the number's power of two, of 2^-9 below 2^-6."""
    y = y.double()
    _, power = torch.frexp(y.abs().clamp_min(2.0**-6))  # y = part * 2^power, part in [0.5, 1)
    step = torch.ldexp(torch.ones_like(y), power - 4)
    out = (torch.round(y / step) * step).clamp(-TOP, TOP)
    return torch.where(torch.isfinite(y), out, torch.full_like(y, math.nan))


def quantised(row: torch.Tensor) -> torch.Tensor:
    """What the cache gives back for rows (the last dimension), in the rows' type."""
    e = exponent_of(row).unsqueeze(-1)
    power = 2.0 ** e.double()
    return (nearest8(row.double() / power) * power).to(row.dtype)


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, past: int, window: int = 0, sink: bool = False) -> torch.Tensor:
    """A sequence's last tokens ``q [T, n_q, d]`` at the positions past .. over its keys and values ``[S, n_kv, d]``, 64 bits."""
    q, k, v = q.double(), k.double(), v.double()
    out = torch.zeros_like(q)
    group = q.shape[1] // k.shape[1]
    for t in range(q.shape[0]):
        pos = past + t
        lo = max(0, pos + 1 - window) if window else 0
        if pos < lo:
            continue
        for h in range(q.shape[1]):
            s = k[lo:pos + 1, h // group] @ q[t, h] * q.shape[2] ** -0.5
            top = s.max().clamp_min(0.0) if sink else s.max()
            p = torch.exp(s - top)
            out[t, h] = (p @ v[lo:pos + 1, h // group]) / (p.sum() + (torch.exp(-top) if sink else 0.0))
    return out
