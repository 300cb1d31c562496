"""Plain 64-bit forms of the operators around a 4-bit paged cache, from their definitions, for the tests.

Tolerances are bounds, not measurements.  A rounding to a type is off by at most eps / 2 of the value (bf16 2^-8, fp16 2^-11,
fp32 2^-24)."""

from __future__ import annotations

import math
from typing import List, Optional, Sequence

import torch

D = 128
GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
# All non-negative e4m3 values by their byte (the byte 0x7f is a not-a-number and never stored).
E4M3 = torch.tensor([(m / 8.0) * 2.0 ** -6 if e == 0 else (1 + m / 8.0) * 2.0 ** (e - 7) for e in range(16) for m in range(8)][:127],
                    dtype=torch.float64)


def _nearest(values: torch.Tensor, table: torch.Tensor) -> torch.Tensor:
    """Index of the nearest entry of an ascending table, ties to the even index."""
    hi = torch.searchsorted(table, values).clamp(1, table.numel() - 1)
    lo = hi - 1
    mid = (table[lo] + table[hi]) / 2
    up = (values > mid) | ((values == mid) & (hi % 2 == 0))
    return torch.where(up, hi, lo)


def quantise(x: torch.Tensor, scale: float = 1.0):
    """(codes uint8 [..., 64], scales uint8 [..., 8]) of bf16 x [..., 128]."""
    y = x.double() / scale
    y = torch.where(torch.isnan(y), torch.zeros_like(y), y).clamp(-2688.0, 2688.0).reshape(*x.shape[:-1], 8, 16)
    s = _nearest(y.abs().amax(-1) / 6.0, E4M3).clamp_min(1)
    mag = _nearest((y.abs() / E4M3[s].unsqueeze(-1)).clamp_max(6.0), GRID)
    neg = torch.signbit(y)
    code = (mag + 8 * neg.long()).to(torch.uint8).reshape(*x.shape[:-1], 64, 2)
    return code[..., 0] | (code[..., 1] << 4), s.to(torch.uint8)


def values(codes: torch.Tensor, scales: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """float64 values [..., 128]."""
    c = torch.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], 8, 16).long()
    v = GRID[c & 7] * torch.where(c >= 8, -1.0, 1.0).double() * E4M3[scales.long()].unsqueeze(-1)
    return v.reshape(*codes.shape[:-1], D) * scale


def attend(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, n: int, scale: float):
    """One request: q [n_q, NH_q, 128], k / v float64 [len, NH_kv, 128] (len = n).  Returns (out, lse, bound) in float64.

    The bound of |kernel - out|: bf16 rounding of the result; probabilities rounded to fp16 (relative 2^-11, or 2^-25 of the
    largest where they are tiny); fp32 scores of 128 products (128 * 2^-23 of the sum of their magnitudes, twice: once
    in the numerator, once in the sum); fp32 sums over n tokens (n * 2^-23)."""
    n_q, nh_q, _ = q.shape
    nh_kv = k.shape[1]
    g = nh_q // nh_kv
    qd = q.double().reshape(n_q, nh_kv, g, D)
    out = torch.zeros(n_q, nh_q, D, dtype=torch.float64)
    lse = torch.full((n_q, nh_q), -math.inf, dtype=torch.float64)
    bound = torch.full((n_q, nh_q, D), 1e-30, dtype=torch.float64)
    for j in range(n_q):
        m = n - n_q + 1 + j
        if m <= 0:
            continue
        kk, vv = k[:m], v[:m]
        s = torch.einsum("hgd,thd->hgt", qd[j], kk) * scale
        size = torch.einsum("hgd,thd->hgt", qd[j].abs(), kk.abs()).amax(-1) * abs(scale)
        lse[j] = torch.logsumexp(s, -1).reshape(-1)
        p = torch.softmax(s, -1)
        o = torch.einsum("hgt,thd->hgd", p, vv)
        a = torch.einsum("hgt,thd->hgd", p, vv.abs())
        delta = size * 128 * 2.0 ** -23
        rel = 2.0 ** -11 + 2 * delta + m * 2.0 ** -23 + 2.0 ** -20
        top = vv.abs().amax(0)[:, None, :]
        b = o.abs() * 2.0 ** -8 + a * rel.unsqueeze(-1) + m * 2.0 ** -25 * top
        out[j], bound[j] = o.reshape(nh_q, D), b.reshape(nh_q, D) + 1e-30
    return out, lse, bound


def slots_of(table_row: Sequence[int], n: int, page_size: int) -> List[int]:
    return [int(table_row[t // page_size]) * page_size + t % page_size for t in range(n)]


def norm_rope(x: torch.Tensor, w: Optional[torch.Tensor], positions: Optional[torch.Tensor], cos_sin: Optional[torch.Tensor], eps: float):
    """(y, bound): float64 of x [T, NH, 128] bf16.  fp32 arithmetic: the mean of 128 squares and its root are off by at most
    130 * 2^-24, the products and the rotation by 8 * 2^-24 of the magnitudes they combine; then one bf16 rounding."""
    y = x.double()
    if w is not None:
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * w.double()
    size = y.abs()
    if cos_sin is not None:
        ok = (positions >= 0) & (positions < cos_sin.shape[0])
        cs = cos_sin.double()[positions.clamp(0, cos_sin.shape[0] - 1).long()]
        c = torch.where(ok[:, None], cs[:, :64], torch.ones_like(cs[:, :64]))[:, None]
        s = torch.where(ok[:, None], cs[:, 64:], torch.zeros_like(cs[:, 64:]))[:, None]
        lo, hi = y[..., :64], y[..., 64:]
        a = size[..., :64] * c.abs() + size[..., 64:] * s.abs()
        b = size[..., 64:] * c.abs() + size[..., :64] * s.abs()
        y, size = torch.cat([lo * c - hi * s, hi * c + lo * s], -1), torch.cat([a, b], -1)
    return y, y.abs() * 2.0 ** -8 + size * 138 * 2.0 ** -24 + 1e-38


class Pages:
    """The stack of free pages and the table, in Python lists."""

    def __init__(self, table: torch.Tensor, free: torch.Tensor, n_free: int, page: int):
        self.table, self.stack, self.n, self.page = table.clone(), free.tolist(), n_free, page

    def assign(self, rows, lens, new):
        slots, positions, cu = [], [], [0]
        for r, a, m in zip(rows, lens, new):
            for t in range(a, a + m):
                if t % self.page == 0:
                    self.n -= 1
                    self.table[r, t // self.page] = self.stack[self.n]
                slots.append(int(self.table[r, t // self.page]) * self.page + t % self.page)
                positions.append(t)
            cu.append(len(slots))
        return slots, positions, [a + m for a, m in zip(lens, new)], cu

    def release(self, rows, lens, keep):
        freed = []
        for r, a, k in zip(rows, lens, keep):
            freed += [int(self.table[r, i]) for i in range(-(-k // self.page), -(-a // self.page))]
        for number in reversed(freed):
            self.stack[self.n] = number
            self.n += 1
