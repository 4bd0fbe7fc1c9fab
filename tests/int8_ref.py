"""The int8 and the grouped operators' definition in 64 bits, and bounds of what the kernels may be off by.

int8. Codes and scales are the definition's own, bit for bit. A product's sum is exact; it is rounded to
float32 once, multiplied by the rounded product of the scales and added to the bias: four roundings to
float32, each of at most 2^-24 of a number that is at most |sum sx sw| + |bias| (and what the others add).

16 bits. A product of two bf16 or fp16 numbers is exact in float32; a sum of K of them has at most K additions,
each off by at most 2^-23 (a unit that also covers sums that round towards zero) of the terms' magnitudes.
"""
from __future__ import annotations

import torch

U = 2.0**-24


def quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales [T, 1]) in 64 bits; x in any type."""
    v = x.double()
    s = (v.abs().amax(1, keepdim=True) / 127).clamp(min=2.0**-126).float().double()
    return torch.round((v / s).float().double()), s


def matmul(q: torch.Tensor, s: torch.Tensor, w: torch.Tensor, ws: torch.Tensor, bias: torch.Tensor | None = None):
    """(y, bound of its error before the last rounding); q, s as quantize gives them, w codes [N, K], ws [N]."""
    y = (q @ w.double().t()) * s * ws.double()
    if bias is None:
        return y, 4 * U * y.abs()
    b = bias.double()
    return y + b, 5 * U * (y.abs() + b.abs())


def matmul16(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor | None = None):
    x, w = x.double(), w.double()
    y, mag = x @ w.t(), x.abs() @ w.abs().t()
    err = (x.shape[1] + 8) * 2 * U * mag
    return (y, err) if bias is None else (y + bias.double(), err + 2 * U * (mag + bias.double().abs()))


def check(got: torch.Tensor, want: torch.Tensor, err: torch.Tensor, what: str = "") -> None:
    """got is want, off by err and one rounding to its dtype (half a step)."""
    eps, tiny = torch.finfo(got.dtype).eps / 2, torch.finfo(got.dtype).tiny
    bound = err + (want.abs() + err) * eps + tiny
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}: "
                           f"{got[bad][0].item()} for {want[bad][0].item()} (bound {bound[bad][0].item()})")


def weights8(g: torch.Generator, *shape, sigma: float = 0.03) -> tuple[torch.Tensor, torch.Tensor]:
    """int8 codes [..., N, K] and scales [..., N] of N(0, sigma) matrices."""
    w = sigma * torch.randn(shape, device=g.device, generator=g)
    s = w.abs().amax(-1) / 127
    return torch.round(w / s.unsqueeze(-1)).clamp(-127, 127).to(torch.int8), s


def grouped(x, w, offsets: list[int], bias=None, rows: list[int] | None = None, top_k: int = 1, int8=None):
    """(y [R, N], bound): x [T, K], w [E, N, K]; int8: the weights' scales [E, N], x (codes, scales)."""
    R = len(rows) if rows is not None else (x[0] if int8 is not None else x).shape[0]
    T = (x[0] if int8 is not None else x).shape[0]
    N, dev = w.shape[1], w.device
    y, err = torch.zeros((R, N), dtype=torch.float64, device=dev), torch.zeros((R, N), dtype=torch.float64, device=dev)
    for e in range(len(offsets) - 1):
        a, b = max(0, offsets[e]), min(R, offsets[e + 1])
        if a >= b:
            continue
        at = [r // top_k if r >= 0 else -1 for r in rows[a:b]] if rows is not None else list(range(a, b))
        at = torch.tensor([t if 0 <= t < T else T for t in at], device=dev)
        be = None if bias is None else bias[e]
        pad = lambda v: torch.cat([v.double(), v.new_zeros((1, v.shape[1])).double()])[at]  # noqa: E731  (row T: zeros)
        if int8 is not None:
            y[a:b], err[a:b] = matmul(pad(x[0]), pad(x[1]), w[e], int8[e], be)
        else:
            y[a:b], err[a:b] = matmul16(pad(x), w[e], be)
    return y, err
