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


def _act(g, ge, u, ue, act: str):
    """(h, bound of its error) of the activation on gate and up with their errors."""
    if act == "silu":
        sg, slope = g * torch.sigmoid(g), 1.1  # |silu'| < 1.1
    else:
        a, lim = 1.702, 7.0
        g, u, slope = g.clamp(max=lim), u.clamp(-lim, lim) + 1, 1.2
        sg = g * torch.sigmoid(a * g)
    h = sg * u
    # exp2 and rcp within 2 units, exp's argument rounded twice: g times 2 units more
    return h, slope * ge * u.abs() + (sg.abs() + slope * ge) * ue + h.abs() * (8 + 4 * g.abs()) * 2 * U


def expert8(q, s, e: dict, act: str = "silu"):
    """(y, bound) of an int8 expert (tensors of synth.int8_layout) for quantised tokens. A code of h may be that of any
    h / s within h's error."""
    h, he = _act(*matmul(q, s, e["gate_proj"], e["gate_proj_scale"]), *matmul(q, s, e["up_proj"], e["up_proj_scale"]), act)
    hq, hs = quantize(h)
    v, top = h / hs, he.amax(1, keepdim=True) / (127 * hs) + 2 * U  # the scale's own relative error, at most
    ve = he / hs + v.abs() * (top + 2 * U)
    qe = torch.maximum((torch.round(v + ve) - hq).abs(), (torch.round(v - ve) - hq).abs()) + hq.abs() * top
    y, ye = matmul(hq, hs, e["down_proj"], e["down_proj_scale"])
    return y, ye + ((qe * hs) @ e["down_proj"].double().abs().t()) * e["down_proj_scale"].double()


def expert16(x, e: dict, act: str = "silu"):
    """(y, bound) of a 16-bit expert: h is rounded to the weights' type, as any number within its error may be."""
    dt = e["down_proj"].dtype
    h, he = _act(*matmul16(x, e["gate_proj"]), *matmul16(x, e["up_proj"]), act)
    hr = h.to(dt).double()
    qe = torch.maximum(((h + he).to(dt).double() - hr).abs(), ((h - he).to(dt).double() - hr).abs())
    y, ye = matmul16(hr, e["down_proj"])
    return y, ye + qe @ e["down_proj"].double().abs().t()


def moe(x, idx, w, experts: list, act: str = "silu"):
    """(y, bound) of the layer; idx < 0 (or an expert that is None) contributes nothing."""
    int8 = next(e for e in experts if e is not None)["down_proj"].dtype == torch.int8
    q, s = quantize(x) if int8 else (x.double(), None)
    y = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    err, mag = torch.zeros_like(y), torch.zeros_like(y)
    for e in torch.unique(idx).tolist():
        if e < 0 or experts[e] is None:
            continue
        t, j = (idx == e).nonzero(as_tuple=True)
        o, oe = expert8(q[t], s[t], experts[e], act) if int8 else expert16(q[t], experts[e], act)
        wt = w[t, j].double().unsqueeze(1)
        y.index_add_(0, t, wt * o)
        err.index_add_(0, t, wt.abs() * oe)
        mag.index_add_(0, t, (wt * o).abs())
    return y, err + mag * (idx.shape[1] + 4) * 2 * U
