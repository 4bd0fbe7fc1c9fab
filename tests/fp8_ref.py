"""The FP8 operators' definition in 64 bits, and bounds of what the kernels may be off by.

Sums. A product of two e4m3 codes is exact in float32, so a float32 sum over K has at most K additions
beside one multiplication by each block's scales and one addition per block: its error is at most (K +
3 G + 8) units of 2^-23 (a unit that also covers sums that round towards zero) of the sum of the
terms' magnitudes. Results of 16 bits come from the FP8 matrix instructions, which add the products of
8 neighbouring values with 13 bits below the largest one's exponent (measured: of one large product
and 7 small ones, the small ones are dropped below 2^-13 of it). Each of up to 7 products of the eight
loses a part spread over at most 2^-13 of the largest, 2^-13 / sqrt(3) rms, sqrt(7 / 3) 2^-13 together;
the eights' parts are independent, and six times their rms bounds them.

Codes. A code's own rounding is part of the definition. h of an expert is computed (gate and up as float32
sums, since a step of a code is far more than what they would lose otherwise), so a code of h may fall to the other side where h / s lies within h's error of the border between two codes, and then it
is off by one step.
"""
from __future__ import annotations

import torch

B = 128


def blocks(n: int) -> int:
    return -(-n // B)


def e4m3(v: torch.Tensor) -> torch.Tensor:
    """v (64 bits) to the nearest e4m3 number, ties to even."""
    step = e4m3_step(v)
    return torch.round(v / step) * step


def e4m3_step(v: torch.Tensor) -> torch.Tensor:
    _, e = torch.frexp(v)
    return torch.exp2((e.double() - 1).clamp(min=-6.0) - 3)


def groups(x: torch.Tensor) -> torch.Tensor:
    K = x.shape[-1]
    return torch.nn.functional.pad(x, (0, blocks(K) * B - K)).unflatten(-1, (-1, B))


def quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes' numbers [T, K], scales [T, G]) in 64 bits; x 64 bits."""
    g = groups(x)
    s = (g.abs().amax(-1) / 448).clamp(min=2.0**-126).float().double()
    return e4m3((g / s.unsqueeze(-1)).float().double()).flatten(-2)[..., : x.shape[-1]], s


def spread(s: torch.Tensor, K: int) -> torch.Tensor:
    return s.repeat_interleave(B, -1)[..., :K]


def weight(w: torch.Tensor, s: torch.Tensor) -> torch.Tensor:
    return w.double() * spread(s.double().repeat_interleave(B, -2)[: w.shape[0]], w.shape[1])


def unit(K: int) -> float:
    return (K + 3 * blocks(K) + 8) * 2.0**-23


def eights(x: torch.Tensor) -> torch.Tensor:
    """Squares of the largest magnitudes of 8 neighbours."""
    return x.unflatten(-1, (-1, 8)).abs().amax(-1) ** 2


def matmul(q: torch.Tensor, s: torch.Tensor, w: torch.Tensor, ws: torch.Tensor, wide: bool = False):
    """(y, bound of its error before the last rounding); wide: float32 sums (float32 results)."""
    x, W = q * spread(s, q.shape[1]), weight(w, ws)
    err = (x.abs() @ W.abs().t()) * unit(q.shape[1])
    if not wide:
        err += 6 * (7 / 3) ** 0.5 * 2.0**-13 * (eights(x) @ eights(W).t()).sqrt()
    return x @ W.t(), err


def check(got: torch.Tensor, want: torch.Tensor, err: torch.Tensor, what: str = "") -> None:
    """got is want, off by err and one rounding to its dtype (half a step)."""
    eps, tiny = torch.finfo(got.dtype).eps / 2, torch.finfo(got.dtype).tiny
    bound = err + (want.abs() + err) * eps + tiny
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}: "
                           f"{got[bad][0].item()} for {want[bad][0].item()} (bound {bound[bad][0].item()})")


def expert(q: torch.Tensor, s: torch.Tensor, e: dict, act: str = "silu"):
    """(y, bound) of one expert (tensors of synth.fp8_layout) for quantised tokens."""
    g, ge = matmul(q, s, e["gate_proj"], e["gate_proj_scale_inv"], wide=True)
    u, ue = matmul(q, s, e["up_proj"], e["up_proj_scale_inv"], wide=True)
    if act == "silu":
        sg, slope = g * torch.sigmoid(g), 1.1  # |silu'| < 1.1
    else:
        a, lim = 1.702, 7.0
        g, u, slope = g.clamp(max=lim), u.clamp(-lim, lim) + 1, 1.2
        sg = g * torch.sigmoid(a * g)
    h = sg * u
    # exp2 and rcp within 2 units, exp's argument rounded twice: g times 2 units more
    he = slope * ge * u.abs() + (sg.abs() + slope * ge) * ue + h.abs() * (8 + 4 * g.abs()) * 2.0**-23
    hq, hs = quantize(h)
    hsx = spread(hs, h.shape[1])
    v, step = h / hsx, e4m3_step(hq)
    top = spread((groups(he).amax(-1) / (448 * hs)), h.shape[1])  # the scale's own relative error, at most
    ve = he / hsx + v.abs() * (top + 2.0**-22)
    d, m = (v - hq).abs(), torch.frexp(hq.abs())[0]
    near = (d - step / 2).abs() <= ve  # a border half a step away, or a quarter below a power of two
    near |= (m == 0.5) & ((d - step / 4).abs() <= ve)
    qe = torch.where(near, step, 0.0) + hq.abs() * top
    y, ye = matmul(hq, hs, e["down_proj"], e["down_proj_scale_inv"])
    return y, ye + (qe * hsx) @ weight(e["down_proj"], e["down_proj_scale_inv"]).abs().t()


def moe(x: torch.Tensor, idx: torch.Tensor, w: torch.Tensor, experts: list, act: str = "silu"):
    """(y, bound) of the layer; idx < 0 (or an expert that is None) contributes nothing."""
    q, s = quantize(x.double())
    y = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    err, mag = torch.zeros_like(y), torch.zeros_like(y)
    for e in torch.unique(idx).tolist():
        if e < 0 or experts[e] is None:
            continue
        t, j = (idx == e).nonzero(as_tuple=True)
        o, oe = expert(q[t], s[t], experts[e], act)
        wt = w[t, j].double().unsqueeze(1)
        y.index_add_(0, t, wt * o)
        err.index_add_(0, t, wt.abs() * oe)
        mag.index_add_(0, t, (wt * o).abs())
    return y, err + mag * (idx.shape[1] + 4) * 2.0**-23
