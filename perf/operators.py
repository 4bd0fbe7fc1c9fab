"""The FP8 operators: weights and activations in e4m3 with a scale for each block of 128.

A weight matrix [N, K] is e4m3 codes and one float32 scale per block of 128 x 128 (the last blocks of
a side may be short). Activations are quantised where they are used, a float32 scale for each token
and 128 columns:

    scale = max(max|x| / 448, 2^-126)        (float32)
    code  = e4m3(x / scale)                  (float32 quotient, then round to nearest even)

``quantize`` is that step by itself, ``linear`` the quantised product y = x W^T (+ bias) from 16-bit
activations, ``matmul`` the same from codes that several projections share, ``decode`` a
mixture-of-experts layer for a few tokens and ``moe`` one for batches and prompts: route, then per
expert h = silu(x Wg^T) * (x Wu^T) in float32, h quantised by the same rule, y = sum_j w_j h Wd^T.

A case is a dict of plain values. Where ``own`` is false, ``run`` is the plain form of the operator in
32 bits; where it is true, the framework's call. ``exact`` is the definition in 64 bits.
"""
from __future__ import annotations

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
E4M3 = torch.float8_e4m3fn
B = 128       # values that share a scale
WSTD = 0.03   # the weights' standard deviation

# the two layer shapes of the benchmark: many small experts, few large ones (whose sides end in half a block)
SMALL = {"H": 2048, "I": 768, "E": 128, "k": 8}
LARGE = {"H": 2880, "I": 2880, "E": 32, "k": 4}


# ----------------------------------------------------------------------------- the cases
def listed() -> list[dict]:
    return [
        # the activations of a decode batch ahead of the projections that share them: launch latency
        {"name": "quantize batch", "op": "quantize", "T": 24, "K": 2880, "dtype": "bf16"},
        # the same over a long prompt; 2880 ends in half a group
        {"name": "quantize prompt", "op": "quantize", "T": 4096, "K": 2880, "dtype": "bf16"},
        # one projection of a decode step, called by itself: launch and call latency
        {"name": "linear one token", "op": "linear", "N": 2880, "K": 2880, "T": 1, "dtype": "bf16", "bias": True},
        # the same kind of layer for a decode batch of 24 sequences
        {"name": "linear batch", "op": "linear", "N": 2048, "K": 4096, "T": 24, "dtype": "bf16", "bias": False},
        # an expert's two halves as a module of their own, over the tokens a prompt sends there
        {"name": "linear 77 tokens", "op": "linear", "N": 5760, "K": 2880, "T": 77, "dtype": "bf16", "bias": False},
        # the query projection over a prompt of 512 tokens, quantised once for q, k and v
        {"name": "matmul prompt", "op": "matmul", "N": 4096, "K": 2048, "T": 512, "dtype": "bf16", "bias": False},
        # the widest projection over a long prompt: where the matrix cores are the bound
        {"name": "linear long prompt", "op": "linear", "N": 5760, "K": 2880, "T": 4096, "dtype": "bf16", "bias": True},
        # one token, and four, through a stack of MoE layers, as a captured decode step replays it
        {"name": "moe decode", "op": "decode", **SMALL, "layers": 8, "T": 1},
        {"name": "moe decode 4", "op": "decode", **LARGE, "layers": 8, "T": 4},
        # a decode batch of 24 sequences through one MoE layer: most experts get a token or two
        {"name": "moe batch", "op": "moe", **SMALL, "T": 24},
        # prompts: 1024 tokens over many experts, 2048 over few
        {"name": "moe prompt", "op": "moe", **SMALL, "T": 1024},
        {"name": "moe long prompt", "op": "moe", **LARGE, "T": 2048},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng) -> dict:
    """One more case of the same kinds: sizes over the logarithm of their range, odd ones among them."""
    op = rng.choice(["quantize", "linear", "linear", "linear", "matmul", "matmul", "decode", "decode", "moe", "moe",
                     "moe"])
    if op == "quantize":
        return {"op": op, "T": _log_int(rng, 1, 4096), "K": 16 * _log_int(rng, 16, 180),
                "dtype": rng.choice(["bf16", "bf16", "f16", "f32"])}
    if op in ("linear", "matmul"):
        N, K = rng.choice([(2880, 2880), (4096, 2048), (2048, 4096), (512, 2048), (768, 2048), (5760, 2880),
                           (_log_int(rng, 300, 5760), 16 * _log_int(rng, 16, 180)),
                           (_log_int(rng, 300, 5760), 16 * _log_int(rng, 16, 180))])
        return {"op": op, "N": N, "K": K, "T": _log_int(rng, 1, 4095), "bias": rng.random() < 0.3,
                "dtype": rng.choice(["bf16", "bf16", "bf16", "f16", "f32"])}
    odd = {"H": 1440, "I": 736, "E": 20, "k": 3}
    shape = rng.choice([SMALL, LARGE, {"H": 1024, "I": 512, "E": 16, "k": 2}, odd])
    if op == "decode":
        return {"op": op, **shape, "layers": 8, "T": rng.randint(1, 4)}
    return {"op": op, **shape, "T": _log_int(rng, 5, 1024 if shape is SMALL else 2047)}


# ----------------------------------------------------------------------------- inputs
def _gen(seed: int) -> torch.Generator:
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _acts(g, *shape, dtype=torch.bfloat16) -> torch.Tensor:
    """N(0, 1), one channel in 256 six times larger, as the residual stream has them."""
    x = torch.randn(shape, device=DEV, generator=g)
    x *= torch.where(torch.rand(shape[-1], device=DEV, generator=g) < 1 / 256, 6.0, 1.0)
    return x.to(dtype)


def _blocks(n: int) -> int:
    return (n + B - 1) // B


def _weights(g, *shape) -> tuple[torch.Tensor, torch.Tensor]:
    """A checkpoint's matrices: codes [..., N, K] and scales [..., N / 128, K / 128] of N(0, WSTD)."""
    N, K = shape[-2:]
    n, k = _blocks(N), _blocks(K)
    w = torch.zeros((*shape[:-2], n * B, k * B), device=DEV)
    w[..., :N, :K] = WSTD * torch.randn(shape, device=DEV, generator=g)
    w = w.view(*shape[:-2], n, B, k, B)
    s = w.abs().amax((-3, -1)) / 448.0
    w /= s[..., :, None, :, None]
    w = w.view(*shape[:-2], n * B, k * B)[..., :N, :K]
    return w.to(E4M3).contiguous(), s.contiguous()


def _logits(g, case: dict) -> torch.Tensor:
    """Router logits: N(0, 1) and a popularity of the experts that falls as rank^-1.1."""
    rank = torch.randperm(case["E"], device=DEV, generator=g) + 1
    return torch.randn((case["T"], case["E"]), device=DEV, generator=g) - 1.1 * rank.double().log().float()


def _layer_seed(seed: int, i: int) -> int:
    return 1000003 * (seed + 1) + i


def _layer(case: dict, seed: int) -> dict:
    """One MoE layer's experts: codes and scales of the gate, up and down matrices, expert first."""
    g, (H, I, E) = _gen(seed), (case["H"], case["I"], case["E"])
    return {"gate": _weights(g, E, I, H), "up": _weights(g, E, I, H), "down": _weights(g, E, H, I)}


def _linear_inputs(case: dict, seed: int):
    g, dt = _gen(seed), DTYPES[case["dtype"]]
    w, s = _weights(g, case["N"], case["K"])
    bias = (0.02 * torch.randn(case["N"], device=DEV, generator=g)).to(torch.bfloat16) if case["bias"] else None
    x = _acts(g, case["T"], case["K"], dtype=torch.bfloat16 if case["op"] == "matmul" else dt)
    return w, s, bias, x


def _moe_inputs(case: dict, seed: int) -> list[tuple[torch.Tensor, torch.Tensor]]:
    g = _gen(seed + 7)
    return [(_acts(g, case["T"], case["H"]), _logits(g, case)) for _ in range(case.get("layers", 1))]


def _pack(case: dict, layer: dict) -> torch.Tensor:
    """The resident slots [E, bytes]: gate, up and down codes, then their scales in that order, filled up
    to a multiple of 16 bytes."""
    E = case["E"]
    parts = [layer[n][0] for n in ("gate", "up", "down")] + [layer[n][1] for n in ("gate", "up", "down")]
    slots = torch.cat([p.reshape(E, -1).view(torch.uint8) for p in parts], 1)
    return torch.nn.functional.pad(slots, (0, -slots.shape[1] % 16))


def _mode(case: dict) -> str:
    return "topk_then_softmax" if case["E"] == 32 else "softmax_then_topk"


def prepare(case: dict, seed: int) -> dict:
    op = case["op"]
    s = {"op": op, "case": case}
    if op == "quantize":
        s["x"] = _acts(_gen(seed), case["T"], case["K"], dtype=DTYPES[case["dtype"]])
    elif op in ("linear", "matmul"):
        s["w"], s["s"], s["bias"], s["x"] = _linear_inputs(case, seed)
        if op == "matmul":
            s["x"] = _quantize(s["x"])
    else:
        n, ins = case.get("layers", 1), _moe_inputs(case, seed)
        s["pools"], s["ins"] = [_pack(case, _layer(case, _layer_seed(seed, i))) for i in range(n)], ins
        if own:
            from tinyserve_amd import ops, synth
            from tinyserve_amd.expert_forward import fp8_expert_layout

            s["L"] = fp8_expert_layout(synth.fp8_layout(case["H"], case["I"]))
            s["slot"] = torch.arange(case["E"], dtype=torch.int32, device=DEV)
            if op == "decode":  # a decode step over the layers, captured once and replayed
                ws = ops.moe_decode_workspace(s["L"], case["T"], case["k"], DEV)
                y = torch.empty((n, case["T"], case["H"]), dtype=torch.bfloat16, device=DEV)

                def step():
                    return [ops.moe_decode_routed(s["L"], p, s["slot"], lg, x, case["k"], _mode(case), out=y[i],
                                                  workspace=ws, return_routing=True)
                            for i, (p, (x, lg)) in enumerate(zip(s["pools"], ins))]

                step()
                torch.cuda.synchronize()
                s["graph"], s["ws"] = torch.cuda.CUDAGraph(), ws
                with torch.cuda.graph(s["graph"]):
                    out = step()
                s["out"] = {"y": y, "idx": [o[1] for o in out], "w": [o[2] for o in out]}
    return s


# ----------------------------------------------------------------------------- the plain form
def _groups(x: torch.Tensor) -> torch.Tensor:
    """[..., K] -> [..., K / 128, 128], the last group filled up with zeros."""
    K = x.shape[-1]
    return torch.nn.functional.pad(x, (0, _blocks(K) * B - K)).unflatten(-1, (-1, B))


def _quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    g = _groups(x.float())
    top = g.abs().amax(-1)
    s = (top / torch.full_like(top, 448.0)).clamp(min=2.0 ** -126)  # a tensor: by a number torch multiplies with 1 / 448
    return (g / s.unsqueeze(-1)).flatten(-2)[..., : x.shape[-1]].to(E4M3).contiguous(), s


def _dequantize(c: torch.Tensor, s: torch.Tensor) -> torch.Tensor:
    return (_groups(c.float()) * s.unsqueeze(-1)).flatten(-2)[..., : c.shape[-1]]


def _dequantize_w(c: torch.Tensor, s: torch.Tensor) -> torch.Tensor:
    N = c.shape[-2]
    return _dequantize(c, s.repeat_interleave(B, -2)[..., :N, :])


def _route(logits: torch.Tensor, case: dict) -> tuple[torch.Tensor, torch.Tensor]:
    v, idx = torch.sort(logits.float(), dim=-1, descending=True, stable=True)
    v, idx = v[:, : case["k"]], idx[:, : case["k"]]
    e = torch.exp(v - v[:, :1])
    return idx.to(torch.int32), e / e.sum(-1, keepdim=True)


def _unpack(pool: torch.Tensor, case: dict) -> list[tuple[torch.Tensor, torch.Tensor]]:
    """(codes as bytes, scales) of gate, up and down for every expert of a pool."""
    H, I = case["H"], case["I"]
    shapes, o = [(I, H), (I, H), (H, I)], 0
    codes, scales = [], []
    for N, K in shapes:
        codes.append(pool[:, o : o + N * K].unflatten(1, (N, K)))
        o += N * K
    for N, K in shapes:
        n = _blocks(N) * _blocks(K)
        scales.append(pool[:, o : o + 4 * n].view(torch.float32).unflatten(1, (_blocks(N), _blocks(K))))
        o += 4 * n
    return list(zip(codes, scales))


def _silu(x: torch.Tensor) -> torch.Tensor:
    return x / (1.0 + torch.exp(-x))


def _plain_decode(pool, x, logits, case):
    idx, w = _route(logits, case)
    at, (T, k) = idx.flatten().long(), idx.shape
    wg, wu, wd = (_dequantize_w(c[at].view(E4M3), s[at]) for c, s in _unpack(pool, case))
    xq = _dequantize(*_quantize(x)).repeat_interleave(k, 0).unsqueeze(-1)
    h = _silu(torch.bmm(wg, xq)) * torch.bmm(wu, xq)
    hq = _dequantize(*_quantize(h.squeeze(-1)))
    y = torch.bmm(wd, hq.unsqueeze(-1)).view(T, k, -1)
    return (w.unsqueeze(-1) * y).sum(1).to(x.dtype), idx, w


def _plain_moe(pool, x, logits, case):
    idx, w = _route(logits, case)
    mats, xq = _unpack(pool, case), _dequantize(*_quantize(x))
    y = torch.zeros(x.shape, device=DEV)
    for e in range(case["E"]):
        t, j = (idx == e).nonzero(as_tuple=True)
        if not t.numel():
            continue
        wg, wu, wd = (_dequantize_w(c[e].view(E4M3), s[e]) for c, s in mats)
        h = _silu(xq[t] @ wg.t()) * (xq[t] @ wu.t())
        y.index_add_(0, t, w[t, j].unsqueeze(1) * (_dequantize(*_quantize(h)) @ wd.t()))
    return y.to(x.dtype), idx, w


def _plain(s: dict):
    op, case = s["op"], s["case"]
    if op == "quantize":
        return _quantize(s["x"])
    if op in ("linear", "matmul"):
        x = _dequantize(*(_quantize(s["x"]) if op == "linear" else s["x"]))
        y = x @ _dequantize_w(s["w"], s["s"]).t()
        if s["bias"] is not None:
            y += s["bias"].float()
        return y.to(DTYPES[case["dtype"]])
    if op == "moe":
        return dict(zip(("y", "idx", "w"), _plain_moe(s["pools"][0], *s["ins"][0], case)))
    out = [_plain_decode(p, x, lg, case) for p, (x, lg) in zip(s["pools"], s["ins"])]
    return {"y": torch.stack([o[0] for o in out]), "idx": [o[1] for o in out], "w": [o[2] for o in out]}


# ----------------------------------------------------------------------------- a pass
def run(s: dict):
    if not own:
        return _plain(s)
    from tinyserve_amd import ops

    op, case = s["op"], s["case"]
    if op == "quantize":
        return ops.fp8_quantize(s["x"])
    if op == "linear":
        return ops.fp8_linear(s["x"], s["w"], s["s"], s["bias"])
    if op == "matmul":
        return ops.fp8_matmul(*s["x"], s["w"], s["s"], s["bias"], out_dtype=DTYPES[case["dtype"]])
    if op == "moe":
        x, logits = s["ins"][0]
        idx, w = ops.route_topk(logits, case["k"], _mode(case))
        return {"y": ops.moe_prefill(s["L"], s["pools"][0], s["slot"], idx, w, x), "idx": idx, "w": w}
    s["graph"].replay()
    return s["out"]


# ----------------------------------------------------------------------------- work
def _distinct(case: dict) -> float:
    """Experts that T tokens' top-k selections reach, on average."""
    rng = np.random.default_rng(1)
    E, k, got = case["E"], case["k"], []
    for _ in range(8):
        lg = rng.normal(size=(case["T"], E)) - 1.1 * np.log(rng.permutation(E) + 1)
        got.append(len(np.unique(np.argpartition(-lg, k - 1, axis=1)[:, :k])))
    return float(np.mean(got))


def work(case: dict) -> dict:
    op, T = case["op"], case["T"]
    if op in ("decode", "moe"):
        H, I, k, layers = case["H"], case["I"], case["k"], case.get("layers", 1)
        expert = 3 * H * I + 4 * (2 * _blocks(I) * _blocks(H) + _blocks(H) * _blocks(I))
        per = _distinct(case) * expert + T * (4 * H + 4 * case["E"] + 8 * k)
        return {"bytes": layers * per, "flops": layers * 2 * T * k * 3 * H * I}
    K, es = case["K"], DTYPES[case["dtype"]].itemsize
    quantized = T * K + 4 * T * _blocks(K)
    if op == "quantize":
        return {"bytes": es * T * K + quantized, "flops": 0}
    N = case["N"]
    weights = N * K + 4 * _blocks(N) * _blocks(K) + (2 * N if case["bias"] else 0)
    x = quantized if op == "matmul" else es * T * K
    return {"bytes": weights + x + es * T * N, "flops": 2 * T * N * K}


# ----------------------------------------------------------------------------- the definition in 64 bits
def _e4m3_64(v: torch.Tensor) -> torch.Tensor:
    """v rounded to the nearest e4m3 number (ties to the even one), in 64 bits."""
    _, e = torch.frexp(v)
    step = torch.exp2((e.double() - 1).clamp(min=-6.0) - 3)
    return torch.round(v / step) * step


def _quantize64(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The numbers the codes stand for, and the scales per value's group."""
    T, K = x.shape
    q, s = torch.empty_like(x), []
    for c in range(0, K, B):
        part = x[:, c : c + B]
        sc = torch.clamp(part.abs().amax(1) / 448, min=2.0 ** -126).float().double()
        q[:, c : c + B] = _e4m3_64((part / sc[:, None]).float().double())
        s.append(sc)
    return q, torch.stack(s, 1)


def _times64(q: torch.Tensor, qs: torch.Tensor, w: torch.Tensor, ws: torch.Tensor) -> torch.Tensor:
    """sum over the blocks of (q . w) qs ws, block by block."""
    (T, K), N = q.shape, w.shape[0]
    rows = torch.arange(N, device=DEV) // B
    y = torch.zeros((T, N), dtype=torch.float64, device=DEV)
    for b in range(qs.shape[1]):
        c = slice(b * B, min(b * B + B, K))
        y += (q[:, c] @ w[:, c].double().t()) * qs[:, b, None] * ws.double()[rows, b]
    return y


def _moe64(case, layer, x, logits):
    v, idx = torch.sort(logits.double(), dim=-1, descending=True, stable=True)
    w, idx = torch.softmax(v[:, : case["k"]], -1), idx[:, : case["k"]]
    q, qs = _quantize64(x.double())
    y = torch.zeros(x.shape, dtype=torch.float64, device=DEV)
    for e in torch.unique(idx).tolist():
        t, j = (idx == e).nonzero(as_tuple=True)
        gate, up, down = ((layer[n][0][e], layer[n][1][e]) for n in ("gate", "up", "down"))
        g = _times64(q[t], qs[t], *gate)
        h = g * torch.sigmoid(g) * _times64(q[t], qs[t], *up)
        y.index_add_(0, t, w[t, j].unsqueeze(1) * _times64(*_quantize64(h), *down))
    return y, w


def exact(case: dict, seed: int):
    op = case["op"]
    if op == "quantize":
        return _quantize64(_acts(_gen(seed), case["T"], case["K"], dtype=DTYPES[case["dtype"]]).double())
    if op in ("linear", "matmul"):
        w, s, bias, x = _linear_inputs(case, seed)
        y = _times64(*_quantize64(x.double()), w, s)
        return y if bias is None else y + bias.double()
    ys, ws = [], []
    for i, (x, lg) in enumerate(_moe_inputs(case, seed)):
        y, w = _moe64(case, _layer(case, _layer_seed(seed, i)), x, lg)
        ys.append(y)
        ws.append(w)
    if op == "moe":
        return {"y": ys[0], "idx": None, "w": ws[0]}
    return {"y": torch.stack(ys), "idx": [None] * len(ys), "w": ws}
