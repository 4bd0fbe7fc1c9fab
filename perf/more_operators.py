"""Products in 8-bit integers and products grouped by expert.

8-bit integers. A weight matrix [N, K] is int8 codes and one float32 scale for each of its rows (output
channels). Activations are quantised where they are used, a float32 scale for each token:

    scale = max(max|x| / 127, 2^-126)            (float32)
    code  = round(x / scale), ties to even       (of the float32 quotient)

``quantize`` is that step by itself, ``linear`` the quantised product y = x W^T (+ bias) from 16- or
32-bit activations, ``matmul`` the same from codes that several projections share.

Grouped. Row r of a batch that is sorted by expert takes row rows[r] // k of the activations and, for
offsets[e] <= r < offsets[e + 1], the matrix of expert e: y[r] = x[rows[r] // k] W_e^T (+ bias_e). Rows
behind the last expert's are zeros. ``grouped`` has 16-bit operands, ``grouped8`` int8 ones with their scales.

``decode`` is a stack of mixture-of-experts layers for a few tokens, ``moe`` one layer for batches and
prompts, over experts in bfloat16, float16 or int8: route, then per expert h = silu(x Wg^T) * (x Wu^T),
h rounded to the weights' type (int8: x and h quantised by the rule above), y = sum_j w_j h Wd^T.

A case is a dict of plain values. Where ``own`` is false, ``run`` is the plain form of the operator in
32 bits; where it is true, the framework's call. ``exact`` is the definition in 64 bits.
"""
from __future__ import annotations

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
WSTD = 0.03   # the weights' standard deviation

# the two layer shapes of the benchmark: many small experts, few large ones
SMALL = {"H": 2048, "I": 768, "E": 128, "k": 8}
LARGE = {"H": 2880, "I": 2880, "E": 32, "k": 4}
# gate and up together, as one product over the same experts
SMALL_UP = {"N": 1536, "K": 2048, "E": 128, "k": 8}
LARGE_UP = {"N": 5760, "K": 2880, "E": 32, "k": 4}


# ----------------------------------------------------------------------------- the cases
def listed() -> list[dict]:
    return [
        # the activations of a decode batch ahead of the projections that share them: launch latency
        {"name": "quantize batch", "op": "quantize", "T": 24, "K": 2880, "dtype": "bf16"},
        # the same over a long prompt
        {"name": "quantize prompt", "op": "quantize", "T": 4096, "K": 2880, "dtype": "bf16"},
        # one projection of a decode step, called by itself: launch and call latency
        {"name": "linear one token", "op": "linear", "N": 2880, "K": 2880, "T": 1, "dtype": "bf16", "bias": True},
        # the same kind of layer for a decode batch of 24 sequences
        {"name": "linear batch", "op": "linear", "N": 2048, "K": 4096, "T": 24, "dtype": "bf16", "bias": False},
        # the query projection over a prompt of 512 tokens, quantised once for q, k and v
        {"name": "matmul prompt", "op": "matmul", "N": 4096, "K": 2048, "T": 512, "dtype": "bf16", "bias": False},
        # the widest projection over a long prompt: where the matrix cores are the bound
        {"name": "linear long prompt", "op": "linear", "N": 5760, "K": 2880, "T": 4096, "dtype": "bf16", "bias": True},
        # gate and up of unquantised experts for a decode batch of 24 sequences: most experts get a row or two
        {"name": "grouped batch", "op": "grouped", **SMALL_UP, "T": 24, "dtype": "bf16", "bias": False, "behind": 0},
        # the same over a long prompt, few large experts with biases
        {"name": "grouped prompt", "op": "grouped", **LARGE_UP, "T": 2048, "dtype": "bf16", "bias": True, "behind": 0},
        # int8 experts: a decode batch, and a prompt whose last rows belong to experts that live elsewhere
        {"name": "grouped int8 batch", "op": "grouped8", **SMALL_UP, "T": 24, "dtype": "bf16", "bias": False, "behind": 0},
        {"name": "grouped int8 prompt", "op": "grouped8", **SMALL_UP, "T": 1024, "dtype": "bf16", "bias": False, "behind": 100},
        # one token through a stack of MoE layers of unquantised experts, as a captured decode step replays it
        {"name": "moe decode", "op": "decode", **SMALL, "layers": 8, "T": 1, "weights": "bf16"},
        # a prompt of 1024 tokens through one MoE layer of int8 experts
        {"name": "moe prompt int8", "op": "moe", **SMALL, "T": 1024, "weights": "int8"},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng) -> dict:
    """One more case of the same kinds: sizes over the logarithm of their range, odd ones among them."""
    op = rng.choice(["quantize", "linear", "linear", "matmul", "grouped", "grouped", "grouped8", "grouped8", "decode", "decode",
                     "moe", "moe", "moe"])
    if op == "quantize":
        return {"op": op, "T": _log_int(rng, 1, 4096), "K": _log_int(rng, 256, 2880),
                "dtype": rng.choice(["bf16", "bf16", "f16", "f32"])}
    if op in ("linear", "matmul"):
        N, K = rng.choice([(2880, 2880), (4096, 2048), (2048, 4096), (512, 2048), (768, 2048), (5760, 2880),
                           (_log_int(rng, 300, 5760), 16 * _log_int(rng, 16, 180)),
                           (_log_int(rng, 300, 5760), 16 * _log_int(rng, 16, 180))])
        return {"op": op, "N": N, "K": K, "T": _log_int(rng, 1, 4095), "bias": rng.random() < 0.3,
                "dtype": rng.choice(["bf16", "bf16", "bf16", "f16", "f32"])}
    if op in ("grouped", "grouped8"):
        shape = rng.choice([SMALL_UP, LARGE_UP, {"N": 2048, "K": 768, "E": 128, "k": 8},
                            {"N": _log_int(rng, 200, 1600), "K": 16 * _log_int(rng, 16, 90), "E": rng.randint(3, 60), "k": 3}])
        T = _log_int(rng, 1, 2047)
        return {"op": op, **shape, "T": T, "dtype": rng.choice(["bf16", "bf16", "f16"]), "bias": rng.random() < 0.3,
                "behind": rng.choice([0, 0, _log_int(rng, 1, T * shape["k"])])}
    odd = {"H": 1440, "I": 736, "E": 20, "k": 3}
    shape = rng.choice([SMALL, LARGE, {"H": 1024, "I": 512, "E": 16, "k": 2}, odd])
    weights = rng.choice(["bf16", "bf16", "f16", "int8", "int8"])
    if op == "decode":
        return {"op": op, **shape, "layers": 2 if shape is LARGE else 8, "T": rng.randint(1, 4), "weights": weights}
    return {"op": op, **shape, "T": _log_int(rng, 5, 1024), "weights": weights}


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


def _weights16(g, *shape, dtype=torch.bfloat16) -> torch.Tensor:
    return (WSTD * torch.randn(shape, device=DEV, generator=g)).to(dtype)


def _weights8(g, *shape) -> tuple[torch.Tensor, torch.Tensor]:
    """A checkpoint's matrices: codes [..., N, K] and scales [..., N] of N(0, WSTD)."""
    w = WSTD * torch.randn(shape, device=DEV, generator=g)
    s = w.abs().amax(-1) / 127.0
    return torch.round(w / s.unsqueeze(-1)).clamp(-127, 127).to(torch.int8), s.contiguous()


def _bias(g, *shape) -> torch.Tensor:
    return (0.02 * torch.randn(shape, device=DEV, generator=g)).to(torch.bfloat16)


def _logits(g, case: dict) -> torch.Tensor:
    """Router logits: N(0, 1) and a popularity of the experts that falls as rank^-1.1."""
    rank = torch.randperm(case["E"], device=DEV, generator=g) + 1
    return torch.randn((case["T"], case["E"]), device=DEV, generator=g) - 1.1 * rank.double().log().float()


def _layer_seed(seed: int, i: int) -> int:
    return 1000003 * (seed + 1) + i


def _layer(case: dict, seed: int) -> dict:
    """One MoE layer's experts, expert first: the gate, up and down matrices; int8: (codes, scales) of each."""
    g, (H, I, E) = _gen(seed), (case["H"], case["I"], case["E"])
    if case["weights"] == "int8":
        return {"gate": _weights8(g, E, I, H), "up": _weights8(g, E, I, H), "down": _weights8(g, E, H, I)}
    dt = DTYPES[case["weights"]]
    return {"gate": _weights16(g, E, I, H, dtype=dt), "up": _weights16(g, E, I, H, dtype=dt), "down": _weights16(g, E, H, I, dtype=dt)}


def _linear_inputs(case: dict, seed: int):
    g = _gen(seed)
    w, s = _weights8(g, case["N"], case["K"])
    bias = _bias(g, case["N"]) if case["bias"] else None
    return w, s, bias, _acts(g, case["T"], case["K"], dtype=DTYPES["bf16" if case["op"] == "matmul" else case["dtype"]])


def _grouped_inputs(case: dict, seed: int):
    """(weights, scales or None, bias or None, x, offsets int32 [E + 1], rows int32 [T k]): the assignments of a
    top-k routing sorted by expert; the last ``behind`` of them are taken out of their groups."""
    g, (E, k, N, K, T) = _gen(seed), (case["E"], case["k"], case["N"], case["K"], case["T"])
    w, s = _weights8(g, E, N, K) if case["op"] == "grouped8" else (_weights16(g, E, N, K, dtype=DTYPES[case["dtype"]]), None)
    bias = _bias(g, E, N) if case["bias"] else None
    x = _acts(g, T, K, dtype=DTYPES[case["dtype"]])
    chosen = torch.topk(_logits(g, case), k, dim=-1).indices.flatten()
    expert, rows = torch.sort(chosen, stable=True)
    ends = torch.searchsorted(expert, torch.arange(E, device=DEV), right=True).clamp(max=T * k - case["behind"])
    offsets = torch.cat([torch.zeros(1, dtype=ends.dtype, device=DEV), ends]).to(torch.int32)
    return w, s, bias, x, offsets, rows.to(torch.int32)


def _moe_inputs(case: dict, seed: int) -> list[tuple[torch.Tensor, torch.Tensor]]:
    g, dt = _gen(seed + 7), DTYPES["bf16" if case["weights"] == "int8" else case["weights"]]
    return [(_acts(g, case["T"], case["H"], dtype=dt), _logits(g, case)) for _ in range(case.get("layers", 1))]


def _pack(case: dict, layer: dict) -> torch.Tensor:
    """The resident slots [E, bytes]: the gate, up and down matrices; int8: then their scales in that order, filled up
    to a multiple of 16 bytes."""
    E, mats = case["E"], [layer[n] for n in ("gate", "up", "down")]
    parts = [c for c, _ in mats] + [s for _, s in mats] if case["weights"] == "int8" else mats
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
    elif op in ("grouped", "grouped8"):
        s["w"], s["s"], s["bias"], s["x"], s["offsets"], s["rows"] = _grouped_inputs(case, seed)
        if op == "grouped8":
            s["x"] = _quantize(s["x"])
        if not own:  # the plain form's loop over the experts
            s["ends"] = s["offsets"].tolist()
    else:
        n, ins = case.get("layers", 1), _moe_inputs(case, seed)
        s["pools"], s["ins"] = [_pack(case, _layer(case, _layer_seed(seed, i))) for i in range(n)], ins
        if own:
            from tinyserve_amd import ops, synth
            from tinyserve_amd.expert_forward import build_expert_layout

            specs = (synth.int8_layout(case["H"], case["I"]) if case["weights"] == "int8"
                     else synth.dense_layout(case["H"], case["I"], DTYPES[case["weights"]]))
            s["L"] = build_expert_layout(specs)
            s["slot"] = torch.arange(case["E"], dtype=torch.int32, device=DEV)
            if op == "decode":  # a decode step over the layers, captured once and replayed
                ws = ops.moe_decode_workspace(s["L"], case["T"], case["k"], DEV)
                y = torch.empty((n, case["T"], case["H"]), dtype=ins[0][0].dtype, device=DEV)

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
def _quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    v = x.float()
    top = v.abs().amax(-1)
    s = (top / torch.full_like(top, 127.0)).clamp(min=2.0 ** -126)  # a tensor: by a number torch multiplies with 1 / 127
    return torch.round(v / s.unsqueeze(-1)).to(torch.int8), s


def _values(c: torch.Tensor, s: torch.Tensor) -> torch.Tensor:
    return c.float() * s.unsqueeze(-1)


def _route(logits: torch.Tensor, case: dict) -> tuple[torch.Tensor, torch.Tensor]:
    v, idx = torch.sort(logits.float(), dim=-1, descending=True, stable=True)
    v, idx = v[:, : case["k"]], idx[:, : case["k"]]
    e = torch.exp(v - v[:, :1])
    return idx.to(torch.int32), e / e.sum(-1, keepdim=True)


def _unpack(pool: torch.Tensor, case: dict) -> list[tuple[torch.Tensor, torch.Tensor | None]]:
    """(matrix or codes, scales or None) of gate, up and down for every expert of a pool."""
    H, I = case["H"], case["I"]
    dt = torch.int8 if case["weights"] == "int8" else DTYPES[case["weights"]]
    shapes, o, mats = [(I, H), (I, H), (H, I)], 0, []
    for N, K in shapes:
        n = N * K * dt.itemsize
        mats.append(pool[:, o : o + n].view(dt).unflatten(1, (N, K)))
        o += n
    if case["weights"] != "int8":
        return [(m, None) for m in mats]
    scales = []
    for N, _ in shapes:
        scales.append(pool[:, o : o + 4 * N].view(torch.float32))
        o += 4 * N
    return list(zip(mats, scales))


def _take(mat: tuple[torch.Tensor, torch.Tensor | None], at) -> torch.Tensor:
    w, s = mat
    return w[at].float() if s is None else _values(w[at], s[at])


def _held(x: torch.Tensor, case: dict) -> torch.Tensor:
    """The numbers that activations stand for where a matrix takes them, in 32 bits."""
    return _values(*_quantize(x)) if case["weights"] == "int8" else x.to(DTYPES[case["weights"]]).float()


def _silu(x: torch.Tensor) -> torch.Tensor:
    return x / (1.0 + torch.exp(-x))


def _plain_decode(pool, x, logits, case):
    idx, w = _route(logits, case)
    at, (T, k) = idx.flatten().long(), idx.shape
    wg, wu, wd = (_take(m, at) for m in _unpack(pool, case))
    xq = _held(x, case).repeat_interleave(k, 0).unsqueeze(-1)
    h = _held((_silu(torch.bmm(wg, xq)) * torch.bmm(wu, xq)).squeeze(-1), case)
    y = torch.bmm(wd, h.unsqueeze(-1)).view(T, k, -1)
    return (w.unsqueeze(-1) * y).sum(1).to(x.dtype), idx, w


def _plain_moe(pool, x, logits, case):
    idx, w = _route(logits, case)
    mats, xq = _unpack(pool, case), _held(x, case)
    y = torch.zeros(x.shape, device=DEV)
    for e in range(case["E"]):
        t, j = (idx == e).nonzero(as_tuple=True)
        if not t.numel():
            continue
        wg, wu, wd = (_take(m, e) for m in mats)
        h = _silu(xq[t] @ wg.t()) * (xq[t] @ wu.t())
        y.index_add_(0, t, w[t, j].unsqueeze(1) * (_held(h, case) @ wd.t()))
    return y.to(x.dtype), idx, w


def _plain_grouped(s: dict) -> torch.Tensor:
    case, ends = s["case"], s["ends"]
    x = _values(*s["x"]) if s["s"] is not None else s["x"].float()
    y = torch.zeros((case["T"] * case["k"], case["N"]), device=DEV)
    for e in range(case["E"]):
        a, b = ends[e], ends[e + 1]
        if a == b:
            continue
        y[a:b] = x[s["rows"][a:b] // case["k"]] @ _take((s["w"], s["s"]), e).t()
        if s["bias"] is not None:
            y[a:b] += s["bias"][e].float()
    return y.to(DTYPES[case["dtype"]])


def _plain(s: dict):
    op, case = s["op"], s["case"]
    if op == "quantize":
        return _quantize(s["x"])
    if op in ("linear", "matmul"):
        x = _values(*(_quantize(s["x"]) if op == "linear" else s["x"]))
        y = x @ _values(s["w"], s["s"]).t()
        if s["bias"] is not None:
            y += s["bias"].float()
        return y.to(DTYPES[case["dtype"]])
    if op in ("grouped", "grouped8"):
        return _plain_grouped(s)
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
        return ops.int8_quantize(s["x"])
    if op == "linear":
        return ops.int8_linear(s["x"], s["w"], s["s"], s["bias"])
    if op == "matmul":
        return ops.int8_matmul(*s["x"], s["w"], s["s"], s["bias"], out_dtype=DTYPES[case["dtype"]])
    if op == "grouped":
        return ops.grouped_matmul(s["x"], s["w"], s["offsets"], s["bias"], rows=s["rows"], top_k=case["k"])
    if op == "grouped8":
        return ops.int8_grouped_matmul(*s["x"], s["w"], s["s"], s["offsets"], s["bias"], rows=s["rows"], top_k=case["k"],
                                       out_dtype=DTYPES[case["dtype"]])
    if op == "moe":
        x, logits = s["ins"][0]
        idx, w = ops.route_topk(logits, case["k"], _mode(case))
        return {"y": ops.moe_prefill(s["L"], s["pools"][0], s["slot"], idx, w, x), "idx": idx, "w": w}
    s["graph"].replay()
    return s["out"]


# ----------------------------------------------------------------------------- work
def _reached(case: dict) -> float:
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
        expert = 3 * H * I + 4 * (2 * I + H) if case["weights"] == "int8" else 6 * H * I
        per = _reached(case) * expert + T * (4 * H + 4 * case["E"] + 8 * k)
        return {"bytes": layers * per, "flops": layers * 2 * T * k * 3 * H * I}
    K, es = case["K"], DTYPES[case["dtype"]].itemsize
    if op == "quantize":
        return {"bytes": es * T * K + T * K + 4 * T, "flops": 0}
    N = case["N"]
    bias = 2 * N if case["bias"] else 0
    if op in ("grouped", "grouped8"):
        R, k = T * case["k"], case["k"]
        matrix, token = (N * K + 4 * N, K + 4) if op == "grouped8" else (2 * N * K, 2 * K)
        live = 1.0 - case["behind"] / R
        return {"bytes": live * _reached(case) * (matrix + bias) + min(T, R * live) * token + es * R * N + 4 * R,
                "flops": 2 * live * R * N * K}
    x = T * K + 4 * T if op == "matmul" else es * T * K
    return {"bytes": N * K + 4 * N + bias + x + es * T * N, "flops": 2 * T * N * K}


# ----------------------------------------------------------------------------- the definition in 64 bits
def _quantize64(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The codes and the scales, both as 64-bit numbers."""
    s = torch.clamp(x.abs().max(1, keepdim=True).values / 127, min=2.0 ** -126).float().double()
    return torch.round((x / s).float().double()), s


def _times64(x: torch.Tensor, w: torch.Tensor, ws: torch.Tensor | None, bias: torch.Tensor | None) -> torch.Tensor:
    """x w^T (+ bias); ws: w and x are codes, x a pair with its scales."""
    y = x @ w.double().t() if ws is None else (x[0] @ w.double().t()) * x[1] * ws.double()
    return y if bias is None else y + bias.double()


def _pick64(x, rows: torch.Tensor):
    return (x[0][rows], x[1][rows]) if isinstance(x, tuple) else x[rows]


def _moe64(case, layer, x, logits):
    v, idx = torch.sort(logits.double(), dim=-1, descending=True, stable=True)
    w, idx = torch.softmax(v[:, : case["k"]], -1), idx[:, : case["k"]]
    int8 = case["weights"] == "int8"
    mat = (lambda n, e: (layer[n][0][e], layer[n][1][e])) if int8 else (lambda n, e: (layer[n][e], None))
    q = _quantize64(x.double()) if int8 else x.double()
    y = torch.zeros(x.shape, dtype=torch.float64, device=DEV)
    for e in torch.unique(idx).tolist():
        t, j = (idx == e).nonzero(as_tuple=True)
        g = _times64(_pick64(q, t), *mat("gate", e), None)
        h = g * torch.sigmoid(g) * _times64(_pick64(q, t), *mat("up", e), None)
        h = _quantize64(h) if int8 else h.to(x.dtype).double()
        y.index_add_(0, t, w[t, j].unsqueeze(1) * _times64(h, *mat("down", e), None))
    return y, w


def exact(case: dict, seed: int):
    op = case["op"]
    if op == "quantize":
        q, s = _quantize64(_acts(_gen(seed), case["T"], case["K"], dtype=DTYPES[case["dtype"]]).double())
        return q.to(torch.int8), s.squeeze(1)
    if op in ("linear", "matmul"):
        w, s, bias, x = _linear_inputs(case, seed)
        return _times64(_quantize64(x.double()), w, s, bias)
    if op in ("grouped", "grouped8"):
        w, s, bias, x, offsets, rows = _grouped_inputs(case, seed)
        q = x.double() if s is None else _quantize64(x.double())
        y = torch.zeros((rows.numel(), case["N"]), dtype=torch.float64, device=DEV)
        token = torch.div(rows, case["k"], rounding_mode="floor").long()
        for e, (a, b) in enumerate(zip(offsets[:-1].tolist(), offsets[1:].tolist())):
            if a < b:
                y[a:b] = _times64(_pick64(q, token[a:b]), w[e], None if s is None else s[e], None if bias is None else bias[e])
        return y
    ys, ws = [], []
    for i, (x, lg) in enumerate(_moe_inputs(case, seed)):
        y, w = _moe64(case, _layer(case, _layer_seed(seed, i)), x, lg)
        ys.append(y)
        ws.append(w)
    if op == "moe":
        return {"y": ys[0], "idx": None, "w": ws[0]}
    return {"y": torch.stack(ys), "idx": [None] * len(ys), "w": ws}
