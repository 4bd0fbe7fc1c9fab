"""MoE layers over bfloat16, float16 and int8 experts on the GPU against their definition in 64 bits
(tests/int8_ref.py): few tokens, batches, prompts, routing inside and outside, experts that are not resident."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from tests import int8_ref as ref
from tinyserve_amd import _lib, ops, synth
from tinyserve_amd.expert_forward import build_expert_layout
from tinyserve_amd.expert_store import pack_tensors

pytestmark = pytest.mark.gpu
KINDS = ["bf16", "f16", "int8"]
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "int8": torch.bfloat16}


def gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def layer(kind: str, H: int, I: int, E: int, seed: int = 0, sigma: float = 0.05):
    """(layout, pool, the experts' tensors)."""
    g, specs = gen(seed + H + I), synth.int8_layout(H, I) if kind == "int8" else synth.dense_layout(H, I, DT[kind])
    pool = torch.zeros((E, specs.total_bytes), dtype=torch.uint8, device="cuda")
    experts = []
    for e in range(E):
        t = {}
        for m, (r, c) in (("gate_proj", (I, H)), ("up_proj", (I, H)), ("down_proj", (H, I))):
            if kind == "int8":
                t[m], t[m + "_scale"] = ref.weights8(g, r, c, sigma=sigma)
            else:
                t[m] = (sigma * torch.randn((r, c), device="cuda", generator=g)).to(DT[kind])
        pack_tensors(pool[e], specs, t)
        experts.append(t)
    return build_expert_layout(specs), pool, experts


def tokens(kind, T, H, E, k, seed=0):
    g = gen(seed + T)
    x = torch.randn((T, H), device="cuda", generator=g)
    x[:, ::131] *= 5
    return x.to(DT[kind]), torch.randn((T, E), device="cuda", generator=g)


SHAPES = [(64, 32, 4, 2), (288, 96, 6, 3), (1440, 736, 5, 4), (2048, 768, 12, 8), (2880, 2880, 5, 4), (96, 4128, 3, 1)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("H,I,E,k", SHAPES)
@pytest.mark.parametrize("T", [1, 2, 4, 5])
def test_decode(kind, H, I, E, k, T):
    """Routed and given selections, the pairs' kernels."""
    L, pool, experts = layer(kind, H, I, E)
    x, lg = tokens(kind, T, H, E, k)
    slot = torch.arange(E, dtype=torch.int32, device="cuda")
    for mode in ("topk_then_softmax", "softmax_then_topk_no_renorm"):
        y, idx, w = ops.moe_decode_routed(L, pool, slot, lg, x, k, mode, return_routing=True)
        ri, rw = ops.route_topk(lg, k, mode)
        assert torch.equal(idx, ri) and (w - rw).abs().max() < 1e-6
        ref.check(y, *ref.moe(x, idx, w, experts), f"routed {mode}")
    ref.check(ops.moe_decode(L, pool, idx, w, x, out_dtype=torch.float32), *ref.moe(x, idx, w, experts), "given")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("H,I,E,k", SHAPES)
@pytest.mark.parametrize("T", [5, 33, 300])
def test_prefill(kind, H, I, E, k, T):
    L, pool, experts = layer(kind, H, I, E)
    x, lg = tokens(kind, T, H, E, k)
    idx, w = ops.route_topk(lg, k)
    slot = torch.arange(E, dtype=torch.int32, device="cuda")
    want = ref.moe(x, idx, w, experts)
    ref.check(ops.moe_prefill(L, pool, slot, idx, w, x), *want)
    ref.check(ops.moe_prefill(L, pool, slot, idx, w, x, out_dtype=torch.float32), *want, "to float32")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T,E,k", [(6, 64, 4), (40, 40, 4), (200, 24, 6), (700, 8, 2), (1500, 4, 2)])
def test_prefill_tiles(kind, T, E, k):
    """Loads that reach each size of token tile, very uneven ones among them."""
    H, I = 160, 224
    L, pool, experts = layer(kind, H, I, E)
    x, lg = tokens(kind, T, H, E, k)
    lg -= 1.5 * torch.arange(1, E + 1, device="cuda").log()
    idx, w = ops.route_topk(lg, k)
    slot = torch.arange(E, dtype=torch.int32, device="cuda")
    ref.check(ops.moe_prefill(L, pool, slot, idx, w, x), *ref.moe(x, idx, w, experts))


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("T", [1, 3, 40])
def test_not_resident(kind, T):
    """Slots below zero and past the pool, ids without an expert: zeros, whatever their weights and the workspace hold."""
    H, I, E, k = 288, 96, 7, 5
    L, pool, experts = layer(kind, H, I, 5)
    slot = torch.tensor([3, -1, 0, 5, 2, 1, 4], dtype=torch.int32, device="cuda")
    here = [experts[s] if 0 <= s < 5 else None for s in slot.tolist()]
    x, lg = tokens(kind, T, H, E, k)
    idx, w = ops.route_topk(lg, k)
    dead = torch.tensor([e is None for e in here], device="cuda")[idx.long()]
    wn = torch.where(dead, float("nan"), w)
    want = ref.moe(x, idx, torch.where(dead, 0.0, w), here)
    n = ops.moe_prefill_workspace(L, T, k, E, "cuda").numel()
    ref.check(ops.moe_prefill(L, pool, slot, idx, wn, x, workspace=torch.full((n,), 255, dtype=torch.uint8, device="cuda")), *want, "prefill")
    gone = idx.clone()
    gone[:, 1] = -1
    ref.check(ops.moe_prefill(L, pool, slot, gone, wn, x), *ref.moe(x, gone, torch.where(dead, 0.0, w), here), "ids below zero")
    ws = torch.full((ops.moe_decode_workspace_size(L, T, k),), 255, dtype=torch.uint8, device="cuda")
    ref.check(ops.moe_decode(L, pool, slot[idx.long()], wn, x, workspace=ws), *want, "decode")
    y, ri, rw = ops.moe_decode_routed(L, pool, slot, lg, x, k, workspace=ws, return_routing=True)
    ref.check(y, *ref.moe(x, ri, rw, here), "routed")


@pytest.mark.parametrize("T", [2, 20])
@pytest.mark.parametrize("xt", [torch.float32, torch.float16, torch.bfloat16])
def test_int8_activations_of_any_type(T, xt):
    L, pool, experts = layer("int8", 288, 96, 6)
    x, lg = tokens("int8", T, 288, 6, 3)
    x = (x.float() * 1.01).to(xt)
    idx, w = ops.route_topk(lg, 3)
    slot = torch.arange(6, dtype=torch.int32, device="cuda")
    want = ref.moe(x, idx, w, experts)
    for out in (torch.float32, torch.float16, torch.bfloat16):
        ref.check(ops.moe_decode(L, pool, idx, w, x, out_dtype=out), *want)
        ref.check(ops.moe_prefill(L, pool, slot, idx, w, x, out_dtype=out), *want)


@pytest.mark.parametrize("kind", ["f16", "int8"])
@pytest.mark.parametrize("T", [2, 40])
def test_clamped_swiglu(kind, T):
    L, pool, experts = layer(kind, 288, 96, 6, sigma=0.2)
    L.act, L.swiglu_limit, L.swiglu_alpha = _lib.ACT_SWIGLU_OAI, 7.0, 1.702
    x, lg = tokens(kind, T, 288, 6, 3)
    idx, w = ops.route_topk(lg, 3)
    want = ref.moe(x, idx, w, experts, "oai")
    ref.check(ops.moe_decode(L, pool, idx, w, x, out_dtype=torch.float32), *want)
    ref.check(ops.moe_prefill(L, pool, torch.arange(6, dtype=torch.int32, device="cuda"), idx, w, x, out_dtype=torch.float32), *want)


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("T", [3, 40])
def test_not_finite(kind, T):
    """A token with a NaN or an infinity gives NaN; the others are as ever."""
    L, pool, experts = layer(kind, 288, 96, 6)
    x, lg = tokens(kind, T, 288, 6, 3)
    idx, w = ops.route_topk(lg, 3)
    want, err = ref.moe(x, idx, w, experts)
    x[1, 5] = float("nan")
    if kind == "int8":
        x[2, 280] = float("inf")
    ok = x.isfinite().all(1)
    for y in (ops.moe_decode(L, pool, idx, w, x), ops.moe_prefill(L, pool, torch.arange(6, dtype=torch.int32, device="cuda"), idx, w, x)):
        assert y[~ok].isnan().all()
        ref.check(y[ok], want[ok], err[ok])


@pytest.mark.parametrize("kind", ["bf16", "int8"])
def test_many_experts_a_token(kind):
    """More experts a token than the routing inside takes, and more than one stage of h in LDS."""
    H, I, E, k = 64, 4128, 40, 24
    L, pool, experts = layer(kind, H, I, E)
    x, lg = tokens(kind, 2, H, E, k)
    y, idx, w = ops.moe_decode_routed(L, pool, torch.arange(E, dtype=torch.int32, device="cuda"), lg, x, k, return_routing=True)
    ref.check(y, *ref.moe(x, idx, w, experts))


@pytest.mark.parametrize("kind", KINDS)
def test_layer_as_grouped_products(kind):
    """The operators together as a layer: route, group, quantise, both grouped products, weighted sums; against the layer call."""
    H, I, E, k, T = 288, 96, 6, 3, 50
    L, pool, experts = layer(kind, H, I, E)
    x, lg = tokens(kind, T, H, E, k)
    idx, w = ops.route_topk(lg, k)
    _, off, perm = ops.group_by_expert(idx, E)
    up = torch.stack([torch.cat([e["gate_proj"], e["up_proj"]]) for e in experts])
    down = torch.stack([e["down_proj"] for e in experts])
    if kind == "int8":
        us = torch.stack([torch.cat([e["gate_proj_scale"], e["up_proj_scale"]]) for e in experts])
        gu = ops.int8_grouped_matmul(*ops.int8_quantize(x), up, us, off, rows=perm, top_k=k, out_dtype=torch.float32)
        h = torch.nn.functional.silu(gu[:, :I]) * gu[:, I:]
        o = ops.int8_grouped_matmul(*ops.int8_quantize(h), down, torch.stack([e["down_proj_scale"] for e in experts]), off, out_dtype=torch.float32)
    else:
        gu = ops.grouped_matmul(x, up, off, rows=perm, top_k=k, out_dtype=torch.float32)
        o = ops.grouped_matmul((torch.nn.functional.silu(gu[:, :I]) * gu[:, I:]).to(x.dtype), down, off, out_dtype=torch.float32)
    y = torch.zeros((T * k, H), device="cuda")
    y[perm.long()] = o
    y = (y.view(T, k, H) * w.unsqueeze(-1)).sum(1)
    want = ref.moe(x, idx, w, experts)
    ref.check(y, *want, "composed")
    ref.check(ops.moe_prefill(L, pool, torch.arange(E, dtype=torch.int32, device="cuda"), idx, w, x), *want, "layer")


@pytest.mark.parametrize("kind", ["bf16", "int8"])
def test_captured(kind):
    """A captured layer replayed on new inputs, with eager work of the same kind between the replays."""
    L, pool, experts = layer(kind, 288, 96, 6)
    slot = torch.arange(6, dtype=torch.int32, device="cuda")
    x, lg = tokens(kind, 2, 288, 6, 3)
    xp, lgp = tokens(kind, 40, 288, 6, 3)
    ws = ops.moe_decode_workspace(L, 2, 3, "cuda")

    def step():
        y, idx, w = ops.moe_decode_routed(L, pool, slot, lg, x, 3, workspace=ws, return_routing=True)
        ip, wp = ops.route_topk(lgp, 3)
        return y, idx, w, ops.moe_prefill(L, pool, slot, ip, wp, xp), ip, wp

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, idx, w, yp, ip, wp = step()
    for seed in range(3):
        a, b = tokens(kind, 2, 288, 6, 3, seed), tokens(kind, 40, 288, 6, 3, seed)
        for dst, src in ((x, a[0]), (lg, a[1]), (xp, b[0]), (lgp, b[1])):
            dst.copy_(src)
        graph.replay()
        got, gotp = y.clone(), yp.clone()
        ref.check(got, *ref.moe(x, idx, w, experts))
        ref.check(gotp, *ref.moe(xp, ip, wp, experts))
        ye, *_ = step()  # eager, on memory of its own but for the workspace
        torch.cuda.synchronize()
        assert torch.equal(ye, got)


def test_modules_and_builders():
    """Int8Linear, the template expert and the inline forwards give the operators' results."""
    from tinyserve_amd.expert_forward import (Int8ExpertModule, _build_cpp_layout_args, _build_dense_inline_forward,
                                              _precompute_param_refs, fast_expert_forward, forward_from_packed)
    from tinyserve_amd.int8 import Int8Linear

    g = gen(7)
    w, ws = ref.weights8(g, 96, 144)
    b = torch.randn(96, device="cuda", generator=g).bfloat16()
    x = torch.randn((2, 3, 144), device="cuda", generator=g).bfloat16()
    y = Int8Linear(w, ws[:, None], b)(x)
    assert y.shape == (2, 3, 96) and torch.equal(y.view(6, 96), ops.int8_linear(x.view(6, 144), w, ws, b))
    H, I = 256, 160
    for kind in KINDS:
        lay = synth.int8_layout(H, I) if kind == "int8" else synth.dense_layout(H, I, DT[kind])
        L, pool, ex = layer(kind, H, I, 1)
        for T in (1, 5, 40):
            h, _ = tokens(kind, T, H, 1, 1)
            zero, one = torch.zeros((T, 1), dtype=torch.int32, device="cuda"), torch.ones((T, 1), device="cuda")
            want = ref.moe(h, zero, one, ex)
            ref.check(_build_dense_inline_forward(lay, None)(pool[0], h), *want)
            ref.check(fast_expert_forward(h, zero, one, pool, **_build_cpp_layout_args(lay, None)), *want)
            if kind == "int8":
                mod = Int8ExpertModule(lay, device="cuda")
                ref.check(forward_from_packed(mod, pool[0], _precompute_param_refs(mod, lay), h), *want)


@pytest.mark.parametrize("kind", ["16-bit", "int8", "fused"])
@pytest.mark.parametrize("T", [1, 3, 40])
def test_pipeline_and_hook(tmp_path, kind, T):
    """A checkpoint on disk through the store, the pipeline, the batcher and an installed MoE block."""
    import torch.nn as nn

    from tests.test_int8_host import save_experts
    from tinyserve_amd.expert_batcher import BatchItem
    from tinyserve_amd.expert_pipeline import ExpertPipeline, install_offloaded_forward
    from tinyserve_amd.expert_store import ExpertStore

    H, I, E, k = 160, 96, 6, 2
    want = save_experts(tmp_path, "int8" if kind == "int8" else "16-bit", np.random.default_rng(3), (0, 1), E, H, I)
    if kind == "fused":
        from safetensors.torch import save_file

        out = {}
        for li in (0, 1):
            out[f"model.layers.{li}.mlp.experts.gate_up_proj"] = torch.stack([torch.cat([want[li, e]["gate_proj"], want[li, e]["up_proj"]]) for e in range(E)])
            out[f"model.layers.{li}.mlp.experts.down_proj"] = torch.stack([want[li, e]["down_proj"] for e in range(E)])
        save_file(out, str(tmp_path / "model.safetensors"))
    store, _ = ExpertStore.from_safetensors(str(tmp_path))
    template = None
    if kind == "fused":
        template = nn.Module()
        template._act_fn = nn.SiLU()
        for n, (shape, dtype) in store.layout.specs.items():
            template.register_parameter(n, nn.Parameter(torch.zeros(shape, dtype=dtype, device="cuda"), requires_grad=False))
    pipe = ExpertPipeline(store, template, "cuda")
    g = gen(T)
    for li in (0, 1):
        ex = [{n: t.cuda() for n, t in want[li, e].items()} for e in range(E)]
        x = torch.randn((T, H), device="cuda", generator=g).bfloat16()
        block = nn.Module()
        block.gate = nn.Linear(H, E, bias=False).to("cuda", torch.bfloat16)
        install_offloaded_forward(block, pipe, li, "gate", k)
        lg = ops.router_logits(x, block.gate.weight)
        idx, w = ops.route_topk(lg.float(), k)
        y = block.forward(x)
        ref.check(y, *ref.moe(x, idx, w if T <= 4 else w.bfloat16(), ex), "hook")
        ref.check(pipe.execute_layer_experts(x, li, idx, w), *ref.moe(x, idx, w, ex), "decode")
        ref.check(pipe.execute_layer_experts_batched(x, li, idx, w), *ref.moe(x, idx, w, ex), "batched")
        items = [BatchItem(x[i : i + 1], idx[i], w[i], i) for i in range(T)]
        ref.check(torch.cat(pipe.execute_batched_experts(items, li)), *ref.moe(x, idx, w, ex), "batcher")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("H,I,E,k,T", [(256, 320, 12, 4, 16), (256, 320, 12, 4, 17), (1024, 1024, 9, 2, 6), (1024, 1024, 9, 2, 7),
                                       (1024, 1024, 9, 2, 12), (1024, 1024, 9, 2, 13), (2048, 768, 10, 8, 2), (2048, 768, 10, 8, 3),
                                       (64, 32, 70, 64, 2), (64, 32, 70, 64, 3), (64, 32, 3, 1, 64), (64, 32, 3, 1, 65)])
def test_last_tokens_as_pairs(kind, H, I, E, k, T):
    """Either side of the most tokens that run as pairs, routed and given; the buffers that a capture would hold."""
    L, pool, experts = layer(kind, H, I, E)
    x, lg = tokens(kind, T, H, E, k)
    slot = torch.arange(E, dtype=torch.int32, device="cuda")
    y, idx, w = ops.moe_decode_routed(L, pool, slot, lg, x, k, return_routing=True, workspace=ops.moe_decode_workspace(L, T, k, "cuda"))
    want = ref.moe(x, idx, w, experts)
    ref.check(y, *want, "routed")
    ref.check(ops.moe_decode(L, pool, idx, w, x), *want, "given")
    ref.check(ops.moe_prefill(L, pool, slot, idx, w, x), *want, "prefill")


@pytest.mark.parametrize("kind", KINDS)
def test_prompt_in_pieces(kind):
    """More assignments than are worked on at a time."""
    H, I, E, k, T = 64, 32, 6, 4, 70_001
    L, pool, experts = layer(kind, H, I, E)
    x, lg = tokens(kind, T, H, E, k)
    idx, w = ops.route_topk(lg, k)
    slot = torch.arange(E, dtype=torch.int32, device="cuda")
    ref.check(ops.moe_prefill(L, pool, slot, idx, w, x), *ref.moe(x, idx, w, experts))


@pytest.mark.parametrize("kind", ["bf16", "int8"])
def test_far_slots(kind):
    """Slots past 2^32 bytes of the pool."""
    H, I, E, k = 256, 96, 6, 3
    L, small, experts = layer(kind, H, I, E)
    L.slot_bytes = 2**30 - 16
    pool = torch.zeros((E, 2**30 - 16), dtype=torch.uint8, device="cuda")
    pool[:, : small.shape[1]] = small
    slot = torch.arange(E, dtype=torch.int32, device="cuda")
    for T in (1, 2, 50):
        x, lg = tokens(kind, T, H, E, k)
        y, idx, w = ops.moe_decode_routed(L, pool, slot, lg, x, k, return_routing=True)
        want = ref.moe(x, idx, w, experts)
        ref.check(y, *want, "routed")
        ref.check(ops.moe_prefill(L, pool, slot, idx, w, x), *want, "prefill")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T", [2, 60])
def test_same_expert_twice(kind, T):
    """A selection that names an expert more than once adds it as often."""
    L, pool, experts = layer(kind, 256, 96, 4)
    x, _ = tokens(kind, T, 256, 4, 3)
    idx = torch.tensor([[1, 1, 3], [2, 2, 2]], dtype=torch.int32, device="cuda").repeat(T // 2, 1)
    w = torch.rand((T, 3), device="cuda", generator=gen(5))
    slot = torch.arange(4, dtype=torch.int32, device="cuda")
    want = ref.moe(x, idx, w, experts)
    ref.check(ops.moe_decode(L, pool, idx, w, x), *want, "decode")
    ref.check(ops.moe_prefill(L, pool, slot, idx, w, x), *want, "prefill")
