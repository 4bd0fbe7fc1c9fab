"""Pipelines over int8 and 16-bit slots on the GPU: templates that the kernels stand in for, templates that they leave
alone, and layers whose results do not depend on what their memory held."""
from __future__ import annotations

import pytest
import torch
import torch.nn as nn

from tests import int8_ref as ref
from tests.test_expert_slots_host import DENSE, GROUP_SCALES, INT8, Template, expert64, store_of
from tests.test_gpu_dense_moe import KINDS, layer, tokens
from tinyserve_amd import ops
from tinyserve_amd.expert_batcher import BatchItem
from tinyserve_amd.expert_forward import Int8ExpertModule
from tinyserve_amd.expert_pipeline import ExpertPipeline

pytestmark = pytest.mark.gpu


def items_of(specs, dtype, seed=3):
    g = torch.Generator().manual_seed(seed)
    hidden = specs["gate_proj"][0][1]
    return [BatchItem(torch.randn((1, hidden), generator=g).to("cuda", dtype), torch.tensor(c, device="cuda"), torch.rand(2, generator=g).cuda(), i)
            for i, c in enumerate(([0, 2], [2, 1], [1, 1], [2, 0], [0, 1]))]


@pytest.mark.parametrize("specs,act,named", [(DENSE[torch.bfloat16], nn.functional.gelu, {"act_fn": nn.GELU()}),
                                             (DENSE[torch.float16], nn.functional.relu, {}), (INT8, nn.functional.gelu, {"_act_fn": nn.GELU()}),
                                             (GROUP_SCALES, None, {"_act_fn": nn.SiLU()})])
def test_batches_of_templates(specs, act, named):
    """Templates with another activation, or scales that the kernels do not take, give their own results."""
    store = store_of(specs)
    pipe = ExpertPipeline(store, Template(specs, act or nn.functional.silu, **named).cuda(), "cuda")
    items = items_of(specs, torch.float32)
    for _ in range(2):
        for it, y in zip(items, pipe.execute_batched_experts(items, 0)):
            want, err = torch.zeros(()), torch.zeros(())
            for e, w in zip(it.expert_indices.tolist(), it.routing_weights.double().cpu()):
                v, d = expert64(store, e, it.hidden_states.cpu(), act)
                want, err = want + w * v, err + w * (d + 3 * 2.0**-24 * (v.abs() + d))
            assert ((y.double().cpu() - want).abs() <= err).all()


@pytest.mark.parametrize("specs,dtype,kind", [(INT8, torch.bfloat16, "own")] + [
    (s, d, kind) for s, d in ((INT8, torch.bfloat16), (DENSE[torch.bfloat16], torch.bfloat16), (DENSE[torch.float16], torch.float16))
    for kind in ("act_fn", "none")])
def test_templates_the_kernels_stand_in_for(specs, dtype, kind):
    """A template that names SiLU, the framework's own int8 one, and none: the kernels' layer."""
    store = store_of(specs)
    t = None if kind == "none" else Int8ExpertModule(store.layout, "cuda") if kind == "own" else Template(specs, act_fn=nn.SiLU()).cuda()
    pipe = ExpertPipeline(store, t, "cuda")
    experts = [{n: store.get_expert_data(0, e)[store.layout.offsets[n] : store.layout.offsets[n] + store.layout.sizes[n]].view(dt).view(shape).cuda()
                for n, (shape, dt) in specs.items()} for e in range(store.num_experts)]
    items = items_of(specs, dtype)
    x = torch.cat([it.hidden_states for it in items])
    idx, w = torch.stack([it.expert_indices for it in items]).int(), torch.stack([it.routing_weights for it in items])
    want = ref.moe(x, idx, w, experts)
    ref.check(torch.cat(pipe.execute_batched_experts(items, 0)), *want, "batcher")
    ref.check(pipe.execute_layer_experts(x, 0, idx, w), *want, "decode")
    ref.check(pipe._inline_fwd(pipe.cache.get_packed(pipe.cache.lookup(0, 1)), x),
              *ref.moe(x, torch.ones((5, 1), dtype=torch.int32, device="cuda"), torch.ones((5, 1), device="cuda"), experts), "inline")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("H,I,E,k,T", [(256, 160, 6, 2, 1), (2048, 768, 12, 8, 1), (256, 160, 6, 2, 90), (2048, 768, 12, 8, 300)])
def test_layers_repeat_bit_for_bit(kind, H, I, E, k, T):
    """Every sum has one order: a layer's results are the same each time, whatever the workspace and the results' memory
    held before (NaN in every type, zeros, what the call before left)."""
    L, pool, _ = layer(kind, H, I, E)
    x, lg = tokens(kind, T, H, E, k)
    slot = torch.arange(E, dtype=torch.int32, device="cuda")
    slot[E - 1] = -1  # an expert that is not resident
    idx, w = ops.route_topk(lg, k)
    ws = ops.moe_prefill_workspace(L, T, k, E, "cuda"), ops.moe_decode_workspace(L, T, k, "cuda")
    got = []
    for fill in (0xFF, 0, None, 0x7F, 0xFF):
        if fill is not None:
            for t in ws:
                t.fill_(fill)
            ws[1][: 32 << 10] = 0  # the part that has to hold one value
        out = [torch.full_like(x, float("nan")) for _ in range(3)]
        ops.moe_prefill(L, pool, slot, idx, w, x, out=out[0], workspace=ws[0])
        ops.moe_decode(L, pool, slot[idx.long()], w, x, out=out[1], workspace=ws[1])
        _, ri, rw = ops.moe_decode_routed(L, pool, slot, lg, x, k, out=out[2], workspace=ws[1], return_routing=True)
        got.append(out + [ri, rw])
    torch.cuda.synchronize()
    assert torch.equal(got[0][3], idx) and not any(torch.isnan(t.float()).any() for t in got[0])
    for g in got[1:]:
        assert all(torch.equal(a, b) for a, b in zip(g, got[0]))
