"""Which packed expert slots get a kernel layout, and what runs those that get none: the layout builders, the store, the
pipeline and the batcher over int8 and 16-bit slots (CPU)."""
from __future__ import annotations

import pytest
import torch
import torch.nn as nn

from tinyserve_amd import _lib, synth
from tinyserve_amd.expert_batcher import BatchItem, ExpertBatcher
from tinyserve_amd.expert_forward import (Int8ExpertModule, _build_cpp_layout_args, _build_dense_inline_forward, build_expert_layout,
                                          int8_expert_layout, template_activation)
from tinyserve_amd.expert_pipeline import ExpertPipeline
from tinyserve_amd.expert_store import ExpertStore, TensorLayout, pack_tensors

H, I, E = 64, 32, 3
INT8 = synth.int8_layout(H, I).specs


def store_of(specs: dict, seed: int = 0) -> ExpertStore:
    """One layer of E experts whose tensors are small random values (scales positive)."""
    lay, g = TensorLayout(specs, align=16), torch.Generator().manual_seed(seed)
    data = torch.zeros((1, E, lay.total_bytes), dtype=torch.uint8)
    for e in range(E):
        tensors = {}
        for n, (shape, dt) in specs.items():
            if dt == torch.int8:
                tensors[n] = torch.randint(-127, 128, shape, generator=g, dtype=torch.int8)
            elif "_scale" in n:
                tensors[n] = (0.0005 + 0.0005 * torch.rand(shape, generator=g)).to(dt)
            else:
                tensors[n] = (0.05 * torch.randn(shape, generator=g)).to(dt)
        pack_tensors(data[0, e], lay, tensors)
    return ExpertStore(data, lay, 1, E)


class Template(nn.Module):
    """An expert whose parameters are the slot's tensors, computed in float32 by torch: weights times their scales (a scale
    for each row or for groups of a row), zero points and biases where the slot has them."""

    def __init__(self, specs: dict, act=nn.functional.silu, **named):
        super().__init__()
        for n, (shape, dt) in specs.items():
            self.register_parameter(n, nn.Parameter(torch.zeros(shape, dtype=dt), requires_grad=False))
        self._computes = [act]
        for n, v in named.items():
            setattr(self, n, v)

    def _times(self, x, mat):
        w = getattr(self, mat).float()
        if hasattr(self, mat + "_zero_point"):
            w = w - getattr(self, mat + "_zero_point").float().reshape(-1, 1)
        if hasattr(self, mat + "_scale"):
            s = getattr(self, mat + "_scale").float().reshape(w.shape[0], -1)
            w = (w.unflatten(1, (s.shape[1], -1)) * s.unsqueeze(-1)).flatten(1)
        y = x @ w.t()
        return y + getattr(self, mat + "_bias").float() if hasattr(self, mat + "_bias") else y

    def forward(self, h):
        x = h.float()
        return self._times(self._computes[0](self._times(x, "gate_proj")) * self._times(x, "up_proj"), "down_proj").to(h.dtype)


def expert64(store: ExpertStore, e: int, h: torch.Tensor, act=None):
    """(expert e of h in 64 bits, how far float32 may be off): a sum of n terms is off by n 2^-24 of the sum of its terms'
    magnitudes, and the activations' slopes are below 2."""
    lay, act = store.layout, act or nn.functional.silu
    w = {n: store.get_expert_data(0, e)[lay.offsets[n] : lay.offsets[n] + lay.sizes[n]].view(dt).view(shape).double()
         for n, (shape, dt) in lay.specs.items()}
    for m in ("gate_proj", "up_proj", "down_proj"):
        if m + "_scale" in w:
            s = w[m + "_scale"].reshape(len(w[m]), -1)
            w[m] = w[m] * s.repeat_interleave(w[m].shape[1] // s.shape[1], 1)
    x = h.double()
    g, u = x @ w["gate_proj"].t(), x @ w["up_proj"].t()
    mid, down = act(g) * u, w["down_proj"].t()
    want, n1, n2 = mid @ down, x.shape[1] + 4, mid.shape[1] + 4
    eg, eu = (n1 * 2.0**-24 * (x.abs() @ w[m].abs().t()) for m in ("gate_proj", "up_proj"))
    emid = 2 * eg * (u.abs() + eu) + act(g).abs() * eu + 8 * 2.0**-24 * (mid.abs() + g.abs() * u.abs())
    return want, emid @ down.abs() + n2 * 2.0**-24 * ((mid.abs() + emid) @ down.abs()) + 2.0**-24 * want.abs()


def no_kernel(lay: TensorLayout, act=None) -> bool:
    return build_expert_layout(lay, act) is None and _build_dense_inline_forward(lay, act) is None and _build_cpp_layout_args(lay, act) is None


# ----------------------------------------------------------------------------- int8 slots that hold more
@pytest.mark.parametrize("more", [{"down_proj_bias": ((H,), torch.float32)}, {"gate_proj_zero_point": ((I,), torch.int8)},
                                  {"input_scale": ((1,), torch.float32)}])
def test_int8_slots_with_further_tensors(more):
    """The kernels would leave them out: no kernel layout, and no module that drops them."""
    specs = {**INT8, **more}
    lay = TensorLayout(specs, align=16)
    assert no_kernel(lay)
    for f in (int8_expert_layout, Int8ExpertModule):
        with pytest.raises(ValueError, match="not an int8"):
            f(lay)
    pipe = ExpertPipeline(store_of(specs), Template(specs, _act_fn=nn.SiLU()), "cpu")
    assert pipe._inline_fwd is None and pipe._cpp_layout_args is None
    with pytest.raises((ValueError, NotImplementedError)):
        pipe.kernel_layout(0)
    assert build_expert_layout(synth.int8_layout(H, I)).format == _lib.EXPERT_INT8


# ----------------------------------------------------------------------------- int8 slots that the kernels do not take
HALF_SCALES = {n: (shape, torch.float16 if n.endswith("_scale") else dt) for n, (shape, dt) in INT8.items()}
GROUP_SCALES = {n: ((shape[0], 2), dt) if n.endswith("_scale") else (shape, dt) for n, (shape, dt) in INT8.items()}
UP_SCALES_FIRST = {n: INT8[n] for n in ("gate_proj", "up_proj", "down_proj", "up_proj_scale", "gate_proj_scale", "down_proj_scale")}


@pytest.mark.parametrize("specs,act", [(INT8, nn.GELU()), (INT8, nn.functional.relu), (HALF_SCALES, None), (GROUP_SCALES, nn.SiLU()),
                                       (UP_SCALES_FIRST, None), (synth.int8_layout(72, 40).specs, None),
                                       (synth.int8_layout(64, 16416).specs, None), (synth.int8_layout(32768, 32).specs, nn.SiLU())])
def test_int8_slots_for_their_template(specs, act):
    """They have no kernel layout: a pipeline over them is built, and their template runs them."""
    from tinyserve_amd.expert_forward import forward_from_packed

    lay = TensorLayout(specs, align=16)
    assert no_kernel(lay, act)
    store, t = store_of(specs), Template(specs, act or nn.functional.silu, _act_fn=act)
    pipe = ExpertPipeline(store, t, "cpu")
    assert pipe._inline_fwd is None and pipe._cpp_layout_args is None
    hidden = specs["gate_proj"][0][1]
    h = torch.randn((2, hidden), generator=torch.Generator().manual_seed(1))
    y = forward_from_packed(t, store.get_expert_data(0, 1), pipe._param_refs, h)
    want, err = expert64(store, 1, h, act)
    assert ((y.double() - want).abs() <= err).all()


def test_int8_slots_the_kernels_take():
    """Scales as vectors or columns, in the builders' order; act None or SiLU."""
    column = {n: ((shape[0], 1), dt) if n.endswith("_scale") else (shape, dt) for n, (shape, dt) in INT8.items()}
    for specs in (INT8, column):
        for act in (None, nn.SiLU(), nn.functional.silu):
            lay = TensorLayout(specs, align=16)
            assert build_expert_layout(lay, act).format == _lib.EXPERT_INT8
            assert _build_dense_inline_forward(lay, act).expert_layout.down_scales_off == lay.offsets["down_proj_scale"]
            assert _build_cpp_layout_args(lay, act)["layout"].slot_bytes == lay.total_bytes


# ----------------------------------------------------------------------------- the template's activation
DENSE = {dt: synth.dense_layout(H, I, dt).specs for dt in (torch.bfloat16, torch.float16)}
SPLIT = [INT8, DENSE[torch.bfloat16], DENSE[torch.float16]]


@pytest.mark.parametrize("specs", SPLIT)
@pytest.mark.parametrize("named", [{}, {"act_fn": nn.GELU()}, {"_act_fn": None}, {"activation_fn": nn.functional.gelu},
                                   {"activation": nn.ReLU()}, {"_act_fn": nn.GELU(), "act_fn": nn.SiLU()}, {"_act_fn": None, "act_fn": nn.Tanh()}])
def test_templates_that_do_not_name_silu(specs, named):
    """The kernels compute SiLU: a template with another activation, whatever it calls it, is not replaced by them."""
    pipe = ExpertPipeline(store_of(specs), Template(specs, nn.functional.gelu, **named), "cpu")
    assert pipe._inline_fwd is None and pipe._cpp_layout_args is None
    with pytest.raises(NotImplementedError, match="activation"):
        pipe.kernel_layout(0)


@pytest.mark.parametrize("specs", SPLIT)
@pytest.mark.parametrize("named", [{"_act_fn": nn.SiLU()}, {"act_fn": nn.SiLU()}, {"_act_fn": None, "act_fn": nn.functional.silu},
                                   {"activation": nn.SiLU()}, None])
def test_templates_that_name_silu(specs, named):
    """They are, and so are slots without a template."""
    pipe = ExpertPipeline(store_of(specs), None if named is None else Template(specs, **named), "cpu")
    L = pipe.kernel_layout(0)
    assert L.format in (_lib.EXPERT_INT8, _lib.EXPERT_DENSE) and L.act == _lib.ACT_SILU
    assert pipe._inline_fwd.expert_layout.format == L.format and pipe._cpp_layout_args["layout"].format == L.format


def test_own_template():
    lay = synth.int8_layout(H, I)
    t = Int8ExpertModule(lay, device="cpu")
    pipe = ExpertPipeline(store_of(INT8), t, "cpu")
    assert pipe.kernel_layout(0).format == _lib.EXPERT_INT8 and pipe._inline_fwd is not None
    assert set(t.state_dict()) == set(INT8) and not list(t.children())


def test_activations_of_other_formats():
    """MXFP4, FP8 and fused slots take the template's _act_fn alone, as they did."""
    for lay in (synth.mxfp4_layout(64, 64), synth.fp8_layout(64, 32), TensorLayout({"gate_up_proj": ((64, 64), torch.bfloat16), "down_proj": ((64, 32), torch.bfloat16)})):
        t = nn.Module()
        t.act_fn = nn.GELU()
        assert template_activation(t, lay) is None and template_activation(None, lay) is None
        t._act_fn = nn.SiLU()
        assert template_activation(t, lay) is t._act_fn


@pytest.mark.parametrize("specs", SPLIT)
@pytest.mark.parametrize("how", ["parameter", "buffer", "module"])
def test_templates_with_further_tensors(specs, how):
    """Biases, scales or adapters that the template holds itself, for all experts: the kernels would leave them out."""
    t = Template(specs, _act_fn=nn.SiLU())
    if how == "parameter":
        t.down_proj_bias = nn.Parameter(torch.ones(H))
    elif how == "buffer":
        t.register_buffer("smooth", torch.ones(H))
    else:
        t.adapter = nn.Linear(H, 4)
    pipe = ExpertPipeline(store_of(specs), t, "cpu")
    assert pipe._inline_fwd is None and pipe._cpp_layout_args is None
    with pytest.raises(NotImplementedError, match="not in the slot"):
        pipe.kernel_layout(0)
    t.__delattr__({"parameter": "down_proj_bias", "buffer": "smooth", "module": "adapter"}[how])
    assert ExpertPipeline(store_of(specs), t, "cpu").kernel_layout(0).act == _lib.ACT_SILU


# ----------------------------------------------------------------------------- the store's layout, and the batcher
UNTAKEN = [(DENSE[torch.bfloat16], nn.GELU(), {"_act_fn": nn.GELU()}), (DENSE[torch.float16], nn.functional.relu, {"act_fn": nn.functional.relu}),
           (synth.dense_layout(72, 40).specs, None, {"_act_fn": nn.SiLU()}), (synth.int8_layout(72, 40).specs, None, {"act_fn": nn.SiLU()}),
           (INT8, nn.functional.gelu, {}), (GROUP_SCALES, None, {"_act_fn": nn.SiLU()}),
           ({n: (shape, torch.float32) for n, (shape, _) in DENSE[torch.bfloat16].items()}, None, {"_act_fn": nn.SiLU()})]


@pytest.mark.parametrize("specs,act,named", UNTAKEN)
def test_batches_over_slots_the_kernels_do_not_take(specs, act, named):
    """The batcher over the framework's own pipeline runs the loop over experts and their template: experts that are not
    cached yet, then cached ones."""
    store = store_of(specs)
    pipe = ExpertPipeline(store, Template(specs, act or nn.functional.silu, **named), "cpu")
    g = torch.Generator().manual_seed(3)
    chosen = [torch.tensor(c) for c in ([0, 2], [2, 1], [1, 1], [2, 0])]
    items = [BatchItem(torch.randn((1, specs["gate_proj"][0][1]), generator=g), c, torch.rand(2, generator=g), i) for i, c in enumerate(chosen)]
    for _ in range(2):
        for it, y in zip(items, pipe.execute_batched_experts(items, 0)):
            want, err = torch.zeros(()), torch.zeros(())
            for e, w in zip(it.expert_indices.tolist(), it.routing_weights.double()):
                v, d = expert64(store, e, it.hidden_states, act)
                want, err = want + w * v, err + w * (d + 3 * 2.0**-24 * (v.abs() + d))
            assert ((y.double() - want).abs() <= err).all()
    assert pipe.cache.hits == 3 and pipe.cache.misses == 3


@pytest.mark.parametrize("specs,act", [(s, a) for s, a, _ in UNTAKEN])
def test_store_and_builders_agree(specs, act):
    """Where build_expert_layout has none, the store's layout is refused, and a batch without a template too."""
    store = store_of(specs)
    assert build_expert_layout(store.layout, act) is None
    with pytest.raises((ValueError, NotImplementedError)):
        store.expert_layout(act)
    if act is None:
        pipe = ExpertPipeline(store, None, "cpu")
        item = BatchItem(torch.zeros((1, specs["gate_proj"][0][1])), torch.tensor([0]), torch.ones(1), 0)
        with pytest.raises((ValueError, NotImplementedError)):
            ExpertBatcher(pipe).batch_execute([item], 0)


@pytest.mark.parametrize("specs", SPLIT)
def test_templates_that_are_no_modules(specs):
    """Any callable with the slot's tensors as attributes serves as a template."""
    from types import SimpleNamespace

    params = {n: nn.Parameter(torch.zeros(shape, dtype=dt), requires_grad=False) for n, (shape, dt) in specs.items()}
    pipe = ExpertPipeline(store_of(specs), SimpleNamespace(**params), "cpu")
    assert pipe._inline_fwd is None and len(pipe._param_refs) == len(specs)
    assert ExpertPipeline(store_of(specs), SimpleNamespace(**params, _act_fn=nn.SiLU()), "cpu").kernel_layout(0).act == _lib.ACT_SILU
