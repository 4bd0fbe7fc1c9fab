"""int8, grouped products and 16-bit / int8 experts without a GPU: refusals of the C ABI and the Python entry
points, slot layouts, the checkpoint store, the module swap."""
from __future__ import annotations

import ctypes
import os

import numpy as np
import pytest
import torch
import torch.nn as nn

from tinyserve_amd import _lib, ops, synth
from tinyserve_amd.expert_forward import (Int8ExpertModule, _build_cpp_layout_args, _build_dense_inline_forward, build_expert_layout,
                                          dense_expert_layout, int8_expert_layout)
from tinyserve_amd.expert_store import ExpertStore, TensorLayout
from tinyserve_amd.int8 import Int8Linear, replace_linear_with_int8

P = ctypes.c_void_p(4096)
BAD, SHAPE = _lib.ERR_INVALID_ARG, _lib.ERR_SHAPE


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built (run __graft_entry__.build())")
    return _lib.load()


# ----------------------------------------------------------------------------- the C ABI
@pytest.mark.parametrize("T,K,N,text", [
    (4, 100, 64, b"multiple of 16"), (4, 0, 64, b"bad shape"), (4, 128, 0, b"bad shape"), (-1, 128, 64, b"bad shape"),
    (4, 131072, 64, b"at most 131056"), (1 << 31, 128, 64, b"too large"), (1, 128, (1 << 30) + 1, b"too large"),
    (1 << 30, 128, 1 << 30, b"too large")])
def test_matmul_refusals(lib, T, K, N, text):
    assert lib.tsa_int8_matmul(P, P, T, K, P, P, N, None, 0, P, 2, None) == SHAPE and text in lib.tsa_last_error()
    assert lib.tsa_int8_linear(P, 2, T, K, P, P, N, None, 0, P, 2, P, 1 << 50, None) == SHAPE and text in lib.tsa_last_error()


def test_matmul_argument_errors(lib):
    assert lib.tsa_int8_matmul(None, P, 4, 128, P, P, 64, None, 0, P, 2, None) == BAD
    assert lib.tsa_int8_matmul(P, P, 4, 128, P, P, 64, None, 0, P, 7, None) == BAD
    assert lib.tsa_int8_matmul(P, P, 4, 128, P, P, 64, P, 9, P, 2, None) == BAD
    assert lib.tsa_int8_matmul(ctypes.c_void_p(4100), P, 4, 128, P, P, 64, None, 0, P, 2, None) == BAD
    assert b"16-byte aligned" in lib.tsa_last_error()
    assert lib.tsa_int8_linear(P, 5, 4, 128, P, P, 64, None, 0, P, 2, P, 1 << 20, None) == BAD
    assert lib.tsa_int8_linear(P, 2, 40, 128, P, P, 64, None, 0, P, 2, P, 100, None) == _lib.ERR_WORKSPACE
    assert lib.tsa_int8_linear(P, 2, 40, 128, P, P, 64, None, 0, P, 2, None, 1 << 20, None) == _lib.ERR_WORKSPACE
    assert lib.tsa_int8_linear(P, 2, 40, 128, P, P, 64, None, 0, P, 2, ctypes.c_void_p(4104), 1 << 20, None) == _lib.ERR_WORKSPACE
    # no tokens: nothing to do, whatever the pointers
    assert lib.tsa_int8_matmul(None, None, 0, 128, None, None, 64, None, 0, None, 2, None) == 0
    assert lib.tsa_int8_linear(None, 2, 0, 128, None, None, 64, None, 0, None, 2, None, 0, None) == 0
    assert lib.tsa_int8_quantize(None, 2, 0, 128, None, None, None) == 0
    assert lib.tsa_int8_quantize(None, 2, 3, 128, None, None, None) == BAD
    assert lib.tsa_int8_quantize(P, 3, 3, 128, P, P, None) == BAD
    assert lib.tsa_int8_quantize(P, 2, 3, 0, P, P, None) == SHAPE
    assert lib.tsa_int8_quantize(P, 2, (1 << 30) + 1, 8, P, P, None) == SHAPE


def test_linear_workspace(lib):
    n = ctypes.c_int64()
    size = lambda T, K: (lib.tsa_int8_linear_workspace_size(T, K, ctypes.byref(n)), n.value)  # noqa: E731
    assert size(1, 2880) == (0, 0) and size(100, 2880)[1] >= 100 * (2880 + 4)
    assert size(-1, 2880)[0] == BAD and size(1, 131072)[0] == BAD
    # rows that do not fit LDS need a workspace whatever their number
    assert size(1, 131056)[1] >= 131056 + 4 or size(1, 131056)[1] == 0
    got = [size(T, 2880)[1] for T in (1, 8, 16, 17, 100, 1000)]
    assert got == sorted(got)


def _grouped(lib, dtype=2, x=P, x_rows=8, K=64, w=P, stride=None, E=4, N=32, off=P, rows=None, R=8, k=1, bias=None, bt=0, y=P, yt=2):
    stride = N * K * 2 if stride is None else stride
    return lib.tsa_grouped_matmul(x, dtype, x_rows, K, w, stride, E, N, off, rows, R, k, bias, bt, y, yt, None)


@pytest.mark.parametrize("kw,rc,text", [
    (dict(dtype=0), BAD, b"bad dtype"), (dict(dtype=3), BAD, b"bad dtype"), (dict(yt=5), BAD, b"bad dtype"), (dict(bias=P, bt=9), BAD, b"bad dtype"),
    (dict(K=0, stride=64), SHAPE, b"bad shape"), (dict(E=0), SHAPE, b"bad shape"), (dict(N=0), SHAPE, b"bad shape"), (dict(R=-1), SHAPE, b"bad shape"),
    (dict(k=0), SHAPE, b"bad shape"), (dict(x_rows=-1), SHAPE, b"bad shape"), (dict(K=60), SHAPE, b"multiple of 8"), (dict(K=131064), SHAPE, b"at most"),
    (dict(E=65537), SHAPE, b"too many"), (dict(R=1 << 30, x_rows=1 << 30), SHAPE, b"too many"), (dict(N=1 << 25), SHAPE, b"too many"),
    (dict(R=1 << 22, x_rows=1 << 22, N=1 << 12), SHAPE, b"too many"), (dict(stride=32 * 64 * 2 - 16), SHAPE, b"overlap"),
    (dict(stride=32 * 64 * 2 + 8), SHAPE, b"16-byte"), (dict(R=9), SHAPE, b"x has 8 rows"), (dict(x_rows=0, rows=P), SHAPE, b"x has 0 rows"),
    (dict(x_rows=1 << 24, rows=P), SHAPE, b"2^31"), (dict(x=None), BAD, b"null"), (dict(w=None), BAD, b"null"), (dict(off=None), BAD, b"null"),
    (dict(y=None), BAD, b"null"), (dict(x=ctypes.c_void_p(4104)), BAD, b"16-byte"), (dict(w=ctypes.c_void_p(4104)), BAD, b"16-byte")])
def test_grouped_refusals(lib, kw, rc, text):
    assert _grouped(lib, **kw) == rc and text in lib.tsa_last_error(), lib.tsa_last_error()


def test_grouped_int8_refusals(lib):
    f = lambda codes=P, scales=P, K=64, ws=P, R=8: lib.tsa_int8_grouped_matmul(  # noqa: E731
        codes, scales, 8, K, P, 32 * K, ws, 4, 32, P, None, R, 1, None, 0, P, 2, None)
    assert f(K=72) == SHAPE and b"multiple of 16" in lib.tsa_last_error()
    assert f(scales=None) == BAD and f(ws=None) == BAD and f(codes=None) == BAD
    assert f(R=0) == 0
    assert _grouped(lib, R=0, x=None, w=None, off=None, y=None) == 0


def _check(lib, L):
    n = ctypes.c_int64()
    return lib.tsa_moe_decode_workspace_size(ctypes.byref(L), 1, 2, ctypes.byref(n)), lib.tsa_last_error()


@pytest.mark.parametrize("kind", ["16-bit", "int8"])
def test_layout_refusals(lib, kind):
    H, I = 288, 736
    lay = synth.int8_layout(H, I) if kind == "int8" else synth.dense_layout(H, I)
    make = lambda: build_expert_layout(lay)  # noqa: E731
    assert lay.total_bytes % 16 == 0 and _check(lib, make())[0] == 0
    cases = [("gate_off", 8, b"multiples of 16"), ("slot_bytes", lay.total_bytes + 4, b"multiple of 16"), ("gate_bias_off", 0, b"biases"),
             ("down_off", lay.total_bytes - 16, b"exceeds slot_bytes"), ("up_off", -1, b"exceeds slot_bytes"), ("hidden", 296, b"multiples of 32"),
             ("mx_tiled", 1, b"mx_tiled"), ("act", 5, b"act"), ("slot_bytes", 1 << 31, b"below 2^31")]
    if kind == "int8":
        cases += [("gate_scales_off", lay.total_bytes - 16, b"exceeds slot_bytes"), ("down_scales_off", -1, b"exceeds slot_bytes"),
                  ("down_scales_off", lay.offsets["down_proj_scale"] - 4, b"multiples of 16")]
    else:
        cases += [("gate_type", 0, b"16-bit experts"), ("down_type", 1, b"16-bit experts")]
    for field, value, text in cases:
        L = make()
        setattr(L, field, value)
        rc, msg = _check(lib, L)
        assert rc != 0 and text in msg, (field, value, msg)


def test_activations_of_another_type(lib):
    """16-bit experts and activations of another type: refused ahead of any launch."""
    L = build_expert_layout(synth.dense_layout(64, 32))
    n = ctypes.c_int64()
    for T in (1, 9):
        lib.tsa_moe_prefill_workspace_size(ctypes.byref(L), T, 2, 4, ctypes.byref(n))
        for xt in (0, 1):
            assert lib.tsa_moe_decode(ctypes.byref(L), P, 1, P, P, T, 2, P, xt, P, 2, P, 1 << 30, None) == BAD
            assert b"own type" in lib.tsa_last_error()
        assert lib.tsa_moe_decode_routed(ctypes.byref(L), P, 1, P, 4, P, 0, 0, T, 2, P, 1, P, 2, None, None, P, 1 << 30, None) == BAD
        assert lib.tsa_moe_decode(ctypes.byref(L), P, 1, P, P, T, 2, ctypes.c_void_p(4104), 2, P, 2, P, 1 << 30, None) == BAD
        assert b"16-byte aligned" in lib.tsa_last_error()
    assert lib.tsa_moe_prefill(ctypes.byref(L), P, 1, P, 4, P, P, 9, 2, P, 1, P, 2, P, n.value, None) == BAD
    assert b"own type" in lib.tsa_last_error()
    assert lib.tsa_moe_prefill(ctypes.byref(L), P, 1, P, 4, P, P, 9, 2, P, 2, P, 2, P, n.value - 1, None) == _lib.ERR_WORKSPACE


@pytest.mark.parametrize("kind", ["16-bit", "int8"])
@pytest.mark.parametrize("H,I,k,E", [(2048, 768, 8, 128), (2880, 2880, 4, 32), (64, 16384, 16, 20), (16384, 64, 1, 4)])
def test_prompt_workspace(lib, kind, H, I, k, E):
    """The workspace of a prompt stops growing where it is worked through in pieces, and a workspace for more tokens
    serves fewer."""
    L, n, got = build_expert_layout(synth.int8_layout(H, I) if kind == "int8" else synth.dense_layout(H, I)), ctypes.c_int64(), []
    for T in (1, 2, 4, 5, 6, 64, 1024, 131072 // k, 131072, 1 << 20, 1 << 24):
        assert lib.tsa_moe_prefill_workspace_size(ctypes.byref(L), T, k, E, ctypes.byref(n)) == 0
        got.append(n.value)
    assert got == sorted(got) and got[7] == got[-1]
    assert got[-1] < 131072 * (5 * H + 5 * I + 64) + (1 << 20)


# ----------------------------------------------------------------------------- the Python entry points
def test_host_tensors_are_refused():
    w, s = synth.make_int8(np.random.default_rng(0), 16, 32)
    x, off = torch.zeros(1, 32, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int32)
    for f in (lambda: ops.int8_quantize(x), lambda: ops.int8_linear(x, w, s), lambda: ops.int8_matmul(w, s, w, s),
              lambda: ops.grouped_matmul(x, x.view(1, 1, 32), off), lambda: ops.int8_grouped_matmul(w, s, w[None], s[None], off)):
        with pytest.raises(RuntimeError, match="must be on CUDA"):
            f()


def test_python_refusals():
    """What the wrappers check themselves (on tensors without data: nothing is launched)."""
    m = lambda *shape, dtype=torch.int8: torch.empty(shape, dtype=dtype, device="meta")  # noqa: E731
    f32, bf = torch.float32, torch.bfloat16
    for args, text in (((m(4, 32, dtype=f32), m(4, dtype=f32)), "must be int8"), ((m(4, 32), m(5, dtype=f32)), "activation scales"),
                       ((m(4, 32), m(4, dtype=bf)), "activation scales")):
        with pytest.raises(RuntimeError, match=text):
            ops._int8_codes(*args)
    for args, text in (((m(4, 32, dtype=f32), m(4), 32), "must be int8"), ((m(4, 32), m(4), 48), "in_features differ"),
                       ((m(4, 32), m(5), 32), "weight scales"), ((m(4, 32), m(2, 2), 32), "weight scales")):
        with pytest.raises(RuntimeError, match=text):
            ops._int8_weight(*args)
    for args, text in (((m(2, 4, 32, dtype=bf), 32, torch.float16), "must be torch.float16"), ((m(4, 32, dtype=bf), 32, bf), "must be"),
                       ((m(2, 4, 32, dtype=bf), 48, bf), "in_features differ"), ((m(0, 4, 32, dtype=bf), 32, bf), "in_features differ")):
        with pytest.raises(RuntimeError, match=text):
            ops._grouped_weight(*args)
    x, i32 = m(6, 32, dtype=bf), torch.int32
    for args, text in (((x, m(3, dtype=torch.int64), None, 1, 2), "offsets"), ((x, m(4, dtype=i32), None, 1, 2), "offsets"),
                       ((x, m(3, dtype=i32), None, 2, 2), "top_k"), ((x, m(3, dtype=i32), m(6, dtype=torch.int64), 1, 2), "rows"),
                       ((x, m(3, dtype=i32), m(2, 3, dtype=i32), 1, 2), "rows"), ((x, m(3, dtype=i32), m(6, dtype=i32), 0, 2), "rows")):
        with pytest.raises(RuntimeError, match=text):
            ops._grouped_rows(*args)
    with pytest.raises(RuntimeError, match="bias must be"):
        ops._grouped_bias(m(8, dtype=bf), 2, 4)


# ----------------------------------------------------------------------------- layouts
def test_layouts_of_slots():
    lay = synth.int8_layout(256, 160)
    L = build_expert_layout(lay)
    assert (L.format, L.hidden, L.inter, L.slot_bytes) == (_lib.EXPERT_INT8, 256, 160, lay.total_bytes)
    assert L.up_off == 160 * 256 and L.gate_scales_off == 3 * 160 * 256 and L.down_scales_off == L.gate_scales_off + 8 * 160
    for dt in (torch.bfloat16, torch.float16):
        lay16 = synth.dense_layout(256, 160, dt)
        L = build_expert_layout(lay16, nn.SiLU())
        assert (L.format, L.gate_type, L.down_type, L.down_off) == (_lib.EXPERT_DENSE, _lib.tsa_dtype(dt), _lib.tsa_dtype(dt), 4 * 160 * 256)
        fused = TensorLayout({"gate_up_proj": ((320, 256), dt), "down_proj": ((256, 160), dt)})
        F = dense_expert_layout(fused, nn.SiLU())
        assert (F.gate_off, F.up_off, F.down_off, F.gate_type) == (0, 2 * 160 * 256, 4 * 160 * 256, _lib.tsa_dtype(dt))
        assert build_expert_layout(fused, nn.SiLU()) is None
        with pytest.raises(ValueError, match="not a 16-bit"):
            dense_expert_layout(fused)  # interleaved rows
        assert _build_dense_inline_forward(lay16, None).expert_layout.format == _lib.EXPERT_DENSE
        assert _build_cpp_layout_args(lay16, None)["layout"].format == _lib.EXPERT_DENSE
    assert _build_dense_inline_forward(lay, None).expert_layout.format == _lib.EXPERT_INT8
    assert _build_dense_inline_forward(fused, None) is None and _build_cpp_layout_args(fused, nn.SiLU()) is None
    for f, l in ((int8_expert_layout, lay), (dense_expert_layout, lay16)):
        with pytest.raises(NotImplementedError, match="activation"):
            f(l, nn.GELU())
        with pytest.raises(ValueError, match="not a"):
            f(synth.mxfp4_layout(64, 64))
    with pytest.raises(ValueError, match="inconsistent"):
        int8_expert_layout(TensorLayout({**lay.specs, "up_proj": ((128, 256), torch.int8)}))
    with pytest.raises(ValueError, match="inconsistent"):
        int8_expert_layout(TensorLayout({**lay.specs, "up_proj_scale": ((128,), torch.float32)}))
    with pytest.raises(ValueError, match="inconsistent"):
        dense_expert_layout(TensorLayout({**lay16.specs, "down_proj": ((256, 160), torch.bfloat16)}))
    with pytest.raises(ValueError, match="not a 16-bit"):  # [in, out] matrices
        dense_expert_layout(TensorLayout({"gate_up_proj": ((256, 320), dt), "down_proj": ((160, 256), dt)}), nn.SiLU())
    names = list(lay.specs)
    with pytest.raises(ValueError, match="must follow"):
        int8_expert_layout(TensorLayout({n: lay.specs[n] for n in names[:3] + [names[4], names[3], names[5]]}))


@pytest.mark.parametrize("H,I,act", [(256, 160, nn.GELU()), (256, 160, torch.nn.functional.relu), (250, 160, None), (256, 48, nn.SiLU()),
                                     (32768, 32, None), (64, 16416, None)])
def test_16_bit_slots_for_their_template(H, I, act):
    """16-bit experts that the kernels do not take have no kernel layout: a pipeline over them is built as before, and forward_from_packed runs its template."""
    from tinyserve_amd.expert_forward import forward_from_packed
    from tinyserve_amd.expert_pipeline import ExpertPipeline

    bf, specs = torch.bfloat16, {"gate_proj": ((I, H), torch.bfloat16), "up_proj": ((I, H), torch.bfloat16), "down_proj": ((H, I), torch.bfloat16)}
    lay = TensorLayout(specs)
    assert build_expert_layout(lay, act) is None and _build_dense_inline_forward(lay, act) is None and _build_cpp_layout_args(lay, act) is None
    assert build_expert_layout(TensorLayout({**specs, "down_proj": ((H, I + 32), bf)})) is None

    class Template(nn.Module):
        def __init__(self):
            super().__init__()
            self._act_fn = act
            for n, (shape, dt) in specs.items():
                self.register_parameter(n, nn.Parameter(torch.zeros(shape, dtype=dt), requires_grad=False))

        def forward(self, h):
            return (self._act_fn or nn.functional.silu)(h @ self.gate_proj.t()) * (h @ self.up_proj.t()) @ self.down_proj.t()

    packed = torch.randn(lay.total_bytes // 2).to(bf).view(torch.uint8)
    t, h = Template(), torch.randn(2, H).to(bf)
    store = type("Store", (), dict(layout=lay, num_layers=1, num_experts=1, expert_bytes=lay.total_bytes))()
    pipe = ExpertPipeline(store, t, torch.device("cpu"), staging_buffer_a=object(), staging_buffer_b=object())
    assert pipe._inline_fwd is None and pipe._cpp_layout_args is None
    y = forward_from_packed(t, packed, pipe._param_refs, h)
    g, u, d = (packed[lay.offsets[n] : lay.offsets[n] + lay.sizes[n]].view(bf).view(specs[n][0]) for n in specs)
    assert torch.equal(y, (act or nn.functional.silu)(h @ g.t()) * (h @ u.t()) @ d.t())


def test_make_int8():
    w, s = synth.make_int8(np.random.default_rng(0), 200, 272)
    assert w.dtype == torch.int8 and s.shape == (200,) and (w.abs().amax(1) == 127).all()
    assert abs(float((w.float() * s[:, None]).std()) - 0.03) < 2e-3


# ----------------------------------------------------------------------------- checkpoints
def save_experts(path, kind: str, rng, layers, E, H, I, drop=None, dtype=torch.bfloat16, flat=False):
    """A checkpoint of per-expert tensors; {(layer, expert): the tensors of the slot}."""
    from safetensors.torch import save_file

    out, want = {}, {}
    for li in layers:
        for e in range(E):
            t = synth.make_int8_expert(rng, H, I) if kind == "int8" else synth.make_dense_expert(rng, H, I, dtype)
            want[li, e] = t
            for n, v in t.items():
                key = n[: -len("_scale")] + ".weight_scale" if n.endswith("_scale") else n + ".weight"
                out[f"model.layers.{li}.mlp.experts.{e}.{key}"] = (v if flat else v[:, None]).clone() if n.endswith("_scale") else v
    if drop:
        del out[drop]
    save_file(out, str(path / "model.safetensors"))
    return want


@pytest.mark.parametrize("kind,dtype,flat", [("int8", torch.bfloat16, False), ("int8", torch.bfloat16, True), ("16-bit", torch.bfloat16, False),
                                             ("16-bit", torch.float16, False)])
def test_store_from_checkpoint(tmp_path, kind, dtype, flat):
    H, I, E = 160, 96, 3
    want = save_experts(tmp_path, kind, np.random.default_rng(1), (1, 4), E, H, I, dtype=dtype, flat=flat)
    st, n = ExpertStore.from_safetensors(str(tmp_path))
    lay = synth.int8_layout(H, I) if kind == "int8" else synth.dense_layout(H, I, dtype)
    assert n == E and st.layer_indices == [1, 4] and st.expert_bytes == lay.total_bytes and st.layout.offsets == lay.offsets
    assert st.layout.specs == lay.specs
    buf = st.allocate_buffer("cpu")
    for s, li in enumerate((1, 4)):
        for e in range(E):
            st.copy_to_buffer(buf, s, e)
            for name, t in want[li, e].items():
                assert torch.equal(buf.get_tensor(name), t)
    assert st.expert_layout().format == (_lib.EXPERT_INT8 if kind == "int8" else _lib.EXPERT_DENSE)
    with pytest.raises(ValueError, match="tiled"):
        ExpertStore.from_safetensors(str(tmp_path), tiled=True)


@pytest.mark.parametrize("kind,drop", [("int8", "1.up_proj.weight"), ("int8", "1.up_proj.weight_scale"), ("16-bit", "1.down_proj.weight")])
def test_store_incomplete(tmp_path, kind, drop):
    save_experts(tmp_path, kind, np.random.default_rng(1), (0,), 2, 64, 32, drop="model.layers.0.mlp.experts." + drop)
    with pytest.raises(ValueError, match="missing"):
        ExpertStore.from_safetensors(str(tmp_path))


def test_store_refuses_other_scales(tmp_path):
    """A scale per tensor, or per group, is not a scale per row; layers of another type are refused."""
    from safetensors.torch import load_file, save_file

    save_experts(tmp_path, "int8", np.random.default_rng(1), (0,), 2, 64, 32)
    f = str(tmp_path / "model.safetensors")
    t = load_file(f)
    key = "model.layers.0.mlp.experts.1.down_proj.weight_scale"
    for bad in (torch.ones(1), torch.ones(64, 2)):
        save_file({**t, key: bad}, f)
        with pytest.raises(ValueError, match="a scale for each row"):
            ExpertStore.from_safetensors(str(tmp_path))
    save_file({**t, "model.layers.0.mlp.experts.1.down_proj.weight": torch.zeros(64, 32)}, f)
    with pytest.raises(ValueError, match="int8|float32"):
        ExpertStore.from_safetensors(str(tmp_path))
    (tmp_path / "b").mkdir()
    save_experts(tmp_path / "b", "16-bit", np.random.default_rng(1), (1,), 2, 64, 32)
    save_file({**t, **load_file(str(tmp_path / "b" / "model.safetensors"))}, f)
    with pytest.raises(ValueError, match="layer 1"):
        ExpertStore.from_safetensors(str(tmp_path))


def test_store_of_fused_experts(tmp_path):
    """Fused unquantised experts keep their slots, and get the kernels' layout where their rows allow it."""
    from safetensors.torch import save_file

    g = torch.Generator().manual_seed(0)
    save_file({"model.layers.0.mlp.experts.gate_up_proj": torch.randn((3, 64, 96), generator=g).bfloat16(),
               "model.layers.0.mlp.experts.down_proj": torch.randn((3, 96, 32), generator=g).bfloat16()}, str(tmp_path / "model.safetensors"))
    st, n = ExpertStore.from_safetensors(str(tmp_path))
    L = st.expert_layout(nn.SiLU())
    off = st.layout.offsets  # in the checkpoint's order
    assert n == 3 and (L.format, L.hidden, L.inter, L.slot_bytes) == (_lib.EXPERT_DENSE, 96, 32, st.expert_bytes)
    assert (L.gate_off, L.up_off, L.down_off) == (off["gate_up_proj"], off["gate_up_proj"] + 2 * 32 * 96, off["down_proj"])


# ----------------------------------------------------------------------------- modules
def test_replace_linear():
    model = nn.Sequential(nn.Linear(32, 48), nn.Sequential(nn.Linear(48, 16, bias=False)), nn.ReLU())
    w = {n: synth.make_int8(np.random.default_rng(0), *s) for n, s in (("0", (48, 32)), ("1.0", (16, 48)), ("2", (4, 16)), ("9.x", (4, 16)))}
    assert replace_linear_with_int8(model, w, device="cpu") == 2
    assert isinstance(model[0], Int8Linear) and model[0].bias is not None and model[1][0].bias is None
    assert model[1][0].weight_scale.shape == (16, 1)
    with pytest.raises(ValueError, match="weight_scale"):
        Int8Linear(w["0"][0], torch.zeros(1), device="cpu")
    with pytest.raises(ValueError, match="multiple of 16"):
        Int8Linear(torch.zeros(4, 24, dtype=torch.int8), torch.zeros(4), device="cpu")
    with pytest.raises(ValueError, match="must be int8"):
        Int8Linear(torch.zeros(4, 32), torch.zeros(4), device="cpu")


@pytest.mark.parametrize("cast", [lambda m: m.to(torch.bfloat16), lambda m: m.half(), lambda m: m.double(), lambda m: m.type(torch.float16),
                                  lambda m: m.to("cpu", torch.float16), lambda m: m.float()])
def test_casts_keep_the_format(cast):
    """A model cast to another type keeps its int8 weights and their scales; biases and the rest change."""
    w, s = synth.make_int8(np.random.default_rng(0), 160, 144)
    model = nn.Sequential(Int8Linear(w, s[:, None], torch.randn(160), device="cpu"), nn.Linear(4, 4))
    lin = cast(model)[0]
    assert torch.equal(lin.weight, w) and lin.weight_scale.dtype == torch.float32 and torch.equal(lin.weight_scale[:, 0], s)
    assert lin.bias.dtype == model[1].weight.dtype and not lin.weight.requires_grad
    lay = synth.int8_layout(128, 96)
    mod = cast(Int8ExpertModule(lay, device="cpu"))
    assert {n: p.dtype for n, p in mod.named_parameters()} == {n: d for n, (_, d) in lay.specs.items()}


def test_module_moves_and_loads():
    w, s = synth.make_int8(np.random.default_rng(0), 32, 48)
    lin = Int8Linear(w, s, device="cpu")
    other = Int8Linear(w, s, device="cpu").to("meta")
    assert other.weight.is_meta and other.weight.dtype == torch.int8 and other.weight_scale.is_meta
    other = other.to_empty(device="cpu")
    other.load_state_dict(lin.state_dict())
    assert torch.equal(other.weight, w) and torch.equal(other.weight_scale[:, 0], s)
