"""FP8 without a GPU: refusals of the C ABI and the Python entry points, slot layouts, the checkpoint
store and the module swap."""
from __future__ import annotations

import ctypes
import os

import numpy as np
import pytest
import torch
import torch.nn as nn

from tests import fp8_ref as ref
from tinyserve_amd import _lib, ops, synth
from tinyserve_amd.expert_forward import build_expert_layout, fp8_expert_layout
from tinyserve_amd.expert_store import ExpertStore, TensorLayout
from tinyserve_amd.fp8 import FP8Linear, replace_linear_with_fp8

P = ctypes.c_void_p(4096)


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built (run __graft_entry__.build())")
    return _lib.load()


@pytest.mark.parametrize("T,K,N,rc,text", [
    (4, 100, 64, _lib.ERR_SHAPE, b"multiple of 16"),
    (4, 0, 64, _lib.ERR_SHAPE, b"bad shape"),
    (4, 128, 0, _lib.ERR_SHAPE, b"bad shape"),
    (-1, 128, 64, _lib.ERR_SHAPE, b"bad shape"),
    (4, (1 << 20) + 16, 64, _lib.ERR_SHAPE, b"multiple of 16"),
    (1 << 31, 128, 64, _lib.ERR_SHAPE, b"too large"),
    (1, 128, (1 << 30) + 1, _lib.ERR_SHAPE, b"too large"),
])
def test_matmul_refusals(lib, T, K, N, rc, text):
    assert lib.tsa_fp8_matmul(P, P, T, K, P, P, N, None, 0, P, 2, None) == rc and text in lib.tsa_last_error()
    assert lib.tsa_fp8_linear(P, 2, T, K, P, P, N, None, 0, P, 2, P, 1 << 50, None) == rc and text in lib.tsa_last_error()


@pytest.mark.parametrize("T,N,y,ok", [(129, 1 << 30, 0, False), (1 << 30, 1 << 20, 2, False), (1 << 30, 1 << 30, 2, False),
                                      (33, 1 << 30, 0, True), (128, 1 << 30, 2, True), (1 << 30, 128, 0, True)])
def test_matmul_more_than_a_launch(lib, T, N, y, ok):
    """Products that no tile covers in one launch are refused before anything runs; the largest others get as
    far as the check of their pointers."""
    assert lib.tsa_fp8_matmul(None, None, T, 16, None, None, N, None, 0, None, y, None) == (_lib.ERR_INVALID_ARG if ok else _lib.ERR_SHAPE)
    assert (b"null pointer" if ok else b"too large") in lib.tsa_last_error()
    assert lib.tsa_fp8_linear(None, 2, T, 16, None, None, N, None, 0, None, y, None, 0, None) == (_lib.ERR_INVALID_ARG if ok else _lib.ERR_SHAPE)


def test_matmul_argument_errors(lib):
    bad = _lib.ERR_INVALID_ARG
    assert lib.tsa_fp8_matmul(None, P, 4, 128, P, P, 64, None, 0, P, 2, None) == bad
    assert lib.tsa_fp8_matmul(P, P, 4, 128, P, P, 64, None, 0, P, 7, None) == bad
    assert lib.tsa_fp8_matmul(P, P, 4, 128, P, P, 64, P, 9, P, 2, None) == bad
    assert lib.tsa_fp8_matmul(ctypes.c_void_p(4100), P, 4, 128, P, P, 64, None, 0, P, 2, None) == bad
    assert b"16-byte aligned" in lib.tsa_last_error()
    assert lib.tsa_fp8_linear(P, 5, 4, 128, P, P, 64, None, 0, P, 2, P, 1 << 20, None) == bad
    assert lib.tsa_fp8_linear(P, 2, 40, 128, P, P, 64, None, 0, P, 2, P, 100, None) == _lib.ERR_WORKSPACE
    assert b"workspace too small" in lib.tsa_last_error()
    assert lib.tsa_fp8_linear(P, 2, 40, 128, P, P, 64, None, 0, P, 2, None, 1 << 20, None) == _lib.ERR_WORKSPACE
    # no tokens: nothing to do, whatever the pointers
    assert lib.tsa_fp8_matmul(None, None, 0, 128, None, None, 64, None, 0, None, 2, None) == 0
    assert lib.tsa_fp8_quantize(None, 2, 0, 128, None, None, None) == 0
    assert lib.tsa_fp8_quantize(None, 2, 3, 128, None, None, None) == bad
    assert lib.tsa_fp8_quantize(P, 3, 3, 128, P, P, None) == bad
    assert lib.tsa_fp8_quantize(P, 2, 3, 0, P, P, None) == _lib.ERR_SHAPE


def test_linear_workspace(lib):
    n = ctypes.c_int64()
    assert lib.tsa_fp8_linear_workspace_size(1, 2880, ctypes.byref(n)) == 0 and n.value == 0
    assert lib.tsa_fp8_linear_workspace_size(100, 2880, ctypes.byref(n)) == 0 and n.value >= 100 * (2880 + 4 * 23)
    assert lib.tsa_fp8_linear_workspace_size(-1, 2880, ctypes.byref(n)) == _lib.ERR_INVALID_ARG


def _check(lib, L):
    n = ctypes.c_int64()
    return lib.tsa_moe_decode_workspace_size(ctypes.byref(L), 1, 2, ctypes.byref(n)), lib.tsa_last_error()


def test_layout_refusals(lib):
    H, I = 2880, 736
    lay = synth.fp8_layout(H, I)
    assert lay.total_bytes % 16 == 0 and _check(lib, fp8_expert_layout(lay))[0] == 0
    for field, value, text in (("gate_off", 8, b"multiples of 16"), ("slot_bytes", lay.total_bytes + 4, b"multiples of 16"),
                               ("gate_bias_off", 0, b"biases"), ("down_scales_off", lay.total_bytes - 8, b"exceeds slot_bytes"),
                               ("down_scales_off", -1, b"exceeds slot_bytes"), ("gate_scales_off", lay.offsets["gate_proj_scale_inv"] + 2, b"multiples of 4"),
                               ("hidden", 2888, b"multiples of 32"), ("mx_tiled", 1, b"mx_tiled"), ("act", 5, b"act")):
        L = fp8_expert_layout(lay)
        setattr(L, field, value)
        rc, msg = _check(lib, L)
        assert rc != 0 and text in msg, (field, msg)
    L = fp8_expert_layout(lay)
    L.format = 4
    assert _check(lib, L)[0] == _lib.ERR_INVALID_ARG


def test_layout_of_slots():
    lay = synth.fp8_layout(256, 160)
    L = build_expert_layout(lay)
    assert (L.format, L.hidden, L.inter, L.slot_bytes) == (_lib.EXPERT_FP8, 256, 160, lay.total_bytes)
    assert L.up_off == 160 * 256 and L.down_scales_off == 3 * 160 * 256 + 2 * 4 * 2 * 2
    fp8_expert_layout(lay, nn.SiLU())
    with pytest.raises(NotImplementedError, match="activation"):
        fp8_expert_layout(lay, nn.GELU())
    with pytest.raises(ValueError, match="not an FP8 expert"):
        fp8_expert_layout(synth.mxfp4_layout(64, 64))
    names = list(lay.specs)
    with pytest.raises(ValueError, match="must follow"):
        fp8_expert_layout(TensorLayout({n: lay.specs[n] for n in names[:3] + [names[4], names[3], names[5]]}))
    with pytest.raises(ValueError, match="inconsistent"):
        fp8_expert_layout(TensorLayout({**lay.specs, "up_proj": ((128, 256), torch.float8_e4m3fn)}))


def test_host_tensors_are_refused():
    w, s = synth.make_fp8(np.random.default_rng(0), 16, 32)
    for f in (lambda: ops.fp8_quantize(torch.zeros(1, 32)), lambda: ops.fp8_linear(torch.zeros(1, 32), w, s),
              lambda: ops.fp8_matmul(w, s, w, s)):
        with pytest.raises(RuntimeError, match="must be on CUDA"):
            f()


def test_make_fp8():
    w, s = synth.make_fp8(np.random.default_rng(0), 200, 272)
    v = ref.weight(w, s)
    assert w.dtype == torch.float8_e4m3fn and s.shape == (2, 3) and abs(float(v.std()) - 0.03) < 2e-3
    assert w.float().abs().max() == 448


def _save(path, rng, layers, E, H, I, drop=None, dtype=torch.float32):
    from safetensors.torch import save_file

    out, want = {}, {}
    for li in layers:
        for e in range(E):
            want[li, e] = synth.make_fp8_expert(rng, H, I)
            for n, t in want[li, e].items():
                key = n.replace("_scale_inv", ".weight_scale_inv") if n.endswith("_scale_inv") else n + ".weight"
                out[f"model.layers.{li}.mlp.experts.{e}.{key}"] = t.to(dtype) if n.endswith("_scale_inv") else t
    if drop:
        del out[drop]
    save_file(out, str(path / "model.safetensors"))
    return want


def test_store_from_checkpoint(tmp_path):
    H, I, E = 160, 96, 3
    want = _save(tmp_path, np.random.default_rng(1), (1, 4), E, H, I)
    st, n = ExpertStore.from_safetensors(str(tmp_path))
    lay = synth.fp8_layout(H, I)
    assert n == E and st.layer_indices == [1, 4] and st.expert_bytes == lay.total_bytes and st.layout.offsets == lay.offsets
    buf = st.allocate_buffer("cpu")
    for s, li in enumerate((1, 4)):
        for e in range(E):
            st.copy_to_buffer(buf, s, e)
            for name, t in want[li, e].items():
                assert torch.equal(buf.get_tensor(name).float(), t.float())
    assert st.expert_layout().format == _lib.EXPERT_FP8
    with pytest.raises(ValueError, match="tiled"):
        ExpertStore.from_safetensors(str(tmp_path), tiled=True)


def test_store_incomplete(tmp_path):
    _save(tmp_path, np.random.default_rng(1), (0,), 2, 64, 32, drop="model.layers.0.mlp.experts.1.up_proj.weight")
    with pytest.raises(ValueError, match="missing"):
        ExpertStore.from_safetensors(str(tmp_path))


def test_replace_linear():
    model = nn.Sequential(nn.Linear(32, 48), nn.Sequential(nn.Linear(48, 16, bias=False)), nn.ReLU())
    w = {n: synth.make_fp8(np.random.default_rng(0), *s) for n, s in (("0", (48, 32)), ("1.0", (16, 48)), ("2", (4, 16)), ("9.x", (4, 16)))}
    assert replace_linear_with_fp8(model, w, device="cpu") == 2
    assert isinstance(model[0], FP8Linear) and model[0].bias is not None and model[1][0].bias is None
    assert model[1][0].weight_scale_inv.shape == (1, 1)
    with pytest.raises(ValueError, match="weight_scale_inv"):
        FP8Linear(w["0"][0], torch.zeros(2, 1), device="cpu")
    with pytest.raises(ValueError, match="multiple of 16"):
        FP8Linear(torch.zeros(4, 24, dtype=torch.float8_e4m3fn), torch.zeros(1, 1), device="cpu")
    with pytest.raises(ValueError, match="float8_e4m3fn"):
        FP8Linear(torch.zeros(4, 32), torch.zeros(1, 1), device="cpu")


@pytest.mark.parametrize("cast", [lambda m: m.to(torch.bfloat16), lambda m: m.half(), lambda m: m.double(), lambda m: m.type(torch.float16),
                                  lambda m: m.to("cpu", torch.float16), lambda m: m.float()])
def test_casts_keep_the_format(cast):
    """A model cast to another type keeps its FP8 weights and their scales; biases and the rest change."""
    from tinyserve_amd.expert_forward import FP8ExpertModule

    w, s = synth.make_fp8(np.random.default_rng(0), 160, 144)
    model = nn.Sequential(FP8Linear(w, s, torch.randn(160), device="cpu"), nn.Linear(4, 4))
    lin = cast(model)[0]
    assert lin.weight.dtype == torch.float8_e4m3fn and torch.equal(lin.weight.view(torch.uint8), w.view(torch.uint8))
    assert lin.weight_scale_inv.dtype == torch.float32 and torch.equal(lin.weight_scale_inv, s)
    assert lin.bias.dtype == model[1].weight.dtype and not lin.weight.requires_grad
    assert set(dict(lin.named_parameters())) == {"weight", "weight_scale_inv", "bias"}
    lay = synth.fp8_layout(128, 96)
    mod = cast(FP8ExpertModule(lay, device="cpu"))
    assert {n: p.dtype for n, p in mod.named_parameters()} == {n: d for n, (_, d) in lay.specs.items()}


def test_module_moves_and_loads():
    w, s = synth.make_fp8(np.random.default_rng(0), 32, 48)
    lin = FP8Linear(w, s, device="cpu")
    other = FP8Linear(w, s, device="cpu").to("meta")
    assert other.weight.is_meta and other.weight.dtype == torch.float8_e4m3fn and other.weight_scale_inv.is_meta
    other = other.to_empty(device="cpu")
    other.load_state_dict(lin.state_dict())
    assert torch.equal(other.weight.view(torch.uint8), w.view(torch.uint8)) and torch.equal(other.weight_scale_inv, s)


@pytest.mark.parametrize("H,I,k,E", [(2048, 768, 8, 128), (2880, 2880, 4, 32), (64, 16384, 16, 20)])
def test_prompt_workspace(lib, H, I, k, E):
    """The workspace of a prompt stops growing where it is worked through in pieces (131072 assignments), and a
    workspace for more tokens serves fewer."""
    L, n, got = fp8_expert_layout(synth.fp8_layout(H, I)), ctypes.c_int64(), []
    for T in (1, 2, 4, 5, 6, 64, 1024, 131072 // k, 131072, 1 << 20, 1 << 24):
        assert lib.tsa_moe_prefill_workspace_size(ctypes.byref(L), T, k, E, ctypes.byref(n)) == 0
        got.append(n.value)
    assert got == sorted(got) and got[7] == got[-1]
    assert got[-1] < 131072 * (5 * H + 2 * I) + (1 << 20)


@pytest.mark.parametrize("E,H,I", [(3, 64, 32), (1, 64, 32), (2, 32, 64), (2, 64, 64)])
def test_store_layers_differ(tmp_path, E, H, I):
    """A layer with more or fewer experts than the first, or others' sizes, is refused (its rest was dropped)."""
    from safetensors.torch import load_file, save_file

    (tmp_path / "b").mkdir()
    _save(tmp_path, np.random.default_rng(1), (0,), 2, 64, 32)
    _save(tmp_path / "b", np.random.default_rng(2), (1,), E, H, I)
    both = {**load_file(str(tmp_path / "model.safetensors")), **load_file(str(tmp_path / "b" / "model.safetensors"))}
    save_file(both, str(tmp_path / "model.safetensors"))
    with pytest.raises(ValueError, match="layer 1"):
        ExpertStore.from_safetensors(str(tmp_path))
