"""FP8 quantisation, products and MoE layers against their definition in 64 bits (fp8_ref)."""
from __future__ import annotations

import pytest
import torch

from tests import fp8_ref as ref
from tinyserve_amd import ops, synth
from tinyserve_amd.expert_forward import fp8_expert_layout

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def acts(seed, *shape, dtype=BF):
    g = gen(seed)
    x = torch.randn(shape, device=DEV, generator=g)
    x *= torch.where(torch.rand(shape[-1], device=DEV, generator=g) < 1 / 64, 8.0, 1.0)
    return x.to(dtype)


def weights(seed, N, K):
    """A matrix of N(0, 0.03) with its blocks' largest value at 448, as checkpoints have them."""
    w = torch.zeros((ref.blocks(N) * 128, ref.blocks(K) * 128), device=DEV)
    w[:N, :K] = 0.03 * torch.randn((N, K), device=DEV, generator=gen(seed))
    b = w.view(ref.blocks(N), 128, ref.blocks(K), 128)
    s = b.abs().amax((1, 3)) / 448
    return (b / s[:, None, :, None]).view_as(w)[:N, :K].to(torch.float8_e4m3fn).contiguous(), s


def same(a, b):
    """Equal numbers, NaN where NaN."""
    a, b = a.double(), b.double()
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a.nan_to_num(), b.nan_to_num())


# ----------------------------------------------------------------------------- quantisation
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("T,K", [(1, 16), (1, 2880), (3, 128), (24, 2880), (7, 200), (5, 1), (2, 131), (257, 2048)])
def test_quantize(T, K, dtype):
    x = acts(T + K, T, K, dtype=dtype)
    c, s = ops.fp8_quantize(x)
    q64, s64 = ref.quantize(x.double())
    assert c.shape == (T, K) and s.shape == (T, ref.blocks(K)) and c.dtype == torch.float8_e4m3fn
    assert torch.equal(s.double(), s64) and torch.equal(c.double(), q64)


def test_quantize_ties():
    """Quotients that are borders between codes, to the even one: maximum 448 makes the scale 1."""
    v = torch.arange(-447, 448, device=DEV).float() / 16
    x = torch.cat([v, torch.zeros(-len(v) % 127, device=DEV)]).view(-1, 127)
    x = torch.cat([torch.full((len(x), 1), 448.0, device=DEV), x], 1)
    for dtype in (F32, HF, BF):
        y = x.to(dtype)
        c, s = ops.fp8_quantize(y)
        assert torch.equal(s, torch.ones_like(s)) and torch.equal(c.double(), ref.e4m3(y.double()))


def test_quantize_small_and_large():
    """Zeros, numbers near the smallest float32 and large ones, groups beside each other (the steps of
    row 2's linspace overflow: it holds infinities and NaN)."""
    x = torch.zeros((6, 384), device=DEV)
    x[1, 128:256] = torch.linspace(-1e-38, 1e-38, 128, device=DEV)
    x[2, :128] = torch.linspace(-3e38, 3e38, 128, device=DEV)
    x[3, 256:] = 1e-42
    x[4, ::3] = 2.0**-120
    x[5] = torch.linspace(1e-30, 1e30, 384, device=DEV)
    for v in (x, x.to(BF)):
        c, s = ops.fp8_quantize(v)
        q64, s64 = ref.quantize(v.double())
        assert same(s, s64) and same(c, q64)


def test_quantize_largest():
    """Numbers up to the largest float32."""
    x = torch.linspace(0.5, 1.0, 256, device=DEV).view(2, 128) * torch.finfo(F32).max
    for v in (x, -x, (x / 2).to(BF)):
        c, s = ops.fp8_quantize(v)
        q64, s64 = ref.quantize(v.double())
        assert same(s, s64) and same(c, q64)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_quantize_not_finite(dtype):
    """A NaN or an infinity takes its own group of its own token, and the product's row, no other."""
    x = acts(3, 4, 256, dtype=dtype)
    x[1, 5], x[2, 200] = float("nan"), float("inf")
    c, s = ops.fp8_quantize(x)
    d = c.float() * ref.spread(s, 256)
    want = torch.zeros((4, 256), dtype=torch.bool, device=DEV)
    want[1, :128] = want[2, 128:] = True
    assert torch.equal(torch.isnan(d), want)
    w, ws = weights(1, 48, 256)
    for y in (ops.fp8_matmul(c, s, w, ws), ops.fp8_linear(x, w, ws)):
        assert torch.isnan(y[1:3]).all() and torch.isfinite(y[0]).all() and torch.isfinite(y[3]).all()


def test_quantize_views():
    """Rows of a wider tensor, a start off the 16-byte boundary, leading dimensions, no token."""
    x = acts(5, 6, 400)
    for v in (x[:, 3:259], x.view(2, 3, 400)[..., :144], x.view(-1)[1 : 1 + 5 * 160].view(5, 160)):
        c, s = ops.fp8_quantize(v)
        c2, s2 = ops.fp8_quantize(v.reshape(-1, v.shape[-1]).clone())
        assert torch.equal(c.view(torch.uint8), c2.view(torch.uint8)) and torch.equal(s, s2)
    c, s = ops.fp8_quantize(x[:0])
    assert c.shape == (0, 400) and s.shape == (0, 4)


# ----------------------------------------------------------------------------- products
SHAPES = [(1, 16, 16), (1, 2880, 2880), (3, 129, 144), (16, 96, 2048), (17, 200, 272), (5, 1, 128), (24, 257, 4096),
          (33, 512, 16), (64, 300, 640), (77, 640, 2880), (129, 255, 1040), (200, 1000, 512), (513, 384, 384)]


@pytest.mark.parametrize("T,N,K", SHAPES)
@pytest.mark.parametrize("dtype,bias", [(BF, None), (F32, BF), (HF, F32)])
def test_matmul(T, N, K, dtype, bias):
    x, (w, ws) = acts(T + K, T, K), weights(N + K, N, K)
    b = None if bias is None else torch.randn(N, device=DEV, generator=gen(9)).to(bias)
    c, s = ops.fp8_quantize(x)
    y = ops.fp8_matmul(c, s, w, ws, b, out_dtype=dtype)
    want, err = ref.matmul(*ref.quantize(x.double()), w, ws, wide=dtype == F32)
    if b is not None:
        want, err = want + b.double(), err + b.double().abs() * 2.0**-23 + want.abs() * 2.0**-23
    ref.check(y, want, err)


@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 40, 300])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_linear(T, dtype):
    """One call from values is the quantisation and the product in two, for any number of tokens."""
    N, K = 272, 1424
    x, (w, ws) = acts(T, T, K, dtype=dtype), weights(2, N, K)
    b = torch.randn(N, device=DEV, generator=gen(1)).to(dtype)
    y = ops.fp8_linear(x, w, ws, b)
    want, err = ref.matmul(*ref.quantize(x.double()), w, ws, wide=dtype == F32)
    ref.check(y, want + b.double(), err + (b.double().abs() + want.abs()) * 2.0**-23)


def test_linear_scales_differ():
    """Scales of neighbouring blocks and tokens that differ by powers of ten: each meets its own block."""
    T, N, K = 40, 400, 656
    x = acts(1, T, K) * (10.0 ** torch.randint(-6, 7, (T, ref.blocks(K)), device=DEV, generator=gen(2))).repeat_interleave(128, 1)[:, :K].to(BF)
    w, ws = weights(3, N, K)
    ws = ws * 10.0 ** torch.randint(-6, 7, ws.shape, device=DEV, generator=gen(4))
    for T2 in (1, 16, T):
        y = ops.fp8_linear(x[:T2], w, ws, out_dtype=F32)
        ref.check(y, *ref.matmul(*ref.quantize(x[:T2].double()), w, ws, wide=True))


def test_linear_one_nan_weight():
    """A NaN code in a weight row makes that output NaN for every token and leaves the others."""
    x, (w, ws) = acts(1, 20, 256), weights(2, 160, 256)
    w.view(torch.uint8)[70, 100] = 0x7F
    for T in (1, 20):
        y = ops.fp8_linear(x[:T], w, ws)
        assert torch.isnan(y[:, 70]).all() and int(torch.isnan(y).sum()) == T


def test_linear_tokens_apart():
    """A token's result does not depend on the tokens beside it in kernels of one kind."""
    x, (w, ws) = acts(1, 16, 512), weights(2, 208, 512)
    y = ops.fp8_linear(x, w, ws)
    assert all(torch.equal(ops.fp8_linear(x[t : t + 1], w, ws), y[t : t + 1]) for t in range(16))


def test_linear_views():
    x, (w, ws) = acts(1, 20, 800), weights(2, 96, 400)
    want = ops.fp8_linear(x[:, 3:403].clone(), w, ws)
    assert torch.equal(ops.fp8_linear(x[:, 3:403], w, ws), want)
    assert torch.equal(ops.fp8_linear(x[:, 3:403].unflatten(0, (4, 5)), w, ws), want)
    off = torch.empty(w.numel() + 1, dtype=torch.uint8, device=DEV)[1:].view(96, 400)
    off.copy_(w.view(torch.uint8))
    wide = torch.zeros((4, 8), device=DEV)
    wide[:1, ::2] = ws
    assert torch.equal(ops.fp8_linear(x[:, 3:403], off, wide[:1, ::2]), want)
    assert ops.fp8_linear(x[:0, :400], w, ws).shape == (0, 96)


def test_linear_past_two_gib():
    """Offsets past 31 bits: a weight of more than 2 GiB, and more than 2 GiB of results."""
    N, K = 140000, 16384
    w = torch.randint(0, 0x60, (N, K), dtype=torch.uint8, device=DEV, generator=gen(1))
    ws = torch.rand((ref.blocks(N), 128), device=DEV, generator=gen(2)) * 1e-3
    rows = torch.tensor([0, 1, 131071, 131072, 139998, 139999], device=DEV)
    for T in (1, 40):
        x = acts(3, T, K)
        y = ops.fp8_linear(x, w, ws, out_dtype=F32)
        W = (w[rows].view(torch.float8_e4m3fn).double() * ref.spread(ws.double()[rows // 128], K))
        q, s = ref.quantize(x.double())
        q = q * ref.spread(s, K)
        ref.check(y[:, rows], q @ W.t(), (q.abs() @ W.abs().t()) * ref.unit(K))
    del w
    T, N, K = 9000, 131072, 16
    x, (w, ws) = acts(4, T, K), weights(5, N, K)
    y = ops.fp8_linear(x, w, ws)
    want, err = ref.matmul(*ref.quantize(x[-300:].double()), w[-512:], ws[-4:])
    ref.check(y[-300:, -512:], want, err)


# ----------------------------------------------------------------------------- MoE layers
def experts(seed, E, H, I):
    out = []
    for e in range(E):
        d = {}
        for i, (n, r, c) in enumerate((("gate_proj", I, H), ("up_proj", I, H), ("down_proj", H, I))):
            d[n], d[n + "_scale_inv"] = weights(seed + 10 * e + i, r, c)
        out.append(d)
    return out


def pool_of(ex, H, I, slots=None):
    lay = synth.fp8_layout(H, I)
    slots = list(range(len(ex))) if slots is None else slots
    pool = torch.zeros((max(slots) + 1, lay.total_bytes), dtype=torch.uint8, device=DEV)
    for e, sl in zip(ex, slots):
        for n, t in e.items():
            o = lay.offsets[n]
            pool[sl, o : o + lay.sizes[n]] = t.reshape(-1).view(torch.uint8)
    return fp8_expert_layout(lay), pool


def routes(seed, T, E, k):
    lg = torch.randn((T, E), device=DEV, generator=gen(seed))
    idx, w = ops.route_topk(lg, k)
    return lg, idx, w


LAYERS = [(4, 2, 64, 32), (8, 4, 256, 384), (5, 3, 1440, 736), (16, 8, 512, 160), (3, 1, 2880, 2880)]


@pytest.mark.parametrize("E,k,H,I", LAYERS)
@pytest.mark.parametrize("T", [1, 3, 8, 33])
def test_moe(E, k, H, I, T):
    """The same layer through the decode call, the routed one and the prompts' one."""
    ex = experts(1, E, H, I)
    L, pool = pool_of(ex, H, I)
    x, (lg, idx, w) = acts(T, T, H), routes(T, T, E, k)
    slot = torch.arange(E, dtype=torch.int32, device=DEV)
    want, err = ref.moe(x, idx, w, ex)
    ref.check(ops.moe_decode(L, pool, idx, w, x), want, err, "decode")
    y, i2, w2 = ops.moe_decode_routed(L, pool, slot, lg, x, k, return_routing=True)
    assert torch.equal(i2, idx)
    ref.check(y, want, err + want.abs() * 2.0**-20 * k, "routed")
    ref.check(ops.moe_prefill(L, pool, slot, idx, w, x), want, err, "prefill")


@pytest.mark.parametrize("E,k,H,I", [(4, 2, 256, 384), (3, 1, 1440, 736), (9, 3, 544, 96)])
@pytest.mark.parametrize("T", [101, 300, 1031])
@pytest.mark.parametrize("route", ["even", "one", "skewed"])
def test_moe_many(E, k, H, I, T, route):
    """Every token tile, with loads that fill it, leave it nearly empty, or all fall on one expert."""
    ex = experts(1, E, H, I)
    L, pool = pool_of(ex, H, I)
    x, g = acts(T, T, H), gen(T)
    p = torch.ones(E, device=DEV) if route != "skewed" else 4.0 ** -torch.arange(E, device=DEV)
    idx = torch.multinomial(p.expand(T, E), k, generator=g).to(torch.int32)
    if route == "one":
        idx[:] = E - 1
    w = torch.rand((T, k), device=DEV, generator=g)
    slot = torch.arange(E, dtype=torch.int32, device=DEV)
    want, err = ref.moe(x, idx, w, ex)
    ref.check(ops.moe_prefill(L, pool, slot, idx, w, x), want, err)


@pytest.mark.parametrize("xd,yd", [(F32, F32), (HF, HF), (BF, F32), (F32, BF)])
@pytest.mark.parametrize("T", [2, 70])
def test_moe_dtypes(xd, yd, T):
    E, k, H, I = 6, 2, 288, 416
    ex = experts(3, E, H, I)
    L, pool = pool_of(ex, H, I)
    x, (_, idx, w) = acts(T, T, H, dtype=xd), routes(T, T, E, k)
    want, err = ref.moe(x, idx, w, ex)
    slot = torch.arange(E, dtype=torch.int32, device=DEV)
    ref.check(ops.moe_decode(L, pool, idx, w, x, out_dtype=yd), want, err)
    ref.check(ops.moe_prefill(L, pool, slot, idx, w, x, out_dtype=yd), want, err)


@pytest.mark.parametrize("T", [1, 4, 90])
def test_moe_missing_and_moved(T):
    """Experts in other slots, some not resident; tokens all of whose experts are missing give zeros."""
    E, k, H, I = 6, 2, 256, 128
    ex = experts(3, E, H, I)
    order = [7, 2, 9, 0, 5, 3]
    L, pool = pool_of(ex, H, I, order)
    slot = torch.tensor([7, -1, 9, 0, -1, 99], dtype=torch.int32, device=DEV)  # 99: past the pool
    left = [ex[0], None, ex[2], ex[3], None, None]
    x, (lg, idx, w) = acts(T, T, H), routes(T, T, E, k)
    idx[0] = torch.tensor([1, 4], device=DEV)
    want, err = ref.moe(x, idx, w, left)
    y = ops.moe_prefill(L, pool, slot, idx, w, x)
    ref.check(y, want, err)
    assert not y[0].any()
    y = ops.moe_decode(L, pool, slot[idx.long()], w, x)
    ref.check(y, want, err)
    _, idx, w = routes(T, T, E, k)
    want, err = ref.moe(x, idx, w, left)
    ref.check(ops.moe_decode_routed(L, pool, slot, lg, x, k), want, err + want.abs() * 2.0**-20 * k + err * 2.0**-18)


def test_moe_swiglu_limits():
    E, k, H, I, T = 4, 2, 256, 256, 5
    ex = experts(3, E, H, I)
    for e in ex:  # gates and ups past the limits of 7
        e["gate_proj_scale_inv"] *= 8
        e["up_proj_scale_inv"] *= 8
    L, pool = pool_of(ex, H, I)
    from tinyserve_amd import _lib

    L.act = _lib.ACT_SWIGLU_OAI
    x, (_, idx, w) = acts(T, T, H), routes(T, T, E, k)
    want, err = ref.moe(x, idx, w, ex, act="swiglu")
    ref.check(ops.moe_decode(L, pool, idx, w, x), want, err)


@pytest.mark.parametrize("T", [1, 50])
def test_moe_same_expert_twice(T):
    """A token that names one expert twice counts it twice."""
    E, k, H, I = 3, 2, 128, 256
    ex = experts(1, E, H, I)
    L, pool = pool_of(ex, H, I)
    x, (_, idx, w) = acts(T, T, H), routes(T, T, E, k)
    idx[:] = 2
    want, err = ref.moe(x, idx, w, ex)
    slot = torch.arange(E, dtype=torch.int32, device=DEV)
    ref.check(ops.moe_decode(L, pool, idx, w, x), want, err)
    ref.check(ops.moe_prefill(L, pool, slot, idx, w, x), want, err)


@pytest.mark.parametrize("T", [1, 6, 80])
def test_moe_nan_token(T):
    """A token with a NaN comes out NaN, the others as without it."""
    E, k, H, I = 4, 2, 256, 160
    ex = experts(1, E, H, I)
    L, pool = pool_of(ex, H, I)
    x, (_, idx, w) = acts(T, T, H), routes(T, T, E, k)
    slot = torch.arange(E, dtype=torch.int32, device=DEV)
    for f in (lambda v: ops.moe_decode(L, pool, idx, w, v), lambda v: ops.moe_prefill(L, pool, slot, idx, w, v)):
        y = f(x)
        bad = x.clone()
        bad[T // 2, 7] = float("nan")
        z = f(bad)
        keep = torch.arange(T, device=DEV) != T // 2
        assert torch.isnan(z[T // 2]).all() and torch.equal(z[keep], y[keep])


def test_moe_captured():
    """A decode step captured once and replayed with other inputs, eager work in between."""
    E, k, H, I, T = 8, 2, 512, 256, 2
    ex = experts(1, E, H, I)
    L, pool = pool_of(ex, H, I)
    slot = torch.arange(E, dtype=torch.int32, device=DEV)
    x, lg = acts(0, T, H), torch.randn((T, E), device=DEV, generator=gen(0))
    ws, y = ops.moe_decode_workspace(L, T, k, DEV), torch.empty((T, H), dtype=BF, device=DEV)
    ws.fill_(255)
    step = lambda: ops.moe_decode_routed(L, pool, slot, lg, x, k, out=y, workspace=ws)  # noqa: E731
    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for i in range(4):
        x.copy_(acts(20 + i, T, H))
        lg.copy_(torch.randn((T, E), device=DEV, generator=gen(30 + i)))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ops.moe_decode_routed(L, pool, slot, lg, x, k))


def test_chain_other_stream():
    """Quantise once, three projections, router, experts: on a stream of its own, equal to one by one."""
    T, H, I, E, k = 20, 512, 256, 8, 2
    x, ex = acts(1, T, H), experts(1, E, H, I)
    L, pool = pool_of(ex, H, I)
    slot = torch.arange(E, dtype=torch.int32, device=DEV)
    ws = [weights(i, n, H) for i, n in enumerate((512, 128, 128))]
    wo = weights(7, H, 512)
    wr = torch.randn((E, H), device=DEV, generator=gen(3)).to(BF)

    def chain():
        c, s = ops.fp8_quantize(x)
        q, k_, v = (ops.fp8_matmul(c, s, *w) for w in ws)
        h = x + ops.fp8_linear(q, *wo)
        idx, wt = ops.route_topk(ops.router_logits(h, wr), k)
        return q, k_, v, ops.moe_prefill(L, pool, slot, idx, wt, h)

    want = chain()
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        got = chain()
    st.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ----------------------------------------------------------------------------- refusals, modules, the pipeline
def test_refusals():
    x, (w, ws) = acts(1, 4, 256), weights(2, 160, 256)
    c, s = ops.fp8_quantize(x)
    for f, text in ((lambda: ops.fp8_linear(x, w, ws[:1]), "weight scales must be"),
                    (lambda: ops.fp8_linear(x[:, :128], w, ws), "in_features differ"),
                    (lambda: ops.fp8_linear(x, w.float(), ws), "must be float8_e4m3fn"),
                    (lambda: ops.fp8_linear(x, w, ws, torch.zeros(3, device=DEV)), "bias must have"),
                    (lambda: ops.fp8_linear(x, w.cpu(), ws), "must be on CUDA"),
                    (lambda: ops.fp8_linear(x[:, :136], w[:, :136], ws), "multiple of 16"),
                    (lambda: ops.fp8_matmul(c, s[:, :1], w, ws), "activation scales must be"),
                    (lambda: ops.fp8_matmul(x, s, w, ws), "activations must be float8_e4m3fn"),
                    (lambda: ops.fp8_matmul(c, s, w, ws.cpu()), "must be on CUDA")):
        with pytest.raises(RuntimeError, match=text):
            f()
    with pytest.raises(TypeError, match="unsupported dtype"):
        ops.fp8_quantize(x.double())


@pytest.mark.parametrize("T", [2, 9])
def test_moe_long_rows(T):
    """The longest rows: hidden past what a workgroup holds of x at once, inter past what it stages of h."""
    for E, k, H, I in ((5, 5, 64, 16384), (3, 2, 16384, 64)):
        ex = experts(1, E, H, I)
        L, pool = pool_of(ex, H, I)
        x, (_, idx, w) = acts(T, T, H), routes(T, T, E, k)
        want, err = ref.moe(x, idx, w, ex)
        ref.check(ops.moe_decode(L, pool, idx, w, x), want, err)


def test_moe_routed_without_workspace_and_many_experts():
    """The allocation-free call, and more experts than the in-kernel routing takes."""
    from tinyserve_amd import _lib
    import ctypes

    for E, k, T in ((7, 3, 2), (300, 4, 3)):
        H, I = 128, 64
        ex = experts(1, 7, H, I)
        L, pool = pool_of(ex, H, I)
        slot = (torch.arange(E, device=DEV) % 7).to(torch.int32)
        x, (lg, idx, w) = acts(T, T, H), routes(T, T, E, k)
        want, err = ref.moe(x, slot[idx.long()], w, ex)
        err = err + want.abs() * 2.0**-20 * k + err * 2.0**-18
        ref.check(ops.moe_decode_routed(L, pool, slot, lg, x, k), want, err)
        y = torch.empty((T, H), dtype=BF, device=DEV)
        _lib.check(_lib.load().tsa_moe_decode_routed_noalloc(
            ctypes.byref(L), pool.data_ptr(), 7, slot.data_ptr(), E, lg.data_ptr(), 0, 0, T, k, x.data_ptr(), 2, y.data_ptr(), 2,
            None, None, torch.cuda.current_stream().cuda_stream))
        ref.check(y, want, err)


def test_modules_and_builders():
    """FP8Linear, the template expert and the inline forward give the operators' results."""
    from tinyserve_amd.expert_forward import (FP8ExpertModule, _build_cpp_layout_args, _build_fp8_inline_forward,
                                              _precompute_param_refs, fast_expert_forward, forward_from_packed)
    from tinyserve_amd.fp8 import FP8Linear

    w, ws = weights(1, 96, 144)
    b = torch.randn(96, device=DEV).to(BF)
    x = acts(2, 2, 3, 144)
    y = FP8Linear(w, ws, b)(x)
    assert y.shape == (2, 3, 96) and torch.equal(y.view(6, 96), ops.fp8_linear(x.view(6, 144), w, ws, b))
    H, I = 256, 160
    ex = experts(3, 1, H, I)
    L, pool = pool_of(ex, H, I)
    lay = synth.fp8_layout(H, I)
    mod = FP8ExpertModule(lay, device=DEV)
    for T in (1, 5, 40):
        h = acts(T, T, H)
        zero, one = torch.zeros((T, 1), dtype=torch.int32, device=DEV), torch.ones((T, 1), device=DEV)
        want, err = ref.moe(h, zero, one, ex)
        ref.check(forward_from_packed(mod, pool[0], _precompute_param_refs(mod, lay), h), want, err)
        ref.check(_build_fp8_inline_forward(lay, None)(pool[0], h), want, err)
        ref.check(fast_expert_forward(h, zero, one, pool, **_build_cpp_layout_args(lay, None)), want, err)


@pytest.mark.parametrize("T", [1, 3, 40])
def test_pipeline_and_hook(tmp_path, T):
    """A checkpoint on disk through the store, the pipeline and an installed MoE block."""
    import numpy as np
    import torch.nn as nn

    from tests.test_fp8_host import _save
    from tinyserve_amd.expert_batcher import BatchItem, ExpertBatcher
    from tinyserve_amd.expert_pipeline import ExpertPipeline, install_offloaded_forward
    from tinyserve_amd.expert_store import ExpertStore

    E, k, H, I = 6, 2, 160, 96
    disk = _save(tmp_path, np.random.default_rng(5), (0, 1), E, H, I)
    store, _ = ExpertStore.from_safetensors(str(tmp_path))
    pipe = ExpertPipeline(store, None, DEV)
    for layer in (0, 1):
        ex = [{n: t.to(DEV) for n, t in disk[layer, e].items()} for e in range(E)]
        x, (lg, idx, w) = acts(T, T, H), routes(T + layer, T, E, k)
        want, err = ref.moe(x, idx, w, ex)
        ref.check(pipe.execute_layer_experts(x, layer, idx, w), want, err)
        ref.check(pipe.execute_layer_experts_batched(x, layer, idx, w), want, err)
        ref.check(pipe.execute_layer_logits(x, layer, lg, k), want, err + want.abs() * 2.0**-20 * k + err * 2.0**-18)
        got = ExpertBatcher(pipe).batch_execute([BatchItem(x[t : t + 1], idx[t], w[t], t) for t in range(T)], layer)
        ref.check(torch.cat(got), want, err)

        class Block(nn.Module):
            def __init__(self):
                super().__init__()
                self.gate = nn.Linear(H, E, bias=False).to(DEV, BF)

        block = Block()
        install_offloaded_forward(block, pipe, layer, "gate", k)
        y = block.forward(x.view(1, T, H))
        idx2, w2 = ops.route_topk(ops.router_logits(x, block.gate.weight), k)
        w2 = w2 if T <= 4 else w2.to(BF).float()
        want, err = ref.moe(x, idx2, w2, ex)
        ref.check(y.view(T, H), want, err + want.abs() * 2.0**-20 * k + err * 2.0**-18)


def test_moe_prompt_in_pieces():
    """More assignments than the grouped kernels take at a time."""
    E, k, H, I, T = 5, 2, 64, 32, 70000
    ex = experts(1, E, H, I)
    L, pool = pool_of(ex, H, I)
    x, (_, idx, w) = acts(T, T, H), routes(T, T, E, k)
    want, err = ref.moe(x, idx, w, ex)
    ref.check(ops.moe_prefill(L, pool, torch.arange(E, dtype=torch.int32, device=DEV), idx, w, x), want, err)


def test_moe_nothing_resident():
    E, k, H, I, T = 4, 2, 96, 64, 9
    L, pool = pool_of(experts(1, E, H, I), H, I)
    x, (_, idx, w) = acts(T, T, H), routes(T, T, E, k)
    slot = torch.full((E,), -1, dtype=torch.int32, device=DEV)
    for n in (1, T):
        assert not ops.moe_prefill(L, pool, slot, idx[:n], w[:n], x[:n]).any()
        assert not ops.moe_decode(L, pool, slot[idx[:n].long()], w[:n], x[:n]).any()


def test_linear_longest_rows():
    """K past what one launch stages, more than 64 blocks."""
    K, N = 131072, 48
    w, ws = weights(1, N, K)
    for T in (2, 40):
        x = acts(T, T, K)
        ref.check(ops.fp8_linear(x, w, ws), *ref.matmul(*ref.quantize(x.double()), w, ws))


def test_prompt_captured():
    """A quantisation, products and a layer of a prompt in one graph, replayed with other inputs; two
    graphs' results do not disturb each other."""
    E, k, H, I, T = 8, 2, 256, 160, 40
    ex = experts(1, E, H, I)
    L, pool = pool_of(ex, H, I)
    slot = torch.arange(E, dtype=torch.int32, device=DEV)
    wq, wo = weights(3, 320, H), weights(4, H, 320)
    xs = [acts(i, T, H) for i in range(2)]
    lg = [torch.randn((T, E), device=DEV, generator=gen(i)) for i in range(2)]

    def step(i):
        c, s = ops.fp8_quantize(xs[i])
        h = ops.fp8_linear(ops.fp8_matmul(c, s, *wq), *wo)
        idx, w = ops.route_topk(lg[i], k)
        return ops.moe_prefill(L, pool, slot, idx, w, h)

    step(0)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(i))
        graphs.append(g)
    for r in range(4):
        for i in range(2):
            xs[i].copy_(acts(50 + 2 * r + i, T, H))
            lg[i].copy_(torch.randn((T, E), device=DEV, generator=gen(70 + 2 * r + i)))
        for g in graphs:
            g.replay()
        want = [step(i) for i in range(2)]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.parametrize("T,N,K", [(33, 1, 16), (40, 3, 32), (65, 2, 144)])
def test_matmul_smallest_buffers(T, N, K):
    """Weights of fewer bytes than the pipeline's blocks ahead of the last."""
    x, (w, ws) = acts(T, T, K), weights(N, N, K)
    ref.check(ops.fp8_linear(x, w, ws), *ref.matmul(*ref.quantize(x.double()), w, ws))


@pytest.mark.parametrize("T", [2, 12])
def test_moe_dead_expert_any_weight(T):
    """The weight of an expert that is not resident is not used: NaN there changes nothing."""
    E, k, H, I = 4, 3, 128, 96
    L, pool = pool_of(experts(1, E, H, I), H, I)
    x, (_, idx, w) = acts(T, T, H), routes(T, T, E, k)
    slot = torch.tensor([0, -1, 2, 3], dtype=torch.int32, device=DEV)
    bad = torch.where(idx == 1, float("nan"), w)
    for f in (lambda v: ops.moe_decode(L, pool, slot[idx.long()], v, x), lambda v: ops.moe_prefill(L, pool, slot, idx, v, x)):
        y = f(bad)
        assert torch.isfinite(y).all() and torch.equal(y, f(w))


@pytest.mark.parametrize("T", [4, 24, 200])
def test_moe_codes_of_h(T):
    """Few codes of h (6144 a token) fall to another side than the definition's: one that does moves a
    token's result by 0.06 / sqrt(6144) = 8e-4 of itself or more. Without one, the down product's sums are
    off by at most sqrt(7 / 3) 2^-13 of the largest of 8 products (2.5 of their rms) per sqrt(8) of it:
    1.7e-4. float32 gate and up sums leave most tokens without one, so the median is below twice that."""
    E, k, H, I = 16, 8, 512, 768
    ex = experts(1, E, H, I)
    L, pool = pool_of(ex, H, I)
    slot = torch.arange(E, dtype=torch.int32, device=DEV)
    off = []
    for seed in range(8 if T < 24 else 1):
        x, (_, idx, w) = acts(seed, T, H, dtype=torch.float32), routes(seed, T, E, k)
        y = ops.moe_prefill(L, pool, slot, idx, w, x) if T > 4 else ops.moe_decode(L, pool, slot[idx.long()], w, x)
        assert y.dtype == torch.float32
        want, _ = ref.moe(x, idx, w, ex)
        off += ((y.double() - want).norm(dim=1) / want.norm(dim=1)).tolist()
    assert sorted(off)[len(off) // 2] < 3.4e-4


@pytest.mark.parametrize("E,k,H,I", [(20, 9, 256, 160), (20, 11, 64, 96), (20, 13, 128, 128), (16, 15, 96, 288), (24, 16, 64, 64),
                                     (40, 33, 64, 32), (11, 10, 64, 6144), (13, 12, 32, 16384)])
@pytest.mark.parametrize("T", [1, 3])
def test_moe_many_experts_a_token(E, k, H, I, T):
    """Each expert's own slot, scales and weight for odd numbers of experts past 8 and for odd pieces of
    them staged at a time (inter 6144: 9 of 10; 16384: 3 of 12), together and each alone. Slot 0 holds no
    expert."""
    ex = experts(1, E, H, I)
    L, pool = pool_of(ex, H, I, list(range(E, 0, -1)))
    slot = torch.arange(E, 0, -1, dtype=torch.int32, device=DEV)
    x, (lg, idx, w) = acts(T, T, H), routes(T, T, E, k)
    want, err = ref.moe(x, idx, w, ex)
    ref.check(ops.moe_decode(L, pool, slot[idx.long()], w, x), want, err, "decode")
    ref.check(ops.moe_prefill(L, pool, slot, idx, w, x), want, err, "prefill")
    y, i2, w2 = ops.moe_decode_routed(L, pool, slot, lg, x, k, return_routing=True)
    ref.check(y, *ref.moe(x, i2, w2, ex), "routed")
    for j in range(k):
        one = torch.nn.functional.one_hot(torch.full((T,), j, device=DEV), k).float()
        ref.check(ops.moe_decode(L, pool, slot[idx.long()], one, x), *ref.moe(x, idx[:, j : j + 1], one[:, j : j + 1], ex), f"place {j}")


@pytest.mark.parametrize("I", [32, 96, 288, 544])
@pytest.mark.parametrize("T", [1, 3])
def test_moe_dead_experts_stale_workspace(I, T):
    """What the workspace holds in place of the h of an expert that is not resident (here NaN) does not
    reach the result, for widths whose last group of channels is short."""
    E, k, H = 20, 16, 64
    ex = experts(1, E, H, I)
    L, pool = pool_of(ex, H, I)
    slot = torch.arange(E, dtype=torch.int32, device=DEV)
    slot[1::2] = -1
    left = [None if e % 2 else x for e, x in enumerate(ex)]
    x, (lg, idx, w) = acts(T, T, H), routes(T, T, E, k)
    want, err = ref.moe(x, idx, w, left)
    ws = ops.moe_decode_workspace(L, T, k, DEV)
    sync = 32 << 10  # not written by these calls
    ws[sync:] = 255
    ref.check(ops.moe_decode(L, pool, slot[idx.long()], w, x, workspace=ws), want, err, "decode")
    ws[sync:] = 255
    y, i2, w2 = ops.moe_decode_routed(L, pool, slot, lg, x, k, workspace=ws, return_routing=True)
    ref.check(y, *ref.moe(x, i2, w2, left), "routed")
    for n in (T, 9):
        x, (_, idx, w) = acts(n, n, H), routes(n, n, E, k)
        wp = ops.moe_prefill_workspace(L, n, k, E, DEV).fill_(255)
        ref.check(ops.moe_prefill(L, pool, slot, idx, w, x, workspace=wp), *ref.moe(x, idx, w, left), "prefill")


def _known_h(H, I, up, up_scales):
    """An expert without down whose h is known exactly: a token of _known_x gives gate sums of 32, so that
    silu(gate) is 32 in float32, and up sums of up_scales[:, b] up[:, b] of each K block b."""
    e = {}
    for n, (r, c) in (("gate_proj", (I, H)), ("up_proj", (I, H)), ("down_proj", (H, I))):
        e[n] = torch.zeros((r, c), device=DEV)
        e[n + "_scale_inv"] = torch.ones((ref.blocks(r), ref.blocks(c)), device=DEV)
    e["gate_proj"][:, 1] = 32
    e["gate_proj_scale_inv"][:] = 2.0**-8
    e["up_proj"][:, 1::128] = up
    e["up_proj_scale_inv"][:] = up_scales * 2.0**-8
    return e


def _known_x(T, H, dtype):
    """Tokens whose scales are 1 and whose code in column 1 of each block is 256."""
    x = torch.zeros((T, H), device=DEV)
    x[:, ::128], x[:, 1::128] = 448, 256
    return x.to(dtype)


def _codes(e):
    return {n: t.to(torch.float8_e4m3fn) if not n.endswith("_scale_inv") else t for n, t in e.items()}


@pytest.mark.parametrize("T", [1, 9, 300])
@pytest.mark.parametrize("dtype", [F32, BF])
def test_moe_float32_sums(T, dtype):
    """A float32 layer result keeps what is 2^-17 of the largest product beside it: two products of 448
    that cancel, the 14 of 2^-9 around them stay. Every sum and product here is exact in float32."""
    from tinyserve_amd.expert_forward import FP8ExpertModule, _precompute_param_refs, forward_from_packed

    H, I = 128, 128
    up = torch.zeros((I, 1), device=DEV)
    up[:16] = 2.0**-9
    up[:16:8] = 448
    e = _known_h(H, I, up, torch.ones((1, 1), device=DEV))
    n = torch.arange(H, device=DEV) % 8 + 1
    e["down_proj"][:, :16] = n.unsqueeze(1).float()
    e["down_proj"][:, 0], e["down_proj"][:, 8] = 1, -1
    L, pool = pool_of([_codes(e)], H, I)
    x, want = _known_x(T, H, dtype), (32 * 14 * 2.0**-9 * n).expand(T, H).float()
    zero, one = torch.zeros((T, 1), dtype=torch.int32, device=DEV), torch.ones((T, 1), device=DEV)
    assert torch.equal(ops.moe_decode(L, pool, zero, one, x, out_dtype=F32), want)
    assert torch.equal(ops.moe_decode_routed(L, pool, zero[0], one, x, 1, out_dtype=F32), want)
    assert torch.equal(ops.moe_prefill(L, pool, zero[0], zero, one, x, out_dtype=F32), want)
    if dtype == F32:
        lay = synth.fp8_layout(H, I)
        mod = FP8ExpertModule(lay, device=DEV)
        assert torch.equal(forward_from_packed(mod, pool[0], _precompute_param_refs(mod, lay), x), want)


@pytest.mark.parametrize("value,scale", [("0x1.800002p-109", "0x1.000002p-100"), ("0x1.400004p-108", "0x1.000004p-100"),
                                         ("0x1.b80004p-104", "0x1.400002p-97"), ("0x1p-104", "0x1.fffffep-95"),
                                         ("0x1.800002p-19", "0x1.000002p-10"), ("0x1.b80004p3", "0x1.400002p10")])
@pytest.mark.parametrize("T", [1, 9, 300])
def test_moe_quotients_of_h(T, value, scale):
    """Codes of h from the correctly rounded quotient: (value, scale) pairs whose quotient rounds onto a
    border between two codes, or next to it."""
    import numpy as np

    v, s = (np.float32(float.fromhex(t)) for t in (value, scale))
    top = next(m for m in (np.float32(448 * float(s)) * np.float32(1 + d * 2.0**-23) for d in (0, 1, -1, 2, -2)) if m / np.float32(448) == s)
    H, I = 256, 128
    up = torch.zeros((I, 2), device=DEV)
    up[0, 0] = up[1, 1] = 1
    e = _known_h(H, I, up, torch.tensor([[float(top) / 32, float(v) / 32]], device=DEV))
    e["down_proj"][:, 1] = 1
    L, pool = pool_of([_codes(e)], H, I)
    code = ref.e4m3(torch.tensor(float(v / s), dtype=torch.float64))
    want = torch.full((T, H), float(code) * float(s), dtype=F32, device=DEV)
    zero, one = torch.zeros((T, 1), dtype=torch.int32, device=DEV), torch.ones((T, 1), device=DEV)
    x = _known_x(T, H, F32)
    assert torch.equal(ops.moe_decode(L, pool, zero, one, x), want)
    assert torch.equal(ops.moe_prefill(L, pool, zero[0], zero, one, x), want)


def _fma(a, b, c):
    """a b + c of float32 values (held in 64 bits) rounded once to float32: the 64-bit sum's own error moves it
    off the border that it may have been rounded onto."""
    p = a * b  # exact
    t = c + p
    big = torch.maximum(c.abs(), p.abs()) == c.abs()
    err = torch.where(big, (c - t) + p, (p - t) + c)
    return torch.where(err != 0, torch.nextafter(t, t + err.sign() * t.abs()), t).float().double()


def test_corrected_quotient_is_the_division():
    """x / s by a rounded reciprocal and one correction equals the division for every significand of s and
    the x within 3 steps of a border between two codes (normal ones: odd 16ths; subnormal ones: odd numbers)."""
    borders = [o / 16 for o in range(17, 32, 2)] + [o / 2 ** (o.bit_length() - 1) for o in range(1, 16, 2)]
    for lo in range(0, 1 << 23, 1 << 20):
        s = 1 + torch.arange(lo, lo + (1 << 20), device=DEV).double() / 2**23
        r = (1 / s).float().double()
        for b in borders:
            x0 = (b * s).float().view(torch.int32)
            for d in range(-3, 4):
                x = (x0 + d).view(torch.float32).double()
                a = (x * r).float().double()
                assert torch.equal(_fma(_fma(-a, s, x), r, a), (x / s).float().double())


@pytest.mark.parametrize("dtype,top,low", [(HF, 15, -5), (BF, 10, -10)])
def test_quantize_every_quotient(dtype, top, low):
    """All significands of a group's maximum with all significands of smaller values down to the ones
    whose code is zero: the codes are the division's."""
    bits = {HF: 10, BF: 7}[dtype]
    sig = 1 + torch.arange(2**bits, device=DEV).double() / 2**bits
    m = sig * 2.0**top
    v = torch.cat([sig * 2.0**e for e in range(low, top + 1)])
    v = torch.nn.functional.pad(v, (0, -len(v) % 127)).view(-1, 127)
    for part in m.split(64):
        x = torch.minimum(v.expand(len(part), -1, -1), part.view(-1, 1, 1))
        x = torch.cat([part.view(-1, 1, 1).expand(-1, len(v), 1), x], 2).reshape(-1, 128)
        c, s = ops.fp8_quantize(x.to(dtype))
        q64, s64 = ref.quantize(x)
        assert torch.equal(s.double(), s64) and torch.equal(c.double(), q64)


def _swiglu_layer(E, H, I):
    """Experts whose gates and ups pass the limits of 7, under the clamped activation."""
    from tinyserve_amd import _lib

    ex = experts(3, E, H, I)
    for e in ex:
        e["gate_proj_scale_inv"] *= 8
        e["up_proj_scale_inv"] *= 8
    L, pool = pool_of(ex, H, I)
    L.act = _lib.ACT_SWIGLU_OAI
    return ex, L, pool


@pytest.mark.parametrize("T", [2, 9, 300])
def test_moe_swiglu_nan_token(T):
    """The limits of the clamped activation let a NaN through: its token comes out NaN, no other changes."""
    E, k, H, I = 4, 2, 256, 160
    _, L, pool = _swiglu_layer(E, H, I)
    x, (_, idx, w) = acts(T, T, H), routes(T, T, E, k)
    slot = torch.arange(E, dtype=torch.int32, device=DEV)
    bad = x.clone()
    bad[T // 2, 7] = float("nan")
    keep = torch.arange(T, device=DEV) != T // 2
    for f in (lambda v: ops.moe_decode(L, pool, idx, w, v), lambda v: ops.moe_prefill(L, pool, slot, idx, w, v)):
        y, z = f(x), f(bad)
        assert torch.isnan(z[T // 2]).all() and torch.equal(z[keep], y[keep])


@pytest.mark.parametrize("T", [9, 60, 300])
def test_moe_swiglu_prompt(T):
    E, k, H, I = 4, 2, 256, 352
    ex, L, pool = _swiglu_layer(E, H, I)
    x, (_, idx, w) = acts(T, T, H), routes(T, T, E, k)
    want, err = ref.moe(x, idx, w, ex, act="swiglu")
    ref.check(ops.moe_prefill(L, pool, torch.arange(E, dtype=torch.int32, device=DEV), idx, w, x), want, err)


@pytest.mark.parametrize("T,K", [((1 << 28) + 5, 1), ((1 << 28) + 300, 8)])
def test_quantize_past_2_28_groups(T, K):
    """More groups than one launch has room for: every one is quantised."""
    x = acts(1, 1 << 20, K).repeat(-(-T // (1 << 20)), 1)[:T]
    c, s = ops.fp8_quantize(x)
    c1, s1 = ops.fp8_quantize(x[: 1 << 20])
    for t in range(0, T, 1 << 20):
        n = min(1 << 20, T - t)
        assert torch.equal(c[t : t + n].view(torch.uint8), c1[:n].view(torch.uint8)) and torch.equal(s[t : t + n], s1[:n])


@pytest.mark.parametrize("T,K", [(2, (1 << 31) - 1), (9, (1 << 31) - 8)])
def test_quantize_longest_rows(T, K):
    """Rows up to 2^31 values, more of them than a launch takes (8)."""
    x = torch.empty((T, K), dtype=BF, device=DEV)
    part = acts(2, 1 << 20)
    for t in range(T):
        for o in range(0, K, 1 << 20):
            x[t, o : o + (1 << 20)] = part[: min(1 << 20, K - o)]
    c, s = ops.fp8_quantize(x)
    del x
    q, qs = ops.fp8_quantize(part.unsqueeze(0))
    last = (K - 1) >> 20 << 20
    for t in range(T):
        for o in (0, 1 << 30, last - (1 << 20)):
            assert torch.equal(c[t, o : o + (1 << 20)].view(torch.uint8), q[0].view(torch.uint8))
            assert torch.equal(s[t, o // 128 : (o + (1 << 20)) // 128], qs[0])
        e, es = ops.fp8_quantize(part[: K - last].unsqueeze(0))
        assert torch.equal(c[t, last:].view(torch.uint8), e[0].view(torch.uint8)) and torch.equal(s[t, last // 128 :], es[0])


@pytest.mark.parametrize("T,dtype", [(1, F32), (17, BF), (33, BF)])
def test_matmul_past_2_27_rows(T, dtype):
    """More weight rows than one launch of the row kernel has room for (2^26 a launch), and as many in tiles."""
    N, K = (1 << 27) + 1000, 16
    g = gen(1)
    w = torch.randint(0, 0x60, (N, K), dtype=torch.uint8, device=DEV, generator=g).view(torch.float8_e4m3fn)
    ws = torch.rand((ref.blocks(N), 1), device=DEV, generator=g) * 1e-2
    b = torch.randn(N, device=DEV, generator=g).to(BF)
    x = acts(2, T, K)
    y = ops.fp8_linear(x, w, ws, b, out_dtype=dtype)
    q, s = ref.quantize(x.double())
    for n in (0, (1 << 26) - 256, (1 << 27) - 256, N // 128 * 128 - 512):
        r = slice(n, min(n + 1024, N))
        want, err = ref.matmul(q, s, w[r], ws[n // 128 :][: ref.blocks(r.stop - n)], wide=dtype == F32)
        bias = b[r].double()
        ref.check(y[:, r], want + bias, err + (bias.abs() + want.abs()) * 2.0**-23)


@pytest.mark.parametrize("T", [1, 9, 150])
def test_moe_largest_experts_past_four_gib(T):
    """The largest hidden and inter, in a pool whose last slot starts past 2^32 bytes."""
    H = I = 16384
    ex = experts(1, 1, H, I)
    L, pool = pool_of(ex, H, I, [6])
    assert 6 * pool.shape[1] > 1 << 32
    x, slot = acts(T, T, H), torch.full((1,), 6, dtype=torch.int32, device=DEV)
    zero, w = torch.zeros((T, 1), dtype=torch.int32, device=DEV), torch.rand((T, 1), device=DEV, generator=gen(T))
    want, err = ref.moe(x, zero, w, ex)
    ref.check(ops.moe_prefill(L, pool, slot, zero, w, x), want, err, "prefill")
    ref.check(ops.moe_decode(L, pool, slot[zero.long()], w, x), want, err, "decode")
