"""int8 quantisation, products and grouped products on the GPU against their definition in 64 bits
(tests/int8_ref.py), at the sizes where tiles, steps and dispatch rules end."""
from __future__ import annotations

import pytest
import torch

from tests import int8_ref as ref
from tinyserve_amd import ops

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def acts(g, *shape, dtype=torch.bfloat16):
    x = torch.randn(shape, device="cuda", generator=g)
    x[..., :: 97] *= 6
    return x.to(dtype)


def check_codes(x, codes, scales):
    q, s = ref.quantize(x)
    assert torch.equal(scales.double(), s.squeeze(1)), "scales differ"
    assert codes.dtype == torch.int8 and torch.equal(codes.double(), q), f"{int((codes.double() != q).sum())} codes differ"


# ----------------------------------------------------------------------------- quantisation
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,K", [(1, 1), (1, 8), (3, 7), (5, 512), (2, 2880), (24, 4096), (7, 4104), (3, 9001), (1023, 130), (1024, 72),
                                 (1500, 2880), (1025, 4099), (1100, 8200)])
def test_quantize(T, K, dtype):
    x = acts(gen(T + K), T, K, dtype=dtype)
    check_codes(x, *ops.int8_quantize(x))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_quantize_every_value_over_every_maximum(dtype):
    """Every positive number of the type, down to 2^-14 of the largest, over the significands of the maxima: ties between
    codes, and quotients next to them, fall as the definition's."""
    n = 128 if dtype == torch.bfloat16 else 1024
    sig = 1 + torch.arange(n, device="cuda", dtype=torch.float64) / n
    small = torch.cat([sig * 2.0**-e for e in range(1, 9)])  # below the maximum, down to codes of zero
    for top in sig.split(64):
        rows = torch.cat([top[:, None], (small[None] * 1.0).expand(len(top), -1), -(sig[None].expand(len(top), -1).minimum(top[:, None]))], 1)
        x = rows.to(dtype)
        check_codes(x, *ops.int8_quantize(x))
        check_codes(x[:, :-1].contiguous(), *ops.int8_quantize(x[:, :-1].contiguous()))


@pytest.mark.parametrize("dtype,scale", [(torch.float32, 1e-38), (torch.float32, 1e-44), (torch.float32, 3e38), (torch.bfloat16, 1e-39),
                                         (torch.bfloat16, 2.0**-90), (torch.bfloat16, 1e38), (torch.float16, 1e-7)])
def test_quantize_extremes(dtype, scale):
    x = (torch.rand((4, 264), device="cuda", generator=gen(1), dtype=torch.float64) * 2 - 1).mul(scale).to(dtype)
    x[3] = 0
    check_codes(x, *ops.int8_quantize(x))


def test_quantize_not_finite():
    """A token with a NaN or an infinity: a NaN as its scale, zeros as its codes, NaN in its outputs; others as ever."""
    x = acts(gen(2), 40, 2880)
    x[1, 7], x[5, 2879], x[39, 0] = float("nan"), float("inf"), float("-inf")
    codes, scales = ops.int8_quantize(x)
    bad = torch.zeros(40, dtype=torch.bool, device="cuda")
    bad[[1, 5, 39]] = True
    assert scales[bad].isnan().all() and not codes[bad].any()
    check_codes(x[~bad], codes[~bad], scales[~bad])
    w, ws = ref.weights8(gen(3), 48, 2880)
    for y in (ops.int8_matmul(codes, scales, w, ws), ops.int8_linear(x, w, ws), ops.int8_linear(x[:6], w, ws)):
        b = bad[: y.shape[0]]
        assert y[b].isnan().all() and y[~b].isfinite().all()


def test_quantize_strides_and_no_tokens():
    x = acts(gen(4), 6, 200)[:, 3:131]  # not contiguous, off 16 bytes
    check_codes(x.contiguous(), *ops.int8_quantize(x))
    codes, scales = ops.int8_quantize(x.new_empty((0, 64)))
    assert codes.shape == (0, 64) and scales.shape == (0,)
    y = acts(gen(5), 2, 3, 64)
    assert ops.int8_quantize(y)[0].shape == (6, 64)


# ----------------------------------------------------------------------------- products
def linear_case(T, K, N, dtype, bias, seed=0):
    g = gen(seed + T * 7 + K * 3 + N)
    w, ws = ref.weights8(g, N, K)
    return acts(g, T, K, dtype=dtype), w, ws, (torch.randn(N, device="cuda", generator=g).to(bias) if bias is not None else None)


@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 31, 32, 33, 64, 65, 100, 129, 300])
@pytest.mark.parametrize("K,N", [(16, 1), (128, 17), (144, 64), (1040, 259), (2880, 320)])
def test_linear(T, K, N):
    x, w, ws, b = linear_case(T, K, N, torch.bfloat16, torch.bfloat16 if N % 2 else None)
    want, err = ref.matmul(*ref.quantize(x), w, ws, b)
    ref.check(ops.int8_linear(x, w, ws, b), want, err, "linear")
    ref.check(ops.int8_matmul(*ops.int8_quantize(x), w, ws, b), want, err, "matmul")
    ref.check(ops.int8_linear(x, w, ws, b, out_dtype=torch.float32), want, err, "linear to float32")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bias", [None, torch.float32, torch.float16])
@pytest.mark.parametrize("T", [1, 9, 24, 200])
def test_linear_types(T, dtype, bias):
    x, w, ws, b = linear_case(T, 1552, 200, dtype, bias)
    want, err = ref.matmul(*ref.quantize(x), w, ws, b)
    for out in DTYPES:
        ref.check(ops.int8_linear(x, w, ws.unsqueeze(1), b, out_dtype=out), want, err, f"{out}")
        ref.check(ops.int8_matmul(*ops.int8_quantize(x), w, ws, b, out_dtype=out), want, err, f"{out}")


@pytest.mark.parametrize("T,N", [(1000, 2880), (777, 5760), (2048, 4104), (4096, 512), (512, 4096), (130, 6000)])
def test_linear_tiles(T, N):
    """Sizes that reach each tile of the dispatch rule, with short last tiles of either side."""
    x, w, ws, b = linear_case(T, 720, N, torch.bfloat16, torch.bfloat16)
    want, err = ref.matmul(*ref.quantize(x), w, ws, b)
    ref.check(ops.int8_linear(x, w, ws, b), want, err)


@pytest.mark.parametrize("T", [1, 20, 40])
def test_sums_are_exact(T):
    """Codes of -128 over the longest rows: sums of nearly 2^31."""
    K = 131056
    codes = torch.full((T, K), -128, dtype=torch.int8, device="cuda")
    w = torch.full((24, K), -128, dtype=torch.int8, device="cuda")
    w[1], w[2, ::2] = 127, 1
    s, ws = torch.full((T,), 2.0**-20, device="cuda"), torch.full((24,), 2.0**-10, device="cuda")
    want, err = ref.matmul(codes.double(), s.double().unsqueeze(1), w, ws)
    ref.check(ops.int8_matmul(codes, s, w, ws, out_dtype=torch.float32), want, err)


def test_linear_views_and_no_tokens():
    x, w, ws, _ = linear_case(3, 288, 64, torch.bfloat16, None)
    want, err = ref.matmul(*ref.quantize(x), w, ws)
    wide = torch.zeros((3, 300), dtype=torch.bfloat16, device="cuda")
    wide[:, 5:293] = x
    ref.check(ops.int8_linear(wide[:, 5:293], w, ws), want, err, "x off 16 bytes")
    wv = torch.zeros((64, 300), dtype=torch.int8, device="cuda")
    wv[:, 4:292] = w
    ref.check(ops.int8_linear(x, wv[:, 4:292], ws), want, err, "w off 16 bytes")
    assert ops.int8_linear(x[:0], w, ws).shape == (0, 64)
    assert ops.int8_linear(x.view(1, 3, 288), w, ws).shape == (3, 64)


# ----------------------------------------------------------------------------- grouped
def ragged(g, E: int, R: int, empty: bool = True) -> list[int]:
    """Ascending offsets with empty groups, one large one, and rows behind the last."""
    p = torch.rand(E, device="cuda", generator=g) ** 4
    if empty:
        p[:: 3] = 0
    c = torch.floor(p / p.sum() * R * 0.95).long().tolist() if float(p.sum()) > 0 else [0] * E
    out = [0]
    for n in c:
        out.append(out[-1] + n)
    return out


def grouped_case(kind, E, N, K, T, k, seed=0, bias=True):
    g = gen(seed + E + N + K + T)
    x = acts(g, T, K, dtype=torch.float16 if kind == "f16" else torch.bfloat16)
    if kind == "int8":
        w, ws = ref.weights8(g, E, N, K)
    else:
        w, ws = (0.03 * torch.randn((E, N, K), device="cuda", generator=g)).to(x.dtype), None
    b = torch.randn((E, N), device="cuda", generator=g).to(torch.bfloat16) if bias else None
    rows = torch.randperm(T * k, device="cuda", generator=g).to(torch.int32)
    return x, w, ws, b, ragged(g, E, T * k), rows


def run_grouped(x, w, ws, off, b=None, rows=None, top_k=1, out=None):
    off = torch.tensor(off, dtype=torch.int32, device="cuda")
    if ws is None:
        return ops.grouped_matmul(x, w, off, b, rows=rows, top_k=top_k, out_dtype=out)
    return ops.int8_grouped_matmul(*ops.int8_quantize(x), w, ws, off, b, rows=rows, top_k=top_k, out_dtype=out or torch.bfloat16)


def want_grouped(x, w, ws, off, b=None, rows=None, top_k=1):
    xr = x if ws is None else ref.quantize(x)
    return ref.grouped(xr, w, off, b, None if rows is None else rows.tolist(), top_k, ws)


@pytest.mark.parametrize("kind", ["bf16", "f16", "int8"])
@pytest.mark.parametrize("E,N,K,T,k", [(1, 1, 16, 1, 1), (3, 40, 144, 7, 2), (8, 128, 256, 24, 4), (20, 300, 528, 100, 3), (60, 64, 64, 90, 2),
                                       (5, 520, 720, 150, 2), (2, 260, 1040, 700, 1), (254, 33, 64, 64, 8), (300, 16, 32, 200, 4),
                                       (1024, 16, 16, 500, 2)])
def test_grouped(kind, E, N, K, T, k):
    x, w, ws, b, off, rows = grouped_case(kind, E, N, K, T, k)
    ref.check(run_grouped(x, w, ws, off, b, rows, k), *want_grouped(x, w, ws, off, b, rows, k), "picked rows")
    y = run_grouped(x, w, ws, [o * T // (T * k) for o in off])
    ref.check(y, *want_grouped(x, w, ws, [o * T // (T * k) for o in off]), "rows in order")


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("out", DTYPES)
def test_grouped_out_types(kind, out):
    x, w, ws, b, off, rows = grouped_case(kind, 6, 70, 272, 50, 2)
    ref.check(run_grouped(x, w, ws, off, b, rows, 2, out), *want_grouped(x, w, ws, off, b, rows, 2))
    ref.check(run_grouped(x, w, ws, off, None, rows, 2, out), *want_grouped(x, w, ws, off, None, rows, 2))


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("off", [[0, 0, 0, 0], [0, 64, 64, 64], [0, 0, 0, 64], [5, 20, 40, 60], [0, 16, 32, 48], [10, 10, 11, 12]])
def test_grouped_edges(kind, off):
    """All rows in one group, none in any, rows ahead of the first and behind the last: zeros there, though their
    entries of ``rows`` point nowhere."""
    x, w, ws, b, _, rows = grouped_case(kind, 3, 72, 160, 64, 1)
    rows = rows.clone()
    rows[: off[0]], rows[off[-1]:] = -(2**31), 2**31 - 1
    y = run_grouped(x, w, ws, off, b, rows)
    ref.check(y, *want_grouped(x, w, ws, off, b, rows))
    assert not y[: off[0]].any() and not y[off[-1]:].any()


@pytest.mark.parametrize("kind", ["bf16", "int8"])
def test_grouped_rows_that_are_not_there(kind):
    """Entries of ``rows`` outside x take a row of zeros; groups are cut to the rows there are."""
    x, w, ws, b, _, rows = grouped_case(kind, 3, 72, 160, 64, 1)
    rows = rows.clone()
    rows[3], rows[20], rows[40], rows[41] = -1, 64, -(2**31), 2**31 - 1
    off = [0, 16, 30, 64]
    ref.check(run_grouped(x, w, ws, off, b, rows), *want_grouped(x, w, ws, off, b, rows))
    ref.check(run_grouped(x, w, ws, [-7, 16, 30, 10**9], b, rows), *want_grouped(x, w, ws, [0, 16, 30, 64], b, rows))


@pytest.mark.parametrize("kind", ["bf16", "int8"])
def test_grouped_over_packed_slots(kind):
    """Weights that are a view of slots which hold more than the matrix: read where they are."""
    x, w, ws, _, off, rows = grouped_case(kind, 5, 48, 160, 40, 2, bias=False)
    es = w.element_size()
    slots = torch.zeros((5, 48 * 160 * es + 112), dtype=torch.uint8, device="cuda")
    slots[:, 32 : 32 + 48 * 160 * es] = w.view(5, -1).view(torch.uint8)
    v = slots.view(w.dtype).as_strided((5, 48, 160), (slots.shape[1] // es, 160, 1), 32 // es)
    assert v.data_ptr() == slots.data_ptr() + 32 and torch.equal(v, w)
    want = want_grouped(x, w, ws, off, None, rows, 2)
    ref.check(run_grouped(x, v, ws, off, None, rows, 2), *want, "slots")
    ref.check(run_grouped(x, w.transpose(1, 2).contiguous().transpose(1, 2), ws, off, None, rows, 2), *want, "transposed")
    ref.check(run_grouped(x, w[:1].expand(5, -1, -1), ws if ws is None else ws[:1].expand(5, -1).contiguous(), off, None, rows, 2),
              *want_grouped(x, w[:1].expand(5, -1, -1), ws if ws is None else ws[:1].expand(5, -1), off, None, rows, 2), "one matrix for all")


@pytest.mark.parametrize("kind", ["bf16", "int8"])
def test_grouped_routing(kind):
    """The rows of a routing as group_by_expert sorts them, some ids without an expert."""
    E, k, T = 12, 3, 50
    x, w, ws, b, _, _ = grouped_case(kind, E, 96, 128, T, k)
    idx = torch.randint(-2, E, (T, k), device="cuda", generator=gen(9)).to(torch.int32)
    idx[idx < 0] = -1
    _, off, perm = ops.group_by_expert(idx, E)
    y = run_grouped(x, w, ws, off.tolist(), b, perm, k)
    perm = perm.clone()
    perm[off[-1]:] = 0
    ref.check(y, *want_grouped(x, w, ws, off.tolist(), b, perm, k))


def test_grouped_nothing():
    x, w, _, b, _, _ = grouped_case("bf16", 3, 72, 160, 8, 1)
    off = torch.zeros(4, dtype=torch.int32, device="cuda")
    assert ops.grouped_matmul(x[:0], w, off, b).shape == (0, 72)
    assert ops.grouped_matmul(x[:0], w, off, b, rows=off[:0]).shape == (0, 72)


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("E", [5, 300, 1000])
def test_grouped_offsets_that_do_not_ascend(kind, E):
    """Offsets are raised to the largest before them and cut to the rows there are: each row is in one group."""
    x, w, ws, b, _, rows = grouped_case(kind, E, 48, 64, 90, 2)
    off = torch.randint(-50, 300, (E + 1,), device="cuda", generator=gen(E)).int()
    off[0] = 7
    top = off.clamp(0, 180).cummax(0).values.tolist()
    ref.check(run_grouped(x, w, ws, off.tolist(), b, rows, 2), *want_grouped(x, w, ws, top, b, rows, 2))
    worst = torch.arange(E, -1, -1, device="cuda").int() * 2**20
    ref.check(run_grouped(x, w, ws, worst.tolist(), b, rows, 2), *want_grouped(x, w, ws, worst.clamp(0, 180).cummax(0).values.tolist(), b, rows, 2))


# ----------------------------------------------------------------------------- where rules change, and far ends
@pytest.mark.parametrize("T", [11, 12, 13, 14, 95, 96, 97, 128, 160, 161, 192, 193, 224, 225, 256, 257, 320])
@pytest.mark.parametrize("K,N", [(2048, 512), (704, 2880), (720, 4096), (256, 5760)])
def test_linear_where_kernels_change(T, K, N):
    """Around the last token count that is quantised inside the product, and that the row kernel takes."""
    x, w, ws, b = linear_case(T, K, N, torch.bfloat16, torch.float32)
    want, err = ref.matmul(*ref.quantize(x), w, ws, b)
    ref.check(ops.int8_linear(x, w, ws, b), want, err)


@pytest.mark.parametrize("T", [1, 2, 3, 12])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K", [8192, 8208, 10912, 10928, 32768, 131056])
def test_linear_long_rows(T, K, dtype):
    """Rows longer than what a wave holds, and than what LDS holds (quantised by a launch of their own)."""
    x, w, ws, b = linear_case(T, K, 40, dtype, None)
    want, err = ref.matmul(*ref.quantize(x), w, ws, b)
    ref.check(ops.int8_linear(x, w, ws, b), want, err)


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("per", [1, 4, 5, 48, 49])
def test_grouped_where_tiles_change(kind, per):
    """Rows per expert on average at the ends of the tiles' ranges."""
    x, w, ws, b, off, rows = grouped_case(kind, 7, 200, 144, 7 * per, 1)
    for R in (7 * per - 1, 7 * per):
        o = [min(v, R) for v in off]
        ref.check(run_grouped(x, w, ws, o, b, rows[:R].contiguous()), *want_grouped(x, w, ws, o, b, rows[:R]))


def test_many_tokens():
    """More tokens than a launch has threads for, results past 2^32 bytes."""
    T, K, N = 2**26 + 17, 16, 40
    x = torch.randn((2**20, K), device="cuda", generator=gen(1)).bfloat16().repeat(65, 1)[:T]
    x[-40:] *= 3
    w, ws = ref.weights8(gen(2), N, K)
    codes, scales = ops.int8_quantize(x)
    y = ops.int8_matmul(codes, scales, w, ws)
    for at in (0, 2**25 - 20, 2**31 // 80 - 100, 2**32 // 80 - 100, 2**26 - 100):
        part = slice(at, min(T, at + 200))
        check_codes(x[part], codes[part], scales[part])
        ref.check(y[part], *ref.matmul(*ref.quantize(x[part]), w, ws), f"from {at}")
    assert torch.equal(y[2**20 : 2**21], y[: 2**20])
    again = ops.int8_linear(x, w, ws)
    assert all(torch.equal(a, b) for a, b in zip(again.split(2**24), y.split(2**24)))


@pytest.mark.parametrize("kind", ["bf16", "int8"])
def test_grouped_far_offsets(kind):
    """Experts whose matrices lie past 2^32 bytes, results that do."""
    es, K, N = (1, 65536, 1024) if kind == "int8" else (2, 32768, 1024)
    E = 70  # of 64 MiB
    w = torch.zeros((E, N, K), dtype=torch.int8 if es == 1 else torch.bfloat16, device="cuda")
    ws = torch.full((E, N), 2.0**-7, device="cuda") if es == 1 else None
    for e in (0, 31, 32, 63, 64, 69):
        r = torch.randint(-127, 128, (N, 128), device="cuda", generator=gen(e))
        w[e, :, ::K // 128] = r.to(w.dtype)
    x = acts(gen(3), 30, K)
    sizes = {0: 5, 31: 3, 32: 4, 63: 6, 64: 5, 69: 7}
    off = [0]
    for e in range(E):
        off.append(off[-1] + sizes.get(e, 0))
    ref.check(run_grouped(x, w, ws, off), *want_grouped(x, w, ws, off))
    del w
    R, N, K = 1_100_000, 2048, 16
    x = acts(gen(4), 4096, K).repeat(R // 4096 + 1, 1)[:R]
    w, ws = ref.weights8(gen(5), 2, N, K) if es == 1 else (0.1 * torch.randn((2, N, K), device="cuda", generator=gen(5)).bfloat16(), None)
    y = run_grouped(x, w, ws, [0, 600_000, R - 50])
    for at in (0, 2**31 // 4096 - 50, 600_000 - 100, 2**32 // 4096 - 50, R - 200):
        n = min(200, R - at)
        cut = [min(n, max(0, o - at)) for o in (0, 600_000, R - 50)]
        ref.check(y[at : at + n], *want_grouped(x[at : at + n], w, None if ws is None else ws, cut), f"from {at}")


@pytest.mark.parametrize("kind", ["bf16", "int8"])
def test_grouped_x_at_its_limit(kind):
    """Rows picked from an x of nearly 2^31 bytes."""
    K = 2048 if kind == "int8" else 1024
    rows_x = 2**20 - 1
    x = acts(gen(6), 1023, K).repeat(1025, 1)[:rows_x]
    w, ws = ref.weights8(gen(7), 2, 48, K) if kind == "int8" else (0.1 * torch.randn((2, 48, K), device="cuda", generator=gen(7)).bfloat16(), None)
    rows = torch.tensor([0, rows_x - 1, 2**19, 2**19 - 1, rows_x, rows_x - 2, 3, rows_x - 1], dtype=torch.int32, device="cuda")
    y = run_grouped(x, w, ws, [0, 5, 8], None, rows)
    small = torch.where(rows < rows_x, torch.arange(8, device="cuda").int(), torch.tensor(8, device="cuda", dtype=torch.int32))
    ref.check(y, *want_grouped(x[rows.long().clamp(max=rows_x - 1)], w, ws, [0, 5, 8], None, small))


def test_captured_and_on_a_stream():
    """Captured calls replayed on new inputs, eager ones between; and the same on a stream of the caller's."""
    w, ws = ref.weights8(gen(1), 200, 288)
    wg, wgs = ref.weights8(gen(2), 4, 80, 288)
    w16 = (0.05 * torch.randn((4, 80, 288), device="cuda", generator=gen(3))).bfloat16()
    xs = [acts(gen(4), T, 288) for T in (1, 12, 40, 300)]
    off = torch.tensor([0, 100, 100, 180, 290], dtype=torch.int32, device="cuda")

    def step():
        out = [ops.int8_linear(x, w, ws) for x in xs]
        codes, scales = ops.int8_quantize(xs[3])
        out += [ops.int8_matmul(codes, scales, w, ws), ops.int8_grouped_matmul(codes, scales, wg, wgs, off), ops.grouped_matmul(xs[3], w16, off)]
        return out

    def check(outs):
        for x, y in zip(xs, outs):
            ref.check(y, *ref.matmul(*ref.quantize(x), w, ws))
        assert torch.equal(outs[4], outs[3])
        o = off.tolist()
        ref.check(outs[5], *ref.grouped(ref.quantize(xs[3]), wg, o, int8=wgs))
        ref.check(outs[6], *ref.grouped(xs[3], w16, o))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in range(3):
        for x in xs:
            x.copy_(acts(gen(100 + seed + len(x)), *x.shape))
        graph.replay()
        got = [y.clone() for y in outs]
        check(got)
        assert all(torch.equal(a, b) for a, b in zip(step(), got))
        torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = step()
    torch.cuda.current_stream().wait_stream(side)
    check(outs)
