"""torch-facing wrappers of the C ABI: device tensors in, device tensors out.

Every function enqueues on the current HIP stream of the tensors' device and returns
without synchronising. Inputs must already be on the GPU; nothing here falls back to
a CPU implementation.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from . import _lib


_stream = _lib.tensor_stream


def _rows(x: torch.Tensor, K: int) -> torch.Tensor:
    """x as contiguous rows of K values (a [T, K] x as it is: no view to make)."""
    if x.dim() == 2 and x.shape[1] == K > 0:
        return x.contiguous()
    return x.reshape(-1, K).contiguous()


def _call(t: torch.Tensor, fn, *args) -> None:
    """fn(*args, stream) on the current stream of t's device, with that device current (kernels are launched on the
    current device). The context only where it changes something: it costs 1 us of a 7 us call."""
    d = t.get_device()
    if d == _lib.device_index():
        rc = fn(*args, _stream(t))
    else:
        with torch.cuda.device(d):
            rc = fn(*args, _stream(t))
    if rc:
        _lib.check(rc)


# ----------------------------------------------------------------------------- GGUF
def gguf_block_info(ggml_type: int) -> tuple[int, int]:
    be, ts = ctypes.c_int64(), ctypes.c_int64()
    _lib.check(_lib.load().tsa_gguf_block_info(int(ggml_type), ctypes.byref(be), ctypes.byref(ts)))
    return be.value, ts.value


def gguf_dequant(data: torch.Tensor, ggml_type: int, shape, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """Bit-exact dequantisation of raw GGUF bytes (uint8, on the GPU) to ``shape``."""
    _lib.require_device(data, what="data")
    if data.dtype != torch.uint8:
        raise RuntimeError("data must be uint8")
    data = data.contiguous()
    shape = tuple(int(s) for s in shape)
    n = 1
    for s in shape:
        n *= s
    out = torch.empty(shape, dtype=dtype, device=data.device)
    _call(data, _lib.load().tsa_gguf_dequant, int(ggml_type), data.data_ptr(), data.numel(), n, out.data_ptr(),
          _lib.tsa_dtype(dtype))
    return out


def gguf_matvec(x: torch.Tensor, w: torch.Tensor, ggml_type: int, out_features: int, in_features: int,
                out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """y[T, N] = x[T, K] @ deq(W)^T for an N x K GGUF matrix stored as raw bytes."""
    _lib.require_device(x, what="activation")
    _lib.require_device(w, what="weight_data")
    if w.dtype != torch.uint8:
        raise RuntimeError("weight_data must be uint8")
    K, N = int(in_features), int(out_features)
    x2 = _rows(x, K) if x.numel() % K == 0 else x.reshape(1, -1).contiguous()
    T = x2.shape[0]
    y = x.new_empty((T, N), dtype=out_dtype or x.dtype)
    w = w.contiguous()
    _call(x2, _lib.load().tsa_gguf_matvec, int(ggml_type), w.data_ptr(), w.numel(), x2.data_ptr(),
          _lib.tsa_dtype(x2.dtype), T, K, y.data_ptr(), _lib.tsa_dtype(y.dtype), N)
    return y


# ----------------------------------------------------------------------------- MXFP4
def mxfp4_dequant(blocks: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.bfloat16,
                  transpose: bool = False, out: torch.Tensor | None = None) -> torch.Tensor:
    """Bit-exact MXFP4 dequantisation: blocks [N, G, 16] + scales [N, G] -> [N, 32G] (or [32G, N])."""
    _lib.require_device(blocks, scales, what="blocks/scales")
    N = blocks.shape[0]
    G = scales.shape[-1] if scales.dim() > 1 else scales.numel() // max(N, 1)
    K = G * 32
    blocks, scales = blocks.contiguous(), scales.contiguous()
    shape = (K, N) if transpose else (N, K)
    if out is None:
        out = torch.empty(shape, dtype=dtype, device=blocks.device)
    elif not out.is_contiguous() or out.numel() != N * K or out.dtype != dtype:
        raise ValueError("out must be a contiguous tensor of N*K elements of the requested dtype")
    _call(blocks, _lib.load().tsa_mxfp4_dequant, blocks.data_ptr(), scales.data_ptr(), N, K, out.data_ptr(),
          _lib.tsa_dtype(dtype), int(transpose))
    return out.view(shape)


def mxfp4_tile_sizes(N: int, K: int) -> tuple[int, int]:
    """(blocks_bytes, scales_bytes) of an [N, K] MXFP4 matrix in the 16-row MFMA tile order."""
    bb, sb = ctypes.c_int64(), ctypes.c_int64()
    _lib.check(_lib.load().tsa_mxfp4_tile_sizes(N, K, ctypes.byref(bb), ctypes.byref(sb)))
    return bb.value, sb.value


def mxfp4_tile(blocks: torch.Tensor, scales: torch.Tensor, out_blocks: torch.Tensor | None = None,
               out_scales: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Repack MXFP4 blocks [N, G, 16] + scales [N, G] (checkpoint order) into the 16-row
    MFMA tile order the fast decode reads (uint8 tensors of mxfp4_tile_sizes bytes)."""
    _lib.require_device(blocks, scales, what="blocks/scales")
    N = blocks.shape[0]
    K = blocks[0].numel() * 2
    bb, sb = mxfp4_tile_sizes(N, K)
    blocks, scales = blocks.contiguous(), scales.contiguous()
    if out_blocks is None:
        out_blocks = torch.empty(bb, dtype=torch.uint8, device=blocks.device)
    if out_scales is None:
        out_scales = torch.empty(sb, dtype=torch.uint8, device=blocks.device)
    if out_blocks.numel() * out_blocks.element_size() < bb or out_scales.numel() * out_scales.element_size() < sb:
        raise ValueError(f"outputs too small: need {bb} and {sb} bytes")
    _call(blocks, _lib.load().tsa_mxfp4_tile, blocks.data_ptr(), scales.data_ptr(), N, K, out_blocks.data_ptr(),
          out_scales.data_ptr())
    return out_blocks, out_scales


def mxfp4_matvec(x: torch.Tensor, blocks: torch.Tensor, scales: torch.Tensor, bias: torch.Tensor | None = None,
                 out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """y[T, N] = x[T, K] @ deq(W)^T + bias with W in MXFP4 ([N, G, 16] or [N, 16G] blocks)."""
    _lib.require_device(x, blocks, scales, what="tensor")
    N = blocks.shape[0]
    K = blocks[0].numel() * 2
    x2 = _rows(x, K)
    T = x2.shape[0]
    y = x.new_empty((T, N), dtype=out_dtype or x.dtype)
    blocks, scales = blocks.contiguous(), scales.contiguous()
    b = None if bias is None else bias.contiguous()
    _call(x2, _lib.load().tsa_mxfp4_matvec, blocks.data_ptr(), scales.data_ptr(), _lib.ptr(b),
          _lib.tsa_dtype(b.dtype) if b is not None else 0, x2.data_ptr(), _lib.tsa_dtype(x2.dtype), T, y.data_ptr(),
          _lib.tsa_dtype(y.dtype), N, K)
    return y


# ----------------------------------------------------------------------------- FP8, blocks of 128
FP8_BLOCK = 128
_FP8_DTYPES = (torch.float8_e4m3fn, torch.uint8)


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """t with contiguous memory from a multiple of 16 bytes on (a copy if it is not there already)."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _one_device(first: torch.Tensor, *others: torch.Tensor | None) -> None:
    d = first.get_device()
    for t in others:
        if t is not None and t.get_device() != d:
            _lib.require_device(first, *others, what="tensor")
            raise RuntimeError(f"all tensors must be on one device (got {first.device} and {t.device})")
    if d < 0:
        _lib.require_device(first, what="tensor")


def _fp8_weight(w: torch.Tensor, scales: torch.Tensor, K: int) -> tuple[torch.Tensor, torch.Tensor, int]:
    """(codes, float32 scales, N) of a weight matrix [N, K], checked."""
    if w.dtype not in _FP8_DTYPES or w.dim() != 2:
        raise RuntimeError(f"FP8 weights must be float8_e4m3fn (or its bytes) [N, K], got {w.dtype} {tuple(w.shape)}")
    N, Kw = w.shape
    if Kw != K:
        raise RuntimeError(f"in_features differ: activations {K}, weight {Kw}")
    if scales.shape != (-(-N // FP8_BLOCK), -(-K // FP8_BLOCK)):
        raise RuntimeError(f"weight scales must be {[-(-N // FP8_BLOCK), -(-K // FP8_BLOCK)]} for an [{N}, {K}] weight, "
                           f"got {list(scales.shape)}")
    return _aligned(w), (scales if scales.dtype == torch.float32 else scales.float()).contiguous(), N


def _bias(bias: torch.Tensor | None, N: int) -> tuple[torch.Tensor | None, int | None, int]:
    """(contiguous bias, its pointer, its tsa_dtype)."""
    if bias is None:
        return None, None, 0
    if bias.numel() != N:
        raise RuntimeError(f"bias must have {N} elements, got {bias.numel()}")
    b = bias.contiguous()
    return b, b.data_ptr(), _lib.tsa_dtype(b.dtype)


def fp8_quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes float8_e4m3fn [T, K], scales float32 [T, ceil(K / 128)]) of x [..., K] (bf16, fp16 or fp32):
    per token and 128 columns, scale = max(max|x| / 448, 2^-126) and code = e4m3(x / scale)."""
    _lib.require_device(x, what="activation")
    dt = _lib.tsa_dtype(x.dtype)
    x2 = _rows(x, x.shape[-1])
    T, K = x2.shape
    codes = x2.new_empty((T, K), dtype=torch.float8_e4m3fn)
    scales = x2.new_empty((T, -(-K // FP8_BLOCK)), dtype=torch.float32)
    _call(x2, _lib.load().tsa_fp8_quantize, x2.data_ptr(), dt, T, K, codes.data_ptr(), scales.data_ptr())
    return codes, scales


def fp8_matmul(codes: torch.Tensor, scales: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor,
               bias: torch.Tensor | None = None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """y [T, N] = deq(codes) @ deq(w)^T (+ bias): codes [T, K] and scales [T, ceil(K / 128)] as
    fp8_quantize returns them, w [N, K] with scales [ceil(N / 128), ceil(K / 128)]; float32 sums. K
    must be a multiple of 16. Projections that share their input share one fp8_quantize."""
    _one_device(codes, scales, w, w_scales, bias)
    if codes.dtype not in _FP8_DTYPES or codes.dim() != 2:
        raise RuntimeError(f"FP8 activations must be float8_e4m3fn (or its bytes) [T, K], got {codes.dtype} {tuple(codes.shape)}")
    T, K = codes.shape
    if scales.shape != (T, -(-K // FP8_BLOCK)) or scales.dtype != torch.float32:
        raise RuntimeError(f"activation scales must be float32 [{T}, {-(-K // FP8_BLOCK)}], got {scales.dtype} {list(scales.shape)}")
    c, sc, (w, ws, N) = _aligned(codes), scales.contiguous(), _fp8_weight(w, w_scales, K)
    b, bp, bt = _bias(bias, N)
    y = c.new_empty((T, N), dtype=out_dtype)
    _call(c, _lib.load().tsa_fp8_matmul, c.data_ptr(), sc.data_ptr(), T, K, w.data_ptr(), ws.data_ptr(), N, bp, bt,
          y.data_ptr(), _lib.tsa_dtype(out_dtype))
    return y


@functools.lru_cache(maxsize=4096)
def _fp8_linear_workspace_size(T: int, K: int) -> int:
    n = ctypes.c_int64()
    _lib.check(_lib.load().tsa_fp8_linear_workspace_size(T, K, ctypes.byref(n)))
    return n.value


def fp8_linear(x: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor, bias: torch.Tensor | None = None,
               out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """y [T, N] = deq(fp8_quantize(x)) @ deq(w)^T (+ bias) for x [..., K] in bf16, fp16 or fp32; y in
    x's dtype unless ``out_dtype`` says otherwise. K must be a multiple of 16."""
    _one_device(x, w, w_scales, bias)
    dt, K = _lib.tsa_dtype(x.dtype), x.shape[-1]
    w, ws, N = _fp8_weight(w, w_scales, K)
    x2 = _aligned(_rows(x, K))
    b, bp, bt = _bias(bias, N)
    T = x2.shape[0]
    y = x2.new_empty((T, N), dtype=out_dtype)
    n = _fp8_linear_workspace_size(T, K)
    scratch = x2.new_empty(n, dtype=torch.uint8) if n else None
    _call(x2, _lib.load().tsa_fp8_linear, x2.data_ptr(), dt, T, K, w.data_ptr(), ws.data_ptr(), N, bp, bt, y.data_ptr(),
          dt if out_dtype is None else _lib.tsa_dtype(out_dtype), _lib.ptr(scratch), n)
    return y


# ----------------------------------------------------------------------------- int8, a scale per token and row
INT8_MAX_K = 131056  # values a row may have: the sums fit 32 bits


def _int8_codes(codes: torch.Tensor, scales: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Quantised tokens (codes int8 [T, K], scales float32 [T]), checked."""
    if codes.dtype != torch.int8 or codes.dim() != 2:
        raise RuntimeError(f"int8 activations must be int8 [T, K], got {codes.dtype} {tuple(codes.shape)}")
    if scales.shape != codes.shape[:1] or scales.dtype != torch.float32:
        raise RuntimeError(f"activation scales must be float32 [{codes.shape[0]}], got {scales.dtype} {list(scales.shape)}")
    return _aligned(codes), scales.contiguous()


def _int8_weight(w: torch.Tensor, scales: torch.Tensor, K: int) -> tuple[torch.Tensor, torch.Tensor, int]:
    """(codes, float32 scales, N) of a weight matrix [N, K], checked."""
    if w.dtype != torch.int8 or w.dim() != 2:
        raise RuntimeError(f"int8 weights must be int8 [N, K], got {w.dtype} {tuple(w.shape)}")
    N, Kw = w.shape
    if Kw != K:
        raise RuntimeError(f"in_features differ: activations {K}, weight {Kw}")
    if scales.numel() != N or scales.shape[0] != N:
        raise RuntimeError(f"weight scales must be [{N}] (or [{N}, 1]) for an [{N}, {K}] weight, got {list(scales.shape)}")
    return _aligned(w), (scales if scales.dtype == torch.float32 else scales.float()).contiguous(), N


def int8_quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes int8 [T, K], scales float32 [T]) of x [..., K] (bf16, fp16 or fp32): per token,
    scale = max(max|x| / 127, 2^-126) and code = round(x / scale), ties to even. A token that holds a NaN or an
    infinity has NaN as its scale and zeros as its codes."""
    _lib.require_device(x, what="activation")
    dt = _lib.tsa_dtype(x.dtype)
    x2 = _rows(x, x.shape[-1])
    T, K = x2.shape
    codes = x2.new_empty((T, K), dtype=torch.int8)
    scales = x2.new_empty(T, dtype=torch.float32)
    _call(x2, _lib.load().tsa_int8_quantize, x2.data_ptr(), dt, T, K, codes.data_ptr(), scales.data_ptr())
    return codes, scales


def int8_matmul(codes: torch.Tensor, scales: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor,
                bias: torch.Tensor | None = None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """y [T, N] = (codes @ w^T) * scales[:, None] * w_scales (+ bias): codes [T, K] and scales [T] as
    int8_quantize returns them, w int8 [N, K] with float32 scales [N] (or [N, 1]); exact sums. K must be a
    multiple of 16 (at most 131056). Projections that share their input share one int8_quantize."""
    _one_device(codes, scales, w, w_scales, bias)
    c, sc = _int8_codes(codes, scales)
    T, K = c.shape
    w, ws, N = _int8_weight(w, w_scales, K)
    b, bp, bt = _bias(bias, N)
    y = c.new_empty((T, N), dtype=out_dtype)
    _call(c, _lib.load().tsa_int8_matmul, c.data_ptr(), sc.data_ptr(), T, K, w.data_ptr(), ws.data_ptr(), N, bp, bt,
          y.data_ptr(), _lib.tsa_dtype(out_dtype))
    return y


@functools.lru_cache(maxsize=4096)
def _int8_linear_workspace_size(T: int, K: int) -> int:
    n = ctypes.c_int64()
    _lib.check(_lib.load().tsa_int8_linear_workspace_size(T, K, ctypes.byref(n)))
    return n.value


def int8_linear(x: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor, bias: torch.Tensor | None = None,
                out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """y [T, N] = int8_matmul(*int8_quantize(x), w, w_scales, bias) for x [..., K] in bf16, fp16 or fp32; y in
    x's dtype unless ``out_dtype`` says otherwise. K must be a multiple of 16 (at most 131056)."""
    _one_device(x, w, w_scales, bias)
    dt, K = _lib.tsa_dtype(x.dtype), x.shape[-1]
    w, ws, N = _int8_weight(w, w_scales, K)
    x2 = _aligned(_rows(x, K))
    b, bp, bt = _bias(bias, N)
    T = x2.shape[0]
    y = x2.new_empty((T, N), dtype=out_dtype)
    n = _int8_linear_workspace_size(T, K)
    scratch = x2.new_empty(n, dtype=torch.uint8) if n else None
    _call(x2, _lib.load().tsa_int8_linear, x2.data_ptr(), dt, T, K, w.data_ptr(), ws.data_ptr(), N, bp, bt, y.data_ptr(),
          dt if out_dtype is None else _lib.tsa_dtype(out_dtype), _lib.ptr(scratch), n)
    return y


# ----------------------------------------------------------------------------- products grouped by expert
def _grouped_weight(w: torch.Tensor, K: int, dtype: torch.dtype) -> tuple[torch.Tensor, int, int]:
    """(w, bytes from one expert's matrix to the next, N) of matrices [E, N, K]: each [N, K] contiguous, the experts
    any multiple of 16 bytes apart (views of packed slots as they are), else a copy."""
    if w.dim() != 3 or w.dtype != dtype:
        raise RuntimeError(f"the experts' weights must be {dtype} [E, N, K], got {w.dtype} {tuple(w.shape)}")
    E, N, Kw = w.shape
    if Kw != K or E < 1 or N < 1:
        raise RuntimeError(f"in_features differ: activations {K}, weights {tuple(w.shape)}")
    es = w.element_size()
    if w.stride(2) != 1 or w.stride(1) != K or w.stride(0) < N * K or w.stride(0) * es % 16 or w.data_ptr() % 16:
        w = _aligned(w)
    return w, max(w.stride(0), N * K) * es, N


def _grouped_rows(x: torch.Tensor, offsets: torch.Tensor, rows: torch.Tensor | None, top_k: int, E: int):
    """(offsets, rows or None, R) of a grouped product over x [T, K], checked."""
    if offsets.dtype != torch.int32 or offsets.numel() != E + 1:
        raise RuntimeError(f"offsets must be int32 [{E + 1}] for {E} experts, got {offsets.dtype} {list(offsets.shape)}")
    if rows is None:
        if top_k != 1:
            raise RuntimeError("top_k divides rows: without them it must be 1")
        return offsets.contiguous(), None, x.shape[0]
    if rows.dtype != torch.int32 or rows.dim() != 1 or top_k < 1:
        raise RuntimeError(f"rows must be an int32 vector and top_k positive, got {rows.dtype} {list(rows.shape)} and {top_k}")
    return offsets.contiguous(), rows.contiguous(), rows.numel()


def _grouped_bias(bias: torch.Tensor | None, E: int, N: int):
    if bias is not None and tuple(bias.shape) != (E, N):
        raise RuntimeError(f"bias must be [{E}, {N}], got {list(bias.shape)}")
    return _bias(bias, E * N)


def grouped_matmul(x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor, bias: torch.Tensor | None = None,
                   rows: torch.Tensor | None = None, top_k: int = 1, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """y [R, N]: y[r] = x[r] @ w[e]^T (+ bias[e]) for offsets[e] <= r < offsets[e + 1], the rows sorted by expert,
    offsets int32 [E + 1] (one that does not ascend counts as the largest before it), any number of rows for each; rows of
    no expert are zeros. x [T, K] and w [E, N, K] in bf16 or fp16 (an expert's matrix
    contiguous, the experts any multiple of 16 bytes apart), bias [E, N]; float32 sums, y in x's dtype unless
    ``out_dtype`` says otherwise. With ``rows`` (int32 [R]), row r takes x[rows[r] // top_k]: group_by_expert's offsets and
    perm with its top_k are the tokens of a routing. K must be a multiple of 8."""
    _one_device(x, w, offsets, bias, rows)
    if x.dim() != 2 or x.dtype not in (torch.bfloat16, torch.float16):
        raise RuntimeError(f"x must be bfloat16 or float16 [T, K], got {x.dtype} {tuple(x.shape)}")
    T, K = x.shape
    w, stride, N = _grouped_weight(w, K, x.dtype)
    E, x2 = w.shape[0], _aligned(x)
    off, rows, R = _grouped_rows(x2, offsets, rows, top_k, E)
    b, bp, bt = _grouped_bias(bias, E, N)
    y = x2.new_empty((R, N), dtype=out_dtype or x.dtype)
    _call(x2, _lib.load().tsa_grouped_matmul, x2.data_ptr(), _lib.tsa_dtype(x.dtype), T, K, w.data_ptr(), stride, E, N, off.data_ptr(),
          _lib.ptr(rows), R, top_k, bp, bt, y.data_ptr(), _lib.tsa_dtype(y.dtype))
    return y


def int8_grouped_matmul(codes: torch.Tensor, scales: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor, offsets: torch.Tensor,
                        bias: torch.Tensor | None = None, rows: torch.Tensor | None = None, top_k: int = 1,
                        out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """grouped_matmul over int8: codes [T, K] and scales [T] as int8_quantize returns them, w int8 [E, N, K] with
    scales [E, N] (or [E, N, 1]). K must be a multiple of 16."""
    _one_device(codes, scales, w, w_scales, offsets, bias, rows)
    c, sc = _int8_codes(codes, scales)
    T, K = c.shape
    w, stride, N = _grouped_weight(w, K, torch.int8)
    E = w.shape[0]
    if w_scales.numel() != E * N or tuple(w_scales.shape[:2]) != (E, N):
        raise RuntimeError(f"weight scales must be [{E}, {N}], got {list(w_scales.shape)}")
    ws = (w_scales if w_scales.dtype == torch.float32 else w_scales.float()).contiguous()
    off, rows, R = _grouped_rows(c, offsets, rows, top_k, E)
    b, bp, bt = _grouped_bias(bias, E, N)
    y = c.new_empty((R, N), dtype=out_dtype)
    _call(c, _lib.load().tsa_int8_grouped_matmul, c.data_ptr(), sc.data_ptr(), T, K, w.data_ptr(), stride, ws.data_ptr(), E, N,
          off.data_ptr(), _lib.ptr(rows), R, top_k, bp, bt, y.data_ptr(), _lib.tsa_dtype(out_dtype))
    return y


# ----------------------------------------------------------------------------- routing
ROUTE_MODES = {
    "topk_then_softmax": _lib.ROUTE_TOPK_SOFTMAX,
    "softmax_then_topk": _lib.ROUTE_SOFTMAX_TOPK_RENORM,
    "softmax_then_topk_no_renorm": _lib.ROUTE_SOFTMAX_TOPK,
}


def route_topk(logits: torch.Tensor, top_k: int, mode: str = "topk_then_softmax") -> tuple[torch.Tensor, torch.Tensor]:
    """(idx int32 [T, k], weights float32 [T, k]) from router logits [T, E]."""
    _lib.require_device(logits, what="logits")
    lg = _rows(logits, logits.shape[-1])
    T, E = lg.shape
    idx = torch.empty((T, top_k), dtype=torch.int32, device=lg.device)
    w = torch.empty((T, top_k), dtype=torch.float32, device=lg.device)
    _call(lg, _lib.load().tsa_route_topk, lg.data_ptr(), _lib.tsa_dtype(lg.dtype), T, E, int(top_k), ROUTE_MODES[mode],
          idx.data_ptr(), w.data_ptr())
    return idx, w


def router_logits(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
                  out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """The router linear on the GPU: [T, E] = x [T, H] @ weight [E, H]^T (+ bias), fp32
    accumulation, rounded once to ``out_dtype`` (default: the weight's dtype, as
    ``F.linear`` returns it)."""
    _lib.require_device(x, weight, *([bias] if bias is not None else []), what="tensor")
    E, H = weight.shape
    x2 = _rows(x, H)
    w = weight.contiguous()
    b = bias.contiguous() if bias is not None else None
    out = x.new_empty((x2.shape[0], E), dtype=out_dtype or weight.dtype)
    _call(x2, _lib.load().tsa_router_logits, x2.data_ptr(), _lib.tsa_dtype(x2.dtype), x2.shape[0], H, w.data_ptr(),
          _lib.tsa_dtype(w.dtype), _lib.ptr(b), _lib.tsa_dtype(b.dtype) if b is not None else 0, E, out.data_ptr(),
          _lib.tsa_dtype(out.dtype))
    return out


# ----------------------------------------------------------------------------- MoE
def _n_slots(pool: torch.Tensor, layout: _lib.ExpertLayout) -> int:
    """Whole slots of ``layout.slot_bytes`` in a contiguous uint8 pool (the kernels index
    slot * slot_bytes, so the pool must hold them all)."""
    if pool.dtype != torch.uint8 or not pool.is_contiguous():
        raise RuntimeError("the expert pool must be a contiguous uint8 tensor")
    n = pool.numel() // int(layout.slot_bytes)
    if n < 1:
        raise RuntimeError(f"expert pool of {pool.numel()} bytes holds no {layout.slot_bytes}-byte slot")
    return n


def _moe_rows(layout: _lib.ExpertLayout, x: torch.Tensor) -> torch.Tensor:
    """x as contiguous rows of ``hidden`` values (from a multiple of 16 bytes on for FP8, 16-bit and int8 experts)."""
    x2 = _rows(x, layout.hidden)
    return _aligned(x2) if layout.format in (_lib.EXPERT_FP8, _lib.EXPERT_DENSE, _lib.EXPERT_INT8) else x2


def _moe_out(out: torch.Tensor | None, x2: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """The result of a layer call on rows x2: new, or the caller's, which the kernels fill from its start."""
    if out is None:
        return torch.empty(x2.shape, dtype=dtype, device=x2.device)
    if not out.is_contiguous() or out.numel() < x2.numel():
        raise RuntimeError(f"out must be contiguous and hold {list(x2.shape)} values, got {list(out.shape)}")
    return out


def moe_decode_workspace_size(layout: _lib.ExpertLayout, T: int, k: int) -> int:
    """Bytes of the decode workspace for T tokens, k experts each; validates the layout
    (host only, raises RuntimeError with the library's message)."""
    n = ctypes.c_int64()
    _lib.check(_lib.load().tsa_moe_decode_workspace_size(ctypes.byref(layout), int(T), int(k), ctypes.byref(n)))
    return n.value


def moe_decode_workspace(layout: _lib.ExpertLayout, T: int, k: int, device) -> torch.Tensor:
    """Decode workspace, zeroed: its leading sync area (the one-launch MXFP4 decode's call
    counter and workgroup flags) must hold one value in every word before the first call."""
    return torch.zeros(max(moe_decode_workspace_size(layout, T, k), 1), dtype=torch.uint8, device=device)


def set_decode_options(tiled_form: int = 1, wait_limit: int = 1 << 18) -> None:
    """Process-wide: the tiled MXFP4 decode in two launches (1, the default) or one (0), and
    the polls a one-launch wait makes before it gives up (tsa_set_decode_options)."""
    _lib.check(_lib.load().tsa_set_decode_options(int(tiled_form), int(wait_limit)))


def decode_workspace_poisoned(workspace: torch.Tensor) -> bool:
    """True if a one-launch wait gave up on this workspace (synchronises the current stream)."""
    out = ctypes.c_int()
    _call(workspace, _lib.load().tsa_moe_decode_workspace_status, workspace.data_ptr(), workspace.numel(), ctypes.byref(out))
    return bool(out.value)


def moe_decode(layout: _lib.ExpertLayout, pool: torch.Tensor, slots: torch.Tensor, weights: torch.Tensor,
               x: torch.Tensor, out: torch.Tensor | None = None, workspace: torch.Tensor | None = None,
               out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """y[t] = sum_j weights[t, j] * FFN_{slots[t, j]}(x[t]) over the resident slot pool."""
    _one_device(x, pool, slots, weights, out, workspace)
    x2 = _moe_rows(layout, x)
    T = x2.shape[0]
    n_slots = _n_slots(pool, layout)
    out = _moe_out(out, x2, out_dtype or x.dtype)
    if T == 0:
        return out
    slots = slots.reshape(T, -1).to(torch.int32).contiguous()
    weights = weights.reshape(T, -1).to(torch.float32).contiguous()
    k = slots.shape[1]
    if weights.shape[1] != k:
        raise RuntimeError(f"{k} slots but {weights.shape[1]} weights a token")
    if workspace is None:
        workspace = moe_decode_workspace(layout, T, k, x.device)
    _call(x2, _lib.load().tsa_moe_decode, ctypes.byref(layout), pool.data_ptr(), n_slots, slots.data_ptr(),
          weights.data_ptr(), T, k, x2.data_ptr(), _lib.tsa_dtype(x2.dtype), out.data_ptr(), _lib.tsa_dtype(out.dtype),
          workspace.data_ptr(), workspace.numel())
    return out


def moe_decode_routed(layout: _lib.ExpertLayout, pool: torch.Tensor, expert_slot: torch.Tensor, logits: torch.Tensor,
                      x: torch.Tensor, top_k: int, mode: str = "topk_then_softmax", out: torch.Tensor | None = None,
                      workspace: torch.Tensor | None = None, out_dtype: torch.dtype | None = None,
                      return_routing: bool = False):
    """Router top-k + fused expert FFN in one call (a single launch for MXFP4, T <= 4)."""
    _one_device(x, pool, expert_slot, logits, out, workspace)
    x2 = _moe_rows(layout, x)
    T = x2.shape[0]
    out = _moe_out(out, x2, out_dtype or x.dtype)
    idx = torch.empty((T, top_k), dtype=torch.int32, device=x.device) if return_routing else None
    w = torch.empty((T, top_k), dtype=torch.float32, device=x.device) if return_routing else None
    if T == 0:
        return (out, idx, w) if return_routing else out
    lg = logits.reshape(T, -1).contiguous()
    E = lg.shape[1]
    expert_slot = expert_slot.to(torch.int32).contiguous()
    if expert_slot.numel() < E:
        raise RuntimeError(f"logits of {E} experts but slots of {expert_slot.numel()}")
    if workspace is None:
        workspace = moe_decode_workspace(layout, T, top_k, x.device)
    _call(x2, _lib.load().tsa_moe_decode_routed, ctypes.byref(layout), pool.data_ptr(), _n_slots(pool, layout),
          expert_slot.data_ptr(), E, lg.data_ptr(), _lib.tsa_dtype(lg.dtype), ROUTE_MODES[mode], T, int(top_k), x2.data_ptr(),
          _lib.tsa_dtype(x2.dtype), out.data_ptr(), _lib.tsa_dtype(out.dtype), _lib.ptr(idx), _lib.ptr(w),
          workspace.data_ptr(), workspace.numel())
    return (out, idx, w) if return_routing else out


def moe_decode_gated(layout: _lib.ExpertLayout, pool: torch.Tensor, expert_slot: torch.Tensor, x: torch.Tensor,
                     router_weight: torch.Tensor, router_bias: torch.Tensor | None, top_k: int,
                     mode: str = "topk_then_softmax", **kw):
    """Hidden states to the weighted expert sum without leaving the GPU: the router linear
    (router_logits), then moe_decode_routed on its logits (keyword arguments pass through)."""
    logits = router_logits(x, router_weight, router_bias)
    return moe_decode_routed(layout, pool, expert_slot, logits, x, top_k, mode, **kw)


def group_by_expert(idx: torch.Tensor, num_experts: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(counts [E], offsets [E+1], perm [n_valid]) — expert-major, token-major within an expert."""
    _lib.require_device(idx, what="idx")
    idx2 = idx.reshape(idx.shape[0], -1).to(torch.int32).contiguous()
    T, k = idx2.shape
    counts = torch.empty(num_experts, dtype=torch.int32, device=idx.device)
    offsets = torch.empty(num_experts + 1, dtype=torch.int32, device=idx.device)
    perm = torch.empty(max(T * k, 1), dtype=torch.int32, device=idx.device)
    _call(idx2, _lib.load().tsa_group_by_expert, idx2.data_ptr(), T, k, int(num_experts), counts.data_ptr(),
          offsets.data_ptr(), perm.data_ptr())
    return counts, offsets, perm[: T * k]


def moe_prefill_workspace(layout: _lib.ExpertLayout, T: int, k: int, E: int, device) -> torch.Tensor:
    n = ctypes.c_int64()
    _lib.check(_lib.load().tsa_moe_prefill_workspace_size(ctypes.byref(layout), int(T), int(k), int(E),
                                                          ctypes.byref(n)))
    return torch.empty(max(n.value, 1), dtype=torch.uint8, device=device)


def moe_prefill(layout: _lib.ExpertLayout, pool: torch.Tensor, expert_slot: torch.Tensor, idx: torch.Tensor,
                weights: torch.Tensor, x: torch.Tensor, out: torch.Tensor | None = None,
                workspace: torch.Tensor | None = None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """Batched (prefill) MoE: out[t] = sum_j weights[t, j] * FFN_{expert_slot[idx[t, j]]}(x[t])."""
    _one_device(x, pool, expert_slot, idx, weights, out, workspace)
    x2 = _moe_rows(layout, x)
    T = x2.shape[0]
    n_slots = _n_slots(pool, layout)
    out = _moe_out(out, x2, out_dtype or x.dtype)
    if T == 0:
        return out
    idx = idx.reshape(T, -1).to(torch.int32).contiguous()
    weights = weights.reshape(T, -1).to(torch.float32).contiguous()
    if weights.shape != idx.shape:
        raise RuntimeError(f"{idx.shape[1]} experts but {weights.shape[1]} weights a token")
    expert_slot = expert_slot.to(torch.int32).contiguous()
    k, E = idx.shape[1], expert_slot.numel()
    if workspace is None:
        workspace = moe_prefill_workspace(layout, T, k, E, x.device)
    _call(x2, _lib.load().tsa_moe_prefill, ctypes.byref(layout), pool.data_ptr(), n_slots, expert_slot.data_ptr(), E,
          idx.data_ptr(), weights.data_ptr(), T, k, x2.data_ptr(), _lib.tsa_dtype(x2.dtype), out.data_ptr(),
          _lib.tsa_dtype(out.dtype), workspace.data_ptr(), workspace.numel())
    return out
