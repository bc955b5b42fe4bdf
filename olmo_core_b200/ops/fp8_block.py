"""
e4m3 products whose operands carry one power-of-two scale per block of 128 along the reduction (``csrc/gemm_block_fp8_sm100.cu``),
and the quantisers that produce such operands (``csrc/block_quant_sm100.cu``).

Three block forms. A block's scale is the smallest power of two, not below ``2^-126``, that brings its largest magnitude to
448 or below, and 1 for a block of zeros, so that the only rounding is the one to e4m3:

* rows: 128 consecutive elements of a row. Activations and output gradients.
* columns: 128 consecutive elements of a column. Both operands of the weight gradient, whose reduction runs over the rows.
* tiles: 128 x 128 elements. Weights: the same codes and scales serve the forward product and the input gradient.

Operands keep the orientation of the tensor they come from; no product needs a transposed copy::

    forward   y  = q_rows(x) q_tiles(W)^T          x [M, K], W [N, K]
    dgrad     dx = q_rows(dy) q_tiles(W)           dy [M, N]
    wgrad     dW = q_columns(dy)^T q_columns(x)    fp32, optionally accumulated into ``main_grad``

Codes are e4m3 bytes (``uint8``, ``float8_e4m3fn`` is accepted too) whose rows start on 16-byte boundaries; the quantisers
return them that way for any width. The scales of an operand with one scale per row of the product are stored with the
reduction block first: ``[ceil(reduction / 128), rows]``. The tensor core applies the scales as exponents: they must be positive
normal powers of two, any other scale makes the results that depend on it NaN (a weight that comes with other scales is
brought into this form by quantising its values: ``quantize_block_tiles(dequantize_block_tiles(codes, scales))``).

On CPU the functions emulate the same arithmetic in PyTorch: the numerical oracle.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from .fp8 import cached_weight_cast
from .gemm import compute_weight, gemm, grouped_gemm_wgrad

__all__ = ["BLOCK", "quantize_block_rows", "quantize_block_columns", "quantize_block_tiles", "dequantize_block_rows",
           "dequantize_block_columns", "dequantize_block_tiles", "gemm_fp8_block", "grouped_gemm_fp8_block",
           "fp8_block_matmul", "fp8_block_grouped_matmul", "fp8_block_linear", "fp8_block_grouped_linear",
           "BlockFloat8LinearFunction", "BlockFloat8GroupedLinearFunction"]

BLOCK = 128

_lib_sigs_done = False


def _lib_block():
    global _lib_sigs_done
    lib = _lib.lib()
    if not _lib_sigs_done:
        from ctypes import c_int, c_longlong, c_void_p

        _lib.register_signature("ocb_quantize_block_fp8", [c_void_p] * 7 + [c_int] * 3 + [c_longlong] * 4 + [c_void_p])
        _lib.register_signature("ocb_gemm_block_fp8", [c_void_p] * 6 + [c_int] * 4 + [c_longlong] * 6 + [c_int]
                                + [c_longlong] * 3 + [c_int] * 4 + [c_void_p] * 2)
        _lib_sigs_done = True
    return lib


def _blocks(n: int) -> int:
    return (n + BLOCK - 1) // BLOCK


# ------------------------------------------------------------------------------------------------------
# Quantisation
# ------------------------------------------------------------------------------------------------------


def _scale_of(amax: torch.Tensor) -> torch.Tensor:
    """Smallest power of two, not below ``2^-126``, with ``amax / scale <= 448``; 1 for zero (bit arithmetic of the kernel)."""
    bits = amax.float().view(torch.int32)
    e = (bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000).to(torch.int32)
    e = torch.where(bits == 0, torch.full_like(e, 127), e.clamp(1, 253))
    return (e << 23).view(torch.float32)


def _emulate_block_quantize(x: torch.Tensor, rows: int, cols: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """``x [..., R, C]`` -> e4m3 bytes and the scale of every block of ``rows x cols`` ``[..., R / rows, C / cols]``."""
    *lead, R, C = x.shape
    xf = torch.nn.functional.pad(x.float(), (0, -C % cols, 0, -R % rows))
    b = xf.view(*lead, xf.shape[-2] // rows, rows, xf.shape[-1] // cols, cols)
    mag = torch.where(b.isnan(), torch.zeros_like(b), b.abs())
    s = _scale_of(mag.amax(dim=(-3, -1), keepdim=True))
    v = b / s
    v = torch.where(v.isinf(), torch.full_like(v, float("nan")), v)
    q = v.to(torch.float8_e4m3fn).view(torch.uint8).view(xf.shape)[..., :R, :C]
    return q.contiguous(), s.squeeze(-1).squeeze(-2)


def _codes(lead, rows: int, cols: int, device) -> torch.Tensor:
    """Uninitialised code matrix (or stack) whose rows start on 16-byte boundaries."""
    return torch.empty((*lead, rows, (cols + 15) // 16 * 16), dtype=torch.uint8, device=device)[..., :cols]


def _check_matrix(x: torch.Tensor, what: str, dims: Tuple[int, ...] = (2,)) -> torch.Tensor:
    if x.dim() not in dims:
        raise ValueError(f"{what} must have {' or '.join(map(str, dims))} dimensions, got shape {tuple(x.shape)}")
    if x.dtype != torch.bfloat16:
        x = x.to(torch.bfloat16)
    return x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()


def _launch_quantize(x: torch.Tensor, q_row, s_row, q_col, s_col, q_tile=None, s_tile=None) -> None:
    R, C = x.shape[-2:]
    groups = x.shape[0] if x.dim() == 3 else 1
    q = next(t for t in (q_row, q_col, q_tile) if t is not None)
    with torch.cuda.device(x.device):
        rc = _lib_block().ocb_quantize_block_fp8(
            x.data_ptr(), _lib.ptr(q_row), _lib.ptr(s_row), _lib.ptr(q_col), _lib.ptr(s_col), _lib.ptr(q_tile),
            _lib.ptr(s_tile), groups, R, C, x.stride(-2), q.stride(-2), x.stride(0) if x.dim() == 3 else 0,
            q.stride(0) if x.dim() == 3 else 0, _lib.stream_ptr())
    _lib.check(rc, "ocb_quantize_block_fp8")


def quantize_block_rows(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """``x [R, C]`` -> (codes ``[R, C]``, scales ``[ceil(C / 128), R]``): one scale per 128 elements of each row."""
    x = _check_matrix(x, "x")
    R, C = x.shape
    if not x.is_cuda:
        q, s = _emulate_block_quantize(x, 1, BLOCK)
        return q, s.t().contiguous()
    q, s = _codes((), R, C, x.device), torch.empty((_blocks(C), R), dtype=torch.float32, device=x.device)
    if x.numel():
        _launch_quantize(x, q, s, None, None)
    return q, s


def quantize_block_columns(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """``x [R, C]`` -> (codes ``[R, C]``, scales ``[ceil(R / 128), C]``): one scale per 128 elements of each column."""
    x = _check_matrix(x, "x")
    R, C = x.shape
    if not x.is_cuda:
        return _emulate_block_quantize(x, BLOCK, 1)
    q, s = _codes((), R, C, x.device), torch.empty((_blocks(R), C), dtype=torch.float32, device=x.device)
    if x.numel():
        _launch_quantize(x, None, None, q, s)
    return q, s


def quantize_block_rows_columns(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """:func:`quantize_block_rows` and :func:`quantize_block_columns` of the same tensor, which is read once."""
    x = _check_matrix(x, "x")
    if not x.is_cuda or not x.numel():
        return (*quantize_block_rows(x), *quantize_block_columns(x))
    R, C = x.shape
    qr, sr = _codes((), R, C, x.device), torch.empty((_blocks(C), R), dtype=torch.float32, device=x.device)
    qc, sc = _codes((), R, C, x.device), torch.empty((_blocks(R), C), dtype=torch.float32, device=x.device)
    _launch_quantize(x, qr, sr, qc, sc)
    return qr, sr, qc, sc


def quantize_block_tiles(w: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """
    ``w [N, K]`` or a stack ``[G, N, K]`` -> (codes of the same shape, scales ``[(G,) ceil(N / 128), ceil(K / 128)]``): one
    scale per 128 x 128 tile.
    """
    w = _check_matrix(w, "w", (2, 3))
    *lead, N, K = w.shape
    if not w.is_cuda:
        return _emulate_block_quantize(w, BLOCK, BLOCK)
    q = _codes(lead, N, K, w.device)
    s = torch.empty((*lead, _blocks(N), _blocks(K)), dtype=torch.float32, device=w.device)
    if w.numel():
        _launch_quantize(w, None, None, None, None, q, s)
    return q, s


def _values(q: torch.Tensor) -> torch.Tensor:
    return (q if q.dtype == torch.float8_e4m3fn else q.view(torch.float8_e4m3fn)).float()


def _exponent_scales(s: torch.Tensor) -> torch.Tensor:
    """``s`` as the products see it: NaN where it is no positive normal power of two."""
    bits = s.contiguous().view(torch.int32)
    return torch.where(((bits & -0x7F800001) == 0) & (bits > 0) & (bits < 0x7F800000), s, float("nan"))


def _spread(s: torch.Tensor, dim: int, n: int) -> torch.Tensor:
    return s.repeat_interleave(BLOCK, dim).narrow(dim, 0, n)


def dequantize_block_rows(q: torch.Tensor, s: torch.Tensor) -> torch.Tensor:
    """fp32 values of an operand from :func:`quantize_block_rows`."""
    return _values(q) * _spread(s.t(), 1, q.shape[1])


def dequantize_block_columns(q: torch.Tensor, s: torch.Tensor) -> torch.Tensor:
    """fp32 values of an operand from :func:`quantize_block_columns`."""
    return _values(q) * _spread(s, 0, q.shape[0])


def dequantize_block_tiles(q: torch.Tensor, s: torch.Tensor) -> torch.Tensor:
    """fp32 values of an operand from :func:`quantize_block_tiles`."""
    return _values(q) * _spread(_spread(s, -2, q.shape[-2]), -1, q.shape[-1])


# ------------------------------------------------------------------------------------------------------
# Products
# ------------------------------------------------------------------------------------------------------


def _check_codes(q: torch.Tensor, what: str, dims: int) -> None:
    if q.dim() != dims:
        raise ValueError(f"{what} must have {dims} dimensions, got shape {tuple(q.shape)}")
    if q.dtype not in (torch.uint8, torch.float8_e4m3fn):
        raise ValueError(f"{what} must hold e4m3 bytes (uint8 or float8_e4m3fn), got {q.dtype}")
    if q.is_cuda and q.numel() and (
            (q.stride(-1) != 1 and q.shape[-1] > 1) or q.data_ptr() % 16
            or any(st % 16 for st, n in zip(q.stride()[:-1], q.shape[:-1]) if n > 1)):
        raise ValueError(f"{what}: rows of codes must be contiguous and start on 16-byte boundaries, got strides {q.stride()}")


def _check_scales(s: torch.Tensor, what: str, shape: Tuple[int, ...], device: torch.device) -> None:
    if tuple(s.shape) != shape:
        raise ValueError(f"{what} must have shape {shape}, got {tuple(s.shape)}")
    if s.dtype != torch.float32:
        raise ValueError(f"{what} must be float32, got {s.dtype}")
    if s.device != device:
        raise ValueError(f"{what} is on {s.device}, the codes are on {device}")


def _epilogue(out: torch.Tensor, accumulate: bool) -> int:
    if out.dtype == torch.bfloat16 and not accumulate:
        return _lib.EPI_BF16
    if out.dtype == torch.float32:
        return _lib.EPI_F32_ACC if accumulate else _lib.EPI_F32
    raise ValueError(f"the product writes bfloat16, or float32 (optionally accumulating), got {out.dtype}"
                     f"{' with accumulation' if accumulate else ''}")


def _check_out(out: Optional[torch.Tensor], shape: Tuple[int, int], accumulate: bool, out_dtype: torch.dtype,
               device: torch.device) -> torch.Tensor:
    if out is None:
        if accumulate:
            raise ValueError("accumulate=True needs an output tensor")
        out = torch.empty(shape, dtype=out_dtype, device=device)
    if tuple(out.shape) != shape or out.device != device:
        raise ValueError(f"output is {tuple(out.shape)} on {out.device}, expected {shape} on {device}")
    if out.stride(1) != 1 and out.shape[1] > 1:
        raise ValueError("output rows must be contiguous")
    _epilogue(out, accumulate)
    return out


def _store(out: torch.Tensor, res: torch.Tensor, accumulate: bool) -> torch.Tensor:
    return out.add_(res) if accumulate else out.copy_(res)


def gemm_fp8_block(
    a_q: torch.Tensor,
    a_s: torch.Tensor,
    b_q: torch.Tensor,
    b_s: torch.Tensor,
    *,
    trans_a: bool = False,
    trans_b: bool = True,
    b_tiles: bool = True,
    out: Optional[torch.Tensor] = None,
    accumulate: bool = False,
    out_dtype: torch.dtype = torch.bfloat16,
) -> torch.Tensor:
    """
    ``out (=|+=) op(a) @ op(b)`` of quantised operands, fp32 accumulation.

    Stored shapes: ``a_q [M, K]`` (``[K, M]`` when ``trans_a``) with scales ``a_s [ceil(K / 128), M]``; ``b_q [N, K]`` when
    ``trans_b``, else ``[K, N]``, with the tile scales of the stored matrix (``b_tiles``) or with ``b_s [ceil(K / 128), N]``.
    ``out`` may be bf16 or, optionally accumulated into, fp32.
    """
    _check_codes(a_q, "a_q", 2)
    _check_codes(b_q, "b_q", 2)
    M, K = a_q.shape[::-1] if trans_a else a_q.shape
    N, Kb = b_q.shape if trans_b else b_q.shape[::-1]
    if K != Kb:
        raise ValueError(f"inner dimensions differ: {K} vs {Kb}")
    if a_q.device != b_q.device:
        raise ValueError(f"operands are on {a_q.device} and {b_q.device}")
    _check_scales(a_s, "a_s", (_blocks(K), M), a_q.device)
    _check_scales(b_s, "b_s", (_blocks(b_q.shape[0]), _blocks(b_q.shape[1])) if b_tiles else (_blocks(K), N), a_q.device)
    out = _check_out(out, (M, N), accumulate, out_dtype, a_q.device)
    if M == 0 or N == 0:
        return out
    if K == 0:
        return out if accumulate else out.zero_()
    if not a_q.is_cuda:
        a_s, b_s = _exponent_scales(a_s), _exponent_scales(b_s)
        a = dequantize_block_columns(a_q, a_s).t() if trans_a else dequantize_block_rows(a_q, a_s)
        if b_tiles:
            b = dequantize_block_tiles(b_q, b_s)
        else:
            b = dequantize_block_rows(b_q, b_s) if trans_b else dequantize_block_columns(b_q, b_s)
        return _store(out, a @ (b.t() if trans_b else b), accumulate)
    if b_tiles:  # scale of (reduction block, block of output columns) wherever the stored tile sits
        sb_k, sb_i = (b_s.stride(1), b_s.stride(0)) if trans_b else (b_s.stride(0), b_s.stride(1))
    else:
        sb_k, sb_i = b_s.stride()
    with torch.cuda.device(a_q.device):
        rc = _lib_block().ocb_gemm_block_fp8(
            a_q.data_ptr(), b_q.data_ptr(), out.data_ptr(), a_s.data_ptr(), b_s.data_ptr(), None, 1, M, N, K, _pitch(a_q),
            _pitch(b_q), out.stride(0), 0, a_s.stride(0), a_s.stride(1), 0, sb_k, sb_i, 0, 7 if b_tiles else 0,
            int(trans_a), int(not trans_b), _epilogue(out, accumulate), _lib.status_buffer(a_q.device).data_ptr(),
            _lib.stream_ptr())
    _lib.check(rc, "ocb_gemm_block_fp8")
    return out


def _pitch(q: torch.Tensor) -> int:
    """Bytes between the rows of a code matrix (a single row may carry any stride)."""
    return q.stride(-2) if q.shape[-2] > 1 else (q.shape[-1] + 15) // 16 * 16


def grouped_gemm_fp8_block(
    a_q: torch.Tensor,
    a_s: torch.Tensor,
    b_q: torch.Tensor,
    b_s: torch.Tensor,
    offsets: torch.Tensor,
    *,
    trans_b: bool = True,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """
    ``out[rows of group g] = a[rows of group g] @ op(b_g)`` in one launch, bf16. ``a_q [R, K]`` sorted by group with scales
    ``[ceil(K / 128), R]``; ``b_q [G, N, K]`` (``trans_b``) or ``[G, K, N]`` with tile scales; ``offsets`` int32 ``[G + 1]`` on
    the same device, non-decreasing row boundaries within ``[0, R]`` (read by the kernel: no host synchronisation). Rows
    outside every group are not written.
    """
    _check_codes(a_q, "a_q", 2)
    _check_codes(b_q, "b_q", 3)
    R, K = a_q.shape
    G = b_q.shape[0]
    N, Kb = b_q.shape[1:] if trans_b else (b_q.shape[2], b_q.shape[1])
    if K != Kb:
        raise ValueError(f"inner dimensions differ: {K} vs {Kb}")
    if a_q.device != b_q.device:
        raise ValueError(f"operands are on {a_q.device} and {b_q.device}")
    _check_offsets(offsets, G, a_q.device)
    _check_scales(a_s, "a_s", (_blocks(K), R), a_q.device)
    _check_scales(b_s, "b_s", (G, _blocks(b_q.shape[1]), _blocks(b_q.shape[2])), a_q.device)
    out = _check_out(out, (R, N), False, torch.bfloat16, a_q.device)
    if out.dtype != torch.bfloat16:
        raise ValueError(f"the grouped product writes bfloat16, got {out.dtype}")
    if R == 0 or N == 0 or G == 0:
        return out
    if K == 0:
        return out.zero_()
    if not a_q.is_cuda:
        a, b = dequantize_block_rows(a_q, _exponent_scales(a_s)), dequantize_block_tiles(b_q, _exponent_scales(b_s))
        bounds = offsets.tolist()
        for g, (lo, hi) in enumerate(zip(bounds[:-1], bounds[1:])):
            out[lo:hi] = (a[lo:hi] @ (b[g].t() if trans_b else b[g])).to(out.dtype)
        return out
    sb_k, sb_i = (b_s.stride(2), b_s.stride(1)) if trans_b else (b_s.stride(1), b_s.stride(2))
    with torch.cuda.device(a_q.device):
        rc = _lib_block().ocb_gemm_block_fp8(
            a_q.data_ptr(), b_q.data_ptr(), out.data_ptr(), a_s.data_ptr(), b_s.data_ptr(), offsets.data_ptr(), G, R, N, K,
            _pitch(a_q), _pitch(b_q), out.stride(0), b_q.stride(0) if G > 1 else b_q.shape[1] * _pitch(b_q), a_s.stride(0),
            a_s.stride(1), 0, sb_k, sb_i, b_s.stride(0), 7, 0, int(not trans_b), _lib.EPI_BF16,
            _lib.status_buffer(a_q.device).data_ptr(), _lib.stream_ptr())
    _lib.check(rc, "ocb_gemm_block_fp8")
    return out


def _check_offsets(offsets: torch.Tensor, groups: int, device: torch.device) -> None:
    if offsets.dtype != torch.int32 or tuple(offsets.shape) != (groups + 1,):
        raise ValueError(f"offsets must be int32 [{groups + 1}], got {offsets.dtype} {tuple(offsets.shape)}")
    if offsets.device != device:
        raise ValueError(f"offsets are on {offsets.device}, the rows are on {device}")
    if not offsets.is_contiguous():
        raise ValueError("offsets must be contiguous")


# ------------------------------------------------------------------------------------------------------
# Layers
# ------------------------------------------------------------------------------------------------------


def fp8_block_matmul(x: torch.Tensor, w_q: torch.Tensor, w_s: torch.Tensor, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """
    ``x @ W^T (+ bias)`` for a weight that is kept in 8 bits: codes ``w_q [N, K]`` with tile scales ``w_s`` (from
    :func:`quantize_block_tiles` or a checkpoint). ``x [..., K]`` is quantised by rows; the result is bf16. No gradient.
    """
    with torch.no_grad():
        x2 = x.reshape(-1, x.shape[-1])
        q, s = quantize_block_rows(x2)
        y = gemm_fp8_block(q, s, w_q, w_s)
    y = y.view(*x.shape[:-1], w_q.shape[0])
    return y if bias is None else y + bias.to(y.dtype)


def fp8_block_grouped_matmul(x: torch.Tensor, w_q: torch.Tensor, w_s: torch.Tensor, offsets: torch.Tensor, *,
                             trans_b: bool = True) -> torch.Tensor:
    """
    The experts' product for weights that are kept in 8 bits: ``y[rows of g] = x[rows of g] @ op(W_g)``; ``x [R, K]`` sorted
    by group, ``w_q [G, N, K]`` (``trans_b``) or ``[G, K, N]`` with tile scales, ``offsets`` int32 ``[G + 1]``. No gradient.
    """
    with torch.no_grad():
        q, s = quantize_block_rows(x)
        return grouped_gemm_fp8_block(q, s, w_q, w_s, offsets, trans_b=trans_b)


class BlockFloat8LinearFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, wgrad_high_precision: bool, cache: Optional[dict] = None):  # type: ignore[override]
        w = compute_weight(weight, torch.bfloat16)
        x2 = _check_matrix(x.reshape(-1, x.shape[-1]), "x")
        wq, sw = cached_weight_cast(cache, "block_tiles", lambda: quantize_block_tiles(w), weight._version)
        needs_dw = ctx.needs_input_grad[1] or getattr(weight, "main_grad", None) is not None
        if needs_dw and not wgrad_high_precision:
            # what the backward pass keeps of x is its column-scaled form: one byte per element
            xq, sx, xc, sxc = quantize_block_rows_columns(x2)
            kept = (xc, sxc)
        else:
            xq, sx = quantize_block_rows(x2)
            kept = (x2,) if needs_dw else ()
        y = gemm_fp8_block(xq, sx, wq, sw)
        ctx.save_for_backward(wq, sw, *kept)
        ctx.wgrad_hp = wgrad_high_precision
        ctx.weight_ref, ctx.x_shape, ctx.x_dtype = weight, x.shape, x.dtype
        return y.view(*x.shape[:-1], w.shape[0])

    @staticmethod
    def backward(ctx, dy):  # type: ignore[override]
        wq, sw, *kept = ctx.saved_tensors
        weight = ctx.weight_ref
        dy2 = _check_matrix(dy.reshape(-1, dy.shape[-1]), "dy")
        main_grad = getattr(weight, "main_grad", None)
        needs_dw = main_grad is not None or ctx.needs_input_grad[1]
        wgrad_fp8 = needs_dw and not ctx.wgrad_hp
        dx = dw = None
        if ctx.needs_input_grad[0] and wgrad_fp8:
            dyq, sdy, dyc, sdyc = quantize_block_rows_columns(dy2)
        elif ctx.needs_input_grad[0]:
            dyq, sdy = quantize_block_rows(dy2)
        elif wgrad_fp8:
            dyc, sdyc = quantize_block_columns(dy2)
        if ctx.needs_input_grad[0]:
            dx = gemm_fp8_block(dyq, sdy, wq, sw, trans_b=False).view(ctx.x_shape).to(ctx.x_dtype)
        if needs_dw:
            if wgrad_fp8:
                args, kwargs = (dyc, sdyc, *kept), dict(trans_a=True, trans_b=False, b_tiles=False)
                product = gemm_fp8_block
            else:
                args, kwargs, product = (dy2, kept[0]), dict(trans_a=True, trans_b=False), gemm
            if main_grad is not None:
                product(*args, **kwargs, out=main_grad, accumulate=True)
                if hasattr(weight, "grad_added_to_main_grad"):
                    weight.grad_added_to_main_grad = True
            elif weight.dtype == torch.bfloat16:
                dw = product(*args, **kwargs, out_dtype=torch.bfloat16)
            else:
                dw = product(*args, **kwargs, out_dtype=torch.float32).to(weight.dtype)
        return dx, dw, None, None


def fp8_block_linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                     wgrad_high_precision: bool = False, weight_cache: Optional[dict] = None) -> torch.Tensor:
    """
    ``x @ weight^T (+ bias)`` with block-scaled e4m3 operands in all three products; any sizes. ``wgrad_high_precision``
    keeps the weight gradient in bf16 (widths must then be multiples of 8). ``weight_cache``: see
    :func:`olmo_core_b200.ops.fp8.cached_weight_cast`.
    """
    if x.shape[-1] != weight.shape[-1]:
        raise ValueError(f"x has {x.shape[-1]} features, the weight takes {weight.shape[-1]}")
    y = BlockFloat8LinearFunction.apply(x, weight, wgrad_high_precision, weight_cache)
    return y if bias is None else y + bias.to(y.dtype)


class BlockFloat8GroupedLinearFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, offsets, trans_b: bool, cache: Optional[dict] = None):  # type: ignore[override]
        w = compute_weight(weight, torch.bfloat16)
        G = offsets.numel() - 1
        x2 = _check_matrix(x, "x")
        wq, sw = cached_weight_cast(cache, "block_tiles", lambda: quantize_block_tiles(w.view(G, -1, w.shape[-1])), weight._version)
        xq, sx = quantize_block_rows(x2)
        y = grouped_gemm_fp8_block(xq, sx, wq, sw, offsets, trans_b=trans_b)
        ctx.save_for_backward(wq, sw, offsets, x2)
        ctx.trans_b, ctx.weight_ref, ctx.w_shape, ctx.x_dtype = trans_b, weight, w.shape, x.dtype
        return y

    @staticmethod
    def backward(ctx, dy):  # type: ignore[override]
        wq, sw, offsets, x2 = ctx.saved_tensors
        trans_b, weight = ctx.trans_b, ctx.weight_ref
        dy2 = _check_matrix(dy, "dy")
        dx = dw = None
        if ctx.needs_input_grad[0]:
            dyq, sdy = quantize_block_rows(dy2)
            dx = grouped_gemm_fp8_block(dyq, sdy, wq, sw, offsets, trans_b=not trans_b).to(ctx.x_dtype)
        main_grad = getattr(weight, "main_grad", None)
        if main_grad is not None or ctx.needs_input_grad[1]:
            a, b = (dy2, x2) if trans_b else (x2, dy2)
            if main_grad is not None:
                dw = main_grad.view(ctx.w_shape)
            else:
                dw = torch.empty(ctx.w_shape, dtype=torch.bfloat16 if weight.dtype == torch.bfloat16 else torch.float32,
                                 device=x2.device)
            if x2.is_cuda:
                grouped_gemm_wgrad(a.contiguous(), b.contiguous(), offsets, dw, accumulate=main_grad is not None)
            else:
                bounds, per = offsets.tolist(), dw.view(offsets.numel() - 1, -1, dw.shape[1])
                for g, (lo, hi) in enumerate(zip(bounds[:-1], bounds[1:])):
                    _store(per[g], a[lo:hi].float().t() @ b[lo:hi].float(), main_grad is not None)
            if main_grad is not None:
                if hasattr(weight, "grad_added_to_main_grad"):
                    weight.grad_added_to_main_grad = True
                dw = None
            else:
                dw = dw.to(weight.dtype)
        return dx, dw, None, None, None


def fp8_block_grouped_linear(x: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor, *, trans_b: bool = True,
                             weight_cache: Optional[dict] = None) -> torch.Tensor:
    """
    The experts' linear layer with block-scaled e4m3 operands in the forward product and in the input gradient; the weight
    gradient is taken in bf16, because the 128-row blocks of a column scale would run across the experts' boundaries.
    ``x [R, K]`` sorted by expert, ``offsets`` int32 ``[G + 1]``, ``weight`` the experts' matrices stacked: ``[G * N, K]`` with
    ``trans_b`` (``y = x W_g^T``) else ``[G * K, N]`` (``y = x W_g``). Widths must be multiples of 8.
    """
    G = offsets.numel() - 1
    w = compute_weight(weight, torch.bfloat16)
    if G < 1 or w.dim() != 2 or w.shape[0] % G:
        raise ValueError(f"a weight of shape {tuple(w.shape)} does not stack {G} equal matrices")
    K = w.shape[1] if trans_b else w.shape[0] // G
    if x.dim() != 2 or x.shape[1] != K:
        raise ValueError(f"x of shape {tuple(x.shape)} does not fit experts that take {K} features")
    if w.shape[1] % 8 or (w.shape[0] // G) % 8:
        raise ValueError("the widths of the experts' matrices must be multiples of 8")
    return BlockFloat8GroupedLinearFunction.apply(x, weight, offsets, trans_b, weight_cache)
