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

import functools
from typing import Optional, Tuple

import torch

from . import _lib
from .fp8 import cached_weight_cast, weight_state
from .gemm import gemm

__all__ = ["BLOCK", "quantize_block_rows", "quantize_block_columns", "quantize_block_tiles", "dequantize_block_rows",
           "dequantize_block_columns", "dequantize_block_tiles", "gemm_fp8_block", "grouped_gemm_fp8_block",
           "fp8_block_matmul", "fp8_block_grouped_matmul", "fp8_block_linear", "fp8_block_grouped_linear",
           "BlockFloat8LinearFunction", "BlockFloat8GroupedLinearFunction"]

BLOCK = 128
MAX_SIZE = 2 ** 31 - 513  # of any dimension: the kernels round 32-bit sizes up to tiles

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


def _pitch(q: torch.Tensor) -> int:
    """Bytes between the rows of a code matrix (a single row may carry any stride)."""
    return q.stride(-2) if q.shape[-2] > 1 else (q.shape[-1] + 15) // 16 * 16


def _check_sizes(t: torch.Tensor, what: str) -> None:
    if any(n > MAX_SIZE for n in t.shape):
        raise ValueError(f"{what} of shape {tuple(t.shape)} is too large: no dimension may exceed {MAX_SIZE}")


def _check_matrix(x: torch.Tensor, what: str, dims: Tuple[int, ...] = (2,)) -> torch.Tensor:
    if x.dim() not in dims:
        raise ValueError(f"{what} must have {' or '.join(map(str, dims))} dimensions, got shape {tuple(x.shape)}")
    _check_sizes(x, what)
    if x.dtype != torch.bfloat16:
        x = x.to(torch.bfloat16)
    return x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()


def _launch_quantize(x: torch.Tensor, q_row, s_row, q_col, s_col, q_tile=None, s_tile=None) -> None:
    R, C = x.shape[-2:]
    groups = x.shape[0] if x.dim() == 3 else 1
    q = next(t for t in (q_row, q_col, q_tile) if t is not None)
    rc = _lib.on_device(
        x.device, _lib_block().ocb_quantize_block_fp8, x.data_ptr(), _lib.ptr(q_row), _lib.ptr(s_row), _lib.ptr(q_col),
        _lib.ptr(s_col), _lib.ptr(q_tile), _lib.ptr(s_tile), groups, R, C, x.stride(-2), _pitch(q),
        x.stride(0) if x.dim() == 3 else 0, q.stride(0) if x.dim() == 3 else 0)
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
    _check_sizes(q, what)
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
    rc = _lib.on_device(
        a_q.device, _lib_block().ocb_gemm_block_fp8, a_q.data_ptr(), b_q.data_ptr(), out.data_ptr(), a_s.data_ptr(),
        b_s.data_ptr(), None, 1, M, N, K, _pitch(a_q), _pitch(b_q), out.stride(0), 0, a_s.stride(0), a_s.stride(1), 0, sb_k,
        sb_i, 0, 7 if b_tiles else 0, int(trans_a), int(not trans_b), _epilogue(out, accumulate),
        _lib.status_buffer(a_q.device).data_ptr())
    _lib.check(rc, "ocb_gemm_block_fp8")
    return out


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
    rc = _lib.on_device(
        a_q.device, _lib_block().ocb_gemm_block_fp8, a_q.data_ptr(), b_q.data_ptr(), out.data_ptr(), a_s.data_ptr(),
        b_s.data_ptr(), offsets.data_ptr(), G, R, N, K, _pitch(a_q), _pitch(b_q), out.stride(0),
        b_q.stride(0) if G > 1 else b_q.shape[1] * _pitch(b_q), a_s.stride(0), a_s.stride(1), 0, sb_k, sb_i, b_s.stride(0), 7,
        0, int(not trans_b), _lib.EPI_BF16, _lib.status_buffer(a_q.device).data_ptr())
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


def _native_product(x: torch.Tensor, w_q: torch.Tensor, w_s: torch.Tensor, offsets: Optional[torch.Tensor], trans_b: bool) -> torch.Tensor:
    """``q_rows(x) @ op(W)`` (bf16) for checked operands on a GPU: quantiser and product in one call."""
    y = _lib.native().block_product.default(x, w_q, w_s, offsets, trans_b, _lib.status_buffer(x.device).data_ptr())
    return y


def fp8_block_matmul(x: torch.Tensor, w_q: torch.Tensor, w_s: torch.Tensor, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """
    ``x @ W^T (+ bias)`` for a weight that is kept in 8 bits: codes ``w_q [N, K]`` with tile scales ``w_s`` (from
    :func:`quantize_block_tiles` or a checkpoint). ``x [..., K]`` is quantised by rows; the result is bf16. No gradient.
    """
    _check_codes(w_q, "w_q", 2)
    N, K = w_q.shape
    if x.dim() == 0 or x.shape[-1] != K:
        raise ValueError(f"x of shape {tuple(x.shape)} does not have the {K} features that the weight takes")
    if x.device != w_q.device:
        raise ValueError(f"x is on {x.device}, the weight on {w_q.device}")
    _check_scales(w_s, "w_s", (_blocks(N), _blocks(K)), w_q.device)
    with torch.no_grad():
        x2 = x if x.dim() == 2 else x.reshape(-1, K)
        y = _native_product(x2, w_q, w_s, None, True) if x2.is_cuda else gemm_fp8_block(*quantize_block_rows(x2), w_q, w_s)
        y = y if x.dim() == 2 else y.view(*x.shape[:-1], N)
        return y if bias is None else y + bias.to(y.dtype)


def fp8_block_grouped_matmul(x: torch.Tensor, w_q: torch.Tensor, w_s: torch.Tensor, offsets: torch.Tensor, *,
                             trans_b: bool = True) -> torch.Tensor:
    """
    The experts' product for weights that are kept in 8 bits: ``y[rows of g] = x[rows of g] @ op(W_g)``; ``x [R, K]`` sorted
    by group, ``w_q [G, N, K]`` (``trans_b``) or ``[G, K, N]`` with tile scales, ``offsets`` int32 ``[G + 1]`` (row boundaries,
    see :func:`grouped_gemm_fp8_block`). Rows outside every group are undefined. No gradient.
    """
    _check_codes(w_q, "w_q", 3)
    G, n, k = w_q.shape
    if x.dim() != 2 or x.shape[1] != (k if trans_b else n):
        raise ValueError(f"x of shape {tuple(x.shape)} does not fit experts that take {k if trans_b else n} features")
    if x.device != w_q.device:
        raise ValueError(f"x is on {x.device}, the weights on {w_q.device}")
    _check_offsets(offsets, G, w_q.device)
    _check_scales(w_s, "w_s", (G, _blocks(n), _blocks(k)), w_q.device)
    with torch.no_grad():
        if x.is_cuda and G:
            return _native_product(x, w_q, w_s, offsets, trans_b)
        return grouped_gemm_fp8_block(*quantize_block_rows(x), w_q, w_s, offsets, trans_b=trans_b)


def _whole(weight: torch.Tensor) -> torch.Tensor:
    """All rows of a weight: of a sharded one, which holds this rank's rows itself, the resident copy, whatever its type."""
    lowp = getattr(weight, "_lowp", None)
    return weight.detach() if lowp is None else lowp


def _cached(cache: Optional[dict], make, weight: torch.Tensor):
    """The 8-bit form of ``weight``, kept in ``cache`` (see :func:`olmo_core_b200.ops.fp8.cached_weight_cast`)."""
    state = weight_state(weight)
    made = cached_weight_cast(cache, "block_tiles", make, state)
    first = made if torch.is_tensor(made) else made[0]
    if cache is not None and first.is_inference() and not torch.is_inference_mode_enabled():
        cache.clear()  # made under inference mode, cannot be saved for a backward pass
        made = cached_weight_cast(cache, "block_tiles", make, state)
    return made


def _check_main_grad(grad: Optional[torch.Tensor], w: torch.Tensor, stacked: bool) -> None:
    """The host's check before anything is written to ``main_grad`` (on a GPU: ``csrc/torch_ops.cpp``)."""
    if grad is None:
        return
    if grad.dtype != torch.float32 or grad.device != w.device:
        raise ValueError(f"main_grad must be float32 on {w.device}, got {grad.dtype} on {grad.device}")
    if stacked:
        fits = grad.numel() == w.numel() and grad.is_contiguous()
    else:
        N, K = w.shape
        fits = grad.shape == w.shape and (K <= 1 or grad.stride(1) == 1) and (N <= 1 or grad.stride(0) >= K)
    if not fits:
        raise ValueError(f"main_grad of shape {tuple(grad.shape)} and strides {grad.stride()} does not fit a weight of shape "
                         f"{tuple(w.shape)}: {'it' if stacked else 'rows'} must be contiguous")


def _weight_gradient(weight: torch.Tensor, main_grad: Optional[torch.Tensor], out: torch.Tensor) -> Optional[torch.Tensor]:
    """What a backward pass returns for the weight: nothing once ``main_grad`` (``out`` then) has it."""
    if main_grad is None:
        return out.to(weight.dtype)
    if hasattr(weight, "grad_added_to_main_grad"):
        weight.grad_added_to_main_grad = True
    return None


def _first_order(backward):
    """For a backward pass whose own derivative is not built: differentiating its result is an error."""

    @functools.wraps(backward)
    def wrapper(ctx, dy):
        with torch.no_grad():
            grads = backward(ctx, dy)
        if not torch.is_grad_enabled():
            return grads
        error = torch._C._functions.DelayedError(b"the block-scaled layers have no second derivative", len(grads))
        return error(*[g if g is None else g.detach().requires_grad_(True) for g in grads])

    return wrapper


class BlockFloat8LinearFunction(torch.autograd.Function):
    """The layer on CPU tensors, through the emulated operations (on a GPU: ``csrc/torch_ops.cpp``)."""

    @staticmethod
    def forward(ctx, x, weight, wgrad_high_precision: bool, cache: Optional[dict] = None):  # type: ignore[override]
        w = _whole(weight).to(torch.bfloat16)
        x2 = _check_matrix(x.reshape(-1, x.shape[-1]), "x")
        wq, sw = _cached(cache, lambda: quantize_block_tiles(w), weight)
        ctx.save_for_backward(wq, sw, x2)
        ctx.wgrad_hp, ctx.has_main_grad = wgrad_high_precision, getattr(weight, "main_grad", None) is not None
        ctx.weight_ref, ctx.x_shape, ctx.x_dtype = weight, x.shape, x.dtype
        return gemm_fp8_block(*quantize_block_rows(x2), wq, sw).view(*x.shape[:-1], w.shape[0])

    @staticmethod
    @_first_order
    def backward(ctx, dy):  # type: ignore[override]
        wq, sw, x2 = ctx.saved_tensors
        weight = ctx.weight_ref
        dy2 = _check_matrix(dy.reshape(-1, wq.shape[0]), "dy")
        main_grad = getattr(weight, "main_grad", None) if ctx.has_main_grad else None
        _check_main_grad(main_grad, wq, False)
        dx = dw = None
        if ctx.needs_input_grad[0]:
            dx = gemm_fp8_block(*quantize_block_rows(dy2), wq, sw, trans_b=False).view(ctx.x_shape).to(ctx.x_dtype)
        if main_grad is not None or ctx.needs_input_grad[1]:
            out = main_grad if main_grad is not None else torch.empty(
                wq.shape, dtype=torch.bfloat16 if weight.dtype == torch.bfloat16 else torch.float32)
            if ctx.wgrad_hp:
                gemm(dy2, x2, trans_a=True, trans_b=False, out=out, accumulate=main_grad is not None)
            else:
                gemm_fp8_block(*quantize_block_columns(dy2), *quantize_block_columns(x2), trans_a=True, trans_b=False,
                               b_tiles=False, out=out, accumulate=main_grad is not None)
            dw = _weight_gradient(weight, main_grad, out)
        return dx, dw, None, None


def fp8_block_linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                     wgrad_high_precision: bool = False, weight_cache: Optional[dict] = None) -> torch.Tensor:
    """
    ``x @ weight^T (+ bias)`` with block-scaled e4m3 operands in all three products; any sizes. ``wgrad_high_precision``
    keeps the weight gradient in bf16 (widths must then be multiples of 8). ``weight_cache``: see
    :func:`olmo_core_b200.ops.fp8.cached_weight_cast`. The gradient of a weight that has a ``main_grad`` (fp32) in the forward pass is
    added to the one that it has in the backward pass. First derivatives only: differentiating the gradients is an error.
    """
    w, main_grad = _whole(weight), getattr(weight, "main_grad", None)
    try:
        (_, K), features = w.shape, x.shape[-1]
    except (ValueError, IndexError):
        raise ValueError(f"the layer takes x [..., K] and a weight [N, K], got shapes {tuple(x.shape)} and {tuple(w.shape)}") from None
    if features != K:
        raise ValueError(f"x has {features} features, the weight takes {K}")
    if x.device != weight.device:
        raise ValueError(f"x is on {x.device}, the weight on {weight.device}")
    if wgrad_high_precision and any(n % 8 for n in w.shape):
        raise ValueError("a weight gradient in bf16 needs widths that are multiples of 8")
    if x.is_cuda:
        native = _lib.native()
        tiles = None if weight_cache is None else _cached(weight_cache, lambda: native.block_tile_buffer.default(w, 1), weight)
        y = native.block_linear.default(x, weight, w, tiles, main_grad, wgrad_high_precision,
                                        _lib.status_buffer(x.device).data_ptr())
    else:
        _check_main_grad(main_grad if torch.is_grad_enabled() else None, w, False)
        y = BlockFloat8LinearFunction.apply(x, weight, wgrad_high_precision, weight_cache)
    return y if bias is None else y + bias.to(y.dtype)


class BlockFloat8GroupedLinearFunction(torch.autograd.Function):
    """The experts' layer on CPU tensors (on a GPU: ``csrc/torch_ops.cpp``)."""

    @staticmethod
    def forward(ctx, x, weight, offsets, trans_b: bool, cache: Optional[dict] = None):  # type: ignore[override]
        w = _whole(weight).to(torch.bfloat16)
        x2 = _check_matrix(x, "x")
        wq, sw = _cached(cache, lambda: quantize_block_tiles(w.view(offsets.numel() - 1, -1, w.shape[-1])), weight)
        ctx.save_for_backward(wq, sw, offsets, x2)
        ctx.trans_b, ctx.weight_ref, ctx.w_shape, ctx.x_dtype = trans_b, weight, w.shape, x.dtype
        ctx.has_main_grad = getattr(weight, "main_grad", None) is not None
        return grouped_gemm_fp8_block(*quantize_block_rows(x2), wq, sw, offsets, trans_b=trans_b)

    @staticmethod
    @_first_order
    def backward(ctx, dy):  # type: ignore[override]
        wq, sw, offsets, x2 = ctx.saved_tensors
        trans_b, weight = ctx.trans_b, ctx.weight_ref
        dy2 = _check_matrix(dy, "dy")
        dx = dw = None
        if ctx.needs_input_grad[0]:
            dx = grouped_gemm_fp8_block(*quantize_block_rows(dy2), wq, sw, offsets, trans_b=not trans_b).to(ctx.x_dtype)
        main_grad = getattr(weight, "main_grad", None) if ctx.has_main_grad else None
        if main_grad is not None or ctx.needs_input_grad[1]:
            _check_main_grad(main_grad, wq, True)
            a, b = (dy2, x2) if trans_b else (x2, dy2)
            out = main_grad.view(ctx.w_shape) if main_grad is not None else torch.empty(ctx.w_shape, dtype=weight.dtype)
            bounds, per = offsets.tolist(), out.view(offsets.numel() - 1, -1, out.shape[1])
            for g, (lo, hi) in enumerate(zip(bounds[:-1], bounds[1:])):
                _store(per[g], a[lo:hi].float().t() @ b[lo:hi].float(), main_grad is not None)
            dw = _weight_gradient(weight, main_grad, out)
        return dx, dw, None, None, None


def fp8_block_grouped_linear(x: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor, *, trans_b: bool = True,
                             weight_cache: Optional[dict] = None) -> torch.Tensor:
    """
    The experts' linear layer with block-scaled e4m3 operands in the forward product and in the input gradient; the weight
    gradient is taken in bf16, because the 128-row blocks of a column scale would run across the experts' boundaries.
    ``x [R, K]`` sorted by expert, ``offsets`` int32 ``[G + 1]`` (row boundaries, see :func:`grouped_gemm_fp8_block`), ``weight``
    the experts' matrices stacked: ``[G * N, K]`` with ``trans_b`` (``y = x W_g^T``) else ``[G * K, N]`` (``y = x W_g``). Widths
    must be multiples of 8. Rows outside every group are undefined. First derivatives only, as :func:`fp8_block_linear`.
    """
    G = offsets.numel() - 1
    w = _whole(weight)
    if G < 1 or w.dim() != 2 or w.shape[0] % G:
        raise ValueError(f"a weight of shape {tuple(w.shape)} does not stack {G} equal matrices")
    K = w.shape[1] if trans_b else w.shape[0] // G
    if x.dim() != 2 or x.shape[1] != K:
        raise ValueError(f"x of shape {tuple(x.shape)} does not fit experts that take {K} features")
    if w.shape[1] % 8 or (w.shape[0] // G) % 8:
        raise ValueError("the widths of the experts' matrices must be multiples of 8")
    _check_offsets(offsets, G, x.device)
    main_grad = getattr(weight, "main_grad", None)
    if x.is_cuda:
        if x.device != weight.device:
            raise ValueError(f"x is on {x.device}, the weights on {weight.device}")
        native = _lib.native()
        tiles = None if weight_cache is None else _cached(weight_cache, lambda: native.block_tile_buffer.default(w, G), weight)
        y = native.block_grouped_linear.default(x, weight, w, offsets, tiles, main_grad, trans_b,
                                                _lib.status_buffer(x.device).data_ptr())
    else:
        _check_main_grad(main_grad if torch.is_grad_enabled() else None, w, True)
        y = BlockFloat8GroupedLinearFunction.apply(x, weight, offsets, trans_b, weight_cache)
    return y
