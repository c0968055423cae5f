"""Products in 8-bit integers: weights with one scale an output channel, activations with one scale a token.

With a = max |x| of a token's row: scale s = a / 127 and q = rint(x * (127 / a)), in float.  Then

    y[t, n] = s[t] c[n] sum_k q[t, k] w[n, k]  (+ bias[n])

with 32-bit integer sums, which are exact, scales multiplied in float and one rounding, to the output's dtype.  A row of
zeros has scale 0; a row that holds a NaN or an infinity has scale NaN, so all of its results are NaN.

Weights are kept in 8 bits (half the bytes that a decode step of bfloat16 weights reads, and the tensor cores' faster
products for prompts); what a product reads of its activations is bfloat16 or float32, a ``PendingNorm`` (the residual add
and the RMS norm in front of a block then run on the way to 8 bits), or rows that are in 8 bits already.

A token's results are the same bits alone and among others, but for those behind a norm: there the row's scale has a float sum of
squares whose order goes by the number of tokens (each such scale is within 2^-18 of the true one).
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Union

import torch

from . import ops
from .build import load_call_binding, load_entry_points
from .ops import KernelError

MAX_K = 131071              # 128 * 128 * K stays below 2^31
MAX_ROWS = 2 ** 31 - 1 - 65536   # tokens, or rows of a weight: the kernels count them (and a step past their end) in 32 bits
_PLAIN, _GLU = 0, 1


class Int8Weight(NamedTuple):
    """``values`` int8 [N, K], rows a multiple of 16 bytes apart; ``scales`` float32 [N]: w[n, k] = scales[n] values[n, k]."""
    values: torch.Tensor
    scales: torch.Tensor

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        return (self.values.float() * self.scales[:, None]).to(dtype)


class Int8Rows(NamedTuple):
    """Tokens in 8 bits: ``values`` int8 [T, K], rows a multiple of 16 bytes apart; ``scales`` float32 [T]."""
    values: torch.Tensor
    scales: torch.Tensor

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        return (self.values.float() * self.scales[:, None]).to(dtype)


def row_pitch(k: int) -> int:
    """Bytes between the rows of a matrix in 8 bits with ``k`` columns."""
    return -(-k // 16) * 16


def _lib(glu: str = "silu"):
    if glu not in ops._GLU_DEFINES:
        raise KernelError(f"the gate {glu!r} is refused: {sorted(ops._GLU_DEFINES)}")
    return load_entry_points("int8_linear.cu", ops._GLU_DEFINES[glu] or None)


def _check_count(rows: int) -> None:
    if rows > MAX_ROWS:
        raise KernelError(f"{rows} rows are refused: at most {MAX_ROWS} a call")


def _check_8_bit(m, what: str) -> None:
    values, scales = m.values, m.scales
    if values.dtype != torch.int8 or scales.dtype != torch.float32:
        raise KernelError(f"{what} in 8 bits are int8 values with float32 scales")
    if values.dim() != 2 or values.stride(1) != 1 or scales.dim() != 1 or scales.numel() != values.shape[0] or not scales.is_contiguous():
        raise KernelError(f"{what} in 8 bits are values [rows, K] with a unit inner stride and one scale a row")
    _check_count(values.shape[0])
    if values.stride(0) % 16 or values.data_ptr() % 16 or values.stride(0) < values.shape[1]:
        raise KernelError(f"the rows of {what} in 8 bits lie a multiple of 16 bytes apart")


def _check_rows(x: torch.Tensor, what: str) -> None:
    ops._code(x)
    if x.dim() != 2 or (x.stride(1) != 1 and x.shape[1] > 1) or (x.shape[0] > 1 and x.stride(0) < x.shape[1]):
        raise KernelError(f"{what} takes rows [T, K] with a unit inner stride")
    _check_count(x.shape[0])


def _check_k(k: int) -> None:
    if not 1 <= k <= MAX_K:
        raise KernelError(f"{k} columns are refused: 1 to {MAX_K} (integer sums of 32 bits)")


def int8_weight(weight: torch.Tensor) -> Int8Weight:
    """A weight matrix [N, K] (bfloat16 or float32) in 8 bits, one scale an output channel; laid out once."""
    return Int8Weight(*quantize_rows(weight))


def int8_weight_from(values: torch.Tensor, scales: torch.Tensor) -> Int8Weight:
    """8-bit values [N, K] and scales [N] of a checkpoint, in the layout that the products take (a copy where it is not)."""
    if values.dtype != torch.int8 or values.dim() != 2 or scales.numel() != values.shape[0]:
        raise KernelError("a weight in 8 bits is int8 [N, K] with N scales")
    n, k = values.shape
    if values.stride(1) != 1 or values.stride(0) % 16 or values.stride(0) < k or values.data_ptr() % 16:
        padded = torch.zeros((n, row_pitch(k)), dtype=torch.int8, device=values.device)
        padded[:, :k] = values
        values = padded[:, :k]
    return Int8Weight(values, scales.reshape(-1).to(torch.float32).contiguous())


def quantize_rows(x: Union[torch.Tensor, ops.PendingNorm]) -> Int8Rows:
    """The rows of x [T, K], or of a norm that has not run (which then runs here), in 8 bits: for several products of the
    same rows."""
    src, residual, gain, kept, eps = _source(x)
    ops._cuda(src, residual, gain, kept)
    tokens, k = src.shape
    values = ops._empty((tokens, row_pitch(k)), torch.int8, src.device)
    scales = ops._empty((tokens,), torch.float32, src.device)
    rc = _lib().b200_int8_rows(src, residual, gain, kept, values, scales, tokens, k, src.stride(0) if tokens > 1 else k, values.shape[1],
                               ops._code(src), 0 if gain is None else ops._code(gain), eps, ops._stream())
    ops._ok(rc, "int8_rows", int(tokens > 0))
    return Int8Rows(values if values.shape[1] == k else values[:, :k], scales)


def _source(x):
    """(rows, residual, gain, where the sum goes, eps) of a tensor or a ``PendingNorm``."""
    if not isinstance(x, ops.PendingNorm):
        _check_rows(x, "a product in 8 bits")
        _check_k(x.shape[1])
        return x, None, None, None, 0.0
    if x.rows is not None:
        x = x.materialize()                      # (the norm's own kernel picks rows)
        _check_k(x.shape[1])
        return x, None, None, None, 0.0
    src, residual, gain, kept = x.x, x.residual, x.weight, x.residual_out
    _check_rows(src, "a norm in front of a product in 8 bits")
    _check_k(src.shape[1])
    ops._code(gain)
    if gain.numel() != src.shape[1] or not gain.is_contiguous():
        raise KernelError(f"norm weight has {gain.numel()} elements, the rows have {src.shape[1]}")
    if residual is not None and (residual.shape != src.shape or residual.dtype != src.dtype or not residual.is_contiguous()):
        raise KernelError("the residual must have the shape and dtype of x")
    return src, residual, gain, kept, x.eps


_byte_product = None             # of the compiled binding, which is loaded at the first product


def _product(x, weight: Int8Weight, bias, out_dtype, mode: int, glu: str, limit: float, alpha: float) -> torch.Tensor:
    global _byte_product
    if ops._held is not None or ops._chain is not None:
        ops.flush_chain()                        # (what waits in the chain may be what is read here)
    w, w_scales = weight
    values = scales = residual = gain = kept = None
    eps = 0.0
    if isinstance(x, Int8Rows):
        src, (values, scales) = None, x
    elif not isinstance(x, ops.PendingNorm):
        src = x
    elif x.rows is None:
        src, residual, gain, kept, eps = x.x, x.residual, x.weight, x.residual_out, x.eps
    else:
        src = x.materialize()                    # (the norm's own kernel picks rows)
    lib = _lib(glu)
    if src is not None and w.is_cuda:
        if _byte_product is None:
            _byte_product = load_call_binding().byte_product
        got = _byte_product(lib.b200_int8_linear, lib.b200_int8_alone, src, w, w_scales, residual, gain, kept, bias, out_dtype, mode,
                            eps, float(limit), float(alpha), ops.error_word(w.device), ops._stream())
        if got is not None:
            out, rc, kernels = got
            ops._ok(rc, "int8_linear", kernels)
            return out
    # Rows that are in 8 bits already, a layer's calls that are being kept, nothing to do, or something that is not as it should be.
    _check_8_bit(weight, "weights")
    if src is None:
        _check_8_bit(x, "rows")
        tokens, k = values.shape
        pitch, out_dtype, x_pitch, x_code = values.stride(0), out_dtype or torch.bfloat16, 0, 0
    else:
        _source(x if gain is not None else src)
        tokens, k = src.shape
        pitch, out_dtype, x_pitch, x_code = row_pitch(k), out_dtype or src.dtype, src.stride(0) if tokens > 1 else k, ops._code(src)
    _check_k(k)
    rows = n = w.shape[0]
    if w.shape[1] != k:
        raise KernelError(f"the rows have {k} columns, the weight has {w.shape[1]}")
    if mode == _GLU:
        if rows % 2:
            raise KernelError("gate and up rows of a gated product are as many")
        n = rows // 2
    if bias is not None and (bias.dtype != torch.float32 or bias.numel() != rows or not bias.is_contiguous()):
        raise KernelError("the bias is float32, one element an output channel")
    if out_dtype not in ops._CODES:
        raise KernelError(f"dtype {out_dtype} is not supported (float32 and bfloat16 are)")
    ops._cuda(src, residual, gain, kept, values, scales, w, w_scales, bias)
    out = ops._empty((tokens, n), out_dtype, w.device)
    if values is None:
        # the tokens in 8 bits and their scales, between the two kernels of the call
        values = ops._empty((tokens * pitch + 4 * tokens,), torch.int8, w.device)
        scales = values.data_ptr() + tokens * pitch
    rc = lib.b200_int8_linear(src, residual, gain, kept, values, scales, w, w_scales, bias, out, tokens, n, k, x_pitch, pitch, w.stride(0),
                              x_code, 0 if gain is None else ops._code(gain), ops._code(out), mode, eps, float(limit), float(alpha),
                              ops.error_word(w.device), ops._stream())
    both = src is not None and n and not lib.b200_int8_alone(tokens, k)
    ops._ok(rc, "int8_linear", 0 if not tokens else 2 if both else int(src is not None or n > 0))
    return out


def int8_linear(x, weight: Int8Weight, bias: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """x . w^T (+ bias) in 8-bit integers.  ``x``: [T, K] bfloat16 or float32 (rows any distance apart), an ``ops.PendingNorm``
    (the residual add and the norm run here and ``residual_out`` is filled) or ``Int8Rows``.  ``out_dtype``: x's unless given
    (``Int8Rows``: bfloat16)."""
    return _product(x, weight, bias, out_dtype, _PLAIN, "silu", 0.0, 1.0)


def int8_glu(x, weight: Int8Weight, glu: str = "silu", limit: float = 0.0, alpha: float = 1.0, bias: Optional[torch.Tensor] = None,
             out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """act(x . gate^T) * (x . up^T) in 8-bit integers, weight = [gate rows; up rows] (``glu``, ``limit``, ``alpha``: the forms of
    ``ops.glu_columns``).  The gate acts on the float sums; the result alone is rounded.  ``x`` as in ``int8_linear``."""
    return _product(x, weight, bias, out_dtype, _GLU, glu, limit, alpha)
