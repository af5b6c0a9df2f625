"""The 8-bit linear ops around the attention layer.

* ``fused_add_rms_norm_quant``: the RMSNorm in front of a projection, with the
  residual's addition, written as 8-bit codes and scales;
* ``fused_silu_mul_quant``: the gated activation of a feed-forward block,
  written the same way;
* ``int8_scaled_mm``: the product of int8 codes under a scale per token and per
  channel.

``dtype=torch.int8`` gives one scale per token (``[T, 1]``), what
``int8_scaled_mm`` takes as ``scale_a``; ``dtype=torch.float8_e4m3fn`` one scale
per 128 columns (``[T, size / 128]``), what ``fp8_einsum`` takes as ``xs`` with
one head: ``fp8_einsum("bhr,hdr->bhd", codes[:, None], scales[:, None], y, ys)``.
A layer with int8 weights runs::

    x8, xs, hidden = fused_add_rms_norm_quant(x, hidden, norm_weight, eps)
    gate_up = int8_scaled_mm(x8, w_gate_up, xs, s_gate_up)
    y8, ys = fused_silu_mul_quant(gate_up)
    x = int8_scaled_mm(y8, w_down, ys, s_down)

The argument checks, output allocation and launch run in C++
(``torch_ops.cpp``) through the C ABI ``fgv_add_rms_norm_quant``,
``fgv_silu_mul_quant`` and ``fgv_int8_scaled_mm``, on torch's current stream of
the tensors' device; a failed check raises AssertionError.  Inference only: a
tensor that requires a gradient (in grad mode) or carries a forward-mode tangent
is refused, and so are lazily negated views and tensors without memory.
"""
from typing import Optional, Tuple

import torch

from .. import _native


def _is_int8(dtype: torch.dtype, what: str) -> bool:
    if dtype is not torch.int8 and dtype is not torch.float8_e4m3fn:
        raise AssertionError(f"{what}: dtype must be torch.int8 or torch.float8_e4m3fn")
    return dtype is torch.int8


def fused_add_rms_norm_quant(
    x: torch.Tensor,
    residual: Optional[torch.Tensor],
    weight: torch.Tensor,
    eps: float,
    dtype: torch.dtype = torch.int8,
    *,
    hidden_out: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``h = x + residual`` and the codes and scales of ``RMSNorm(h) * weight``.

    Args:
        x: [T, size] bfloat16 or float16, contiguous rows of any row stride.
        residual: like x, or None (then h is x).
        weight: [size], of x's type or float32.
        eps: added to the mean of h^2, positive and finite.
        dtype: torch.int8 (a scale per token) or torch.float8_e4m3fn (a scale
            per 128 columns; size a multiple of 128).  size is at most 65536.
        hidden_out: where h is written (x or residual itself, or a tensor apart
            from the inputs); a new tensor if not given.

    Returns:
        codes [T, size] of dtype; scales [T, 1] or [T, size / 128] float32; h
        rounded to x's type (x itself when there is no residual).  The codes
        are the nearest ones to h * weight over the scale, ties to even,
        computed as in 64 bits.  A row (block of 128) of zeros has scale 0; a
        row that holds a NaN or an infinity has NaN scales, and under a
        largest magnitude that is not finite the codes are 0.
    """
    rc, codes, scales, hidden = _native.torch_ext().add_rms_norm_quant(
        x, residual, weight, eps, _is_int8(dtype, "fused_add_rms_norm_quant"), hidden_out)
    if rc:
        _native.raise_status(rc, "fused_add_rms_norm_quant")
    return codes, scales, hidden


def fused_silu_mul_quant(x: torch.Tensor, dtype: torch.dtype = torch.int8) -> Tuple[torch.Tensor, torch.Tensor]:
    """The codes and scales of ``silu(gate) * up``, ``x = [gate | up]``.

    Args:
        x: [T, 2 * size] bfloat16 or float16, contiguous rows of any row stride.
        dtype: as in ``fused_add_rms_norm_quant``.

    Returns:
        codes [T, size] of dtype; scales [T, 1] or [T, size / 128] float32.
    """
    rc, codes, scales = _native.torch_ext().silu_mul_quant(x, _is_int8(dtype, "fused_silu_mul_quant"))
    if rc:
        _native.raise_status(rc, "fused_silu_mul_quant")
    return codes, scales


def int8_scaled_mm(
    a: torch.Tensor,
    b: torch.Tensor,
    scale_a: torch.Tensor,
    scale_b: torch.Tensor,
    bias: Optional[torch.Tensor] = None,
    out_dtype: torch.dtype = torch.bfloat16,
    *,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """``out[m, n] = scale_a[m] * scale_b[n] * sum_k a[m, k] * b[n, k] + bias[n]``.

    Args:
        a: [M, K] int8, contiguous rows; K at most 131071, M at most 2^20, N at most 2^24.
        b: [N, K] int8, contiguous rows (the weight, a channel a row).
        scale_a: float32 [M], [M, 1] or one scale.
        scale_b: float32 [N], [N, 1], [1, N] or one scale.
        bias: [N], float32 or of out_dtype.
        out_dtype: bfloat16, float16 or float32.
        out: [M, N] of out_dtype to write into, contiguous rows, apart from the
            inputs; a new tensor if not given.

    The sum is exact; the scales and the bias are applied in float32, in that
    order, and the result is rounded once.
    """
    rc, result = _native.torch_ext().int8_mm(a, b, scale_a, scale_b, bias, out_dtype, out)
    if rc:
        _native.raise_status(rc, "int8_scaled_mm")
    return result


__all__ = ["fused_add_rms_norm_quant", "fused_silu_mul_quant", "int8_scaled_mm"]
