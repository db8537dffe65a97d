"""Linear layers in 8-bit floating point: e4m3 operands with one fp32 scale for each block of 128 along the inner
axis (of every row of the activations, of every 128 rows of the weight), fp32 sums, bias and GELU in the
epilogue, the result in 16 or 32 bits or as e4m3 rows for the next layer.

The projections around the attention are the reference's fp8 linears (``xfuser/model_executor/layers/fp8_linear.py``);
weights come from :func:`quantize_weight` or from a checkpoint with block scales.  Forward only, like everything in
this package.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Tuple, Union

import torch

from . import ops


@dataclass(frozen=True)
class Fp8Rows:
    """Activations in e4m3: ``data`` ``[rows, K]`` and fp32 ``scale`` ``[rows, ceil(K/128)]``; row ``r`` stands for
    ``data[r, k] * scale[r, k // 128]``.  ``lead``: the leading axes that ``rows`` flattens (``(rows,)`` when ``None``)."""

    data: torch.Tensor
    scale: torch.Tensor
    lead: Optional[Tuple[int, ...]] = None

    @property
    def shape(self) -> Tuple[int, ...]:
        return (self.lead if self.lead is not None else (self.data.shape[0],)) + (self.data.shape[1],)


@dataclass(frozen=True)
class Fp8Weight:
    """A weight in e4m3: ``data`` ``[N, K]`` and fp32 ``scale`` ``[ceil(N/128), ceil(K/128)]`` of any values."""

    data: torch.Tensor
    scale: torch.Tensor


def quantize_rows(x: torch.Tensor) -> Fp8Rows:
    """``x`` ``[..., K]`` (bf16, fp16 or fp32; K a multiple of 16, rows on 16-byte boundaries) as e4m3 rows.  A block's scale
    is the smallest power of two that brings its values within 448, so a value is rounded once; a block with an infinity
    or a NaN gets the scale NaN, and so does every result computed from it."""
    rows = x if x.dim() == 3 else x.unsqueeze(0) if x.dim() == 2 else x.reshape(1, -1, x.shape[-1])
    data, scale = ops.quantize_rows(rows)
    return Fp8Rows(data, scale, tuple(x.shape[:-1]))


def quantize_weight(weight: torch.Tensor) -> Fp8Weight:
    """``weight`` ``[N, K]`` as an e4m3 weight with a power-of-two scale for each block of 128 x 128."""
    return Fp8Weight(*ops.quantize_weight(weight))


def fp8_linear(x: Union[torch.Tensor, Fp8Rows], weight: Fp8Weight, bias: Optional[torch.Tensor] = None, *,
               activation: Optional[str] = None, out_dtype: Optional[torch.dtype] = None,
               quantize_out: bool = False) -> Union[torch.Tensor, Fp8Rows]:
    """``activation(x @ weight.T + bias)`` -> ``[..., N]``.

    ``x``: a tensor ``[..., K]``, quantised by the rule of :func:`quantize_rows` (rows on 16-byte boundaries), or
    :class:`Fp8Rows` with scales of any value.  ``activation``: ``None`` or ``"gelu_tanh"``.  ``out_dtype``: bf16, fp16 or fp32 (the dtype of ``x`` when it is a tensor, else
    bf16).  ``quantize_out``: the result as :class:`Fp8Rows` (N a multiple of 16), quantised from the fp32 sums.  The sums of
    a block of 128 run in the tensor cores in fp32, their scaled sum in fp32 registers; the product of two scales is taken in
    fp32 too and has to be within its range."""
    w, ws = weight.data, weight.scale
    if isinstance(x, torch.Tensor):
        out_dtype = x.dtype if out_dtype is None else out_dtype
        lead = x.shape[:-1]
        data, scale = x if x.dim() == 3 else x.unsqueeze(0) if x.dim() == 2 else x.reshape(1, -1, x.shape[-1]), None
        M = data.shape[0] * data.shape[1]
    else:
        out_dtype = torch.bfloat16 if out_dtype is None else out_dtype
        lead, data, scale = x.shape[:-1], x.data, x.scale
        M = data.shape[0]
    if torch.compiler.is_compiling():
        from . import compile_ops

        made = compile_ops.fp8_linear(data, scale, w, ws, bias, activation or "", out_dtype, quantize_out)
        return Fp8Rows(made[0], made[1], tuple(lead)) if quantize_out else made[0].view(*lead, w.shape[0])
    if quantize_out:
        q, s = ops.empty_fp8_rows(M, w.shape[0], data.device)
        ops.fp8_linear(data, scale, w, ws, bias, activation=activation, out_q=q, out_scale=s)
        return Fp8Rows(q, s, tuple(lead))
    out = torch.empty(M, w.shape[0], dtype=out_dtype, device=data.device)
    ops.fp8_linear(data, scale, w, ws, bias, activation=activation, out=out)
    return out if len(lead) == 1 else out.view(*lead, w.shape[0])
