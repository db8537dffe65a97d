"""``torch.library`` custom operators over the attention path, so that ``torch.compile`` traces a DiT
block around ``USP`` / ``xFuserLongContextAttention`` as one opaque node instead of breaking the graph at
the ctypes calls (the reference wraps its own non-traceable kernels the same way,
``xfuser/core/distributed/attention_backend.py:383-399``).

* ``xdit_b200::attn``  -- one dense attention call, ``(q, k, v[, joint k, v]) -> (out, lse)``;
* ``xdit_b200::usp``   -- a whole ``USP`` call under the current sequence-parallel state (pack, collectives,
  attention, return exchange), ``(q, k, v[, joint q, k, v]) -> out``.

* ``xdit_b200::rotary_axes``, ``xdit_b200::gated_residual_norm``, ``xdit_b200::fp8_linear`` -- the steps of a block around its
  attention, each a list of what the step makes (e4m3 rows as two tensors, values and scales).

All are functional (they allocate their results) and carry shape-only "fake" implementations for
tracing.  ``xdit_b200.USP``, the ``[B,S,H,D]`` layer and the block's functions route through them while Dynamo is
tracing and call the kernels directly otherwise.
"""
from __future__ import annotations

from typing import List, Optional, Tuple

import torch
from torch.library import custom_op, register_fake

from . import ops


@custom_op("xdit_b200::attn", mutates_args=())
def attn(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, joint_key: Optional[torch.Tensor],
         joint_value: Optional[torch.Tensor], is_causal: bool, scale: float) -> Tuple[torch.Tensor, torch.Tensor]:
    out, lse = ops.attn_fwd(query, key, value, joint_key, joint_value, causal=is_causal,
                            scale=scale if scale > 0 else None, want_lse=True)
    return out, lse


@register_fake("xdit_b200::attn")
def _attn_fake(query, key, value, joint_key, joint_value, is_causal, scale):
    B, H, Sq, D = query.shape
    return (torch.empty((B, H, Sq, D), dtype=query.dtype, device=query.device),
            torch.empty((B, H, Sq), dtype=torch.float32, device=query.device))


@custom_op("xdit_b200::usp", mutates_args=())
def usp(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, joint_query: Optional[torch.Tensor],
        joint_key: Optional[torch.Tensor], joint_value: Optional[torch.Tensor], joint_strategy: str,
        is_causal: bool, scale: float) -> torch.Tensor:
    from . import usp as _usp
    from .distributed import (PROCESS_GROUP, get_ring_parallel_world_size, get_ulysses_parallel_rank,
                              get_ulysses_parallel_world_size)

    out = _usp.usp_native(query, key, value, joint_query, joint_key, joint_value, joint_strategy or None, None,
                          is_causal, scale if scale > 0 else None, get_ulysses_parallel_world_size(),
                          get_ring_parallel_world_size(),
                          get_ulysses_parallel_rank(), PROCESS_GROUP.ULYSSES_PG, PROCESS_GROUP.RING_PG)
    # a custom operator may not return a view of an input; the data path never does, but the result can
    # be a permuted view of a fresh buffer, which is fine
    return out


@register_fake("xdit_b200::usp")
def _usp_fake(query, key, value, joint_query, joint_key, joint_value, joint_strategy, is_causal, scale):
    B, H, s, D = query.shape
    sj = joint_query.shape[2] if joint_query is not None else 0
    return torch.empty((B, H, s + sj, D), dtype=query.dtype, device=query.device)


def _fp8_like(x, rows: int, K: int):
    return (torch.empty((rows, K), dtype=torch.float8_e4m3fn, device=x.device),
            torch.empty((-(-K // 128), rows), dtype=torch.float32, device=x.device).t())


@custom_op("xdit_b200::rotary_axes", mutates_args=())
def rotary_axes(query: torch.Tensor, key: Optional[torch.Tensor], positions: Optional[torch.Tensor], axes_dim: List[int],
                grid: Optional[List[int]], start: int, theta: float, ladder: str, frequencies: Optional[List[float]],
                pairing: str) -> List[torch.Tensor]:
    from .rotary import RotaryEmbedding, rotary_embed

    e = RotaryEmbedding(tuple(axes_dim), positions, grid, start, theta, ladder, frequencies, pairing)
    return [t for t in rotary_embed(query, key, e) if t is not None]


@register_fake("xdit_b200::rotary_axes")
def _rotary_axes_fake(query, key, positions, axes_dim, grid, start, theta, ladder, frequencies, pairing):
    return [torch.empty_like(t) for t in (query, key) if t is not None]


@custom_op("xdit_b200::gated_residual_norm", mutates_args=())
def gated_residual_norm(residual: torch.Tensor, branch: Optional[torch.Tensor], gate: Optional[torch.Tensor],
                        residual_scale: float, post_norm: str, post_weight: Optional[torch.Tensor],
                        post_bias: Optional[torch.Tensor], norm: str, weight: Optional[torch.Tensor],
                        bias: Optional[torch.Tensor], scale: Optional[torch.Tensor], shift: Optional[torch.Tensor],
                        eps: float, quantize: bool) -> List[torch.Tensor]:
    """What the step makes: ``hidden`` where there is a branch, then ``normed``, or e4m3 rows and their scales."""
    from .modulation import gated_residual_norm as step

    hidden, normed = step(residual, branch, gate=gate, residual_scale=residual_scale, post_norm=post_norm or None,
                          post_weight=post_weight, post_bias=post_bias, norm=norm or None, weight=weight, bias=bias,
                          scale=scale, shift=shift, eps=eps, quantize=quantize)
    made = [hidden] if branch is not None else []
    return made + ([] if normed is None else [normed.data, normed.scale] if quantize else [normed])


@register_fake("xdit_b200::gated_residual_norm")
def _gated_residual_norm_fake(residual, branch, gate, residual_scale, post_norm, post_weight, post_bias, norm, weight,
                              bias, scale, shift, eps, quantize):
    made = [torch.empty_like(residual)] if branch is not None else []
    if quantize:
        return made + list(_fp8_like(residual, residual.shape[0] * residual.shape[1], residual.shape[2]))
    return made + ([torch.empty_like(residual)] if norm else [])


@custom_op("xdit_b200::fp8_linear", mutates_args=())
def fp8_linear(x: torch.Tensor, x_scale: Optional[torch.Tensor], weight: torch.Tensor, weight_scale: torch.Tensor,
               bias: Optional[torch.Tensor], activation: str, out_dtype: torch.dtype, quantize_out: bool) -> List[torch.Tensor]:
    """``x``: ``[B, s, K]`` as it is, or e4m3 rows ``[M, K]`` with ``x_scale``.  ``[M, N]``, or e4m3 rows and their scales."""
    from .fp8_linear import Fp8Rows, Fp8Weight
    from .fp8_linear import fp8_linear as layer

    y = layer(x if x_scale is None else Fp8Rows(x, x_scale), Fp8Weight(weight, weight_scale), bias,
              activation=activation or None, out_dtype=out_dtype, quantize_out=quantize_out)
    return [y.data, y.scale] if quantize_out else [y.view(-1, weight.shape[0])]


@register_fake("xdit_b200::fp8_linear")
def _fp8_linear_fake(x, x_scale, weight, weight_scale, bias, activation, out_dtype, quantize_out):
    M = x.shape[0] if x_scale is not None else x.shape[0] * x.shape[1]
    if quantize_out:
        return list(_fp8_like(x, M, weight.shape[0]))
    return [torch.empty((M, weight.shape[0]), dtype=out_dtype, device=x.device)]
