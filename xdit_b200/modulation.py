"""What a DiT block does between two sub-layers, in one pass over the hidden states: the gated residual of the
sub-layer that just ended and the modulated norm of the one that follows.

It stands for ``hidden = hidden + gate * attn_output; normed = norm(hidden) * (1 + scale) + shift`` in the blocks that
the reference's wrappers run, for blocks with a second norm behind the sub-layer, and for the modulated norm alone.
Forward only, like everything in this package.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from . import ops
from .fp8_linear import Fp8Rows


def gated_residual_norm(residual: torch.Tensor, branch: Optional[torch.Tensor] = None, *,
                        gate: Optional[torch.Tensor] = None, residual_scale: float = 1.0,
                        post_norm: Optional[str] = None, post_weight: Optional[torch.Tensor] = None,
                        post_bias: Optional[torch.Tensor] = None, norm: Optional[str] = "layer",
                        weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                        scale: Optional[torch.Tensor] = None, shift: Optional[torch.Tensor] = None, eps: float = 1e-6,
                        quantize: bool = False, out_residual: Optional[torch.Tensor] = None
                        ) -> Tuple[torch.Tensor, Union[torch.Tensor, Fp8Rows, None]]:
    """``hidden = residual_scale * residual + gate * post_norm(branch)`` and ``normed = norm(hidden) * (1 + scale) + shift``;
    returns ``(hidden, normed)``.

    ``residual`` and ``branch``: ``[B, s, C]`` in bf16, fp16 or fp32, contiguous last axis, C up to 16384.  Without a branch
    ``hidden`` is ``residual`` itself, whatever ``residual_scale``.  ``norm`` and ``post_norm``: ``"layer"``, ``"rms"`` or ``None``
    (``norm=None``: ``normed`` is ``None``), each with an optional ``weight`` and ``bias`` ``[C]``.  ``gate``, ``scale`` and ``shift``: ``[C]``, ``[B, C]``, ``[B, 1, C]`` or,
    for each token, ``[B, s, C]``.  Rows of parameters are in the tensors' dtype or fp32.  ``hidden`` is summed in fp32,
    rounded once where it is written, and ``norm`` takes the unrounded sum; ``out_residual`` (``residual`` or ``branch``
    itself, for an update in place; it must not overlap an input in another way) receives it.  With ``quantize`` ``normed`` is
    an :class:`~xdit_b200.fp8_linear.Fp8Rows` for the 8-bit projection that follows (C a multiple of 16, and all
    rows, those of modulation too, on 16-byte boundaries)."""
    if residual.dim() != 3:
        raise ValueError("expected [B, s, C]")
    if torch.compiler.is_compiling() and out_residual is None:
        from . import compile_ops

        made = list(compile_ops.gated_residual_norm(residual, branch, gate, float(residual_scale), post_norm or "",
                                                    post_weight, post_bias, norm or "", weight, bias, scale, shift,
                                                    float(eps), quantize))
        hidden = made.pop(0) if branch is not None else residual
        return hidden, Fp8Rows(*made, tuple(residual.shape[:2])) if quantize else made[0] if made else None
    if quantize and (norm is None or residual.shape[2] % 16):
        raise ValueError("quantize needs a norm and rows of a multiple of 16 values")
    if branch is None and out_residual is not None:
        raise ValueError("out_residual needs a branch")
    hidden = residual
    if branch is not None:
        hidden = out_residual if out_residual is not None else torch.empty_like(residual)
    normed = data = scales = None
    if quantize:
        data, scales = ops.empty_fp8_rows(residual.shape[0] * residual.shape[1], residual.shape[2], residual.device)
    elif norm is not None:
        normed = torch.empty_like(residual)
    if branch is None and norm is None:
        raise ValueError("nothing to do without a branch and a norm")
    ops.gated_residual_norm(residual, branch, out_residual=hidden if branch is not None else None, out=normed,
                            out_q=data, out_scale=scales, gate=gate, residual_scale=residual_scale,
                            post_norm=post_norm, post_weight=post_weight, post_bias=post_bias, norm=norm,
                            weight=weight, bias=bias, scale=scale, shift=shift, eps=eps)
    if quantize:
        normed = Fp8Rows(data, scales, tuple(residual.shape[:2]))
    return hidden, normed
