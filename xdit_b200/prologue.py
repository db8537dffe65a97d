"""The slice of a DiT attention processor that sits between the q/k/v projections and the output
projection, as one call: RMSNorm(q, k) + rotary embedding + head split + Ulysses pack in a single
kernel, the all-to-all, the attention kernel on the receive buffer, the output all-to-all and the
head merge.

It stands for these lines of the reference's processors::

    query = attn.norm_q(query); key = attn.norm_k(key)            # transformer_wan.py:99-100
    query = query.unflatten(2, (attn.heads, -1)) ...               # :102-104
    query = apply_rotary_emb(query, *rotary_emb) ...               # :106-122
    hidden_states = USP(query.transpose(1, 2), ...).transpose(1, 2)  # :143-150
    hidden_states = hidden_states.flatten(2, 3)                    # :151

(the same steps with a per-head norm in ``transformer_flux.py:113-147,170-219``).  The norm modules
and Flux's rotary helper come from diffusers, which the reference does not vendor: the norm is
``torch.nn.RMSNorm`` semantics, the rotary embedding is the interleaved-pair form that the Wan
processor defines inline.  In place of cos/sin tables every function here takes a
:class:`~xdit_b200.rotary.RotaryEmbedding`, and :func:`attention_from_hidden_states` starts and ends one step further out, with
projections in 8-bit floating point.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
import torch.distributed as dist

from . import ops
from . import usp as _usp
from .distributed import (PROCESS_GROUP, get_ring_parallel_world_size, get_ulysses_parallel_rank,
                          get_ulysses_parallel_world_size)
from .fp8_linear import Fp8Rows, Fp8Weight, fp8_linear
from .rotary import RotaryEmbedding, rotary_embed


def qk_norm_rope_heads(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, heads: int, *,
                       norm_q_weight: Optional[torch.Tensor] = None, norm_k_weight: Optional[torch.Tensor] = None,
                       eps: float = 1e-6, norm_per_head: bool = False,
                       rotary_emb: Union[RotaryEmbedding, Tuple[torch.Tensor, torch.Tensor], None] = None
                       ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Projections ``[B, s, heads*D]`` -> normalised, rotated ``q, k`` and ``v`` as ``[B, heads, s, D]``
    tensors (what the processor passes to ``USP``).  One launch; for ``B > 1`` the results are
    ``[heads, B, s, D]`` buffers viewed with the batch axis first."""
    B, s, HD = query.shape
    D = HD // heads
    cos, sin, late = _rotary(rotary_emb, B, s, D, query.device)
    n = heads * B * s * D
    buf = torch.empty(3 * n, dtype=query.dtype, device=query.device)
    ops.qk_norm_rope_pack(query, key, value, heads, buf, buf[n:], buf[2 * n:], (n, n, n), 1,
                          norm_q_weight=norm_q_weight, norm_k_weight=norm_k_weight, eps=eps,
                          norm_per_head=norm_per_head, cos=cos, sin=sin)
    q, k, v = (buf[i * n:(i + 1) * n].view(heads, B, s, D).permute(1, 0, 2, 3) for i in range(3))
    if late is not None:
        rotary_embed(q, k, late, out_query=q, out_key=k)
    return q, k, v


def _rotary(rotary_emb, B, s, D, device):
    """``(cos, sin, late)``: the tables of the prologue kernel, which rotates interleaved pairs by one set of positions for
    all samples, or the embedding that is applied behind it (halves, positions of each sample's own)."""
    if isinstance(rotary_emb, RotaryEmbedding):
        p = rotary_emb.positions
        if rotary_emb.pairing != "interleaved" or (B > 1 and p is not None and p.dim() == 3 and p.shape[0] > 1):
            rotary_emb._fit(B, s, D, device)  # what does not fit is refused before anything is written
            return None, None, rotary_emb
        return (*rotary_emb.tables(s, D, device), None)
    return (*_cos_sin(rotary_emb, s, D), None)


def _cos_sin(rotary_emb, s, D):
    if rotary_emb is None:
        return None, None
    cos, sin = rotary_emb
    # the processors carry [1, s, 1, D] tables (transformer_wan.py:108-120); [s, D] is accepted as well
    cos = cos.reshape(s, D) if cos.numel() == s * D else cos
    sin = sin.reshape(s, D) if sin.numel() == s * D else sin
    if cos.shape != (s, D) or sin.shape != (s, D):
        raise ValueError("rotary_emb must hold cos and sin tables of s x D elements")
    return cos.float().contiguous(), sin.float().contiguous()


def attention_from_projections(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, heads: int, *,
                               norm_q_weight: Optional[torch.Tensor] = None,
                               norm_k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                               norm_per_head: bool = False,
                               rotary_emb: Union[RotaryEmbedding, Tuple[torch.Tensor, torch.Tensor], None] = None,
                               softmax_scale: Optional[float] = None,
                               out_proj_weight: Union[torch.Tensor, Fp8Weight, None] = None,
                               out_proj_bias: Optional[torch.Tensor] = None, attn_layer=None) -> torch.Tensor:
    """Self-attention of one DiT layer from its q/k/v projections ``[B, s_local, heads*D]`` to the
    tensor the output projection takes, ``[B, s_local, heads*D]``, under the current sequence-parallel
    degrees.  With a Ulysses degree ``U > 1`` and no ring the prologue kernel writes straight into the
    all-to-all send buffer; otherwise it produces ``[B, heads, s, D]`` tensors for ``USP``'s data path.

    With ``out_proj_weight`` (``[hidden, heads*D]`` or an ``Fp8Weight`` of it, optional bias) the layer's output projection
    (``attn.to_out[0]``, ``transformer_wan.py:152``, ``transformer_flux.py:210-219``) is applied as well and
    ``[B, s_local, hidden]`` is returned: the attention kernel writes its rows head-merged, so the
    projection reads them where they lie.

    ``attn_layer`` (PipeFusion, no sequence parallelism): the layer's stale-KV buffers are the attention's
    keys and values, and the prologue kernel writes the fresh K and V rows of the current patch straight
    into them -- no separate patch-update pass (``attention_processor.py:286-292`` ->
    ``cache_manager.py:103-135``)."""
    if attn_layer is not None:
        out = _attention_with_stale_kv(query, key, value, heads, norm_q_weight, norm_k_weight, eps, norm_per_head,
                                       rotary_emb, softmax_scale, attn_layer)
        return _project(out, out_proj_weight, out_proj_bias)
    out = _attention_from_projections(query, key, value, heads, norm_q_weight, norm_k_weight, eps, norm_per_head,
                                      rotary_emb, softmax_scale)
    return _project(out, out_proj_weight, out_proj_bias)


def _project(x, weight, bias, out_dtype=None):
    if weight is None:
        return x
    if isinstance(weight, Fp8Weight):
        return fp8_linear(x, weight, bias, out_dtype=out_dtype)
    return torch.nn.functional.linear(x, weight, bias)


def attention_from_hidden_states(hidden_states: Union[torch.Tensor, Fp8Rows], qkv_weight: Union[torch.Tensor, Fp8Weight],
                                 heads: int, *, qkv_bias: Optional[torch.Tensor] = None,
                                 out_proj_weight: Union[torch.Tensor, Fp8Weight, None] = None,
                                 out_proj_bias: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.bfloat16,
                                 **kwargs) -> torch.Tensor:
    """Self-attention of one DiT layer from its (normed) hidden states ``[B, s_local, hidden]``: the fused q, k, v projection
    ``qkv_weight`` ``[3 * heads*D, hidden]``, :func:`attention_from_projections` with ``kwargs`` on its three column slices, and the
    output projection where one is given.  A weight may be an :class:`~xdit_b200.fp8_linear.Fp8Weight`; ``hidden_states`` may then
    be the :class:`~xdit_b200.fp8_linear.Fp8Rows` that ``gated_residual_norm(quantize=True)`` makes, and ``dtype`` is the type that
    the attention runs in.  Forward only: tensors that record a gradient are refused."""
    given = (hidden_states, qkv_weight, qkv_bias, out_proj_weight, out_proj_bias, *kwargs.values())
    ops._refuse_gradient(*(t for t in given if isinstance(t, torch.Tensor)))
    if isinstance(hidden_states, Fp8Rows):
        if not isinstance(qkv_weight, Fp8Weight):
            raise TypeError("e4m3 hidden states need an Fp8Weight as qkv_weight")
    else:
        dtype = hidden_states.dtype
    qkv = _project(hidden_states, qkv_weight, qkv_bias, dtype)
    if qkv.dim() != 3 or qkv.shape[2] % (3 * heads):
        raise ValueError(f"expected [B, s, hidden] and a weight of 3 x {heads} heads, got a projection {tuple(qkv.shape)}")
    query, key, value = qkv.chunk(3, dim=2)
    return attention_from_projections(query, key, value, heads, out_proj_weight=out_proj_weight,
                                      out_proj_bias=out_proj_bias, **kwargs)


def _attention_with_stale_kv(query, key, value, heads, norm_q_weight, norm_k_weight, eps, norm_per_head, rotary_emb,
                             softmax_scale, attn_layer):
    from .cache_manager import get_cache_manager

    if get_ulysses_parallel_world_size() * get_ring_parallel_world_size() != 1:
        raise NotImplementedError("the fused stale-KV path serves PipeFusion without sequence parallelism; "
                                  "use USP(..., attn_layer=...) otherwise")
    B, n, HD = query.shape
    D = HD // heads
    cos, sin, late = _rotary(rotary_emb, B, n, D, query.device)
    kc, vc, start = get_cache_manager().rows_for_producer(attn_layer, B, heads, n, D, query.dtype, query.device)
    S = kc.shape[2]
    q_buf = torch.empty(heads * B * n * D, dtype=query.dtype, device=query.device)
    # q in the packed [H][B][n][D] layout; k and v rows at [start, start + n) of the [B,H,S,D] buffers
    ops.qk_norm_rope_pack(query, key, value, heads, q_buf, kc.view(-1)[start * D:], vc.view(-1)[start * D:],
                          (q_buf.numel(), 0, 0), 1, norm_q_weight=norm_q_weight, norm_k_weight=norm_k_weight, eps=eps,
                          norm_per_head=norm_per_head, cos=cos, sin=sin,
                          dst_strides=[None, (S * D, heads * S * D), (S * D, heads * S * D)])
    q4 = q_buf.view(heads, B, n, D).permute(1, 0, 2, 3)
    if late is not None:
        k_new = kc[:, :, start:start + n]
        rotary_embed(q4, k_new, late, out_query=q4, out_key=k_new)
    out = torch.empty(B, n, heads, D, dtype=query.dtype, device=query.device)
    ops.attn_fwd(q4, kc, vc, out=out.permute(0, 2, 1, 3), scale=softmax_scale)
    return out.view(B, n, HD)


def _attention_from_projections(query, key, value, heads, norm_q_weight, norm_k_weight, eps, norm_per_head,
                                rotary_emb, softmax_scale):
    B, s, HD = query.shape
    if HD % heads:
        raise ValueError("hidden size must be divisible by the number of heads")
    D = HD // heads
    U, R = get_ulysses_parallel_world_size(), get_ring_parallel_world_size()
    if U == 1 and R == 1:
        # one GPU: the attention kernel writes its rows straight into [B, s, heads, D], which is the
        # head-merged tensor the output projection takes
        q, k, v = qk_norm_rope_heads(query, key, value, heads, norm_q_weight=norm_q_weight,
                                     norm_k_weight=norm_k_weight, eps=eps, norm_per_head=norm_per_head,
                                     rotary_emb=rotary_emb)
        out = torch.empty(B, s, heads, D, dtype=query.dtype, device=query.device)
        ops.attn_fwd(q, k, v, out=out.permute(0, 2, 1, 3), scale=softmax_scale)
        return out.view(B, s, HD)
    if U == 1 or R > 1:
        q, k, v = qk_norm_rope_heads(query, key, value, heads, norm_q_weight=norm_q_weight,
                                     norm_k_weight=norm_k_weight, eps=eps, norm_per_head=norm_per_head,
                                     rotary_emb=rotary_emb)
        out = _usp.usp_native(q, k, v, None, None, None, None, None, False, softmax_scale, U, R,
                              get_ulysses_parallel_rank(), PROCESS_GROUP.ULYSSES_PG, PROCESS_GROUP.RING_PG)
        # [B, heads, s, D] -> [B, s, heads*D]
        return out.permute(0, 2, 1, 3).reshape(B, s, HD)
    assert heads % U == 0, "h must be divisible by world_size, got {} and {}".format(heads, U)
    Hl = heads // U
    cos, sin, late = _rotary(rotary_emb, B, s, D, query.device)
    blk = Hl * B * s * D
    stride = 3 * blk
    send = torch.empty(U * stride, dtype=query.dtype, device=query.device)
    ops.qk_norm_rope_pack(query, key, value, heads, send, send[blk:], send[2 * blk:], (stride, stride, stride), U,
                          norm_q_weight=norm_q_weight, norm_k_weight=norm_k_weight, eps=eps,
                          norm_per_head=norm_per_head, cos=cos, sin=sin)
    for peer in range(U if late is not None else 0):
        q, k = (send.as_strided((B, Hl, s, D), (s * D, B * s * D, D, 1), peer * stride + i * blk) for i in range(2))
        rotary_embed(q, k, late, out_query=q, out_key=k)
    recv = torch.empty_like(send)
    dist.all_to_all_single(recv, send, group=PROCESS_GROUP.ULYSSES_PG)
    shape, strides = (B, Hl, U, s, D), (s * D, B * s * D, stride, D, 1)
    q5 = recv.as_strided(shape, strides, 0)
    k5 = recv.as_strided(shape, strides, blk)
    v5 = recv.as_strided(shape, strides, 2 * blk)
    out_send = torch.empty(U * blk, dtype=query.dtype, device=query.device)
    out5 = out_send.as_strided(shape, (s * D, B * s * D, blk, D, 1), 0)
    ops.attn_fwd(q5, k5, v5, out=out5, scale=softmax_scale)
    out_recv = torch.empty_like(out_send)
    dist.all_to_all_single(out_recv, out_send, group=PROCESS_GROUP.ULYSSES_PG)
    # received [heads][B][s][D] -> [B, s, heads*D]
    return out_recv.view(heads, B, s, D).permute(1, 2, 0, 3).reshape(B, s, HD)
