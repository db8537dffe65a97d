"""Rotary positions with several axes: the embedding of a DiT's image and video tokens (time, height, width
of a latent grid) and of text tokens that share a sequence with them, straight from the positions.

``RotaryEmbedding`` says where the tokens are and which frequencies their pairs turn with;
``rotary_embed`` rotates queries and keys ``[B, heads, s, D]`` by it in one launch, and
``attention_from_projections`` / ``qk_norm_rope_heads`` take it in place of cos/sin tables.  It stands for the
position tables that the reference's models build and slice per rank and the ``apply_rotary_emb`` of its processors
(``transformer_wan.py:106-122, 311-319``).  Forward only, like everything in this package.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass
from functools import lru_cache
from typing import Optional, Sequence, Tuple

import torch

from . import _capi, ops


@lru_cache(maxsize=64)
def _pairs(axes_dim: Tuple[int, ...], theta: float, ladder: str, frequencies: Optional[Tuple[float, ...]]):
    """``(frequencies, axis, pairs)``: ctypes pointers to every rotated pair's frequency (radians at position one) and
    axis (they keep their arrays alive)."""
    if not 1 <= len(axes_dim) <= _capi.XDIT_ROTARY_MAX_AXES or any(d < 0 or d % 2 for d in axes_dim):
        raise ValueError(f"axes_dim {axes_dim}: 1 to {_capi.XDIT_ROTARY_MAX_AXES} even numbers of elements")
    n = sum(axes_dim) // 2
    if not 1 <= n <= _capi.XDIT_ROTARY_MAX_PAIRS:
        raise ValueError(f"axes_dim {axes_dim}: 2 to {2 * _capi.XDIT_ROTARY_MAX_PAIRS} elements may be rotated")
    axis = [a for a, d in enumerate(axes_dim) for _ in range(d // 2)]
    if frequencies is not None:
        freq = frequencies
        if len(freq) != n:
            raise ValueError(f"{len(freq)} frequencies for {n} pairs")
    elif ladder == "axis":
        freq = [theta ** (-2.0 * i / d) for d in axes_dim for i in range(d // 2)]
    elif ladder == "shared":
        freq = [theta ** (-float(i) / n) for i in range(n)]
    else:
        raise ValueError(f"ladder {ladder!r}: 'axis' or 'shared'")
    return (C.cast((C.c_double * n)(*freq), C.POINTER(C.c_double)), C.cast((C.c_uint8 * n)(*axis), C.POINTER(C.c_uint8)), n)


@dataclass(eq=False)
class RotaryEmbedding:
    """Where tokens are, and how far their pairs turn.

    ``axes_dim``: how many elements of a head belong to each axis (the elements behind their sum pass unrotated).
    ``positions``: ids of the tokens, int32, int64 or fp32, ``[s, axes]`` or ``[B, s, axes]``; or ``grid``: the sides of the
    latent grid, e.g. ``(frames, height, width)``, which the tokens walk row by row from token ``start`` on (a
    sequence-parallel rank passes its first token; tokens behind the grid, the padding of a shard, are not rotated).
    ``ladder``: ``"axis"`` gives each axis frequencies of its own, ``theta ** (-2i / axes_dim[a])``; ``"shared"`` cuts one
    ladder ``theta ** (-2i / sum(axes_dim))`` into the axes.  ``frequencies``: one value per pair instead.
    ``pairing``: ``"interleaved"`` rotates elements ``(2i, 2i+1)``, ``"halves"`` ``(i, i + sum(axes_dim) / 2)``."""

    axes_dim: Tuple[int, ...]
    positions: Optional[torch.Tensor] = None
    grid: Optional[Sequence[int]] = None
    start: int = 0
    theta: float = 10000.0
    ladder: str = "axis"
    frequencies: Optional[Sequence[float]] = None
    pairing: str = "interleaved"

    def _params(self, batch: int, rows: int):
        if self.pairing not in ("interleaved", "halves"):
            raise ValueError(f"pairing {self.pairing!r}: 'interleaved' or 'halves'")
        f = self.frequencies
        freq, axis, pairs = _pairs(tuple(self.axes_dim), self.theta, self.ladder, f if f is None else tuple(map(float, f)))
        return ops.rotary_positions(freq, axis, pairs, len(self.axes_dim), positions=self.positions, grid=self.grid,
                                    start=self.start, batch=batch, rows=rows)

    def _fit(self, batch: int, rows: int, D: int, device) -> Tuple[_capi.RotaryPositions, torch.device]:
        """``(positions, device)`` for ``rows`` tokens of heads of ``D`` on ``device``, or the refusal that a launch would meet."""
        device = torch.device(device)
        if D < sum(self.axes_dim):
            raise ValueError(f"{sum(self.axes_dim)} elements to rotate in a head of {D}")
        if self.positions is not None:
            ops._check_tensors(self.positions)
            at = self.positions.device
            if device.type != at.type or device.index not in (None, at.index):
                raise ValueError(f"positions on {at} for tensors on {device}")
            device = at
        return self._params(batch, rows), device

    def tables(self, s: int, D: int, device) -> Tuple[torch.Tensor, torch.Tensor]:
        """``(cos, sin)``, fp32 ``[s, D]``, as the attention prologue takes them: interleaved pairs, one set of positions for
        all samples."""
        if self.pairing != "interleaved":
            raise ValueError("the attention prologue rotates interleaved pairs")
        positions, device = self._fit(1, s, D, device)
        return ops.rotary_tables(positions, s, D, device)


def rotary_embed(query: torch.Tensor, key: Optional[torch.Tensor], embedding: RotaryEmbedding, *,
                 out_query: Optional[torch.Tensor] = None, out_key: Optional[torch.Tensor] = None
                 ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """``(query, key)`` rotated by ``embedding``.  ``query`` ``[B, H, s, D]`` and ``key`` ``[B, Hk, s, D]`` (or ``None``; its heads may be
    fewer) in bf16, fp16 or fp32, any strides with a contiguous last axis.  The results lie in memory like the inputs, or
    go to ``out_query`` / ``out_key``, which may be the inputs themselves (each its own) but not overlap them in another
    way.  Angles are taken in 64 bits and their cos and sin in 32; a result is rounded once."""
    if torch.compiler.is_compiling() and out_query is None and out_key is None:
        from . import compile_ops

        e = embedding
        got = compile_ops.rotary_axes(query, key, e.positions, list(e.axes_dim), None if e.grid is None else list(e.grid),
                                      e.start, e.theta, e.ladder, None if e.frequencies is None else list(e.frequencies),
                                      e.pairing)
        return got[0], got[1] if key is not None else None
    if query.dim() != 4 or (key is not None and key.dim() != 4):
        raise ValueError("query and key must be [B, heads, s, D]")
    if key is None and out_key is not None:
        raise ValueError("out_key without a key")
    p = embedding._params(query.shape[0], query.shape[2])
    if embedding.positions is not None:
        ops._check_tensors(query, embedding.positions)
    out_query = torch.empty_like(query) if out_query is None else out_query
    if key is not None and out_key is None:
        out_key = torch.empty_like(key)
    ops.rotary_axes(query, key, p, embedding.pairing == "halves", out_query, out_key)
    return out_query, out_key
