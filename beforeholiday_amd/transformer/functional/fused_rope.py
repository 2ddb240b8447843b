"""RMS norm of query / key heads and rotary position embedding in one pass (kernels/qk_norm_rope.hip).

The reference's transformer has neither (its positions are a learned table,
apex/transformer/testing/standalone_transformer_lm.py:770-900); models that normalise and rotate run it as a
chain of elementwise passes over query and key. Here each is read and written once.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from ..._native import submodule


def rotary_tables(n_positions: int, rotary_dim: int, base: float = 10000.0, device=None,
                  position_scale: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """cos and sin [n_positions, rotary_dim // 2] of the angles position * position_scale * base^(-2 i / rotary_dim),
    computed in fp64 (a far position's angle loses its fraction in fp32) and rounded once to fp32."""
    if rotary_dim < 2 or rotary_dim % 2 or n_positions < 1:
        raise ValueError(f"rotary_tables: need an even rotary_dim and a position, got {rotary_dim}, {n_positions}")
    inv = float(base) ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim)
    ang = (torch.arange(n_positions, dtype=torch.float64, device=device) * position_scale)[:, None] * inv
    return ang.cos().float(), ang.sin().float()


def _rotate(x, cos, sin, interleaved):
    h = cos.size(-1)
    a, b = (x[..., 0:2 * h:2], x[..., 1:2 * h:2]) if interleaved else (x[..., :h], x[..., h:2 * h])
    y, z = a * cos - b * sin, b * cos + a * sin
    yz = torch.stack((y, z), -1).flatten(-2) if interleaved else torch.cat((y, z), -1)
    return torch.cat((yz, x[..., 2 * h:]), -1)


def _qk_norm_rope_torch(q, k, wq, wk, cos, sin, positions, offset, eps, interleaved):
    """The same function in torch operations (CPU tensors)."""
    ct = torch.promote_types(q.dtype, torch.float32)
    if cos is not None:
        if positions is None:
            positions = torch.arange(offset, offset + q.size(0), device=q.device)
        pos = positions.long() if positions.dim() == 2 else positions.long()[:, None]
        ok = (pos >= 0) & (pos < cos.size(0))
        at = pos.clamp(0, cos.size(0) - 1)
        cos, sin = (t[at].masked_fill(~ok[..., None], float("nan"))[:, :, None].to(ct) for t in (cos, sin))
    outs = []
    for x, w in ((q, wq), (k, wk)):
        y = x.to(ct)
        if w is not None:
            y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps) * w.to(ct)
        if cos is not None:
            y = _rotate(y, cos, sin, interleaved)
        outs.append(y.to(x.dtype).contiguous())
    return tuple(outs)


def _check(query, key, query_weight, key_weight, cos, sin, positions, offset):
    for name, t in (("query", query), ("key", key)):
        if t.dim() != 4:
            raise ValueError(f"fused_qk_norm_rope: {name} must be [s, b, heads, head_dim], got {tuple(t.shape)}")
    hn = query.size(3)
    if key.shape[:2] != query.shape[:2] or key.size(3) != hn or key.dtype != query.dtype or key.device != query.device:
        raise ValueError(f"fused_qk_norm_rope: query {tuple(query.shape)} and key {tuple(key.shape)} do not fit")
    if (query_weight is None) != (key_weight is None):
        raise ValueError("fused_qk_norm_rope: give both norm weights or none")
    if (cos is None) != (sin is None):
        raise ValueError("fused_qk_norm_rope: give both angle tables or none")
    if query_weight is None and cos is None:
        raise ValueError("fused_qk_norm_rope: neither norm weights nor angle tables")
    if query_weight is not None:
        for w in (query_weight, key_weight):
            if w.dim() != 1 or w.size(0) != hn or w.dtype != query_weight.dtype or w.device != query.device:
                raise ValueError("fused_qk_norm_rope: norm weights must be [head_dim], of one dtype, on the query's device")
    if cos is not None:
        if cos.dim() != 2 or cos.shape != sin.shape or not 2 <= 2 * cos.size(1) <= hn or \
                cos.dtype != torch.float32 or sin.dtype != torch.float32 or cos.device != query.device or \
                sin.device != query.device:
            raise ValueError("fused_qk_norm_rope: cos / sin must be fp32 [positions, at most head_dim / 2] tables on the "
                             "query's device")
        if positions is not None:
            if tuple(positions.shape) not in ((query.size(0),), tuple(query.shape[:2])) or \
                    positions.dtype not in (torch.int32, torch.int64) or positions.device != query.device:
                raise ValueError("fused_qk_norm_rope: positions must be int32 / int64 [s] or [s, b] on the query's device")
            if offset:
                raise ValueError("fused_qk_norm_rope: an offset goes without positions")
        elif offset < 0 or offset + query.size(0) > cos.size(0):
            raise ValueError(f"fused_qk_norm_rope: positions {offset} .. {offset + query.size(0) - 1} do not fit tables of "
                             f"{cos.size(0)}")


def fused_qk_norm_rope(query: torch.Tensor, key: torch.Tensor, query_weight: Optional[torch.Tensor] = None,
                       key_weight: Optional[torch.Tensor] = None, cos: Optional[torch.Tensor] = None,
                       sin: Optional[torch.Tensor] = None, *, positions: Optional[torch.Tensor] = None, offset: int = 0,
                       eps: float = 1e-6, interleaved: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """RMS-normalises every head of ``query`` [s, b, np, hn] and ``key`` [s, b, ng, hn] over hn, scales it by
    ``query_weight`` / ``key_weight`` [hn], then rotates its first ``2 * cos.size(1)`` values by the angle of its
    position; the rest of the head passes through. Math in fp32, one rounding. Differentiable (once) in query, key and
    the weights.

    Args:
        query, key: fp32 / fp16 / bf16, any strides (head_dim not contiguous: copied), hn even and at most
            512; on the GPU fewer than 2^26 tokens.
        query_weight, key_weight: both or none (no norm); fp32 / fp16 / bf16.
        cos, sin: fp32 [positions, rot / 2] tables (:func:`rotary_tables`), both or none (no rotation). Not
            differentiated.
        positions: integer [s] or [s, b] rows of the tables; one outside them gives NaN in the rotated values.
            Default: offset + 0 .. s - 1, which must fit the tables.
        interleaved: pairs are neighbours (2 i, 2 i + 1); default: (i, i + rot / 2).

    Returns the new query and key, contiguous."""
    offset = int(offset)
    if query.is_cuda:  # the native call checks the operands
        return tuple(submodule("qk_norm_rope").norm_rope(query, key, query_weight, key_weight, cos, sin, positions, offset,
                                                         eps, interleaved))
    _check(query, key, query_weight, key_weight, cos, sin, positions, offset)
    return _qk_norm_rope_torch(query, key, query_weight, key_weight, cos, sin, positions, offset, eps, interleaved)
