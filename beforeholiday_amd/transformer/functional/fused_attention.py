"""Grouped-query attention with a backward pass that recomputes the probabilities.

The reference materialises the [b * heads, sq, sk] scores (apex/transformer/testing/standalone_transformer_lm.py:
309-470, CoreAttention) or is limited to one head size (apex/contrib/fmha). Here scores never leave the chip:
kernels/grouped_attn.hip keeps one number per query (the log-sum of its exponentials) and rebuilds the
probabilities from it in the backward pass.
"""
from __future__ import annotations

from typing import Optional

import torch

from ..._autocast_utils import _cast_if_autocast_enabled
from ..._native import submodule

_M32 = 0xFFFFFFFF


def _signed64(x: int) -> int:
    x &= (1 << 64) - 1
    return x - (1 << 64) if x >= 1 << 63 else x


def _mix32(x):
    x = x ^ (x >> 16)
    x = (x * 0x7FEB352D) & _M32
    x = x ^ (x >> 15)
    x = (x * 0x846CA68B) & _M32
    return x ^ (x >> 16)


def attention_dropout_keep(seed: int, batch_heads: int, sq: int, sk: int, p: float, device=None) -> torch.Tensor:
    """The keep flags [batch_heads, sq, sk] that :func:`fused_grouped_attention` draws for ``seed``: a hash of
    (seed, batch * heads + head, query), then one of (that, key // 2), whose low / high 16 bits decide about the
    even / odd key."""
    seed &= (1 << 64) - 1
    h = (torch.arange(batch_heads, device=device) * 0x9E3779B1)[:, None] & _M32
    q = (torch.arange(sq, device=device) * 0x85EBCA77)[None] & _M32
    row = _mix32((seed & _M32) ^ _mix32((seed >> 32) ^ h ^ q))
    x = (row[..., None] + (torch.arange((sk + 1) // 2, device=device) * 0x9E3779B9)) & _M32
    x = x ^ (x >> 16)
    x = (x * 0x7FEB352D) & _M32
    x = x ^ (x >> 16)
    t = min(65536, int((1.0 - p) * 65536.0))
    return torch.stack(((x & 0xFFFF) < t, (x >> 16) < t), -1).flatten(-2)[..., :sk]


def _attention_torch(q, k, v, lens, causal, window, scale, p, seed):
    """The same function in torch operations (CPU tensors)."""
    sq, b, np_, hn = q.shape
    sk, ng = k.size(0), k.size(2)
    ct = torch.promote_types(q.dtype, torch.float32)
    qf = q.to(ct).permute(1, 2, 0, 3)
    kf, vf = (t.to(ct).permute(1, 2, 0, 3).repeat_interleave(np_ // ng, 1) for t in (k, v))
    i = torch.arange(sq, device=q.device)[:, None] + (sk - sq)
    j = torch.arange(sk, device=q.device)[None]
    see = torch.ones(sq, sk, dtype=torch.bool, device=q.device)
    if causal:
        see = see & (j <= i) & (j > i - window) if window else see & (j <= i)
    see = see.expand(b, 1, sq, sk)
    if lens is not None:
        here = (j < lens.view(-1, 1, 1, 1))
        see = see & here
        vf = vf.masked_fill(~here.transpose(-1, -2), 0.0)  # keys past a length are not read
        kf = kf.masked_fill(~here.transpose(-1, -2), 0.0)
    s = torch.matmul(qf, kf.transpose(-1, -2)) * scale
    s = s.masked_fill(~see, float("-inf"))
    some = see.any(-1, keepdim=True)
    prob = torch.softmax(s.masked_fill(~some, 0.0), -1) * some
    if p > 0:
        keep = attention_dropout_keep(seed, b * np_, sq, sk, p, q.device).view(b, np_, sq, sk)
        prob = prob * keep / (1.0 - p)
    return torch.matmul(prob, vf).permute(2, 0, 1, 3).to(q.dtype).contiguous()


def _check(query, key, value):
    for name, t in (("query", query), ("key", key), ("value", value)):
        if t.dim() != 4:
            raise ValueError(f"fused_grouped_attention: {name} must be [s, b, heads, head_dim], got {tuple(t.shape)}")
    if key.shape != value.shape or key.size(1) != query.size(1) or key.size(3) != query.size(3):
        raise ValueError(f"fused_grouped_attention: query {tuple(query.shape)}, key {tuple(key.shape)} and value "
                         f"{tuple(value.shape)} do not fit")
    if key.size(2) < 1 or query.size(2) < 1 or query.size(2) % key.size(2):
        raise ValueError(f"fused_grouped_attention: {query.size(2)} query heads are no multiple of {key.size(2)} key heads")
    if not query.dtype == key.dtype == value.dtype:
        raise ValueError("fused_grouped_attention: query, key and value must have one dtype")


def fused_grouped_attention(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, *, causal: bool = False,
                            window: Optional[int] = None, key_lengths: Optional[torch.Tensor] = None,
                            dropout_p: float = 0.0, training: bool = True, scale: Optional[float] = None,
                            seed: Optional[int] = None) -> torch.Tensor:
    """softmax(scale Q K^T) V for grouped heads, without the scores in memory. Differentiable in query, key, value
    (once).

    Args:
        query: [sq, b, np, hn]; key, value: [sk, b, ng, hn]. np is a multiple of ng; query head j reads key head
            j // (np / ng). Any strides (views of a fused projection output, transposed batch-first tensors);
            a layout the kernels cannot address is copied (b * heads * hn of 2^24 and more cannot be). On the GPU
            fp16 / bf16, hn a multiple of 8 up to 128, b * heads * ceil(s / 128) below 2^22; on the CPU any floating
            type and head size.
        causal: query i sees keys up to i + sk - sq: the last query is aligned with the last key.
        window: with ``causal``, a query sees at most this many keys, its own position's included.
        key_lengths: int [b]; keys from key_lengths[n] on are not seen and not read (they may hold anything, and
            take zero gradients). Values outside 0 .. sk count as the nearer bound. Alignment of the causal mask
            stays with sk.
        dropout_p: probability of dropping a softmax weight while ``training`` (the rest is scaled by
            1 / (1 - dropout_p)); resolved to 1 / 65536. The mask is a function of ``seed`` and is regenerated in
            the backward pass (:func:`attention_dropout_keep`).
        scale: default hn ** -0.5; in 1e-30 .. 1e30 (the kernels hold it in fp32).
        seed: default: drawn like the other fused attention dropouts (tensor-parallel ranks differ; replayable
            through ``utils.graph_rng``).

    A query that sees no key gives zeros and takes no gradient. Contents that only key_lengths hides are never read; a
    NaN or infinity in a value that the causal mask or the window hides may still reach a query (0 * NaN), as in the
    written-out product. Returns [sq, b, np, hn], contiguous."""
    if window is not None and (not causal or int(window) < 1):
        raise ValueError("fused_grouped_attention: window needs causal=True and must be at least 1")
    if not 0.0 <= dropout_p < 1.0:
        raise ValueError(f"fused_grouped_attention: dropout_p must be in [0, 1), got {dropout_p}")
    scale = float(scale) if scale is not None else query.size(-1) ** -0.5
    if not 1e-30 <= scale <= 1e30:
        raise ValueError(f"fused_grouped_attention: scale must be in [1e-30, 1e30], got {scale}")
    if key_lengths is not None:
        if key_lengths.dim() != 1 or key_lengths.size(0) != query.size(1) or key_lengths.is_floating_point():
            raise ValueError("fused_grouped_attention: key_lengths must be an integer [batch] tensor")
        if key_lengths.device != query.device:
            raise ValueError("fused_grouped_attention: key_lengths must be on the query's device")
    query, key, value = _cast_if_autocast_enabled(query, key, value)
    p = float(dropout_p) if training else 0.0
    seed_dev = None
    if p > 0 and seed is None:
        from ...contrib.multihead_attn._core import _seed_pair

        seed, seed_dev = _seed_pair()
    seed = _signed64(int(seed)) if p > 0 else 0
    window = 0 if window is None else int(window)
    if query.is_cuda:  # the native call checks the operands
        if key_lengths is not None:
            if key_lengths.dtype != torch.int32:
                key_lengths = key_lengths.clamp(0, key.size(0)).to(torch.int32)
            key_lengths = key_lengths.contiguous()
        return submodule("grouped_attention").attention(query, key, value, key_lengths, causal, window, scale, p, seed,
                                                        seed_dev)
    _check(query, key, value)
    lens = None if key_lengths is None else key_lengths.clamp(0, key.size(0))
    return _attention_torch(query, key, value, lens, causal, window, scale, p, seed)
