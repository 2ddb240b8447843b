"""Counter-based dropout: the mask is a function of the seed and never stored (kernels/counter_dropout.hip).

torch's dropout, which the reference's embedding and attention use
(apex/transformer/testing/standalone_transformer_lm.py:840-900), keeps a byte per element for the backward pass; here
the backward pass draws the same mask again from the seed.
"""
from __future__ import annotations

from typing import Optional

import torch

from ..._native import submodule
from .fused_attention import _signed64

_M32 = 0xFFFFFFFF


def _threshold(p: float) -> int:
    return min(_M32, int((1.0 - p) * 4294967296.0))


def dropout_keep(seed: int, n: int, p: float, device=None) -> torch.Tensor:
    """The keep flags [n] that :func:`fused_dropout` draws for ``seed``: element i is kept when word i % 4 of
    Philox4x32-7 (counter i // 4, key ``seed``) is below (1 - p) 2^32."""
    seed &= (1 << 64) - 1
    calls = torch.arange((n + 3) // 4, device=device)
    c0, c1 = calls & _M32, calls >> 32
    c2, c3 = torch.zeros_like(calls), torch.zeros_like(calls)
    k0, k1 = seed & _M32, seed >> 32
    for _ in range(7):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # the low 64 bits are right also where int64 wraps
        c0, c1, c2, c3 = ((p1 >> 32) & _M32) ^ c1 ^ k0, p1 & _M32, ((p0 >> 32) & _M32) ^ c3 ^ k1, p0 & _M32
        k0, k1 = (k0 + 0x9E3779B9) & _M32, (k1 + 0xBB67AE85) & _M32
    return torch.stack((c0, c1, c2, c3), -1).flatten()[:n] < _threshold(p)


class CounterDropoutFn(torch.autograd.Function):
    """x -> keep ? x / (1 - p) : 0 on the CPU; its backward is itself on the gradient (any number of times)."""

    @staticmethod
    def forward(ctx, x, p, seed):
        ctx.args = (p, seed)
        scale = 1.0 / (1.0 - p) if p < 1.0 else 0.0
        keep = dropout_keep(seed, x.numel(), p, x.device).view(x.shape)
        y = x.to(torch.promote_types(x.dtype, torch.float32)) * scale
        return torch.where(keep, y, torch.zeros((), dtype=y.dtype)).to(x.dtype)

    @staticmethod
    def backward(ctx, dy):
        return CounterDropoutFn.apply(dy, *ctx.args), None, None


def fused_dropout(x: torch.Tensor, p: float = 0.5, training: bool = True, *, seed: Optional[int] = None,
                  model_parallel: bool = False) -> torch.Tensor:
    """Drops elements of ``x`` with probability ``p`` and scales the rest by 1 / (1 - p); ``x`` itself when not
    ``training`` or p = 0. A dropped element gives 0 whatever it held.

    The mask depends on ``seed`` and the element's position in ``x`` (row-major over its shape), not on strides, dtype
    or device. ``seed`` defaults to the next one of the dropout seed stream that ``bias_dropout_add`` uses:
    replicated over tensor-parallel ranks, or (``model_parallel=True``: sequence-parallel shards) one of this rank's
    own; with ``utils.graph_rng`` enabled a captured step draws a new mask on every replay.

    On the GPU fp32 / fp16 / bf16; on the CPU any floating type."""
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"fused_dropout: p must be in [0, 1], got {p}")
    if not x.is_floating_point() or (x.is_cuda and x.dtype not in (torch.float32, torch.float16, torch.bfloat16)):
        raise ValueError(f"fused_dropout: unsupported dtype {x.dtype}")
    if not training or p == 0.0:
        return x
    seed_dev = None
    if seed is None:
        from ...utils import graph_rng
        from ..tensor_parallel.random import dropout_seed

        if x.is_cuda and graph_rng.active():
            stream = 0
            if model_parallel:
                from .. import parallel_state

                stream = 1 + parallel_state.get_tensor_model_parallel_rank()
            seed, seed_dev = graph_rng.next_salt(stream), graph_rng.step_seed()
        else:
            seed = dropout_seed(model_parallel)
    p, seed = float(p), _signed64(int(seed))
    if x.is_cuda:
        return submodule("counter_dropout").dropout(x, _threshold(p), 1.0 / (1.0 - p) if p < 1.0 else 0.0, seed, seed_dev)
    return CounterDropoutFn.apply(x, p, seed)
