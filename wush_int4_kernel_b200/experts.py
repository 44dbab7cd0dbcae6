"""Tokens ordered by expert and back, with gradients: the moves around the experts' products of a mixture-of-experts block.

No counterpart in the reference, which has dense layers only.  ``ExpertRoute`` holds the order of one batch; its two moves
are differentiable (the experts' own products are not: 8-bit codes have no gradient).

    route = ExpertRoute.sort(ids, n_experts)     # ids (tokens, k); ids outside [0, n_experts) name no expert
    rows = route.gather(x)                       # (tokens * k, H), sorted by expert
    ...                                          # rows route.offsets[e]:route.offsets[e + 1] belong to expert e
    y = route.combine(rows, weights)             # y[t] = sum_j weights[t, j] * rows[route.pos[t, j]]
"""
from __future__ import annotations

from dataclasses import dataclass

import torch
from torch.autograd.function import once_differentiable


def _ops():
    from . import _C          # ImportError when the extension is not built: no fallback
    return _C


class _Gather(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, pos, offsets):
        ctx.save_for_backward(pos)
        return _ops().expert_gather(x, pos, offsets)

    @staticmethod
    @once_differentiable
    def backward(ctx, d_rows):
        (pos,) = ctx.saved_tensors
        return _ops().expert_combine(d_rows.contiguous(), pos), None, None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, pos, offsets):
        ctx.save_for_backward(rows, weights, pos, offsets)
        return _ops().expert_combine(rows, pos, weights)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        rows, weights, pos, offsets = ctx.saved_tensors
        d_rows, d_weights = _ops().expert_combine_grad(dy.contiguous(), rows, pos, offsets, weights)
        return d_rows, d_weights, None, None


@dataclass
class ExpertRoute:
    """Order of the entries (token, choice) of one batch by expert."""
    pos: torch.Tensor          # (tokens, k) int32: row of the entry, -1 where there is no expert
    offsets: torch.Tensor      # (experts + 1) int32: first row of each expert

    @classmethod
    def sort(cls, ids: torch.Tensor, n_experts: int) -> "ExpertRoute":
        return cls(*_ops().expert_sort(ids.contiguous(), n_experts))

    def gather(self, x: torch.Tensor) -> torch.Tensor:
        """(tokens, H) -> (tokens * k, H) sorted by expert; the rows behind the last entry are zero."""
        return _Gather.apply(x.contiguous(), self.pos, self.offsets)

    def gather_quant_int8(self, x: torch.Tensor):
        """Codes and scales of ``gather(x)``; every token is quantised once.  No gradient."""
        return tuple(_ops().expert_gather_quant_int8(x.contiguous(), self.pos, self.offsets))

    def combine(self, rows: torch.Tensor, weights: torch.Tensor) -> torch.Tensor:
        """(tokens * k, H) and fp32 weights (tokens, k) -> (tokens, H); differentiable in both."""
        return _Combine.apply(rows.contiguous(), weights.contiguous(), self.pos, self.offsets)


@dataclass
class W8A8Experts:
    """Mixture-of-experts feed-forward block on 8-bit weights: y[t] = sum_j weights[t, j] * down_e(silu(gate_e) * up_e)
    with e = ids[t, j].  Six kernels in one call; tokens whose ids name no expert get zero."""
    w13q: torch.Tensor         # (experts, 2 * I, H) int8, the I gate channels first
    w13s: torch.Tensor         # (experts, 2 * I) fp32
    w2q: torch.Tensor          # (experts, H, I) int8
    w2s: torch.Tensor          # (experts, H) fp32

    @classmethod
    def from_weights(cls, w13: torch.Tensor, w2: torch.Tensor) -> "W8A8Experts":
        """Quantises (experts, 2 * I, H) and (experts, H, I) weights, one scale per channel."""
        return cls(*_ops().quant_int8(w13.contiguous()), *_ops().quant_int8(w2.contiguous()))

    @property
    def n_experts(self) -> int:
        return self.w13q.shape[0]

    def __call__(self, x: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor) -> torch.Tensor:
        lead = x.shape[:-1]
        x2, ids2, w2 = (t.reshape(-1, t.shape[-1]).contiguous() for t in (x, ids, weights))
        y = _ops().w8a8_expert_ffn(x2, ids2, w2, self.w13q, self.w13s, self.w2q, self.w2s)
        return y.reshape(*lead, x.shape[-1])

    def by_operators(self, x: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor) -> torch.Tensor:
        """The same block as a composition of the single operators; bit for bit the result of ``__call__``."""
        ops = _ops()
        route = ExpertRoute.sort(ids, self.n_experts)
        xq, xs = route.gather_quant_int8(x)
        h = ops.w8a8_grouped_gated(xq, xs, self.w13q, self.w13s, route.offsets)
        hq, hs = ops.quant_int8(h)
        fp32 = 4 * ids.numel() * x.shape[1] <= 64 << 20           # what the block keeps in fp32 before the weighted sum
        o = ops.w8a8_grouped_gemm(hq, hs, self.w2q, self.w2s, route.offsets, torch.float32 if fp32 else x.dtype)
        return ops.expert_combine(o, route.pos, weights, x.dtype)

    def to(self, device) -> "W8A8Experts":
        return W8A8Experts(*(t.to(device) for t in (self.w13q, self.w13s, self.w2q, self.w2s)))
