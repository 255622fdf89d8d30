"""Differentiable forms of the tensor-level operators.

Each function runs the same kernel as its namesake in :mod:`sinkattn_b200.ops`
(sink_dynamic_attention: sink_dynamic_attn) and records what its gradient needs;
without a differentiable input (or under torch.no_grad()) nothing is recorded.
The gradients are first-order only. reference_api's drop-ins call these where
an input requires a gradient. Results may be written over; where the gradient
needs the output (both attentions) the backward pass then refuses.

A backward pass may be captured into a CUDA graph like any other torch one:
warm it up on a side stream and let no graph of the same leaves that was
recorded eagerly stay alive beside it (torch ties a leaf's accumulation to the
stream it was first recorded on).
"""
from __future__ import annotations

import math
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import ops


def needs_grad(*tensors: Optional[torch.Tensor]) -> bool:
    """Whether a call on these tensors has to be recorded."""
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


class _BlockSparseAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, block_mask, softmax_scale, head_mask_type):
        out, lse = ops.bsattn_fwd(q, k, v, block_mask, softmax_scale=softmax_scale,
                                  head_mask_type=head_mask_type)
        out = out.detach()  # torch refuses to write over one of several results that is a view
        ctx.save_for_backward(q, k, v, out, lse, block_mask, head_mask_type)
        ctx.softmax_scale = softmax_scale
        ctx.set_materialize_grads(False)
        return out, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dlse):
        if dout is None and dlse is None:
            return (None,) * 6
        q, k, v, out, lse, block_mask, head_mask_type = ctx.saved_tensors
        if dout is None:
            dout = torch.zeros_like(out)
        dq, dk, dv = ops.bsattn_bwd(dout, q, k, v, out, lse, block_mask,
                                    softmax_scale=ctx.softmax_scale,
                                    head_mask_type=head_mask_type, dlse=dlse)
        return dq, dk, dv, None, None, None


def block_sparse_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                           block_mask: torch.Tensor, softmax_scale: Optional[float] = None,
                           head_mask_type: Optional[torch.Tensor] = None):
    """ops.bsattn_fwd with gradients for q, k and v, through both results.

    Arguments as for ops.bsattn_fwd. Returns (out [B,H,Sq,D] bf16, lse fp32
    [B,H,Sq]). Keys and values broadcast over heads (expanded views) get their
    gradients summed over them by autograd. The backward pass takes at most
    131072 queries and keys and refuses more."""
    return _BlockSparseAttention.apply(q, k, v, block_mask, softmax_scale, head_mask_type)


def _like(grad: Optional[torch.Tensor], w: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return None if grad is None or w is None else grad.to(w.dtype)


class _QKHeadNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, eps, w_q, w_k, cos, sin, positions, interleaved):
        out_q, out_k = ops.qk_head_norm_rope(q, k, eps, w_q, w_k, cos, sin, positions=positions,
                                             interleaved=interleaved)
        ctx.save_for_backward(q, k, w_q, w_k, cos, sin, positions)
        ctx.eps, ctx.interleaved = eps, interleaved
        return out_q, out_k

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk):
        q, k, w_q, w_k, cos, sin, positions = ctx.saved_tensors
        dq, dk, dw_q, dw_k = ops.qk_head_norm_rope_bwd(
            dq, None if k is None else dk, q, k, ctx.eps, w_q, w_k, cos, sin,
            positions=positions, interleaved=ctx.interleaved)
        return dq, dk, None, _like(dw_q, w_q), _like(dw_k, w_k), None, None, None, None


def qk_head_norm_rope(q: torch.Tensor, k: Optional[torch.Tensor], eps: float,
                      w_q: Optional[torch.Tensor] = None, w_k: Optional[torch.Tensor] = None,
                      cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None,
                      positions: Optional[torch.Tensor] = None, interleaved: bool = True):
    """ops.qk_head_norm_rope with gradients for q, k, w_q and w_k (the tables
    get none). The weights' gradients are summed in fp32 and returned in the
    weights' type."""
    return _QKHeadNormRope.apply(q, k, eps, w_q, w_k, cos, sin, positions, interleaved)


class _QKNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, head_dim, eps, w_q, w_k, cos, sin):
        out_q, out_k = ops.qk_norm_rope(q, k, head_dim, eps, w_q, w_k, cos, sin)
        ctx.save_for_backward(q, k, w_q, w_k, cos, sin)
        ctx.head_dim, ctx.eps = head_dim, eps
        return out_q, out_k

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk):
        q, k, w_q, w_k, cos, sin = ctx.saved_tensors
        dq, dk, dw_q, dw_k = ops.qk_norm_rope_bwd(dq, dk, q, k, ctx.head_dim, ctx.eps, w_q, w_k,
                                                  cos, sin)
        return dq, dk, None, None, _like(dw_q, w_q), _like(dw_k, w_k), None, None


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, head_dim: int, eps: float,
                 w_q: Optional[torch.Tensor] = None, w_k: Optional[torch.Tensor] = None,
                 cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None):
    """ops.qk_norm_rope (out of place) with gradients for q, k, w_q and w_k
    (the tables get none); the bf16 rounding between the norm and the rotation
    counts as the identity."""
    return _QKNormRope.apply(q, k, head_dim, eps, w_q, w_k, cos, sin)


class _MeanPool(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, pool, prefix):
        ctx.size, ctx.pool, ctx.prefix = x.shape[2], pool, prefix
        return ops.mean_pool_seq(x, pool, prefix).detach()

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        pooled = dout[:, :, ctx.prefix:]
        tokens = ctx.size - ctx.prefix
        # the last pool counts the final token once more for each token it lacks
        last = 1 + pooled.shape[2] * ctx.pool - tokens
        spread = (pooled.float() / ctx.pool).to(dout.dtype)
        dx = spread.repeat_interleave(ctx.pool, dim=2)[:, :, :tokens]
        if last > 1:
            dx[:, :, -1] = (pooled[:, :, -1].float() * (last / ctx.pool)).to(dout.dtype)
        return torch.cat([dout[:, :, :ctx.prefix], dx], dim=2), None, None


def mean_pool_seq(x: torch.Tensor, pool: int, prefix: int = 0) -> torch.Tensor:
    """ops.mean_pool_seq with a gradient for x (torch operations, one rounding)."""
    prefix = min(max(int(prefix), 0), x.shape[2])
    if pool <= 1 or prefix == x.shape[2]:
        return x
    return _MeanPool.apply(x, int(pool), prefix)


class _MixOutputs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, sink_out, sink_lse, dyn_out, dyn_lse, sample_gap):
        ctx.save_for_backward(sink_out, sink_lse, dyn_out, dyn_lse)
        ctx.log_gap = math.log(float(max(1, int(sample_gap))))
        return ops.mix_outputs(sink_out, sink_lse, dyn_out, dyn_lse, sample_gap).detach()

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        sink_out, sink_lse, dyn_out, dyn_lse = ctx.saved_tensors
        rows = (*sink_out.shape[:3], 1)
        lead = sink_lse.reshape(rows).float() - (dyn_lse.reshape(rows).float() + ctx.log_gap)
        w_sink, w_dyn = torch.sigmoid(lead), torch.sigmoid(-lead)
        d = dout.float()
        dlead = w_sink * w_dyn * (d * (sink_out.float() - dyn_out.float())).sum(-1, keepdim=True)
        return ((d * w_sink).to(sink_out.dtype), dlead.reshape(sink_lse.shape).to(sink_lse.dtype),
                (d * w_dyn).to(dyn_out.dtype), -dlead.reshape(dyn_lse.shape).to(dyn_lse.dtype), None)


def mix_outputs(sink_out: torch.Tensor, sink_lse: torch.Tensor, dyn_out: torch.Tensor,
                dyn_lse: torch.Tensor, sample_gap: int) -> torch.Tensor:
    """ops.mix_outputs with gradients for both outputs and both log-sum-exps
    (torch operations in fp32, one rounding)."""
    return _MixOutputs.apply(sink_out, sink_lse, dyn_out, dyn_lse, sample_gap)


class _SinkDynamicAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, block_mask, k_pool, v_pool, sample_gap, softmax_scale,
                head_mask_type):
        out, lse = ops.sink_dynamic_attn(q, k, v, block_mask, k_pool, v_pool, sample_gap,
                                         softmax_scale=softmax_scale,
                                         head_mask_type=head_mask_type, return_lse=True)
        out = out.detach()  # as above
        if head_mask_type is not None:
            head_mask_type = head_mask_type.to(torch.int32)
        ctx.save_for_backward(q, k, v, k_pool, v_pool, out, lse, block_mask, head_mask_type)
        ctx.softmax_scale = softmax_scale
        ctx.log_gap = math.log(float(max(1, int(sample_gap))))
        ctx.set_materialize_grads(False)
        return out, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dlse):
        if dout is None and dlse is None:
            return (None,) * 9
        q, k, v, k_pool, v_pool, out, lse, block_mask, head_mask_type = ctx.saved_tensors
        if dout is None:
            dout = torch.zeros_like(out)
        # One softmax over both kinds of keys: with the joint output and log-sum-exp the
        # backward pass of either kind is that of the attention alone. The pooled keys' logits
        # are raised by ln(gap), which taken from the log-sum-exp is the same probability.
        dq, dk, dv = ops.bsattn_bwd(dout, q, k, v, out, lse, block_mask,
                                    softmax_scale=ctx.softmax_scale,
                                    head_mask_type=head_mask_type, dlse=dlse)
        dense = torch.zeros(q.shape[1], dtype=torch.int32, device=q.device)
        blocks = [-(-t.shape[2] // ops.BLOCK) for t in (q, k_pool)]
        unread = torch.ones(1, 1, *blocks, dtype=torch.bool, device=q.device)
        dq2, dk_pool, dv_pool = ops.bsattn_bwd(dout, q, k_pool, v_pool, out, lse - ctx.log_gap,
                                               unread, softmax_scale=ctx.softmax_scale,
                                               head_mask_type=dense, dlse=dlse)
        return dq.add_(dq2), dk, dv, None, dk_pool, dv_pool, None, None, None


def sink_dynamic_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                           block_mask: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                           sample_gap: int, softmax_scale: Optional[float] = None,
                           head_mask_type: Optional[torch.Tensor] = None):
    """ops.sink_dynamic_attn with gradients for q, k, v, k_pool and v_pool, through
    both results. Returns (out, lse); the backward pass takes at most 131072
    queries and keys and refuses more."""
    return _SinkDynamicAttention.apply(q, k, v, block_mask, k_pool, v_pool, sample_gap,
                                       softmax_scale, head_mask_type)
