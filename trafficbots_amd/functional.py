"""Autograd forms of the engine's training operators: what a transformer layer of the reference (`src/models/modules/transformer.py:98-240`,
`attention.py:9-154`, `mlp.py:20-85`) needs to be trained on the device -- attention, layer norm, Linear with bias, ReLU, row mask and
residual.  Every function takes the engine that runs it first (`HipEngine`, or `wm.engine`); the arithmetic is
`HipEngine.attention / layer_norm / linear` and their `_backward` twins, there is no host fallback.

The gradients are not differentiable once more (a second backward raises).  To capture a training step into a graph, capture the engine's
calls themselves, or make sure that no eager graph of the same leaves is alive (torch's accumulation into a leaf would wait for work
outside the capture)."""
from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, engine, q, k, v, query_valid, key_valid, attn_mask, causal, scale):
        out, lse = engine.attention(q, k, v, query_valid, key_valid, attn_mask, causal, scale)
        ctx.engine, ctx.causal, ctx.scale = engine, causal, scale
        ctx.save_for_backward(q, k, v, out, lse, query_valid, key_valid, attn_mask)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out):
        dq, dk, dv = ctx.engine.attention_backward(d_out, *ctx.saved_tensors, ctx.causal, ctx.scale)
        return None, dq, dk, dv, None, None, None, None, None


def attention(engine, q: Tensor, k: Tensor, v: Tensor, query_valid: Optional[Tensor] = None, key_valid: Optional[Tensor] = None,
              attn_mask: Optional[Tensor] = None, causal: bool = False, scale: Optional[float] = None) -> Tensor:
    """:meth:`HipEngine.attention` with gradients of q, k and v: [B, Lq, H, D]."""
    return _Attention.apply(engine, q, k, v, query_valid, key_valid, attn_mask, causal, scale)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, engine, x, weight, bias, eps):
        y, mean, rstd = engine.layer_norm(x, weight, bias, eps)
        ctx.engine = engine
        ctx.save_for_backward(x, weight, mean, rstd)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out):
        x, weight, mean, rstd = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, dw, db = ctx.engine.layer_norm_backward(d_out, x, weight, mean, rstd, want_dx=need[1], want_dweight=need[2] or need[3])
        return None, dx, dw if need[2] else None, db if need[3] else None, None


def layer_norm(engine, x: Tensor, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None, eps: float = 1e-5) -> Tensor:
    """:meth:`HipEngine.layer_norm` with gradients of x, weight and bias."""
    return _LayerNorm.apply(engine, x, weight, bias, eps)


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, engine, x, weight, bias, residual, activation, row_valid):
        y, act = engine.linear(x, weight, bias, activation, row_valid, residual, want_act=True) if activation else \
            (engine.linear(x, weight, bias, activation, row_valid, residual), None)
        ctx.engine = engine
        ctx.save_for_backward(x, weight, act, row_valid)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out):
        x, weight, act, row_valid = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx = dw = db = None
        if any(need[1:4]):
            dx, dw, db = ctx.engine.linear_backward(d_out, x, weight, act=act, row_valid=row_valid, want_dx=need[1], want_dweight=need[2], want_dbias=need[3])
        return None, dx, dw, db, d_out if need[4] else None, None, None


def linear(engine, x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, activation: Optional[str] = None, row_valid: Optional[Tensor] = None,
           residual: Optional[Tensor] = None) -> Tensor:
    """:meth:`HipEngine.linear` with gradients of x, weight, bias and residual."""
    return _Linear.apply(engine, x, weight, bias, residual, activation, row_valid)
