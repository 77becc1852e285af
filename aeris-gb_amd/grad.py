"""The block's operators outside its attention, differentiable: what a training step calls in place of ``ops.norm_modulate``,
``ops.gemm`` and the gated MLP.  (The reference trains these modules by autograd over ATen operations, model.py:121-159,311-325,395-403.)

``norm_modulate``, ``linear`` and ``feed_forward`` return tensors that autograd differentiates once, with the gradients of
``ops.norm_modulate_backward``, ``ops.linear_backward`` and ``ops.feed_forward_backward``; their results are those of the calls without
gradients, and gradients have their tensors' types.  Only the gradients that are asked for are computed.

Streams and graphs: calls follow the current stream and hold no scratch memory beyond it, and a forward pass with its backward pass may
be captured into a HIP graph.  torch's own rule for that holds here too: while the graph is captured, no eager graph of the same leaves
may be alive on another stream (torch would tie that stream to the capture and the process would end).  A captured call on a
leaf for which an eager result of this module still lives is refused with a RuntimeError; release the result, or do the eager passes on
the stream that captures.
"""
from __future__ import annotations

import weakref
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import ops

__all__ = ["feed_forward", "linear", "norm_modulate"]

# leaf -> the eager graphs through it that may still be alive: (weak reference to the node, raw stream)
_EAGER = torch.utils.weak.WeakIdKeyDictionary()


def _record(result, leaves):
    """Notes which eager graph ``result`` made of ``leaves``."""
    node = result.grad_fn
    if node is None or torch._C._cuda_isCurrentStreamCapturing():
        return result
    entry = (weakref.ref(node), ops._stream())
    for t in leaves:
        if t is not None and t.requires_grad and t.is_leaf:
            live = [e for e in _EAGER.get(t, ()) if e[0]() is not None]
            _EAGER[t] = live + [entry]
    return result


def _refuse_under_capture(leaves):
    if not torch._C._cuda_isCurrentStreamCapturing() or not torch.is_grad_enabled():
        return
    raw = ops._stream()
    for t in leaves:
        if t is not None and any(ref() is not None and stream != raw for ref, stream in _EAGER.get(t, ())):
            raise RuntimeError("an eager graph of a tensor of this captured call is still alive on another stream: release its result before the capture "
                               "(torch ties that stream to the capture in the backward pass, which ends the process)")


def _rows(t: Optional[torch.Tensor]):
    """Modulation rows with memory of their own (a row expanded over the members is copied: each member has a gradient)."""
    return t.contiguous() if t is not None and t.dim() == 2 and t.shape[0] > 1 and t.stride(0) == 0 else t


class _NormModulate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gamma, beta, shift, scale, kind, order, eps, out_dtype):
        shift, scale = _rows(shift), _rows(scale)
        if x.numel() == 0:
            y = torch.empty(x.shape, dtype=out_dtype, device=x.device)
        else:
            y = ops.norm_modulate(x, gamma, beta, shift, scale, kind=kind, order=order, eps=eps, out_dtype=out_dtype)
        ctx.save_for_backward(x, gamma, beta, shift, scale)
        ctx.how = kind, order, eps
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        kind, order, eps = ctx.how
        return (*ops.norm_modulate_backward(dy.contiguous(), *ctx.saved_tensors, kind=kind, order=order, eps=eps, wanted=ctx.needs_input_grad[:5]),
                None, None, None, None)


def norm_modulate(x: torch.Tensor, gamma: torch.Tensor, beta: Optional[torch.Tensor] = None, shift: Optional[torch.Tensor] = None,
                  scale: Optional[torch.Tensor] = None, *, kind: str = "layernorm", order: str = "norm_then_mod", eps: float = 1e-5,
                  out_dtype=torch.bfloat16) -> torch.Tensor:
    """``ops.norm_modulate``, differentiable in x, gamma, beta, shift and scale.

    x [B, S, d] (bf16 | f32, contiguous) -> [B, S, d] in out_dtype; gamma, beta bf16 | f32 [d]; shift, scale f32 [1 | B, d], both of one shape."""
    if kind not in ops._KIND or order not in ops._ORDER:
        raise RuntimeError(f"kind must be one of {sorted(ops._KIND)} and order one of {sorted(ops._ORDER)}, got {kind!r}, {order!r}")
    ops._on_current_device(x.device, dict(x=x, gamma=gamma, beta=beta, shift=shift, scale=scale))
    if x.dtype not in ops._DT or gamma.dtype not in ops._DT or out_dtype not in ops._DT:
        raise RuntimeError(f"x, gamma and the result must be bf16 or f32, got {x.dtype}, {gamma.dtype} and {out_dtype}")
    if x.dim() != 3 or gamma.shape != x.shape[2:] or (beta is not None and beta.shape != gamma.shape):
        raise RuntimeError(f"x must be [B, S, d], gamma and beta [d], got {tuple(x.shape)}, {tuple(gamma.shape)}")
    if shift is not None and scale is not None and shift.shape != scale.shape:
        raise RuntimeError(f"shift and scale must be of one shape, got {tuple(shift.shape)} and {tuple(scale.shape)}")
    leaves = (x, gamma, beta, shift, scale)
    _refuse_under_capture(leaves)
    return _record(_NormModulate.apply(*leaves, kind, order, eps, out_dtype), leaves)


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, a, w, bias, residual, act, out_dtype):
        y, z = ops.linear_train(a, w, bias, act=act, residual=residual, out_dtype=out_dtype)
        ctx.save_for_backward(a, w, z)
        ctx.act, ctx.res_dtype = act, None if residual is None else residual.dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        a, w, z = ctx.saved_tensors
        need_a, need_w, need_bias, need_res = ctx.needs_input_grad[:4]
        plain = ctx.act in (None, "none")
        dy = dy.contiguous()
        round_res = need_res and ctx.res_dtype is not dy.dtype and plain and dy.dtype is torch.float32  # dz is what a bf16 residual gets
        da, dw, dbias, dz = ops.linear_backward(dy, a, w, z, act=ctx.act, wanted=(need_a, need_w, need_bias, round_res))
        dres = None
        if need_res:
            dres = dz if round_res else dy.to(ctx.res_dtype)
        return da, dw, dbias, dres, None, None


def linear(a: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor] = None, *, act: Optional[str] = None,
           residual: Optional[torch.Tensor] = None, out_dtype=torch.bfloat16) -> torch.Tensor:
    """act(a[.., K] @ w[N, K]^T + bias) + residual, differentiable in all four; act None | "gelu" (erf) | "silu".

    a, w, bias bf16, residual [.., N] bf16 | f32, the result in out_dtype (bf16 | f32); contiguous; N a multiple of 8, K of 64 (with an
    activation: of 8).  With an activation the bf16 value it is applied to is kept for the backward pass, otherwise a and w alone."""
    leaves = (a, w, bias, residual)
    ops._on_current_device(a.device, dict(a=a, w=w, bias=bias, residual=residual))
    _refuse_under_capture(leaves)
    return _record(_Linear.apply(*leaves, act, out_dtype), leaves)


class _FeedForward(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w1, w2):
        y, gate_up, h = ops.feed_forward_train(x, w1, w2)
        ctx.save_for_backward(x, w1, w2, gate_up, h)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        return ops.feed_forward_backward(dy.contiguous(), *ctx.saved_tensors, wanted=ctx.needs_input_grad)


def feed_forward(x: torch.Tensor, w1: torch.Tensor, w2: torch.Tensor) -> torch.Tensor:
    """The gated MLP ``FeedForward`` (model.py:148-159), w2 (silu(gate) * up) with [gate | up] = w1 x, differentiable in x, w1 and w2.

    x bf16 [.., d], w1 bf16 [2H, d], w2 bf16 [d, H], contiguous, d and H multiples of 8 -> bf16 [.., d].  gate, up and their product (bf16,
    3 H numbers a token) are kept for the backward pass."""
    leaves = (x, w1, w2)
    ops._on_current_device(x.device, dict(x=x, w1=w1, w2=w2))
    _refuse_under_capture(leaves)
    return _record(_FeedForward.apply(*leaves), leaves)
