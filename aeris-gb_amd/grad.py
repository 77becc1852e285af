"""The block's operators outside its attention, differentiable: what a training step calls in place of ``ops.norm_modulate``,
``ops.gemm`` and the gated MLP.  (The reference trains these modules by autograd over ATen operations, model.py:121-159,311-325,395-403.)

``norm_modulate``, ``linear`` and ``feed_forward`` return tensors that autograd differentiates once, with the gradients of
``ops.norm_modulate_backward``, ``ops.linear_backward`` and ``ops.feed_forward_backward``; their results are those of the calls without
gradients, and gradients have their tensors' types.  Only the gradients that are asked for are computed, and nothing is kept where
none is.

Streams and graphs: calls follow the current stream and hold no scratch memory beyond it, and a forward pass with its backward pass may
be captured into a HIP graph.  torch's own rule for that holds here too: while the graph is captured, no eager graph of the same leaves
may be alive on another stream (torch would tie that stream to the capture and the process would end).  A captured call on
tensors whose leaves an eager result of this module still has behind it is refused with a RuntimeError; release the result, or do the eager
passes on the stream that captures.
"""
from __future__ import annotations

import weakref
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import ops

__all__ = ["feed_forward", "linear", "norm_modulate"]

_capturing = torch._C._cuda_isCurrentStreamCapturing
_EAGER = weakref.WeakSet()  # nodes of eager graphs that are alive, each with its stream


def _wants_grad(leaves):
    if torch.is_grad_enabled():
        for t in leaves:
            if t is not None and t.requires_grad:
                return True
    return False


def _leaves(nodes):
    """Identities of the tensors whose gradients the graphs behind these nodes accumulate."""
    seen, found, todo = set(), set(), [n for n in nodes if n is not None]
    while todo:
        node = todo.pop()
        if id(node) in seen:
            continue
        seen.add(id(node))
        found.add(id(getattr(node, "variable", None)))
        todo += [n for n, _ in node.next_functions if n is not None]
    return found - {id(None)}


def _note(ctx, inputs):
    """Notes an eager graph's node; under a capture, refuses inputs whose leaves an eager graph of another stream has too."""
    raw = ops._stream()
    if not _capturing():
        ctx.stream = raw
        _EAGER.add(ctx)
        return
    others = [node for node in list(_EAGER) if node.stream != raw]
    if others:
        inputs = [t for t in inputs if t is not None and t.requires_grad]
        mine = {id(t) for t in inputs if t.is_leaf} | _leaves([t.grad_fn for t in inputs])
        if not mine.isdisjoint(_leaves(others)):
            raise RuntimeError("an eager graph of a tensor of this captured call is still alive on another stream: release its result before the capture "
                               "(torch ties that stream to the capture in the backward pass, which ends the process)")


def _incoming(dy):
    """A result's gradient as the kernels read it: contiguous, its address a multiple of 16."""
    dy = dy.contiguous()
    return dy.clone() if dy.data_ptr() & 15 else dy


def _rows(t: Optional[torch.Tensor]):
    """Modulation rows with memory of their own (a row expanded over the members is copied: each member has a gradient)."""
    return t.contiguous() if t is not None and t.dim() == 2 and t.shape[0] > 1 and t.stride(0) == 0 else t


def _norm(x, gamma, beta, shift, scale, kind, order, eps, out_dtype):
    if x.numel() == 0:
        return torch.empty(x.shape, dtype=out_dtype, device=x.device)
    return ops.norm_modulate(x, gamma, beta, shift, scale, kind=kind, order=order, eps=eps, out_dtype=out_dtype)


class _NormModulate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gamma, beta, shift, scale, kind, order, eps, out_dtype):
        _note(ctx, (x, gamma, beta, shift, scale))
        shift, scale = _rows(shift), _rows(scale)
        y = _norm(x, gamma, beta, shift, scale, kind, order, eps, out_dtype)
        ctx.save_for_backward(x, gamma, beta, shift, scale)
        mod = shift if shift is not None else scale
        ctx.how = mod.stride(0) if mod is not None and mod.shape[0] > 1 else 0, ops._KIND[kind], ops._ORDER[order], eps
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        return (*ops._norm_grads(_incoming(dy), *ctx.saved_tensors, *ctx.how, ctx.needs_input_grad[:5]), None, None, None, None)


def norm_modulate(x: torch.Tensor, gamma: torch.Tensor, beta: Optional[torch.Tensor] = None, shift: Optional[torch.Tensor] = None,
                  scale: Optional[torch.Tensor] = None, *, kind: str = "layernorm", order: str = "norm_then_mod", eps: float = 1e-5,
                  out_dtype=torch.bfloat16) -> torch.Tensor:
    """``ops.norm_modulate``, differentiable in x, gamma, beta, shift and scale.

    x [B, S, d] (bf16 | f32, contiguous) -> [B, S, d] in out_dtype; gamma, beta bf16 | f32 [d]; shift, scale f32 [1 | B, d], both of one shape."""
    if kind not in ops._KIND or order not in ops._ORDER:
        raise RuntimeError(f"kind must be one of {sorted(ops._KIND)} and order one of {sorted(ops._ORDER)}, got {kind!r}, {order!r}")
    leaves = (x, gamma, beta, shift, scale)
    ops._on_current_device(x.device, dict(x=x, gamma=gamma, beta=beta, shift=shift, scale=scale))
    if x.dtype not in ops._DT or gamma.dtype not in ops._DT or out_dtype not in ops._DT:
        raise RuntimeError(f"x, gamma and the result must be bf16 or f32, got {x.dtype}, {gamma.dtype} and {out_dtype}")
    if x.dim() != 3 or gamma.shape != x.shape[2:] or (beta is not None and beta.shape != gamma.shape):
        raise RuntimeError(f"x must be [B, S, d], gamma and beta [d], got {tuple(x.shape)}, {tuple(gamma.shape)}")
    if shift is not None and scale is not None and (shift.shape != scale.shape or shift.stride(0) != scale.stride(0)):
        raise RuntimeError(f"shift and scale must be of one shape and layout, got {tuple(shift.shape)} and {tuple(scale.shape)}")
    if not _wants_grad(leaves):
        return _norm(*leaves, kind, order, eps, out_dtype)
    return _NormModulate.apply(*leaves, kind, order, eps, out_dtype)


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, a, w, bias, residual, act, out_dtype, M, N, K):
        _note(ctx, (a, w, bias, residual))
        y, z = ops._linear_forward(a, w, bias, residual, act, out_dtype, M, N, K, ctx.needs_input_grad[0] or ctx.needs_input_grad[1] or ctx.needs_input_grad[2])
        ctx.save_for_backward(a, w, z)
        ctx.how = ops._ACT[act], M, N, K
        ctx.residual = None if residual is None else (residual.dtype, residual.shape)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        need_a, need_w, need_bias, need_res = ctx.needs_input_grad[:4]
        dy = _incoming(dy)
        res_dtype, res_shape = ctx.residual if need_res else (None, None)
        round_res = need_res and res_dtype is not dy.dtype and dy.dtype is torch.float32 and ctx.how[0] == ops.L.ACT_NONE  # dz is what a bf16 residual gets
        da, dw, dbias, dres = ops._linear_grads(dy, *ctx.saved_tensors, *ctx.how, (need_a, need_w, need_bias, round_res))
        if need_res:
            dres = (dres if round_res else dy.to(res_dtype)).view(res_shape)
        return da, dw, dbias, dres, None, None, None, None, None


def linear(a: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor] = None, *, act: Optional[str] = None,
           residual: Optional[torch.Tensor] = None, out_dtype=torch.bfloat16) -> torch.Tensor:
    """act(a[.., K] @ w[N, K]^T + bias) + residual, differentiable in all four; act None | "gelu" (erf) | "silu".

    a, w, bias bf16, residual [.., N] bf16 | f32, the result in out_dtype (bf16 | f32); contiguous; N a multiple of 8, K of 64 (with an
    activation: of 8).  With an activation the value it is applied to is kept for the backward pass too (24 bits), otherwise a and w alone."""
    leaves = (a, w, bias, residual)
    ops._on_current_device(a.device, dict(a=a, w=w, bias=bias, residual=residual))
    sizes = ops._checked_linear(a, w, bias, residual, act, out_dtype)
    if not _wants_grad(leaves):
        return ops._linear_forward(a, w, bias, residual, act, out_dtype, *sizes, False)[0]
    return _Linear.apply(*leaves, act, out_dtype, *sizes)


class _FeedForward(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w1, w2, M, d, H):
        _note(ctx, (x, w1, w2))
        y, gate_up, h = ops._feed_forward(x, w1, w2, M, d, H, True)
        ctx.save_for_backward(x, w1, w2, gate_up, h)
        ctx.sizes = M, d, H
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        return (*ops._feed_forward_grads(_incoming(dy), *ctx.saved_tensors, *ctx.sizes, ctx.needs_input_grad[:3]), None, None, None)


def feed_forward(x: torch.Tensor, w1: torch.Tensor, w2: torch.Tensor) -> torch.Tensor:
    """The gated MLP ``FeedForward`` (model.py:148-159), w2 (silu(gate) * up) with [gate | up] = w1 x, differentiable in x, w1 and w2.

    x bf16 [.., d], w1 bf16 [2H, d], w2 bf16 [d, H], contiguous, d and H multiples of 8 -> bf16 [.., d].  gate and up (24
    bits) and their product (bf16) are kept for the backward pass: 8 H bytes a token."""
    ops._on_current_device(x.device, dict(x=x, w1=w1, w2=w2))
    sizes = ops._checked_feed_forward(x, w1, w2)
    if not _wants_grad((x, w1, w2)):
        return ops._feed_forward(x, w1, w2, *sizes, False)[0]
    return _FeedForward.apply(x, w1, w2, *sizes)
