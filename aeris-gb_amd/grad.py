"""The block's operators outside its attention, differentiable: what a training step calls in place of ``ops.norm_modulate``,
``ops.gemm`` and the gated MLP.  (The reference trains these modules by autograd over ATen operations, model.py:121-159,311-325,395-403.)

``norm_modulate``, ``linear`` and ``feed_forward`` return tensors that autograd differentiates once, in reverse mode, with the gradients of
``ops.norm_modulate_backward``, ``ops.linear_backward`` and ``ops.feed_forward_backward``, in their tensors' types.  A result has the same bits
whether or not it is to be differentiated; those of ``ops.norm_modulate`` and of ``ops.gemm`` without activation are the same too, ``ops.gemm`` with
GELU or SiLU and the module ``FeedForward`` differ in the last roundings (up to 64 tokens ``feed_forward`` keeps h in two bf16).  Only the gradients
that are asked for are computed, and nothing is kept where none is; how their products are cut and in what order their sums are added depends on
the sizes, the types and which of them are asked for.  The nodes of the autograd graph are C++ (csrc/grad_functions.cpp, built to csrc/aeris_grad.so): a small block's pass is bound by the host.

Streams and graphs: calls follow the current stream and hold no scratch memory beyond it, and a forward pass with its backward pass may
be captured into a HIP graph.  torch's own rule for that holds here too: what the captured graph differentiates must have no autograd nodes of
another stream - an eager graph of the same leaves that is still alive, or an input computed outside the capture - or torch would tie that stream to
the capture and the process would end.  Such a call is refused with a RuntimeError; release the eager result, or do the eager passes on the stream
that captures.  (A backward pass alone, of a forward pass outside the capture, is torch's to start and cannot be refused here: capture both.)
``ops.profile_begin`` records the calls of ``ops``, not these.
"""
from __future__ import annotations

import importlib.machinery
import importlib.util
import os
from typing import Optional

import torch

from . import _lib as L
from . import build, ops

__all__ = ["feed_forward", "linear", "norm_modulate"]

EXTENSION_PATH = os.path.join(os.path.dirname(L.LIB_PATH), "aeris_grad.so")
_ACT = {None: L.ACT_NONE, "none": L.ACT_NONE, "gelu": L.ACT_GELU, "silu": L.ACT_SILU}
_F32 = {torch.bfloat16: False, torch.float32: True}
_loaded = None


def _functions():
    """The extension, loaded once, behind the library whose calls it makes."""
    global _loaded
    if _loaded is None:
        if not os.path.exists(EXTENSION_PATH):
            raise RuntimeError(f"{EXTENSION_PATH} is missing: build it with `python aeris-gb_amd/build.py` (there is no fallback path)")
        if not build.grad_built_for_this_torch(EXTENSION_PATH):
            raise RuntimeError(f"{EXTENSION_PATH} was built against another torch than {torch.__version__}: build it again with `python aeris-gb_amd/build.py`")
        L.lib()
        loader = importlib.machinery.ExtensionFileLoader("aeris_grad", EXTENSION_PATH)
        module = importlib.util.module_from_spec(importlib.util.spec_from_loader("aeris_grad", loader))
        loader.exec_module(module)
        _loaded = module
    return _loaded


def norm_modulate(x: torch.Tensor, gamma: torch.Tensor, beta: Optional[torch.Tensor] = None, shift: Optional[torch.Tensor] = None,
                  scale: Optional[torch.Tensor] = None, *, kind: str = "layernorm", order: str = "norm_then_mod", eps: float = 1e-5,
                  out_dtype=torch.bfloat16) -> torch.Tensor:
    """``ops.norm_modulate``, differentiable in x, gamma, beta, shift and scale.

    x [B, S, d] (bf16 | f32, contiguous) -> [B, S, d] in out_dtype; gamma, beta bf16 | f32 [d]; shift, scale f32 [1 | B, d], both of one shape and
    layout (columns of one matrix, or a row expanded over the members)."""
    if kind not in ops._KIND or order not in ops._ORDER or out_dtype not in _F32:
        raise RuntimeError(f"kind must be one of {sorted(ops._KIND)}, order one of {sorted(ops._ORDER)} and the result bf16 or f32, got {kind!r}, {order!r}, {out_dtype}")
    return (_loaded or _functions()).norm_modulate(x, gamma, beta, shift, scale, ops._KIND[kind], ops._ORDER[order], eps, _F32[out_dtype])


def linear(a: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor] = None, *, act: Optional[str] = None,
           residual: Optional[torch.Tensor] = None, out_dtype=torch.bfloat16) -> torch.Tensor:
    """act(a[.., K] @ w[N, K]^T + bias) + residual, differentiable in all four; act None | "gelu" (erf) | "silu".

    a, w, bias bf16, residual [.., N] bf16 | f32, the result in out_dtype (bf16 | f32); contiguous; N a multiple of 8, K of 64 (with an
    activation: of 8).  With an activation the value it is applied to is kept for the backward pass too (24 bits), otherwise a and w alone."""
    if act not in _ACT or out_dtype not in _F32:
        raise RuntimeError(f"act must be None, 'gelu' or 'silu' and the result bf16 or f32, got {act!r}, {out_dtype}")
    return (_loaded or _functions()).linear(a, w, bias, _ACT[act], residual, _F32[out_dtype])


def feed_forward(x: torch.Tensor, w1: torch.Tensor, w2: torch.Tensor) -> torch.Tensor:
    """The gated MLP ``FeedForward`` (model.py:148-159), w2 (silu(gate) * up) with [gate | up] = w1 x, differentiable in x, w1 and w2.

    x bf16 [.., d], w1 bf16 [2H, d], w2 bf16 [d, H], contiguous, d and H multiples of 8 -> bf16 [.., d].  gate and up (24
    bits) and their product (bf16) are kept for the backward pass: 8 H bytes a token."""
    return (_loaded or _functions()).feed_forward(x, w1, w2)
