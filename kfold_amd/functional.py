"""Differentiable forms of the training operators of ``kfold_amd.ops``.

Each is one ``torch.autograd.Function`` around the forward and backward entry points; what is kept
between the two is the operator's inputs (for the layer norm also two fp32 statistics per row).  First
derivatives in reverse mode only: forward-mode tangents are refused.  To record a step into a HIP graph, call the forward and backward functions of
``ops`` themselves: they only enqueue kernels on the current stream.
"""

from __future__ import annotations

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import ops


def _differentiated(*tensors: torch.Tensor | None) -> bool:
    """Whether the call has to go through the autograd function: gradients are wanted, or an argument
    carries a tangent, which the function refuses (the kernels would drop it)."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        return True
    # tangents exist inside a dual level only; asking each tensor costs microseconds
    if getattr(forward_ad, "_current_level", 0) < 0:
        return False
    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = ops.layer_norm_forward(x, weight, bias, eps, stats=True)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.bias_dtype = None if bias is None else bias.dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, mean, rstd = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dx, dw, db = ops.layer_norm_backward(dy, x, mean, rstd, weight, need_dx=need_x, need_dparams=need_w or need_b)
        return dx, dw.to(weight.dtype) if need_w else None, db.to(ctx.bias_dtype) if need_b else None, None


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """Layer norm over the last dim of x (bf16 or fp32, any width), result in x.dtype."""
    if _differentiated(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, eps)
    return ops.layer_norm_forward(x, weight, bias, eps)


class _GatedFFN(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_in, w_out):
        ctx.save_for_backward(x, w_in, w_out)
        return ops.gated_ffn_forward(x, w_in.to(x.dtype), w_out.to(x.dtype))

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w_in, w_out = ctx.saved_tensors
        need_x, need_i, need_o = ctx.needs_input_grad
        # one rounding to the weights' type: in the kernel where both have the type it writes
        same = w_in.dtype == w_out.dtype == torch.bfloat16
        dx, dwi, dwo = ops.gated_ffn_backward(dy, x, w_in.to(x.dtype), w_out.to(x.dtype), need_dx=need_x,
                                              need_dw=(need_i, need_o), dw_dtype=torch.bfloat16 if same else torch.float32)
        return dx, dwi.to(w_in.dtype) if need_i else None, dwo.to(w_out.dtype) if need_o else None


def gated_ffn(x: torch.Tensor, w_in: torch.Tensor, w_out: torch.Tensor) -> torch.Tensor:
    """``(silu(u) * v) w_out^T`` with ``u, v = chunk(x w_in^T, 2)``: the SwiGLU block with its output
    projection.  Weights of another dtype are rounded to x's first; their gradients come in their own."""
    if _differentiated(x, w_in, w_out):
        return _GatedFFN.apply(x, w_in, w_out)
    return ops.gated_ffn_forward(x, w_in.to(x.dtype), w_out.to(x.dtype))


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed, offset, shared_dim):
        # a seed in device memory is kept as a saved tensor: changing it in place before the backward
        # pass, which draws the mask again, is then an error
        if isinstance(seed, torch.Tensor):
            ctx.save_for_backward(seed)
        ctx.args = (p, None if isinstance(seed, torch.Tensor) else seed, offset, shared_dim)
        return ops.dropout_forward(x, p, seed, offset, shared_dim, residual)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        p, seed, offset, shared_dim = ctx.args
        if seed is None:
            (seed,) = ctx.saved_tensors
        dx = ops.dropout_backward(dy, p, seed, offset, shared_dim) if ctx.needs_input_grad[0] else None
        return dx, dy if ctx.needs_input_grad[1] else None, None, None, None, None


def dropout(x: torch.Tensor, p: float, seed, offset: int = 0, shared_dim: int | None = None,
            residual: torch.Tensor | None = None) -> torch.Tensor:
    """``(residual or 0) + dropout(x)`` with the mask of ``ops.dropout_forward``."""
    if _differentiated(x, residual):
        return _Dropout.apply(x, residual, p, seed, offset, shared_dim)
    return ops.dropout_forward(x, p, seed, offset, shared_dim, residual)
