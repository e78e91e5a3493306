"""Differentiable dense-head operators over rows: layer norm, a linear layer whose input is kept in 8 bits, and log
probabilities over the item catalogue.

Each is one autograd node over the typed wrappers of ``kernels`` (csrc/layer_norm.hip, act8.hip, log_prob.hip); tensors
live on the GPU, in float32, bfloat16 or float16.  Inputs of more than two dimensions are taken as rows of their last
one (``log_probs`` takes two: its items belong to the rows).  Gradients of gradients are not available.  The types are the tensors' own: autocast changes nothing.

``needs_input_grad`` is what the inputs ask for, also under ``torch.no_grad``, and inside ``forward`` the grad mode is
always off: the nodes that keep something for the backward are told the caller's grad mode (``grad``).
"""
from __future__ import annotations

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _lib, kernels


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x as [n, d] with unit stride in the last dimension (a copy only where a view cannot show it)."""
    if x.dim() == 0:
        raise ValueError("expected rows, got a scalar")
    x = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    return x if x.stride(1) == 1 else x.contiguous()


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, grad):
        rows = _rows(x)
        if not (grad and any(ctx.needs_input_grad)):
            return kernels.layer_norm_fwd(rows, weight, bias, eps).view(x.shape)
        y, mean, rstd = kernels.layer_norm_fwd(rows, weight, bias, eps, stats=True)
        ctx.save_for_backward(x, mean, rstd, weight)
        ctx.bias_dtype = None if bias is None else bias.dtype
        return y.view(x.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, mean, rstd, weight = ctx.saved_tensors
        dx, dw, db = kernels.layer_norm_bwd(_rows(dy), _rows(x), mean, rstd, weight, *ctx.needs_input_grad[:3])
        if db is not None:
            db = db.to(ctx.bias_dtype)
        return None if dx is None else dx.view(x.shape), dw, db, None, None


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """Layer norm over the last dimension, in x's type; weight / bias in float32 or x's type (kernels.layer_norm_fwd)."""
    return _LayerNorm.apply(x, weight, bias, eps, torch.is_grad_enabled())


class LayerNorm(nn.LayerNorm):
    """``nn.LayerNorm`` over one dimension (the same parameters and state_dict keys) on the HIP path."""

    def __init__(self, normalized_shape: int, eps: float = 1e-5, elementwise_affine: bool = True, bias: bool = True,
                 device=None, dtype=None) -> None:
        super().__init__(normalized_shape, eps, elementwise_affine, bias, device, dtype)
        if len(self.normalized_shape) != 1:
            raise ValueError("LayerNorm normalises the last dimension only")

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.shape[-1:] != self.normalized_shape:
            raise ValueError(f"expected a last dimension of {self.normalized_shape[0]}, got {list(x.shape)}")
        return layer_norm(x, self.weight, self.bias, self.eps)


def _product(a: torch.Tensor, b: torch.Tensor, trans_b: bool, bias: torch.Tensor | None = None) -> torch.Tensor:
    """a [n, k] times b [k, m] (or its transpose b [m, k]), plus bias [m]: the library's fp32 GEMM where it takes the
    widths, else torch's plain product.  A 16-bit result is rounded once: the bias goes into the product's 32-bit sum."""
    if a.dtype is torch.float32 and kernels.gemm_supported(a, b):
        y = kernels.gemm(a, b, trans_b=trans_b)
        return y if bias is None else y.add_(bias)
    b = b.t() if trans_b else b
    with torch.autocast(a.device.type, enabled=False):
        return a @ b if bias is None else torch.addmm(bias, a, b)


class _LinearAct8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, grad):
        rows = _rows(x)
        kernels._req_rows(rows, "x")
        if weight.device != rows.device or (bias is not None and bias.device != rows.device):
            raise ValueError(f"weight and bias: on {rows.device} expected")
        if weight.dim() != 2 or weight.shape[1] != rows.shape[1]:
            raise ValueError(f"weight: [out, {rows.shape[1]}] expected, got {list(weight.shape)}")
        if bias is not None and bias.shape != weight.shape[:1]:
            raise ValueError(f"bias: [{weight.shape[0]}] expected, got {list(bias.shape)}")
        if ctx.needs_input_grad[1] and not 1 <= rows.shape[1] <= _lib.KGAT_ACT8_MAX_D:
            raise ValueError(f"x: width must be in [1, {_lib.KGAT_ACT8_MAX_D}], got {rows.shape[1]}")
        w = weight.to(rows.dtype)
        y = _product(rows, w, True, None if bias is None else bias.to(rows.dtype))
        if grad and any(ctx.needs_input_grad):
            a = kernels.act8_pack(rows) if ctx.needs_input_grad[1] else None
            ctx.save_for_backward(weight, *((a.q, a.e) if a is not None else ()))
            ctx.rows = (tuple(rows.shape), rows.dtype)
            ctx.bias_dtype = None if bias is None else bias.dtype
        ctx.x_shape = x.shape
        return y.view(*x.shape[:-1], weight.shape[0])

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        weight, *packed = ctx.saved_tensors
        shape, dtype = ctx.rows
        dy = _rows(dy)
        dx = dW = db = None
        if ctx.needs_input_grad[0]:
            dx = _product(dy, weight.to(dtype), False).view(ctx.x_shape)
        if ctx.needs_input_grad[1]:
            dW, db = kernels.act8_wgrad(dy, kernels.Act8(*packed, shape, dtype), bias=ctx.needs_input_grad[2])
            dW = dW.to(weight.dtype)
        elif ctx.needs_input_grad[2]:
            db = dy.sum(0, dtype=torch.float32)
        return dx, dW, None if db is None else db.to(ctx.bias_dtype), None


def linear_act8(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None) -> torch.Tensor:
    """``F.linear`` that keeps its input for the backward in 8 bits (1.03 bytes an element against 4 or 2;
    kernels.act8_pack).  The output, rounded once, and the input's gradient are those of the exact input (products by
    kgat_gemm_f32 in float32 where the widths are multiples of 4, else torch's); the weight's gradient is the exact product
    with the 8-bit values, within 2^-7 of each block's largest (kernels.act8_wgrad)."""
    return _LinearAct8.apply(x, weight, bias, torch.is_grad_enabled())


class LinearAct8(nn.Linear):
    """``nn.Linear`` (the same parameters, initialisation and state_dict keys) whose backward reads its input from an
    8-bit checkpoint (linear_act8)."""

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return linear_act8(x, self.weight, self.bias)


class _LogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, scores, items, k, scale):
        ctx.set_materialize_grads(False)
        rows = scores if scores.dim() != 2 or scores.stride(1) == 1 else scores.contiguous()
        r = kernels.log_prob_fwd(rows, items, k, scale)
        ctx.save_for_backward(scores, items, r.stats)
        ctx.scale = scale
        # entropy and lse are rows of stats: outputs of their own, so that the saved rows stay what the backward reads
        entropy, lse = r.entropy.clone(), r.lse.clone()
        ctx.mark_non_differentiable(*[t for t in (lse, r.top_items, r.top_logp, r.stats) if t is not None])
        return r.logp, entropy, lse, r.top_items, r.top_logp, r.stats

    @staticmethod
    @once_differentiable
    def backward(ctx, dlogp, dentropy, *_):
        scores, items, stats = ctx.saved_tensors
        if dlogp is None and dentropy is None:
            return None, None, None, None
        dlogp = torch.zeros(items.shape, dtype=torch.float32, device=scores.device) if dlogp is None else \
            dlogp.contiguous()
        ds = kernels.log_prob_bwd(_rows(scores), items, stats, dlogp,
                                  None if dentropy is None else dentropy.contiguous(), ctx.scale)
        return ds, None, None, None


def log_probs(scores: torch.Tensor, items: torch.Tensor, k: int = 0, scale: float = 1.0) -> kernels.LogProbs:
    """kernels.log_prob_fwd with a gradient: ``logp`` and ``entropy`` are differentiable in the scores, the other results
    are not.  A listwise training loss is ``-log_probs(scores, items).logp.mean()``."""
    return kernels.LogProbs(*_LogProbs.apply(scores, items, k, scale))
