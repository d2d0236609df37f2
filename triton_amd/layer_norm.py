"""Layer norm of the rows of an activation, with its gradients (no counterpart in the reference's operator library).

`layer_norm` is what stands in front of a router or a projection: one pass over the rows, statistics in fp32, one rounding to
the activation's type.  Its backward pass gives the gradients of the activation, the weight and the bias; the sums over rows
are taken in an order that depends on the sizes alone, so that equal calls give equal bits.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _native as nt
from ._autograd import check_capture, check_forward_mode, once

DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def _check(x, weight, bias, eps):
    if x.ndim < 1 or x.shape[-1] == 0:
        raise ValueError(f"x must have columns to normalise (got shape {tuple(x.shape)})")
    for name, t in (("x", x), ("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if t.dtype not in DTYPES:
            raise NotImplementedError(f"layer_norm: {name} must be fp32, bf16 or fp16 (got {t.dtype})")
        if t is not x and (t.shape != x.shape[-1:] or t.device != x.device):
            raise ValueError(f"{name} must be [{x.shape[-1]}] on {x.device} (got {tuple(t.shape)} on {t.device})")
    if not 0.0 <= float(eps) < float("inf"):
        raise ValueError(f"eps must be finite and not negative (got {eps})")


def _rows(t):
    t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 else t.contiguous()


def _vector(t):
    return t if t is None or t.stride(0) == 1 else t.contiguous()


def _type(t):
    return nt.TK_F32 if t is None else nt.TORCH_TO_TK[t.dtype]


def layer_norm_forward(x, weight=None, bias=None, eps: float = 1e-5, *, with_stats: bool = True):
    """`(y, mean, rstd)`; the statistics (fp32, one a row, flattened) are None unless `with_stats`."""
    _check(x, weight, bias, eps)
    nt.require_gpu(x, "x")
    x2, weight, bias = _rows(x), _vector(weight), _vector(bias)
    M, C = x2.shape
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    mean = rstd = None
    if with_stats:
        mean, rstd = torch.empty((2, M), dtype=torch.float32, device=x.device)
    with nt.on_device(x.device):
        nt.check(
            nt.lib().tk_layer_norm(x2.data_ptr(), _type(x), M, C, x2.stride(0), nt.ptr(weight), _type(weight), nt.ptr(bias), _type(bias), eps,
                                   y.data_ptr(), C, nt.ptr(mean), nt.ptr(rstd), nt.stream_ptr(x.device)))
    return y, mean, rstd


def layer_norm_backward(dy, x, mean, rstd, weight=None, bias=None, *, need_dx: bool = True, need_dweight: bool = True, need_dbias: bool = True):
    """`(dx, dweight, dbias)` for the gradient `dy` of `layer_norm(x, weight, bias)` and its statistics; an entry is None where it is
    not needed or there is no such parameter.  Gradients have their parameters' types."""
    _check(x, weight, bias, 0.0)
    if dy.shape != x.shape or dy.device != x.device:
        raise ValueError(f"dy must be {tuple(x.shape)} on {x.device} (got {tuple(dy.shape)} on {dy.device})")
    C = x.shape[-1]
    M = x.numel() // C
    for name, t in (("mean", mean), ("rstd", rstd)):
        if t.shape != (M, ) or t.dtype != torch.float32 or t.device != x.device or not t.is_contiguous():
            raise ValueError(f"{name} must be the contiguous fp32 [{M}] of the forward pass")
    nt.require_gpu(x, "x")
    x2, dy2, weight = _rows(x), _rows(dy if dy.dtype == x.dtype else dy.to(x.dtype)), _vector(weight)
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need_dx else None
    dweight = torch.empty((C, ), dtype=weight.dtype, device=x.device) if need_dweight and weight is not None else None
    dbias = torch.empty((C, ), dtype=bias.dtype, device=x.device) if need_dbias and bias is not None else None
    ws = None
    if dweight is not None or dbias is not None:
        ws = torch.empty(nt.lib().tk_layer_norm_backward_workspace_bytes(M, C), dtype=torch.uint8, device=x.device)
    with nt.on_device(x.device):
        nt.check(
            nt.lib().tk_layer_norm_backward(dy2.data_ptr(), dy2.stride(0), x2.data_ptr(), _type(x), M, C, x2.stride(0), nt.ptr(weight), _type(weight),
                                            mean.data_ptr(), rstd.data_ptr(), nt.ptr(dx), C, nt.ptr(dweight), nt.ptr(dbias), _type(bias), nt.ptr(ws),
                                            nt.stream_ptr(x.device)))
    return dx, dweight, dbias


class _LayerNorm(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = layer_norm_forward(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, bias, mean, rstd)
        return y

    @staticmethod
    @once
    def backward(ctx, dy):
        x, weight, bias, mean, rstd = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, dweight, dbias = layer_norm_backward(dy, x, mean.contiguous(), rstd.contiguous(), weight, bias, need_dx=need[0], need_dweight=need[1], need_dbias=need[2])
        return dx, dweight, dbias, None


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, eps: float = 1e-5) -> torch.Tensor:
    """`(x - mean) / sqrt(var + eps) * weight + bias` over the last dimension of `x [..., C]` (biased variance), in x's type.

    x, weight and bias are fp32, bf16 or fp16, each its own; weight and bias are `[C]` and optional.  Rows may have any stride.
    Statistics are taken in fp32; the mean is good to its own rounding also where it is large against the deviation, and a row of equal
    elements gives the bias.  So does a row whose squared distances from its mean add up to more than fp32 holds (distances of about 1e18 on),
    which has no deviation to speak of.
    Differentiable once in all three."""
    host = nt.host()
    y = host.layer_norm(x, weight, bias, eps) if host is not None else None
    if y is not None:
        return y
    check_forward_mode("layer_norm", x, weight, bias)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        check_capture(x, weight, bias)
        return _LayerNorm.apply(x, weight, bias, eps)
    return layer_norm_forward(x, weight, bias, eps, with_stats=False)[0]


from .torch_twins import layer_norm_torch  # noqa: E402,F401  (plain twin; never called by `layer_norm`)
