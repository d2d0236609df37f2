"""What the operators' autograd functions share."""
from __future__ import annotations

import functools

import torch

from torch.autograd import forward_ad

from . import _native as nt


def check_capture(*tensors):
    """Refuses a captured call with leaves that an earlier graph on the default stream still uses, and with what was made of such leaves: their
    gradients are accumulated on that stream, and the backward pass would make it wait for the capture, which ends the process.  Asked of the
    caller's own tensors, since a copy of a leaf is no leaf."""
    if torch.cuda.is_current_stream_capturing() and any(t is not None and nt.rules().kept_by_default_stream(t) for t in tensors):
        raise RuntimeError("a result computed on the default stream from the same leaf tensors is still alive: delete it before the capture "
                           "(or compute it on another stream; without a backward pass, capture the call under torch.no_grad())")


def check_forward_mode(who, *tensors):
    """Refuses dual tensors, which ask for no gradient: an operator that computes from their primals alone would drop their tangents."""
    if forward_ad._current_level >= 0 and any(isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{who} has no derivative in forward mode")


def once(backward):
    """For the backward pass of a function that is differentiable once: gradients that are themselves to be differentiated
    (`create_graph`) raise an error when they are, whatever they were made from."""

    @functools.wraps(backward)
    def wrapper(ctx, *grads):
        with torch.no_grad():
            out = backward(ctx, *grads)
        if not torch.is_grad_enabled():
            return out
        many = out if isinstance(out, tuple) else (out, )
        node = torch._C._functions.DelayedError(b"the row operators are differentiable once", sum(t is not None for t in many))
        made = node(*[t.detach().requires_grad_() for t in many if t is not None])
        made = iter(made if isinstance(made, tuple) else (made, ))
        many = tuple(None if t is None else next(made) for t in many)
        return many if isinstance(out, tuple) else many[0]

    return wrapper
