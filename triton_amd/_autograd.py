"""What the operators' autograd functions share."""
from __future__ import annotations

import functools

import torch


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
