"""Row operators and autograd without a GPU."""
import types

import pytest
import torch

from triton_amd import _native as nt
from triton_kernels.distill import distill_topk
from triton_kernels.layer_norm import layer_norm
from triton_kernels.logprobs import token_logprobs

T, V, K, C = 6, 40, 5, 24


def _inputs():
    z, tokens = torch.randn((T, V)), torch.randint(V, (T, ))
    q, at = torch.randn((T, K)), torch.randint(V, (T, K))
    return z, tokens, q, at, torch.randn((T, C)), torch.randn(C), torch.randn(C)


def _calls():
    z, tokens, q, at, x, w, b = _inputs()
    return ((lambda t: token_logprobs(t, tokens, 3).logprobs, z), (lambda t: distill_topk(t, q, at), z), (lambda t: layer_norm(t, w, b), x),
            (lambda t: layer_norm(x, t, b), w), (lambda t: layer_norm(x, w, t), b))


def test_captures_are_checked_for_the_tensors_of_the_caller(monkeypatch):
    """With the two questions of the check answered by stubs: "is the stream being captured" with yes, "is it kept by the default stream" for leaves.
    Rows that are copied for their strides are asked for as they come."""
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    monkeypatch.setattr(nt, "rules", lambda: types.SimpleNamespace(kept_by_default_stream=lambda t: t.requires_grad and t.grad_fn is None))
    for f, t in _calls():
        strided = t.t().contiguous().t() if t.ndim == 2 else torch.stack((t, t), 1)[:, 0]
        for leaf in (t.clone(), strided.detach()):
            with pytest.raises(RuntimeError, match="same leaf"):
                f(leaf.requires_grad_())
            with pytest.raises(RuntimeError, match="HIP device"), torch.no_grad():
                f(leaf)


def test_forward_mode_is_refused():
    """Dual tensors ask for no gradient; without a refusal the result would be that of the primal, with a derivative of zero."""
    import torch.autograd.forward_ad as fwad
    z, tokens, q, at, x, w, b = _inputs()
    calls = _calls() + ((lambda t: distill_topk(z, t, at), q), )
    for f, t in calls:
        with pytest.raises(NotImplementedError, match="forward mode"), fwad.dual_level():
            f(fwad.make_dual(t, torch.ones_like(t)))
        with pytest.raises((NotImplementedError, RuntimeError), match="forward mode|storage"):
            torch.func.jvp(f, (t, ), (torch.ones_like(t), ))
        with fwad.dual_level(), pytest.raises(RuntimeError, match="HIP device"):  # (others are taken in such a level)
            fwad.make_dual(t, torch.ones_like(t))
            f(t)


def test_forward_mode_is_refused_by_the_other_differentiable_operators():
    import torch.autograd.forward_ad as fwad
    from triton_kernels.reduce import reduce
    from triton_kernels.topk import topk
    x, y, scale = torch.randn((T, 8)), torch.randn((T, 2, 16)), torch.rand((T, 2, 1))
    for f, t in ((lambda s: topk(s, 2), x), (lambda s: reduce(s, 1), y), (lambda s: reduce(y, 1, scale=s), scale)):
        with pytest.raises(NotImplementedError, match="forward mode"), fwad.dual_level():
            f(fwad.make_dual(t, torch.ones_like(t)))
        with pytest.raises(RuntimeError, match="HIP device"):
            f(t)
