"""The row operators where autograd does more than call their backward pass: other streams than the default one, captures, hooks on saved tensors,
recomputation."""
import pytest
import torch

from triton_amd import _native as nt
from triton_kernels.distill import distill_topk
from triton_kernels.layer_norm import layer_norm
from triton_kernels.logprobs import token_logprobs

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
T, V, K, C = 20, 501, 5, 72


def _inputs(dtype=F32, seed=0):
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn((T, V), generator=g) * 3).to(dtype).cuda()
    tokens = torch.randint(V, (T, ), generator=g).cuda()
    q, at = torch.randn((T, K), generator=g).cuda(), torch.randint(V, (T, K), generator=g).cuda()
    x, w, b = (torch.randn(s, generator=g).cuda() for s in ((T, C), C, C))
    return z, tokens, q, at, x.to(dtype), w, b


def _calls(z, tokens, q, at, x, w, b):
    """(operator of one tensor to differentiate, that tensor)"""
    return ((lambda t: token_logprobs(t, tokens, 3).logprobs, z), (lambda t: token_logprobs(t, tokens, 3).entropy, z), (lambda t: distill_topk(t, q, at), z),
            (lambda t: layer_norm(t, w, b), x), (lambda t: layer_norm(x, t, b), w), (lambda t: layer_norm(x, w, t), b))


def test_native_nodes_on_a_side_stream():
    """Also where the leaves belong to a graph of the default stream, and with the same results."""
    for f, t in _calls(*_inputs()):
        leaf = t.clone().requires_grad_()
        living = f(leaf)
        want, = torch.autograd.grad(living.square().sum(), leaf, retain_graph=True)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            y = f(leaf)
            got, = torch.autograd.grad(y.square().sum(), leaf)
        torch.cuda.synchronize()
        assert type(y.grad_fn) is type(living.grad_fn)
        assert torch.equal(y, living) and torch.equal(got, want)
        del living


@pytest.mark.parametrize("native", [True, False])
def test_captures_of_what_was_made_of_a_living_graphs_leaves_are_refused(native, monkeypatch):
    """Transposed leaves, views and casts of leaves, results of the default stream; without gradients they are captured, and leaves of no other graph are with
    them.  The refusal comes from the forward pass: no backward pass is captured."""
    if not native:
        monkeypatch.setattr(nt, "host", lambda: None)
    for f, t in _calls(*_inputs()):
        turned = t.t().contiguous().t() if t.ndim == 2 else torch.stack((t, t), 1)[:, 0]
        fresh = t.clone().requires_grad_()
        for leaf, made in ((turned.detach(), lambda s: s), (t.clone(), lambda s: s.view(s.shape)), (t.clone(), lambda s: s.to(BF16)), (t.clone(), lambda s: (s * 2).exp())):
            leaf.requires_grad_()
            living = f(made(leaf))
            before = made(leaf)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                for s in (lambda: made(leaf), lambda: before):
                    with pytest.raises(RuntimeError, match="same leaf"):
                        f(s())
                with torch.no_grad():
                    out = f(made(leaf))
                own = f(fresh)
                g, = torch.autograd.grad(own.sum(), fresh)
            own, want = own.detach(), f(t)
            for _ in range(2):
                graph.replay()
                torch.cuda.synchronize()
                assert torch.equal(out, living) and torch.equal(own, want) and g.isfinite().all()
            assert torch.autograd.grad(living.sum(), leaf)[0].isfinite().all()
            del living, before


def _both(monkeypatch, native):
    if not native:
        monkeypatch.setattr(nt, "host", lambda: None)


def _gradient(f, leaf):
    y = f(leaf)
    return y.detach(), torch.autograd.grad(y.square().sum(), leaf)[0]


HOOKS = {"offloaded": (lambda t: t.cpu(), lambda t: t.cuda()),
         "other strides": (lambda t: (t.ndim, t.t().contiguous() if t.ndim == 2 else torch.stack((t, t), -1)), lambda p: p[1].t() if p[0] == 2 else p[1][..., 0]),
         "rows between others": (lambda t: torch.stack((t, t), 1), lambda t: t[:, 1])}


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("hook", list(HOOKS))
def test_saved_tensors_that_come_back_otherwise(hook, native, monkeypatch):
    _both(monkeypatch, native)
    for dtype in (F32, BF16):
        for f, t in _calls(*_inputs(dtype)):
            leaf = t.clone().requires_grad_()
            want = _gradient(f, leaf)
            with torch.autograd.graph.saved_tensors_hooks(*HOOKS[hook]):
                got = _gradient(f, leaf)
            assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("native", [True, False])
def test_saved_tensors_that_are_not_what_was_saved(native, monkeypatch):
    """Refused by the backward pass on the host: another device, other sizes, a type that their place does not take."""
    _both(monkeypatch, native)
    wrong = {"left on the host": lambda t: t.cpu(), "fewer": lambda t: t[:-1], "in 64 bits": lambda t: t.double(), "flat": lambda t: t[None]}
    for unpack in wrong.values():
        for f, t in _calls(*_inputs()):
            leaf = t.clone().requires_grad_()
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
                y = f(leaf)
            with pytest.raises((RuntimeError, ValueError, NotImplementedError)):
                torch.autograd.grad(y.sum(), leaf)
    x = torch.randn((6, 40), device="cuda", requires_grad=True)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.to(BF16), lambda t: t.float()):  # (rows kept in fewer bits are those rows)
        y = layer_norm(x)
    g, = torch.autograd.grad(y.sum(), x)
    assert g.dtype == F32 and g.isfinite().all()


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("reentrant", [True, False])
def test_recomputed_in_the_backward_pass(reentrant, native, monkeypatch):
    from torch.utils.checkpoint import checkpoint
    _both(monkeypatch, native)
    for f, t in _calls(*_inputs()):
        leaf = t.clone().requires_grad_()
        want = _gradient(f, leaf)
        y = checkpoint(lambda u: f(u * 1), leaf, use_reentrant=reentrant)
        y.square().sum().backward()
        assert torch.equal(y, want[0]) and torch.equal(leaf.grad, want[1])


@pytest.mark.parametrize("native", [True, False])
def test_other_transforms_are_refused(native, monkeypatch):
    """Forward mode, whose dual tensors ask for no gradient, with and without a leaf beside them; vmap and grad of torch.func."""
    import torch.autograd.forward_ad as fwad
    _both(monkeypatch, native)
    z, tokens, q, at, x, w, b = _inputs()
    for f, t in _calls(z, tokens, q, at, x, w, b) + ((lambda s: distill_topk(z, s, at), q), (lambda s: layer_norm(x.clone().requires_grad_(), s, b), w)):
        want = f(t)
        with fwad.dual_level():
            with pytest.raises(NotImplementedError, match="forward mode"):
                f(fwad.make_dual(t, torch.ones_like(t)))
            assert torch.equal(f(t), want)
        for call in (lambda: torch.func.jvp(f, (t, ), (torch.ones_like(t), )), lambda: torch.func.vmap(f)(torch.stack((t, t))),
                     lambda: torch.func.grad(lambda s: f(s).sum())(t)):
            with pytest.raises((RuntimeError, NotImplementedError)):
                call()
        assert torch.equal(f(t), want)


@pytest.mark.parametrize("turned", [True, False])
@pytest.mark.parametrize("native", [True, False])
def test_results_changed_in_place(native, turned, monkeypatch):
    """A mask over the log probabilities before they are added up; the entropies are theirs alone."""
    _both(monkeypatch, native)
    z, tokens, *_ = _inputs()
    leaf = (z.t().contiguous().t() if turned else z.clone()).requires_grad_()
    mask = (torch.arange(T, device="cuda") % 3 != 0).float()
    want = token_logprobs(leaf, tokens)
    g, = torch.autograd.grad((want.logprobs * mask).sum() + want.entropy.sum(), leaf)
    r = token_logprobs(leaf, tokens)
    r.logprobs.mul_(mask)
    assert torch.equal(r.entropy, want.entropy) and torch.equal(r.logprobs, want.logprobs * mask)
    assert torch.equal(torch.autograd.grad(r.logprobs.sum() + r.entropy.sum(), leaf)[0], g)
    y = layer_norm(z.clone().requires_grad_())
    loss = distill_topk(leaf, *_inputs()[2:4])
    for out in (y, loss):
        out.mul_(2).sum().backward()
