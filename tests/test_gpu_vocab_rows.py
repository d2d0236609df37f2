"""Log probabilities of tokens, entropies and alternatives, and distillation from top logits, with their gradients, against the 64-bit oracle: from
one column to half a million, the three types, ties, masks of -inf and of the lowest value, rows that are no distribution, padding,
strided and shifted rows, tokens and teacher entries out of range or named twice; other streams, graph capture, a run of them together."""
import math

import pytest
import torch

from oracle import rows as orc
from triton_amd import _native as nt
from triton_kernels.distill import _forward as distill_forward
from triton_kernels.distill import distill_topk, distill_topk_backward
from triton_kernels.layer_norm import layer_norm
from triton_kernels.logprobs import _forward as logprobs_forward
from triton_kernels.logprobs import check_logits, token_logprobs, token_logprobs_backward

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
INF = float("inf")
SIZES = [(1, 1), (1, 2), (2, 5), (3, 63), (4, 64), (5, 65), (7, 1000), (2, 2049), (2, 4097), (9, 8192), (3, 32000), (2, 50001), (1, 131072), (300, 513)]


def _logits(T, V, dtype, seed=0):
    g = torch.Generator().manual_seed(seed * 7919 + T * 131 + V)
    z = torch.randn((T, V), generator=g) * 2.5 + torch.randn((T, 1), generator=g) * 3 - 4
    z.scatter_add_(1, torch.randint(V, (T, 8), generator=g), torch.rand((T, 8), generator=g) * 12)
    tokens = torch.randint(V, (T, ), generator=g)
    return z.to(dtype).cuda(), tokens.cuda(), torch.randn(T, generator=g).cuda(), (torch.randn(T, generator=g) * 0.1).cuda()


def _teacher(logits, K, seed=0, dtype=None):
    T, V = logits.shape
    g = torch.Generator().manual_seed(seed * 31 + T + V + K)
    at = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(T)]).to(torch.int32)
    q = (torch.randn((T, K), generator=g) * 2).to(dtype or logits.dtype)
    return q.cuda(), at.cuda()


def _check_logprobs(z, tokens, k, t=1.0, grads=None):
    lp, h, top_lp, top, stats = logprobs_forward(check_logits(z, t), tokens, k, t, True)
    want = orc.token_logprobs(z, tokens, k, t)
    orc.check(lp, *want["logprobs"], "logprobs")
    orc.check(h, *want["entropy"], "entropy")
    if k:
        assert top.dtype == torch.int32 and torch.equal(top.cpu().long(), want["top_indx"][0])
        orc.check(top_lp, *want["top_logprobs"], "top_logprobs")
    else:
        assert top is None and top_lp is None
    if grads is not None:
        for a, b in (grads, (grads[0], None), (None, grads[1])):
            g = token_logprobs_backward(z, tokens, h, stats, a, b, t)
            assert g.dtype == z.dtype and g.is_contiguous()
            orc.check(g, *orc.token_logprobs_backward(z, tokens, a, b, t), "dlogits")
    return lp, h, top_lp, top


def _check_distill(z, q, at, t=1.0, grad=None):
    loss, stats = distill_forward(check_logits(z, t), q, at, t, True)
    orc.check(loss, *orc.distill_topk(z, q, at, t), "loss")
    if grad is not None:
        g = distill_topk_backward(z, q, at, stats, grad, t)
        assert g.dtype == z.dtype and g.is_contiguous()
        orc.check(g, *orc.distill_topk_backward(z, q, at, grad, t), "dlogits")
    return loss


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("T,V", SIZES)
def test_logprobs_sizes_and_types(T, V, dtype):
    z, tokens, a, b = _logits(T, V, dtype)
    _check_logprobs(z, tokens, min(20, V), 1.0, (a, b))
    _check_logprobs(z, tokens.int(), 0, 0.7, (a, b))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("T,V", SIZES)
def test_distill_sizes_and_types(T, V, dtype):
    z, _, a, _ = _logits(T, V, dtype)
    for K in {1, min(V, 16), min(V, 100)}:
        _check_distill(z, *_teacher(z, K), 1.0, a)
    _check_distill(z, *_teacher(z, min(V, 7), dtype=F32), 2.0, a)


@pytest.mark.parametrize("k", [1, 2, 3, 31, 64, 65, 127, 128])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_numbers_of_alternatives(k, dtype):
    for T, V in ((3, 128), (2, 5000), (2, 70001)):
        z, tokens, _, _ = _logits(T, V, dtype)
        _check_logprobs(z, tokens, k)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_ties_go_to_the_lower_index(dtype):
    g = torch.Generator().manual_seed(3)
    for V in (200, 4096, 30011):
        z = torch.randint(-3, 3, (6, V), generator=g).to(dtype).cuda()
        z[1] = 0.0
        z[2] = torch.where(torch.rand(V, generator=g) < 0.5, 0.0, -0.0).to(dtype)  # the two zeros are one value
        z[3] = -5.0
        z[3, V - 70:] = 7.0  # more of the largest than asked for, at the end
        z[4] = -INF
        z[4, V // 2::3] = 1.0
        z[5] = torch.linspace(-4, 4, V).to(dtype)
        for k in (1, 20, 64, 100):
            _check_logprobs(z, torch.zeros(6, dtype=torch.int64, device="cuda"), k)
            _check_logprobs(z.flip(1), torch.zeros(6, dtype=torch.int64, device="cuda"), k)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("V", [70, 3000, 40000])
def test_sorted_rows(V, dtype):
    """The largest logits all side by side, at either end or in the middle."""
    up = torch.linspace(-20, 8, V)
    z = torch.stack((up, up.flip(0), torch.roll(up, V // 2))).to(dtype).cuda()
    for k in (1, 50, min(V, 128)):
        _check_logprobs(z, torch.tensor([0, V - 1, V // 3], device="cuda"), k)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("V", [33, 1000, 20001])
def test_masked_logits(V, dtype):
    """Half of a vocabulary ruled out, all but one, all but a few that stand at the end; with -inf and with the type's lowest value."""
    for low in (-INF, torch.finfo(dtype).min):
        z, tokens, a, b = _logits(5, V, dtype)
        g = torch.Generator().manual_seed(V)
        z.masked_fill_((torch.rand(V, generator=g) < 0.5).cuda(), low)
        z[1] = low
        z[1, V // 2] = 0.5
        z[2, :V - 3] = low
        tokens[0] = int(z[0].argmax())
        tokens[1] = V // 2
        tokens[2] = 0
        _check_logprobs(z, tokens, min(V, 40), 1.0, (a, b))
        q, at = _teacher(z, 9)
        _check_distill(z, q, at, 1.0, a)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T,V", [(6, 30000), (1001, 1500), (1001, 20003)])
@pytest.mark.parametrize("low", [-5e4, -1e9, -1e10, -1e20, -1e30])
def test_masked_with_large_numbers(T, V, dtype, low):
    """Masks whose products with log2(e) are further from whole numbers than an exponent can hold: in front of the logits that count, behind
    them, in every other place, everywhere."""
    z, tokens, a, b = _logits(T, V, dtype)
    z[0::6, :V - 40] = low
    z[1::6, 40:] = low
    z[2::6, ::2] = low
    z[3::6] = low
    z[4::6, :V // 2] = low
    z[4::6, V // 2:] = 2 * low
    tokens[0::6] = V - 1
    q, at = _teacher(z, 9)
    n, k = 12, 20  # (rows that are compared; the others are there for the kernels that many rows have)
    for t in (1.0, 0.7):
        lp, h, top_lp, top, stats = logprobs_forward(z, tokens, k, t, True)
        loss, distill_stats = distill_forward(z, q, at, t, True)
        want = orc.token_logprobs(z[:n], tokens[:n], k, t)
        assert torch.equal(top[:n].cpu().long(), want["top_indx"][0])
        for name, got in (("logprobs", lp), ("entropy", h), ("top_logprobs", top_lp)):
            orc.check(got[:n], *want[name], name)
        orc.check(loss[:n], *orc.distill_topk(z[:n], q[:n], at[:n], t), "loss")
        g = token_logprobs_backward(z, tokens, h, stats, a, b, t)
        orc.check(g[:n], *orc.token_logprobs_backward(z[:n], tokens[:n], a[:n], b[:n], t), "dlogits")
        g = distill_topk_backward(z, q, at, distill_stats, a, t)
        orc.check(g[:n], *orc.distill_topk_backward(z[:n], q[:n], at[:n], a[:n], t), "dlogits of the distillation")


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("V", [5, 777, 9000])
def test_rows_that_are_no_distribution(V, dtype):
    z, tokens, a, b = _logits(10, V, dtype)
    z[1] = -INF
    z[2] = torch.finfo(dtype).min  # a uniform row
    z[3, V // 2] = float("nan")
    z[4, V - 1] = INF
    z[5, 0], z[5, 1] = INF, float("nan")
    z[6] = -INF
    z[6, V // 3] = float("nan")
    z[7] = INF
    z[8] = torch.finfo(dtype).max / 2  # another
    tokens[4] = V - 1
    _check_logprobs(z, tokens, min(V, 6), 1.0, (a, b))
    q, at = _teacher(z, min(V, 6))
    _check_distill(z, q, at, 1.0, a)


def test_large_logits_of_either_sign():
    for c in (1e4, 3e4, 1e30, 3e38):
        z = torch.tensor([[c, -c, 0.0, c, 1.0], [-c, -c, -c, -c, -c], [c, c, c, c, c]], device="cuda")
        tokens = torch.tensor([3, 0, 4], device="cuda")
        lp, h, _, top = _check_logprobs(z, tokens, 3)
        assert torch.allclose(h.cpu(), torch.tensor([math.log(2), math.log(5), math.log(5)]))
        assert top.tolist() == [[0, 3, 4], [0, 1, 2], [0, 1, 2]]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T,V", [(5, 20001), (1001, 700)])
@pytest.mark.parametrize("temperature", [2.0**-100, 2.0**-20, 2.0**20, 2.0**100])
def test_temperatures_far_from_one(T, V, dtype, temperature):
    z, tokens, a, b = _logits(T, V, dtype)
    z[2] = z[2].round()  # (several largest ones)
    _check_logprobs(z, tokens, 7, temperature, (a, b))
    q, at = _teacher(z, 9)
    _check_distill(z, q, at, temperature, a)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_tokens_out_of_range_and_no_gradient(dtype):
    z, tokens, a, b = _logits(8, 3001, dtype)
    tokens[0], tokens[1], tokens[2], tokens[3] = -1, -100, 3001, 2**40
    z[2, 5] = float("nan")
    lp, h, _, _ = _check_logprobs(z, tokens, 4, 1.0, (a, b))
    assert not lp[:4].any()
    a[5], b[5] = 0, 0
    _check_logprobs(z, tokens, 0, 1.0, (a, b))
    i32 = tokens.clone().clamp(-(2**31), 2**31 - 1).int()
    for x, y in zip(_check_logprobs(z, i32, 4), _check_logprobs(z, tokens, 4)):
        assert torch.equal(x.nan_to_num(), y.nan_to_num())


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_teacher_entries_that_do_not_count(dtype):
    V = 2500
    z, _, a, _ = _logits(12, V, dtype)
    q, at = _teacher(z, 10)
    at[0, 3:] = -1
    at[1] = V
    at[2] = -1
    q[3] = -INF
    q[4, ::2] = -INF
    q[5, 4] = float("nan")
    q[6, 0] = INF
    q[7, 0] = float("nan")
    at[7, 0] = -1
    z[8, at[8, 0].long()] = -INF  # a student that rules out what the teacher holds possible
    at[9] = at[9, 0]  # the same index ten times
    at[10, 5], at[10, 9] = at[10, 0], at[10, 2]
    z[2] = float("nan")
    loss = _check_distill(z, q, at, 1.0, a)
    assert loss[8].item() == INF and not loss[1:4].any()
    _check_distill(z, q, at.long() + 0, 0.7, a)
    big = at.long()
    big[0, 3] = 2**33 + 1
    _check_distill(z, q, big, 1.0, a)
    _check_distill(z, q[:, :0], at[:, :0], 1.0, a)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("first", [1, 3, 5, 7])
def test_padding_beside_rows_that_begin_between_boundaries(first, dtype):
    """Entries and tokens of -1 where a row's loads begin in front of its first column: nothing in front of it is read or written."""
    for T, V in ((7, 501), (5, 20003), (1200, 301)):
        wide, tokens, a, b = _logits(T, V + 8, dtype)
        z = wide[:, first:first + V]
        tokens = tokens % V
        tokens[::2] = -1
        q, at = _teacher(z, 9)
        at[:, ::2] = -1
        at[1::3, 1] = 0
        at[2::3, 3] = V - 1
        _check_distill(z, q, at, 1.0, a)
        wide[:, :first] = float("nan")
        wide[:, first + V:] = INF
        _check_logprobs(z, tokens, 5, 1.0, (a, b))
        _check_distill(z, q, at, 1.0, a)


def test_the_largest_number_of_teacher_entries():
    z, _, a, _ = _logits(3, 5003, BF16)
    _check_distill(z, *_teacher(z, 1024, dtype=F32), 1.0, a)
    _check_distill(z, *_teacher(z, 1023, dtype=F16), 1.0, a)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("V", [64, 1001, 20000])
def test_rows_at_any_stride_and_address(V, dtype):
    wide, tokens, a, b = _logits(9, 2 * V + 5, dtype)
    tokens = tokens % V
    for z in (wide[:, 1:V + 1], wide[:, V + 3:2 * V + 3], wide[::2, 2:V + 2], wide[:, :V].t().contiguous().t(), wide[:1, 3:V + 3].expand(9, V)):
        n = z.shape[0]
        _check_logprobs(z, tokens[:n], 17, 1.0, (a[:n], b[:n]))
        q, at = _teacher(z, 20)
        _check_distill(z, q, at, 1.0, a[:n])
        _check_distill(z, torch.cat((q, q), 1)[:, 3:13], torch.cat((at, at), 1)[:, 3:13], 1.0, a[:1].expand(n))
    pairs = torch.stack((tokens, tokens), 1)
    _check_logprobs(wide[:, :V], pairs[:, 1], 3, 1.0, (torch.stack((a, b), 1)[:, 0], b[:1].expand(9)))


def test_the_widest_vocabulary():
    z, tokens, a, b = _logits(1, 524288, BF16)
    z[0, 524287] = 30.0
    _check_logprobs(z, tokens, 128, 1.0, (a, b))
    z, tokens, a, b = _logits(1, 600001, F32)
    _check_logprobs(z, tokens, 0, 1.0, (a, b))
    _check_distill(z, *_teacher(z, 50), 1.0, a)


def test_no_rows():
    z, tokens, a, b = _logits(4, 100, BF16)
    r = token_logprobs(z[:0], tokens[:0], 5)
    assert r.logprobs.shape == (0, ) and r.top_indx.shape == (0, 5)
    leaf = z[:0].clone().requires_grad_()
    r = token_logprobs(leaf, tokens[:0], 5)
    assert torch.autograd.grad(r.logprobs.sum(), leaf)[0].shape == (0, 100)
    q, at = _teacher(z, 3)
    leaf = z[:0].clone().requires_grad_()
    assert torch.autograd.grad(distill_topk(leaf, q[:0], at[:0]).sum(), leaf)[0].shape == (0, 100)


@pytest.mark.parametrize("native", [True, False])
def test_autograd(native, monkeypatch):
    """Through the native host path and through the general one."""
    if not native:
        monkeypatch.setattr(nt, "host", lambda: None)
    z, tokens, a, b = _logits(40, 3001, F32)
    lp, h, _, _, stats = logprobs_forward(z, tokens, 6, 0.7, True)
    for ga, gb in ((a, b), (a, None), (None, b)):
        leaf = z.clone().requires_grad_()
        r = token_logprobs(leaf, tokens, 6, temperature=0.7)
        assert torch.equal(r.logprobs, lp) and torch.equal(r.entropy, h)
        assert not r.top_logprobs.requires_grad and not r.top_indx.requires_grad
        outs = [(o, g) for o, g in ((r.logprobs, ga), (r.entropy, gb)) if g is not None]
        torch.autograd.backward([o for o, _ in outs], [g for _, g in outs])
        assert torch.equal(leaf.grad, token_logprobs_backward(z, tokens, h, stats, ga, gb, 0.7))
    leaf = z.clone().requires_grad_()
    token_logprobs(leaf, tokens).logprobs.sum().backward()  # a gradient of one value for all rows
    orc.check(leaf.grad, *orc.token_logprobs_backward(z, tokens, torch.ones(1), None), "dlogits")
    q, at = _teacher(z, 12)
    leaf = z.clone().requires_grad_()
    distill_topk(leaf, q, at, temperature=2.0).mean().backward()
    orc.check(leaf.grad, *orc.distill_topk_backward(z, q, at, torch.full((1, ), 1 / 40), 2.0), "dlogits")
    leaf = z.clone().requires_grad_()
    for f in (lambda t: distill_topk(t, q, at), lambda t: token_logprobs(t, tokens, 3).entropy):
        g, = torch.autograd.grad(f(leaf).sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiable once"):
            g.sum().backward()
    turned = z.t().contiguous().t().requires_grad_()  # (goes the general way)
    token_logprobs(turned, tokens, temperature=0.7).logprobs.backward(a)
    assert torch.equal(turned.grad, token_logprobs_backward(z, tokens, h, stats, a, None, 0.7))
    with torch.no_grad():
        assert not token_logprobs(leaf, tokens).logprobs.requires_grad
    with pytest.raises(NotImplementedError, match="teacher"):
        distill_topk(leaf, q.clone().requires_grad_(), at)


@pytest.mark.parametrize("V", [1000, 9001])
def test_many_rows(V):
    z, tokens, a, b = _logits(1500, V, BF16)
    _check_logprobs(z, tokens, 9, 1.0, (a, b))
    _check_distill(z, *_teacher(z, 9), 1.0, a)


def _everything(z, tokens, q, at, a, b):
    lp, h, tlp, top, stats = logprobs_forward(z, tokens, 20, 1.0, True)
    loss, dstats = distill_forward(z, q, at, 1.0, True)
    return (lp, h, tlp, top, token_logprobs_backward(z, tokens, h, stats, a, b), loss, distill_topk_backward(z, q, at, dstats, a))


def test_equal_calls_give_equal_bits_on_any_stream():
    sets = []
    for T, V in ((3, 60001), (200, 5000)):
        z, tokens, a, b = _logits(T, V, BF16)
        sets.append((z, tokens, *_teacher(z, 30), a, b))
    want = [_everything(*s) for s in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(_everything(*sets[i]))
    torch.cuda.synchronize()
    for i in (0, 1):
        for out in got[i]:
            for x, y in zip(out, want[i]):
                assert torch.equal(x, y)


@pytest.mark.parametrize("T,V", [(2, 30001), (120, 3000)])
def test_in_graphs_that_are_replayed_in_turn(T, V):
    graphs, ins, outs = [], [], []
    for i in (0, 1):
        z, tokens, a, b = _logits(T, V, BF16, seed=i)
        ins.append((z, tokens, *_teacher(z, 30), a, b))
        _everything(*ins[i])
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_everything(*ins[i]))
        graphs.append(g)
    for seed in (5, 6, 7):
        for i in (0, 1):
            ins[i][0].copy_(_logits(T, V, BF16, seed=seed + 10 * i)[0])
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        torch.cuda.synchronize()
        for i in (0, 1):
            for x, y in zip(outs[i], _everything(*ins[i])):
                assert torch.equal(x, y)


def test_training_steps_in_a_graph():
    """Forward and backward passes through autograd, captured together and replayed with other inputs between eager steps."""
    T, V, K = 60, 3001, 20
    z, tokens, a, b = _logits(T, V, BF16)
    q, at = _teacher(z, K)
    leaf = z.clone().requires_grad_()

    def step(leaf):
        r = token_logprobs(leaf, tokens, 5)
        g1, = torch.autograd.grad((r.logprobs, r.entropy), leaf, (a, b))
        loss = distill_topk(leaf, q, at, temperature=2.0)
        g2, = torch.autograd.grad(loss, leaf, a)
        y = layer_norm(leaf)
        g3, = torch.autograd.grad(y, leaf, g2)
        return r.logprobs.detach(), r.entropy.detach(), r.top_indx, g1, loss.detach(), g2, y.detach(), g3

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(leaf)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(leaf)
    for seed in (3, 4, 5):
        new = _logits(T, V, BF16, seed=seed)[0]
        with torch.no_grad():
            leaf.copy_(new)
        graph.replay()
        want = step(new.clone().requires_grad_())
        torch.cuda.synchronize()
        for x, y in zip(out, want):
            assert torch.equal(x, y)


@pytest.mark.parametrize("native", [True, False])
def test_a_capture_beside_a_living_graph_of_the_same_leaves_is_refused(native, monkeypatch):
    """The refusal comes from the forward pass; nothing of a backward pass is captured while the leaves' gradients belong to the default stream."""
    if not native:
        monkeypatch.setattr(nt, "host", lambda: None)
    z, tokens, a, _ = _logits(20, 500, BF16)
    q, at = _teacher(z, 5)
    x, w, b = (torch.randn(s, device="cuda") for s in ((20, 64), 64, 64))
    leaf, w = z.clone().requires_grad_(), w.requires_grad_()
    calls = (lambda: token_logprobs(leaf, tokens).logprobs, lambda: distill_topk(leaf, q, at), lambda: layer_norm(x, w, b))
    for f, wrt in zip(calls, (leaf, leaf, w)):
        living = f()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            doubled = a * 2
            with pytest.raises(RuntimeError, match="same leaf"):
                f()
            with torch.no_grad():
                out = f()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, living) and torch.equal(doubled, a * 2)
        assert torch.autograd.grad(living.sum(), wrt)[0].isfinite().all()
        del living


def test_calls_from_several_threads():
    import threading
    sets, want, got = [], [], [None] * 4
    for i in range(4):
        z, tokens, a, b = _logits(30 + i, 4000 + 111 * i, F16, seed=i)
        sets.append((z, tokens, *_teacher(z, 30), a, b))
        want.append(_everything(*sets[i]))
    torch.cuda.synchronize()

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                got[i] = _everything(*sets[i])
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i, )) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(4):
        for x, y in zip(got[i], want[i]):
            assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_many_short_rows(dtype):
    """Rows that have a wave each: with few and many alternatives, ties, masks, rows that are no distribution, more teacher entries than a wave holds."""
    for T, V in ((1000, 1), (1100, 37), (1003, 1000), (1500, 2047), (1024, 2049), (1000, 8192)):
        z, tokens, a, b = _logits(T, V, dtype)
        z[3] = -INF
        z[4, V // 2] = float("nan")
        z[5] = 2.0
        z[6, : V // 2] = -INF
        z[7] = torch.finfo(dtype).min
        tokens[8] = -1
        for k in {min(V, 1), min(V, 32), min(V, 33), min(V, 128)}:
            _check_logprobs(z, tokens, k, 1.0, (a, b) if k == min(V, 32) else None)
        _check_logprobs(z, tokens, 0, 0.5, (a, b))
        for K in {min(V, 5), min(V, 256), min(V, 300)}:
            _check_distill(z, *_teacher(z, K, dtype=F32), 1.0, a)


def test_rows_beyond_32_bit_offsets():
    T, V = 40000, 60000  # 4.8 GB
    z = torch.zeros((T, V), dtype=BF16, device="cuda")
    small, tokens, a, b = _logits(3, V, BF16)
    z[-3:] = small
    tok = torch.zeros(T, dtype=torch.int64, device="cuda")
    tok[-3:] = tokens
    leaf = z.requires_grad_()
    r = token_logprobs(leaf, tok, 5)
    want = orc.token_logprobs(small, tokens, 5)
    for name in ("logprobs", "entropy", "top_logprobs"):  # (few rows are summed in pieces, so that the bits are those of the number of rows)
        orc.check(getattr(r, name)[-3:], *want[name], name)
    assert torch.equal(r.top_indx[-3:].cpu().long(), want["top_indx"][0])
    assert r.top_indx[T // 2].tolist() == [0, 1, 2, 3, 4]
    ga = torch.zeros(T, device="cuda")
    ga[-3:] = a
    g, = torch.autograd.grad(r.logprobs, leaf, ga)
    orc.check(g[-3:], *orc.token_logprobs_backward(small, tokens, a, None), "dlogits")
    assert not g[:-3].any()


def test_teacher_and_student_together():
    """A teacher's and a student's last norm and projection, the teacher's top logits taken, the student's gradient brought back to the
    norm's parameters: against the same chain in 64 bits from the student's own logits on."""
    g = torch.Generator().manual_seed(0)
    T, C, V, K = 24, 96, 1501, 12
    x = torch.randn((T, C), generator=g).cuda()
    w, b = (torch.randn(C, generator=g) * 0.1 + 1).cuda(), (torch.randn(C, generator=g) * 0.1).cuda()
    head, head_t = (torch.randn((V, C), generator=g) * 0.3).cuda(), (torch.randn((V, C), generator=g) * 0.3).cuda()
    tokens = torch.randint(V, (T, ), generator=g).cuda()
    teacher = token_logprobs(layer_norm(x, w, b) @ head_t.t(), tokens, K)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    logits = layer_norm(*leaves) @ head.t()
    logits.retain_grad()
    loss = distill_topk(logits, teacher.top_logprobs, teacher.top_indx, temperature=1.5)
    loss.mean().backward()
    want, bound = orc.distill_topk(logits, teacher.top_logprobs, teacher.top_indx, 1.5)
    orc.check(loss, want, bound, "loss")
    want, bound = orc.distill_topk_backward(logits, teacher.top_logprobs, teacher.top_indx, torch.full((1, ), 1 / T), 1.5)
    orc.check(logits.grad, want, bound, "dlogits")
    # (the product's gradient in 64 bits from the kernel's; its own rounding is 32 bits over V terms)
    dy = logits.grad.double() @ head.double()
    off = (logits.grad.double().abs() @ head.double().abs()) * V * orc.U
    grads = orc.layer_norm_backward(dy.float(), x, w, 1e-5, b)
    slack = off.sum(0).max().item() * 8 + off.max().item() * 8
    for leaf, name in zip(leaves, ("dx", "dweight", "dbias")):
        orc.check(leaf.grad, grads[name][0], grads[name][1] + slack, name)
