"""Calls of the experts in 8 bits as programs make them: hooks that change what the backward pass was to read, weights
that begin at any address, other transforms than a backward pass, several threads, and a rank's own
experts."""
import pytest
import torch

from oracle import fp8_blocks as orc
from oracle.rows import check
from triton_amd import _native as nt
from triton_kernels.fp8_blocks import (downcast_to_fp8_blocks, linear_fp8_blocks, matmul_fp8_blocks, quantize_fp8_weight, swiglu_fp8_backward, swiglu_fp8_checkpoint,
                                       swiglu_fp8_forward, upcast_from_fp8_blocks, weight_gradient_fp8_blocks)
from triton_kernels.tensor import make_ragged_tensor_metadata

pytestmark = pytest.mark.gpu

F32, BF16, F16, E4M3 = torch.float32, torch.bfloat16, torch.float16, torch.float8_e4m3fn


def _both(monkeypatch, native):
    if not native:
        monkeypatch.setattr(nt, "host", lambda: None)


def _rows(g, R, C, dtype=BF16, scale=1.0):
    return (torch.randn((R, C), generator=g) * (torch.rand((R, 1), generator=g) * 2 + 0.1) * scale).to(dtype).cuda()


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,K,N", [(40, 200, 72), (2300, 4104, 264)])       # (the second one's input gradient goes by tiles of 256)
def test_scales_that_a_hook_gives_back_count_whole(T, K, N, dtype, native, monkeypatch):
    _both(monkeypatch, native)
    g = torch.Generator().manual_seed(T)
    x = _rows(g, T, K, dtype).requires_grad_()
    w = (torch.randn((1, K, N), generator=g) * 0.05).cuda().requires_grad_()
    dy = _rows(g, T, N, dtype, 0.01)
    md = make_ragged_tensor_metadata(torch.tensor([T], dtype=torch.int32, device="cuda"), T)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t * 1.25 if t.dtype == F32 else t):  # (the scales alone are fp32; three more bits)
        y = linear_fp8_blocks(x, w, md)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    x8, xs = downcast_to_fp8_blocks(x.detach())
    w8, ws = downcast_to_fp8_blocks(w.detach(), 128)
    d8, ds = downcast_to_fp8_blocks(dy)
    some = torch.arange(0, T, max(1, T // 40), device="cuda")
    check(dx[some], *orc.product(d8.view(torch.uint8)[some].view(E4M3), ds[some], w8.transpose(1, 2), ws.transpose(1, 2) * 1.25, out_dtype=dtype)[:2], "dx")
    check(dw, *orc.weight_gradient(x8, xs * 1.25, dy), "dw")


def test_scales_that_a_hook_of_one_node_gives_back_count_whole(monkeypatch):
    """Hooks on the saved tensors of a node that Python has (weights that were handed in)."""
    g = torch.Generator().manual_seed(1)
    x = _rows(g, 40, 200).requires_grad_()
    w = (torch.randn((200, 72), generator=g) * 0.05).cuda().requires_grad_()
    dy = _rows(g, 40, 72, BF16, 0.01)
    y = linear_fp8_blocks(x, w, quantized=quantize_fp8_weight(w))
    for saved in y.grad_fn._raw_saved_tensors:
        saved.register_hooks(lambda t: t, lambda t: t * 1.25 if t.dtype == F32 else t)
    dw, = torch.autograd.grad(y, w, dy)
    x8, xs = downcast_to_fp8_blocks(x.detach())
    check(dw[None], *orc.weight_gradient(x8, xs * 1.25, dy), "dw")


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("shift,apart", [(1, 0), (0, 8), (8, 0)])
@pytest.mark.parametrize("M", [900, 2**21 + 100])                          # (beyond 2^21 rows in slices only the kernels for lines at sixteen-byte boundaries run)
def test_weights_of_even_lines_that_begin_anywhere(M, shift, apart, native, monkeypatch):
    """Lines a multiple of sixteen bytes apart, matrices not: `shift` bytes behind a boundary, or `apart` bytes between them."""
    _both(monkeypatch, native)
    K, N, E = 32, 16, 2
    g = torch.Generator().manual_seed(3)
    a = torch.randint(0, 120, (M, K), generator=g, dtype=torch.uint8).cuda().view(E4M3)
    a_scale = (torch.rand((M, 1), generator=g) + 0.5).cuda()
    w = (torch.randn((E, N, K), generator=g) * 100).clamp(-448, 448).to(E4M3).cuda()
    w_scale = (torch.rand((E, 1, 1), generator=g) + 0.5).cuda()
    odd = torch.zeros(E * (N * K + apart) + 16, dtype=torch.uint8, device="cuda").as_strided((E, N, K), (N * K + apart, K, 1), shift)
    odd.copy_(w.view(torch.uint8))
    sizes = [M - 70, 60]
    md = make_ragged_tensor_metadata(torch.tensor(sizes, dtype=torch.int32, device="cuda"), M)
    y = matmul_fp8_blocks(a, a_scale, odd.view(E4M3).transpose(1, 2), w_scale, None, md)
    for lo, hi, e in ((0, 300, 0), (M - 300, M - 70, 0), (M - 70, M - 10, 1)):
        check(y[lo:hi], *orc.product(a[lo:hi], a_scale[lo:hi], w[e:e + 1].transpose(1, 2), w_scale[e:e + 1])[:2], "y")


@pytest.mark.parametrize("native", [True, False])
def test_fp32_results_come_without_copies_of_the_operands(native, monkeypatch):
    """Their kernel takes lines that begin anywhere."""
    _both(monkeypatch, native)
    M, K, N = 600, 1001, 264
    g = torch.Generator().manual_seed(4)
    a = torch.randint(0, 120, (M, K), generator=g, dtype=torch.uint8).cuda().view(E4M3)
    w = torch.randint(0, 120, (1, N, K), generator=g, dtype=torch.uint8).cuda().view(E4M3).transpose(1, 2)
    a_scale, w_scale = torch.ones((M, 8), device="cuda"), torch.ones((1, 8, 3), device="cuda")
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    y = matmul_fp8_blocks(a, a_scale, w, w_scale, out_dtype=F32)
    assert torch.cuda.max_memory_allocated() - before < y.numel() * 4 + 4096
    some = torch.arange(0, M, 37, device="cuda")
    check(y[some], *orc.product(a.view(torch.uint8)[some].view(E4M3), a_scale[some], w, w_scale, out_dtype=F32)[:2], "y")


@pytest.mark.parametrize("source", [BF16, F16, F32])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_what_the_weights_gradient_reads_in_16_bits(dtype, source):
    """With the unit matrix behind it the gradient is x times its scale as it is multiplied: exact in fp16 where it is a multiple of 2^-24 within 65504, as all that was
    quantised from fp16 is, the nearest such number otherwise; exact in bf16 from 2^-126 on."""
    g = torch.Generator().manual_seed(6)
    T, K = 64, 256
    x = torch.randn((T, K), generator=g) * torch.ldexp(torch.ones(T, 1), torch.arange(T)[:, None] - 44)  # (up to 2^19 and more, beyond fp16, and far below 2^-24)
    x = (x.clamp(-65504, 65504) if source == F16 else x).to(source).cuda()
    x8, s = downcast_to_fp8_blocks(x)
    dw = weight_gradient_fp8_blocks(x8, s, torch.eye(T, dtype=dtype, device="cuda"), None, F32).cpu().double().T
    exact = orc.upcast(x8, s)
    if dtype == BF16:
        assert torch.equal(dw, exact)
        return
    held = exact.clamp(-65504, 65504)
    whole = held * 2.0**24 == (held * 2.0**24).round()
    assert torch.equal(dw[whole], held[whole]) and ((dw - held).abs() <= 2.0**-25).all()
    assert whole.all() == (source == F16)


@pytest.mark.parametrize("sa,sw", [(1.3 * 2.0**-63, 1.1 * 2.0**-62), (1.9 * 2.0**100, 1.1 * 2.0**-100), (1.7 * 2.0**60, 1.3 * 2.0**40), (1.1 * 2.0**-126, 1.9)])
@pytest.mark.parametrize("M,K,N,out_dtype", [(3, 300, 64, BF16), (300, 304, 264, BF16), (300, 300, 264, F32), (6000, 272, 4201, BF16)])  # few rows, ring, any lines, tiles
def test_scales_whose_product_is_a_normal_number(M, K, N, out_dtype, sa, sw):
    g = torch.Generator().manual_seed(7)
    a = torch.randint(0, 120, (M, -(-K // 16) * 16), generator=g, dtype=torch.uint8).cuda().view(E4M3)[:, :K]
    w = (torch.randn((1, N, -(-K // 16) * 16), generator=g) * 100).clamp(-448, 448).cuda().to(E4M3)[:, :, :K].transpose(1, 2)
    a_scale, w_scale = torch.full((M, -(-K // 128)), sa, device="cuda"), torch.full((1, -(-K // 128), -(-N // 128)), sw, device="cuda")
    y = matmul_fp8_blocks(a, a_scale, w, w_scale, out_dtype=out_dtype)
    some = torch.arange(0, M, max(1, M // 50), device="cuda")
    check(y[some], *orc.product(a.view(torch.uint8)[some].view(E4M3), a_scale[some], w, w_scale, out_dtype=out_dtype)[:2], "y")


def _calls(g):
    """(operator of one tensor, that tensor, whether it has a gradient)"""
    x, w = _rows(g, 40, 256), (torch.randn((256, 64), generator=g) * 0.1).cuda()
    x8, s = downcast_to_fp8_blocks(x)
    q = quantize_fp8_weight(w)
    h, v, t = swiglu_fp8_forward(x, 1.7, 2.0)
    dy, bias, gammas = _rows(g, 40, 64), torch.randn((1, 64), generator=g).cuda(), torch.rand(40, generator=g).cuda()
    return ((lambda p: downcast_to_fp8_blocks(p)[1], x, False), (lambda p: downcast_to_fp8_blocks(p, 128)[1], x, False), (lambda p: upcast_from_fp8_blocks(x8, p), s, False),
            (lambda p: matmul_fp8_blocks(x8, p, q.values, q.scales), s, False), (lambda p: matmul_fp8_blocks(x8, s, q.values, p), q.scales, False),
            (lambda p: matmul_fp8_blocks(x8, s, q.values, q.scales, p), bias, False), (lambda p: matmul_fp8_blocks(x8, s, q.values, q.scales, gammas=p), gammas, False),
            (lambda p: weight_gradient_fp8_blocks(x8, s, p), dy, False), (lambda p: weight_gradient_fp8_blocks(x8, p, dy), s, False),
            (lambda p: linear_fp8_blocks(p, w), x, True), (lambda p: linear_fp8_blocks(x, p), w, True), (lambda p: linear_fp8_blocks(p, w, quantized=q), x, True),
            (lambda p: swiglu_fp8_forward(p, 1.7, 2.0)[0], x, False), (lambda p: swiglu_fp8_checkpoint(p, 1.7, 2.0), x, True), (lambda p: swiglu_fp8_backward(p, v, t, 1.7, 2.0), h, False))


@pytest.mark.parametrize("native", [True, False])
def test_other_transforms_are_refused(native, monkeypatch):
    """Forward mode, whose dual tensors ask for no gradient; vmap and grad of torch.func."""
    import torch.autograd.forward_ad as fwad
    _both(monkeypatch, native)
    for f, t, differentiable in _calls(torch.Generator().manual_seed(8)):
        want = f(t)
        with fwad.dual_level():
            with pytest.raises(NotImplementedError, match="forward mode"):
                f(fwad.make_dual(t, torch.ones_like(t)))
            assert torch.equal(f(t), want)
        for call in (lambda: torch.func.jvp(f, (t, ), (torch.ones_like(t), )), lambda: torch.func.vmap(f)(torch.stack((t, t))), lambda: torch.func.grad(lambda s: f(s).float().sum())(t)):
            with pytest.raises((RuntimeError, NotImplementedError)):
                call()
        if not differentiable:
            with pytest.raises(NotImplementedError, match="no gradient for"):
                f(t.clone().requires_grad_())
        assert torch.equal(f(t), want)


@pytest.mark.parametrize("native", [True, False])
def test_threads_side_by_side(native, monkeypatch):
    """Each on a stream of its own, forward and backward, many times over; a workspace of its own for each weights' gradient."""
    import threading
    _both(monkeypatch, native)
    g = torch.Generator().manual_seed(9)
    T, K, N = 2100, 144, 272                                               # (a gradient in parts)
    sets = [(_rows(g, T, K), (torch.randn((K, N), generator=g) * 0.1).cuda(), _rows(g, T, N, BF16, 0.1), _rows(g, 60, 256)) for _ in range(4)]

    def step(x, w, dy, a):
        x, w, a = x.detach().requires_grad_(), w.detach().requires_grad_(), a.detach().requires_grad_()
        y, h = linear_fp8_blocks(x, w), swiglu_fp8_checkpoint(a, 1.7, 2.0)
        return (y, h) + torch.autograd.grad(y, (x, w), dy) + torch.autograd.grad(h, a, torch.ones_like(h))

    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    wrong = []

    def run(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(20):
                    got = step(*sets[i])
                    stream.synchronize()
                    if not all(torch.equal(p, q) for p, q in zip(got, want[i])):
                        wrong.append(i)
        except Exception as e:  # noqa: BLE001
            wrong.append(e)

    threads = [threading.Thread(target=run, args=(i, )) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_dual_weights_are_not_quantised():
    import torch.autograd.forward_ad as fwad
    w = torch.ones((256, 64), device="cuda")
    with fwad.dual_level():
        with pytest.raises(NotImplementedError, match="forward mode"):
            quantize_fp8_weight(fwad.make_dual(w, torch.ones_like(w)))
    assert quantize_fp8_weight(w.requires_grad_()).scales.shape == (1, 2, 1)  # (a leaf's values: the linear layer has its gradient)


@pytest.mark.parametrize("sizes,K,N,out_dtype", [([4, 1, 0, 13, 3, 5, 6, 1], 384, 96, BF16), ([40, 17, 0, 130, 33, 5, 64, 11], 400, 200, BF16), ([40, 17, 0, 130, 33, 5, 64, 11], 400, 200, F32),
                                                 ([900, 300, 0, 2000, 77, 1100, 500, 1], 256, 4200, BF16)])  # few rows, ring, any lines, tiles
def test_a_rank_multiplies_by_its_own_experts(sizes, K, N, out_dtype):
    """Metadata of all slices restricted to a few: their rows are at their places, the other rows stay as they were."""
    from triton_amd.tensor import remap_ragged_tensor_metadata
    g = torch.Generator().manual_seed(10)
    M, E, local = sum(sizes), len(sizes), [1, 3, 4, 6]
    smap = torch.full((E, ), -1, dtype=torch.int32)
    smap[local] = torch.arange(len(local), dtype=torch.int32)
    a, a_scale = downcast_to_fp8_blocks(_rows(g, M, K))
    w = (torch.randn((E, N, -(-K // 16) * 16), generator=g) * 100).clamp(-448, 448).cuda().to(E4M3)[:, :, :K].transpose(1, 2)
    w_scale = (torch.rand((E, -(-K // 128), -(-N // 128)), generator=g) + 0.5).cuda()
    md = remap_ragged_tensor_metadata(make_ragged_tensor_metadata(torch.tensor(sizes, dtype=torch.int32, device="cuda"), M), smap.cuda())
    before = torch.are_deterministic_algorithms_enabled()
    torch.use_deterministic_algorithms(True)                               # (new memory holds NaN)
    try:
        mine = w.transpose(1, 2).view(torch.uint8)[local].view(E4M3).transpose(1, 2)
        y = matmul_fp8_blocks(a, a_scale, mine, w_scale[local], None, md, out_dtype=out_dtype)
    finally:
        torch.use_deterministic_algorithms(before)
    for e in range(E):
        lo, hi = sum(sizes[:e]), sum(sizes[:e + 1])
        if e not in local:
            assert y[lo:hi].isnan().all()
            continue
        some = torch.arange(lo, hi, max(1, (hi - lo) // 40), device="cuda")
        check(y[some], *orc.product(a.view(torch.uint8)[some].view(E4M3), a_scale[some], w[e:e + 1], w_scale[e:e + 1], out_dtype=out_dtype)[:2], "y")
        assert y[lo:hi].isfinite().all()


HOOKS = {"offloaded": (lambda t: t.cpu(), lambda t: t.cuda()),
         "other strides": (lambda t: t.transpose(-1, -2).contiguous() if t.ndim > 1 else torch.stack((t, t), 1), lambda p: p.transpose(-1, -2) if p.dtype != torch.int32 or p.shape[1] != 2 else p[:, 0]),
         "rows between others": (lambda t: torch.stack((t, t), t.ndim - 1), lambda p: p.select(p.ndim - 2, 1))}


@pytest.mark.parametrize("hooks", HOOKS)
@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_saved_tensors_with_other_strides(dtype, native, hooks, monkeypatch):
    _both(monkeypatch, native)
    g = torch.Generator().manual_seed(11)
    T, K, N, E = 90, 200, 72, 3
    md = make_ragged_tensor_metadata(torch.tensor([30, 0, 50], dtype=torch.int32, device="cuda"), T)
    x, a = _rows(g, T, K, dtype).requires_grad_(), _rows(g, 20, 300, dtype).requires_grad_()
    w = (torch.randn((E, K, N), generator=g) * 0.05).cuda().requires_grad_()
    k_first = w.detach().transpose(1, 2).contiguous().transpose(1, 2).requires_grad_()
    dy, dh = _rows(g, T, N, dtype, 0.1), _rows(g, 20, 150, dtype)
    step = lambda v: (linear_fp8_blocks(x, v, md), swiglu_fp8_checkpoint(a, 1.7, 2.0))  # noqa: E731
    for v in (w, k_first):
        y, h = step(v)
        want = torch.autograd.grad(y, (x, v), dy) + torch.autograd.grad(h, a, dh)
        with torch.autograd.graph.saved_tensors_hooks(*HOOKS[hooks]):
            y, h = step(v)
        got = torch.autograd.grad(y, (x, v), dy) + torch.autograd.grad(h, a, dh)
        assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("reentrant", [True, False])
def test_recomputed_layers(reentrant, native, monkeypatch):
    from torch.utils.checkpoint import checkpoint
    _both(monkeypatch, native)
    g = torch.Generator().manual_seed(12)
    T, d, f, E = 120, 136, 200, 2
    md = make_ragged_tensor_metadata(torch.tensor([50, 70], dtype=torch.int32, device="cuda"), T)
    x = _rows(g, T, d).requires_grad_()
    w1, w2 = ((torch.randn(s, generator=g) * 0.05).cuda().requires_grad_() for s in ((E, d, 2 * f), (E, f, d)))
    dy = _rows(g, T, d, BF16, 0.1)
    block = lambda x, w1, w2: linear_fp8_blocks(swiglu_fp8_checkpoint(linear_fp8_blocks(x, w1, md), 1.7, 7.0), w2, md)  # noqa: E731

    def gradients(y):
        for t in (x, w1, w2):
            t.grad = None
        y.backward(dy)
        return [t.grad for t in (x, w1, w2)]

    y = block(x, w1, w2)
    z = checkpoint(block, x, w1, w2, use_reentrant=reentrant)
    assert torch.equal(y, z) and all(torch.equal(p, q) for p, q in zip(gradients(y), gradients(z)))


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("changed", ["slice_sizes", "slice_offs", "block_schedule_data"])
def test_metadata_changed_before_the_backward_pass(changed, native, monkeypatch):
    """Slices written over for the next batch: the gradients of this one are gone, and the backward pass says so."""
    _both(monkeypatch, native)
    g = torch.Generator().manual_seed(13)
    md = make_ragged_tensor_metadata(torch.tensor([30, 10, 50], dtype=torch.int32, device="cuda"), 90)
    x = _rows(g, 90, 200).requires_grad_()
    w = (torch.randn((3, 200, 72), generator=g) * 0.05).cuda().requires_grad_()
    y = linear_fp8_blocks(x, w, md)
    getattr(md, changed).add_(0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
