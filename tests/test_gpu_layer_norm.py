"""Layer norm and its gradients against the 64-bit oracle: sizes from one element to rows of tens of thousands, the three types of
activations and of weights, strided, shifted and transposed rows, rows that are constant or hold infinities, no rows; equal bits
from equal calls, other streams, graph capture."""
import pytest
import torch

from oracle import rows as orc
from triton_amd import _native as nt
from triton_kernels.layer_norm import layer_norm, layer_norm_backward, layer_norm_forward

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
SIZES = [(1, 1), (1, 7), (3, 8), (5, 63), (2, 64), (17, 100), (4, 128), (33, 257), (9, 512), (70, 520), (5, 1023), (3, 2049), (16, 2880), (2, 4096), (3, 8191),
         (1, 16384), (3, 10000), (2, 16385), (2, 33001), (300, 72), (1000, 130)]


def _make(M, C, dtype, weights, seed=0, shift=0.0):
    g = torch.Generator().manual_seed(seed + M * 131 + C)
    x = (torch.randn((M, C), generator=g) * 1.5 + torch.randn((M, 1), generator=g) * 0.5 + shift).to(dtype).cuda()
    w = b = None
    if weights is not None:
        w = (torch.randn(C, generator=g) * 0.2 + 1).to(weights).cuda()
        b = (torch.randn(C, generator=g) * 0.2).to(weights).cuda()
    dy = torch.randn((M, C), generator=g).to(dtype).cuda()
    return x, w, b, dy


def _check(x, w, b, dy, eps=1e-5):
    y, mean, rstd = layer_norm_forward(x, w, b, eps)
    want, bound = orc.layer_norm(x, w, b, eps)
    assert y.dtype == x.dtype and y.shape == x.shape and y.is_contiguous()
    orc.check(y, want, bound, "y")
    assert torch.equal(layer_norm(x, w, b, eps), y)
    dx, dw, db = layer_norm_backward(dy, x, mean, rstd, w, b)
    want = orc.layer_norm_backward(dy, x, w, eps, b)
    assert dx.dtype == x.dtype and dx.shape == x.shape
    orc.check(dx.reshape(-1, x.shape[-1]), *want["dx"], "dx")
    if w is not None:
        assert dw.dtype == w.dtype
        orc.check(dw, *want["dweight"], "dweight")
    else:
        assert dw is None
    if b is not None:
        assert db.dtype == b.dtype
        orc.check(db, *want["dbias"], "dbias")
    else:
        assert db is None
    return y, dx, dw, db


@pytest.mark.parametrize("dtype,weights", [(BF16, BF16), (F16, F32), (F32, F32), (BF16, None)])
@pytest.mark.parametrize("M,C", SIZES)
def test_sizes_and_types(M, C, dtype, weights):
    _check(*_make(M, C, dtype, weights))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_more_long_rows_than_partial_sums(dtype):
    _check(*_make(301, 16389, dtype, F32))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_weight_and_bias_of_other_types_or_alone(dtype):
    x, w, b, dy = _make(37, 264, dtype, F32)
    _check(x, w.to(BF16), b.to(F16), dy)
    _check(x, w.to(F16), b, dy)
    _check(x, w, None, dy)
    _check(x, None, b.to(BF16), dy)


@pytest.mark.parametrize("M,C", [(4099, 256), (4099, 40), (1031, 2880), (6000, 1023), (2050, 7), (3001, 3), (2048, 512), (2047, 513), (2500, 1537), (2100, 2050), (2049, 4096),
                                 (2200, 4100), (9001, 130), (2051, 8)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_many_rows(M, C, dtype):
    _check(*_make(M, C, dtype, F32))


@pytest.mark.parametrize("C", [65, 128, 1000, 2880])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_at_any_stride_and_address(C, dtype):
    """Column slices (rows that start between 16-byte boundaries), every second row, transposed storage, broadcast gradients."""
    wide, w, b, dy = _make(21, 2 * C + 3, dtype, F32, seed=1)
    w, b = w[:C], b[:C]
    for x in (wide[:, 1:C + 1], wide[:, C + 2:2 * C + 2], wide[::2, 3:C + 3], wide[:, :C].t().contiguous().t()):
        _check(x, w, b, dy[:x.shape[0], 5:C + 5].contiguous())
        _check(x, w, b, dy[:x.shape[0], 1:C + 1])
    x = wide[:, :C]
    _check(x, w, b, dy[:, :1].expand(21, C))
    _check(x, w, b, dy[:1, :C].expand(21, C))
    _check(x[:1].expand(21, C), w, b, dy[:, :C])
    both = torch.stack((w, b), dim=1)
    _check(x, both[:, 0], both[:, 1], dy[:, :C])


def test_more_dimensions():
    x, w, b, dy = _make(60, 96, BF16, BF16)
    y, dx, dw, db = _check(x.view(3, 4, 5, 96), w, b, dy.view(3, 4, 5, 96))
    flat = _check(x, w, b, dy)
    for a, c in zip((y.view(60, 96), dx.view(60, 96), dw, db), flat):
        assert torch.equal(a, c)
    assert layer_norm(x[0], w, b).shape == (96, )
    assert torch.equal(layer_norm(x[0], w, b), flat[0][0])


def test_constant_rows_large_means_and_eps():
    x, w, b, dy = _make(12, 384, F32, F32)
    x[0] = 3.0
    x[1] = 0.0
    _check(x, w, b, dy)
    _check(x[2:], w, b, dy[2:], eps=0.0)
    _check(x, w, b, dy, eps=0.5)
    _check(*_make(12, 384, F32, F32, shift=100.0))
    _check(*_make(12, 384, BF16, F32, shift=-30.0))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("C", [2, 9, 100, 1000])
def test_constant_rows_of_large_numbers(C, dtype):
    """Where the reciprocal deviation times the mean is beyond 32 bits, but no element's distance from the mean is."""
    x, w, b, dy = _make(11, C, dtype, dtype)
    x[3] = 2.0**121 if C <= 100 else 2.0**117
    x[10] = -x[3]
    _check(x, w, b, dy, eps=1e-5 if C <= 100 else 1e-9)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_infinities_and_nan_stay_in_their_rows(dtype):
    x, w, b, dy = _make(9, 200, dtype, dtype)
    clean = layer_norm(x, w, b)
    x[2, 7], x[5, 199], x[6, 0] = float("inf"), float("nan"), float("-inf")
    y = layer_norm(x, w, b)
    rows = [0, 1, 3, 4, 7, 8]
    assert torch.equal(y[rows], clean[rows])
    assert y[[2, 5, 6]].isnan().all()


def test_no_rows():
    x, w, b, dy = _make(0, 64, BF16, F32)
    y, mean, rstd = layer_norm_forward(x, w, b)
    assert y.shape == (0, 64)
    dx, dw, db = layer_norm_backward(dy, x, mean, rstd, w, b)
    assert dx.shape == (0, 64) and not dw.any() and not db.any() and dw.shape == (64, )
    assert layer_norm(x.view(3, 0, 64), w, b).shape == (3, 0, 64)


@pytest.mark.parametrize("native", [True, False])
def test_autograd_gives_the_same_and_only_what_is_asked(native, monkeypatch):
    """Through the native host path and through the general one."""
    if not native:
        monkeypatch.setattr(nt, "host", lambda: None)
    x, w, b, dy = _make(50, 300, BF16, F32)
    y0, mean, rstd = layer_norm_forward(x, w, b)
    want = layer_norm_backward(dy, x, mean, rstd, w, b)
    for mask in range(1, 8):
        leaves = [t.clone().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate((x, w, b))]
        y = layer_norm(*leaves)
        assert torch.equal(y, y0)
        y.backward(dy)
        for i, t in enumerate(leaves):
            if mask >> i & 1:
                assert torch.equal(t.grad, want[i]), (mask, i)
            else:
                assert t.grad is None
    for weight, bias in ((None, None), (w, None), (None, b)):  # parameters that there are not
        leaves = [t if t is None else t.clone().requires_grad_() for t in (x, weight, bias)]
        y = layer_norm(*leaves)
        y.backward(dy)
        f = layer_norm_forward(x, weight, bias)
        assert torch.equal(y, f[0])
        for t, g in zip(leaves, layer_norm_backward(dy, x, f[1], f[2], weight, bias)):
            assert t is None and g is None or torch.equal(t.grad, g)
    leaf = x.clone().requires_grad_()
    g, = torch.autograd.grad(layer_norm(leaf, w, b).sum(), leaf)
    assert torch.equal(g, layer_norm_backward(torch.ones_like(x), x, mean, rstd, w, b)[0])
    g, = torch.autograd.grad(layer_norm(leaf, w, b), leaf, dy, create_graph=True)
    assert torch.equal(g, want[0])
    with pytest.raises(RuntimeError, match="differentiable once"):
        g.sum().backward()
    leaf = x.clone().requires_grad_()
    y = layer_norm(leaf, w, b)
    with torch.no_grad():
        leaf.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()
    turned = x.t().contiguous().t().requires_grad_()  # (goes the general way)
    layer_norm(turned, w, b).backward(dy.t().contiguous().t())
    assert torch.equal(turned.grad, want[0])


def test_equal_calls_give_equal_bits():
    x, w, b, dy = _make(3000, 520, BF16, F32)
    y, mean, rstd = layer_norm_forward(x, w, b)
    first = layer_norm_backward(dy, x, mean, rstd, w, b)
    for _ in range(3):
        for a, c in zip(first, layer_norm_backward(dy, x, mean, rstd, w, b)):
            assert torch.equal(a, c)


def test_two_streams_at_once():
    x, w, b, dy = _make(2000, 776, BF16, F32)
    x2, _, _, dy2 = _make(1999, 776, BF16, F32, seed=5)
    want = [layer_norm_forward(t, w, b) for t in (x, x2)]
    want = [(f[0], *layer_norm_backward(d, t, f[1], f[2], w, b)) for f, t, d in zip(want, (x, x2), (dy, dy2))]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(5):
        for i, (s, t, d) in enumerate(zip(streams, (x, x2), (dy, dy2))):
            with torch.cuda.stream(s):
                y, mean, rstd = layer_norm_forward(t, w, b)
                got[i].append((y, *layer_norm_backward(d, t, mean, rstd, w, b)))
    torch.cuda.synchronize()
    for i in (0, 1):
        for out in got[i]:
            for a, c in zip(out, want[i]):
                assert torch.equal(a, c)


def test_in_a_graph():
    x, w, b, dy = _make(700, 520, BF16, F32)
    layer_norm_forward(x, w, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, mean, rstd = layer_norm_forward(x, w, b)
        out = (y, *layer_norm_backward(dy, x, mean, rstd, w, b))
    for seed in range(3):
        nx, _, _, ndy = _make(700, 520, BF16, F32, seed=10 + seed)
        x.copy_(nx)
        dy.copy_(ndy)
        graph.replay()
        f = layer_norm_forward(nx, w, b)
        want = (f[0], *layer_norm_backward(ndy, nx, f[1], f[2], w, b))
        torch.cuda.synchronize()
        for a, c in zip(out, want):
            assert torch.equal(a, c)


def test_rows_beyond_32_bit_offsets():
    """The last rows of an activation of more than 2^32 bytes."""
    M, C = 1 << 21, 1032
    x = torch.zeros((M, C), dtype=BF16, device="cuda")
    small, w, b, dy = _make(4, C, BF16, F32)
    x[-4:] = small
    y = layer_norm(x, w, b)
    assert torch.equal(y[-4:], layer_norm(small, w, b))
    assert torch.equal(y[0], b.to(BF16)) and torch.equal(y[M // 2 + 1], b.to(BF16))
