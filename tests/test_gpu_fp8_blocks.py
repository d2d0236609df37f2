"""e4m3 in blocks of 128 on the GPU against the 64-bit oracle: the quantiser bit for bit, the ragged product, the weights' gradient, the linear layer and
swiglu with their gradients; sizes from one element on, odd lengths and strides, empty slices, dropped and gathered rows, what is not finite, other streams, captured graphs."""
import pytest
import torch

from oracle import fp8_blocks as orc
from oracle.rows import check
from triton_kernels.fp8_blocks import (downcast_to_fp8_blocks, linear_fp8_blocks, matmul_fp8_blocks, quantize_fp8_weight, swiglu_fp8_backward,
                                       swiglu_fp8_checkpoint, swiglu_fp8_forward, upcast_from_fp8_blocks, weight_gradient_fp8_blocks)
from triton_kernels.matmul import FnSpecs, FusedActivation
from triton_kernels.swiglu import swiglu_fn
from triton_kernels.tensor import make_ragged_tensor_metadata

pytestmark = pytest.mark.gpu

F32, BF16, F16, E4M3 = torch.float32, torch.bfloat16, torch.float16, torch.float8_e4m3fn
NAN, INF = float("nan"), float("inf")
ACT = (1.702, 7.0)
SWIGLU = FusedActivation(FnSpecs("swiglu", swiglu_fn, ("alpha", "limit"), reduction_n=2), ACT)


def _gen(*seed):
    return torch.Generator().manual_seed(hash(seed) % (1 << 31))


def _rows(g, R, C, dtype=BF16, scale=1.0):
    x = torch.randn((R, C), generator=g) * (torch.rand((R, 1), generator=g) * 2 + 0.1) * scale
    x[:, ::37] *= 20
    return x.to(dtype).cuda()


def _same(values, scales, want):
    assert values.dtype == E4M3 and scales.dtype == F32
    v, w = values.float().cpu().double(), want[0]
    assert torch.equal(torch.nan_to_num(v, nan=1e9), torch.nan_to_num(w, nan=1e9))
    assert torch.equal(scales.cpu().double(), want[1])


# ---- quantiser ---------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("R,C", [(1, 1), (3, 7), (2, 128), (5, 129), (17, 264), (1, 1000), (33, 2880), (260, 72), (7, 4104)])
def test_rows_quantised_and_read_back(R, C, dtype):
    x = _rows(_gen(R, C), R, C, dtype)
    values, scales = downcast_to_fp8_blocks(x)
    assert values.shape == x.shape and scales.shape == (R, -(-C // 128)) and values.stride(0) % 16 == 0
    _same(values, scales, orc.downcast(x))
    for out in (BF16, F16, F32):
        back = upcast_from_fp8_blocks(values, scales, out)
        assert back.dtype == out and torch.equal(back.cpu(), orc.upcast(values, scales).to(out))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shape", [(1, 1), (128, 128), (5, 300), (300, 5), (129, 257), (2, 130, 136), (3, 256, 40)])
def test_blocks_of_128_rows(shape, dtype):
    x = torch.randn(shape, generator=_gen(*shape)).mul(0.05).to(dtype).cuda()
    values, scales = downcast_to_fp8_blocks(x, 128)
    _same(values, scales, orc.downcast(x, 128))
    assert torch.equal(upcast_from_fp8_blocks(values, scales, F32, 128).cpu().double(), orc.upcast(values, scales, 128))
    q = quantize_fp8_weight(x)
    w3 = x if x.ndim == 3 else x[None]
    want = orc.downcast(w3, 128)
    for t, unit in ((q.values, 1), (q.values_n, 2)):
        assert t.shape == w3.shape and (t.stride(unit) == 1 or t.shape[unit] == 1)
        _same(t, q.scales, want)
    k_first = quantize_fp8_weight(x.transpose(-1, -2).contiguous().transpose(-1, -2))
    assert torch.equal(k_first.values.float(), q.values.float()) and torch.equal(k_first.scales, q.scales) and torch.equal(k_first.values_n.float(), q.values_n.float())


def test_extremes_of_the_quantiser():
    f = torch.finfo(F32)
    x = torch.zeros((9, 256))
    x[1, 3], x[1, 200] = f.max, f.smallest_normal
    x[2, 0], x[2, 129] = 2.0**-149, -2.0**-140
    x[3, :4] = torch.tensor([448.0, 448.0 * (1 + 2**-23), 2.0**-9, 17.0])  # just beyond a power's reach: the next scale
    x[4, :3] = torch.tensor([448.0, 1.0625, 1.1875])                      # ties to even
    x[5, 0], x[5, 1], x[5, 2] = INF, NAN, 3.0
    x[6, 5] = -INF
    x[7, :] = -0.0
    x[8] = torch.logspace(-30, 3, 256)
    for shape in (x, x[:, :250], x[:, 1:]):
        t = shape.cuda()
        values, scales = downcast_to_fp8_blocks(t)
        _same(values, scales, orc.downcast(t))
    t = x.cuda()
    _same(*downcast_to_fp8_blocks(t, 128), orc.downcast(t, 128))


def test_shapes_and_strides_of_the_quantiser():
    x = _rows(_gen(5), 24, 400)
    for t in (x[:, 8:264], x[:, 3:300], x[::3], x.T, x[:, ::2], x[0], x[:0], x[:, :0], x.view(2, 12, 400), x.view(2, 3, 4, 400)[:, 1:], x[:1].expand(5, 400)):
        values, scales = downcast_to_fp8_blocks(t)
        assert values.shape == t.shape and scales.shape == (*t.shape[:-1], -(-t.shape[-1] // 128))
        if t.numel():
            d = t[None] if t.ndim == 1 else t
            _same(values if t.ndim > 1 else values[None], scales if t.ndim > 1 else scales[None], orc.downcast(d))
        back = upcast_from_fp8_blocks(values, scales)
        assert back.shape == t.shape
    neighbours = torch.full((4, 512), 5.0, device="cuda").to(E4M3)
    back = upcast_from_fp8_blocks(neighbours[:, 3:260], torch.full((4, 3), 0.3, device="cuda"), F32)
    assert torch.equal(back, torch.full((4, 257), 5.0 * torch.tensor(0.3).item(), device="cuda"))


# ---- product -----------------------------------------------------------------------------------------------------------------

def _operands(seed, rows, K, N, E=1, pitch=None):
    g = _gen(seed, rows, K, N, E)
    a, a_scale = downcast_to_fp8_blocks(_rows(g, rows, K))
    if pitch is not None:
        full = torch.full((rows, pitch), NAN, device="cuda").to(E4M3)
        full[:, :K] = a
        a = full[:, :K]
    wv = (torch.randn((E, N, K), generator=g) * 120).clamp(-448, 448).to(E4M3).cuda()
    w_scale = (torch.rand((E, -(-N // 128), -(-K // 128)), generator=g) * 1e-3 + 1e-5).cuda()
    return g, a, a_scale, wv.transpose(1, 2), w_scale.transpose(1, 2)


def _deal(g, rows, E):
    if E == 1:
        return [rows]
    cut = torch.randint(0, rows + 1, (E - 1, ), generator=g).sort().values.tolist()
    return [b - a for a, b in zip([0] + cut, cut + [rows])]


def _metadata(sizes, rows=None):
    return make_ragged_tensor_metadata(torch.tensor(sizes, dtype=torch.int32, device="cuda"), sum(sizes) if rows is None else rows)


def _check_product(a, a_scale, w, w_scale, out_dtype=BF16, sizes=None, rows=None, **kw):
    swiglu = kw.pop("swiglu", False)
    md = None if sizes is None else _metadata(sizes, rows)
    y = matmul_fp8_blocks(a, a_scale, w, w_scale, kw.get("bias"), md, gather_indx=kw.get("gather"), scatter_indx=kw.get("scatter"), gammas=kw.get("gammas"),
                          fused_activation=SWIGLU if swiglu else None, out_dtype=out_dtype)
    want, bound, written = orc.product(a, a_scale, w, w_scale, sizes, swiglu=ACT if swiglu else None, out_dtype=out_dtype, **kw)
    assert y.dtype == out_dtype and y.shape == want.shape
    check(y[written.cuda()], want[written], bound[written], "y")
    return y


@pytest.mark.parametrize("M,K,N", [(1, 1, 1), (1, 128, 128), (3, 7, 5), (1, 4096, 512), (2, 130, 33), (16, 256, 48), (17, 384, 64), (33, 1000, 129), (64, 640, 256),
                                   (65, 128, 300), (128, 512, 384), (129, 1040, 512), (200, 96, 1023), (257, 720, 264), (520, 2880, 256), (300, 16, 640), (1000, 144, 2048)])
@pytest.mark.parametrize("out_dtype,swiglu", [(BF16, False), (F16, True), (F32, False), (BF16, True), (F32, True)])
def test_product_sizes(M, K, N, out_dtype, swiglu):
    N += N % 2 if swiglu else 0
    _check_product(*_operands(1, M, K, N)[1:], out_dtype, swiglu=swiglu)


@pytest.mark.parametrize("E,rows,K,N", [(3, 5, 256, 64), (8, 64, 384, 96), (32, 70, 512, 128), (5, 700, 1000, 1023), (8, 900, 640, 512), (4, 2000, 272, 384), (300, 400, 128, 64), (7, 1600, 256, 520)])
@pytest.mark.parametrize("options", ["plain", "bias", "gather", "scatter", "all"])
def test_ragged_products(E, rows, K, N, options):
    swiglu = options in ("gather", "all") and N % 2 == 0
    tokens = max(1, rows // 2) if options in ("gather", "all") else rows
    g, a, a_scale, w, w_scale = _operands(2, tokens, K, N, E)
    kw = {}
    sizes = _deal(g, rows, E)
    if options in ("gather", "all"):
        kw["gather"] = torch.randint(tokens, (rows, ), generator=g, dtype=torch.int32).cuda()
    if options in ("bias", "all"):
        kw["bias"] = torch.randn((E, N), generator=g).to(BF16 if options == "all" else F32).cuda()
        kw["gammas"] = torch.rand(rows, generator=g).to(F32 if options == "all" else BF16).cuda()
    if options in ("scatter", "all"):
        at = torch.randperm(rows, generator=g).to(torch.int32)
        at[::7] = -1
        kw["scatter"] = at.cuda()
    _check_product(a, a_scale, w, w_scale, BF16, sizes, swiglu=swiglu, **kw)


@pytest.mark.parametrize("pitch", [None, 277, 288, 400])
@pytest.mark.parametrize("M", [1, 40, 300])
def test_strides_of_the_product(M, pitch):
    K, N, E = 272, 136, 2
    g, a, a_scale, w, w_scale = _operands(3, M, K, N, E, pitch)
    sizes = _deal(g, M, E)
    y = _check_product(a, a_scale, w, w_scale, BF16, sizes)
    md = _metadata(sizes)
    n_first = w.contiguous()                                              # contiguous along N: copied
    wide = torch.full((E, N, K + 16), NAN, device="cuda").to(E4M3)
    wide[:, :, :K] = w.transpose(1, 2)
    odd = torch.empty((E, N + 1, K + 3), device="cuda").to(E4M3)
    odd[:, :N, 1:K + 1] = w.transpose(1, 2)
    for other in (n_first, wide[:, :, :K].transpose(1, 2), odd[:, :N, 1:K + 1].transpose(1, 2)):
        assert torch.equal(matmul_fp8_blocks(a, a_scale, other, w_scale, None, md).cpu(), y.cpu())
    for s, t in ((a_scale.T.contiguous().T, w_scale.contiguous()), (torch.stack((a_scale, a_scale), 2)[:, :, 0], torch.stack((w_scale, w_scale), 3)[..., 1])):
        assert torch.equal(matmul_fp8_blocks(a, s, w, t, None, md), y)
    assert torch.equal(matmul_fp8_blocks(a.T.contiguous().T, a_scale, w, w_scale, None, md), y)


@pytest.mark.parametrize("M", [1, 30, 300])
def test_what_is_not_finite_stays_in_its_row_or_column(M):
    K, N = 400, 200
    _, a, a_scale, w, w_scale = _operands(4, M + 2, K, N)
    a[M // 2, 399] = NAN
    a_scale[M, 1] = INF
    w = w.transpose(1, 2).contiguous().transpose(1, 2)
    w[0, 5, 7] = NAN
    y = matmul_fp8_blocks(a, a_scale, w, w_scale, out_dtype=F32)
    bad = torch.zeros((M + 2, N), dtype=torch.bool)
    bad[M // 2], bad[M], bad[:, 7] = True, True, True
    assert torch.equal(y.isfinite().cpu(), ~bad)


def test_rows_behind_the_slices_and_dropped_ones_stay():
    g, a, a_scale, w, w_scale = _operands(6, 90, 256, 64, 3)
    sizes = [20, 0, 31]
    before = torch.are_deterministic_algorithms_enabled()
    torch.use_deterministic_algorithms(True)                               # (new memory holds NaN)
    try:
        y = matmul_fp8_blocks(a, a_scale, w, w_scale, None, _metadata(sizes, 90))
        at = torch.arange(90, dtype=torch.int32, device="cuda")
        at[::4] = -1
        z = matmul_fp8_blocks(a, a_scale, w, w_scale, None, _metadata(sizes, 90), scatter_indx=at)
    finally:
        torch.use_deterministic_algorithms(before)
    assert y[51:].isnan().all() and z[51:].isnan().all() and z[::4].isnan().all()
    want, bound, _ = orc.product(a[:51], a_scale[:51], w, w_scale, sizes)
    check(y[:51], want, bound, "y")
    assert torch.equal(z[1::4][:13], y[1::4][:13])


def test_no_rows_no_columns_no_depth():
    for M, K, N in ((0, 128, 64), (5, 128, 0), (5, 0, 64)):
        a, w = torch.zeros((M, K), device="cuda").to(E4M3), torch.zeros((2, N, K), device="cuda").to(E4M3).transpose(1, 2)
        y = matmul_fp8_blocks(a, torch.ones((M, -(-K // 128)), device="cuda"), w, torch.ones((2, -(-K // 128), -(-N // 128)), device="cuda"),
                              torch.full((2, N), 3.0, device="cuda"), _metadata([M, 0]))
        assert y.shape == (M, N) and (y == 3).all()


# ---- gradients ---------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("out_dtype", [F32, BF16, F16])
@pytest.mark.parametrize("T,K,N,E", [(1, 1, 1, 1), (5, 130, 7, 1), (31, 64, 64, 2), (33, 128, 128, 3), (200, 264, 136, 4), (300, 520, 776, 5), (513, 256, 512, 2), (1000, 100, 300, 40), (2100, 144, 272, 1)])
def test_weight_gradients(T, K, N, E, dtype, out_dtype):
    g = _gen(T, K, N, E)
    sizes = None if E == 1 else _deal(g, T, E)
    x, s = downcast_to_fp8_blocks(_rows(g, T, K, dtype))
    dy = _rows(g, T, N, dtype, 0.02)
    md = None if sizes is None else _metadata(sizes)
    dw = weight_gradient_fp8_blocks(x, s, dy, md, out_dtype)
    assert dw.dtype == out_dtype and dw.shape == ((K, N) if md is None else (E, K, N))
    check(dw.view(E, K, N), *orc.weight_gradient(x, s, dy, sizes, out_dtype), "dw")
    assert torch.equal(weight_gradient_fp8_blocks(x, s, dy, md, out_dtype), dw)


def test_weight_gradient_strides_scales_and_rows_outside():
    g = _gen(9)
    T, K, N = 150, 200, 72
    x, s = downcast_to_fp8_blocks(_rows(g, T, K))
    s = s * 1.37                                                           # scales of any size: rounded to 16 bits behind them
    dy = _rows(g, T, N + 5, BF16, 0.1)[:, 2:N + 2]
    check(weight_gradient_fp8_blocks(x, s, dy, None, F32)[None], *orc.weight_gradient(x, s, dy), "dw")
    x[100:], dy[100:] = torch.full((50, K), NAN, device="cuda").to(E4M3), NAN   # rows that no slice holds
    sizes = [60, 0, 40]
    dw = weight_gradient_fp8_blocks(x, s, dy, _metadata(sizes, T), F32)
    check(dw, *orc.weight_gradient(x[:100], s[:100], dy[:100], sizes), "dw")
    assert (dw[1] == 0).all()
    for xv, d in ((x[:100].T.contiguous().T, dy[:100]), (x[:100], dy[:100].T.contiguous().T), (x[:100].clone(), dy[:100].contiguous())):
        assert torch.equal(weight_gradient_fp8_blocks(xv, s[:100], d, _metadata(sizes), F32), dw)
    one = dy[:1].expand(100, N)
    check(weight_gradient_fp8_blocks(x[:100], s[:100], one, None, F32)[None], *orc.weight_gradient(x[:100], s[:100], one), "dw")


def test_weight_gradient_of_large_fp16():
    x, s = downcast_to_fp8_blocks(torch.full((4, 128), 65504.0, device="cuda", dtype=F16))
    dy = torch.ones((4, 8), device="cuda", dtype=F16)
    assert torch.equal(weight_gradient_fp8_blocks(x, s, dy, None, F32), torch.full((128, 8), 4 * 65504.0, device="cuda"))


@pytest.mark.parametrize("dtype,weights", [(BF16, BF16), (F16, F32), (BF16, F32), (F16, F16)])
@pytest.mark.parametrize("T,K,N,E", [(1, 128, 64, 1), (40, 256, 192, 3), (333, 520, 776, 5), (600, 384, 256, 2)])
def test_linear_and_its_gradients(T, K, N, E, dtype, weights):
    g = _gen(T, K, N)
    sizes = None if E == 1 else _deal(g, T, E)
    md = None if sizes is None else _metadata(sizes)
    x = _rows(g, T, K, dtype).requires_grad_()
    w = (torch.randn((E, K, N) if E > 1 else (K, N), generator=g) * 0.05).to(weights).cuda().requires_grad_()
    dy = _rows(g, T, N, dtype, 0.01)
    y = linear_fp8_blocks(x, w, md)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    w3 = w.detach().view(E, K, N)
    x8, xs = downcast_to_fp8_blocks(x.detach())
    w8, ws = downcast_to_fp8_blocks(w3, 128)
    d8, ds = downcast_to_fp8_blocks(dy)
    check(y, *orc.product(x8, xs, w8, ws, sizes, out_dtype=dtype)[:2], "y")
    check(dx, *orc.product(d8, ds, w8.transpose(1, 2), ws.transpose(1, 2), sizes, out_dtype=dtype)[:2], "dx")
    check(dw.view(E, K, N), *orc.weight_gradient(x8, xs, dy, sizes, weights), "dw")
    assert y.dtype == dx.dtype == dtype and dw.dtype == weights and dw.shape == w.shape
    with torch.no_grad():
        assert torch.equal(linear_fp8_blocks(x, w, md), y)
    q = quantize_fp8_weight(w)
    k_first = w.detach().transpose(-1, -2).contiguous().transpose(-1, -2).requires_grad_()
    for other, given in ((w, q), (k_first, None)):
        z = linear_fp8_blocks(x, other, md, given)
        assert torch.equal(z, y)
        assert all(torch.equal(p, r) for p, r in zip(torch.autograd.grad(z, (x, other), dy), (dx, dw)))
    dx1, = torch.autograd.grad(linear_fp8_blocks(x, w.detach(), md), x, dy)
    dw1, = torch.autograd.grad(linear_fp8_blocks(x.detach(), w, md), w, dy)
    assert torch.equal(dx1, dx) and torch.equal(dw1, dw)


def test_linear_gives_zeros_behind_the_slices():
    g = _gen(11)
    x = _rows(g, 100, 256).requires_grad_()
    w = (torch.randn((2, 256, 64), generator=g) * 0.05).to(BF16).cuda().requires_grad_()
    y = linear_fp8_blocks(x, w, _metadata([30, 27], 100))
    assert (y[57:] == 0).all() and (y[:57] != 0).any(1).all()
    y.backward(torch.ones_like(y))
    assert (x.grad[57:] == 0).all() and (x.grad[:57] != 0).any(1).all()
    y = linear_fp8_blocks(x, w, _metadata([0, 0], 100))
    dx, dw = torch.autograd.grad(y.sum(), (x, w))                          # (the sum's gradient is one number expanded)
    assert (y == 0).all() and (dx == 0).all() and (dw == 0).all()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("limit", [None, 7.0, 0.5])
@pytest.mark.parametrize("M,n", [(1, 1), (3, 5), (2, 64), (17, 65), (33, 500), (16, 2880), (5, 4099)])
def test_swiglu_and_its_gradient(M, n, limit, dtype):
    g = _gen(M, n)
    a = _rows(g, M, 2 * n, dtype, 1.5).requires_grad_()
    dh = torch.randn((M, n), generator=g).to(dtype).cuda()
    h = swiglu_fp8_checkpoint(a, 1.702, limit)
    da, = torch.autograd.grad(h, a, dh)
    check(h, *orc.swiglu(a, 1.702, limit), "h")
    h2, values, scales = swiglu_fp8_forward(a.detach(), 1.702, limit)
    v, s = downcast_to_fp8_blocks(a.detach())
    assert torch.equal(h2, h) and torch.equal(values.float(), v.float()) and torch.equal(scales, s)
    check(da, *orc.swiglu_backward(dh, values, scales, 1.702, limit), "da")
    assert torch.equal(swiglu_fp8_backward(dh, values, scales, 1.702, limit), da)
    with torch.no_grad():
        assert torch.equal(swiglu_fp8_checkpoint(a, 1.702, limit), h)


def test_swiglu_far_and_not_finite():
    a = torch.tensor([[90.0, 2.0, -90.0, 3.0, 1e4, -1.0, -1e4, 2.0, NAN, 1.0, 1.0, NAN, 0.0, 5.0, -100.0, 1e3]], device="cuda")
    for limit in (None, 7.0):
        h, values, scales = swiglu_fp8_forward(a, 1.0, limit)
        want, bound = orc.swiglu(a, 1.0, limit)
        live = torch.isfinite(want)
        assert torch.equal(h.cpu().isnan(), want.isnan())
        check(h.cpu()[live], want[live], bound[live], "h")
        da = swiglu_fp8_backward(torch.ones_like(h), values, scales, 1.0, limit)
        want, bound = orc.swiglu_backward(torch.ones_like(h), values, scales, 1.0, limit)
        assert torch.equal(da.cpu().isnan(), want.isnan())
        live = ~want.isnan()
        check(da.cpu()[live], want[live], bound[live], "da")


def test_strides_of_swiglu():
    g = _gen(13)
    wide = _rows(g, 20, 300)
    for a in (wide[:, 4:260], wide[:, 1:261], wide.T[:, :20], wide.view(4, 5, 300)[1:, :, :64], wide[:0], wide[:, :0], wide[0, :128]):
        x = a.detach().clone().contiguous().requires_grad_()
        y = a.detach().requires_grad_()
        hx, hy = swiglu_fp8_checkpoint(x, 1.0, 2.0), swiglu_fp8_checkpoint(y, 1.0, 2.0)
        assert hx.shape == (*a.shape[:-1], a.shape[-1] // 2) and torch.equal(hx, hy)
        d = torch.randn((*hx.shape[:-1], hx.shape[-1] * 2), generator=torch.Generator().manual_seed(1)).to(BF16).cuda()[..., ::2]
        assert torch.equal(torch.autograd.grad(hx, x, d)[0], torch.autograd.grad(hy, y, d.contiguous())[0])


# ---- together ----------------------------------------------------------------------------------------------------------------

def _block(x, w1, w2, md):
    return linear_fp8_blocks(swiglu_fp8_checkpoint(linear_fp8_blocks(x, w1, md), 1.702, 7.0), w2, md)


def test_a_training_step_of_the_feed_forward_block():
    """Projection, activation and projection, forward and back, with every intermediate checked where it is used."""
    g = _gen(21)
    T, d, f, E = 260, 256, 320, 4
    sizes = _deal(g, T, E)
    md = _metadata(sizes)
    x = _rows(g, T, d).requires_grad_()
    w1 = (torch.randn((E, d, 2 * f), generator=g) * 0.05).to(BF16).cuda().requires_grad_()
    w2 = (torch.randn((E, f, d), generator=g) * 0.05).cuda().requires_grad_()
    dy = _rows(g, T, d, BF16, 0.01)
    y = _block(x, w1, w2, md)
    dx, dw1, dw2 = torch.autograd.grad(y, (x, w1, w2), dy)
    with torch.no_grad():
        a = linear_fp8_blocks(x, w1, md)
        h, a8, as_ = swiglu_fp8_forward(a, 1.702, 7.0)
        h8, hs = downcast_to_fp8_blocks(h)
        q2, s2 = downcast_to_fp8_blocks(w2, 128)
        d8, ds = downcast_to_fp8_blocks(dy)
        check(y, *orc.product(h8, hs, q2, s2, sizes)[:2], "y")
        check(dw2, *orc.weight_gradient(h8, hs, dy, sizes, F32), "dw2")
        dh = matmul_fp8_blocks(d8, ds, q2.transpose(1, 2).contiguous().transpose(1, 2).transpose(1, 2), s2.transpose(1, 2), None, md)
        check(dh, *orc.product(d8, ds, q2.transpose(1, 2), s2.transpose(1, 2), sizes)[:2], "dh")
        da = swiglu_fp8_backward(dh, a8, as_, 1.702, 7.0)
        x8, xs = downcast_to_fp8_blocks(x)
        check(dw1, *orc.weight_gradient(x8, xs, da, sizes, BF16), "dw1")
        q1, s1 = downcast_to_fp8_blocks(w1, 128)
        g8, gs = downcast_to_fp8_blocks(da)
        check(dx, *orc.product(g8, gs, q1.transpose(1, 2), s1.transpose(1, 2), sizes)[:2], "dx")


def test_a_served_layer_from_router_to_combine():
    """routing -> gathered product with swiglu -> quantiser -> scattered product with gate weights -> sum over a token's experts."""
    from triton_kernels.legacy import routing
    from triton_kernels.reduce import reduce
    g = _gen(22)
    T, d, f, E, k = 90, 256, 384, 8, 2
    logits = torch.randn((T, E), generator=g).cuda()
    x8, xs = downcast_to_fp8_blocks(_rows(g, T, d))
    _, _, _, w1, s1 = _operands(31, 1, d, 2 * f, E)
    _, _, _, w2, s2 = _operands(32, 1, f, d, E)
    rdata, gather, scatter = routing(logits, k)
    sizes = rdata.expt_hist.tolist()
    h = matmul_fp8_blocks(x8, xs, w1, s1, None, rdata.expt_data, gather_indx=rdata.token_indx, fused_activation=SWIGLU)
    h8, hs = downcast_to_fp8_blocks(h)
    y = matmul_fp8_blocks(h8, hs, w2, s2, None, rdata.expt_data, scatter_indx=scatter.dst_indx, gammas=rdata.gate_scal)
    out, _ = reduce(y.view(T, k, -1), dim=1)
    check(h, *orc.product(x8, xs, w1, s1, sizes, gather=rdata.token_indx, swiglu=ACT)[:2], "h")
    want, bound, written = orc.product(h8, hs, w2, s2, sizes, scatter=scatter.dst_indx, gammas=rdata.gate_scal)
    assert written.all()
    check(y, want, bound, "y")
    check(out, want.view(T, k, -1).sum(1), bound.view(T, k, -1).sum(1) + 2.0**-8 * want.view(T, k, -1).sum(1).abs() + 2.0**-130, "out")


def test_another_stream():
    g, a, a_scale, w, w_scale = _operands(41, 200, 384, 256)
    want = matmul_fp8_blocks(a, a_scale, w, w_scale)
    x = _rows(g, 64, 256).requires_grad_()
    wp = (torch.randn((256, 128), generator=g) * 0.1).cuda().requires_grad_()
    dy = _rows(g, 64, 128)
    grads = torch.autograd.grad(linear_fp8_blocks(x, wp), (x, wp), dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = matmul_fp8_blocks(a, a_scale, w, w_scale)
        again = torch.autograd.grad(linear_fp8_blocks(x, wp), (x, wp), dy)
    side.synchronize()
    assert torch.equal(y, want) and all(torch.equal(p, q) for p, q in zip(grads, again))


def test_captured_and_replayed():
    g = _gen(43)
    T, d, f, E = 96, 256, 128, 3
    md = _metadata([40, 0, 56])
    x = _rows(g, T, d)
    w1, w2 = ((torch.randn(s, generator=g) * 0.05).to(BF16).cuda() for s in ((E, d, 2 * f), (E, f, d)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.no_grad():
        _block(x, w1, w2, md)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        y = _block(x, w1, w2, md)
    for _ in range(4):
        x.copy_(_rows(g, T, d))
        graph.replay()
        torch.cuda.synchronize()
        with torch.no_grad():
            assert torch.equal(y, _block(x, w1, w2, md))


def test_a_captured_training_step():
    g = _gen(44)
    T, d, f, E = 96, 256, 128, 3
    md = _metadata([40, 0, 56])
    leaves = [_rows(g, T, d).requires_grad_()] + [(torch.randn(s, generator=g) * 0.05).to(BF16).cuda().requires_grad_() for s in ((E, d, 2 * f), (E, f, d))]
    dy = _rows(g, T, d)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(_block(*leaves, md), leaves, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = _block(*leaves, md)
        grads = torch.autograd.grad(y, leaves, dy)
    for _ in range(3):
        with torch.no_grad():
            leaves[0].copy_(_rows(g, T, d))
            leaves[1].mul_(1.1)
        graph.replay()
        torch.cuda.synchronize()
        z = _block(*leaves, md)
        assert torch.equal(y, z) and all(torch.equal(p, q) for p, q in zip(grads, torch.autograd.grad(z, leaves, dy)))
        del z


def test_a_capture_beside_a_living_graph_is_refused():
    x = _rows(_gen(45), 8, 128).requires_grad_()
    w = torch.ones((128, 64), device="cuda", dtype=BF16, requires_grad=True)
    alive, alive_h = linear_fp8_blocks(x, w), swiglu_fp8_checkpoint(x, 1.0)
    graph = torch.cuda.CUDAGraph()
    seen = []
    with torch.cuda.graph(graph):
        y = torch.zeros(4, device="cuda") + 1
        for call in (lambda: linear_fp8_blocks(x, w), lambda: swiglu_fp8_checkpoint(x, 1.0)):
            try:
                call()
            except RuntimeError as e:
                seen.append("still alive" in str(e))
    assert seen == [True, True]
    graph.replay()
    torch.cuda.synchronize()
    assert (y == 1).all() and alive.shape == (8, 64) and alive_h.shape == (8, 64)


def test_second_derivatives_are_refused():
    x = _rows(_gen(46), 8, 128).requires_grad_()
    w = torch.ones((128, 64), device="cuda", dtype=BF16, requires_grad=True)
    for y in (linear_fp8_blocks(x, w), swiglu_fp8_checkpoint(x, 1.0)):
        d, = torch.autograd.grad(y.float().square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiable once"):
            d.sum().backward()


def test_hooks_on_saved_tensors():
    x = _rows(_gen(47), 40, 200).requires_grad_()
    w = (torch.randn((200, 72), generator=_gen(48)) * 0.1).cuda().requires_grad_()
    dy, dh = _rows(_gen(49), 40, 72), _rows(_gen(50), 40, 100)
    want = torch.autograd.grad(linear_fp8_blocks(x, w), (x, w), dy) + torch.autograd.grad(swiglu_fp8_checkpoint(x, 1.0), x, dh)
    with torch.autograd.graph.save_on_cpu():
        y, h = linear_fp8_blocks(x, w), swiglu_fp8_checkpoint(x, 1.0)
    got = torch.autograd.grad(y, (x, w), dy) + torch.autograd.grad(h, x, dh)
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t[:1]):
        y, h = linear_fp8_blocks(x, w), swiglu_fp8_checkpoint(x, 1.0)
    for out, d in ((y, dy), (h, dh)):
        with pytest.raises((ValueError, RuntimeError), match="as the forward pass saved it"):
            torch.autograd.grad(out, x, d)


@pytest.mark.parametrize("T,K,N,sizes", [(8192, 128, 72, None), (5000, 136, 520, [700, 0, 3300, 64, 900]), (4100, 256, 256, [4100, 0]), (1025, 16, 8, None), (20000, 64, 24, [1, 19999])])
def test_weight_gradients_of_long_slices_in_parts(T, K, N, sizes):
    g = _gen(T, K, N)
    x, s = downcast_to_fp8_blocks(_rows(g, T, K))
    dy = _rows(g, T, N, BF16, 0.02)
    md = None if sizes is None else _metadata(sizes, T)
    total = T if sizes is None else sum(sizes)
    for out_dtype in (F32, BF16, F16):
        dw = weight_gradient_fp8_blocks(x, s, dy, md, out_dtype)
        check(dw.view(-1, K, N), *orc.weight_gradient(x[:total], s[:total], dy[:total], sizes, out_dtype), "dw")
        assert torch.equal(weight_gradient_fp8_blocks(x, s, dy, md, out_dtype), dw)


@pytest.mark.parametrize("M,K,N,E", [(48, 264, 520, 1), (130, 1000, 1032, 4), (500, 384, 1024, 8), (400, 1048, 640, 280), (2500, 160, 264, 300), (20, 144, 4104, 12)])
@pytest.mark.parametrize("out_dtype,swiglu", [(BF16, False), (F16, True)])
def test_products_of_middle_sizes(M, K, N, E, out_dtype, swiglu):
    g, a, a_scale, w, w_scale = _operands(12, M, K, N, E)
    sizes = _deal(g, M, E)
    _check_product(a, a_scale, w, w_scale, out_dtype, sizes, swiglu=swiglu, bias=torch.randn((E, N), generator=g).cuda())
    at = torch.randint(M, (M, ), generator=g, dtype=torch.int32).cuda()
    _check_product(a, a_scale, w, w_scale, out_dtype, sizes, swiglu=swiglu, gather=at)


@pytest.mark.parametrize("M,E", [(900, 3), (257, 1)])
def test_many_rows_of_lines_that_begin_anywhere(M, E):
    K, N = 300, 136
    g, a, a_scale, w, w_scale = _operands(13, M, K, N, E, 307)
    odd = torch.full((E, N, K + 3), NAN, device="cuda").to(E4M3)
    odd[:, :, 1:K + 1] = w.transpose(1, 2)
    sizes = _deal(g, M, E)
    y = _check_product(a, a_scale, odd[:, :, 1:K + 1].transpose(1, 2), w_scale, BF16, sizes)
    assert torch.equal(matmul_fp8_blocks(a.contiguous(), a_scale, w, w_scale, None, _metadata(sizes)), y)


def test_a_slice_of_more_rows_than_the_schedule_counts():
    M, K, N = 2**21 + 300, 16, 16
    g = _gen(14)
    a = torch.randint(0, 120, (M, K), generator=g, dtype=torch.uint8).cuda().view(E4M3)
    a_scale = (torch.rand((M, 1), generator=g) + 0.5).cuda()
    _, _, _, w, w_scale = _operands(15, 4, K, N, 2)
    sizes = [M - 100, 60]
    md = _metadata(sizes, M)
    y = matmul_fp8_blocks(a, a_scale, w, w_scale, None, md)
    for lo, hi, e in ((0, 500, 0), (2**21 - 300, M - 100, 0), (M - 100, M - 40, 1)):
        want, bound, _ = orc.product(a[lo:hi], a_scale[lo:hi], w[e:e + 1], w_scale[e:e + 1])
        check(y[lo:hi], want, bound, "y")
    with pytest.raises(NotImplementedError, match="more than 2097152 rows"):
        matmul_fp8_blocks(a, a_scale, w, w_scale, None, md, out_dtype=F32)


def test_linear_without_slices_or_row_blocks():
    x = _rows(_gen(16), 30, 256)
    before = torch.are_deterministic_algorithms_enabled()
    torch.use_deterministic_algorithms(True)                               # (new memory holds NaN)
    try:
        for E in (0, 2):
            w = torch.ones((E, 256, 64), device="cuda", dtype=BF16)
            for rows in (0, 30):                                           # (metadata of no rows have no row block)
                xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
                y = linear_fp8_blocks(xg, wg, _metadata([0] * E, rows))
                dx, dw = torch.autograd.grad(y, (xg, wg), torch.ones_like(y))
                assert y.shape == (30, 64) and (y == 0).all() and (dx == 0).all() and (dw == 0).all() and dw.shape == w.shape
    finally:
        torch.use_deterministic_algorithms(before)


@pytest.mark.parametrize("T,K,N", [(300, 264, 136), (2600, 512, 2056)])
def test_linear_with_weights_of_other_scales(T, K, N):
    from triton_kernels.fp8_blocks import Fp8Weight
    g = _gen(T, K, N)
    sizes = [T // 2, T - T // 2]
    md = _metadata(sizes)
    x, dy = _rows(g, T, K).requires_grad_(), _rows(g, T, N, BF16, 0.01)
    w = (torch.randn((2, K, N), generator=g) * 0.05).cuda().requires_grad_()
    q = quantize_fp8_weight(w)
    q = Fp8Weight(q.values, q.values_n, q.scales * (torch.rand(q.scales.shape, generator=g).cuda() + 0.51))
    y = linear_fp8_blocks(x, w, md, q)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    x8, xs = downcast_to_fp8_blocks(x.detach())
    d8, ds = downcast_to_fp8_blocks(dy)
    check(y, *orc.product(x8, xs, q.values, q.scales, sizes)[:2], "y")
    check(dx, *orc.product(d8, ds, q.values_n.transpose(1, 2), q.scales.transpose(1, 2), sizes)[:2], "dx")
    check(dw, *orc.weight_gradient(x8, xs, dy, sizes, F32), "dw")


@pytest.mark.parametrize("E,T,K,N", [(70, 900, 136, 200), (70, 45000, 16, 40), (129, 3000, 264, 520)])
def test_weight_gradients_of_many_slices(E, T, K, N):
    g = _gen(E, T, K, N)
    sizes = _deal(g, T, E)
    x, s = downcast_to_fp8_blocks(_rows(g, T, K))
    dy = _rows(g, T, N, BF16, 0.02)
    for out_dtype in (F32, BF16):
        check(weight_gradient_fp8_blocks(x, s, dy, _metadata(sizes), out_dtype), *orc.weight_gradient(x, s, dy, sizes, out_dtype), "dw")


def test_gradients_of_one_row_expanded():
    x = _rows(_gen(17), 40, 256).requires_grad_()
    w = (torch.randn((256, 64), generator=_gen(18)) * 0.1).cuda().requires_grad_()
    row = _rows(_gen(19), 1, 64)
    want = torch.autograd.grad(linear_fp8_blocks(x, w), (x, w), row.expand(40, 64).contiguous())
    got = torch.autograd.grad(linear_fp8_blocks(x, w), (x, w), row.expand(40, 64))
    assert all(torch.equal(p, q) for p, q in zip(want, got))


def test_offsets_past_32_bits():
    R, K, N = 2**20 + 70_000, 4096, 64                                     # 4.6 GB in 8 bits
    at = torch.tensor([0, 1, R // 2, 2**19 + 1, 2**20 + 3] + list(range(R - 60, R)), device="cuda")
    a = torch.randint(0, 120, (R, K), dtype=torch.uint8, device="cuda").view(E4M3)
    a_scale = torch.ldexp(torch.ones((), device="cuda"), torch.randint(-6, 6, (R, K // 128), device="cuda"))
    _, _, _, w, w_scale = _operands(20, 4, K, N)
    rows, scales = a.view(torch.uint8)[at].view(E4M3), a_scale[at]
    for out_dtype in (BF16, F32):
        want, bound, _ = orc.product(rows, scales, w, w_scale, out_dtype=out_dtype)
        check(matmul_fp8_blocks(a, a_scale, w, w_scale, out_dtype=out_dtype)[at], want, bound, "y")
        check(matmul_fp8_blocks(a, a_scale, w, w_scale, gather_indx=at.int(), out_dtype=out_dtype), want, bound, "gathered")
    dy = torch.zeros((R, N), dtype=BF16, device="cuda")
    dy[at] = _rows(_gen(21), len(at), N, BF16, 0.1)
    check(weight_gradient_fp8_blocks(a, a_scale, dy, None, F32)[None], *orc.weight_gradient(rows, scales, dy[at]), "dw")
    x = upcast_from_fp8_blocks(a, a_scale)
    assert torch.equal(x[at].cpu(), orc.upcast(rows, scales).to(BF16))
    v, s = downcast_to_fp8_blocks(x)
    _same(v.view(torch.uint8)[at].view(E4M3), s[at], orc.downcast(x[at]))
    h, v2, s2 = swiglu_fp8_forward(x, *ACT)
    check(h[at], *orc.swiglu(x[at], *ACT), "h")
    assert torch.equal(v2.view(torch.uint8), v.view(torch.uint8)) and torch.equal(s2, s)
    check(swiglu_fp8_backward(h, v, s, *ACT)[at], *orc.swiglu_backward(h[at], v.view(torch.uint8)[at].view(E4M3), s[at], *ACT), "da")


@pytest.mark.parametrize("M,K,N,E", [(70, 2057, 136, 1), (300, 2100, 520, 3), (40, 2176, 264, 1), (130, 4000, 1024, 2), (64, 2048, 16, 1), (97, 6150, 72, 2)])
@pytest.mark.parametrize("out_dtype,swiglu", [(BF16, True), (F16, False)])
def test_products_of_few_columns_and_long_rows(M, K, N, E, out_dtype, swiglu):
    g, a, a_scale, w, w_scale = _operands(22, M, K, N, E)
    wide = torch.full((E, N, -(-K // 16) * 16), NAN, device="cuda").to(E4M3)  # lines at sixteen-byte boundaries, NaN behind their ends
    wide[:, :, :K] = w.transpose(1, 2)
    a2 = torch.full((M, wide.shape[2]), NAN, device="cuda").to(E4M3)
    a2[:, :K] = a
    sizes = _deal(g, M, E)
    y = _check_product(a2[:, :K], a_scale, wide[:, :, :K].transpose(1, 2), w_scale, out_dtype, sizes, swiglu=swiglu)
    at = torch.arange(M, dtype=torch.int32, device="cuda")
    assert torch.equal(_check_product(a2[:, :K], a_scale, wide[:, :, :K].transpose(1, 2), w_scale, out_dtype, sizes, swiglu=swiglu, gather=at), y)
