"""The product in 8 bits on the kernels of large calls, tiles of 128 and of 256, each call shown to take them: one stage and many, several tiles a workgroup,
ends of K and N inside a piece and a tile, gathered and scattered rows, the epilogue, scales of any size and exponents in the instruction.  Against the 64-bit oracle at rows
around the tiles' borders."""
import pytest
import torch

from fp8_cases import kernel_of, product_desc
from oracle import fp8_blocks as orc
from oracle.rows import check
from triton_kernels.fp8_blocks import downcast_to_fp8_blocks, linear_fp8_blocks, matmul_fp8_blocks
from triton_kernels.matmul import FnSpecs, FusedActivation
from triton_kernels.swiglu import swiglu_fn
from triton_kernels.tensor import make_ragged_tensor_metadata

pytestmark = pytest.mark.gpu

F32, BF16, F16, E4M3 = torch.float32, torch.bfloat16, torch.float16, torch.float8_e4m3fn
NAN, INF = float("nan"), float("inf")
ACT = (1.702, 7.0)
SWIGLU = FusedActivation(FnSpecs("swiglu", swiglu_fn, ("alpha", "limit"), reduction_n=2), ACT)

# rows, K, N, slices, tile: K of one, two and many blocks, with a whole, a part and none of its last piece; N that ends within a tile, at odd columns too; more tiles than
# workgroups (512 of 128, 256 of 256) and fewer
CASES = [(4000, 100, 2000, 40, 128), (4000, 250, 2001, 40, 128), (4000, 256, 2000, 40, 128), (2600, 1000, 1544, 7, 128), (2048, 1024, 2304, 1, 128), (2400, 600, 2900, 30, 128),
         (6000, 100, 4200, 4, 256), (6000, 250, 4201, 3, 256), (6000, 128, 4200, 4, 256), (6000, 1000, 3000, 2, 256), (4100, 1040, 4097, 1, 256), (5000, 520, 5000, 5, 256), (5000, 272, 3001, 12, 256)]


def _cus():
    return torch.cuda.get_device_properties(0).multi_processor_count


def _sizes(g, rows, E):
    """Uneven slices, an empty one and one of a single row among them."""
    if E == 1:
        return None
    cut = torch.randint(0, rows + 1, (E - 1, ), generator=g).sort().values.tolist()
    sizes = [b - a for a, b in zip([0] + cut, cut + [rows])]
    if E > 3:
        sizes[0], sizes[1] = sizes[0] + sizes[1], 0
        sizes[3], sizes[2] = sizes[3] + max(sizes[2] - 1, 0), min(sizes[2], 1)
    return sizes


def _some(g, sizes, rows):
    """Rows of each slice: its ends, those around the first and last tiles' borders, a few others; and how many of each."""
    some, counts, lo = [], [], 0
    for n in [rows] if sizes is None else sizes:
        near = {0, 1, 15, 16, 63, 64, 127, 128, 255, 256, n // 128 * 128 - 1, n // 128 * 128, n // 256 * 256, n - 1} | set(torch.randint(max(n, 1), (4, ), generator=g).tolist())
        near = sorted(r for r in near if 0 <= r < n)
        some += [lo + r for r in near]
        counts.append(len(near))
        lo += n
    return torch.tensor(some, device="cuda"), counts


def _metadata(sizes, rows):
    return None if sizes is None else make_ragged_tensor_metadata(torch.tensor(sizes, dtype=torch.int32, device="cuda"), rows)


def _pick(t, rows):
    return t.view(torch.uint8)[rows].view(E4M3)


def _padded(values, pitch):
    """The same lines with NaN between them, each at a sixteen-byte boundary."""
    out = torch.full((*values.shape[:-1], pitch), NAN, device="cuda").to(E4M3)
    out[..., :values.shape[-1]] = values
    return out[..., :values.shape[-1]]


def _operands(g, rows, K, N, E):
    x = torch.randn((rows, K), generator=g) * (torch.rand((rows, 1), generator=g) * 2 + 0.1)
    a, a_scale = downcast_to_fp8_blocks(x.cuda())
    a_scale = a_scale * (torch.rand(a_scale.shape, generator=g).cuda() + 0.5)  # (of any size)
    w = (torch.randn((E, N, K), generator=g) * 120).clamp(-448, 448).cuda().to(E4M3)
    w_scale = (torch.rand((E, -(-N // 128), -(-K // 128)), generator=g) * 1e-3 + 1e-5).cuda()
    pitch = -(-K // 16) * 16 + 16
    return _padded(a, pitch), a_scale, _padded(w, pitch).transpose(1, 2), w_scale.transpose(1, 2)


@pytest.mark.parametrize("out_dtype", [BF16, F16])
@pytest.mark.parametrize("options", ["plain", "gather", "scatter", "all"])
@pytest.mark.parametrize("rows,K,N,E,tile", CASES)
def test_products_on_tiles(rows, K, N, E, tile, options, out_dtype):
    g = torch.Generator().manual_seed(rows + K)
    swiglu = options in ("gather", "all")
    N += N % 2 if swiglu else 0
    tokens = 1500 if options in ("gather", "all") else rows
    a, a_scale, w, w_scale = _operands(g, tokens, K, N, E)
    sizes = _sizes(g, rows, E)
    behind = 100 if sizes is not None else 0                               # rows that no slice holds
    kw, total = {}, rows + behind
    if options in ("gather", "all"):
        kw["gather_indx"] = torch.randint(tokens, (total, ), generator=g, dtype=torch.int32).cuda()
    else:
        a, a_scale = torch.cat([a.view(torch.uint8), a.view(torch.uint8)[:behind]]).view(E4M3), torch.cat([a_scale, a_scale[:behind]])
        a = _padded(a, w.stride(2))
    if options in ("scatter", "all"):
        at = torch.randperm(total, generator=g).to(torch.int32)
        at[::7] = -1
        kw["scatter_indx"] = at.cuda()
        kw["gammas"] = torch.rand(total, generator=g).cuda()
    if options in ("all", "scatter"):
        kw["bias"] = torch.randn((E, N), generator=g).to(BF16 if options == "all" else F32).cuda()
    d = product_desc(total, K, N, E, out_dtype=out_dtype, x_stride=a.stride(0), w_stride=w.stride(2), x_rows=a.shape[0], gather="gather_indx" in kw)
    assert kernel_of(d, _cus()) == tile and a.data_ptr() % 16 == 0 and w.data_ptr() % 16 == 0
    call = lambda: matmul_fp8_blocks(a, a_scale, w, w_scale, a_ragged_metadata=_metadata(sizes, total), fused_activation=SWIGLU if swiglu else None, out_dtype=out_dtype, **kw)  # noqa: E731
    before = torch.are_deterministic_algorithms_enabled()
    torch.use_deterministic_algorithms(True)                               # (new memory holds NaN)
    try:
        y = call()
    finally:
        torch.use_deterministic_algorithms(before)
    to = torch.arange(total, device="cuda") if "scatter_indx" not in kw else kw["scatter_indx"].long()
    written = torch.zeros(total, dtype=torch.bool, device="cuda")
    written[to[:rows][to[:rows] >= 0]] = True
    assert torch.equal(y.isfinite().all(1), written) and y[~written].isnan().all()
    some, counts = _some(g, sizes, rows)
    src = some if "gather_indx" not in kw else kw["gather_indx"].long()[some]
    want, bound, _ = orc.product(_pick(a, src), a_scale[src], w, w_scale, counts, bias=kw.get("bias"), swiglu=ACT if swiglu else None, out_dtype=out_dtype,
                                 gammas=None if "gammas" not in kw else kw["gammas"][some])
    live = to[some] >= 0
    check(y[to[some][live]], want[live.cpu()], bound[live.cpu()], "y")
    z = call()
    assert torch.equal(z[written], y[written])


@pytest.mark.parametrize("rows,K,N,E,tile", [(2600, 1000, 1544, 7, 128), (6000, 272, 4200, 3, 256)])
def test_what_is_not_finite_stays_in_its_row_or_column_of_a_tile(rows, K, N, E, tile):
    g = torch.Generator().manual_seed(5)
    a, a_scale, w, w_scale = _operands(g, rows, K, N, E)
    a[rows // 2, K - 1], a_scale[rows - 1, 1] = NAN, INF
    w.transpose(1, 2)[E - 1, 7, 5] = NAN
    sizes = _sizes(g, rows, E)
    assert kernel_of(product_desc(rows, K, N, E, x_stride=a.stride(0), w_stride=w.stride(2)), _cus()) == tile
    y = matmul_fp8_blocks(a, a_scale, w, w_scale, a_ragged_metadata=_metadata(sizes, rows))
    bad = torch.zeros((rows, N), dtype=torch.bool)
    bad[rows // 2], bad[rows - 1], bad[rows - sizes[-1]:, 7] = True, True, True
    assert torch.equal(y.isfinite().cpu(), ~bad)


# rows, K, N, slices, the output's tile and that of the input's gradient
LINEAR = [(6000, 1000, 1500, 1, 256, 128), (6000, 1000, 1500, 3, 256, 128), (6200, 520, 5000, 5, 256, 64), (4000, 2000, 100, 40, 64, 128), (5000, 3001, 272, 12, 64, 256), (6000, 3000, 1000, 2, 128, 256)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,K,N,E,tile_y,tile_dx", LINEAR)
def test_linear_layers_on_tiles(T, K, N, E, tile_y, tile_dx, dtype):
    """Scales that are powers of two: exponents in the matrix instruction."""
    g = torch.Generator().manual_seed(T + K)
    sizes = _sizes(g, T, E)
    total = T + (100 if E > 1 else 0)
    x = (torch.randn((total, K), generator=g) * torch.ldexp(torch.ones(total, 1), torch.randint(-6, 4, (total, 1), generator=g))).to(dtype).cuda().requires_grad_()
    w = (torch.randn((E, K, N), generator=g) * 0.05).cuda().requires_grad_()
    dy = (torch.randn((total, N), generator=g) * 0.1).to(dtype).cuda()
    assert kernel_of(product_desc(total, K, N, E, out_dtype=dtype), _cus()) == tile_y and kernel_of(product_desc(total, N, K, E, out_dtype=dtype), _cus()) == tile_dx
    md = _metadata(sizes, total)
    y = linear_fp8_blocks(x, w if E > 1 else w[0], md)
    dx, = torch.autograd.grad(y, x, dy)
    assert (y[T:] == 0).all() and (dx[T:] == 0).all() and y.isfinite().all() and dx.isfinite().all()
    x8, xs = downcast_to_fp8_blocks(x.detach())
    d8, ds = downcast_to_fp8_blocks(dy)
    w8, ws = downcast_to_fp8_blocks(w.detach(), 128)
    some, counts = _some(g, sizes, T)
    check(y[some], *orc.product(_pick(x8, some), xs[some], w8, ws, counts, out_dtype=dtype)[:2], "y")
    check(dx[some], *orc.product(_pick(d8, some), ds[some], w8.transpose(1, 2), ws.transpose(1, 2), counts, out_dtype=dtype)[:2], "dx")
