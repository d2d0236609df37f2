"""The weights' gradient in 8 bits on the tiles that training steps take, each call shown to take them: tiles of 256 and 128, many and few tiles a slice (an XCD's own eighth
of each slice, and every eighth of all), more tiles than workgroups, uneven and empty slices, and exponents in the conversion.  Against the 64-bit oracle at columns around
the tiles' borders."""
import pytest
import torch

from fp8_cases import gradient_desc, gradient_kernel_of
from oracle import fp8_blocks as orc
from oracle.rows import check
from triton_kernels.fp8_blocks import downcast_to_fp8_blocks, linear_fp8_blocks, weight_gradient_fp8_blocks
from triton_kernels.tensor import make_ragged_tensor_metadata

pytestmark = pytest.mark.gpu

F32, BF16, F16, E4M3 = torch.float32, torch.bfloat16, torch.float16, torch.float8_e4m3fn
NAN = float("nan")

# rows, K, N, slices, tile; tiles a slice beside it
CASES = [(300, 2300, 2100, 7, 256),   # 81, no multiple of 8
         (900, 2048, 2056, 8, 256),   # 72
         (1500, 2300, 2001, 8, 256),  # 72, odd columns (copied lines), slices of several stages
         (2000, 520, 776, 50, 256),   # 12: every eighth of all
         (70, 5800, 5900, 1, 256),    # 552
         (400, 1100, 1100, 3, 128),   # 81
         (500, 1600, 1601, 5, 128),   # 169, more than workgroups
         (1200, 2000, 520, 6, 128)]   # 80


def _sizes(g, rows, E):
    if E == 1:
        return None
    cut = torch.randint(0, rows + 1, (E - 1, ), generator=g).sort().values.tolist()
    sizes = [b - a for a, b in zip([0] + cut, cut + [rows])]
    sizes[0], sizes[1] = sizes[0] + sizes[1], 0
    return sizes


def _metadata(sizes, rows):
    return None if sizes is None else make_ragged_tensor_metadata(torch.tensor(sizes, dtype=torch.int32, device="cuda"), rows)


def _some(g, N):
    near = {0, 1, 7, 8, 63, 64, 127, 128, 255, 256, N // 256 * 256 - 1, N // 256 * 256, N // 128 * 128 - 1, N // 128 * 128, N - 1} | set(torch.randint(N, (40, ), generator=g).tolist())
    return torch.tensor(sorted(n for n in near if 0 <= n < N), device="cuda")


def _rows(g, R, C, dtype, scale=1.0):
    return (torch.randn((R, C), generator=g) * (torch.rand((R, 1), generator=g) * 2 + 0.1) * scale).to(dtype).cuda()


@pytest.mark.parametrize("dtype,out_dtype", [(BF16, F32), (BF16, BF16), (F16, F32), (F16, F16), (F16, BF16)])
@pytest.mark.parametrize("T,K,N,E,tile", CASES)
def test_gradients_on_tiles(T, K, N, E, tile, dtype, out_dtype):
    g = torch.Generator().manual_seed(T + K)
    assert gradient_kernel_of(gradient_desc(T + 20, K, N, E, dy_dtype=dtype), torch.cuda.get_device_properties(0).multi_processor_count) == (tile, 1)
    sizes = _sizes(g, T, E)
    total = T + (20 if E > 1 else 0)                                       # rows that no slice holds
    x, s = downcast_to_fp8_blocks(_rows(g, total, K, dtype))
    s = s * (1.0 if out_dtype == F32 else 1.37)                            # scales of any size: rounded to 16 bits behind them
    dy = _rows(g, total, N, dtype, 0.02)
    x[T:], dy[T:] = torch.full((total - T, K), NAN, device="cuda").to(E4M3), NAN
    md = _metadata(sizes, total)
    dw = weight_gradient_fp8_blocks(x, s, dy, md, out_dtype).view(E, K, N)
    some = _some(g, N)
    want, bound = orc.weight_gradient(x[:T], s[:T], dy[:T][:, some], sizes, out_dtype)
    check(dw[:, :, some], want, bound, "dw")
    assert dw.isfinite().all() and (sizes is None or (dw[1] == 0).all())
    assert torch.equal(weight_gradient_fp8_blocks(x, s, dy, md, out_dtype).view(E, K, N), dw)


@pytest.mark.parametrize("dtype,weights", [(BF16, F32), (BF16, BF16), (F16, F32)])
@pytest.mark.parametrize("T,K,N,E,tile", CASES)
def test_gradients_of_linear_layers_on_tiles(T, K, N, E, tile, dtype, weights):
    """Scales that are powers of two: exponents in the conversion to bf16, which is exact as the product is."""
    g = torch.Generator().manual_seed(T + N)
    assert gradient_kernel_of(gradient_desc(T, K, N, E, dy_dtype=dtype, pow2_scales=1), torch.cuda.get_device_properties(0).multi_processor_count) == (tile, 1)
    sizes = _sizes(g, T, E)
    x = _rows(g, T, K, dtype)
    w = torch.zeros((E, K, N) if E > 1 else (K, N), dtype=weights, device="cuda", requires_grad=True)
    dy = _rows(g, T, N, dtype, 0.02)
    md = _metadata(sizes, T)
    dw, = torch.autograd.grad(linear_fp8_blocks(x, w, md), w, dy)
    x8, xs = downcast_to_fp8_blocks(x)
    some = _some(g, N)
    want, bound = orc.weight_gradient(x8, xs, dy[:, some], sizes, weights)
    check(dw.view(E, K, N)[:, :, some], want, bound, "dw")
    assert torch.equal(weight_gradient_fp8_blocks(x8, xs, dy, md, weights).view(E, K, N), dw.view(E, K, N))
