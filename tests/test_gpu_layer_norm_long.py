"""Layer norm of rows far longer than a model's: sums of tens of thousands of numbers a lane, and parameters of more columns than one launch has threads for."""
import pytest
import torch

from oracle import rows as orc
from triton_kernels.layer_norm import layer_norm_backward, layer_norm_forward

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.parametrize("C", [2**27 + 17, 2**28 + 33])
def test_parameters_of_many_columns(C):
    """Of one row, where each of their gradients is a single product: the same bits as torch's."""
    g = torch.Generator(device="cuda").manual_seed(C)
    x, dy = (torch.randn((1, C), generator=g, device="cuda", dtype=BF16) for _ in range(2))
    w, b = torch.ones(C, dtype=F32, device="cuda"), torch.zeros(C, dtype=F32, device="cuda")
    mean, rstd = torch.full((1, ), 0.25, device="cuda"), torch.full((1, ), 1.5, device="cuda")
    dx, dw, db = layer_norm_backward(dy, x, mean, rstd, w, b, need_dx=False)
    assert dx is None
    assert torch.equal(db, dy[0].float())
    assert torch.equal(dw, dy[0].float() * ((x[0].float() - 0.25) * 1.5))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("size", [1.1**0.5, 0.7])
def test_sums_of_long_rows(dtype, size):
    """Elements of one size, whose squares each round the same way when they are added to a large sum; gradients likewise."""
    C = 2**24 + 300
    sign = torch.ones(C)
    sign[1::2] = -1
    x = (sign * size).to(dtype).cuda()[None]
    dy = (sign * 0.3 + 0.2).to(dtype).cuda()[None]
    y, mean, rstd = layer_norm_forward(x)
    orc.check(y, *orc.layer_norm(x), "y")
    want = 1 / (x.double().square().mean().item() + 1e-5)**0.5
    assert abs(rstd.item() - want) <= (orc.LN_DEPTH / 2 + 8) * orc.U * want
    orc.check(layer_norm_backward(dy, x, mean, rstd)[0], *orc.layer_norm_backward(dy, x)["dx"], "dx")
