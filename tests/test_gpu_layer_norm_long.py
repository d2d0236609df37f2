"""Layer norm of long rows and of many: sums of tens of thousands of numbers a lane, parameters of more columns than one launch has threads for,
workgroups that take several of the longest rows that fit one, fp16."""
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


@pytest.mark.parametrize("dtype", [F32, BF16, torch.float16])
@pytest.mark.parametrize("M,C", [(600, 8200), (1100, 16384), (1030, 12001)])
def test_many_rows_of_a_workgroup_each(M, C, dtype):
    """More rows of 8193 to 16384 columns than the backward pass has workgroups for: the two buffers of its barrier, the row requested ahead, the running sums."""
    g = torch.Generator(device="cuda").manual_seed(M + C)
    x = (torch.randn((M, C), generator=g, device="cuda") * 1.5 + 0.3).to(dtype)
    dy = torch.randn((M, C), generator=g, device="cuda").to(dtype)
    w, b = torch.randn(C, generator=g, device="cuda"), torch.randn(C, generator=g, device="cuda")
    y, mean, rstd = layer_norm_forward(x, w, b)
    orc.check(y, *orc.layer_norm(x, w, b), "y")
    want = orc.layer_norm_backward(dy, x, w, 1e-5, b)
    for name, got in zip(("dx", "dweight", "dbias"), layer_norm_backward(dy, x, mean, rstd, w, b)):
        orc.check(got, *want[name], name)
    for name, got in zip(("dx", "dweight", "dbias"), layer_norm_backward(dy, x, mean, rstd, w, b, need_dx=False)):
        assert got is None if name == "dx" else orc.check(got, *want[name], name) is None


@pytest.mark.parametrize("M,C", [(4099, 256), (4099, 40), (6000, 1023), (2050, 7), (2048, 512), (2047, 513), (2049, 4096), (2200, 4100), (9001, 130)])
def test_many_rows_in_fp16(M, C):
    g = torch.Generator(device="cuda").manual_seed(M + C)
    x, dy = (torch.randn((M, C), generator=g, device="cuda") for _ in range(2))
    x, dy = (x * 1.5 + 0.3).half(), dy.half()
    w, b = torch.randn(C, generator=g, device="cuda"), torch.randn(C, generator=g, device="cuda")
    y, mean, rstd = layer_norm_forward(x, w, b)
    orc.check(y, *orc.layer_norm(x, w, b), "y")
    want = orc.layer_norm_backward(dy, x, w, 1e-5, b)
    for name, got in zip(("dx", "dweight", "dbias"), layer_norm_backward(dy, x, mean, rstd, w, b)):
        orc.check(got, *want[name], name)
