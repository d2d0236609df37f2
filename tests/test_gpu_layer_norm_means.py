"""Layer norm of rows whose mean is large against their deviation, in 32 bits, where the mean's error counts: against a bound that knows the mean's own
rounding alone, and not the roundings of a sum of elements as large as the mean."""
import pytest
import torch

from oracle import rows as orc
from triton_kernels.layer_norm import layer_norm, layer_norm_backward, layer_norm_forward

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
# a part of a wave, a wave, a workgroup a row, a workgroup of 1024, rows that do not fit registers; few rows and many
SIZES = [(5, 9), (7, 130), (6, 1023), (3, 2880), (2, 4096), (3, 8191), (2, 16384), (2, 20000), (2050, 130), (2049, 500), (2051, 1023), (2048, 2880), (2053, 4096),
         (2050, 5000)]
VALUES = [12345.678, 1000.1, 333333.33, -7.7e8, 1e-3]


def _weights(C, seed=0):
    g = torch.Generator().manual_seed(C + seed)
    return (torch.randn(C, generator=g) * 0.2 + 1).cuda(), (torch.randn(C, generator=g) * 0.2).cuda()


@pytest.mark.parametrize("M,C", SIZES)
def test_rows_of_one_value_are_their_mean(M, C):
    """The differences are zero, so y is the bias, the weight's gradient zero, and the deviation that of eps."""
    w, b = _weights(C)
    x = torch.tensor(VALUES, device="cuda").repeat(M // len(VALUES) + 1)[:M, None].expand(M, C).contiguous()
    y, mean, rstd = layer_norm_forward(x, w, b)
    assert torch.equal(mean, x[:, 0])
    assert torch.equal(y, b.expand(M, C))
    want = 1e-5**-0.5  # (eps in 32 bits, the root and the reciprocal: two units each at most)
    assert ((rstd.double() - want).abs() <= 4 * orc.U * want).all()
    dy = torch.randn((M, C), generator=torch.Generator().manual_seed(1)).cuda()
    dx, dw, db = layer_norm_backward(dy, x, mean, rstd, w, b)
    assert not dw.any()
    zero = orc.layer_norm_backward(dy, torch.zeros_like(x), w, 1e-5, b)  # (the same rows, shifted)
    orc.check(dx, *zero["dx"], "dx")
    orc.check(db, *zero["dbias"], "dbias")


@pytest.mark.parametrize("dtype,value", [(torch.float16, 1023.5), (torch.float16, -61.9375), (BF16, 255.0), (BF16, -0.00390625 * 129)])
@pytest.mark.parametrize("M,C", [(2, 16383), (2, 20001), (2048, 3001)])
def test_rows_of_one_value_in_16_bits(M, C, dtype, value):
    """Values with all bits that the type has, whose sums need more than 24."""
    w, b = _weights(C)
    x = torch.full((M, C), value, dtype=dtype, device="cuda")
    y, mean, _ = layer_norm_forward(x, w, b)
    assert (x.float() == value).all() and (mean == value).all()
    assert torch.equal(y, b.to(dtype).expand(M, C))


def _bound(x, y, w, b, eps):
    """The mean is off by its own rounding, by those of the sum of the distances (which are no larger than a deviation and the first mean's last bits), and the
    variance by those of a sum of their squares; then as in the oracle."""
    xd = orc.d64(x)
    C = x.shape[-1]
    depth = min(C, orc.LN_DEPTH) + 2
    mu = xd.mean(-1, keepdim=True)
    d = xd - mu
    var = d.square().mean(-1, keepdim=True)
    r = 1 / torch.sqrt(var + eps)
    h = (d * r).abs()
    ulp = 2 * orc.U * mu.abs()
    off_mu = ulp / 2 + depth * orc.U * (d.abs().mean(-1, keepdim=True) + var.sqrt() + ulp)
    off_r = 0.5 * depth * orc.U * (1.1 * var + ulp.square()) * r.square() + 8 * orc.U  # relative
    aw = orc.d64(w).abs()
    return aw * (h * off_r + r * off_mu + 2 * orc.U * h) + orc.U * y.abs() + orc.U * orc.d64(b).abs() + orc.half_step(x.dtype, y)


@pytest.mark.parametrize("M,C", SIZES)
@pytest.mark.parametrize("spread", ["a last bit", "one element", "a thousandth", "a hundredth of the mean"])
def test_rows_beside_a_large_mean(M, C, spread):
    w, b = _weights(C)
    g = torch.Generator().manual_seed(M + C)
    x = torch.tensor(VALUES).repeat(M // len(VALUES) + 1)[:M, None].expand(M, C).clone()
    if spread == "a last bit":
        x = torch.where(torch.rand((M, C), generator=g) < 0.5, torch.nextafter(x, torch.full_like(x, float("inf"))), x)
    elif spread == "one element":
        x[:, C // 2] = torch.nextafter(x[:, 0], torch.full_like(x[:, 0], float("inf")))
    else:
        x *= 1 + torch.randn((M, C), generator=g) * (1e-3 if spread == "a thousandth" else 1e-2)
    x = x.cuda()
    n = min(M, 200)  # (rows that are compared)
    for eps in (1e-5, 1e-12):
        y = layer_norm(x, w, b, eps)
        want, _ = orc.layer_norm(x[:n], w, b, eps)
        orc.check(y[:n], want, _bound(x[:n], want, w, b, eps), f"y, eps {eps}")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,C", [(3, 300), (2, 4096), (2, 16384), (3, 20000), (2050, 300), (2050, 4096)])
def test_rows_whose_sum_is_beyond_32_bits(M, C, dtype):
    """Their mean is not: equal elements give the bias, and so do distances whose squares are beyond 32 bits."""
    w, b = _weights(C)
    x = torch.full((M, C), 2.0**126, device="cuda", dtype=dtype)
    x[1] = -x[1]
    y, mean, rstd = layer_norm_forward(x, w, b)
    assert torch.equal(mean, x[:, 0].float()) and torch.equal(y, b.to(dtype).expand(M, C))
    x[0, ::2] = 2.0**125
    assert torch.equal(layer_norm(x, w, b), b.to(dtype).expand(M, C))
