"""The gradients over a vocabulary against the statistics that the forward pass left: what is added to the statistics' own rounding."""
import pytest
import torch

from oracle import rows as orc
from triton_kernels.distill import _forward as distill_forward
from triton_kernels.distill import distill_topk_backward
from triton_kernels.logprobs import _forward as logprobs_forward
from triton_kernels.logprobs import token_logprobs_backward

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V,step", [(131072, 353), (2000, 9)])
def test_probabilities_are_those_of_the_stored_sum(V, step):
    """Rows with another number of equal logits each, whose probabilities are 1 / s in every place that is not masked.  Counted: two units for each of two exponentials
    of base two, and half a step for each of four products and roundings; the logarithm of s turned to base two is no rounding among them."""
    T = 200
    live = V - step * torch.arange(T, device="cuda")
    z = torch.where(torch.arange(V, device="cuda") < live[:, None], 0.0, float("-inf"))
    tokens, one = torch.zeros(T, dtype=torch.int64, device="cuda"), torch.ones(T, device="cuda")

    def check(g, stats, sign):
        p = torch.exp(-stats[1].double())
        assert not torch.where(torch.isfinite(z), torch.zeros_like(g), g).any()
        assert ((g[:, 1].double() - sign * p).abs() <= 8 * orc.U * p).all()  # (a place that every row has; the others of a row have the same bits)
        assert torch.equal(g[:, 1:], torch.where(torch.isfinite(z), g[:, 1:2], torch.zeros_like(g))[:, 1:])

    _, h, _, _, stats = logprobs_forward(z, tokens, 0, 1.0, True)
    check(token_logprobs_backward(z, tokens, h, stats, one, None), stats, -1)
    _, stats = distill_forward(z, torch.zeros((T, 1), device="cuda"), torch.zeros((T, 1), dtype=torch.int64, device="cuda"), 1.0, True)
    check(distill_topk_backward(z, torch.zeros((T, 1), device="cuda"), torch.zeros((T, 1), dtype=torch.int64, device="cuda"), stats, one), stats, 1)


def test_logarithms_beyond_32_bits():
    """Logits masked with the lowest value of fp32 at a temperature below one: their log probability is -inf in 32 bits, and so the loss of a teacher that holds
    one of them possible +inf; its gradient is that of a probability of zero."""
    z = torch.zeros((2, 300), device="cuda")
    z[:, 100:] = torch.finfo(torch.float32).min
    q, at = torch.zeros((2, 2), device="cuda"), torch.tensor([[3, 200], [3, 4]], device="cuda")
    one = torch.ones(2, device="cuda")
    lp, h, _, _, _ = logprobs_forward(z, torch.tensor([200, 4], device="cuda"), 0, 0.7, True)
    loss, stats = distill_forward(z, q, at, 0.7, True)
    g = distill_topk_backward(z, q, at, stats, one, 0.7)
    assert lp[0] == -float("inf") and loss[0] == float("inf")
    orc.check(lp[1:], *orc.token_logprobs(z[1:], torch.tensor([4]), 0, 0.7)["logprobs"], "logprobs")
    orc.check(loss[1:], *orc.distill_topk(z[1:], q[1:], at[1:], 0.7), "loss")
    orc.check(g, *orc.distill_topk_backward(z, q, at, one, 0.7), "dlogits")
