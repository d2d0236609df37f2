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
