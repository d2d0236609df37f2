"""The row operators' twins and workspaces where there is little to compute: no teacher entries, no rows, no alternatives, one column."""
import pytest
import torch

from oracle import rows as orc
from triton_kernels.distill import distill_topk_torch
from triton_kernels.layer_norm import layer_norm_torch
from triton_kernels.logprobs import token_logprobs_torch


@pytest.mark.parametrize("T", [0, 1, 5])
@pytest.mark.parametrize("V", [1, 9])
@pytest.mark.parametrize("K", [0, 1, 4])
def test_distillation_from_few_entries(T, V, K):
    g = torch.Generator().manual_seed(0)
    z, q, at = torch.randn((T, V), generator=g), torch.randn((T, K), generator=g), torch.randint(-1, V, (T, K), generator=g)
    loss = distill_topk_torch(z, q, at, 0.8)
    assert loss.shape == (T, ) and loss.dtype == torch.float32
    if K == 0:
        assert not loss.any()
    if T and K:
        orc.check(loss, *orc.distill_topk(z, q, at, 0.8), "loss")


@pytest.mark.parametrize("T", [0, 1, 5])
@pytest.mark.parametrize("V", [1, 9])
def test_other_twins(T, V):
    z, tokens = torch.randn((T, V), generator=torch.Generator().manual_seed(1)), torch.zeros(T, dtype=torch.int64)
    for k in (0, 1):
        r = token_logprobs_torch(z, tokens, k)
        assert r.logprobs.shape == r.entropy.shape == (T, )
        assert (r.top_indx is None) == (k == 0) and (k == 0 or r.top_indx.shape == r.top_logprobs.shape == (T, k))
    assert layer_norm_torch(z).shape == (T, V)


def test_no_rows_need_no_workspace():
    from triton_amd import _native as nt
    lib = nt.lib()
    for M, C in ((0, 8), (0, 20000), (5, 0), (-1, 8)):
        assert lib.tk_layer_norm_backward_workspace_bytes(M, C) == 0
    assert lib.tk_layer_norm_backward_workspace_bytes(3, 100) == 2 * 3 * 100 * 4
    for T, V, k in ((0, 50000, 20), (-1, 50000, 0), (4, 0, 0), (2000, 50000, 20)):
        assert lib.tk_vocab_workspace_bytes(T, V, k) == 0
    assert lib.tk_vocab_workspace_bytes(1, 50000, 20) > 0
