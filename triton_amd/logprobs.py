"""Log probabilities of given tokens over a whole vocabulary, with entropy and top alternatives (no counterpart in the reference's
operator library; `topk` is the selection over a router's few columns).

One pass over the logits gives a row's softmax statistics and the candidates of its largest entries; nothing of the logits'
size is written.  The backward pass reads the logits once more and writes their gradient.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Optional

import torch

from . import _native as nt
from ._autograd import check_capture, check_forward_mode, once

DTYPES = (torch.float32, torch.bfloat16, torch.float16)
MAX_ROWS, MAX_COLUMNS = 2**31 - 1, 2**30
MAX_TOP = 128
MAX_TOP_COLUMNS = 524288


@dataclass
class TokenLogprobs:
    logprobs: torch.Tensor  # [T] fp32: log probability of the row's token
    entropy: torch.Tensor  # [T] fp32
    top_logprobs: Optional[torch.Tensor] = None  # [T, k] fp32: the k largest, larger first
    top_indx: Optional[torch.Tensor] = None  # [T, k] int32: their tokens, equal logits by index


def check_logits(logits, temperature):
    """The logits as the kernels take them: unit stride along the vocabulary."""
    if logits.ndim != 2 or logits.shape[1] == 0:
        raise ValueError(f"logits must be [rows, vocabulary] (got shape {tuple(logits.shape)})")
    if logits.dtype not in DTYPES:
        raise NotImplementedError(f"logits must be fp32, bf16 or fp16 (got {logits.dtype})")
    if logits.shape[0] > MAX_ROWS or logits.shape[1] > MAX_COLUMNS:
        raise NotImplementedError(f"logits have at most {MAX_ROWS} rows and {MAX_COLUMNS} columns (got shape {tuple(logits.shape)})")
    if not (temperature > 0 and math.isfinite(temperature)):
        raise ValueError(f"temperature must be positive and finite (got {temperature})")
    return logits if logits.stride(1) == 1 else logits.contiguous()


def check_index(indx, shape, logits, name):
    if indx.shape != shape or indx.device != logits.device:
        raise ValueError(f"{name} must be {tuple(shape)} on {logits.device} (got {tuple(indx.shape)} on {indx.device})")
    if indx.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name} must be int32 or int64 (got {indx.dtype})")


def logits_desc(logits, temperature):
    d = nt.VocabDesc()
    d.logits, d.logits_dtype, d.logits_stride_m = logits.data_ptr(), nt.TORCH_TO_TK[logits.dtype], logits.stride(0)
    d.n_rows, d.vocab = logits.shape
    d.temperature = temperature
    return d


def workspace(logits, k):
    """Scratch of this call's own, or None where it needs none: a captured graph's pool then owns it."""
    n = nt.lib().tk_vocab_workspace_bytes(logits.shape[0], logits.shape[1], k)
    return torch.empty(n, dtype=torch.uint8, device=logits.device) if n else None


def check_saved(t, shape, logits, name):
    if t.shape != shape or t.dtype != torch.float32 or t.device != logits.device or not t.is_contiguous():
        raise ValueError(f"{name} must be the contiguous fp32 {list(shape)} of the forward pass")


def row_gradient(g, logits, name):
    """A gradient of a row's output: its pointer, element stride and the tensor to keep alive."""
    if g is None:
        return None, 0, None
    T = logits.shape[0]
    if g.shape != (T, ) or g.device != logits.device:
        raise ValueError(f"{name} must be [{T}] on {logits.device} (got {tuple(g.shape)} on {g.device})")
    g = g if g.dtype == torch.float32 else g.float()
    return g.data_ptr(), g.stride(0) if T > 1 else 0, g


def _forward(logits, tokens, k, temperature, with_stats):
    check_index(tokens, logits.shape[:1], logits, "tokens")
    T, V = logits.shape
    if not 0 <= k <= V:
        raise ValueError(f"k must lie in [0, {V}] (got {k})")
    if k > MAX_TOP or (k and V > MAX_TOP_COLUMNS):
        raise NotImplementedError(f"token_logprobs gives at most {MAX_TOP} alternatives, of at most {MAX_TOP_COLUMNS} columns (got {k} of {V})")
    dev = logits.device
    nt.require_gpu(logits, "logits")
    tokens = tokens if tokens.is_contiguous() else tokens.contiguous()
    logprobs, entropy = (torch.empty((T, ), dtype=torch.float32, device=dev) for _ in range(2))  # (not of one buffer: a caller may change one of them in place)
    stats = torch.empty((2, T), dtype=torch.float32, device=dev) if with_stats else None
    top_logprobs = torch.empty((T, k), dtype=torch.float32, device=dev) if k else None
    top_indx = torch.empty((T, k), dtype=torch.int32, device=dev) if k else None
    ws = workspace(logits, k)
    d = logits_desc(logits, temperature)
    d.tokens, d.tokens_i64 = tokens.data_ptr(), int(tokens.dtype == torch.int64)
    d.logprobs, d.entropy, d.stats = logprobs.data_ptr(), entropy.data_ptr(), nt.ptr(stats)
    d.k, d.top_logprobs, d.top_indx, d.workspace = k, nt.ptr(top_logprobs), nt.ptr(top_indx), nt.ptr(ws)
    nt.submit(nt.lib().tk_token_logprobs, d, dev)
    return logprobs, entropy, top_logprobs, top_indx, stats


def token_logprobs_backward(logits, tokens, entropy, stats, d_logprobs, d_entropy, temperature: float = 1.0):
    """The gradient of `logits` for those of the log probabilities and entropies (`[T]`, either may be None)."""
    logits = check_logits(logits, temperature)
    check_index(tokens, logits.shape[:1], logits, "tokens")
    T = logits.shape[0]
    check_saved(entropy, (T, ), logits, "entropy")
    check_saved(stats, (2, T), logits, "stats")
    d_lp, lp_stride, keep_lp = row_gradient(d_logprobs, logits, "d_logprobs")
    d_h, h_stride, keep_h = row_gradient(d_entropy, logits, "d_entropy")
    nt.require_gpu(logits, "logits")
    tokens = tokens if tokens.is_contiguous() else tokens.contiguous()
    d_logits = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    d = logits_desc(logits, temperature)
    d.tokens, d.tokens_i64 = tokens.data_ptr(), int(tokens.dtype == torch.int64)
    d.entropy, d.stats = entropy.data_ptr(), stats.data_ptr()
    d.d_logprobs, d.d_logprobs_stride, d.d_entropy, d.d_entropy_stride = d_lp, lp_stride, d_h, h_stride
    d.d_logits, d.d_logits_stride_m = d_logits.data_ptr(), d_logits.stride(0)
    nt.submit(nt.lib().tk_token_logprobs_backward, d, logits.device)
    del keep_lp, keep_h
    return d_logits


class _TokenLogprobs(torch.autograd.Function):
    """The log probabilities and entropies carry the gradient; the alternatives are returned as non-differentiable tensors."""

    @staticmethod
    def forward(ctx, logits, tokens, k, temperature):
        logprobs, entropy, top_logprobs, top_indx, stats = _forward(logits, tokens, k, temperature, True)
        ctx.save_for_backward(logits, tokens, entropy, stats)
        ctx.temperature = temperature
        ctx.set_materialize_grads(False)
        if k:
            ctx.mark_non_differentiable(top_logprobs, top_indx)
        return logprobs, entropy, top_logprobs, top_indx

    @staticmethod
    @once
    def backward(ctx, d_logprobs, d_entropy, *_unused):
        logits, tokens, entropy, stats = ctx.saved_tensors
        if d_logprobs is None and d_entropy is None:
            return None, None, None, None
        return token_logprobs_backward(logits, tokens, entropy.contiguous(), stats.contiguous(), d_logprobs, d_entropy, ctx.temperature), None, None, None


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, k: int = 0, temperature: float = 1.0) -> TokenLogprobs:
    """Log probability of `tokens [T]` (int32 or int64) under `softmax(logits / temperature)` of `logits [T, V]`, the entropy of each
    row, and its `k` most likely tokens (ties to the lower index).

    Logits are fp32, bf16 or fp16, results fp32; rows may have any stride.  Logits of -inf have probability zero; a row of nothing else
    has log probabilities of -inf, entropy 0 and no gradient.  A row with a NaN or +inf gives NaN, and -1 as its alternatives.  A token
    outside `[0, V)` (padding) has the log probability 0 and no gradient through it.  The log probabilities and the entropies are
    differentiable once in the logits, the alternatives are not."""
    host = nt.host()
    r = host.token_logprobs(logits, tokens, k, temperature) if host is not None else None
    if r is not None:
        return TokenLogprobs(*r)
    check_forward_mode("token_logprobs", logits)
    if logits.requires_grad and torch.is_grad_enabled():
        check_capture(logits)
        logits = check_logits(logits, temperature)
        return TokenLogprobs(*_TokenLogprobs.apply(logits, tokens, k, temperature))
    return TokenLogprobs(*_forward(check_logits(logits, temperature), tokens, k, temperature, False)[:4])


from .torch_twins import token_logprobs_torch  # noqa: E402,F401  (plain twin; never called by `token_logprobs`)
