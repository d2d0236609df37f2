"""Distillation from a teacher that is known by its largest logits of each row (no counterpart in the reference's operator library).

The teacher's entries are what `token_logprobs(teacher_logits, ..., k)` returns as `top_logprobs` and `top_indx`: log probabilities
serve as logits, since the softmax over a row's entries is the same.  The loss reads the student's logits once, its backward pass
once more.
"""
from __future__ import annotations

import torch

from . import _native as nt
from ._autograd import check_capture, check_forward_mode, once
from .logprobs import DTYPES, check_index, check_logits, check_saved, logits_desc, row_gradient, workspace

MAX_TEACHER = 1024


def _desc(logits, teacher_logits, teacher_indx, temperature):
    T = logits.shape[0]
    if teacher_logits.ndim != 2 or teacher_logits.shape[0] != T or teacher_logits.device != logits.device:
        raise ValueError(f"teacher_logits must be [{T}, entries] on {logits.device} (got {tuple(teacher_logits.shape)} on {teacher_logits.device})")
    if teacher_logits.dtype not in DTYPES:
        raise NotImplementedError(f"teacher_logits must be fp32, bf16 or fp16 (got {teacher_logits.dtype})")
    check_index(teacher_indx, teacher_logits.shape, logits, "teacher_indx")
    if teacher_logits.shape[1] > MAX_TEACHER:
        raise NotImplementedError(f"distill_topk takes at most {MAX_TEACHER} teacher entries a row (got {teacher_logits.shape[1]})")
    nt.require_gpu(logits, "logits")
    teacher_logits = teacher_logits if teacher_logits.stride(1) == 1 else teacher_logits.contiguous()
    teacher_indx = teacher_indx if teacher_indx.stride(1) == 1 else teacher_indx.contiguous()
    d = logits_desc(logits, temperature)
    d.teacher_logits, d.teacher_dtype, d.teacher_stride_m = teacher_logits.data_ptr(), nt.TORCH_TO_TK[teacher_logits.dtype], teacher_logits.stride(0)
    d.teacher_indx, d.teacher_indx_i64, d.teacher_indx_stride_m = teacher_indx.data_ptr(), int(teacher_indx.dtype == torch.int64), teacher_indx.stride(0)
    d.n_teacher = teacher_logits.shape[1]
    return d, (teacher_logits, teacher_indx)


def _forward(logits, teacher_logits, teacher_indx, temperature, with_stats):
    d, keep = _desc(logits, teacher_logits, teacher_indx, temperature)
    T, dev = logits.shape[0], logits.device
    loss = torch.empty((T, ), dtype=torch.float32, device=dev)
    stats = torch.empty((4, T), dtype=torch.float32, device=dev) if with_stats else None
    ws = workspace(logits, 0)
    d.loss, d.workspace = loss.data_ptr(), nt.ptr(ws)
    if with_stats:
        d.stats, d.teacher_stats = stats.data_ptr(), stats.data_ptr() + 8 * T
    nt.submit(nt.lib().tk_distill_topk, d, dev)
    del keep
    return loss, stats


def distill_topk_backward(logits, teacher_logits, teacher_indx, stats, d_loss, temperature: float = 1.0):
    """The gradient of `logits` for that of the losses (`[T]`) and the forward pass' statistics."""
    logits = check_logits(logits, temperature)
    T = logits.shape[0]
    check_saved(stats, (4, T), logits, "stats")
    d_l, stride, keep_g = row_gradient(d_loss, logits, "d_loss")
    d, keep = _desc(logits, teacher_logits, teacher_indx, temperature)
    d_logits = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    d.stats, d.teacher_stats = stats.data_ptr(), stats.data_ptr() + 8 * T
    d.d_loss, d.d_loss_stride = d_l, stride
    d.d_logits, d.d_logits_stride_m = d_logits.data_ptr(), d_logits.stride(0)
    nt.submit(nt.lib().tk_distill_topk_backward, d, logits.device)
    del keep, keep_g
    return d_logits


class _DistillTopK(torch.autograd.Function):

    @staticmethod
    def forward(ctx, logits, teacher_logits, teacher_indx, temperature):
        loss, stats = _forward(logits, teacher_logits, teacher_indx, temperature, True)
        ctx.save_for_backward(logits, teacher_logits, teacher_indx, stats)
        ctx.temperature = temperature
        return loss

    @staticmethod
    @once
    def backward(ctx, d_loss):
        logits, teacher_logits, teacher_indx, stats = ctx.saved_tensors
        return distill_topk_backward(logits, teacher_logits, teacher_indx, stats.contiguous(), d_loss, ctx.temperature), None, None, None


def distill_topk(logits: torch.Tensor, teacher_logits: torch.Tensor, teacher_indx: torch.Tensor, temperature: float = 1.0) -> torch.Tensor:
    """Kullback-Leibler divergence of each row's student from its teacher, `[T]` fp32:

        a = softmax(teacher_logits / temperature) over the row's entries
        loss = sum_j a_j (ln a_j - ln softmax(logits / temperature)[teacher_indx_j])

    `logits [T, V]` are the student's (fp32, bf16 or fp16), `teacher_logits [T, K]` the teacher's at `teacher_indx [T, K]` (int32 or
    int64; K up to 1024).  An entry whose index lies outside `[0, V)` or whose logit is -inf carries no weight; a row without any
    other has the loss 0 and no gradient (padding, fewer alternatives than K).  A student that gives one of the others no
    probability, or one whose logarithm is beyond fp32 (a mask of fp32's lowest value at a temperature below one), has the loss +inf; one with a
    NaN or +inf, or a teacher with one, NaN.  Differentiable once in `logits`."""
    host = nt.host()
    loss = host.distill_topk(logits, teacher_logits, teacher_indx, temperature) if host is not None else None
    if loss is not None:
        return loss
    check_forward_mode("distill_topk", logits, teacher_logits)
    if teacher_logits.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError("distill_topk has no gradient for the teacher: pass its logits detached")
    if logits.requires_grad and torch.is_grad_enabled():
        check_capture(logits)
        return _DistillTopK.apply(check_logits(logits, temperature), teacher_logits, teacher_indx, temperature)
    return _forward(check_logits(logits, temperature), teacher_logits, teacher_indx, temperature, False)[0]


from .torch_twins import distill_topk_torch  # noqa: E402,F401  (plain twin; never called by `distill_topk`)
