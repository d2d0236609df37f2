"""Experts in 8 bits: e4m3 values with one fp32 scale for each block of 128 (no counterpart in the reference's operator library).

    downcast_to_fp8_blocks, upcast_from_fp8_blocks   rows in blocks of 128 (activations), matrices in blocks of 128 x 128 (weights)
    matmul_fp8_blocks                                the ragged product of such operands, with the options of `matmul` that serving uses
    linear_fp8_blocks                                the experts' linear layer for training: products in 8 bits, and the input kept in 8 bits for the gradient of the weights
    swiglu_fp8_checkpoint                            the activation between two of them, its input kept in 8 bits for the backward pass

A matrix stands for `values * scales`.  Scales made here are powers of two: the value is then a number of four significant bits, so the products of the
backward pass take it in 16 bits as it is.  Scales that a checkpoint brings may have any size.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch

from . import _native as nt
from ._autograd import check_capture, check_forward_mode, once
from .tensor import RaggedTensorMetadata
from .tensor_details.ragged_tensor import _BLOCK_SIZES

FP8_BLOCK = 128
DTYPES = (torch.float32, torch.bfloat16, torch.float16)
_E4M3 = torch.float8_e4m3fn
_MOST = 0x7FFFFF00  # of rows, K and N
_SCHEDULE = 64  # row blocks of the kernel that goes by the schedule


def _blocks(n: int) -> int:
    return -(-n // FP8_BLOCK)


def _type(t, what, types=DTYPES):
    if t.dtype not in types:
        raise NotImplementedError(f"{what} must be {', '.join(str(d)[6:] for d in types)} (got {t.dtype})")


def _no_gradient(who, **tensors):
    if torch.is_grad_enabled():
        for name, t in tensors.items():
            if t is not None and t.requires_grad:
                raise NotImplementedError(f"{who} has no gradient for {name}: pass it detached (linear_fp8_blocks and swiglu_fp8_checkpoint have gradients)")
    check_forward_mode(who, *tensors.values())


def _matrices(t: torch.Tensor, what: str):
    """`t [..., R, C]` as `[B, R, C]` with unit stride along C, copied if there is no such view."""
    if t.ndim < 1:
        raise ValueError(f"{what} must have a row (got a scalar)")
    t = t[None] if t.ndim == 1 else t
    t = t.reshape(math.prod(t.shape[:-2]), *t.shape[-2:]) if t.ndim != 3 else t
    return t if t.stride(2) == 1 or t.shape[2] <= 1 else t.contiguous()


def _pitch(n: int) -> int:
    return (n + 15) // 16 * 16


def _new_values(shape, device):
    """e4m3 `[..., R, C]` whose rows begin at sixteen-byte boundaries."""
    return torch.empty((*shape[:-1], _pitch(shape[-1])), dtype=_E4M3, device=device)[..., :shape[-1]]


def _downcast(x3, block_rows, values, scales, values_t=None):
    B, R, C = x3.shape
    with nt.on_device(x3.device):
        nt.check(
            nt.lib().tk_fp8_block_downcast(x3.data_ptr(), nt.TORCH_TO_TK[x3.dtype], B, R, C, x3.stride(0), x3.stride(1), block_rows, values.data_ptr(),
                                           values.stride(0), values.stride(1), nt.ptr(values_t), values_t.stride(0) if values_t is not None else 0,
                                           values_t.stride(1) if values_t is not None else 0, scales.data_ptr(), scales.stride(0), scales.stride(1),
                                           scales.stride(2), nt.stream_ptr(x3.device)))


def _check_block_rows(block_rows):
    if block_rows not in (1, FP8_BLOCK):
        raise NotImplementedError(f"blocks have 1 or {FP8_BLOCK} rows (got {block_rows})")


def downcast_to_fp8_blocks(x: torch.Tensor, block_rows: int = 1):
    """`(values, scales)` of `x [..., R, C]` (fp32, bf16 or fp16) in blocks of `block_rows` x 128 elements: `values` e4m3 of x's shape, its rows at
    sixteen-byte boundaries; `scales [..., ceil(R / block_rows), ceil(C / 128)]` fp32.  `block_rows` is 1 (activations) or 128 (weights).

    A block's scale is the smallest power of two that leaves its largest finite magnitude at most 448 (1 for a block of zeros, at least
    2^-126); elements are rounded to the nearest e4m3, ties to even.  Infinities and NaN become NaN and do not count for the scale."""
    host = nt.host()
    r = host.fp8_downcast(x, block_rows) if host is not None else None
    if r is not None:
        return r
    _check_block_rows(block_rows)
    _type(x, "x")
    _no_gradient("downcast_to_fp8_blocks", x=x)
    x3 = _matrices(x, "x")
    nt.require_gpu(x, "x")
    values = _new_values(x3.shape, x.device)
    scales = torch.empty((x3.shape[0], -(-x3.shape[1] // block_rows), _blocks(x3.shape[2])), dtype=torch.float32, device=x.device)
    _downcast(x3, block_rows, values, scales)
    if x.ndim == 1:
        return values[0, 0], scales[0, 0]
    if x.ndim == 3:
        return values, scales
    return values.unflatten(0, x.shape[:-2]) if x.ndim > 3 else values[0], scales.view(*x.shape[:-2], *scales.shape[1:])


def upcast_from_fp8_blocks(values: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.bfloat16, block_rows: int = 1) -> torch.Tensor:
    """`values * scales` in fp32, rounded to `dtype` (fp32, bf16 or fp16): two roundings where scales are no powers of two and `dtype` has 16 bits.  The arguments as
    `downcast_to_fp8_blocks` returns them, scales of any size."""
    host = nt.host()
    r = host.fp8_upcast(values, scales, dtype, block_rows) if host is not None else None
    if r is not None:
        return r
    _check_block_rows(block_rows)
    _type(values, "values", (_E4M3, ))
    if dtype not in DTYPES:
        raise NotImplementedError(f"the result is float32, bfloat16 or float16 (got {dtype})")
    if values.ndim < 1:
        raise ValueError("values must have a row (got a scalar)")
    lead = values.shape[:-1]
    want = (*lead[:-1], -(-lead[-1] // block_rows), _blocks(values.shape[-1])) if lead else (_blocks(values.shape[-1]), )
    if tuple(scales.shape) != want or scales.dtype != torch.float32 or scales.device != values.device:
        raise ValueError(f"scales must be fp32 {want} on {values.device} (got {scales.dtype} {tuple(scales.shape)} on {scales.device})")
    _no_gradient("upcast_from_fp8_blocks", values=values, scales=scales)
    nt.require_gpu(values, "values")
    v3 = _matrices(values, "values")
    s3 = scales.reshape(v3.shape[0], *((1, ) if not lead else ()), *scales.shape[-2:])
    out = torch.empty(values.shape, dtype=dtype, device=values.device)
    with nt.on_device(values.device):
        nt.check(
            nt.lib().tk_fp8_block_upcast(v3.data_ptr(), *v3.shape, v3.stride(0), v3.stride(1), block_rows, s3.data_ptr(), *s3.stride(), out.data_ptr(),
                                         nt.TORCH_TO_TK[dtype], v3.shape[1] * v3.shape[2], v3.shape[2], nt.stream_ptr(values.device)))
    return out


# ---- the product -----------------------------------------------------------------------------------------------------------

def _operand_rows(a, a_scale, what="a"):
    """`a [rows, K]` with K contiguous and its scales, checked."""
    _type(a, what, (_E4M3, ))
    if a.ndim != 2:
        raise ValueError(f"{what} must be [rows, K] (got {tuple(a.shape)})")
    want = (a.shape[0], _blocks(a.shape[1]))
    if tuple(a_scale.shape) != want or a_scale.dtype != torch.float32 or a_scale.device != a.device:
        raise ValueError(f"{what}_scale must be fp32 {want} on {a.device} (got {a_scale.dtype} {tuple(a_scale.shape)} on {a_scale.device})")
    return a if a.stride(1) == 1 or a.shape[1] <= 1 else a.contiguous()


def _index(t, what, device, length=None):
    if t.dtype != torch.int32 or t.ndim != 1 or t.device != device or (length is not None and t.shape[0] != length):
        raise ValueError(f"{what} must be int32 [{'rows' if length is None else length}] on {device} (got {t.dtype} {tuple(t.shape)} on {t.device})")
    return t.contiguous()


def _check_metadata(md, n_slices, device):
    if md.n_slices != n_slices:
        raise ValueError(f"{n_slices} weight slices for {md.n_slices} ragged slices")
    if md.slice_sizes.device != device:
        raise ValueError(f"a_ragged_metadata must live on {device} (got {md.slice_sizes.device})")


def _fit(**sizes):
    for name, n in sizes.items():
        if n > _MOST:
            raise NotImplementedError(f"sizes up to {_MOST} (got {name}={n})")


def _gemm(a, a_scale, w, w_scale, bias, md, gather, scatter, gammas, act, out_dtype, zero_rest=False, pow2=False):
    """One launch; operands as checked by the callers, `w [E, K, N]` with K contiguous.  `zero_rest`: rows behind the slices become zero; `pow2`: all scales are the
    quantiser's."""
    M = a.shape[0] if gather is None else gather.shape[0]
    K, N = w.shape[1], w.shape[2]
    _fit(rows=M, K=K, N=N, scatter=0 if scatter is None else scatter.shape[0])
    swiglu = act is not None
    y = torch.empty((scatter.shape[0] if scatter is not None else M, N // 2 if swiglu else N), dtype=out_dtype, device=a.device)
    if y.numel() == 0 or M == 0 or w.shape[0] == 0:
        return y.zero_() if zero_rest else y
    d = nt.Fp8GemmDesc()
    d.x, d.x_stride_m, d.x_rows = a.data_ptr(), a.stride(0), a.shape[0]
    d.x_scale, d.xs_stride_m, d.xs_stride_k = a_scale.data_ptr(), a_scale.stride(0), a_scale.stride(1)
    d.w, d.w_stride_e, d.w_stride_n = w.data_ptr(), w.stride(0), w.stride(2)
    d.w_scale, d.ws_stride_e, d.ws_stride_k, d.ws_stride_n = w_scale.data_ptr(), *w_scale.stride()
    if bias is not None:
        d.bias, d.bias_dtype, d.bias_stride_e = bias.data_ptr(), nt.TORCH_TO_TK[bias.dtype], bias.stride(0)
    d.gather_indx, d.scatter_indx = nt.ptr(gather), nt.ptr(scatter)
    d.scatter_len = scatter.shape[0] if scatter is not None else 0
    if gammas is not None:
        d.gammas, d.gammas_dtype = gammas.data_ptr(), nt.TORCH_TO_TK[gammas.dtype]
    d.n_slices = w.shape[0]
    if md is not None:
        i = _BLOCK_SIZES.index(_SCHEDULE)
        schedule = md.block_schedule_data
        d.slice_sizes, d.slice_offs = md.slice_sizes.data_ptr(), md.slice_offs.data_ptr()
        d.block_schedule = schedule.data_ptr() + 4 * i * schedule.stride(0)
        d.grid_m = min(RaggedTensorMetadata.n_blocks(md.n_slices, M, _SCHEDULE), schedule.shape[1])
    d.M, d.N, d.K = M, N, K
    d.y, d.y_dtype, d.y_stride_m = y.data_ptr(), nt.TORCH_TO_TK[out_dtype], y.stride(0)
    if swiglu:
        d.activation, d.act_alpha = nt.TK_ACT_SWIGLU, act[0]
        d.act_limit, d.act_has_limit = (act[1], 1) if act[1] is not None else (0.0, 0)
    d.zero_rest, d.pow2_scales = int(zero_rest), int(pow2)
    nt.submit(nt.lib().tk_fp8_block_gemm, d, a.device)
    return y


def _aligned(t, unit):
    """`t [.., lines, length]` with lines at sixteen-byte boundaries (`unit` elements), copied if they are elsewhere."""
    if t.data_ptr() % 16 == 0 and all(s % unit == 0 for s in t.stride()[:-1]):
        return t
    out = torch.empty((*t.shape[:-1], -(-t.shape[-1] // unit) * unit), dtype=t.dtype, device=t.device)[..., :t.shape[-1]]
    return out.copy_(t)


def _activation(fused_activation):
    """`(alpha, limit)` of a fused swiglu, None without one."""
    if fused_activation is None or (fused_activation.specs.fn is None and fused_activation.specs.name == "dflt"):
        return None
    if fused_activation.specs.name != "swiglu" or fused_activation.specs.reduction_n != 2:
        raise NotImplementedError(f"fused activation {fused_activation.specs.name!r} is not supported")
    args = fused_activation.fn_args
    limit = args[1] if len(args) > 1 else None
    return float(args[0]), None if limit is None else float(limit)


def matmul_fp8_blocks(a: torch.Tensor, a_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, bias: Optional[torch.Tensor] = None,
                      a_ragged_metadata: Optional[RaggedTensorMetadata] = None, gather_indx: Optional[torch.Tensor] = None,
                      scatter_indx: Optional[torch.Tensor] = None, gammas: Optional[torch.Tensor] = None, fused_activation=None,
                      out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The ragged product of operands in 8 bits:

        y[dst(r)] = act((a * a_scale)[src(r)] @ (w * w_scale)[e(r)] + bias[e(r)]) * gammas[r]

    `a [rows, K]` e4m3 with `a_scale [rows, ceil(K / 128)]`; `w [E, K, N]` (or `[K, N]`) e4m3 with `w_scale [E, ceil(K / 128), ceil(N / 128)]`, scales fp32
    of any size and any strides (the product of two of them is taken first, and is to be a normal number of fp32).  Weights are contiguous along K, as a checkpoint's `[E, N, K]` transposed; others are copied for the call.  `a_ragged_metadata`, `gather_indx`,
    `scatter_indx`, `gammas` and `fused_activation` (swiglu) as in `matmul`: the rows of the slices in order, src(r) = gather_indx[r], dst(r) =
    scatter_indx[r] (negative: dropped).  `bias [E, N]` and `gammas [rows]` are fp32 or bf16.  Blocks of 128 products are summed by themselves and added, times their scales,
    in fp32; the result is rounded once, to `out_dtype` (bf16, fp16 or fp32).  For results of 16 bits the products are those of the 8-bit matrix instructions, which add eight at a time
    and keep of each what reaches 2^-13 of the largest one (small beside the rounding of typical sums, not of sums that cancel); for fp32 results they are taken from the exact
    16-bit form of the values, at half to a third of the speed for many rows.

    Rows that no slice holds, and rows of the output that no index names, are not written.  No gradients: `linear_fp8_blocks` has them."""
    host = nt.host()
    y = host.fp8_matmul(a, a_scale, w, w_scale, bias, a_ragged_metadata, gather_indx, scatter_indx, gammas, fused_activation, out_dtype) if host is not None else None
    if y is not None:
        return y
    _no_gradient("matmul_fp8_blocks", a=a, w=w, a_scale=a_scale, w_scale=w_scale, bias=bias, gammas=gammas)
    _type(w, "w", (_E4M3, ))
    a = _operand_rows(a, a_scale)
    if w.ndim == 2:
        w, w_scale = w[None], w_scale[None]
    if w.ndim != 3 or w.device != a.device:
        raise ValueError(f"w must be [E, K, N] on {a.device} (got {tuple(w.shape)} on {w.device})")
    E, K, N = w.shape
    if K != a.shape[1]:
        raise ValueError(f"reduction dims differ: a has K={a.shape[1]}, w has K={K}")
    want = (E, _blocks(K), _blocks(N))
    if tuple(w_scale.shape) != want or w_scale.dtype != torch.float32 or w_scale.device != a.device:
        raise ValueError(f"w_scale must be fp32 {want} on {a.device} (got {w_scale.dtype} {tuple(w_scale.shape)} on {w_scale.device})")
    if out_dtype not in DTYPES:
        raise NotImplementedError(f"the output is float32, bfloat16 or float16 (got {out_dtype})")
    act = _activation(fused_activation)
    if act is not None and N % 2:
        raise ValueError(f"swiglu needs an even number of columns (got {N})")
    if gather_indx is not None:
        gather_indx = _index(gather_indx, "gather_indx", a.device)
    M = a.shape[0] if gather_indx is None else gather_indx.shape[0]
    if scatter_indx is not None:
        scatter_indx = _index(scatter_indx, "scatter_indx", a.device)
    if bias is not None:
        bias = bias[None] if bias.ndim == 1 else bias
        if tuple(bias.shape) != (E, N) or bias.device != a.device:
            raise ValueError(f"bias must be [{E}, {N}] on {a.device} (got {tuple(bias.shape)} on {bias.device})")
        _type(bias, "bias", (torch.float32, torch.bfloat16))
        bias = bias if bias.stride(1) == 1 else bias.contiguous()
    if gammas is not None:
        if tuple(gammas.shape) != (M, ) or gammas.device != a.device:
            raise ValueError(f"gammas must be [{M}] on {a.device} (got {tuple(gammas.shape)} on {gammas.device})")
        _type(gammas, "gammas", (torch.float32, torch.bfloat16))
        gammas = gammas.contiguous()
    nt.require_gpu(a, "a")
    md = a_ragged_metadata
    if md is not None and getattr(md, "remapped_from", None) is not None:
        from .matmul import _localise_remapped_metadata
        md = _localise_remapped_metadata(md, E, M)
    if md is not None:
        _check_metadata(md, E, a.device)
    elif E != 1:
        raise NotImplementedError("batched weights need ragged metadata")
    if w.stride(1) != 1 and K > 1:
        w = w.transpose(1, 2).contiguous().transpose(1, 2)
    if M > 256 * E and out_dtype != torch.float32:
        # (the fast kernels take lines at sixteen-byte boundaries; beyond 256 rows an expert a copy of all weights costs less than the kernel for any lines.  fp32 results
        # have no other kernel than that one: us, copied / not: 700 rows, 1000 x 1023 32 / 12; 2000, 2057 x 2048 57 / 44; eight experts, 16384, 2881 x 2880 600 / 566)
        a, w = _aligned(a, 16), _aligned(w.transpose(1, 2), 16).transpose(1, 2)
    return _gemm(a, a_scale, w, w_scale, bias, md, gather_indx, scatter_indx, gammas, act, out_dtype)


# ---- the linear layer for training -----------------------------------------------------------------------------------------

class Fp8Weight(NamedTuple):
    """Weights `[E, K, N]` in 8 bits for both directions of a linear layer: the same values contiguous along K (the output's product) and along N (the
    input's gradient), and the scales `[E, ceil(K / 128), ceil(N / 128)]` of both."""
    values: torch.Tensor
    values_n: torch.Tensor
    scales: torch.Tensor


def quantize_fp8_weight(w: torch.Tensor) -> Fp8Weight:
    """The 8-bit form of `w [E, K, N]` or `[K, N]` (fp32, bf16 or fp16; contiguous along either) that `linear_fp8_blocks` multiplies with, in one pass: for steps that
    use the same weights several times (accumulated gradients)."""
    _type(w, "w")
    if w.ndim not in (2, 3):
        raise ValueError(f"w must be [E, K, N] (got {tuple(w.shape)})")
    check_forward_mode("quantize_fp8_weight", w)
    nt.require_gpu(w, "w")
    w = w.detach()
    w3 = w[None] if w.ndim == 2 else w
    turned = w3.stride(1) == 1 and w3.stride(2) != 1  # contiguous along K: the blocks of the transposed matrix are the transposed blocks
    if turned:
        w3 = w3.transpose(1, 2)
    w3 = _matrices(w3, "w")
    E, R, C = w3.shape
    values, other = _new_values((E, R, C), w.device), _new_values((E, C, R), w.device)
    scales = torch.empty((E, _blocks(R), _blocks(C)), dtype=torch.float32, device=w.device)
    _downcast(w3, FP8_BLOCK, values, scales, other)
    if turned:  # values [E, N, K], other [E, K, N]
        return Fp8Weight(values.transpose(1, 2), other, scales.transpose(1, 2))
    return Fp8Weight(other.transpose(1, 2), values, scales)


def weight_gradient_fp8_blocks(x: torch.Tensor, x_scale: torch.Tensor, dy: torch.Tensor, ragged_metadata: Optional[RaggedTensorMetadata] = None,
                               out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """`dw[e] = (x * x_scale)^T dy` over the rows of slice e: `x [T, K]` e4m3 with `x_scale [T, ceil(K / 128)]` as `downcast_to_fp8_blocks` returns them, `dy [T, N]`
    bf16 or fp16; the result `[E, K, N]` (`[K, N]` without metadata) in `out_dtype` (dy's if not given).  fp32 sums; `x * x_scale` is rounded to dy's type first.  Where the
    scales are powers of two that changes nothing in bf16, and in fp16 nothing of what was quantised from fp16 but numbers beyond 65504, which are held to it; of what was
    quantised from bf16 or fp32 it loses in fp16 what lies below 2^-24: pass dy in bf16 there.  A slice without rows has the gradient zero."""
    _no_gradient("weight_gradient_fp8_blocks", x=x, x_scale=x_scale, dy=dy)
    _type(dy, "dy", (torch.bfloat16, torch.float16))
    out_dtype = out_dtype or dy.dtype
    if out_dtype not in DTYPES:
        raise NotImplementedError(f"the gradient is float32, bfloat16 or float16 (got {out_dtype})")
    x = _operand_rows(x, x_scale, "x")
    if dy.ndim != 2 or dy.shape[0] != x.shape[0] or dy.device != x.device:
        raise ValueError(f"dy must be [{x.shape[0]}, N] on {x.device} (got {tuple(dy.shape)} on {dy.device})")
    nt.require_gpu(x, "x")
    md = ragged_metadata
    if md is not None:
        if getattr(md, "remapped_from", None) is not None:
            raise NotImplementedError("weight gradients need the metadata of all slices")
        _check_metadata(md, md.n_slices, x.device)
    return _weight_gradient(x, x_scale, dy, md, out_dtype, False)


def _weight_gradient(x, x_scale, dy, md, out_dtype, pow2):
    """One launch; operands as checked by the callers.  `pow2`: the scales are the quantiser's."""
    dy = dy if dy.stride(1) == 1 or dy.shape[1] <= 1 else dy.contiguous()
    # (a copy costs less than the kernel for lines that begin anywhere, or overlap: a row expanded)
    x, dy = (_aligned(t if t.stride(0) >= t.shape[1] else t.contiguous(), unit) for t, unit in ((x, 16), (dy, 8)))
    (T, K), N, E = x.shape, dy.shape[1], 1 if md is None else md.n_slices
    _fit(rows=T, K=K, N=N)
    y = torch.empty((E, K, N), dtype=out_dtype, device=x.device)
    d = nt.Fp8WgradDesc()
    d.x, d.x_stride_t, d.x_scale, d.xs_stride_t, d.xs_stride_k = x.data_ptr(), x.stride(0), x_scale.data_ptr(), *x_scale.stride()
    d.dy, d.dy_dtype, d.dy_stride_t = dy.data_ptr(), nt.TORCH_TO_TK[dy.dtype], dy.stride(0)
    if md is not None:
        d.slice_sizes, d.slice_offs = md.slice_sizes.data_ptr(), md.slice_offs.data_ptr()
    d.n_slices, d.T, d.K, d.N = E, T, K, N
    d.y, d.y_dtype, d.y_stride_e, d.y_stride_k = y.data_ptr(), nt.TORCH_TO_TK[out_dtype], y.stride(0), y.stride(1)
    d.pow2_scales = int(pow2)
    n_ws = nt.lib().tk_fp8_block_wgrad_workspace_bytes(T, K, N, E)
    ws = torch.empty(n_ws, dtype=torch.uint8, device=x.device) if n_ws else None
    d.workspace = nt.ptr(ws)
    nt.submit(nt.lib().tk_fp8_block_wgrad, d, x.device)
    return y if md is not None else y[0]


def _quantize_rows(x):
    x = x if x.stride(1) == 1 or x.shape[1] <= 1 else x.contiguous()
    values = _new_values(x.shape, x.device)
    scales = torch.empty((x.shape[0], _blocks(x.shape[1])), dtype=torch.float32, device=x.device)
    _downcast(x[None], 1, values[None], scales[None])
    return values, scales


def _check_saved(t, like, what):
    """A hook on saved tensors may have put another tensor in the place of one of `like` = (shape, dtype, device)."""
    if (tuple(t.shape), t.dtype, t.device) != like:
        raise ValueError(f"{what} must be {like[1]} {like[0]} on {like[2]}, as the forward pass saved it (got {t.dtype} {tuple(t.shape)} on {t.device})")
    return t


def _like(t):
    return tuple(t.shape), t.dtype, t.device


class _LinearFp8(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, w, values, values_n, scales, md, pow2):
        x8, xs = _quantize_rows(x)
        y = _gemm(x8, xs, values, scales, None, md, None, None, None, None, x.dtype, True, pow2)
        slices = () if md is None else (md.slice_sizes, md.slice_offs, md.block_schedule_data)  # (saved, so that a change of them before the backward pass is an error)
        ctx.save_for_backward(x8, xs, values_n, scales, *slices)
        ctx.md, ctx.pow2, ctx.w_shape, ctx.w_dtype = md, pow2, w.shape, w.dtype
        ctx.like = [_like(t) for t in (x8, xs, values_n, scales, *slices)]
        return y

    @staticmethod
    @once
    def backward(ctx, dy):
        names = ("x8", "x_scale", "w8", "w_scale", "slice_sizes", "slice_offs", "block_schedule_data")
        own = all(r.unpack_hook is None for r in ctx._raw_saved_tensors)  # (what a hook gives back for the scales need not be the quantiser's)
        x8, xs, values_n, scales, *slices = (_check_saved(*v) for v in zip(ctx.saved_tensors, ctx.like, names))
        md = None
        if slices:
            sizes, offs, schedule = (t.contiguous() for t in slices)
            md = RaggedTensorMetadata(sizes, offs, ctx.md.block_offs_data, schedule)
        x8 = x8 if x8.stride(1) == 1 or x8.shape[1] <= 1 else x8.contiguous()
        values_n = values_n if values_n.stride(2) == 1 or values_n.shape[2] <= 1 else values_n.contiguous()
        dx = dw = None
        if ctx.needs_input_grad[0]:
            d8, ds = _quantize_rows(dy)
            dx = _gemm(d8, ds, values_n.transpose(1, 2), scales.transpose(1, 2), None, md, None, None, None, None, dy.dtype, True, ctx.pow2 and own)
        if ctx.needs_input_grad[1]:
            dw = _weight_gradient(x8, xs, dy, md, ctx.w_dtype, own).view(ctx.w_shape)
        return dx, dw, None, None, None, None, None


def linear_fp8_blocks(x: torch.Tensor, w: torch.Tensor, a_ragged_metadata: Optional[RaggedTensorMetadata] = None, quantized: Optional[Fp8Weight] = None) -> torch.Tensor:
    """The experts' linear layer with products in 8 bits, differentiable once in `x` and `w`.

        y  = x8 @ w8          x8, w8: x in blocks of 128 elements, w in blocks of 128 x 128 (`downcast_to_fp8_blocks`)
        dx = dy8 @ w8^T
        dw = x8^T @ dy        in 16 bits, from the 8-bit copy of x: the only thing that is kept of it

    `x [rows, K]` is bf16 or fp16, the rows of the slices of `a_ragged_metadata` in order; `w [E, K, N]` (`[K, N]` without metadata) fp32, bf16 or fp16,
    contiguous along either of its last dimensions.  y and dx have x's type, dw has w's.  `quantized` = `quantize_fp8_weight(w)`, for steps that use the same weights several
    times, or a `Fp8Weight` of other scales (a checkpoint's); without it the call quantises w.  Handed in, it takes the slower host path and products without exponents: it pays where
    the conversion of the weights costs more than some 100 us (eight experts, 2880 x 5760: 512 rows 310 -> 191 us a step, 16384 rows 1470 -> 1388; five, 520 x 776 78 -> 182).  Rows behind the last slice give and receive zeros."""
    host = nt.host() if quantized is None else None
    y = host.fp8_linear(x, w, a_ragged_metadata) if host is not None else None
    if y is not None:
        return y
    _type(x, "x", (torch.bfloat16, torch.float16))
    _type(w, "w")
    if x.ndim != 2 or w.ndim not in (2, 3) or w.device != x.device or w.shape[-2] != x.shape[1]:
        raise ValueError(f"x [rows, K] and w [E, K, N] do not go together (got {tuple(x.shape)} on {x.device} and {tuple(w.shape)} on {w.device})")
    check_forward_mode("linear_fp8_blocks", x, w)
    nt.require_gpu(x, "x")
    md, E = a_ragged_metadata, 1 if w.ndim == 2 else w.shape[0]
    if md is not None:
        if getattr(md, "remapped_from", None) is not None:
            raise NotImplementedError("linear_fp8_blocks needs the metadata of all slices")
        _check_metadata(md, E, x.device)
    elif E != 1:
        raise NotImplementedError("batched weights need ragged metadata")
    if quantized is not None:
        K, N = w.shape[-2:]
        for name, t, shape, dtype in (("values", quantized.values, (E, K, N), _E4M3), ("values_n", quantized.values_n, (E, K, N), _E4M3),
                                      ("scales", quantized.scales, (E, _blocks(K), _blocks(N)), torch.float32)):
            if tuple(t.shape) != shape or t.dtype != dtype or t.device != x.device:
                raise ValueError(f"quantized.{name} must be {dtype} {shape} on {x.device} (got {t.dtype} {tuple(t.shape)} on {t.device})")
        if (quantized.values.stride(1) != 1 and K > 1) or (quantized.values_n.stride(2) != 1 and N > 1):
            raise ValueError("quantized must be as quantize_fp8_weight returns it (values contiguous along K, values_n along N)")
    pow2 = quantized is None  # (nobody vouches for the scales of weights that are handed in)
    if torch.is_grad_enabled() and (x.requires_grad or w.requires_grad):
        check_capture(x, w)
        q = quantize_fp8_weight(w) if quantized is None else quantized
        return _LinearFp8.apply(x, w, *q, md, pow2)
    q = quantize_fp8_weight(w) if quantized is None else quantized
    x8, xs = _quantize_rows(x.detach())
    return _gemm(x8, xs, q.values, q.scales, None, md, None, None, None, None, x.dtype, True, pow2)


# ---- swiglu ----------------------------------------------------------------------------------------------------------------

def _swiglu_rows(a, what):
    if a.ndim < 1 or a.shape[-1] % 2:
        raise ValueError(f"{what} must have an even number of columns (got shape {tuple(a.shape)})")
    a2 = a.reshape(math.prod(a.shape[:-1]), a.shape[-1])
    return a2 if a2.stride(1) == 1 or a2.shape[1] <= 1 else a2.contiguous()


def _limit(limit):
    if limit is not None and not float(limit) >= 0.0:
        raise ValueError(f"limit must not be negative (got {limit})")
    return (0.0, 0) if limit is None else (float(limit), 1)


def swiglu_fp8_forward(a: torch.Tensor, alpha: float, limit: Optional[float] = None, *, keep: bool = True):
    """`(h, values, scales)`: swiglu of `a [..., 2n]`, and a's 8-bit copy as `downcast_to_fp8_blocks` makes it, from one pass over a (rows flattened; None unless
    `keep`)."""
    _type(a, "a")
    _no_gradient("swiglu_fp8_forward", a=a)
    nt.require_gpu(a, "a")
    a2 = _swiglu_rows(a, "a")
    M, C = a2.shape
    h = torch.empty((*a.shape[:-1], C // 2), dtype=a.dtype, device=a.device)
    values = _new_values((M, C), a.device) if keep else None
    scales = torch.empty((M, _blocks(C)), dtype=torch.float32, device=a.device) if keep else None
    bound, has = _limit(limit)
    with nt.on_device(a.device):
        nt.check(
            nt.lib().tk_swiglu_fp8(a2.data_ptr(), nt.TORCH_TO_TK[a.dtype], M, C // 2, a2.stride(0), h.data_ptr(), C // 2, nt.ptr(values),
                                   values.stride(0) if keep else 0, nt.ptr(scales), scales.stride(0) if keep else 0, 1, float(alpha), bound, has,
                                   nt.stream_ptr(a.device)))
    return h, values, scales


def swiglu_fp8_backward(dh: torch.Tensor, values: torch.Tensor, scales: torch.Tensor, alpha: float, limit: Optional[float] = None) -> torch.Tensor:
    """The gradient of a for that of `swiglu_fp8_forward`'s output, at the 8-bit copy of a: `[..., 2n]` in dh's type."""
    _type(dh, "dh")
    _no_gradient("swiglu_fp8_backward", dh=dh, values=values, scales=scales)
    values = _operand_rows(values, scales, "values")
    M, C = values.shape
    if dh.ndim < 1 or C % 2 or dh.shape[-1] * 2 != C or dh.numel() * 2 != M * C or dh.device != values.device:
        raise ValueError(f"dh must be [{M}, {C // 2}] on {values.device} (got {tuple(dh.shape)} on {dh.device})")
    nt.require_gpu(dh, "dh")
    d2 = dh.reshape(M, C // 2)
    d2 = d2 if d2.stride(1) == 1 or C <= 2 else d2.contiguous()
    da = torch.empty((*dh.shape[:-1], C), dtype=dh.dtype, device=dh.device)
    bound, has = _limit(limit)
    with nt.on_device(dh.device):
        nt.check(
            nt.lib().tk_swiglu_fp8_backward(d2.data_ptr(), nt.TORCH_TO_TK[dh.dtype], M, C // 2, d2.stride(0), values.data_ptr(), values.stride(0), scales.data_ptr(),
                                            *scales.stride(), da.data_ptr(), C, float(alpha), bound, has, nt.stream_ptr(dh.device)))
    return da


class _SwigluFp8(torch.autograd.Function):

    @staticmethod
    def forward(ctx, a, alpha, limit):
        h, values, scales = swiglu_fp8_forward(a, alpha, limit)
        ctx.save_for_backward(values, scales)
        ctx.alpha, ctx.limit, ctx.like = alpha, limit, [_like(values), _like(scales)]
        return h

    @staticmethod
    @once
    def backward(ctx, dh):
        values, scales = (_check_saved(*v) for v in zip(ctx.saved_tensors, ctx.like, ("values", "scales")))
        return swiglu_fp8_backward(dh, values, scales, ctx.alpha, ctx.limit), None, None


def swiglu_fp8_checkpoint(a: torch.Tensor, alpha: float, limit: Optional[float] = None) -> torch.Tensor:
    """swiglu of `a [..., 2n]` with interleaved (gate, linear) columns -> `[..., n]` in a's type (fp32, bf16 or fp16); for the backward pass a is kept in 8 bits
    (`downcast_to_fp8_blocks` of its rows), and the gradient is that at the kept values.  The same formula as `swiglu`, but NaN stays NaN also in front of a limit.  An element
    beyond the limit has the gradient zero.  Differentiable once; where no gradient is asked for nothing is kept."""
    host = nt.host()
    h = host.fp8_swiglu(a, alpha, limit) if host is not None else None
    if h is not None:
        return h
    check_forward_mode("swiglu_fp8_checkpoint", a)
    if torch.is_grad_enabled() and a.requires_grad:
        check_capture(a)
        _limit(limit)
        return _SwigluFp8.apply(a, float(alpha), limit)
    return swiglu_fp8_forward(a, alpha, limit, keep=False)[0]


from .torch_twins import (downcast_to_fp8_blocks_torch, matmul_fp8_blocks_torch, swiglu_fp8_backward_torch,  # noqa: E402,F401  (plain twins; never
                          upcast_from_fp8_blocks_torch, weight_gradient_fp8_blocks_torch)  # called by the operators)
