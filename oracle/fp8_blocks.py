"""e4m3 with one scale for each block of 128, the ragged product of such operands, the weights' gradient from 8-bit activations and swiglu with its
gradient, in 64 bits on the CPU from the definitions; and how far a 32-bit evaluation may be from them.

Values and scales of the quantiser have no bound: they are numbers that have to be met.  The other bounds count roundings: u = 2^-24 is half a step of fp32, a matrix
instruction is taken to lose up to a whole step (2 u) for each number that it adds, exp2 and the reciprocal are good to two units u, and the results end with half a
step of their type.

The matrix instructions on e4m3 do not keep 24 bits of every product: they add eight products of consecutive k at a time, and cut off what of a product
lies below 2^-13 of the power of two in the largest of the eight (found with one large product and one small one at every distance and place: 2^-13 of it comes through whole from any of the seven other
places, 2^-14 not at all, 1.75 * 2^-13 as 2^-13, with either sign; beyond the eight, and against the running sum, 23 places do).  So eight products are off by less than 7 * 2^-13 of their largest one, next to
what fp32 sums lose.  fp32 results are taken from sums without that.
"""
from __future__ import annotations

import torch

from .rows import U, d64, half_step

BLOCK = 128


def _spread(s, block_rows, R, C):
    return s.repeat_interleave(block_rows, -2)[..., :R, :].repeat_interleave(BLOCK, -1)[..., :C]


def e4m3(v):
    """The nearest e4m3 of numbers within 448, ties to even; NaN for what is not finite."""
    step = torch.ldexp(torch.ones_like(v), (torch.frexp(v.abs().clamp_min(2.0**-6)).exponent - 4).to(torch.int32))
    return torch.where(v.isfinite(), torch.round(v / step) * step, torch.full_like(v, float("nan")))


def downcast(x, block_rows=1):
    """`(values, scales)` of `[..., R, C]`, values as the numbers they stand for before scaling."""
    x = d64(x)
    R, C = x.shape[-2:]
    scales = torch.ones((*x.shape[:-2], -(-R // block_rows), -(-C // BLOCK)), dtype=torch.float64)
    for r in range(scales.shape[-2]):
        for c in range(scales.shape[-1]):
            part = x[..., r * block_rows:(r + 1) * block_rows, c * BLOCK:(c + 1) * BLOCK]
            top = torch.where(part.isfinite(), part.abs(), torch.zeros_like(part)).amax((-2, -1))
            s = torch.full_like(top, 2.0**-126)
            while (top > 448 * s).any():
                s = torch.where(top > 448 * s, s * 2, s)
            scales[..., r, c] = torch.where(top == 0, torch.ones_like(s), s)
    return e4m3(x / _spread(scales, block_rows, R, C)), scales


def upcast(values, scales, block_rows=1):
    return values.detach().cpu().to(torch.float32).to(torch.float64) * _spread(d64(scales), block_rows, *values.shape[-2:])


def _act(a, off, alpha, limit):
    """swiglu of interleaved columns that are off by up to `off`, and how far the result may be."""
    gate, lin, eg, el = a[..., 0::2], a[..., 1::2], off[..., 0::2], off[..., 1::2]
    if limit is not None:
        gate, lin = gate.clamp(max=limit), lin.clamp(-limit, limit)
    s = gate * torch.sigmoid(alpha * gate)
    h = s * lin + s
    slope = 1.1 + abs(alpha)  # of s, whose derivative is sigma (1 + alpha gate (1 - sigma))
    return h, slope * eg * (lin.abs() + 1) + s.abs() * el + slope * eg * el + ((alpha * gate).abs() * 2 + 10) * U * ((s * lin).abs() + s.abs())


def slices(sizes, rows):
    out, at = [], 0
    for n in [rows] if sizes is None else sizes:
        out.append((at, at + n))
        at += n
    return out


def _largest_of_eight(x):
    return torch.nn.functional.pad(x.abs(), (0, -x.shape[1] % 8)).unflatten(1, (-1, 8)).amax(2)


def product(a, a_scale, w, w_scale, sizes=None, bias=None, gather=None, scatter=None, gammas=None, swiglu=None, out_dtype=torch.bfloat16):
    """`(y, bound, written)`: w [E, K, N]; `written` says which rows of y anything is written to; swiglu = (alpha, limit)."""
    x = upcast(a, a_scale)
    x = x if gather is None else x[gather.cpu().long()]
    wd = upcast(w, w_scale, BLOCK)
    M, K, N = x.shape[0], x.shape[1], wd.shape[2]
    y, off, done = torch.zeros((M, N), dtype=torch.float64), torch.zeros((M, N), dtype=torch.float64), torch.zeros(M, dtype=torch.bool)
    depth = min(K, BLOCK) + -(-K // BLOCK) + 6
    for e, (lo, hi) in enumerate(slices(sizes, M)):
        y[lo:hi] = x[lo:hi] @ wd[e]
        off[lo:hi] = 2 * U * depth * (x[lo:hi].abs() @ wd[e].abs())
        if out_dtype != torch.float32:  # (of eight products none is larger than the product of the largest factors)
            off[lo:hi] += 7 * 2.0**-13 * (_largest_of_eight(x[lo:hi]) @ _largest_of_eight(wd[e].T).T)
        if bias is not None:
            y[lo:hi] += d64(bias)[e]
            off[lo:hi] += U * (y[lo:hi].abs() + d64(bias)[e].abs())
        done[lo:hi] = True
    if swiglu is not None:
        y, off = _act(y, off, *swiglu)
    if gammas is not None:
        g = d64(gammas)[:, None]
        y, off = y * g, off * g.abs() + U * (y * g).abs()
    if scatter is not None:
        at = scatter.cpu().long()
        out, o, d = torch.zeros((at.shape[0], y.shape[1]), dtype=torch.float64), torch.zeros((at.shape[0], y.shape[1]), dtype=torch.float64), torch.zeros(at.shape[0], dtype=torch.bool)
        for r in range(min(M, at.shape[0])):
            if done[r] and at[r] >= 0:
                out[at[r]], o[at[r]], d[at[r]] = y[r], off[r], True
        y, off, done = out, o, d
    return y, off + half_step(out_dtype, y), done


def weight_gradient(x, x_scale, dy, sizes=None, out_dtype=torch.float32):
    """`(dw, bound)` [E, K, N]; the scaled values are rounded to dy's type first."""
    top = torch.finfo(dy.dtype).max
    xd = upcast(x, x_scale).to(torch.float32).clamp(-top, top).to(dy.dtype).to(torch.float64)
    g = d64(dy)
    dw, off = [], []
    for lo, hi in slices(sizes, xd.shape[0]):
        dw.append(xd[lo:hi].T @ g[lo:hi])
        off.append(2 * U * min(hi - lo + 2, 4096) * (xd[lo:hi].T.abs() @ g[lo:hi].abs()))
    dw, off = torch.stack(dw), torch.stack(off)
    return dw, off + half_step(out_dtype, dw)


def swiglu(a, alpha, limit=None):
    x = d64(a)
    h, off = _act(x, torch.zeros_like(x), alpha, limit)
    return h, off + half_step(a.dtype, h)


def swiglu_backward(dh, values, scales, alpha, limit=None):
    a, d = upcast(values, scales), d64(dh)
    gate, lin = a[:, 0::2], a[:, 1::2]
    if limit is not None:
        gate, lin = gate.clamp(max=limit), lin.clamp(-limit, limit)
    t = torch.sigmoid(alpha * gate)
    u = alpha * gate
    dg, dl = d * (lin + 1) * t * (1 + u * (1 - t)), d * gate * t
    rel = (u.abs() * 2 + 12) * U
    # (1 - sigma is off by sigma's own error, u times that by as much more)
    og = (d * (lin.abs() + 1)).abs() * t * (rel * (1 + u.abs() * (1 - t)) + u.abs() * t * rel + 4 * U * (1 + u.abs()))
    ol = dl.abs() * rel
    if limit is not None:
        over_g, over_l = a[:, 0::2] > limit, a[:, 1::2].abs() > limit
        dg, dl = torch.where(over_g, torch.zeros_like(dg), dg), torch.where(over_l, torch.zeros_like(dl), dl)
    da, off = torch.stack((dg, dl), -1).flatten(-2), torch.stack((og, ol), -1).flatten(-2)
    return da, off + half_step(dh.dtype, da)
