"""Row operators in 64 bits on the CPU: layer norm, token log probabilities, distillation from top logits, and their gradients, written
from the definitions; and how far a 32-bit evaluation may be from them.

The bounds count roundings.  u = 2^-24 is half a step of fp32; a sum of n terms in any order that adds at most `depth` numbers one
after the other is off by at most depth * u times the sum of the terms' magnitudes (first order); exp, log, rsqrt and division are taken as good to
two units u each (the hardware's are good to one unit in the last place).  Each bound ends with the output's own rounding: half a step of its type, and half
the smallest subnormal number.
"""
from __future__ import annotations

import math

import torch

U = 2.0**-24
INF = float("inf")


def half_step(dtype, value):
    f = torch.finfo(dtype)
    return f.eps / 2 * value.abs() + f.smallest_normal * f.eps / 2 + (2.0**-126 if dtype == torch.float32 else 0.0)


def d64(t):
    return None if t is None else t.detach().cpu().to(torch.float64)


# ---- layer norm -------------------------------------------------------------------------------------------

LN_DEPTH = 300  # numbers that a row's sums add one after the other: C / 128 of a thread at the longest rows tested, and the joins


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """`(y, bound)` of rows in 64 bits; the bound is for a result in x's type."""
    xd, w, b = d64(x), d64(weight), d64(bias)
    C = xd.shape[-1]
    depth = min(C, LN_DEPTH) + 2
    mu = xd.mean(-1, keepdim=True)
    var = (xd - mu).square().mean(-1, keepdim=True)
    r = 1 / torch.sqrt(var + eps)
    h = (xd - mu) * r
    y = h if w is None else h * w
    y = y if b is None else y + b
    off_mu = depth * U * xd.abs().mean(-1, keepdim=True)
    off_h = h.abs() * (depth / 2 + 8) * U + r * off_mu + h.abs() * r.square() * off_mu.square()
    aw = 1.0 if w is None else w.abs()
    bound = aw * (off_h + 2 * U * h.abs()) + U * y.abs() + (0 if b is None else U * b.abs())
    return y, bound + half_step(x.dtype, y)


def layer_norm_backward(dy, x, weight=None, eps=1e-5, bias=None):
    """`{name: (value, bound)}` for dx, dweight, dbias in 64 bits (rows flattened)."""
    C = x.shape[-1]
    xd, g0, w = d64(x).reshape(-1, C), d64(dy).reshape(-1, C), d64(weight)
    M = xd.shape[0]
    depth = min(C, LN_DEPTH) + 2
    mu = xd.mean(1, keepdim=True)
    r = 1 / torch.sqrt((xd - mu).square().mean(1, keepdim=True) + eps)
    h = (xd - mu) * r
    off_mu = depth * U * xd.abs().mean(1, keepdim=True)
    off_h = h.abs() * (depth / 2 + 8) * U + r * off_mu + h.abs() * r.square() * off_mu.square()
    g = g0 if w is None else g0 * w
    mean = lambda t: t.mean(1, keepdim=True)  # noqa: E731
    mg, mgh = mean(g), mean(g * h)
    dx = r * (g - mg - h * mgh)
    off_mg = (depth + 2) * U * mean(g.abs())
    off_mgh = (depth + 4) * U * mean((g * h).abs()) + mean(g.abs() * off_h)
    bound = r * (4 * U * (g.abs() + mg.abs() + (h * mgh).abs()) + off_mg + h.abs() * off_mgh + off_h * mgh.abs()) + dx.abs() * (depth / 2 + 8) * U
    out = dict(dx=(dx, bound + half_step(x.dtype, dx)))
    rows = min(M, M / 64 + 160)  # rows that the sums over rows add one after the other
    if w is not None:
        dw = (g0 * h).sum(0)
        out["dweight"] = (dw, (rows + 3) * U * (g0 * h).abs().sum(0) + (g0.abs() * off_h).sum(0) + half_step(weight.dtype, dw))
    if bias is not None:
        db = g0.sum(0)
        out["dbias"] = (db, (rows + 1) * U * g0.abs().sum(0) + half_step(bias.dtype, db))
    return out


# ---- rows over a vocabulary -------------------------------------------------------------------------------


class Rows:
    """A row's softmax in 64 bits: `lp` (log probabilities), `p`, the entropy, which rows are `bad` (a NaN or +inf) or `empty`
    (-inf alone), and bounds of a 32-bit evaluation (`off_lp` per element, `off_h` per row)."""

    def __init__(self, logits, temperature):
        x = d64(logits)
        V = x.shape[1]
        self.bad = (torch.isnan(x) | (x == INF)).any(1)
        self.empty = ~self.bad & (x == -INF).all(1)
        odd = self.bad | self.empty
        x = torch.where(odd[:, None], torch.zeros_like(x), x)
        m = x.amax(1, keepdim=True)
        d = (x - m) / temperature
        s = d.exp().sum(1, keepdim=True)
        self.lp = d - s.log()
        self.p = self.lp.exp()
        live = self.p > 0
        dl = torch.where(live, d.abs(), torch.zeros_like(d))
        self.lpl = torch.where(live, self.lp, torch.zeros_like(d))
        self.entropy = -(self.p * self.lpl).sum(1)
        depth = min(V, V / 256 + 40)
        ed, ed2 = (self.p * dl).sum(1, keepdim=True), (self.p * dl * dl).sum(1, keepdim=True)
        off_s = U * (depth + 3 + 3 * ed)  # relative, and so what ln s is off by beside its own rounding
        ln_s = s.log().abs()
        finite = lambda t: torch.where(torch.isfinite(t), t, torch.zeros_like(t))  # noqa: E731
        self.off_lp = U * (3 * finite(d.abs()) + 3 * ln_s + finite(self.lp.abs()) + 2) + off_s
        self.off_h = (off_s * (1 + ed) + U * (3 * ed2 + (depth + 5) * ed + 4 * ln_s) + 2 * U * self.entropy.abs()[:, None])[:, 0]


def _rows_of(cond, yes, no):
    return torch.where(cond.reshape(-1, *[1] * (no.ndim - 1)), torch.full_like(no, yes), no)


def token_logprobs(logits, tokens, k=0, temperature=1.0):
    """`{name: (value, bound)}`; top_indx has no bound."""
    R, V, tok = Rows(logits, temperature), logits.shape[1], tokens.detach().cpu().long()
    live = (tok >= 0) & (tok < V)
    at = torch.where(live, tok, torch.zeros_like(tok))[:, None]
    lp = _rows_of(R.empty, -INF, _rows_of(R.bad, math.nan, R.lp.gather(1, at)[:, 0]))
    lp = torch.where(live, lp, torch.zeros_like(lp))
    h = _rows_of(R.bad, math.nan, _rows_of(R.empty, 0.0, R.entropy))
    out = dict(logprobs=(lp, R.off_lp.gather(1, at)[:, 0] + half_step(torch.float32, lp)), entropy=(h, R.off_h + half_step(torch.float32, h)))
    if k:
        top = torch.sort(d64(logits).nan_to_num(nan=0.0, posinf=0.0), dim=1, descending=True, stable=True).indices[:, :k]
        tlp = _rows_of(R.empty, -INF, _rows_of(R.bad, math.nan, R.lp.gather(1, top)))
        out["top_logprobs"] = (tlp, R.off_lp.gather(1, top) + half_step(torch.float32, tlp))
        out["top_indx"] = (_rows_of(R.bad, -1, top), None)
    return out


def token_logprobs_backward(logits, tokens, d_logprobs, d_entropy, temperature=1.0):
    R, (T, V), tok = Rows(logits, temperature), logits.shape, tokens.detach().cpu().long()
    live = (tok >= 0) & (tok < V)
    at = torch.where(live, tok, torch.zeros_like(tok))[:, None]
    zero = torch.zeros(T, dtype=torch.float64)
    a = torch.where(live, zero if d_logprobs is None else d64(d_logprobs).expand(T), zero)[:, None]
    b = (zero if d_entropy is None else d64(d_entropy).expand(T))[:, None]
    one = torch.zeros_like(R.p).scatter_(1, at, 1.0)
    H = R.entropy[:, None]
    g = (a * (one - R.p) - b * R.p * (R.lpl + H)) / temperature
    size = a.abs() + b.abs() * (R.lpl.abs() + H)
    bound = (R.p * size * (R.off_lp + 6 * U) + R.p * b.abs() * (R.off_lp + R.off_h[:, None]) + one * 4 * U * a.abs()) / temperature + 3 * U * g.abs()
    still = ((a == 0) & (b == 0))[:, 0] | R.empty
    g = _rows_of(still, 0.0, _rows_of(R.bad, math.nan, g))
    # (32-bit probabilities below the smallest normal number are zero)
    return g, bound + half_step(logits.dtype, g) + 2.0**-126 * size / temperature


class Teacher:

    def __init__(self, logits, teacher_logits, teacher_indx, temperature):
        V, q, i = logits.shape[1], d64(teacher_logits), teacher_indx.detach().cpu().long()
        self.live = (i >= 0) & (i < V) & (q != -INF)
        self.at = torch.where(self.live, i, torch.zeros_like(i))
        self.none = ~self.live.any(1)
        self.bad = (self.live & (torch.isnan(q) | (q == INF))).any(1)
        q = torch.where(self.live, q, torch.full_like(q, -INF))
        q = _rows_of(self.none | self.bad, 0.0, q)
        m = q.amax(1, keepdim=True) if q.shape[1] else q.sum(1, keepdim=True)
        d = (q - m) / temperature
        ls = d.exp().sum(1, keepdim=True).log()
        la = d - ls
        self.a = torch.where(self.live, la.exp(), torch.zeros_like(la))
        self.la = torch.where(self.a > 0, la, torch.zeros_like(la))
        size = torch.where(self.a > 0, d.abs(), torch.zeros_like(d))
        mean = (self.a * size).sum(1, keepdim=True)
        self.off_la = U * (3 * size + 3 * ls.abs() + self.la.abs() + 5 + min(q.shape[1], 40) + 3 * mean)


def distill_topk(logits, teacher_logits, teacher_indx, temperature=1.0):
    """`(loss, bound)`."""
    R, t = Rows(logits, temperature), Teacher(logits, teacher_logits, teacher_indx, temperature)
    lp = _rows_of(R.empty, -INF, R.lp).gather(1, t.at)
    on = t.a > 0
    lp = torch.where(on, lp, torch.zeros_like(lp))
    loss = (t.a * (t.la - lp)).sum(1)
    size = torch.where(torch.isfinite(lp), lp.abs(), torch.zeros_like(lp)) + t.la.abs()
    off = t.a * (size * (t.off_la + 40 * U) + t.off_la + torch.where(on, R.off_lp.gather(1, t.at), torch.zeros_like(lp)))
    loss = _rows_of(t.none, 0.0, _rows_of(R.bad | t.bad, math.nan, loss))
    # (entries of a probability that 32 bits do not hold count nothing)
    return loss, off.sum(1) + half_step(torch.float32, loss) + 2.0**-126 * size.sum(1)


def distill_topk_backward(logits, teacher_logits, teacher_indx, d_loss, temperature=1.0):
    R, t = Rows(logits, temperature), Teacher(logits, teacher_logits, teacher_indx, temperature)
    n = t.a.shape[1]
    c = d64(d_loss).expand(logits.shape[0])[:, None]
    named = torch.zeros_like(R.p).scatter_add_(1, t.at, t.a)
    off_named = torch.zeros_like(R.p).scatter_add_(1, t.at, t.a * (t.off_la + (n + 2) * U))
    g = c * (R.p - named) / temperature
    bound = c.abs() * (R.p * (R.off_lp + 4 * U) + off_named) / temperature + 4 * U * g.abs()
    still = (c == 0)[:, 0] | t.none | R.empty
    g = _rows_of(still, 0.0, _rows_of(R.bad | t.bad, math.nan, g))
    return g, bound + half_step(logits.dtype, g) + 2.0**-126 * (1 + c.abs()) / temperature


def check(got, want, bound, what):
    """Every element within its bound; NaN and infinities in the same places.  A finite value whose bound reaches past the largest
    number F of the result's type may come out as the infinity of its sign: the exact sum of the rounded terms, up to `bound` away, is
    then allowed to exceed F, and rounding such a number gives that infinity."""
    largest = torch.finfo(got.dtype).max
    got = got.detach().cpu().to(torch.float64)
    over = torch.isinf(got) & torch.isfinite(want) & (want.abs() + bound > largest) & (got.sign() == want.sign())
    got = torch.where(over, want, got)
    assert got.shape == want.shape, f"{what}: shape {tuple(got.shape)} for {tuple(want.shape)}"
    assert torch.equal(got.isnan(), want.isnan()), f"{what}: NaN in other places"
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(got), inf) and torch.equal(got[inf], want[inf]), f"{what}: infinities in other places"
    fine = torch.isfinite(want)
    over = ((got - want).abs() - bound.expand_as(want))[fine]
    if over.numel():
        worst = int(over.argmax())
        assert over[worst] <= 0, f"{what}: {got[fine][worst].item()!r} for {want[fine][worst].item()!r}, bound {bound.expand_as(want)[fine][worst].item():.3g}"
