"""Row operators around the experts, as their users call them: the layer norm in front of a router or a projection, the
log probabilities of given tokens over a whole vocabulary, and the distillation loss against a teacher's top logits.

A case is a dict of plain values.  `listed()` names the fixed ones, `draw(rng)` gives more of the same ranges,
`prepare(case, seed)` makes what a program holds before the call, `run(state)` is one pass, through the package's
operators where `own` is true and in plain torch operations where it is not, `exact(case, seed)` the same results in
64 bits, and `work(case)` the bytes and operations that a pass cannot do without.

Kinds:

  norm      layer norm of the rows of an activation; `train` adds the gradients of the activation, the weight and the bias
  logprobs  log probability of one given token a row, entropy and the `k` most likely tokens; `train` adds the gradient of
            the logits for given gradients of the log probabilities and entropies
  distill   Kullback-Leibler divergence from a teacher known by its `k` largest logits a row; `train` adds the gradient
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda:0"
FLOATS = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-5


def _norm(name, rows, cols, dtype, weights, train):
    return dict(name=name, kind="norm", rows=rows, cols=cols, dtype=dtype, weights=weights, train=train)


def _logits(name, kind, rows, vocab, dtype, k, temperature, masked, train):
    return dict(name=name, kind=kind, rows=rows, vocab=vocab, dtype=dtype, k=k, temperature=temperature, masked=masked, train=train)


def listed():
    return [
        # the norm in front of one layer of a decode batch: a latency
        _norm("norm_t16", 16, 2880, "bf16", "bf16", False),
        # norms of the heads of a projection: many short rows
        _norm("norm_heads", 135168, 128, "fp16", "fp16", False),
        # the activations of a prefill batch
        _norm("norm_t16384", 16384, 4096, "bf16", "bf16", False),
        # a training step's activations, weights held in 32 bits
        _norm("norm_train", 16384, 2880, "bf16", "fp32", True),
        # odd sizes, everything in 32 bits
        _norm("norm_train_odd", 4097, 1023, "fp32", "fp32", True),
        # one sequence of an interactive decode loop that reports alternatives
        _logits("logprobs_t1", "logprobs", 1, 131072, "bf16", 20, 1.0, 0.0, False),
        # a decode batch under a grammar that rules out half of an odd vocabulary
        _logits("logprobs_t61", "logprobs", 61, 50001, "fp16", 8, 0.7, 0.5, False),
        # a teacher's pass over a batch of text, its largest logits kept for distillation
        _logits("logprobs_t4096", "logprobs", 4096, 131072, "bf16", 64, 1.0, 0.0, False),
        # a policy gradient step with an entropy bonus
        _logits("logprobs_train", "logprobs", 2048, 32000, "fp32", 0, 1.0, 0.0, True),
        # a small step of distillation
        _logits("distill_t32", "distill", 32, 32000, "fp32", 16, 2.0, 0.0, True),
        # the loss of an evaluation batch over an odd vocabulary
        _logits("distill_eval", "distill", 1000, 50001, "fp16", 100, 1.0, 0.0, False),
        # a training step's batch
        _logits("distill_train", "distill", 4096, 131072, "bf16", 64, 1.0, 0.0, True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm", "logprobs", "distill"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    train = rng.random() < 0.5
    if kind == "norm":
        cols = _log_int(rng, 64, 8192)
        if rng.random() < 0.5:
            cols = max(64, cols // 64 * 64)
        rows = _log_int(rng, 1, min(135168, 64 * 1024 * 1024 // cols))
        return dict(kind=kind, rows=rows, cols=cols, dtype=dtype, weights=rng.choice([dtype, "fp32"]), train=train)
    vocab = _log_int(rng, 1000, 131072)
    if rng.random() < 0.5:
        vocab = vocab // 64 * 64
    rows = _log_int(rng, 1, min(16384, (256 if dtype == "fp32" else 512) * 1024 * 1024 // vocab))
    k = _log_int(rng, 1, 100)
    if kind == "logprobs" and rng.random() < 0.25:
        k = 0
    return dict(kind=kind, rows=rows, vocab=vocab, dtype=dtype, k=k, temperature=rng.choice([0.7, 1.0, 1.0, 2.0]),
                masked=rng.choice([0.0, 0.0, 0.5]) if kind == "logprobs" else 0.0, train=train)


def _randn(g, shape, scale=1.0, shift=0.0, dtype=torch.float32):
    return torch.randn(shape, generator=g, device=DEVICE).mul_(scale).add_(shift).to(dtype)


def _vocabulary_logits(g, rows, vocab, dtype, masked):
    """Logits as a trained model's: a bulk, a level of each row's own, some tokens that stand out, and tokens ruled out."""
    z = torch.randn((rows, vocab), generator=g, device=DEVICE, dtype=torch.float32).mul_(2.5)
    z += torch.randn((rows, 1), generator=g, device=DEVICE) * 3 - 4
    likely = torch.randint(vocab, (rows, 40), generator=g, device=DEVICE)
    z.scatter_add_(1, likely, torch.rand((rows, 40), generator=g, device=DEVICE) * 12)
    if masked:
        z.masked_fill_(torch.rand((1, vocab), generator=g, device=DEVICE) < masked, -math.inf)
    return z.to(dtype)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype, rows, train = FLOATS[case["dtype"]], case["rows"], case["train"]
    state = dict(kind=case["kind"], train=train)
    if case["kind"] == "norm":
        cols, weights = case["cols"], FLOATS[case["weights"]]
        state["x"] = (_randn(g, (rows, cols), 1.5) + _randn(g, (rows, 1), 0.5)).to(dtype)
        state["weight"] = _randn(g, (cols, ), 0.1, 1.0, weights)
        state["bias"] = _randn(g, (cols, ), 0.1, 0.0, weights)
        if train:
            state["dy"] = _randn(g, (rows, cols), 1.0, 0.0, dtype)
            for name in ("x", "weight", "bias"):
                state[name].requires_grad_()
        return state
    vocab, k = case["vocab"], case["k"]
    z = _vocabulary_logits(g, rows, vocab, dtype, case["masked"])
    state.update(logits=z, k=k, temperature=case["temperature"])
    if case["kind"] == "logprobs":
        # the tokens that a sampler took: the most likely of a handful that the mask, if any, leaves
        some = torch.randint(vocab, (rows, 64), generator=g, device=DEVICE)
        state["tokens"] = some.gather(1, z.gather(1, some).float().argmax(1, keepdim=True)).squeeze(1)
        if train:
            state["d_logprobs"] = _randn(g, (rows, ))
            state["d_entropy"] = _randn(g, (rows, ), 0.01, 0.01)
    else:
        # a teacher that mostly agrees: the student's scores with noise, at the places that it holds likely
        scores = z.float() + torch.randn((rows, vocab), generator=g, device=DEVICE)
        values, indices = scores.topk(k, dim=1)
        state["teacher_logits"], state["teacher_indx"] = values.to(dtype), indices.to(torch.int32)
        if train:
            state["d_loss"] = torch.full((rows, ), 1.0 / rows, device=DEVICE)
    if train:
        state["logits"].requires_grad_()
    return state


# ---- plain forms: 32 bits throughout, rounded once --------------------------------------------------------------------

def _plain_norm(s):
    x, w, b = s["x"].detach(), s["weight"].detach(), s["bias"].detach()
    xf, wf = x.float(), w.float()
    centred = xf - xf.mean(1, keepdim=True)
    r = torch.rsqrt(centred.square().mean(1, keepdim=True) + EPS)
    h = centred * r
    out = dict(y=(h * wf + b.float()).to(x.dtype))
    if s["train"]:
        dy = s["dy"].float()
        g = dy * wf
        out["dx"] = ((g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True)) * r).to(x.dtype)
        out["dweight"], out["dbias"] = (dy * h).sum(0).to(w.dtype), dy.sum(0).to(b.dtype)
    return out


def _plain_softmax(logits, temperature):
    z = logits.float() / temperature
    z = z - z.amax(1, keepdim=True)
    e = z.exp()
    total = e.sum(1, keepdim=True)
    return z, e, total, total.log()


def _plain_logprobs(s):
    logits, k = s["logits"].detach(), s["k"]
    z, e, total, log_total = _plain_softmax(logits, s["temperature"])
    at = s["tokens"][:, None]
    out = dict(logprobs=(z.gather(1, at) - log_total).squeeze(1))
    entropy = log_total - (e * z.clamp_min(-200.0)).sum(1, keepdim=True) / total
    out["entropy"] = entropy.squeeze(1)
    if k:
        # a stable sort leaves equal logits in the order of their indices
        indices = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :k]
        out["top_logprobs"], out["top_indx"] = z.gather(1, indices) - log_total, indices.to(torch.int32)
    if s["train"]:
        p = e / total
        g = -p * s["d_logprobs"][:, None] - s["d_entropy"][:, None] * p * ((z - log_total).clamp_min(-200.0) + entropy)
        g.scatter_add_(1, at, s["d_logprobs"][:, None])
        out["dlogits"] = (g / s["temperature"]).to(logits.dtype)
    return out


def _plain_distill(s):
    logits = s["logits"].detach()
    z, e, total, log_total = _plain_softmax(logits, s["temperature"])
    a_z, a_e, a_total, a_log = _plain_softmax(s["teacher_logits"], s["temperature"])
    a = a_e / a_total
    at = s["teacher_indx"].long()
    out = dict(loss=(a * ((a_z - a_log) - (z.gather(1, at) - log_total))).sum(1))
    if s["train"]:
        g = (e / total).scatter_add_(1, at, -a) * s["d_loss"][:, None]
        out["dlogits"] = (g / s["temperature"]).to(logits.dtype)
    return out


# ---- the package's operators ---------------------------------------------------------------------------------------

def _own_norm(s):
    from triton_kernels.layer_norm import layer_norm
    y = layer_norm(s["x"], s["weight"], s["bias"], eps=EPS)
    if not s["train"]:
        return dict(y=y)
    dx, dweight, dbias = torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["dy"])
    return dict(y=y, dx=dx, dweight=dweight, dbias=dbias)


def _own_logprobs(s):
    from triton_kernels.logprobs import token_logprobs
    r = token_logprobs(s["logits"], s["tokens"], s["k"], temperature=s["temperature"])
    out = dict(logprobs=r.logprobs, entropy=r.entropy)
    if s["k"]:
        out["top_logprobs"], out["top_indx"] = r.top_logprobs, r.top_indx
    if s["train"]:
        out["dlogits"], = torch.autograd.grad((r.logprobs, r.entropy), s["logits"], (s["d_logprobs"], s["d_entropy"]))
    return out


def _own_distill(s):
    from triton_kernels.distill import distill_topk
    loss = distill_topk(s["logits"], s["teacher_logits"], s["teacher_indx"], temperature=s["temperature"])
    out = dict(loss=loss)
    if s["train"]:
        out["dlogits"], = torch.autograd.grad(loss, s["logits"], s["d_loss"])
    return out


def run(state):
    if own:
        return {"norm": _own_norm, "logprobs": _own_logprobs, "distill": _own_distill}[state["kind"]](state)
    return {"norm": _plain_norm, "logprobs": _plain_logprobs, "distill": _plain_distill}[state["kind"]](state)


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "norm":
        x, w, b = (s[n].detach().double() for n in ("x", "weight", "bias"))
        if case["train"]:
            for t in (x, w, b):
                t.requires_grad_()
        var, mean = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
        y = (x - mean) / torch.sqrt(var + EPS) * w + b
        out = dict(y=y.detach())
        if case["train"]:
            out["dx"], out["dweight"], out["dbias"] = torch.autograd.grad(y, (x, w, b), s["dy"].double())
        return out
    t = case["temperature"]
    z = s["logits"].detach().double().div_(t)
    lse = torch.logsumexp(z, dim=1, keepdim=True)
    logp = z.sub_(lse)
    p = torch.exp(logp)
    if case["kind"] == "logprobs":
        at = s["tokens"][:, None]
        surprise = torch.where(p > 0, logp, torch.zeros((), dtype=torch.float64, device=DEVICE))
        entropy = -torch.sum(p * surprise, dim=1)
        out = dict(logprobs=logp.gather(1, at)[:, 0], entropy=entropy)
        if case["k"]:
            order = torch.argsort(-s["logits"].detach().float(), dim=1, stable=True)[:, :case["k"]]
            out["top_logprobs"], out["top_indx"] = logp.gather(1, order), order.to(torch.int32)
        if case["train"]:
            one = torch.zeros_like(p).scatter_(1, at, 1.0)
            g_lp, g_h = s["d_logprobs"].double()[:, None], s["d_entropy"].double()[:, None]
            out["dlogits"] = (g_lp * (one - p) - g_h * p * (surprise + entropy[:, None])) / t
        return out
    at = s["teacher_indx"].long()
    log_a = torch.log_softmax(s["teacher_logits"].double() / t, dim=1)
    a = torch.exp(log_a)
    out = dict(loss=torch.sum(a * (log_a - logp.gather(1, at)), dim=1))
    if case["train"]:
        full = torch.zeros_like(p).scatter_add_(1, at, a)
        out["dlogits"] = s["d_loss"].double()[:, None] * (p - full) / t
    return out


def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    rows, es = case["rows"], size[case["dtype"]]
    if case["kind"] == "norm":
        n, ws = rows * case["cols"], size[case["weights"]]
        weights = 2 * case["cols"] * ws
        if case["train"]:  # x and dy read, y and dx written, the weights read and their gradients written
            return dict(bytes=4 * n * es + 2 * weights, flops=24 * n)
        return dict(bytes=2 * n * es + weights, flops=8 * n)
    n, k = rows * case["vocab"], case["k"]
    if case["kind"] == "logprobs":  # an index in 64 bits read, two floats written, and k pairs of value and index
        small = rows * (8 + 8 + 8 * k)
    else:  # k pairs read, a float written
        small = rows * (4 + k * (es + 4))
    if case["train"]:  # the gradients of the row's outputs read, those of the logits written
        return dict(bytes=2 * n * es + small + rows * 8, flops=14 * n)
    return dict(bytes=n * es + small, flops=8 * n)
