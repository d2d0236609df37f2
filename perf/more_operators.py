"""Experts in 8 bits, as their users call them: values of e4m3 with one fp32 scale for each block of 128, the ragged product of
such operands, the linear layer that is trained on them and keeps its input in 8 bits for the backward pass, and the swiglu
between two of them that does the same.

A case is a dict of plain values.  `listed()` names the fixed ones, `draw(rng)` gives more of the same ranges,
`prepare(case, seed)` makes what a program holds before the call, `run(state)` is one pass, through the package's
operators where `own` is true and in plain torch operations where it is not, `exact(case, seed)` the same results in
64 bits, and `work(case)` the bytes and operations that a pass cannot do without.

Kinds:

  store    an activation written as an 8-bit checkpoint (one scale for 128 elements of a row) and read back
  product  the product of 8-bit rows with the 8-bit weights of their experts (one scale for 128 x 128 elements), with swiglu behind it or
           a bias; `gathered`: rows are fetched by index
  linear   a training step of the experts' linear layer: the output, the gradient of the input, and that of the weights from the
           input's 8-bit checkpoint
  swiglu   a training step of the activation: its output, and the gradient of its input, taken at the input's 8-bit checkpoint

A block's scale is the smallest power of two that leaves its largest element at most 448 (1 for a block of zeros), and an element is
rounded to the nearest e4m3, ties to even.  The weights that `product` is given have scales of any size, as checkpoints hold them.
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda:0"
FLOATS = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BLOCK = 128
ALPHA, LIMIT = 1.702, 7.0


def _store(name, rows, cols, dtype):
    return dict(name=name, kind="store", rows=rows, cols=cols, dtype=dtype)


def _product(name, rows, experts, k, n, dtype, swiglu=False, gathered=False):
    return dict(name=name, kind="product", rows=rows, experts=experts, k=k, n=n, dtype=dtype, swiglu=swiglu, gathered=gathered)


def _linear(name, rows, experts, k, n, dtype, weights):
    return dict(name=name, kind="linear", rows=rows, experts=experts, k=k, n=n, dtype=dtype, weights=weights)


def _swiglu(name, rows, cols, dtype, limited):
    return dict(name=name, kind="swiglu", rows=rows, cols=cols, dtype=dtype, limited=limited)


def listed():
    return [
        # the activations of a decode batch, quantised for the product that follows: a latency
        _store("store_t16", 16, 2880, "bf16"),
        # the activations of a training step's layer
        _store("store_t16384", 16384, 4096, "bf16"),
        # one token of an interactive decode loop through a dense projection
        _product("product_t1", 1, 1, 4096, 4096, "bf16"),
        # a decode batch: a few rows for each of many experts, both projections and their activation
        _product("product_t128_e32", 128, 32, 2880, 5760, "bf16", swiglu=True, gathered=True),
        # a short prefill with odd sizes, a few experts
        _product("product_odd", 700, 3, 1000, 1023, "fp16"),
        # a prefill batch through the experts' down projection
        _product("product_t4096_e32", 4096, 32, 2880, 2880, "bf16"),
        # a long prefill through a few large experts
        _product("product_t16384_e8", 16384, 8, 4096, 14336, "bf16", swiglu=True, gathered=True),
        # the gradient step of a small layer with odd sizes, weights held in 32 bits
        _linear("linear_odd", 333, 5, 520, 776, "fp16", "fp32"),
        # a training step's micro-batch through the experts' first projection
        _linear("linear_train", 16384, 8, 2880, 5760, "bf16", "bf16"),
        # a few rows through the activation: a latency
        _swiglu("swiglu_t16", 16, 5760, "bf16", True),
        # odd sizes, everything in 32 bits
        _swiglu("swiglu_odd", 1111, 1030, "fp32", False),
        # the activations of a training step
        _swiglu("swiglu_train", 16384, 11520, "bf16", True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi):
    """A length: any, even, or whole blocks."""
    n = _log_int(rng, lo, hi)
    unit = rng.choice([1, 16, 64, 128])
    return max(lo, n // unit * unit)


def draw(rng):
    kind = rng.choice(["store", "product", "product", "linear", "linear", "swiglu"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind == "store":
        cols = _size(rng, 64, 16384)
        return dict(kind=kind, rows=_log_int(rng, 1, min(65536, 64 * 1024 * 1024 // cols)), cols=cols, dtype=dtype)
    if kind == "swiglu":
        cols = _size(rng, 64, 16384) // 2 * 2
        return dict(kind=kind, rows=_log_int(rng, 1, min(65536, 128 * 1024 * 1024 // cols)), cols=cols, dtype=dtype, limited=rng.random() < 0.5)
    k, n = _size(rng, 128, 4096), _size(rng, 128, 8192) // 2 * 2
    experts = rng.choice([1, 2, 5, 8, 32])
    rows = _log_int(rng, 1, 16384)
    if kind == "product":
        return dict(kind=kind, rows=rows, experts=experts, k=k, n=n, dtype=rng.choice(["bf16", "bf16", "fp16"]), swiglu=rng.random() < 0.5,
                    gathered=rng.random() < 0.5)
    experts = min(experts, 8)
    # (a step is three products)
    rows = min(rows, max(1, 16384 * 2880 * 5760 // (k * n)))
    return dict(kind=kind, rows=rows, experts=experts, k=k, n=n, dtype=rng.choice(["bf16", "bf16", "fp16"]), weights=rng.choice(["bf16", "fp32"]))


def _randn(g, shape, scale=1.0, dtype=torch.float32):
    return torch.randn(shape, generator=g, device=DEVICE).mul_(scale).to(dtype)


def _activation(g, rows, cols, dtype, scale=1.0):
    """Rows as a trained model's: levels of their own, and a few columns that stand out."""
    x = torch.randn((rows, cols), generator=g, device=DEVICE)
    x *= torch.rand((rows, 1), generator=g, device=DEVICE) * 1.5 + 0.25
    x[:, torch.randint(cols, (max(1, cols // 200), ), generator=g, device=DEVICE)] *= 12
    return x.mul_(scale).to(dtype)


def _slices(g, rows, experts):
    """How many rows each expert has, as a router deals them: uneven, now and then none."""
    if experts == 1:
        return [rows]
    weights = torch.rand((experts, ), generator=g, device=DEVICE).square() + 0.02
    owner = torch.multinomial(weights, rows, replacement=True, generator=g)
    return torch.bincount(owner, minlength=experts).tolist()


def _metadata(sizes):
    """The row offsets that the router of this package hands to the products behind it."""
    if not own or len(sizes) == 1:
        return None
    from triton_kernels.tensor import make_ragged_tensor_metadata
    return make_ragged_tensor_metadata(torch.tensor(sizes, dtype=torch.int32, device=DEVICE), sum(sizes))


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype, rows = FLOATS[case["dtype"]], case["rows"]
    state = dict(kind=case["kind"], dtype=dtype)
    if case["kind"] == "store":
        state["x"] = _activation(g, rows, case["cols"], dtype)
        return state
    if case["kind"] == "swiglu":
        state["a"] = _activation(g, rows, case["cols"], dtype, 1.5).requires_grad_()
        state["dh"] = _randn(g, (rows, case["cols"] // 2), 1.0, dtype)
        state["limit"] = LIMIT if case["limited"] else None
        return state
    E, K, N = case["experts"], case["k"], case["n"]
    sizes = _slices(g, rows, E)
    state["sizes"], state["metadata"] = sizes, _metadata(sizes)
    if case["kind"] == "product":
        # one token for every two rows where rows are fetched by index: each token goes to two experts
        tokens = max(1, rows // 2) if case["gathered"] else rows
        state["gather"] = torch.randint(tokens, (rows, ), generator=g, device=DEVICE, dtype=torch.int32) if case["gathered"] else None
        state["a"], state["a_scale"] = _plain_downcast(_activation(g, tokens, K, torch.bfloat16))
        # the weights as a checkpoint holds them: output by input, scales of any size
        values = torch.empty((E, N, K), dtype=torch.float8_e4m3fn, device=DEVICE)
        scale = torch.empty((E, -(-N // BLOCK), -(-K // BLOCK)), device=DEVICE)
        for e in range(E):
            w = _randn(g, (N, K), 0.03)
            amax = _blocks(w, BLOCK).abs().amax((1, 3))
            scale[e] = amax / 448
            values[e] = _from_blocks((_blocks(w, BLOCK) / scale[e][:, None, :, None]).clamp_(-448, 448), N, K).to(values.dtype)
        state["w"], state["w_scale"] = values.transpose(1, 2), scale.transpose(1, 2)
        state["swiglu"] = case["swiglu"]
        state["bias"] = None if case["swiglu"] else _randn(g, (E, N), 0.1)
        return state
    state["x"] = _activation(g, rows, K, dtype).requires_grad_()
    state["w"] = _randn(g, (E, K, N), 0.03, FLOATS[case["weights"]]).requires_grad_()
    state["dy"] = _activation(g, rows, N, dtype, 0.01)
    return state


# ---- plain forms: 32 bits throughout, rounded once --------------------------------------------------------------------

def _blocks(x, block_rows):
    """[R, C] as [R / block_rows, block_rows, C / 128, 128], filled up with zeros."""
    R, C = x.shape
    r, c = -(-R // block_rows), -(-C // BLOCK)
    full = torch.zeros((r * block_rows, c * BLOCK), dtype=x.dtype, device=x.device) if (r * block_rows, c * BLOCK) != (R, C) else x
    if full is not x:
        full[:R, :C] = x
    return full.view(r, block_rows, c, BLOCK)


def _from_blocks(b, R, C):
    return b.reshape(b.shape[0] * b.shape[1], -1)[:R, :C]


def _plain_downcast(x, block_rows=1):
    b = _blocks(x.float(), block_rows)
    amax = b.abs().amax((1, 3))
    fraction, exponent = torch.frexp(amax)
    exponent = torch.where(fraction <= 0.875, exponent - 9, exponent - 8).clamp_min(-126)
    scale = torch.where(amax == 0, torch.ones_like(amax), torch.ldexp(torch.ones_like(amax), exponent))
    values = _from_blocks(b / scale[:, None, :, None], *x.shape).to(torch.float8_e4m3fn)
    return values, scale


def _plain_upcast(values, scale, block_rows=1):
    return _from_blocks(_blocks(values.float(), block_rows) * scale[:, None, :, None], *values.shape)


def _plain_act(a, limit):
    gate, linear = a[:, 0::2], a[:, 1::2]
    if limit is not None:
        gate, linear = gate.clamp(max=limit), linear.clamp(-limit, limit)
    sigmoid = 1 / (1 + torch.exp(-ALPHA * gate))
    return gate, linear, sigmoid


def _plain_store(s):
    values, scale = _plain_downcast(s["x"])
    return dict(x=_plain_upcast(values, scale).to(s["dtype"]), scale=scale)


def _plain_product(s):
    E, K, N = s["w"].shape
    a = _plain_upcast(s["a"], s["a_scale"])
    if s["gather"] is not None:
        a = a[s["gather"].long()]
    out = torch.empty((a.shape[0], N // 2 if s["swiglu"] else N), dtype=s["dtype"], device=a.device)
    at = 0
    for e, rows in enumerate(s["sizes"]):
        if rows == 0:
            continue
        w = _plain_upcast(s["w"][e].T, s["w_scale"][e].T, BLOCK)
        y = a[at:at + rows] @ w.T
        if s["bias"] is not None:
            y += s["bias"][e]
        if s["swiglu"]:
            gate, linear, sigmoid = _plain_act(y, LIMIT)
            y = gate * sigmoid * (linear + 1)
        out[at:at + rows] = y
        at += rows
    return dict(y=out)


def _plain_linear(s):
    x, w, dy = s["x"].detach(), s["w"].detach(), s["dy"]
    E, K, N = w.shape
    x8 = _plain_upcast(*_plain_downcast(x))
    dy8 = _plain_upcast(*_plain_downcast(dy))
    y = torch.empty((x.shape[0], N), dtype=x.dtype, device=x.device)
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    at = 0
    for e, rows in enumerate(s["sizes"]):
        if rows == 0:
            dw[e] = 0
            continue
        w8 = _plain_upcast(*_plain_downcast(w[e], BLOCK), BLOCK)
        here = slice(at, at + rows)
        y[here] = x8[here] @ w8
        dx[here] = dy8[here] @ w8.T
        dw[e] = x8[here].T @ dy[here].float()
        at += rows
    return dict(y=y, dx=dx, dw=dw)


def _plain_swiglu(s):
    a, dh, limit = s["a"].detach(), s["dh"].float(), s["limit"]
    gate, linear, sigmoid = _plain_act(a.float(), limit)
    h = gate * sigmoid * (linear + 1)
    a8 = _plain_upcast(*_plain_downcast(a))
    gate, linear, sigmoid = _plain_act(a8, limit)
    da = torch.empty_like(a8)
    d_gate = dh * (linear + 1) * sigmoid * (1 + ALPHA * gate * (1 - sigmoid))
    d_linear = dh * gate * sigmoid
    if limit is not None:
        d_gate = torch.where(a8[:, 0::2] <= limit, d_gate, 0.0)
        d_linear = torch.where(a8[:, 1::2].abs() <= limit, d_linear, 0.0)
    da[:, 0::2], da[:, 1::2] = d_gate, d_linear
    return dict(h=h.to(s["dtype"]), da=da.to(s["dtype"]))


# ---- the package's operators ---------------------------------------------------------------------------------------

def _own_store(s):
    from triton_kernels.fp8_blocks import downcast_to_fp8_blocks, upcast_from_fp8_blocks
    values, scale = downcast_to_fp8_blocks(s["x"])
    return dict(x=upcast_from_fp8_blocks(values, scale, s["dtype"]), scale=scale)


def _own_product(s):
    from triton_kernels.fp8_blocks import matmul_fp8_blocks
    from triton_kernels.matmul import FnSpecs, FusedActivation
    from triton_kernels.swiglu import swiglu_fn
    act = FusedActivation(FnSpecs("swiglu", swiglu_fn, ("alpha", "limit"), reduction_n=2), (ALPHA, LIMIT)) if s["swiglu"] else None
    y = matmul_fp8_blocks(s["a"], s["a_scale"], s["w"], s["w_scale"], s["bias"], s["metadata"], gather_indx=s["gather"], fused_activation=act,
                          out_dtype=s["dtype"])
    return dict(y=y)


def _own_linear(s):
    from triton_kernels.fp8_blocks import linear_fp8_blocks
    y = linear_fp8_blocks(s["x"], s["w"], s["metadata"])
    dx, dw = torch.autograd.grad(y, (s["x"], s["w"]), s["dy"])
    return dict(y=y, dx=dx, dw=dw)


def _own_swiglu(s):
    from triton_kernels.fp8_blocks import swiglu_fp8_checkpoint
    h = swiglu_fp8_checkpoint(s["a"], ALPHA, s["limit"])
    da, = torch.autograd.grad(h, s["a"], s["dh"])
    return dict(h=h, da=da)


def run(state):
    if own:
        return {"store": _own_store, "product": _own_product, "linear": _own_linear, "swiglu": _own_swiglu}[state["kind"]](state)
    return {"store": _plain_store, "product": _plain_product, "linear": _plain_linear, "swiglu": _plain_swiglu}[state["kind"]](state)


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------

def _grid(v):
    """The nearest e4m3 of numbers within 448, ties to even: four significant bits, steps of 2^-9 below 2^-6."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0**-6))) - 3)
    return torch.round(v / step) * step


def _stored(x, tall=1):
    """A matrix as its 8-bit form stands for it, and the scales, strip by strip of 128 columns."""
    x = x.detach().double()
    out = torch.empty_like(x)
    scales = []
    for c in range(0, x.shape[1], 128):
        part = x[:, c:c + 128]
        if tall == 1:
            top = part.abs().max(dim=1, keepdim=True).values
        else:
            top = torch.cat([p.abs().max().expand(p.shape[0], 1) for p in part.split(tall)])
        s = torch.exp2(torch.ceil(torch.log2(top / 448)).clamp_min(-126))
        s = torch.where(top > 0, s, torch.ones_like(s))
        out[:, c:c + 128] = _grid(part / s) * s
        scales.append(s)
    return out, torch.cat(scales, dim=1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "store":
        x, scale = _stored(s["x"])
        return dict(x=x, scale=scale)
    if case["kind"] == "swiglu":
        def act(a):
            gate, lin = a.unflatten(1, (-1, 2)).unbind(2)
            if s["limit"] is not None:
                gate, lin = torch.clamp(gate, max=s["limit"]), torch.clamp(lin, min=-s["limit"], max=s["limit"])
            return gate * torch.sigmoid(ALPHA * gate) * (lin + 1)
        kept = _stored(s["a"])[0].requires_grad_()
        da, = torch.autograd.grad(act(kept), kept, s["dh"].double())
        return dict(h=act(s["a"].detach().double()), da=da)
    if case["kind"] == "product":
        K, N = case["k"], case["n"]
        a = s["a"].double() * s["a_scale"].double().repeat_interleave(128, 1)[:, :K]
        if s["gather"] is not None:
            a = a.index_select(0, s["gather"].to(torch.int64))
        parts = []
        for e, rows in enumerate(a.split(s["sizes"])):
            w = s["w"][e].double() * s["w_scale"][e].double().repeat_interleave(128, 0)[:K].repeat_interleave(128, 1)[:, :N]
            y = rows @ w
            if s["bias"] is not None:
                y = y + s["bias"][e].double()
            if s["swiglu"]:
                gate, lin = y.unflatten(1, (-1, 2)).unbind(2)
                gate, lin = torch.clamp(gate, max=LIMIT), torch.clamp(lin, min=-LIMIT, max=LIMIT)
                y = gate * torch.sigmoid(ALPHA * gate) * (lin + 1)
            parts.append(y)
        return dict(y=torch.cat(parts))
    x, dy = _stored(s["x"])[0], s["dy"].double()
    dy8 = _stored(s["dy"])[0]
    y, dx, dw = [], [], []
    for e, (x_e, dy_e, dy8_e) in enumerate(zip(x.split(s["sizes"]), dy.split(s["sizes"]), dy8.split(s["sizes"]))):
        w = _stored(s["w"][e], 128)[0]
        y.append(x_e @ w)
        dx.append(dy8_e @ w.mT)
        dw.append(x_e.mT @ dy_e)
    return dict(y=torch.cat(y), dx=torch.cat(dx), dw=torch.stack(dw))


def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    es = size[case["dtype"]]
    if case["kind"] == "store":  # read, written in 8 bits with its scales, both read, written again, and the scales are a result
        n, groups = case["rows"] * case["cols"], case["rows"] * -(-case["cols"] // BLOCK)
        return dict(bytes=n * (2 * es + 2) + 8 * groups, flops=4 * n)
    if case["kind"] == "swiglu":  # the input read, its 8 bits written and read, its gradient written; the output and its gradient
        n, groups = case["rows"] * case["cols"], case["rows"] * -(-case["cols"] // BLOCK)
        return dict(bytes=n * (2 * es + 2) + 8 * groups + n * es, flops=20 * n)
    R, E, K, N = case["rows"], case["experts"], case["k"], case["n"]
    used = min(R, E)  # experts that have rows: at least one, and no more than this
    if case["kind"] == "product":
        tokens = max(1, R // 2) if case["gathered"] else R
        out = R * (N // 2 if case["swiglu"] else N) * es
        return dict(bytes=tokens * K + used * K * N + out + 4 * (tokens * -(-K // BLOCK) + used * -(-K // BLOCK) * -(-N // BLOCK)), flops=2 * R * K * N)
    ws = size[case["weights"]]  # the gradient of every expert's weights is written, the weights of those with rows are read
    return dict(bytes=R * (2 * K + 2 * N) * es + used * K * N * ws + E * K * N * ws, flops=6 * R * K * N)
