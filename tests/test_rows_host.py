"""Row operators without a GPU: the oracle's gradients against differences of its values, the plain twins against the oracle, and what
the operators and their C entries refuse."""
import ctypes

import pytest
import torch

from oracle import rows as orc
from triton_amd import _native as nt

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
INF = float("inf")


def _slope(f, x, v, h=1e-4):
    """Central difference of f along v; its error is h^2 / 6 times the third derivative, and 1e-16 f / h."""
    return (f(x + h * v) - f(x - h * v)) / (2 * h)


def test_oracle_gradients_are_slopes():
    g = torch.Generator().manual_seed(0)
    M, C = 5, 37
    x, dy = torch.randn((M, C), generator=g, dtype=torch.float64), torch.randn((M, C), generator=g, dtype=torch.float64)
    w, b = torch.randn(C, generator=g, dtype=torch.float64), torch.randn(C, generator=g, dtype=torch.float64)
    grads = orc.layer_norm_backward(dy, x, w, 1e-5, b)
    for name, at, f in (("dx", x, lambda t: (orc.layer_norm(t, w, b)[0] * dy).sum()), ("dweight", w, lambda t: (orc.layer_norm(x, t, b)[0] * dy).sum()),
                        ("dbias", b, lambda t: (orc.layer_norm(x, w, t)[0] * dy).sum())):
        v = torch.randn(at.shape, generator=g, dtype=torch.float64)
        assert abs(_slope(f, at, v) - (grads[name][0] * v).sum()) < 1e-5
    T, V, K = 4, 29, 6
    z = torch.randn((T, V), generator=g, dtype=torch.float64) * 2
    tokens = torch.tensor([3, 0, -1, 28])
    a, c = torch.randn(T, generator=g, dtype=torch.float64), torch.randn(T, generator=g, dtype=torch.float64)
    q, at = torch.randn((T, K), generator=g, dtype=torch.float64), torch.randint(V, (T, K), generator=g)
    at[1, 2], at[3, 1] = -1, at[3, 0]
    v = torch.randn(z.shape, generator=g, dtype=torch.float64)

    def scores(t):
        r = orc.token_logprobs(t, tokens, 0, 0.7)
        return (r["logprobs"][0] * a + r["entropy"][0] * c).sum()

    assert abs(_slope(scores, z, v) - (orc.token_logprobs_backward(z, tokens, a, c, 0.7)[0] * v).sum()) < 1e-5
    assert abs(_slope(lambda t: (orc.distill_topk(t, q, at, 1.3)[0] * a).sum(), z, v) - (orc.distill_topk_backward(z, q, at, a, 1.3)[0] * v).sum()) < 1e-5


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_twins_match_the_oracle(dtype):
    from triton_kernels.distill import distill_topk_torch
    from triton_kernels.layer_norm import layer_norm_torch
    from triton_kernels.logprobs import token_logprobs_torch
    g = torch.Generator().manual_seed(1)
    x, w, b = torch.randn((6, 50), generator=g).to(dtype), torch.randn(50, generator=g), torch.randn(50, generator=g)
    for weight, bias in ((w, b), (None, b), (w, None), (None, None)):
        orc.check(layer_norm_torch(x, weight, bias), *orc.layer_norm(x, weight, bias), "y")
    z = (torch.randn((7, 60), generator=g) * 3).to(dtype)
    z[1] = -INF
    z[2, 4] = float("nan")
    z[3, 0] = INF
    z[4, ::2] = -INF
    z[5] = 1.0
    tokens = torch.tensor([5, 5, 5, 0, 3, -1, 60])
    r, want = token_logprobs_torch(z, tokens, 9, 0.8), orc.token_logprobs(z, tokens, 9, 0.8)
    assert torch.equal(r.top_indx.long(), want["top_indx"][0])
    for name in ("logprobs", "entropy", "top_logprobs"):
        orc.check(getattr(r, name), *want[name], name)
    q, at = torch.randn((7, 8), generator=g), torch.randint(60, (7, 8), generator=g)
    at[0, 1:] = -1
    at[5] = 60
    q[6, 2] = -INF
    orc.check(distill_topk_torch(z, q, at, 0.8), *orc.distill_topk(z, q, at, 0.8), "loss")


def test_operators_refuse_what_they_do_not_take():
    from triton_kernels.distill import distill_topk
    from triton_kernels.layer_norm import layer_norm, layer_norm_backward
    from triton_kernels.logprobs import token_logprobs
    x, w = torch.zeros((4, 8)), torch.ones(8)
    with pytest.raises(RuntimeError, match="HIP device"):
        layer_norm(x, w)
    for args, error in (((x[:, :0], ), ValueError), ((x[0, 0], ), ValueError), ((x.double(), ), NotImplementedError), ((x, w.double()), NotImplementedError),
                        ((x, w[:7]), ValueError), ((x, w, w[None]), ValueError), ((x, w, w, -1.0), ValueError), ((x, w, w, float("nan")), ValueError)):
        with pytest.raises(error):
            layer_norm(*args)
    with pytest.raises(ValueError, match="dy must be"):
        layer_norm_backward(x[:3], x, None, None)
    for stats in (torch.zeros(3), torch.zeros(4, dtype=torch.float64), torch.zeros(8)[::2]):
        with pytest.raises(ValueError, match="forward pass"):
            layer_norm_backward(x, x, stats, torch.zeros(4), w)
    with pytest.raises(RuntimeError, match="HIP device"):
        layer_norm_backward(x, x, torch.zeros(4), torch.zeros(4), w)
    z, tokens = torch.zeros((3, 10)), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="HIP device"):
        token_logprobs(z, tokens, 2)
    for args, error in (((z[0], tokens), ValueError), ((z[:, :0], tokens), ValueError), ((z.double(), tokens), NotImplementedError), ((z, tokens[:2]), ValueError),
                        ((z, tokens.short()), ValueError), ((z, tokens, 11), ValueError), ((z, tokens, -1), ValueError), ((z, tokens, 0, 0.0), ValueError),
                        ((z, tokens, 0, -1.0), ValueError), ((z, tokens, 0, INF), ValueError), ((z, tokens, 0, float("nan")), ValueError),
                        ((torch.zeros((3, 200)), tokens, 129), NotImplementedError), ((torch.zeros((3, 524289)), tokens, 1), NotImplementedError)):
        with pytest.raises(error):
            token_logprobs(*args)
    for many in (torch.zeros((1, 1)).expand(2**31, 1), torch.zeros((1, 1)).expand(1, 2**30 + 1), torch.zeros((1, 1)).expand(1, 2**32 + 5)):
        with pytest.raises(NotImplementedError, match="at most"):
            token_logprobs(many, torch.zeros(1, dtype=torch.int64).expand(many.shape[0]))
        with pytest.raises(NotImplementedError, match="at most"):
            distill_topk(many, many[:, :1], torch.zeros((1, 1), dtype=torch.int64).expand(many.shape[0], 1))
    q, at = torch.zeros((3, 4)), torch.zeros((3, 4), dtype=torch.int32)
    with pytest.raises(RuntimeError, match="HIP device"):
        distill_topk(z, q, at)
    for args, error in (((z, q[:2], at[:2]), ValueError), ((z, q, at[:, :3]), ValueError), ((z, q.double(), at), NotImplementedError), ((z, q, at.short()), ValueError),
                        ((z, q[0], at[0]), ValueError), ((z, q, at, 0.0), ValueError),
                        ((z, torch.zeros((3, 1025)), torch.zeros((3, 1025), dtype=torch.int32)), NotImplementedError)):
        with pytest.raises(error):
            distill_topk(*args)


def test_backward_passes_refuse_what_no_forward_pass_gave():
    from triton_kernels.distill import distill_topk_backward
    from triton_kernels.logprobs import token_logprobs_backward
    z, tokens, h, stats, g = torch.zeros((3, 10)), torch.zeros(3, dtype=torch.int64), torch.zeros(3), torch.zeros((2, 3)), torch.ones(3)
    with pytest.raises(RuntimeError, match="HIP device"):
        token_logprobs_backward(z, tokens, h, stats, g, None)
    for args in ((z, tokens, h[:2], stats, g, g), (z, tokens, h.double(), stats, g, g), (z, tokens, h, stats[0], g, g), (z, tokens, h, torch.zeros((3, 2)).t(), g, g),
                 (z, tokens, h, stats, g[:2], g), (z, tokens, h, stats, g, g[:, None]), (z, tokens[:2], h, stats, g, g)):
        with pytest.raises(ValueError):
            token_logprobs_backward(*args)
    q, at, stats = torch.zeros((3, 4)), torch.zeros((3, 4), dtype=torch.int32), torch.zeros((4, 3))
    with pytest.raises(RuntimeError, match="HIP device"):
        distill_topk_backward(z, q, at, stats, g)
    for args in ((z, q, at, stats[:2], g), (z, q, at, stats.double(), g), (z, q, at, stats, g[:1]), (z, q, at, stats, g[None]), (z, q[:2], at[:2], stats, g)):
        with pytest.raises(ValueError):
            distill_topk_backward(*args)


def test_c_entries_refuse_bad_calls_before_any_launch():
    lib, p = nt.lib(), 64  # (an address that no entry reads)
    ln = lambda x=p, dt=nt.TK_BF16, m=4, c=8, w=p, wt=nt.TK_F32, eps=1e-5, y=p: lib.tk_layer_norm(x, dt, m, c, c, w, wt, None, 0, eps, y, c, None, None, None)  # noqa: E731
    assert ln(m=0) == nt.TK_OK
    for bad in (dict(m=-1), dict(c=0), dict(c=2**31), dict(eps=-1.0), dict(eps=float("nan")), dict(x=None), dict(y=None)):
        assert ln(**bad) == nt.TK_ERR_INVALID, bad
        assert "tk_layer_norm" in nt.last_error()
    assert ln(dt=nt.TK_E4M3) == nt.TK_ERR_UNSUPPORTED and ln(wt=nt.TK_U8) == nt.TK_ERR_UNSUPPORTED
    bw = lambda dt=nt.TK_BF16, m=4, c=8, mean=p, dw=p, ws=p, wt=nt.TK_F32: lib.tk_layer_norm_backward(  # noqa: E731
        p, c, p, dt, m, c, c, p, wt, mean, p, p, c, dw, None, 0, ws, None)
    for bad in (dict(m=-1), dict(c=0), dict(mean=None), dict(ws=None)):
        assert bw(**bad) == nt.TK_ERR_INVALID, bad
    assert bw(dt=nt.TK_U8) == nt.TK_ERR_UNSUPPORTED and bw(wt=nt.TK_I32) == nt.TK_ERR_UNSUPPORTED
    assert [lib.tk_layer_norm_backward_workspace_bytes(5000, C) // (8 * C) for C in (1, 512, 513, 16384, 16385)] == [768, 768, 512, 512, 128]
    assert lib.tk_layer_norm_backward_workspace_bytes(0, 8) >= 0 and lib.tk_layer_norm_backward_workspace_bytes(5, 0) == 0

    def desc(**more):
        d = nt.VocabDesc()
        for name, kind in d._fields_:
            if kind is ctypes.c_void_p:
                setattr(d, name, p)
        d.logits_dtype, d.n_rows, d.vocab, d.temperature, d.k, d.n_teacher, d.teacher_dtype = nt.TK_BF16, 3, 100, 1.0, 4, 5, nt.TK_F32
        for name, value in more.items():
            setattr(d, name, value)
        return d

    entries = {e: getattr(lib, e) for e in ("tk_token_logprobs", "tk_token_logprobs_backward", "tk_distill_topk", "tk_distill_topk_backward")}
    shared = [dict(n_rows=-1), dict(vocab=0), dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=1e-39), dict(temperature=INF), dict(temperature=float("nan")), dict(logits=None)]
    own = {"tk_token_logprobs": [dict(k=-1), dict(k=101), dict(tokens=None), dict(logprobs=None), dict(entropy=None), dict(top_indx=None), dict(top_logprobs=None)],
           "tk_token_logprobs_backward": [dict(tokens=None), dict(entropy=None), dict(stats=None), dict(d_logits=None)],
           "tk_distill_topk": [dict(n_teacher=-1), dict(teacher_logits=None), dict(teacher_indx=None), dict(loss=None)],
           "tk_distill_topk_backward": [dict(n_teacher=-1), dict(teacher_logits=None), dict(stats=None), dict(teacher_stats=None), dict(d_logits=None)]}
    for name, entry in entries.items():
        assert entry(None, None) == nt.TK_ERR_INVALID
        assert entry(desc(n_rows=0), None) == nt.TK_OK
        for bad in shared + own[name]:
            assert entry(desc(**bad), None) == nt.TK_ERR_INVALID, (name, bad)
            assert name in nt.last_error()
        assert entry(desc(logits_dtype=nt.TK_U8), None) == nt.TK_ERR_UNSUPPORTED
    assert entries["tk_token_logprobs"](desc(vocab=1000, k=129), None) == nt.TK_ERR_UNSUPPORTED
    assert entries["tk_token_logprobs"](desc(vocab=524289), None) == nt.TK_ERR_UNSUPPORTED
    for name in ("tk_distill_topk", "tk_distill_topk_backward"):
        assert entries[name](desc(n_teacher=1025), None) == nt.TK_ERR_UNSUPPORTED
        assert entries[name](desc(teacher_dtype=nt.TK_I32), None) == nt.TK_ERR_UNSUPPORTED


def test_descriptor_matches_the_header(tmp_path):
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    fields = [f[0] for f in nt.VocabDesc._fields_]
    src = tmp_path / "probe.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "triton_amd.h"\nint main(void){printf("%zu", sizeof(tk_vocab_desc));\n'
                   + "".join(f'printf(" %zu", offsetof(tk_vocab_desc, {f}));\n' for f in fields) + "return 0;}\n")
    exe = tmp_path / "probe"
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-pedantic", "-I", os.path.join(root, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(nt.VocabDesc)] + [getattr(nt.VocabDesc, f).offset for f in fields]
