"""e4m3 in blocks of 128 without a GPU: the oracle against definitions and differences, the plain twins against the oracle, the descriptors against the header, and
what the operators and their C entries refuse."""
import ctypes
import os
import re
import subprocess

import pytest
import torch

from oracle import fp8_blocks as orc
from oracle.rows import check
from triton_amd import _native as nt
from triton_kernels import fp8_blocks as ops
from triton_kernels.matmul import FnSpecs, FusedActivation
from triton_kernels.swiglu import swiglu_fn

F32, BF16, F16, E4M3 = torch.float32, torch.bfloat16, torch.float16, torch.float8_e4m3fn
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_oracle_rounds_to_the_nearest_number():
    every = torch.arange(256, dtype=torch.uint8).view(E4M3).to(torch.float64)
    every = every[every.isfinite()].unique()
    v = torch.cat([every, (every[1:] + every[:-1]) / 2, torch.linspace(-448, 448, 5001, dtype=torch.float64)])
    assert torch.equal(orc.e4m3(v), v.to(F32).to(E4M3).to(torch.float64))
    near = every[(v[:, None] - every).abs().argmin(1)]
    assert torch.equal((orc.e4m3(v) - v).abs(), (near - v).abs())


def test_oracle_scales_are_the_smallest_powers_of_two():
    x = torch.randn((3, 500), generator=torch.Generator().manual_seed(0)) * torch.logspace(-20, 20, 500)
    values, scales = orc.downcast(x)
    top = torch.stack([p.abs().amax(1) for p in x.double().split(128, 1)], 1)
    assert (top <= 448 * scales).all() and (top > 224 * scales).all()
    assert torch.equal(torch.frexp(scales).mantissa, torch.full_like(scales, 0.5))
    assert ((values * scales.repeat_interleave(128, 1)[:, :500] - x).abs() <= 2.0**-4 * x.abs() + 2.0**-10 * scales.repeat_interleave(128, 1)[:, :500]).all()


def test_oracle_gradients_are_slopes():
    g = torch.Generator().manual_seed(1)
    a = torch.randn((4, 20), generator=g, dtype=torch.float64) * 2
    d = torch.randn((4, 10), generator=g, dtype=torch.float64)
    v = torch.randn((4, 20), generator=g, dtype=torch.float64)
    one = torch.ones((4, 1))
    for limit in (None, 1.5):
        kept = (a * 16).round().clamp(-448, 448).to(F32).to(E4M3)           # numbers that 8 bits hold
        at = kept.double()
        f = lambda t: (orc._act(t, torch.zeros_like(t), 0.7, limit)[0] * d).sum()  # noqa: E731
        slope = (f(at + 1e-5 * v) - f(at - 1e-5 * v)) / 2e-5
        assert abs(slope - (orc.swiglu_backward(d.float(), kept, one, 0.7, limit)[0] * v).sum()) < 1e-4 * (1 + abs(slope))
    x, s = orc.downcast(a.float())
    dy, w = torch.randn((4, 6), generator=g), torch.randn((20, 6), generator=g, dtype=torch.float64)
    dw = orc.weight_gradient(x.float().to(E4M3), s.float(), dy.to(BF16))[0][0]
    xs = x * s.repeat_interleave(128, 1)[:, :20]
    f = lambda t: ((xs @ t) * dy.to(BF16).double()).sum()  # noqa: E731
    u = torch.randn(w.shape, generator=g, dtype=torch.float64)
    assert abs((f(w + u) - f(w - u)) / 2 - (dw * u).sum()) < 1e-9


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_twins_match_the_oracle(dtype):
    g = torch.Generator().manual_seed(2)
    x = (torch.randn((5, 300), generator=g) * 3).to(dtype)
    x[1, 2], x[2, 3], x[3] = float("nan"), float("inf"), 0
    for rows in (1, 128):
        values, scales = ops.downcast_to_fp8_blocks_torch(x, rows)
        want = orc.downcast(x, rows)
        assert torch.equal(values.double().nan_to_num(1e9), want[0].nan_to_num(1e9)) and torch.equal(scales.double(), want[1])
        back = ops.upcast_from_fp8_blocks_torch(values, scales, F32, rows)
        assert torch.equal(back.double().nan_to_num(1e9), orc.upcast(values, scales, rows).nan_to_num(1e9))
    x = (torch.randn((9, 200), generator=g) * 2).to(dtype)
    a, a_scale = ops.downcast_to_fp8_blocks_torch(x)
    w, w_scale = ops.downcast_to_fp8_blocks_torch(torch.randn((1, 200, 70), generator=g), 128)
    act = FusedActivation(FnSpecs("swiglu", swiglu_fn, ("alpha", "limit"), reduction_n=2), (1.7, 2.0))
    for swiglu in (None, (1.7, 2.0)):
        y = ops.matmul_fp8_blocks_torch(a, a_scale, w, w_scale, fused_activation=act if swiglu else None, out_dtype=BF16)
        check(y, *orc.product(a, a_scale, w, w_scale, swiglu=swiglu)[:2], "y")
    dy = torch.randn((9, 30), generator=g).to(BF16)
    check(ops.weight_gradient_fp8_blocks_torch(a, a_scale, dy, None, F32)[None], *orc.weight_gradient(a, a_scale, dy), "dw")
    dh = torch.randn((9, 100), generator=g).to(dtype)
    for limit in (None, 1.0):
        check(ops.swiglu_fp8_backward_torch(dh, a, a_scale, 1.7, limit), *orc.swiglu_backward(dh, a, a_scale, 1.7, limit), "da")


def _fields(name):
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "triton_amd.h")).read(), flags=re.S)
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, flags=re.S).group(1)
    return [re.search(r"(\w+)\s*$", part).group(1) for decl in body.split(";") if decl.strip() for part in decl.strip().split(",")]


def test_descriptors_match_the_header(tmp_path):
    pairs = (("tk_fp8_gemm_desc", nt.Fp8GemmDesc), ("tk_fp8_wgrad_desc", nt.Fp8WgradDesc))
    for name, cls in pairs:
        assert _fields(name) == [f[0] for f in cls._fields_]
    src = tmp_path / "probe.c"
    src.write_text('#include <stdio.h>\n#include "triton_amd.h"\nint main(void){printf("%zu %zu\\n", sizeof(tk_fp8_gemm_desc), sizeof(tk_fp8_wgrad_desc));return 0;}\n')
    exe = tmp_path / "probe"
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-pedantic", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    assert [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()] == [ctypes.sizeof(c) for _, c in pairs]


def _raises(kind, match, f, *args, **kw):
    with pytest.raises(kind, match=match):
        f(*args, **kw)


def test_what_the_operators_refuse():
    x, q = torch.ones((4, 256)), torch.ones((4, 256)).to(E4M3)
    s = torch.ones((4, 2))
    w, ws = torch.ones((2, 64, 256)).to(E4M3).transpose(1, 2), torch.ones((2, 2, 1))
    i = torch.zeros(4, dtype=torch.int32)
    _raises(RuntimeError, "no CPU path", ops.downcast_to_fp8_blocks, x)
    _raises(NotImplementedError, "1 or 128 rows", ops.downcast_to_fp8_blocks, x, 64)
    _raises(NotImplementedError, "must be float32", ops.downcast_to_fp8_blocks, x.double())
    _raises(ValueError, "must have a row", ops.downcast_to_fp8_blocks, torch.ones(()))
    _raises(NotImplementedError, "no gradient for x", ops.downcast_to_fp8_blocks, x.clone().requires_grad_())
    _raises(NotImplementedError, "values must be", ops.upcast_from_fp8_blocks, x, s)
    _raises(ValueError, "scales must be", ops.upcast_from_fp8_blocks, q, s[:3])
    _raises(ValueError, "scales must be", ops.upcast_from_fp8_blocks, q, s, block_rows=128)
    _raises(NotImplementedError, "result is", ops.upcast_from_fp8_blocks, q, s, torch.float64)
    good = (q, s, w[:1], ws[:1])
    for match, kind, args, kw in (
        ("no CPU path", RuntimeError, good, {}),
        ("a must be", NotImplementedError, (x, s, w, ws), {}),
        ("a_scale must be", ValueError, (q, s.double(), w, ws), {}),
        ("a must be", ValueError, (q[0], s, w, ws), {}),
        ("w must be", NotImplementedError, (q, s, w.float(), ws), {}),
        ("w must be", ValueError, (q, s, w[None], ws), {}),
        ("reduction dims", ValueError, (q, s, w[:1, :200], ws[:1]), {}),
        ("w_scale must be", ValueError, (q, s, w[:1], ws), {}),
        ("bias must be", ValueError, good, dict(bias=torch.ones((1, 63)))),
        ("bias must be", NotImplementedError, good, dict(bias=torch.ones((1, 64), dtype=F16))),
        ("gammas must be", ValueError, good, dict(gammas=torch.ones(5))),
        ("gather_indx must be", ValueError, good, dict(gather_indx=i.long())),
        ("scatter_indx must be", ValueError, good, dict(scatter_indx=i[:, None])),
        ("output is", NotImplementedError, good, dict(out_dtype=E4M3)),
        ("even number", ValueError, (q, s, w[:1, :, :63], ws[:1]), dict(fused_activation=FusedActivation(FnSpecs("swiglu", swiglu_fn, ("alpha", "limit"), reduction_n=2), (1.0, None)))),
        ("not supported", NotImplementedError, good, dict(fused_activation=FusedActivation(FnSpecs("gelu", swiglu_fn, (), reduction_n=1), ()))),
        ("no gradient for bias", NotImplementedError, good, dict(bias=torch.ones((1, 64), requires_grad=True))),
    ):
        _raises(kind, match, ops.matmul_fp8_blocks, *args, **kw)
    dy = torch.ones((4, 8), dtype=BF16)
    _raises(RuntimeError, "no CPU path", ops.weight_gradient_fp8_blocks, q, s, dy)
    _raises(NotImplementedError, "dy must be", ops.weight_gradient_fp8_blocks, q, s, dy.float())
    _raises(ValueError, "dy must be", ops.weight_gradient_fp8_blocks, q, s, dy[:3])
    _raises(NotImplementedError, "gradient is", ops.weight_gradient_fp8_blocks, q, s, dy, None, torch.float64)
    xb, wf = x.to(BF16), torch.ones((256, 64))
    _raises(RuntimeError, "no CPU path", ops.linear_fp8_blocks, xb, wf)
    _raises(NotImplementedError, "x must be", ops.linear_fp8_blocks, x, wf)
    _raises(ValueError, "do not go together", ops.linear_fp8_blocks, xb, wf[:200])
    _raises(RuntimeError, "no CPU path", ops.quantize_fp8_weight, wf)
    _raises(ValueError, "w must be", ops.quantize_fp8_weight, wf[0])
    _raises(RuntimeError, "no CPU path", ops.swiglu_fp8_checkpoint, x, 1.0)
    _raises(RuntimeError, "no CPU path", ops.swiglu_fp8_backward, torch.ones((4, 128)), q, s, 1.0)
    _raises(ValueError, "dh must be", ops.swiglu_fp8_backward, torch.ones((4, 127)), q, s, 1.0)


def test_what_the_entries_refuse():
    lib, p = nt.lib(), 4096                                                  # (a pointer that no refused call follows)
    down = lambda **k: lib.tk_fp8_block_downcast(*{**dict(x=p, dt=nt.TK_BF16, b=1, r=4, c=8, xb=0, xr=8, rows=1, v=p, vb=0, vr=16, t=None, tb=0, tc=0, s=p, sb=0, sr=1, sc=1, st=None), **k}.values())  # noqa: E731
    assert down(b=0) == nt.TK_OK and down(r=0) == nt.TK_OK and down(c=0) == nt.TK_OK
    assert down(x=None) == nt.TK_ERR_INVALID and down(r=-1) == nt.TK_ERR_INVALID and down(s=None) == nt.TK_ERR_INVALID
    assert down(dt=nt.TK_E4M3) == nt.TK_ERR_UNSUPPORTED and down(rows=32) == nt.TK_ERR_UNSUPPORTED and down(t=p) == nt.TK_ERR_UNSUPPORTED
    up = lambda **k: lib.tk_fp8_block_upcast(*{**dict(v=p, b=1, r=4, c=8, vb=0, vr=16, rows=1, s=p, sb=0, sr=1, sc=1, o=p, dt=nt.TK_BF16, ob=0, or_=8, st=None), **k}.values())  # noqa: E731
    assert up(r=0) == nt.TK_OK and up(o=None) == nt.TK_ERR_INVALID and up(dt=nt.TK_U8) == nt.TK_ERR_UNSUPPORTED and up(rows=2) == nt.TK_ERR_UNSUPPORTED

    def gemm(**k):
        d = nt.Fp8GemmDesc()
        for name, v in {**dict(x=p, x_rows=4, x_scale=p, w=p, w_scale=p, n_slices=1, M=4, N=8, K=128, y=p, y_dtype=nt.TK_BF16), **k}.items():
            setattr(d, name, v)
        return lib.tk_fp8_block_gemm(d, None)

    assert gemm(M=0) == nt.TK_OK and gemm(N=0) == nt.TK_OK and lib.tk_fp8_block_gemm(None, None) == nt.TK_ERR_INVALID
    for bad in (dict(M=-1), dict(y=None), dict(x=None), dict(w_scale=None), dict(n_slices=2), dict(slice_sizes=p), dict(activation=7), dict(activation=1, N=7)):
        assert gemm(**bad) == nt.TK_ERR_INVALID, bad
    for bad in (dict(y_dtype=nt.TK_E4M3), dict(bias=p, bias_dtype=nt.TK_F16), dict(gammas=p, gammas_dtype=nt.TK_I32), dict(slice_sizes=p, slice_offs=p, block_schedule=p, n_slices=70000)):
        assert gemm(**bad) == nt.TK_ERR_UNSUPPORTED, bad

    def wgrad(**k):
        d = nt.Fp8WgradDesc()
        for name, v in {**dict(x=p, x_scale=p, dy=p, dy_dtype=nt.TK_BF16, n_slices=1, T=4, K=8, N=8, y=p, y_dtype=nt.TK_F32), **k}.items():
            setattr(d, name, v)
        return lib.tk_fp8_block_wgrad(d, None)

    assert wgrad(n_slices=0) == nt.TK_OK and wgrad(K=0) == nt.TK_OK and lib.tk_fp8_block_wgrad(None, None) == nt.TK_ERR_INVALID
    for bad in (dict(T=-1), dict(y=None), dict(dy=None), dict(n_slices=2), dict(slice_sizes=p)):
        assert wgrad(**bad) == nt.TK_ERR_INVALID, bad
    for bad in (dict(dy_dtype=nt.TK_F32), dict(y_dtype=nt.TK_U8)):
        assert wgrad(**bad) == nt.TK_ERR_UNSUPPORTED, bad
    act = lambda **k: lib.tk_swiglu_fp8(*{**dict(a=p, dt=nt.TK_BF16, m=4, n=4, am=8, o=p, om=4, v=p, vm=16, s=p, sm=1, sc=1, al=1.0, li=0.0, has=0, st=None), **k}.values())  # noqa: E731
    assert act(m=0) == nt.TK_OK and act(v=None) == nt.TK_ERR_INVALID and act(o=None) == nt.TK_ERR_INVALID and act(dt=nt.TK_E4M3) == nt.TK_ERR_UNSUPPORTED
    back = lambda **k: lib.tk_swiglu_fp8_backward(*{**dict(d=p, dt=nt.TK_BF16, m=4, n=4, dm=4, v=p, vm=16, s=p, sm=1, sc=1, o=p, om=8, al=1.0, li=0.0, has=0, st=None), **k}.values())  # noqa: E731
    assert back(n=0) == nt.TK_OK and back(s=None) == nt.TK_ERR_INVALID and back(m=-1) == nt.TK_ERR_INVALID and back(dt=nt.TK_U8) == nt.TK_ERR_UNSUPPORTED


def test_sizes_beyond_32_bits_and_long_slices_are_refused():
    lib, p = nt.lib(), 4096

    def gemm(**k):
        d = nt.Fp8GemmDesc()
        for name, v in {**dict(x=p, x_rows=4, x_stride_m=128, x_scale=p, w=p, w_stride_e=1024, w_stride_n=128, w_scale=p, n_slices=1, M=4, N=8, K=128, y=p, y_dtype=nt.TK_BF16), **k}.items():
            setattr(d, name, v)
        return lib.tk_fp8_block_gemm(d, None)

    for bad in (dict(M=2**31 - 1), dict(N=2**31 - 256 + 1), dict(K=2**31 - 1)):
        assert gemm(**bad) == nt.TK_ERR_UNSUPPORTED, bad
    # a schedule counts up to 2^15 row blocks of 64 in a slice: beyond it only the kernels that need none
    ragged = dict(slice_sizes=p, slice_offs=p, block_schedule=p, grid_m=2**15 + 1, n_slices=2, M=2**21 + 1)
    for bad in (dict(y_dtype=nt.TK_F32), dict(x=p + 1), dict(w_stride_n=136), dict(K=0), dict(n_slices=300)):
        assert gemm(**{**ragged, **bad}) == nt.TK_ERR_UNSUPPORTED, bad
    d = nt.Fp8WgradDesc()
    for name, v in dict(x=p, x_scale=p, dy=p, dy_dtype=nt.TK_BF16, n_slices=1, T=2**31 - 1, K=8, N=8, y=p, y_dtype=nt.TK_F32).items():
        setattr(d, name, v)
    assert lib.tk_fp8_block_wgrad(d, None) == nt.TK_ERR_UNSUPPORTED
    for name in ("rows", "K", "N"):
        _raises(NotImplementedError, f"got {name}=2147483648", ops._fit, **{name: 2**31})


def test_operands_that_want_a_gradient_are_refused():
    q, s = torch.ones((4, 256)).to(E4M3), torch.ones((4, 2))
    w, ws = torch.ones((1, 64, 256)).to(E4M3).transpose(1, 2), torch.ones((1, 2, 1))
    wants = lambda t: t.clone().requires_grad_()  # noqa: E731
    _raises(NotImplementedError, "no gradient for a", ops.matmul_fp8_blocks, wants(q), s, w, ws)
    _raises(NotImplementedError, "no gradient for w", ops.matmul_fp8_blocks, q, s, wants(w), ws)
    _raises(NotImplementedError, "no gradient for values", ops.upcast_from_fp8_blocks, wants(q), s)
    _raises(NotImplementedError, "no gradient for x", ops.weight_gradient_fp8_blocks, wants(q), s, torch.ones((4, 8), dtype=BF16))
    _raises(NotImplementedError, "no gradient for a", ops.swiglu_fp8_forward, torch.ones((4, 8), requires_grad=True), 1.0)
    _raises(NotImplementedError, "no gradient for dh", ops.swiglu_fp8_backward, torch.ones((4, 128), requires_grad=True), q, s, 1.0)


@pytest.mark.parametrize("case,kernel", [
    (dict(M=1, K=4096, N=4096), 16), (dict(M=1, K=4096, N=14336), 64), (dict(M=32, K=4096, N=4096), 16), (dict(M=64, K=4096, N=4096), 64), (dict(M=700, K=1000, N=1023, E=3), 64),
    (dict(M=700, K=1000, N=1023, E=3, x=4097), 1), (dict(M=1, K=4096, N=4096, out_dtype=F32), 16), (dict(M=4096, K=4096, N=4096, out_dtype=F32), 1), (dict(M=128, K=2880, N=5760, E=32), 64),
    (dict(M=4096, K=2880, N=2880, E=32), 128), (dict(M=2048, K=1024, N=2304), 128), (dict(M=16384, K=4096, N=14336, E=8, gather=True), 256), (dict(M=16384, K=2880, N=5760, E=8), 256),
    (dict(M=16384, K=2880, N=5760, E=8, w_stride=2888), 1), (dict(M=4096, K=2880, N=2880, E=300), 64), (dict(M=2**21 + 64, K=16, N=16, E=2), 128), (dict(M=100, K=64, N=64, E=2, grid_m=0), 0),
    (dict(M=100, K=64, N=64, E=2, grid_m=0, zero_rest=1), 2), (dict(M=0, K=64, N=64), 0)])
def test_the_kernel_that_a_product_takes(case, kernel):
    from fp8_cases import kernel_of, product_desc
    assert kernel_of(product_desc(**case)) == kernel


def test_the_kernel_of_a_refused_product():
    from fp8_cases import kernel_of, product_desc
    _raises(NotImplementedError, "sizes up to", kernel_of, product_desc(2**31 - 1, 16, 16))
    _raises(ValueError, "bad argument", kernel_of, product_desc(1, 16, 16), 0)


@pytest.mark.parametrize("case,kernel", [
    (dict(T=16384, K=2880, N=5760, E=8), (256, 1)), (dict(T=333, K=520, N=776, E=5), (128, 1)), (dict(T=300, K=2300, N=2100, E=7), (256, 1)), (dict(T=400, K=1100, N=1100, E=3), (128, 1)),
    (dict(T=8192, K=128, N=72), (128, 32)), (dict(T=8192, K=128, N=72, workspace=False), (128, 1)), (dict(T=8192, K=512, N=2048), (128, 8)), (dict(T=100, K=128, N=72, x=4097), (64, 1)),
    (dict(T=100, K=128, N=72, dy_stride_t=76), (64, 1)), (dict(T=100, K=0, N=72), (0, 0)), (dict(T=0, K=128, N=72), (128, 1))])
def test_the_kernel_that_a_gradient_takes(case, kernel):
    from fp8_cases import gradient_desc, gradient_kernel_of
    assert gradient_kernel_of(gradient_desc(**case)) == kernel


def test_the_kernel_of_a_refused_gradient():
    from fp8_cases import gradient_desc, gradient_kernel_of
    _raises(ValueError, "not 16-byte aligned", gradient_kernel_of, gradient_desc(8192, 128, 72, workspace=4100))
    _raises(ValueError, "bad argument", gradient_kernel_of, gradient_desc(1, 16, 16), 0)


def test_gathered_rows_of_two_gibibytes():
    """Beyond the reach of a buffer resource the kernel for any lines takes them, and where the schedule does not suffice the refusal says what for."""
    from fp8_cases import kernel_of, product_desc
    rows = 2**31 // 4096
    for n, kernel in ((rows - 1, 256), (rows, 1)):
        assert kernel_of(product_desc(16384, 4096, 14336, 8, gather=True, x_rows=n)) == kernel
    assert kernel_of(product_desc(16384, 4096, 14336, 8, x_rows=rows)) == 256
    assert kernel_of(product_desc(2**21 + 64, 4096, 256, 2, gather=True, x_rows=rows - 1)) in (128, 256)
    _raises(NotImplementedError, "less than 2 GiB to gather from", kernel_of, product_desc(2**21 + 64, 4096, 256, 2, gather=True, x_rows=rows))
