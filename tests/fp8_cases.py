"""The kernel that a product in 8 bits takes, asked of the library by its sizes, strides and addresses."""
import ctypes

import torch

from triton_amd import _native as nt
from triton_amd.tensor import RaggedTensorMetadata

ANY, FEW, RING = 1, 16, 64


def product_desc(M, K, N, E=1, *, ragged=None, out_dtype=torch.bfloat16, x=4096, x_stride=None, x_rows=None, w=4096, w_stride=None, gather=False, **more):
    """A descriptor of a product with lines of `x_stride` and `w_stride` bytes at addresses `x` and `w` that nothing follows."""
    x_stride, w_stride = x_stride or -(-K // 16) * 16, w_stride or -(-K // 16) * 16
    d = nt.Fp8GemmDesc()
    d.x, d.x_stride_m, d.x_rows, d.x_scale, d.xs_stride_m, d.xs_stride_k = x, x_stride, M if x_rows is None else x_rows, 4096, -(-K // 128), 1
    d.w, d.w_stride_e, d.w_stride_n = w, N * w_stride, w_stride
    d.w_scale, d.ws_stride_e, d.ws_stride_k, d.ws_stride_n = 4096, -(-K // 128) * -(-N // 128), 1, -(-K // 128)
    d.n_slices, d.M, d.N, d.K, d.y, d.y_dtype = E, M, N, K, 4096, nt.TORCH_TO_TK[out_dtype]
    if gather:
        d.gather_indx = 4096
    if E > 1 if ragged is None else ragged:
        d.slice_sizes, d.slice_offs, d.block_schedule, d.grid_m = 4096, 4096, 4096, RaggedTensorMetadata.n_blocks(E, M, 64)
    for name, v in more.items():
        setattr(d, name, v)
    return d


def kernel_of(desc, cus=256):
    kernel = ctypes.c_int32(-1)
    nt.check(nt.lib().tk_host_fp8_block_gemm_kernel(desc, cus, kernel))
    return kernel.value


def gradient_desc(T, K, N, E=1, *, workspace=True, dy_dtype=torch.bfloat16, **more):
    """A descriptor of a weights' gradient from lines at sixteen-byte boundaries that nothing follows."""
    d = nt.Fp8WgradDesc()
    d.x, d.x_stride_t, d.x_scale, d.xs_stride_t, d.xs_stride_k = 4096, -(-K // 16) * 16, 4096, -(-K // 128), 1
    d.dy, d.dy_dtype, d.dy_stride_t = 4096, nt.TORCH_TO_TK[dy_dtype], -(-N // 8) * 8
    if E > 1:
        d.slice_sizes, d.slice_offs = 4096, 4096
    d.n_slices, d.T, d.K, d.N, d.y, d.y_dtype, d.y_stride_e, d.y_stride_k = E, T, K, N, 4096, nt.TK_F32, K * N, N
    d.workspace = 4096 if workspace is True else workspace or None
    for name, v in more.items():
        setattr(d, name, v)
    return d


def gradient_kernel_of(desc, cus=256):
    """`(tile, parts)`"""
    tile, parts = ctypes.c_int32(-1), ctypes.c_int32(-1)
    nt.check(nt.lib().tk_host_fp8_block_wgrad_kernel(desc, cus, tile, parts))
    return tile.value, parts.value
