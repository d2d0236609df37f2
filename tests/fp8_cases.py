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
