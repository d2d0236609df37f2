// Gradient of the experts' weights from 8-bit activations: y[e] = (x scales)^T dy over the rows of slice e (tk_fp8_block_wgrad).
#include "fp8_blocks.h"
#include "ragged_k.h"

namespace tk {
namespace {

struct WgradParams {
  const uint8_t* x;
  int64_t x_t;
  const float* xs;
  int64_t xs_t, xs_k;
  const uint16_t* dy;
  int64_t dy_t;
  const int32_t* slice_sizes;
  const int32_t* slice_offs;
  int32_t n_slices, T, K, N;
  uint8_t* y;
  int64_t y_e, y_k;
  int32_t tiles_k, tiles_n;
};

// an e4m3 times its scale in dy's type (in fp16 at most its largest number)
template <int DT>
__device__ __forceinline__ uint32_t scaled_pair(float a, float b, float s) {
  a *= s, b *= s;
  if constexpr (DT == TK_F16) a = at_least(at_most(a, 65504.f), -65504.f), b = at_least(at_most(b, 65504.f), -65504.f);
  return pack_out2<DT == TK_F16>(a, b);
}

// Any strides and alignments: 64 x 64 tiles, four waves of 32 x 32, stages of 32 rows, turned into K-contiguous lines on their way into LDS.
template <int DT, int YT>
__global__ __launch_bounds__(256) void fp8_wgrad_any_kernel(const WgradParams p) {
  constexpr int STAGE = 32, PITCH = STAGE + 8;  // elements of a line
  __shared__ __attribute__((aligned(16))) uint16_t xs[64 * PITCH], ds[64 * PITCH];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int lr = lane & 31, h = lane >> 5, mw = wave & 1, nw = wave >> 1;
  int id = blockIdx.x;
  const int tn = id % p.tiles_n;
  id /= p.tiles_n;
  const int tk = id % p.tiles_k, e = id / p.tiles_k;
  const int k0 = tk * 64, n0 = tn * 64;
  const int rows = p.slice_sizes ? p.slice_sizes[e] : p.T;
  const int64_t first = p.slice_sizes ? p.slice_offs[e] : 0;
  const int row = tid >> 3, c = (tid & 7) * 8;  // this thread's row of the stage, and its eight columns of either operand
  f32x16_t acc = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int t0 = 0; t0 < rows; t0 += STAGE) {
    const int64_t t = first + t0 + row;
    const bool in = t0 + row < rows;
    uint16_t xv[8], dv[8];
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      float a[2] = {0.f, 0.f};
      float s = 0.f;
      if (in && k0 + c < p.K) s = p.xs[t * p.xs_t + (int64_t)(k0 / kFp8Block) * p.xs_k];
#pragma unroll
      for (int q = 0; q < 2; ++q)
        if (in && k0 + c + i + q < p.K) a[q] = __builtin_amdgcn_cvt_f32_fp8((int)p.x[t * p.x_t + k0 + c + i + q], 0);
      const uint32_t w = scaled_pair<DT>(a[0], a[1], s);
      xv[i] = (uint16_t)w, xv[i + 1] = (uint16_t)(w >> 16);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) dv[i] = in && n0 + c + i < p.N ? p.dy[t * p.dy_t + n0 + c + i] : 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) xs[(c + i) * PITCH + row] = xv[i], ds[(c + i) * PITCH + row] = dv[i];
    __syncthreads();
#pragma unroll
    for (int u = 0; u < STAGE / 16; ++u) {
      const u32x4_t a = *reinterpret_cast<const u32x4_t*>(ds + (nw * 32 + lr) * PITCH + u * 16 + h * 8);
      const u32x4_t b = *reinterpret_cast<const u32x4_t*>(xs + (mw * 32 + lr) * PITCH + u * 16 + h * 8);
      acc = mfma_k16<DT>(a, b, acc);
    }
  }
  const int k = k0 + mw * 32 + lr;
  if (k >= p.K) return;
  uint8_t* line = p.y + (e * p.y_e + k * p.y_k) * (YT == TK_F32 ? 4 : 2);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int n = n0 + nw * 32 + Frag<32>::n_of(i, h);
    if (n < p.N) store_elem<YT>(line, n, acc[i]);
  }
}

int32_t launch_any(WgradParams p, int dt, int yt, hipStream_t st) {
  p.tiles_k = (int)cdiv(p.K, 64), p.tiles_n = (int)cdiv(p.N, 64);
  const int64_t grid = (int64_t)p.tiles_k * p.tiles_n * p.n_slices;
  if (grid > 0x7FFFFFFF) return fail(TK_ERR_UNSUPPORTED, "tk_fp8_block_wgrad: grid too large");
  auto launch = [&](auto kern) { hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(256), 0, st, p); };
  if (dt == TK_BF16)
    yt == TK_F32 ? launch(fp8_wgrad_any_kernel<TK_BF16, TK_F32>) : yt == TK_BF16 ? launch(fp8_wgrad_any_kernel<TK_BF16, TK_BF16>) : launch(fp8_wgrad_any_kernel<TK_BF16, TK_F16>);
  else
    yt == TK_F32 ? launch(fp8_wgrad_any_kernel<TK_F16, TK_F32>) : yt == TK_BF16 ? launch(fp8_wgrad_any_kernel<TK_F16, TK_BF16>) : launch(fp8_wgrad_any_kernel<TK_F16, TK_F16>);
  return check_launch("fp8_wgrad_any_kernel");
}

}  // namespace
}  // namespace tk

using namespace tk;

extern "C" int32_t tk_fp8_block_wgrad(const tk_fp8_wgrad_desc* d, tk_stream_t stream) {
  if (!d) return fail(TK_ERR_INVALID, "tk_fp8_block_wgrad: null descriptor");
  if (d->T < 0 || d->K < 0 || d->N < 0 || d->n_slices < 0) return fail(TK_ERR_INVALID, "tk_fp8_block_wgrad: negative size");
  if (d->dy_dtype != TK_BF16 && d->dy_dtype != TK_F16) return fail(TK_ERR_UNSUPPORTED, "tk_fp8_block_wgrad: dy must be bf16 or fp16 (dtype %d)", d->dy_dtype);
  if (d->y_dtype != TK_F32 && d->y_dtype != TK_BF16 && d->y_dtype != TK_F16) return fail(TK_ERR_UNSUPPORTED, "tk_fp8_block_wgrad: the gradient is fp32, bf16 or fp16 (dtype %d)", d->y_dtype);
  if (d->slice_sizes ? !d->slice_offs : d->n_slices > 1) return fail(TK_ERR_INVALID, "tk_fp8_block_wgrad: slices need their sizes and offsets");
  if (d->n_slices == 0 || d->K == 0 || d->N == 0) return TK_OK;
  if (!d->y || (d->T > 0 && (!d->x || !d->x_scale || !d->dy))) return fail(TK_ERR_INVALID, "tk_fp8_block_wgrad: null operand");
  WgradParams p = {};
  p.x = d->x, p.x_t = d->x_stride_t, p.xs = d->x_scale, p.xs_t = d->xs_stride_t, p.xs_k = d->xs_stride_k;
  p.dy = static_cast<const uint16_t*>(d->dy), p.dy_t = d->dy_stride_t;
  p.slice_sizes = d->slice_sizes, p.slice_offs = d->slice_offs, p.n_slices = d->n_slices;
  p.T = d->T, p.K = d->K, p.N = d->N;
  p.y = static_cast<uint8_t*>(d->y), p.y_e = d->y_stride_e, p.y_k = d->y_stride_k;
  return launch_any(p, d->dy_dtype, d->y_dtype, static_cast<hipStream_t>(stream));
}
