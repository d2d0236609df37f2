// Layer norm of rows, forward and backward.
#include "row_math.h"

namespace tk {
namespace {

template <int DT>
__global__ __launch_bounds__(256) void layer_norm_kernel(const void* x, int64_t M, int64_t C, int64_t sx, const void* w, int wt, const void* b, int bt,
                                                         float eps, void* y, int64_t sy, float* mean, float* rstd) {
  __shared__ float buf[3][4];
  for (int64_t m = blockIdx.x; m < M; m += gridDim.x) {
    float s = 0.f;
    for (int64_t c = threadIdx.x; c < C; c += 256) s += RowType<DT>::load(x, m * sx + c);
    const float mu = block_sum<256>(s, buf[0]) / (float)C;
    s = 0.f;
    for (int64_t c = threadIdx.x; c < C; c += 256) {
      const float d = RowType<DT>::load(x, m * sx + c) - mu;
      s = fmaf(d, d, s);
    }
    const float r = 1.0f / sqrtf(block_sum<256>(s, buf[1]) / (float)C + eps);
    for (int64_t c = threadIdx.x; c < C; c += 256) {
      const float h = (RowType<DT>::load(x, m * sx + c) - mu) * r;
      RowType<DT>::store(y, m * sy + c, fmaf(h, w ? load_any(w, wt, c) : 1.0f, b ? load_any(b, bt, c) : 0.0f));
    }
    if (threadIdx.x == 0) {
      if (mean) mean[m] = mu;
      if (rstd) rstd[m] = r;
    }
  }
}

template <int DT>
__global__ __launch_bounds__(256) void layer_norm_dx_kernel(const void* dy, int64_t sdy, const void* x, int64_t M, int64_t C, int64_t sx, const void* w, int wt,
                                                            const float* mean, const float* rstd, void* dx, int64_t sdx) {
  __shared__ float buf[3][4];
  for (int64_t m = blockIdx.x; m < M; m += gridDim.x) {
    const float mu = mean[m], r = rstd[m];
    float sg = 0.f, sgh = 0.f;
    for (int64_t c = threadIdx.x; c < C; c += 256) {
      const float g = RowType<DT>::load(dy, m * sdy + c) * (w ? load_any(w, wt, c) : 1.0f);
      sg += g;
      sgh = fmaf(g, (RowType<DT>::load(x, m * sx + c) - mu) * r, sgh);
    }
    sg = block_sum<256>(sg, buf[0]) / (float)C;
    sgh = block_sum<256>(sgh, buf[1]) / (float)C;
    for (int64_t c = threadIdx.x; c < C; c += 256) {
      const float g = RowType<DT>::load(dy, m * sdy + c) * (w ? load_any(w, wt, c) : 1.0f), h = (RowType<DT>::load(x, m * sx + c) - mu) * r;
      RowType<DT>::store(dx, m * sdx + c, (g - sg - h * sgh) * r);
    }
  }
}

constexpr int DW_PARTS = 128;  // workgroups along the rows that a column's sum is split over

// Partial sums of part blockIdx.y: parts [2][DW_PARTS][C].
template <int DT>
__global__ __launch_bounds__(256) void layer_norm_dw_parts_kernel(const void* dy, int64_t sdy, const void* x, int64_t M, int64_t C, int64_t sx,
                                                                  const float* mean, const float* rstd, float* parts) {
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= C) return;
  float dw = 0.f, db = 0.f;
  for (int64_t m = blockIdx.y; m < M; m += DW_PARTS) {
    const float g = RowType<DT>::load(dy, m * sdy + c);
    dw = fmaf(g, (RowType<DT>::load(x, m * sx + c) - mean[m]) * rstd[m], dw);
    db += g;
  }
  parts[blockIdx.y * C + c] = dw;
  parts[(DW_PARTS + blockIdx.y) * C + c] = db;
}

__global__ __launch_bounds__(256) void layer_norm_dw_kernel(const float* parts, int64_t C, void* dw, int wt, void* db, int bt) {
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= C) return;
  float a = 0.f, b = 0.f;
  for (int p = 0; p < DW_PARTS; ++p) {
    a += parts[p * C + c];
    b += parts[(DW_PARTS + p) * C + c];
  }
  if (dw) store_any(dw, wt, c, a);
  if (db) store_any(db, bt, c, b);
}

constexpr int64_t MAX_COLS = 0x7FFFFFFF;
unsigned rows_grid(int64_t M) { return (unsigned)(M < 65536 ? M : 65536); }

template <int DT>
void backward(const void* dy, int64_t sdy, const void* x, int64_t M, int64_t C, int64_t sx, const void* w, int wt, const float* mean, const float* rstd,
              void* dx, int64_t sdx, void* dw, void* db, int bt, float* parts, hipStream_t s) {
  if (dx && M) hipLaunchKernelGGL(layer_norm_dx_kernel<DT>, dim3(rows_grid(M)), dim3(256), 0, s, dy, sdy, x, M, C, sx, w, wt, mean, rstd, dx, sdx);
  if (!dw && !db) return;
  const unsigned cols = (unsigned)cdiv(C, 256);
  hipLaunchKernelGGL(layer_norm_dw_parts_kernel<DT>, dim3(cols, DW_PARTS), dim3(256), 0, s, dy, sdy, x, M, C, sx, mean, rstd, parts);
  hipLaunchKernelGGL(layer_norm_dw_kernel, dim3(cols), dim3(256), 0, s, parts, C, dw, wt, db, bt);
}

}  // namespace
}  // namespace tk

using namespace tk;

extern "C" int32_t tk_layer_norm(const void* x, int32_t dtype, int64_t n_rows, int64_t n_cols, int64_t stride_xm, const void* weight, int32_t weight_dtype,
                                 const void* bias, int32_t bias_dtype, float eps, void* y, int64_t stride_ym, float* mean, float* rstd,
                                 tk_stream_t stream) {
  if (n_rows < 0 || n_cols <= 0 || n_cols > MAX_COLS) return fail(TK_ERR_INVALID, "tk_layer_norm: bad sizes %lld x %lld", (long long)n_rows, (long long)n_cols);
  if (!(eps >= 0.f)) return fail(TK_ERR_INVALID, "tk_layer_norm: eps must not be negative");
  if (!is_row_dtype(dtype) || (weight && !is_row_dtype(weight_dtype)) || (bias && !is_row_dtype(bias_dtype)))
    return fail(TK_ERR_UNSUPPORTED, "tk_layer_norm: fp32, bf16 and fp16 only");
  if (n_rows == 0) return TK_OK;
  if (!x || !y) return fail(TK_ERR_INVALID, "tk_layer_norm: null pointer");
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto k = dtype == TK_F32 ? layer_norm_kernel<TK_F32> : dtype == TK_BF16 ? layer_norm_kernel<TK_BF16> : layer_norm_kernel<TK_F16>;
  hipLaunchKernelGGL(k, dim3(rows_grid(n_rows)), dim3(256), 0, s, x, n_rows, n_cols, stride_xm, weight, weight_dtype, bias, bias_dtype, eps, y, stride_ym,
                     mean, rstd);
  return check_launch("layer_norm_kernel");
}

extern "C" int64_t tk_layer_norm_backward_workspace_bytes(int64_t n_rows, int64_t n_cols) { return n_cols > 0 ? 2 * DW_PARTS * n_cols * 4 : 0; }

extern "C" int32_t tk_layer_norm_backward(const void* dy, int64_t stride_dym, const void* x, int32_t dtype, int64_t n_rows, int64_t n_cols,
                                          int64_t stride_xm, const void* weight, int32_t weight_dtype, const float* mean, const float* rstd, void* dx,
                                          int64_t stride_dxm, void* dweight, void* dbias, int32_t bias_dtype, void* workspace, tk_stream_t stream) {
  if (n_rows < 0 || n_cols <= 0 || n_cols > MAX_COLS)
    return fail(TK_ERR_INVALID, "tk_layer_norm_backward: bad sizes %lld x %lld", (long long)n_rows, (long long)n_cols);
  if (!is_row_dtype(dtype) || ((weight || dweight) && !is_row_dtype(weight_dtype)) || (dbias && !is_row_dtype(bias_dtype)))
    return fail(TK_ERR_UNSUPPORTED, "tk_layer_norm_backward: fp32, bf16 and fp16 only");
  if (n_rows && (!dy || !x || !mean || !rstd)) return fail(TK_ERR_INVALID, "tk_layer_norm_backward: null pointer");
  if ((dweight || dbias) && !workspace) return fail(TK_ERR_INVALID, "tk_layer_norm_backward: the sums over rows need a workspace");
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto f = dtype == TK_F32 ? backward<TK_F32> : dtype == TK_BF16 ? backward<TK_BF16> : backward<TK_F16>;
  f(dy, stride_dym, x, n_rows, n_cols, stride_xm, weight, weight_dtype, mean, rstd, dx, stride_dxm, dweight, dbias, bias_dtype,
    static_cast<float*>(workspace), s);
  return check_launch("layer_norm_backward");
}
