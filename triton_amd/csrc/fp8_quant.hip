// e4m3 with one fp32 scale for each block of 128: writing it (rows, with swiglu in front where asked for, and 128 x 128 blocks), reading it back, and the
// backward pass of swiglu from it.
//
// HBM bounds all of it: a pass over the data, eight consecutive elements a lane.  us: 16384 x 4096 bf16 written and read back 73 (5.5 TB/s; a copy of 1 GiB 5.0), eight matrices of 2880 x 5760 in both orders 111
// (4.8), swiglu of 16384 x 11520 with its 8-bit copy and its gradient 291 (5.2).
#include "fp8_blocks.h"

namespace tk {
namespace {

struct RowsParams {
  const void* x;  // what is quantised [batch, rows, cols]
  int64_t x_b, x_r;
  uint8_t* v;
  int64_t v_b, v_r;
  float* s;
  int64_t s_b, s_r, s_c;
  void* y;  // swiglu: its output; reading back: the result
  int64_t y_b, y_r;
  const void* d;  // swiglu's backward pass: the gradient of its output
  int64_t d_r;
  int64_t rows, cols, groups;  // groups = batch * rows * blocks of a row
  uint32_t blocks;
  int32_t block_rows;
  float alpha, limit;
};

// Sixteen lanes have one block of a row, eight consecutive elements each.
struct Where {
  int64_t b, r;
  uint32_t c;  // the block
  int64_t col;  // the lane's first element
};
__device__ __forceinline__ Where locate(const RowsParams& p, int64_t g) {
  Where w;
  int64_t line;
  if (g < (int64_t)1 << 32) {
    line = (uint32_t)g / p.blocks;
  } else {
    line = g / p.blocks;
  }
  w.c = (uint32_t)(g - line * p.blocks);
  w.b = 0, w.r = line;
  if (line >= p.rows) {
    w.b = line / p.rows;
    w.r = line - w.b * p.rows;
  }
  w.col = (int64_t)w.c * kFp8Block + (threadIdx.x & 15) * 8;
  return w;
}

// The maximum over the block through the sixteen lanes, the scale from its bits, eight conversions.  (QUANT: without it swiglu alone.)
template <int DT, bool SWIGLU, bool QUANT>
__global__ __launch_bounds__(256) void fp8_rows_kernel(const RowsParams p) {
  for (int64_t g = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4); g < p.groups; g += (int64_t)gridDim.x * 16) {
    const Where w = locate(p, g);
    const int64_t at = w.b * p.x_b + w.r * p.x_r + w.col;
    const bool whole = w.col + 8 <= p.cols;
    float v[8];
    if (whole) {
      load_vec<DT, 8>(p.x, at, v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = w.col + i < p.cols ? load_elem<DT>(p.x, at + i) : 0.f;
    }
    if constexpr (SWIGLU) {
      float o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = swiglu_of<DT == TK_F32>(v[2 * i], v[2 * i + 1], p.alpha, p.limit);
      const int64_t to = w.r * p.y_r + w.col / 2;
      if (whole) {
        store_vec<DT, 4>(p.y, to, o);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (w.col + 2 * i < p.cols) store_elem<DT>(p.y, to + i, o[i]);
      }
    }
    if constexpr (!QUANT) continue;
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t u = finite_bits(v[i]);
      m = u > m ? u : m;
    }
    const float s = fp8_scale(max16(m)), inv = fp8_inverse(s);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = no_infinity(v[i]) * inv;
    const u32x2_t q = {to_e4m3(v[0], v[1], v[2], v[3]), to_e4m3(v[4], v[5], v[6], v[7])};
    uint8_t* out = p.v + w.b * p.v_b + w.r * p.v_r + w.col;
    if (whole) {
      store_wide(out, q);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (w.col + i < p.cols) out[i] = (uint8_t)(q[i >> 2] >> (i & 3) * 8);
    }
    if ((threadIdx.x & 15) == 0) p.s[w.b * p.s_b + w.r * p.s_r + (int64_t)w.c * p.s_c] = s;
  }
}

// Values times scale, rounded once.
template <int DT>
__global__ __launch_bounds__(256) void fp8_upcast_kernel(const RowsParams p) {
  for (int64_t g = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4); g < p.groups; g += (int64_t)gridDim.x * 16) {
    const Where w = locate(p, g);
    if (w.col >= p.cols) continue;
    const bool whole = w.col + 8 <= p.cols;
    const float s = p.s[w.b * p.s_b + (p.block_rows == 1 ? w.r : w.r / p.block_rows) * p.s_r + (int64_t)w.c * p.s_c];
    const uint8_t* from = p.v + w.b * p.v_b + w.r * p.v_r + w.col;
    u32x2_t q = {0, 0};
    if (whole) {
      q = load_wide<u32x2_t>(from);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (w.col + i < p.cols) q[i >> 2] |= (uint32_t)from[i] << (i & 3) * 8;
    }
    float v[8];
    from_e4m3(q[0], v), from_e4m3(q[1], v + 4);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= s;
    const int64_t to = w.b * p.y_b + w.r * p.y_r + w.col;
    if (whole) {
      store_vec<DT, 8>(p.y, to, v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (w.col + i < p.cols) store_elem<DT>(p.y, to + i, v[i]);
    }
  }
}

// d gate = d out (linear + 1) sigma (1 + alpha gate (1 - sigma)), d linear = d out gate sigma, none beyond the limit.
template <int DT>
__global__ __launch_bounds__(256) void swiglu_fp8_backward_kernel(const RowsParams p) {
  constexpr bool EXACT = DT == TK_F32;
  for (int64_t g = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4); g < p.groups; g += (int64_t)gridDim.x * 16) {
    const Where w = locate(p, g);
    if (w.col >= p.cols) continue;
    const bool whole = w.col + 8 <= p.cols;
    const float s = p.s[w.r * p.s_r + (int64_t)w.c * p.s_c];
    const uint8_t* from = p.v + w.r * p.v_r + w.col;
    const int64_t d_at = w.r * p.d_r + w.col / 2;
    u32x2_t q = {0, 0};
    float d[4];
    if (whole) {
      q = load_wide<u32x2_t>(from);
      load_vec<DT, 4>(p.d, d_at, d);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (w.col + i < p.cols) q[i >> 2] |= (uint32_t)from[i] << (i & 3) * 8;
#pragma unroll
      for (int i = 0; i < 4; ++i) d[i] = w.col + 2 * i < p.cols ? load_elem<DT>(p.d, d_at + i) : 0.f;
    }
    float v[8];
    from_e4m3(q[0], v), from_e4m3(q[1], v + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float gate0 = v[2 * i] * s, lin0 = v[2 * i + 1] * s;
      const float gate = at_most(gate0, p.limit), lin = at_least(at_most(lin0, p.limit), -p.limit);
      const Sigmoid t = sigmoid_of<EXACT>(p.alpha * gate);
      v[2 * i] = gate0 > p.limit ? 0.f : d[i] * (lin + 1.0f) * fmaf(p.alpha * gate, t.rest, 1.0f) * t.u * t.v;
      v[2 * i + 1] = fabsf(lin0) > p.limit ? 0.f : d[i] * gate * t.u * t.v;
    }
    const int64_t to = w.r * p.y_r + w.col;
    if (whole) {
      store_vec<DT, 8>(p.y, to, v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (w.col + i < p.cols) store_elem<DT>(p.y, to + i, v[i]);
    }
  }
}

// A workgroup has a block of 128 x 128: sixteen rows of sixteen lanes at a time, eight times; the converted block goes out in its own order and, through
// LDS, in the other one.
template <int DT>
__global__ __launch_bounds__(256) void fp8_tile_kernel(const RowsParams p, uint8_t* vt, int64_t t_b, int64_t t_c) {
  __shared__ uint32_t wave_max[4];
  __shared__ __attribute__((aligned(16))) uint8_t turned[128 * 132];
  const uint32_t row_blocks = (uint32_t)((p.rows + kFp8Block - 1) / kFp8Block);
  const int64_t id = blockIdx.x;
  const int64_t b = id / ((int64_t)row_blocks * p.blocks);
  const uint32_t in = (uint32_t)(id - b * row_blocks * p.blocks), rb = in / p.blocks, cb = in - rb * p.blocks;
  const int64_t row0 = (int64_t)rb * kFp8Block, col0 = (int64_t)cb * kFp8Block;
  const int lane = threadIdx.x & 15, line = threadIdx.x >> 4;
  const int64_t col = col0 + lane * 8;
  const bool whole = col + 8 <= p.cols;
  float v[8][8];
  uint32_t m = 0;
#pragma unroll
  for (int t = 0; t < 8; ++t) {
    const int64_t r = row0 + t * 16 + line;
    const int64_t at = b * p.x_b + r * p.x_r + col;
    if (r < p.rows && whole) {
      load_vec<DT, 8>(p.x, at, v[t]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[t][i] = r < p.rows && col + i < p.cols ? load_elem<DT>(p.x, at + i) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t u = finite_bits(v[t][i]);
      m = u > m ? u : m;
    }
  }
  m = max16(m);
  for (int step = 16; step < 64; step *= 2) {
    const uint32_t o = (uint32_t)__shfl_xor((int)m, step);
    m = o > m ? o : m;
  }
  if ((threadIdx.x & 63) == 0) wave_max[threadIdx.x >> 6] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) m = wave_max[i] > m ? wave_max[i] : m;
  const float s = fp8_scale(m), inv = fp8_inverse(s);
  if (threadIdx.x == 0) p.s[b * p.s_b + (int64_t)rb * p.s_r + (int64_t)cb * p.s_c] = s;
#pragma unroll
  for (int t = 0; t < 8; ++t) {
    const int64_t r = row0 + t * 16 + line;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[t][i] = no_infinity(v[t][i]) * inv;
    const u32x2_t q = {to_e4m3(v[t][0], v[t][1], v[t][2], v[t][3]), to_e4m3(v[t][4], v[t][5], v[t][6], v[t][7])};
    if (r < p.rows) {
      uint8_t* out = p.v + b * p.v_b + r * p.v_r + col;
      if (whole) {
        store_wide(out, q);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (col + i < p.cols) out[i] = (uint8_t)(q[i >> 2] >> (i & 3) * 8);
      }
    }
    if (vt) {
#pragma unroll
      for (int i = 0; i < 8; ++i) turned[(lane * 8 + i) * 132 + t * 16 + line] = (uint8_t)(q[i >> 2] >> (i & 3) * 8);
    }
  }
  if (!vt) return;
  __syncthreads();
  // row c of the turned block: eight bytes a lane, sixteen lanes
  for (int c = line; c < kFp8Block; c += 16) {
    if (col0 + c >= p.cols) break;
    const uint32_t* from = reinterpret_cast<const uint32_t*>(turned + c * 132 + lane * 8);
    const u32x2_t q = {from[0], from[1]};
    uint8_t* out = vt + b * t_b + (col0 + c) * t_c + row0 + lane * 8;
    if (row0 + lane * 8 + 8 <= p.rows) {
      store_wide(out, q);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (row0 + lane * 8 + i < p.rows) out[i] = (uint8_t)(q[i >> 2] >> (i & 3) * 8);
    }
  }
}

bool is_float(int dtype) { return dtype == TK_F32 || dtype == TK_BF16 || dtype == TK_F16; }
// Workgroups, sixteen blocks a turn.  Eight times as many as a CU has room for: those that run have work side by side in memory, and few turns each.  us, 8 a CU / 16 / 64 / one turn each: 16384 x 11520
// bf16 quantised 127 / 120 / 114 / 131, read back 110 / 109 / 101 / 108, swiglu's gradient 173 / 166 / 153 / 167; 16384 x 4096 fp32 read back 98 / 91 / 79 / 64.
unsigned groups_grid(int64_t groups) {
  const int64_t n = cdiv(groups, 16), most = (int64_t)device_cu_count() * 64;
  return (unsigned)(n < most ? n : most);
}

template <class F>
int32_t by_type(int dtype, F&& f) {
  switch (dtype) {
    case TK_F32:
      f(template_int<TK_F32>{});
      break;
    case TK_BF16:
      f(template_int<TK_BF16>{});
      break;
    default:
      f(template_int<TK_F16>{});
  }
  return TK_OK;
}

}  // namespace
}  // namespace tk

using namespace tk;

extern "C" int32_t tk_fp8_block_downcast(const void* x, int32_t dtype, int64_t batch, int64_t rows, int64_t cols, int64_t x_stride_b, int64_t x_stride_r,
                                         int32_t block_rows, uint8_t* values, int64_t v_stride_b, int64_t v_stride_r, uint8_t* values_t,
                                         int64_t t_stride_b, int64_t t_stride_c, float* scales, int64_t s_stride_b, int64_t s_stride_r, int64_t s_stride_c,
                                         tk_stream_t stream) {
  if (batch < 0 || rows < 0 || cols < 0) return fail(TK_ERR_INVALID, "tk_fp8_block_downcast: negative size");
  if (!is_float(dtype)) return fail(TK_ERR_UNSUPPORTED, "tk_fp8_block_downcast: x must be fp32, bf16 or fp16 (dtype %d)", dtype);
  if (block_rows != 1 && block_rows != kFp8Block) return fail(TK_ERR_UNSUPPORTED, "tk_fp8_block_downcast: blocks of 1 or 128 rows (got %d)", block_rows);
  if (values_t && block_rows == 1) return fail(TK_ERR_UNSUPPORTED, "tk_fp8_block_downcast: transposed values go with blocks of 128 rows");
  if (batch == 0 || rows == 0 || cols == 0) return TK_OK;
  if (!x || !values || !scales) return fail(TK_ERR_INVALID, "tk_fp8_block_downcast: null pointer");
  RowsParams p = {};
  p.x = x, p.x_b = x_stride_b, p.x_r = x_stride_r;
  p.v = values, p.v_b = v_stride_b, p.v_r = v_stride_r;
  p.s = scales, p.s_b = s_stride_b, p.s_r = s_stride_r, p.s_c = s_stride_c;
  p.rows = rows, p.cols = cols;
  if (cdiv(cols, kFp8Block) > 0x7FFFFFFF) return fail(TK_ERR_UNSUPPORTED, "tk_fp8_block_downcast: too many columns");
  p.blocks = (uint32_t)cdiv(cols, kFp8Block);
  p.groups = batch * rows * p.blocks;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (block_rows == 1) {
    by_type(dtype, [&](auto dt) { hipLaunchKernelGGL((fp8_rows_kernel<decltype(dt)::value, false, true>), dim3(groups_grid(p.groups)), dim3(256), 0, st, p); });
    return check_launch("fp8_rows_kernel");
  }
  const int64_t tiles = batch * cdiv(rows, kFp8Block) * p.blocks;
  if (tiles > 0x7FFFFFFF) return fail(TK_ERR_UNSUPPORTED, "tk_fp8_block_downcast: too many blocks");
  by_type(dtype, [&](auto dt) { hipLaunchKernelGGL(fp8_tile_kernel<decltype(dt)::value>, dim3((unsigned)tiles), dim3(256), 0, st, p, values_t, t_stride_b, t_stride_c); });
  return check_launch("fp8_tile_kernel");
}

extern "C" int32_t tk_fp8_block_upcast(const uint8_t* values, int64_t batch, int64_t rows, int64_t cols, int64_t v_stride_b, int64_t v_stride_r, int32_t block_rows,
                                       const float* scales, int64_t s_stride_b, int64_t s_stride_r, int64_t s_stride_c, void* out, int32_t out_dtype,
                                       int64_t o_stride_b, int64_t o_stride_r, tk_stream_t stream) {
  if (batch < 0 || rows < 0 || cols < 0) return fail(TK_ERR_INVALID, "tk_fp8_block_upcast: negative size");
  if (!is_float(out_dtype)) return fail(TK_ERR_UNSUPPORTED, "tk_fp8_block_upcast: the result is fp32, bf16 or fp16 (dtype %d)", out_dtype);
  if (block_rows != 1 && block_rows != kFp8Block) return fail(TK_ERR_UNSUPPORTED, "tk_fp8_block_upcast: blocks of 1 or 128 rows (got %d)", block_rows);
  if (batch == 0 || rows == 0 || cols == 0) return TK_OK;
  if (!values || !scales || !out) return fail(TK_ERR_INVALID, "tk_fp8_block_upcast: null pointer");
  RowsParams p = {};
  p.v = const_cast<uint8_t*>(values), p.v_b = v_stride_b, p.v_r = v_stride_r;
  p.s = const_cast<float*>(scales), p.s_b = s_stride_b, p.s_r = s_stride_r, p.s_c = s_stride_c;
  p.y = out, p.y_b = o_stride_b, p.y_r = o_stride_r;
  p.rows = rows, p.cols = cols, p.block_rows = block_rows;
  if (cdiv(cols, kFp8Block) > 0x7FFFFFFF) return fail(TK_ERR_UNSUPPORTED, "tk_fp8_block_upcast: too many columns");
  p.blocks = (uint32_t)cdiv(cols, kFp8Block);
  p.groups = batch * rows * p.blocks;
  by_type(out_dtype, [&](auto dt) { hipLaunchKernelGGL(fp8_upcast_kernel<decltype(dt)::value>, dim3(groups_grid(p.groups)), dim3(256), 0, static_cast<hipStream_t>(stream), p); });
  return check_launch("fp8_upcast_kernel");
}

extern "C" int32_t tk_swiglu_fp8(const void* a, int32_t dtype, int64_t M, int64_t n_out, int64_t a_stride_m, void* out, int64_t out_stride_m, uint8_t* values,
                                 int64_t v_stride_m, float* scales, int64_t s_stride_m, int64_t s_stride_c, float alpha, float limit, int32_t has_limit,
                                 tk_stream_t stream) {
  if (M < 0 || n_out < 0) return fail(TK_ERR_INVALID, "tk_swiglu_fp8: negative size");
  if (!is_float(dtype)) return fail(TK_ERR_UNSUPPORTED, "tk_swiglu_fp8: a must be fp32, bf16 or fp16 (dtype %d)", dtype);
  if (M == 0 || n_out == 0) return TK_OK;
  if (!a || !out || !values != !scales) return fail(TK_ERR_INVALID, "tk_swiglu_fp8: null pointer");
  RowsParams p = {};
  p.x = a, p.x_r = a_stride_m;
  p.v = values, p.v_r = v_stride_m;
  p.s = scales, p.s_r = s_stride_m, p.s_c = s_stride_c;
  p.y = out, p.y_r = out_stride_m;
  p.rows = M, p.cols = 2 * n_out;
  if (cdiv(p.cols, kFp8Block) > 0x7FFFFFFF) return fail(TK_ERR_UNSUPPORTED, "tk_swiglu_fp8: too many columns");
  p.blocks = (uint32_t)cdiv(p.cols, kFp8Block);
  p.groups = M * p.blocks;
  p.alpha = alpha, p.limit = has_limit ? limit : INFINITY;
  by_type(dtype, [&](auto dt) {
    auto kern = values ? fp8_rows_kernel<decltype(dt)::value, true, true> : fp8_rows_kernel<decltype(dt)::value, true, false>;
    hipLaunchKernelGGL(kern, dim3(groups_grid(p.groups)), dim3(256), 0, static_cast<hipStream_t>(stream), p);
  });
  return check_launch("fp8_rows_kernel");
}

extern "C" int32_t tk_swiglu_fp8_backward(const void* d_out, int32_t dtype, int64_t M, int64_t n_out, int64_t d_out_stride_m, const uint8_t* values,
                                          int64_t v_stride_m, const float* scales, int64_t s_stride_m, int64_t s_stride_c, void* d_a, int64_t d_a_stride_m,
                                          float alpha, float limit, int32_t has_limit, tk_stream_t stream) {
  if (M < 0 || n_out < 0) return fail(TK_ERR_INVALID, "tk_swiglu_fp8_backward: negative size");
  if (!is_float(dtype)) return fail(TK_ERR_UNSUPPORTED, "tk_swiglu_fp8_backward: gradients must be fp32, bf16 or fp16 (dtype %d)", dtype);
  if (M == 0 || n_out == 0) return TK_OK;
  if (!d_out || !values || !scales || !d_a) return fail(TK_ERR_INVALID, "tk_swiglu_fp8_backward: null pointer");
  RowsParams p = {};
  p.d = d_out, p.d_r = d_out_stride_m;
  p.v = const_cast<uint8_t*>(values), p.v_r = v_stride_m;
  p.s = const_cast<float*>(scales), p.s_r = s_stride_m, p.s_c = s_stride_c;
  p.y = d_a, p.y_r = d_a_stride_m;
  p.rows = M, p.cols = 2 * n_out;
  if (cdiv(p.cols, kFp8Block) > 0x7FFFFFFF) return fail(TK_ERR_UNSUPPORTED, "tk_swiglu_fp8_backward: too many columns");
  p.blocks = (uint32_t)cdiv(p.cols, kFp8Block);
  p.groups = M * p.blocks;
  p.alpha = alpha, p.limit = has_limit ? limit : INFINITY;
  by_type(dtype, [&](auto dt) { hipLaunchKernelGGL(swiglu_fp8_backward_kernel<decltype(dt)::value>, dim3(groups_grid(p.groups)), dim3(256), 0, static_cast<hipStream_t>(stream), p); });
  return check_launch("swiglu_fp8_backward_kernel");
}
