// The ragged product of e4m3 operands with one scale for each block of 128, few rows: what takes the time is the stream of the weights.
//
//   * A workgroup has 16 columns of the weights and up to 64 rows of a slice (a block of the schedule); its eight waves take every eighth block of K, and their
//     sums are joined in LDS in the waves' order.  So a single row spreads 4096 columns over 256 workgroups, and a wave has all of its share of K = 4096 in flight at once.
//   * Operands go from memory into registers as the matrix instruction wants them: a lane's 32 consecutive k of one column are a quarter of a cache line, and four
//     lanes have the whole.
//   * us: one row, 4096 x 4096 6.8 (2.5 TB/s of weights; an empty kernel takes 2), eight experts of a row, 1024 x 1024 4.7.
#include "fp8_blocks.h"

namespace tk {
namespace {

constexpr int kFewCols = 16, kFewRows = 64, kFewWaves = 8;

// ALIGNED: lines begin at sixteen-byte boundaries
template <bool ALIGNED>
__device__ __forceinline__ i32x8_t load_frag(const uint8_t* line, int k, int K) {
  u32x4_t lo, hi;
  if (ALIGNED && k + 32 <= K) {
    lo = *reinterpret_cast<const u32x4_t*>(line + k), hi = *reinterpret_cast<const u32x4_t*>(line + k + 16);
  } else {
    lo = load_piece(line, k, K), hi = load_piece(line, k + 16, K);
  }
  return __builtin_bit_cast(i32x8_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

// MF row fragments of 16 (the last rows of which need not be there)
template <int YT, bool SWIGLU, bool ALIGNED, int MF>
__device__ __forceinline__ void few_rows(const Fp8GemmParams& p, float* sums, int expert, int off_m, int start_m, int eM, int n0) {
  constexpr int DEPTH = MF == 1 ? 4 : 2;  // blocks of K in flight a wave
  const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nb = (p.K + kFp8Block - 1) / kFp8Block;
  // (columns and rows that are not there read the last one's; nobody writes them)
  const int n = n0 + lr < p.N ? n0 + lr : p.N - 1;
  const uint8_t* w_line = p.w + expert * p.w_e + n * p.w_n;
  const float* w_scale = p.ws + expert * p.ws_e + (int64_t)(n0 / kFp8Block) * p.ws_n;
  const uint8_t* x_line[MF];
  const float* x_scale[MF];
#pragma unroll
  for (int j = 0; j < MF; ++j) {
    int m = off_m + j * 16 + lr;
    m = start_m + (m < eM ? m : eM - 1);
    const int64_t src = p.gather ? p.gather[m] : m;
    x_line[j] = p.x + src * p.x_stride_m, x_scale[j] = p.xs + src * p.xs_m;
  }
  const f32x4_t zero = {0.f, 0.f, 0.f, 0.f};
  f32x4_t acc[MF];
#pragma unroll
  for (int j = 0; j < MF; ++j) acc[j] = zero;
  i32x8_t w[DEPTH], x[DEPTH][MF];
  float sw[DEPTH], sx[DEPTH][MF];
  auto load = [&](int d, int b) __attribute__((always_inline)) {
    if (b >= nb) return;  // (uniform)
    const int k = b * kFp8Block + g * 32;
    w[d] = load_frag<ALIGNED>(w_line, k, p.K);
    sw[d] = w_scale[b * p.ws_k];
#pragma unroll
    for (int j = 0; j < MF; ++j) {
      x[d][j] = load_frag<ALIGNED>(x_line[j], k, p.K);
      sx[d][j] = x_scale[j][b * p.xs_k];
    }
  };
#pragma unroll
  for (int d = 0; d < DEPTH; ++d) load(d, wave + d * kFewWaves);
  for (int b0 = wave; b0 < nb; b0 += DEPTH * kFewWaves) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      const int b = b0 + d * kFewWaves;
      if (b >= nb) break;
#pragma unroll
      for (int j = 0; j < MF; ++j) {
        const f32x4_t part = YT == TK_F32 ? mfma_block_exact(w[d], x[d][j], zero) : mfma_block(w[d], x[d][j], zero);
        const float s = sx[d][j] * sw[d];
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[j][i] = fmaf(part[i], s, acc[j][i]);
      }
      load(d, b + DEPTH * kFewWaves);
    }
  }
  // sums[wave][row][column], columns side by side
#pragma unroll
  for (int j = 0; j < MF; ++j) *reinterpret_cast<f32x4_t*>(sums + (wave * MF * 16 + j * 16 + lr) * kFewCols + g * 4) = acc[j];
  __syncthreads();
  // a thread has two columns of a row
  const int r = tid >> 3, c = (tid & 7) * 2, row = off_m + r, col = n0 + c;
  if (r >= MF * 16 || row >= eM || col >= p.N) return;
  float v[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < kFewWaves; ++i) {
    const f32x2_t s = *reinterpret_cast<const f32x2_t*>(sums + (i * MF * 16 + r) * kFewCols + c);
    v[0] += s[0], v[1] += s[1];
  }
  const int src = start_m + row;
  int dst = src;
  if (p.scatter) dst = src < p.scatter_len ? p.scatter[src] : -1;
  if (dst < 0) return;
  const bool two = col + 1 < p.N;
  if (p.bias) {
    v[0] += load_scalar(p.bias, expert * p.bias_e + col, p.bias_is_f32);
    if (two) v[1] += load_scalar(p.bias, expert * p.bias_e + col + 1, p.bias_is_f32);
  }
  const float gam = p.gammas ? load_scalar(p.gammas, src, p.gammas_is_f32) : 1.0f;
  const int64_t to = dst * p.y_stride_m;
  if constexpr (SWIGLU) {
    store_elem<YT>(p.y, to + col / 2, swiglu_of<YT == TK_F32>(v[0], v[1], p.alpha, p.limit) * gam);
  } else {
    store_elem<YT>(p.y, to + col, v[0] * gam);
    if (two) store_elem<YT>(p.y, to + col + 1, v[1] * gam);
  }
}

// ONE: no slice has more than 16 rows; two workgroups share a CU then (the compiler moves up to 19 of the registers to memory for it, before and after the loop), where
// the registers for 64 rows allow one
template <int YT, bool SWIGLU, bool ALIGNED, bool ONE>
__global__ __launch_bounds__(kFewWaves * 64, ONE ? 4 : 2) void fp8_block_few_kernel(const Fp8GemmParams p) {
  __shared__ __attribute__((aligned(16))) float sums[kFewWaves * (ONE ? 16 : kFewRows) * kFewCols];
  fp8_zero_rest<YT, SWIGLU>(p);
  const int tile_m = blockIdx.x / p.grid_n, n0 = (blockIdx.x - tile_m * p.grid_n) * kFewCols;
  int expert = 0, off_m = tile_m * kFewRows, start_m = 0, eM = p.M;
  if (p.slice_sizes) {
    const int32_t where = p.block_sched[tile_m];
    if (where < 0) return;
    expert = where & 0xFFFF, off_m = (where >> 16) * kFewRows;
    start_m = p.slice_offs[expert], eM = p.slice_sizes[expert];
  }
  if (off_m >= eM) return;
  const int rows = eM - off_m;
  if (ONE || rows <= 16)
    few_rows<YT, SWIGLU, ALIGNED, 1>(p, sums, expert, off_m, start_m, eM, n0);
  else if constexpr (!ONE) {
    if (rows <= 32)
      few_rows<YT, SWIGLU, ALIGNED, 2>(p, sums, expert, off_m, start_m, eM, n0);
    else
      few_rows<YT, SWIGLU, ALIGNED, 4>(p, sums, expert, off_m, start_m, eM, n0);
  }
}

}  // namespace

int32_t fp8_gemm_launch_few(const Fp8GemmParams& q, bool aligned, int yt, bool swiglu, hipStream_t st) {
  Fp8GemmParams p = q;
  p.grid_n = (int)cdiv(p.N, kFewCols);
  const int64_t grid = (int64_t)p.grid_m * p.grid_n;
  if (grid > 0x7FFFFFFF) return fail(TK_ERR_UNSUPPORTED, "tk_fp8_block_gemm: grid too large");
  auto go = [&](auto kern) -> int32_t {
    hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(kFewWaves * 64), 0, st, p);
    return check_launch("fp8_block_few_kernel");
  };
  auto by_rows = [&](auto yt_c, auto swiglu_c, auto aligned_c) -> int32_t {
    constexpr int YT = decltype(yt_c)::value;
    constexpr bool SWIGLU = decltype(swiglu_c)::value, ALIGNED = decltype(aligned_c)::value;
    return p.M <= 16 ? go(fp8_block_few_kernel<YT, SWIGLU, ALIGNED, true>) : go(fp8_block_few_kernel<YT, SWIGLU, ALIGNED, false>);
  };
  auto by_type = [&](auto yt_c) -> int32_t {
    if (swiglu) return aligned ? by_rows(yt_c, std::true_type{}, std::true_type{}) : by_rows(yt_c, std::true_type{}, std::false_type{});
    return aligned ? by_rows(yt_c, std::false_type{}, std::true_type{}) : by_rows(yt_c, std::false_type{}, std::false_type{});
  };
  return yt == TK_F32 ? by_type(template_int<TK_F32>{}) : yt == TK_BF16 ? by_type(template_int<TK_BF16>{}) : by_type(template_int<TK_F16>{});
}

}  // namespace tk
