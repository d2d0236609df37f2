// The ragged product of e4m3 operands with one scale for each block of 128: the entry point, and the kernel for operands of any alignment.
//
// A block's sum is one MFMA (16 x 16 x 128) on a cleared accumulator; it is then added to the running sum times the row's and the weights' scale of the block: one fused
// operation for each accumulator register and block of K.  With the weights as the first operand a lane's registers are output columns of one row, so a lane needs
// one row scale a fragment, and the columns of a fragment share the weights' scale.
#include "fp8_blocks.h"

namespace tk {
namespace {

constexpr int kAnyRows = 64, kAnyCols = 64;

// 64 x 64 tiles, four waves of 32 x 32 (two fragments by two).  A block of K and its scales are asked for into registers a block ahead, and go from there into one of two buffers in LDS; four
// workgroups share a CU (the sixteen bit form of fp32 results leaves room for three).  us, this / three blocks ahead and two workgroups / one buffer and two barriers: three slices, 700 rows, K 1000, N
// 1023 10.2 / 10.5 / 14.0; 128 rows, K 4100, N 4096 24 / 25 / 37; 16 slices, 1000 rows, K 1000, N 4099 35 / 41 / 42.
template <int YT, bool SWIGLU>
__global__ __launch_bounds__(256, YT == TK_F32 ? 3 : 4) void fp8_block_any_kernel(const Fp8GemmParams p) {
  constexpr int PITCH = kFp8Block + 16, OPERAND = 64 * PITCH;
  static_assert(kAnyRows == 64 && kAnyCols == 64, "lines of an operand");
  __shared__ __attribute__((aligned(16))) uint8_t lds[2][2 * OPERAND];  // rows, columns
  fp8_zero_rest<YT, SWIGLU>(p);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int lr = lane & 15, g = lane >> 4, mw = wave & 1, nw = wave >> 1;
  const int tile_n = blockIdx.x % p.grid_n, tile_m = blockIdx.x / p.grid_n;
  int expert = 0, off_m = tile_m * kAnyRows, start_m = 0, eM = p.M;
  if (p.slice_sizes) {
    const int32_t where = p.block_sched[tile_m];
    if (where < 0) return;
    expert = where & 0xFFFF, off_m = (where >> 16) * kAnyRows;
    start_m = p.slice_offs[expert], eM = p.slice_sizes[expert];
  }
  if (off_m >= eM) return;
  const int n0 = tile_n * kAnyCols;
  const int piece = (tid & 7) * 16, line = tid >> 3;
  const uint8_t *x_row[2], *w_row[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int m = off_m + line + i * 32, n = n0 + line + i * 32;
    x_row[i] = w_row[i] = nullptr;
    if (m < eM) x_row[i] = p.x + (int64_t)(p.gather ? p.gather[start_m + m] : start_m + m) * p.x_stride_m;
    if (n < p.N) w_row[i] = p.w + expert * p.w_e + n * p.w_n;
  }
  const float* row_scale[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {  // (rows that are not there have the last one's)
    const int m = off_m + (j * 2 + mw) * 16 + lr, r = start_m + (m < eM ? m : eM - 1);
    row_scale[j] = p.xs + (int64_t)(p.gather ? p.gather[r] : r) * p.xs_m;
  }
  const int n_wave = n0 + nw * 32;
  const float* col_scale = p.ws + expert * p.ws_e + (int64_t)((n_wave < p.N ? n_wave : 0) / kFp8Block) * p.ws_n;

  const f32x4_t zero = {0.f, 0.f, 0.f, 0.f};
  f32x4_t acc[2][2] = {{zero, zero}, {zero, zero}};
  const int nb = (p.K + kFp8Block - 1) / kFp8Block;
  u32x4_t xr[2], wr[2];
  float sx[2], sc = 0.f, s[2];
  auto load = [&](int b) __attribute__((always_inline)) {
    if (b >= nb) return;
    const int k = b * kFp8Block + piece;
#pragma unroll
    for (int i = 0; i < 2; ++i) xr[i] = load_piece(x_row[i], k, p.K), wr[i] = load_piece(w_row[i], k, p.K);
#pragma unroll
    for (int j = 0; j < 2; ++j) sx[j] = row_scale[j][b * p.xs_k];
    sc = col_scale[b * p.ws_k];
  };
  load(0);
  for (int b = 0; b < nb; ++b) {
    uint8_t *xs = lds[b & 1], *ws = xs + OPERAND;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      *reinterpret_cast<u32x4_t*>(xs + (line + i * 32) * PITCH + piece) = xr[i];
      *reinterpret_cast<u32x4_t*>(ws + (line + i * 32) * PITCH + piece) = wr[i];
      s[i] = sx[i] * sc;
    }
    load(b + 1);
    // (one barrier a block: the buffer that is written next is the one that was read before it.  No wait for what is on its way from memory.)
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    i32x8_t a[2], c[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      __builtin_memcpy(&a[i], ws + (nw * 32 + i * 16 + lr) * PITCH + g * 32, 32);
      __builtin_memcpy(&c[i], xs + ((i * 2 + mw) * 16 + lr) * PITCH + g * 32, 32);
    }
#pragma unroll
    for (int f = 0; f < 2; ++f)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const f32x4_t part = YT == TK_F32 ? mfma_block_exact(a[f], c[j], zero) : mfma_block(a[f], c[j], zero);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[f][j][i] = fmaf(part[i], s[j], acc[f][j][i]);
      }
  }
  fp8_epilogue<YT, SWIGLU, 2, 2, 2>(p, acc, expert, off_m, start_m, eM, n_wave, p.N, mw, lane);
}

int32_t launch_any(Fp8GemmParams p, int yt, bool swiglu, hipStream_t st) {
  p.grid_n = (int)cdiv(p.N, kAnyCols);
  const int64_t grid = (int64_t)p.grid_m * p.grid_n;
  if (grid > 0x7FFFFFFF) return fail(TK_ERR_UNSUPPORTED, "tk_fp8_block_gemm: grid too large");
  auto launch = [&](auto kern) { hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(256), 0, st, p); };
  switch (yt) {
    case TK_F32:
      swiglu ? launch(fp8_block_any_kernel<TK_F32, true>) : launch(fp8_block_any_kernel<TK_F32, false>);
      break;
    case TK_BF16:
      swiglu ? launch(fp8_block_any_kernel<TK_BF16, true>) : launch(fp8_block_any_kernel<TK_BF16, false>);
      break;
    default:
      swiglu ? launch(fp8_block_any_kernel<TK_F16, true>) : launch(fp8_block_any_kernel<TK_F16, false>);
  }
  return check_launch("fp8_block_any_kernel");
}

// rows behind the slices alone: a call whose metadata have no row block
template <int YT, bool SWIGLU>
__global__ __launch_bounds__(256) void fp8_rest_kernel(const Fp8GemmParams p) {
  fp8_zero_rest<YT, SWIGLU>(p);
}
int32_t launch_rest(const Fp8GemmParams& p, int yt, bool swiglu, hipStream_t st) {
  auto launch = [&](auto kern) { hipLaunchKernelGGL(kern, dim3((unsigned)(p.M < 1024 ? p.M : 1024)), dim3(256), 0, st, p); };
  if (swiglu)
    yt == TK_F32 ? launch(fp8_rest_kernel<TK_F32, true>) : yt == TK_BF16 ? launch(fp8_rest_kernel<TK_BF16, true>) : launch(fp8_rest_kernel<TK_F16, true>);
  else
    yt == TK_F32 ? launch(fp8_rest_kernel<TK_F32, false>) : yt == TK_BF16 ? launch(fp8_rest_kernel<TK_BF16, false>) : launch(fp8_rest_kernel<TK_F16, false>);
  return check_launch("fp8_rest_kernel");
}

// What the kernels with memory-to-LDS transfers need: lines that begin at sixteen-byte boundaries, and offsets within a buffer resource (2 GiB) from the start of a
// tile, or of x and its scales where rows are gathered (beyond it such a call takes the kernel for any lines).
bool fp8_tiles_run(Fp8GemmParams& p, int64_t x_rows, int yt) {
  const int64_t limit = (int64_t)1 << 31, K16 = (p.K + 15) & ~15, blocks = cdiv(p.K, kFp8Block), rows = p.gather ? x_rows : 256;
  if (yt == TK_F32 || p.K == 0) return false;
  if ((reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.w) | (uint64_t)p.x_stride_m | (uint64_t)p.w_e | (uint64_t)p.w_n) & 15) return false;
  if (p.x_stride_m < 0 || p.w_n < 0 || p.xs_m < 0 || p.xs_k < 0 || p.ws_k < 0 || p.ws_n < 0) return false;
  const int64_t x_bytes = (rows - 1) * p.x_stride_m + K16;
  if (x_bytes >= limit || 255 * p.w_n + K16 >= limit) return false;
  if (((rows - 1) * p.xs_m + blocks * p.xs_k) * 4 >= limit || (p.ws_n + blocks * p.ws_k) * 4 >= limit) return false;
  p.x_bytes = (uint32_t)x_bytes;
  return true;
}

// Tiles of a size that a call is expected to have: every slice's last row block is half full (a single slice's is known).
int64_t expected_tiles(const Fp8GemmParams& p, int64_t slices, int64_t size) {
  return (p.slice_sizes ? cdiv(2 * p.M + slices * size, 2 * size) : cdiv(p.M, size)) * cdiv(p.N, size);
}

// Whether the kernel for few rows runs: it reads each column's weights once for 64 rows and each row once for 16 columns, and a CU takes about as long for 32 rows as for two workgroups of 16,
// so what decides is rows (16 for a slice that has fewer) times workgroups of columns (in brackets).  us (three numbers: rows, K, N of one slice; four: slices first),
// it / the ring (which runs beyond 32 rows a slice in any case): 1 4096 4096 (4096) 6.8 / 12.5; 4 40 560 896 (3584) 4.3 / 5.6; 32 4096 4096 (8192) 11.3 / 12.8; 1 4096 8192 (8192) 10.9 / 12.7; 2 64 7168 2048 (8192) 20.8 / 19.1; 512 16384 256 (8192) 53 / 36; 8 8 1024 1024 (8192) 4.7 / 7.1; 1 4096 14336 (14336)
// 18.7 / 13.8; 64 4096 4096 (16384) 17 / 12.9; 8 256 1024 1024 (16384) 10.9 / 6.9; 8 16 2048 2048 (16384) 8.8 / 9.0; 8 16 1024 4096 (32768) 9.9 / 7.9; 256 4096 4096 (65536) 62 / 14.3;
// it / `any`: 1 4100 4096 (4096) 8.1 / 23; 16 4100 16384 (16384) 22.5 / 24.8; 8 256 1000 1023 (16384) 9.8 / 10.1; 3 300 1000 1023 (19200) 9.8 / 10.2; 96 4100 4096 (24576) 23 / 25; 8 16 1000 4096 (32768)
// 12.5 / 10.3; 128 4100 4096 (32768) 27.9 / 25.4; 3 700 1000 1023 (44800) 15.6 / 10.5.
bool few_rows_run(const Fp8GemmParams& p, int64_t slices, bool dma) {
  const int64_t in_use = slices < p.M ? slices : p.M, rows = p.M > 16 * in_use ? p.M : 16 * in_use;
  return dma ? p.M <= 32 * in_use && rows * cdiv(p.N, 16) <= 8192 : rows * cdiv(p.N, 16) <= 24576;
}

// Size of the tiles: 64 (the ring), 128 or 256, whichever is expected to take the least time.  A round of tiles (of 64 and 128 two a CU, of 256 one) takes the time of its blocks of K and
// of a start and an end, in us (fitted to what is measured below).  With up to 16 rows a slice the weights' stream is all that counts, which the ring keeps up best.
// us, 64 / 128 / 256 (a name of three numbers: rows, K and N of one slice; of four: slices first): 64 4096 4096 12.9 / 32.6 / 58.9; 256 4096 4096 14.3 / 33.6 / 61; 512 4096 4096 21.3 / 38 / 68; 1024 4096 4096 40.1 / 41.2 / 72;
// 2048 4096 4096 86 / 50 / 76; 4096 4096 4096 - / 91 / 80; 1024 2048 2048 12.9 / 21 / 37; 2048 2048 2048 25.2 / 23.4 / 42; 4096 512 2048 21 / 16 / 20.6; 8 512 1024 1024 7.2 / 14.1 / 22.6; 8 1024 1024 1024 8.6 / 14.3 / 24.2; 8 2048
// 1024 1024 14 / 14.7 / 24.5; 8 4096 1024 1024 22 / 18.3 / 25.4; 8 800 608 7296 26 / 23.1 / 23; 8 294 640 7312 17.5 / 14.5 / 19.4; 8 64 4096 4096 22.6 / 36.5 / 60; 32 128 2880 5760 90 / 113 / -; 32 512 2880 5760
// 120 / 131 / 158; 32 1024 2880 5760 148 / 139 / 166; 32 2048 2880 2880 90 / 82 / 104; 32 4096 2880 2880 147 / 110 / 118; 8 4096 2880 2880 - / 70 / 62.
int tile_size(const Fp8GemmParams& p, int64_t slices, int64_t cus) {
  if (p.M <= slices * 16) return 64;
  const int64_t n64 = (int64_t)p.grid_m * cdiv(p.N, 64), n128 = expected_tiles(p, slices, 128), n256 = expected_tiles(p, slices, 256);
  const double blocks = (double)cdiv(p.K, kFp8Block);
  const double t64 = n64 <= cus ? 0.36 * blocks + 4.3 : (double)cdiv(n64, 2 * cus) * (0.56 * blocks + 3.4);
  const double t128 = n128 <= cus / 2 ? 0.8 * blocks + 8 : (double)cdiv(n128, 2 * cus) * (1.3 * blocks + 6) + 6;
  const double t256 = (double)cdiv(n256, cus) * (2.1 * blocks + 6) + 6;
  return t64 <= t128 && t64 <= t256 ? 64 : t128 <= t256 ? 128 : 256;
}

// The kernels' numbers as the host check hook has them; tiles go by their size.
enum { kNothing = 0, kAny = 1, kRest = 2, kFew = 16, kRing64 = 64 };

// Checks a call and chooses its kernel, on a card with `cus` compute units.
int32_t plan(const tk_fp8_gemm_desc* d, int64_t cus, Fp8GemmParams& p, int32_t& kernel) {
  kernel = kNothing;
  if (!d) return fail(TK_ERR_INVALID, "tk_fp8_block_gemm: null descriptor");
  if (d->M < 0 || d->N < 0 || d->K < 0 || d->n_slices < 0 || d->grid_m < 0) return fail(TK_ERR_INVALID, "tk_fp8_block_gemm: negative size");
  if (d->M > kFp8Most || d->N > kFp8Most || d->K > kFp8Most) return fail(TK_ERR_UNSUPPORTED, "tk_fp8_block_gemm: sizes up to %d (got %d x %d x %d)", kFp8Most, d->M, d->K, d->N);
  if (d->y_dtype != TK_F32 && d->y_dtype != TK_BF16 && d->y_dtype != TK_F16) return fail(TK_ERR_UNSUPPORTED, "tk_fp8_block_gemm: the output is fp32, bf16 or fp16 (dtype %d)", d->y_dtype);
  if (d->activation != TK_ACT_NONE && d->activation != TK_ACT_SWIGLU) return fail(TK_ERR_INVALID, "tk_fp8_block_gemm: bad activation %d", d->activation);
  const bool swiglu = d->activation == TK_ACT_SWIGLU;
  if (swiglu && d->N % 2) return fail(TK_ERR_INVALID, "tk_fp8_block_gemm: swiglu needs an even number of columns (got %d)", d->N);
  if (d->bias && d->bias_dtype != TK_F32 && d->bias_dtype != TK_BF16) return fail(TK_ERR_UNSUPPORTED, "tk_fp8_block_gemm: the bias is fp32 or bf16 (dtype %d)", d->bias_dtype);
  if (d->gammas && d->gammas_dtype != TK_F32 && d->gammas_dtype != TK_BF16) return fail(TK_ERR_UNSUPPORTED, "tk_fp8_block_gemm: gammas are fp32 or bf16 (dtype %d)", d->gammas_dtype);
  if (d->M == 0 || d->N == 0) return TK_OK;
  if (!d->y || (d->K > 0 && (!d->x || !d->x_scale || (d->n_slices > 0 && (!d->w || !d->w_scale))))) return fail(TK_ERR_INVALID, "tk_fp8_block_gemm: null operand");
  if (d->slice_sizes) {
    if (!d->slice_offs || !d->block_schedule) return fail(TK_ERR_INVALID, "tk_fp8_block_gemm: slices need their offsets and block schedule");
    if (d->n_slices > 0xFFFF) return fail(TK_ERR_UNSUPPORTED, "tk_fp8_block_gemm: up to 65535 slices (got %d)", d->n_slices);
  } else if (d->n_slices != 1) {
    return fail(TK_ERR_INVALID, "tk_fp8_block_gemm: %d slices without their sizes", d->n_slices);
  }
  p = Fp8GemmParams{};
  p.x = d->x, p.x_stride_m = d->x_stride_m, p.xs = d->x_scale, p.xs_m = d->xs_stride_m, p.xs_k = d->xs_stride_k;
  p.w = d->w, p.w_e = d->w_stride_e, p.w_n = d->w_stride_n;
  p.ws = d->w_scale, p.ws_e = d->ws_stride_e, p.ws_k = d->ws_stride_k, p.ws_n = d->ws_stride_n;
  p.bias = d->bias, p.bias_e = d->bias_stride_e, p.bias_is_f32 = d->bias_dtype == TK_F32;
  p.gather = d->gather_indx, p.scatter = d->scatter_indx, p.scatter_len = d->scatter_len;
  p.gammas = d->gammas, p.gammas_is_f32 = d->gammas_dtype == TK_F32;
  p.slice_sizes = d->slice_sizes, p.slice_offs = d->slice_offs, p.block_sched = d->block_schedule;
  p.n_slices = d->n_slices, p.grid_m = d->slice_sizes ? d->grid_m : (int)cdiv(d->M, kAnyRows);
  p.M = d->M, p.N = d->N, p.K = d->K;
  p.y = d->y, p.y_stride_m = d->y_stride_m;
  p.alpha = d->act_alpha, p.limit = d->act_has_limit ? d->act_limit : INFINITY;
  p.zero_rest = d->zero_rest, p.pow2 = d->pow2_scales;
  if (p.grid_m == 0) {
    kernel = p.zero_rest ? kRest : kNothing;
    return TK_OK;
  }
  const int64_t slices = d->slice_sizes ? d->n_slices : 1;
  const bool dma = fp8_tiles_run(p, d->x_rows, d->y_dtype);
  // A schedule has 15 bits for a row block of 64: a slice that may have more goes by tiles, which need none.
  const bool long_slices = d->slice_sizes && d->M > (1 << 15) * kAnyRows;
  if (long_slices && !(dma && slices <= kDmaSlices))
    return fail(TK_ERR_UNSUPPORTED, "tk_fp8_block_gemm: more than %d rows in slices need 16-bit results, up to %d slices, operands whose lines begin at sixteen-byte boundaries and, where rows are gathered, less than 2 GiB to gather from (got %d rows)",
                (1 << 15) * kAnyRows, kDmaSlices, d->M);
  if (few_rows_run(p, slices, dma)) {
    kernel = kFew;
  } else if (!dma) {
    kernel = kAny;
  } else {
    const int tile = tile_size(p, slices, cus);
    kernel = (tile == 64 && !long_slices) || slices > kDmaSlices ? kRing64 : tile == 256 ? 256 : 128;
  }
  return TK_OK;
}

}  // namespace
}  // namespace tk

using namespace tk;

extern "C" int32_t tk_fp8_block_gemm(const tk_fp8_gemm_desc* d, tk_stream_t stream) {
  Fp8GemmParams p;
  int32_t kernel;
  if (const int32_t rc = plan(d, device_cu_count(), p, kernel)) return rc;
  const bool swiglu = kernel != kNothing && d->activation == TK_ACT_SWIGLU;
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (kernel) {
    case kNothing:
      return TK_OK;
    case kRest:
      return launch_rest(p, d->y_dtype, swiglu, st);
    case kAny:
      return launch_any(p, d->y_dtype, swiglu, st);
    case kFew:
      return fp8_gemm_launch_few(p, ((reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.w) | (uint64_t)p.x_stride_m | (uint64_t)p.w_e | (uint64_t)p.w_n) & 15) == 0, d->y_dtype, swiglu, st);
    case kRing64:
      return fp8_gemm_launch_ring(p, d->y_dtype, swiglu, st);
    default:
      return fp8_gemm_launch_tiles(p, kernel, d->y_dtype, swiglu, st);
  }
}

extern "C" int32_t tk_host_fp8_block_gemm_kernel(const tk_fp8_gemm_desc* d, int32_t cus, int32_t* kernel) {
  if (!kernel || cus <= 0) return fail(TK_ERR_INVALID, "tk_host_fp8_block_gemm_kernel: bad argument");
  Fp8GemmParams p;
  return plan(d, cus, p, *kernel);
}
