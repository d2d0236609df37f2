// The ragged product of e4m3 operands with one scale for each block of 128, small and middle sizes and few rows of many experts: 64 x 64 tiles on a ring of stages.
//
//   * What takes the time here is a stage's way from memory, so stages are small (64 rows and 64 columns of a block of K, with their scales) and many: four of them are in
//     LDS, three on their way while the next one is read from it, and two workgroups share a CU.  (Eight stages and one workgroup: no change.)
//   * Four waves of 32 x 32, four products of 16 x 16 each a stage, added to the running sums times the scales as in the kernel for large tiles.  A stage's operands are read from
//     LDS behind the products of the one before.  One barrier a stage: behind it the next stage has landed and this one has been read, so its buffer is filled again.
//   * Where there is a workgroup a CU at most and K is long, a workgroup has two such groups of four waves with a ring each, which take every other block of K.
//   * Each wave makes the same number of transfers a stage (two of rows, two of columns, one of scales), so that one count of those in flight holds for all.
//   * Row blocks of a slice that share columns run next to each other on one XCD.
//   * us: one slice of 64 to 256 rows, 4096 x 4096 13 to 14 (64 to 256 workgroups that each take in 50 GB/s, as a CU does however its stages are cut); 32 experts, 128 rows, K 2880, N 5760 with swiglu 89 (6 TB/s: HBM and the last-level
//     cache); eight, 512 rows, 1024 x 1024 7.1.
#include "fp8_blocks.h"
#include "gemm_tiles.h"

namespace tk {
namespace {

constexpr int kRingTile = 64, kRingOperand = kRingTile * kFp8Block, kRingScales = 512, kRingStage = 2 * kRingOperand + kRingScales;
constexpr int kRing = 4, kRingLds = kRing * kRingStage, kRingTransfers = 5;  // stages; transfers of a wave and stage
static_assert(kRingLds <= 80 * 1024, "two workgroups of a CU");

// KG groups of four waves: a stage is KG blocks of K, one for each group, and their sums are joined in the groups' order.
template <int YT, bool SWIGLU, int KG>
__global__ __launch_bounds__(256 * KG, 2) void fp8_block_ring_kernel(const Fp8GemmParams p) {
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  fp8_zero_rest<YT, SWIGLU>(p);
  const int id = xcd_remap((int)blockIdx.x, (int)gridDim.x);
  const int tile_n = id / p.grid_m, tile_m = id - tile_n * p.grid_m, n0 = tile_n * kRingTile;
  int expert = 0, off_m = tile_m * kRingTile, start_m = 0, eM = p.M;
  if (p.slice_sizes) {
    const int32_t where = p.block_sched[tile_m];
    if (where < 0) return;
    expert = where & 0xFFFF, off_m = (where >> 16) * kRingTile;
    start_m = p.slice_offs[expert], eM = p.slice_sizes[expert];
  }
  if (off_m >= eM) return;
  const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, g4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6) & 3, group = KG == 1 ? 0 : __builtin_amdgcn_readfirstlane(tid >> 8);
  const int mw = wave & 1, nw = wave >> 1;
  const int nb = (p.K + kFp8Block - 1) / kFp8Block, nst = (nb + KG - 1) / KG, tail = p.K & 15;
  const uint32_t mine = (uint32_t)group * kRingLds, lds0 = lds_addr(lds) + mine;
  const int rows = eM - off_m < kRingTile ? eM - off_m : kRingTile, cols = p.N - n0 < kRingTile ? p.N - n0 : kRingTile, first = start_m + off_m;

  // ---- transfers: eight lines each, as in the kernel for large tiles (lane -> line lane / 8, piece (lane % 8) ^ (line >> 1 & 7)) ------------------------------
  const uint32_t K16 = (uint32_t)((p.K + 15) & ~15), x_row = (uint32_t)p.x_stride_m, w_row = (uint32_t)p.w_n;
  const buf_desc_t xdesc = p.gather ? make_buf_desc(p.x, p.x_bytes) : make_buf_desc(p.x + first * p.x_stride_m, (uint32_t)(rows - 1) * x_row + K16);
  const buf_desc_t wdesc = make_buf_desc(p.w + (int64_t)expert * p.w_e + (int64_t)n0 * p.w_n, (uint32_t)(cols - 1) * w_row + K16);
  const int pc[2] = {(lane & 7) ^ (lane >> 4), (lane & 7) ^ (lane >> 4) ^ 4};
  uint32_t x_off[2], w_off[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int line = (wave * 2 + i) * 8 + (lane >> 3);
    const uint32_t src = line < rows ? (p.gather ? (uint32_t)p.gather[first + line] : (uint32_t)line) : 0u;
    x_off[i] = line < rows ? src * x_row + pc[i] * 16u : kOutOfRange;
    w_off[i] = line < cols ? (uint32_t)line * w_row + pc[i] * 16u : kOutOfRange;
  }
  // the even waves fetch the rows' scales, the odd ones the columns' (of which there is one block)
  buf_desc_t sdesc;
  uint32_t s_off, s_step;
  if (wave & 1) {
    sdesc = make_buf_desc(p.ws + (int64_t)expert * p.ws_e + (int64_t)(n0 / kFp8Block) * p.ws_n, 0x7FFFFFFFu);
    s_off = 0, s_step = (uint32_t)p.ws_k * 4u;
  } else {
    const uint32_t src = lane < rows ? (p.gather ? (uint32_t)p.gather[first + lane] : (uint32_t)lane) : 0u;
    sdesc = make_buf_desc(p.gather ? p.xs : p.xs + first * p.xs_m, 0x7FFFFFFFu);
    s_off = lane < rows ? src * (uint32_t)p.xs_m * 4u : kOutOfRange, s_step = (uint32_t)p.xs_k * 4u;
  }
  auto fetch = [&](int s) __attribute__((always_inline)) {
    const uint32_t at = lds0 + (uint32_t)(s % kRing) * kRingStage;
    const int k = (s * KG + group) * kFp8Block;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const bool in = k + pc[i] * 16 < p.K;  // (none behind the last block)
      lds_dma16(wdesc, at + kRingOperand + (wave * 2 + i) * 1024, in ? w_off[i] + (uint32_t)k : kOutOfRange);
      lds_dma16(xdesc, at + (wave * 2 + i) * 1024, in ? x_off[i] + (uint32_t)k : kOutOfRange);
    }
    lds_dma4(sdesc, at + 2 * kRingOperand + (wave & 1) * 256, k < p.K ? s_off + (uint32_t)(s * KG + group) * s_step : kOutOfRange);
  };

  // ---- LDS read side --------------------------------------------------------------------------------------------------------------------------------------
  const int sw = (lr >> 1) & 7;
  const uint32_t pos0 = (uint32_t)(((2 * g4) ^ sw) * 16 + lr * 128), pos1 = (uint32_t)(((2 * g4 + 1) ^ sw) * 16 + lr * 128);
  auto ld = [&](uint32_t at) __attribute__((always_inline)) -> u32x4_t { return *reinterpret_cast<const u32x4_t*>(lds + at); };
  auto frag = [&](uint32_t at) __attribute__((always_inline)) -> i32x8_t {
    return __builtin_bit_cast(i32x8_t, __builtin_shufflevector(ld(at + pos0), ld(at + pos1), 0, 1, 2, 3, 4, 5, 6, 7));
  };
  auto barrier = [&]() __attribute__((always_inline)) {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  // clears what the last piece of each line of the last block holds past K
  auto clear_tail = [&](uint32_t at) __attribute__((always_inline)) {
    at += (uint32_t)((nb - 1) % KG) * kRingLds;
    if (tid < 2 * kRingTile) {
      const int l = tid & 63, piece = ((p.K % kFp8Block) >> 4) ^ ((l >> 1) & 7);
      uint8_t* last = lds + at + (tid >> 6) * kRingOperand + l * 128 + piece * 16;
      u32x4_t v = *reinterpret_cast<const u32x4_t*>(last);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int keep = tail - 4 * i;  // bytes of this word
        v[i] = keep >= 4 ? v[i] : keep <= 0 ? 0u : v[i] & ((1u << 8 * keep) - 1u);
      }
      *reinterpret_cast<u32x4_t*>(last) = v;
    }
    barrier();
  };
  i32x8_t w[2], x[2];
  float sx[2], sc;
  auto read = [&](int s) __attribute__((always_inline)) {
    const uint32_t at = mine + (uint32_t)(s % kRing) * kRingStage;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      w[i] = frag(at + kRingOperand + (uint32_t)((nw * 2 + i) * 2048));
      x[i] = frag(at + (uint32_t)((i * 2 + mw) * 2048));
      sx[i] = *reinterpret_cast<const float*>(lds + at + 2 * kRingOperand + ((i * 2 + mw) * 16 + lr) * 4);
    }
    sc = *reinterpret_cast<const float*>(lds + at + 2 * kRingOperand + 256);
  };
#pragma unroll
  for (int s = 0; s < kRing; ++s) fetch(s);
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"((kRing - 1) * kRingTransfers) : "memory");
  barrier();
  if (tail && nst == 1) clear_tail(0);
  read(0);
  const f32x4_t zero = {0.f, 0.f, 0.f, 0.f};
  f32x4_t acc[2][2] = {{zero, zero}, {zero, zero}};
#pragma unroll 1
  for (int s = 0; s < nst; ++s) {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((kRing - 2) * kRingTransfers) : "memory");
    barrier();
    fetch(s + kRing);
    if (tail && s + 2 == nst) clear_tail((uint32_t)((s + 1) % kRing) * kRingStage);
    f32x4_t part[2][2];
    const float scale[2] = {sx[0] * sc, sx[1] * sc};
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        part[f][j] = mfma_block(w[f], x[j], zero);
        asm volatile("" : "+v"(part[f][j]));  // (an empty use: the products stay in front of the reads, which take their operands' registers)
      }
    __builtin_amdgcn_sched_barrier(0);
    read(s + 1);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int f = 0; f < 2; ++f)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[f][j][i] = fmaf(part[f][j][i], scale[j], acc[f][j][i]);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (the last transfers write into this workgroup's LDS)
  if constexpr (KG > 1) {
    barrier();
    f32x4_t* sums = reinterpret_cast<f32x4_t*>(lds) + (tid & 255);
    if (group > 0) {
#pragma unroll
      for (int f = 0; f < 4; ++f) sums[((group - 1) * 4 + f) * 256] = acc[f >> 1][f & 1];
    }
    barrier();
    if (group > 0) return;
#pragma unroll
    for (int g = 0; g < KG - 1; ++g)
#pragma unroll
      for (int f = 0; f < 4; ++f) acc[f >> 1][f & 1] += sums[(g * 4 + f) * 256];
  }
  fp8_epilogue<YT, SWIGLU, 2, 2, 2>(p, acc, expert, off_m, start_m, eM, n0 + nw * 32, p.N, mw, lane);
}

}  // namespace

int32_t fp8_gemm_launch_ring(const Fp8GemmParams& q, int yt, bool swiglu, hipStream_t st) {
  Fp8GemmParams p = q;
  p.grid_n = (int)cdiv(p.N, kRingTile);
  const int64_t grid = (int64_t)p.grid_m * p.grid_n;
  if (grid > 0x7FFFFFFF) return fail(TK_ERR_UNSUPPORTED, "tk_fp8_block_gemm: grid too large");
  // A workgroup a CU at most, and long chains of stages: two groups.  us, two / one: 64 rows, 4096 x 4096 12.9 / 14.8; 256 rows 14.3 / 15.7; 512 rows, 2048 x 2048 9.8 / 10.1; K 16384, N 256 36 / 46; but
  // eight slices, 256 rows, 1024 x 1024 7.1 / 6.9; 2048 rows, 512 x 512 6.3 / 5.8.
  const int groups = grid <= device_cu_count() && p.K >= 16 * kFp8Block ? 2 : 1;
  auto go = [&](auto kern, int groups) -> int32_t {
    if (const int32_t rc = allow_dynamic_lds(reinterpret_cast<const void*>(kern), groups * kRingLds)) return rc;
    hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(256 * groups), groups * kRingLds, st, p);
    return check_launch("fp8_block_ring_kernel");
  };
  auto by_groups = [&](auto yt_c, auto swiglu_c) -> int32_t {
    constexpr int YT = decltype(yt_c)::value;
    constexpr bool SWIGLU = decltype(swiglu_c)::value;
    return groups == 2 ? go(fp8_block_ring_kernel<YT, SWIGLU, 2>, 2) : go(fp8_block_ring_kernel<YT, SWIGLU, 1>, 1);
  };
  if (yt == TK_BF16) return swiglu ? by_groups(template_int<TK_BF16>{}, std::true_type{}) : by_groups(template_int<TK_BF16>{}, std::false_type{});
  return swiglu ? by_groups(template_int<TK_F16>{}, std::true_type{}) : by_groups(template_int<TK_F16>{}, std::false_type{});
}

}  // namespace tk
