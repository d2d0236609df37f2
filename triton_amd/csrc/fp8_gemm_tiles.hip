// The ragged product of e4m3 operands with one scale for each block of 128, full row blocks: both operands staged by memory-to-LDS transfers.
//
//   * A workgroup multiplies 256 rows of one expert by 256 columns with eight waves of 128 x 64 (one workgroup per CU), or 128 by 128 with four waves of
//     64 x 64 (two per CU).  A stage is 128 k of both operands: one block of scales, and whole cache lines.  Two stages are in LDS.
//   * A wave takes its 64 columns of a stage into registers and goes through its row fragments of 16: a product of 16 x 16 over the whole block on a cleared
//     accumulator, and three products later four fused operations that add it to the running sums times the scales.  The order is pinned product by product: what
//     the compiler makes of it needs more registers than there are.
//   * Scales that are powers of two (a caller that had both operands quantised here says so) go into the matrix instruction as exponents, and it adds
//     to the running sum itself.
//   * The scales of a stage (one a row, one or two for the columns) come by transfers of four bytes a lane beside the operands.
//   * A stage's columns are in registers from the end of the one before, so a second barrier frees their buffer and the transfers of the stage after next begin there; those of the rows
//     follow behind the stage's last reads.  The barrier stands in the stage's middle for tiles of 256, at its start for tiles of 128, whose stages are short beside a transfer's way (us, start /
//     middle: 32 experts, 4096 rows, 2880 x 2880 108 / 113; 2048 rows 76 / 81; tiles of 256: one of 8192 rows, 8192 x 8192 608 / 575).
//   * Transfers, the order of 16-byte pieces in LDS, the list of tiles and the run across tiles are those of moe_gemm_dma_kernel.h.
//   * What bounds it (8192 rows, 8192 x 8192): 575 us = 1.91 PFLOP/s, with exponents in the matrix instruction 514 = 2.14; the same without the transfers' data 444, with all of them from one line of
//     the cache 536; the matrix unit is busy 0.42 of the cycles and LDS 0.35, at 1.93 GHz (eight experts, 16384 rows, K 4096, N 14336).  Two waves a SIMD meet twice a stage.  Tried, and slower or no faster: half of the rows' transfers in the
//     middle, others' order of pieces in LDS (its conflicts are half of its cycles), a word of each line asked for two stages ahead, three stages of 128 x 256, a stage of 128 x 128 as a whole in registers.
//   * K that is no multiple of 16: the last piece of a row holds bytes of whatever follows; they are cleared in LDS before the last stage is read.
#include "fp8_blocks.h"
#include "gemm_tiles.h"

namespace tk {
namespace {

template <int TILE>
struct TilesCfg {
  static constexpr int WM = 2, WN = TILE / 64, NW = WM * WN;  // waves along rows / columns
  static constexpr int MFW = TILE / 32, NFW = 4;              // fragments of a wave
  static constexpr int BYTES = TILE * kFp8Block;              // of an operand's stage
  static constexpr int TR = TILE / 8 / NW;                    // transfers of a wave, operand and stage
  static constexpr int SCALES = TILE * 4 + 256;               // a stage's scales: rows, then columns
  static constexpr int LDS = 4 * BYTES + 2 * SCALES;
  static constexpr int PER_CU = TILE == 256 ? 1 : 2;
};
static_assert(TilesCfg<256>::LDS <= 160 * 1024 && TilesCfg<128>::LDS <= 80 * 1024, "one / two workgroups of a CU");

template <int TILE, int YT, bool SWIGLU, bool POW2>
__global__ __launch_bounds__(TilesCfg<TILE>::NW * 64, 2) void fp8_block_tiles_kernel(const Fp8GemmParams p) {
  typedef TilesCfg<TILE> C;
  constexpr int MFW = C::MFW, NFW = C::NFW;
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  fp8_zero_rest<YT, SWIGLU>(p);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int mw = wave % C::WM, nw = wave / C::WM;
  const int lr = lane & 15, g4 = lane >> 4;
  const int nst = (p.K + kFp8Block - 1) / kFp8Block;
  const int tail = p.K & 15;
  const uint32_t lds0 = lds_addr(lds);

  TileList<TILE, TILE> tiles;
  int tile = tiles.init(p, lane, (p.N + TILE - 1) / TILE);
  const int t_step = tiles.t_step, t_end = tiles.t_end;
  if (tile >= t_end) return;

  // ---- transfer side: transfer i of a wave and operand = lines (wave * TR + i) * 8 .. + 7, lane -> line lane / 8, LDS position lane % 8, i.e. piece (lane % 8) ^
  // (line >> 1 & 7), where line >> 1 & 7 = (i & 1) * 4 + (lane >> 4) ------------------------------------------------------------------------------------
  static_assert(C::TR % 2 == 0, "a transfer's parity is that of its index in the wave");
  const int pc0 = (lane & 7) ^ (lane >> 4), pc1 = pc0 ^ 4;
  buf_desc_t xdesc, wdesc, sdesc;
  uint32_t x_off[C::TR], w_off[C::TR], s_off;
  uint32_t s_step;  // bytes from a block's scale to the next one's, of what this wave fetches
  const uint32_t x_row = (uint32_t)p.x_stride_m, w_row = (uint32_t)p.w_n;
  constexpr int SW = TILE / 64;  // waves 0 .. SW - 1 fetch the rows' scales, 64 each, wave SW the columns'
  // (what depends on the lane alone would be kept in registers over the whole loop, beside sums that need them: a lane number the compiler cannot follow is not)
  auto own_lane = [&]() __attribute__((always_inline)) -> int {
    int l = tid & 63;
    asm volatile("" : "+v"(l));
    return l;
  };
  auto aim = [&](const Tile& c) __attribute__((always_inline)) {
    const int lane = own_lane(), pc0 = (lane & 7) ^ (lane >> 4), pc1 = pc0 ^ 4;
    const int rows = c.eM - c.off_m < TILE ? c.eM - c.off_m : TILE, cols = p.N - c.n_tile < TILE ? p.N - c.n_tile : TILE;
    const int first = c.start_m + c.off_m;
    // (to the end of the last row's last piece: its bytes lie in memory that holds the row's end)
    xdesc = p.gather ? make_buf_desc(p.x, p.x_bytes) : make_buf_desc(p.x + first * p.x_stride_m, (uint32_t)(rows - 1) * x_row + (uint32_t)((p.K + 15) & ~15));
    wdesc = make_buf_desc(p.w + (int64_t)c.expert * p.w_e + (int64_t)c.n_tile * p.w_n, (uint32_t)(cols - 1) * w_row + (uint32_t)((p.K + 15) & ~15));
#pragma unroll
    for (int i = 0; i < C::TR; ++i) {
      const int line = (wave * C::TR + i) * 8 + (lane >> 3);
      const uint32_t piece = (uint32_t)((i & 1) ? pc1 : pc0) * 16u;
      const uint32_t src = line < rows ? (p.gather ? (uint32_t)p.gather[first + line] : (uint32_t)line) : 0u;
      x_off[i] = line < rows ? src * x_row + piece : kOutOfRange;
      w_off[i] = line < cols ? (uint32_t)line * w_row + piece : kOutOfRange;
    }
    if (wave < SW) {
      const int line = wave * 64 + lane;
      const uint32_t src = line < rows ? (p.gather ? (uint32_t)p.gather[first + line] : (uint32_t)line) : 0u;
      sdesc = make_buf_desc(p.gather ? p.xs : p.xs + first * p.xs_m, 0x7FFFFFFFu);
      s_off = line < rows ? src * (uint32_t)p.xs_m * 4u : kOutOfRange;
      s_step = (uint32_t)p.xs_k * 4u;
    } else if (wave == SW) {
      sdesc = make_buf_desc(p.ws + (int64_t)c.expert * p.ws_e + (int64_t)(c.n_tile / kFp8Block) * p.ws_n, 0x7FFFFFFFu);
      s_off = lane * kFp8Block < cols ? (uint32_t)lane * (uint32_t)p.ws_n * 4u : kOutOfRange;
      s_step = (uint32_t)p.ws_k * 4u;
    }
  };
  uint32_t fill = 0;  // the buffers that the next transfers fill: 0 or 1
  int fs = 0;         // the stage of the tile aimed at that they fetch
  bool more = true;
  int f_tile = tile;
  auto fetch_x = [&](int i) __attribute__((always_inline)) {
    const int k = fs * kFp8Block;
    const bool in = more && k + ((i & 1) ? pc1 : pc0) * 16 < p.K;
    lds_dma16(xdesc, lds0 + fill * C::BYTES + (wave * C::TR + i) * 1024, in ? x_off[i] + (uint32_t)k : kOutOfRange);
  };
  auto fetch_w = [&](int i) __attribute__((always_inline)) {
    const int k = fs * kFp8Block;
    const bool in = more && k + ((i & 1) ? pc1 : pc0) * 16 < p.K;
    lds_dma16(wdesc, lds0 + (2 + fill) * C::BYTES + (wave * C::TR + i) * 1024, in ? w_off[i] + (uint32_t)k : kOutOfRange);
  };
  auto fetch_s = [&]() __attribute__((always_inline)) {
    if (wave <= SW) lds_dma4(sdesc, lds0 + 4 * C::BYTES + fill * C::SCALES + wave * 256, more ? s_off + (uint32_t)fs * s_step : kOutOfRange);
  };
  auto advance = [&]() __attribute__((always_inline)) {
    fill ^= 1;
    if (++fs == nst) {
      fs = 0;
      f_tile += t_step;
      more = more && f_tile < t_end;
      if (more) aim(tiles.locate(f_tile));
    }
  };

  // ---- LDS read side: the lane's pieces 2 g4 and 2 g4 + 1 of its line -----------------------------------------------------------------------------------
  const int sw = (lr >> 1) & 7;
  const uint32_t pos0 = (uint32_t)(((2 * g4) ^ sw) * 16 + lr * 128), pos1 = (uint32_t)(((2 * g4 + 1) ^ sw) * 16 + lr * 128);
  auto ld = [&](uint32_t at) __attribute__((always_inline)) -> u32x4_t { return *reinterpret_cast<const u32x4_t*>(lds + at); };
  auto frag = [&](uint32_t at) __attribute__((always_inline)) -> i32x8_t {
    return __builtin_bit_cast(i32x8_t, __builtin_shufflevector(ld(at + pos0), ld(at + pos1), 0, 1, 2, 3, 4, 5, 6, 7));
  };
  i32x8_t w[NFW], x[2];
  float sx[2], sc;
  auto read_w = [&](uint32_t b, int f) __attribute__((always_inline)) { w[f] = frag((2 + b) * C::BYTES + (uint32_t)((nw * NFW + f) * 2048)); };
  auto read_sc = [&](uint32_t b) __attribute__((always_inline)) {
    sc = *reinterpret_cast<const float*>(lds + 4 * C::BYTES + b * C::SCALES + TILE * 4 + (nw * 64 / kFp8Block) * 4);
  };
  auto read_x = [&](uint32_t b, int j) __attribute__((always_inline)) {
    x[j & 1] = frag(b * C::BYTES + (uint32_t)((j * C::WM + mw) * 2048));
    sx[j & 1] = *reinterpret_cast<const float*>(lds + 4 * C::BYTES + b * C::SCALES + ((j * C::WM + mw) * 16 + lr) * 4);
  };
  auto barrier = [&]() __attribute__((always_inline)) {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  // clears what the last piece of each line of stage buffer b holds past K
  auto clear_tail = [&](uint32_t b) __attribute__((always_inline)) {
    for (int line = wave * 64 + own_lane(); line < 2 * TILE; line += C::NW * 64) {
      const int l = line % TILE, piece = ((p.K % kFp8Block) >> 4) ^ ((l >> 1) & 7);
      uint8_t* at = lds + (line < TILE ? b : 2 + b) * C::BYTES + l * 128 + piece * 16;
      u32x4_t v = *reinterpret_cast<const u32x4_t*>(at);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int keep = tail - 4 * i;  // bytes of this word
        v[i] = keep >= 4 ? v[i] : keep <= 0 ? 0u : v[i] & ((1u << 8 * keep) - 1u);
      }
      *reinterpret_cast<u32x4_t*>(at) = v;
    }
    barrier();
  };

  Tile cur = tiles.locate(tile);
  aim(cur);
#pragma unroll 1
  for (int n = 0; n < 2; ++n) {
#pragma unroll
    for (int i = 0; i < C::TR; ++i) fetch_w(i);
#pragma unroll
    for (int i = 0; i < C::TR; ++i) fetch_x(i);
    fetch_s();
    advance();
  }
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * C::TR) : "memory");  // (a wave without scales to fetch has no more in flight; the others wait for one more)
  barrier();
  if (tail && nst == 1) clear_tail(0);
  uint32_t b = 0;
  const f32x4_t zero = {0.f, 0.f, 0.f, 0.f};
  f32x4_t acc[NFW][MFW], part[NFW];

  // A stage; its columns and its first row fragment are in registers.
  auto stage = [&](bool next_has_tail) __attribute__((always_inline)) {
    constexpr int MID = TILE == 128 ? 0 : MFW / 2 - 1, ALL = MFW * NFW, SKEW = 3;  // (up to NFW - 1: a result's registers are taken again NFW products later)
    float s[2];
    auto add = [&](auto t_c) __attribute__((always_inline)) {  // product T's sums, times the scales
      constexpr int T = decltype(t_c)::value, J = T / NFW, F = T % NFW;
      if constexpr (!POW2) {
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[F][J][i] = fmaf(part[F][i], s[J & 1], acc[F][J][i]);
        asm volatile("" : "+v"(acc[F][J]));
      }
    };
    static_for<0, ALL>([&](auto t_c) __attribute__((always_inline)) {
      constexpr int T = decltype(t_c)::value, J = T / NFW, F = T % NFW;
      constexpr bool END = J == MFW - 1;
      if constexpr (END && F == 0) {
        // every wave has read this stage, and the next one has landed (in flight behind it: the columns that MID asked for)
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(C::TR) : "memory");
        barrier();
        if (next_has_tail) clear_tail(b ^ 1);
      }
      if constexpr (T == 0 && MID == 0) barrier();  // every wave has this stage's columns in registers
      if constexpr (F == 0) s[J & 1] = sx[J & 1] * sc;
      if constexpr (POW2)
        acc[F][J] = mfma_block(w[F], x[J & 1], acc[F][J], f32_bits(sc) >> 23, f32_bits(sx[J & 1]) >> 23);
      else
        part[F] = mfma_block(w[F], x[J & 1], zero);
      // (an empty use of the results: the compiler otherwise sinks the products to the end of the loop, where all operands live at once)
      if constexpr (POW2)
        asm volatile("" : "+v"(acc[F][J]));
      else
        asm volatile("" : "+v"(part[F]));
      if constexpr (!END) {
        if constexpr (F == 0) read_x(b, J + 1);
      } else {
        if constexpr (F == 0) read_x(b ^ 1, 0);
        read_w(b ^ 1, F);
        fetch_x(F);
        if constexpr (F == NFW - 1) fetch_s();
      }
      if constexpr (J == MID) {
        if constexpr (F == 0 && MID > 0) {
          // every wave has this stage's columns in registers (and multiplied by them)
          __builtin_amdgcn_s_barrier();
          asm volatile("" ::: "memory");
        }
        fetch_w(F);
      }
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (T >= SKEW) add(template_int<T - SKEW>{});
      __builtin_amdgcn_sched_barrier(0);
    });
    static_assert(C::TR == NFW, "a transfer of either operand beside each of the last products");
    static_for<ALL - SKEW, ALL>([&](auto t_c) __attribute__((always_inline)) { add(t_c); });
    read_sc(b ^ 1);
    advance();
    b ^= 1;
  };

  auto begin = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int f = 0; f < NFW; ++f)
#pragma unroll
      for (int j = 0; j < MFW; ++j) acc[f][j] = zero;
#pragma unroll
    for (int f = 0; f < NFW; ++f) read_w(b, f);
    read_sc(b);
    read_x(b, 0);
  };
  begin();
  // (one loop over the stages of all tiles: a second copy of the stage for a tile's last one needs its results and its sums in registers of their own)
#pragma unroll 1
  for (int s = 0;;) {
    stage(tail && (s + 2 == nst || nst == 1));
    if (++s < nst) continue;
    fp8_epilogue<YT, SWIGLU, C::WM, MFW, NFW>(p, acc, cur.expert, cur.off_m, cur.start_m, cur.eM, cur.n_tile + nw * 64, p.N, mw, own_lane());
    tile += t_step;
    if (tile >= t_end) break;
    cur = tiles.locate(tile);
    s = 0;
    begin();  // (what the stage read ahead, once more: the epilogue needs the registers)
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (the last transfers write into this workgroup's LDS)
}

template <int TILE>
int32_t launch(Fp8GemmParams p, int yt, bool swiglu, hipStream_t st) {
  typedef TilesCfg<TILE> C;
  p.grid_n = (int)cdiv(p.N, TILE);
  const int64_t tiles = (cdiv(p.M, TILE) + (p.slice_sizes ? p.n_slices - 1 : 0)) * p.grid_n;
  if (tiles > 0x7FFFFFFF) return fail(TK_ERR_UNSUPPORTED, "tk_fp8_block_gemm: grid too large");
  int64_t grid = (int64_t)device_cu_count() * C::PER_CU / 8 * 8;
  if (grid > cdiv(tiles, 8) * 8) grid = cdiv(tiles, 8) * 8;
  auto go = [&](auto kern) -> int32_t {
    if (const int32_t rc = allow_dynamic_lds(reinterpret_cast<const void*>(kern), C::LDS)) return rc;
    hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(C::NW * 64), C::LDS, st, p);
    return check_launch("fp8_block_tiles_kernel");
  };
  auto by_act = [&](auto yt_c) -> int32_t {
    constexpr int YT = decltype(yt_c)::value;
    if (p.pow2 && !swiglu) return go(fp8_block_tiles_kernel<TILE, YT, false, true>);
    return swiglu ? go(fp8_block_tiles_kernel<TILE, YT, true, false>) : go(fp8_block_tiles_kernel<TILE, YT, false, false>);
  };
  return yt == TK_BF16 ? by_act(template_int<TK_BF16>{}) : by_act(template_int<TK_F16>{});
}

}  // namespace

int32_t fp8_gemm_launch_tiles(const Fp8GemmParams& p, int tile, int yt, bool swiglu, hipStream_t st) {
  return tile == 256 ? launch<256>(p, yt, swiglu, st) : launch<128>(p, yt, swiglu, st);
}

}  // namespace tk
