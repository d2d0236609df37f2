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
  int32_t parts;  // parts of a slice's rows, each with sums of its own (y is the workspace then)
  int32_t pow2;
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

// ---- lines that begin at sixteen-byte boundaries -------------------------------------------------------------------------------------------------------
//
//   * A workgroup multiplies a T x T tile of a slice: 256 with eight waves of 128 x 64 (one per CU), or 128 with four waves of 64 x 64 (two per CU).  A stage is
//     64 rows; two are in LDS, in the operands' own order, and are turned by the reads (read_frag_tr).
//   * Both operands come through registers, asked for a stage and more ahead: that is where x is scaled and becomes dy's type, once for all waves.  (A transfer straight
//     into LDS would have x converted on its way out of it, by each of the waves that share it, row scales and all.)
//   * One barrier a stage, in front of the last of its four steps of sixteen rows: until there the next stage is written into the buffer that the last one has
//     been read from, piece by piece beside the products of the other three steps, and the one behind it asked for.
//   * Workgroups are persistent and the stream of stages runs on across tiles.  Every XCD takes an eighth of each slice's tiles, from the longest slice to the
//     shortest (up to 64 of them), and its workgroups walk their list forth and back.
//   * us: eight slices of 16384 rows in all, 2880 x 5760 545 to 640, by box (850 to 1000 TFLOP/s), 4096 x 14336 1770 (1086; a library product of 8192 cubed in bf16 reaches 1200).  The matrix unit is busy
//     0.55 of the cycles at 1.98 GHz, LDS 0.42.  Four waves of 128 x 96 or 128 x 128, which read a third less from LDS, have one wave a SIMD and take 1.5 to 3 times as long.

constexpr int kStage = 64;
template <int T>
struct WgradCfg {
  static constexpr int WM = 2, WN = T / 64, NW = WM * WN;
  static constexpr int MF = T / WM / 32, NF = 2;  // fragments of a wave
  static constexpr int PITCH = T * 2, OPERAND = kStage * PITCH, STAGE = 2 * OPERAND, LDS = 2 * STAGE;
  static constexpr int THREADS = NW * 64;
  static constexpr int PER_CU = T == 256 ? 1 : 2;
  static constexpr int XP = kStage * T / 16 / THREADS, DP = kStage * T / 8 / THREADS;  // pieces of sixteen bytes a thread: x, dy
};

// POW2: bf16, and all scales powers of two: the conversion multiplies by the exponent.
template <int DT, int YT, int T, bool POW2>
__global__ __launch_bounds__(WgradCfg<T>::THREADS, 2) void fp8_wgrad_kernel(const WgradParams p) {
  typedef WgradCfg<T> C;
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = lane >> 5, mw = wave & 1, nw = wave >> 1;
  const uint32_t lds0 = lds_addr(lds);

  // ---- the slices, longest first (lane l: that of rank l), and this workgroup's tiles ----------------------------------------------------------------
  const bool sorted = p.n_slices <= 64;
  int sz = 0, so = 0, id = lane;
  if (sorted) {
    int mine = lane < p.n_slices ? p.T : -1, first = 0;  // (no slices: one of T rows)
    if (p.slice_sizes && lane < p.n_slices) mine = p.slice_sizes[lane], first = p.slice_offs[lane];
    int rank = 0;
    for (int o = 0; o < p.n_slices; ++o) {
      const int other = __builtin_amdgcn_readlane(mine, o);
      rank += other > mine || (other == mine && o < lane) ? 1 : 0;
    }
    // (a lane's rank is a place of its own; lanes without a slice keep theirs)
    rank = lane < p.n_slices ? rank : lane;
    sz = __builtin_amdgcn_ds_permute(rank * 4, mine);
    so = __builtin_amdgcn_ds_permute(rank * 4, first);
    id = __builtin_amdgcn_ds_permute(rank * 4, lane);
  }
  // (of few tiles a slice, and of parts, an XCD takes every eighth)
  const uint32_t per_e = (uint32_t)(p.tiles_k * p.tiles_n), parts = (uint32_t)p.parts, units = per_e * (uint32_t)p.n_slices * parts;
  const bool flat = per_e < 64 || parts > 1;
  const uint32_t q = (per_e + 7) / 8, total = flat ? (units + 7) / 8 : q * (uint32_t)p.n_slices;
  const uint32_t xcd = blockIdx.x & 7, i8 = blockIdx.x >> 3, wgs = gridDim.x >> 3, rounds = (total + wgs - 1) / wgs;
  struct Where {
    int id, rows, first, k0, n0;
  };
  auto next = [&](uint32_t& r, Where& w) __attribute__((always_inline)) -> bool {
    for (; r < rounds; ++r) {
      const uint32_t l = r * wgs + (r & 1 ? wgs - 1 - i8 : i8), v = flat ? (l * 8 + xcd) / per_e : l / q, in = flat ? l * 8 + xcd - v * per_e : xcd * q + (l - v * q);
      if (l >= total || in >= per_e || v >= parts * (uint32_t)p.n_slices) continue;
      const uint32_t rank = (uint32_t)__builtin_amdgcn_readfirstlane((int)(v / parts)), part = v - rank * parts;
      // (bands of eight tiles down, in a band column by column, so that those in hand on an XCD share few operand columns)
      const uint32_t band = in / (8u * (uint32_t)p.tiles_n), left = (uint32_t)p.tiles_k - band * 8u, bh = left < 8u ? left : 8u;
      const uint32_t in_b = in - band * 8u * (uint32_t)p.tiles_n, tn = in_b / bh, tk = band * 8u + in_b - tn * bh;
      if (sorted) {
        w.id = __builtin_amdgcn_readlane(id, (int)rank), w.rows = __builtin_amdgcn_readlane(sz, (int)rank), w.first = __builtin_amdgcn_readlane(so, (int)rank);
      } else {
        // (scalar loads: the wait for a vector one would be a wait for the stages in flight)
        typedef const __attribute__((address_space(4))) int32_t* scalar_t;
        w.id = (int)rank, w.rows = reinterpret_cast<scalar_t>(reinterpret_cast<uintptr_t>(p.slice_sizes))[rank];
        w.first = reinterpret_cast<scalar_t>(reinterpret_cast<uintptr_t>(p.slice_offs))[rank];
      }
      if (parts > 1) {  // whole stages
        const uint32_t stages = ((uint32_t)w.rows + kStage - 1) / kStage, from = (uint32_t)((uint64_t)stages * part / parts) * kStage;
        const uint32_t to = (uint32_t)((uint64_t)stages * (part + 1) / parts) * kStage;
        w.rows = (int)(to < (uint32_t)w.rows ? to : (uint32_t)w.rows) - (int)from, w.first += (int)from, w.id = w.id * (int)parts + (int)part;
      }
      // (all of it is the same in every lane, which the compiler loses sight of)
      w.id = __builtin_amdgcn_readfirstlane(w.id), w.rows = __builtin_amdgcn_readfirstlane(w.rows), w.first = __builtin_amdgcn_readfirstlane(w.first);
      w.k0 = __builtin_amdgcn_readfirstlane((int)tk * T), w.n0 = __builtin_amdgcn_readfirstlane((int)tn * T);
      r = (uint32_t)__builtin_amdgcn_readfirstlane((int)r);
      return true;
    }
    return false;
  };
  uint32_t cur_r = 0;
  Where cur;
  if (!next(cur_r, cur)) return;

  // ---- loads: the next stage to ask for ------------------------------------------------------------------------------------------------------------------
  uint32_t f_r = cur_r;
  Where aim = cur;
  constexpr int XL = T / 16, DL = T / 8;  // threads of a row
  constexpr int XR = C::THREADS / XL, DR = C::THREADS / DL;  // rows of a piece of all threads
  // what a thread holds of the stage to be written next: the pieces of x with their scales, and those of dy
  u32x4_t lx[C::XP], ld[C::DP];
  float ls[C::XP];
  // A stage's resources begin at its first row, and end with the slice's last one: rows behind it read zeros, and no scale.  Columns behind K or N read what follows,
  // or zeros, and end in rows and columns that are not there.
  const uint32_t x_at = (uint32_t)(tid / XL) * (uint32_t)p.x_t + tid % XL * 16u, d_at = ((uint32_t)(tid / DL) * (uint32_t)p.dy_t + tid % DL * 8u) * 2u;
  const uint32_t s_at = ((uint32_t)(tid / XL) * (uint32_t)p.xs_t + (uint32_t)(tid % XL * 16 / kFp8Block) * (uint32_t)p.xs_k) * 4u;
  const bool s_in = tid % XL * 16 / kFp8Block == 0;  // (of a tile that ends within its first block of K the second has no scales)
  const uint8_t* xb;
  const uint16_t* db;
  const float* sb;
  int left;  // rows of the slice from the next stage on
  int x_end, d_end;
  bool second;
  auto start = [&]() __attribute__((always_inline)) {
    const int64_t t = aim.first;
    xb = p.x + t * p.x_t + aim.k0, db = p.dy + t * p.dy_t + aim.n0, sb = p.xs + t * p.xs_t + (int64_t)(aim.k0 / kFp8Block) * p.xs_k;
    left = aim.rows;
    x_end = ((p.K + 15) & ~15) - aim.k0, d_end = (((p.N + 7) & ~7) - aim.n0) * 2;
    second = aim.k0 + kFp8Block < p.K;
  };
  start();
  typedef decltype(__builtin_amdgcn_make_buffer_rsrc((void*)nullptr, 0, 0, 0)) resource_t;
  resource_t xr, dr, sr;
  int rows;
  auto resources = [&]() __attribute__((always_inline)) {  // of the stage to ask for
    rows = left < kStage ? left : kStage;
    const int x_bytes = __builtin_amdgcn_readfirstlane(rows > 0 ? (rows - 1) * (int)p.x_t + x_end : 0);
    const int d_bytes = __builtin_amdgcn_readfirstlane(rows > 0 ? (rows - 1) * (int)p.dy_t * 2 + d_end : 0);
    xr = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(xb), 0, x_bytes, 0x00020000);
    dr = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(db), 0, d_bytes, 0x00020000);
    sr = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(sb), 0, 0x7FFFFFFF, 0x00020000);
  };
  auto load_x = [&](int i) __attribute__((always_inline)) {
    lx[i] = __builtin_amdgcn_raw_buffer_load_b128(xr, x_at + (uint32_t)(i * XR) * (uint32_t)p.x_t, 0, 0);
    const bool in = tid / XL + i * XR < rows && (second || s_in);
    ls[i] = bits_f32(__builtin_amdgcn_raw_buffer_load_b32(sr, in ? s_at + (uint32_t)(i * XR) * (uint32_t)p.xs_t * 4u : 0x80000000u, 0, 0));
  };
  auto load_d = [&](int i) __attribute__((always_inline)) { ld[i] = __builtin_amdgcn_raw_buffer_load_b128(dr, d_at + (uint32_t)(i * DR) * (uint32_t)p.dy_t * 2u, 0, 0); };
  auto advance = [&]() __attribute__((always_inline)) {
    left -= kStage;
    if (left > 0) {
      xb += kStage * p.x_t, db += kStage * p.dy_t, sb += kStage * p.xs_t;
    } else if (f_r < rounds) {
      ++f_r;
      if (next(f_r, aim)) start();
    }
  };
  auto store_x = [&](int i, uint32_t buf) __attribute__((always_inline)) {
    const int row = tid / XL + i * XR, piece = (tid % XL * 2) ^ ((row & 3) * 4);
    const float s = ls[i];
    u32x4_t o[2];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      if constexpr (POW2) {
        o[c >> 1][(c & 1) * 2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lx[i][c], s, false));
        o[c >> 1][(c & 1) * 2 + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lx[i][c], s, true));
      } else {
        float v[4];
        from_e4m3(lx[i][c], v);
        o[c >> 1][(c & 1) * 2] = scaled_pair<DT>(v[0], v[1], s);
        o[c >> 1][(c & 1) * 2 + 1] = scaled_pair<DT>(v[2], v[3], s);
      }
    }
    u32x4_t* to = reinterpret_cast<u32x4_t*>(lds + buf + row * C::PITCH + piece * 16);
    to[0] = o[0], to[1] = o[1];
  };
  auto store_d = [&](int i, uint32_t buf) __attribute__((always_inline)) {
    const int row = tid / DL + i * DR, piece = (tid % DL) ^ ((row & 3) * 4);
    *reinterpret_cast<u32x4_t*>(lds + buf + C::OPERAND + row * C::PITCH + piece * 16) = ld[i];
  };
  // part i of four of the stage held: written, and the same part of the one behind it asked for
  static_assert(C::DP == 4 && C::XP == 2, "parts");
  auto part = [&](auto i_c, uint32_t buf) __attribute__((always_inline)) {
    constexpr int I = decltype(i_c)::value;
    if constexpr (I < 2) store_x(I, buf), load_x(I);
    store_d(I, buf), load_d(I);
  };

  // ---- fragment reads: a lane's row of four, four columns; columns 32 j on are pieces 4 j on ----------------------------------------------------------------
  const int l16 = lane & 15, pp = ((lane >> 4) & 1) * 2 + ((l16 & 3) >> 1);
  const uint32_t rd0 = lds0 + (uint32_t)((h * 8 + (l16 >> 2)) * C::PITCH + (l16 & 1) * 8);
  uint32_t at_a[C::MF], at_b[C::NF];
#pragma unroll
  for (int j = 0; j < C::MF; ++j) at_a[j] = rd0 + (uint32_t)(((mw * C::MF * 4 + j * 4 + pp) ^ ((l16 >> 2) * 4)) * 16);
#pragma unroll
  for (int f = 0; f < C::NF; ++f) at_b[f] = rd0 + C::OPERAND + (uint32_t)(((nw * C::NF * 4 + f * 4 + pp) ^ ((l16 >> 2) * 4)) * 16);
  u32x4_t af[2][C::MF], bf[2][C::NF];
  f32x16_t acc[C::NF][C::MF];
  // step S of a stage: its products, while the operands of the next step (of the same stage, or the next one's first) are read from `from`; behind the first ones
  // what `between` does
  auto step = [&](auto s_c, uint32_t from, auto&& between) __attribute__((always_inline)) {
    constexpr int S = decltype(s_c)::value, P = S & 1, NEXT = (S + 1) & 3;
#pragma unroll
    for (int f = 0; f < C::NF; ++f) bf[1 - P][f] = read_frag_tr(at_b[f] + (uint32_t)(NEXT * 16 * C::PITCH) + from, C::PITCH);
#pragma unroll
    for (int j = 0; j < C::MF; ++j) {
      af[1 - P][j] = read_frag_tr(at_a[j] + (uint32_t)(NEXT * 16 * C::PITCH) + from, C::PITCH);
#pragma unroll
      for (int f = 0; f < C::NF; ++f) {
        acc[f][j] = mfma_k16<DT>(bf[P][f], af[P][j], acc[f][j]);
        asm volatile("" : "+v"(acc[f][j]));  // (an empty use: the products stay where they are written)
      }
      if (j == 0) between();
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto barrier = [&]() __attribute__((always_inline)) {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int f = 0; f < C::NF; ++f)
#pragma unroll
      for (int j = 0; j < C::MF; ++j)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[f][j][i] = 0.f;
  };
  auto write = [&](const Where& w) __attribute__((always_inline)) {
    int l = tid & 63;
    asm volatile("" : "+v"(l));  // (so that nothing of what follows is worked out before the loop and kept in registers)
    const int lr = l & 31, h = l >> 5;
#pragma unroll
    for (int j = 0; j < C::MF; ++j) {
      const int k = w.k0 + (mw * C::MF + j) * 32 + lr;
#pragma unroll
      for (int f = 0; f < C::NF; ++f)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float v[8];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const auto s = __builtin_amdgcn_permlane32_swap(f32_bits(acc[f][j][8 * u + i]), f32_bits(acc[f][j][8 * u + 4 + i]), false, false);
            v[i] = bits_f32(s[0]), v[4 + i] = bits_f32(s[1]);
          }
          const int n = w.n0 + (nw * C::NF + f) * 32 + 16 * u + 8 * h;
          if (k >= p.K || n >= p.N) continue;
          const int64_t to = w.id * p.y_e + k * p.y_k + n;
          if (n + 8 <= p.N) {
            store_vec<YT, 8>(p.y, to, v);
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (n + i < p.N) store_elem<YT>(p.y, to + i, v[i]);
          }
        }
    }
  };

  // the first stage into LDS, the second into registers
  resources();
  static_for<0, 4>([&](auto i_c) __attribute__((always_inline)) {
    constexpr int I = decltype(i_c)::value;
    if constexpr (I < 2) load_x(I);
    load_d(I);
  });
  advance();
  resources();
  static_for<0, 4>([&](auto i_c) __attribute__((always_inline)) { part(i_c, 0); });
  advance();
  barrier();
#pragma unroll
  for (int f = 0; f < C::NF; ++f) bf[0][f] = read_frag_tr(at_b[f], C::PITCH);
#pragma unroll
  for (int j = 0; j < C::MF; ++j) af[0][j] = read_frag_tr(at_a[j], C::PITCH);
  clear();
  int t = 0;
  uint32_t buf = 0;
#pragma unroll 1
  for (;;) {
    const uint32_t other = buf ^ C::STAGE;
    resources();
    step(template_int<0>{}, buf, [&]() __attribute__((always_inline)) { part(template_int<0>{}, other); });
    step(template_int<1>{}, buf, [&]() __attribute__((always_inline)) { part(template_int<1>{}, other); });
    step(template_int<2>{}, buf, [&]() __attribute__((always_inline)) { part(template_int<2>{}, other), part(template_int<3>{}, other); });
    barrier();
    step(template_int<3>{}, other, []() {});
    advance();
    buf = other;
    t += kStage;
    if (t >= cur.rows) {
      write(cur);
      clear();
      t = 0, ++cur_r;
      if (!next(cur_r, cur)) break;
    }
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

// The parts' sums of one slice, added in their order.
template <int YT>
__global__ __launch_bounds__(256) void fp8_wgrad_join_kernel(const float* ws, int parts, int64_t n_slices, int64_t K, int64_t N, int64_t pitch, void* y, int64_t y_e, int64_t y_k) {
  const int64_t quads = pitch / 4, all = n_slices * K * quads;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
    const int64_t line = i / quads, n = (i - line * quads) * 4, e = line / K, k = line - e * K;
    const float* from = ws + (e * parts * K + k) * pitch + n;
    f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < parts; ++s) sum += *reinterpret_cast<const f32x4_t*>(from + s * K * pitch);
    for (int c = 0; c < 4; ++c)
      if (n + c < N) store_elem<YT>(y, e * y_e + k * y_k + n + c, sum[c]);
  }
}

// Parts of a slice's rows: where tiles of 128 are fewer than half of the places for them and a slice has (expected) eight stages and more, so many that they fill those
// places, of four stages at least.  (Two places on each of 256 compute units, a constant: the workspace is asked for by sizes alone, before it is known on which device the call
// will run, and both have to come to the same number.)
int wgrad_parts(int64_t T, int64_t K, int64_t N, int64_t n_slices) {
  const int64_t tiles = cdiv(K, 128) * cdiv(N, 128) * n_slices, places = 512, stages = n_slices > 0 ? T / n_slices / kStage : 0;
  if (tiles == 0 || tiles * 2 > places || stages < 8) return 1;
  const int64_t by_places = places / tiles, by_stages = stages / 4;
  return (int)(by_places < by_stages ? by_places : by_stages);
}

template <int T>
int32_t launch_tiles(WgradParams p, int dt, int yt, hipStream_t st) {
  typedef WgradCfg<T> C;
  p.tiles_k = (int)cdiv(p.K, T), p.tiles_n = (int)cdiv(p.N, T);
  const int64_t per_e = (int64_t)p.tiles_k * p.tiles_n;
  const int64_t lists = per_e < 64 || p.parts > 1 ? cdiv(per_e * p.n_slices * p.parts, 8) : cdiv(per_e, 8) * p.n_slices;  // tiles of an XCD
  if (lists * 8 > 0x7FFFFFFF) return fail(TK_ERR_UNSUPPORTED, "tk_fp8_block_wgrad: grid too large");
  const int64_t most = (int64_t)device_cu_count() * C::PER_CU / 8;
  const unsigned grid = (unsigned)((lists < most ? lists : most) * 8);
  auto launch = [&](auto kern) -> int32_t {
    if (const int32_t rc = allow_dynamic_lds(reinterpret_cast<const void*>(kern), C::LDS)) return rc;
    hipLaunchKernelGGL(kern, dim3(grid), dim3(C::THREADS), C::LDS, st, p);
    return check_launch("fp8_wgrad_kernel");
  };
  auto by_out = [&](auto dt_c, auto pow2_c) -> int32_t {
    constexpr int DT = decltype(dt_c)::value;
    constexpr bool POW2 = decltype(pow2_c)::value;
    return yt == TK_F32 ? launch(fp8_wgrad_kernel<DT, TK_F32, T, POW2>) : yt == TK_BF16 ? launch(fp8_wgrad_kernel<DT, TK_BF16, T, POW2>) : launch(fp8_wgrad_kernel<DT, TK_F16, T, POW2>);
  };
  if (dt == TK_F16) return by_out(template_int<TK_F16>{}, std::false_type{});
  return p.pow2 ? by_out(template_int<TK_BF16>{}, std::true_type{}) : by_out(template_int<TK_BF16>{}, std::false_type{});
}

// Checks a call and chooses its kernel, on a card with `cus` compute units: tiles of 256 or 128 (with p.parts), 64 the one for any lines, 0 none.
int32_t plan(const tk_fp8_wgrad_desc* d, int64_t cus, WgradParams& p, int32_t& tile) {
  tile = 0;
  if (!d) return fail(TK_ERR_INVALID, "tk_fp8_block_wgrad: null descriptor");
  if (d->T < 0 || d->K < 0 || d->N < 0 || d->n_slices < 0) return fail(TK_ERR_INVALID, "tk_fp8_block_wgrad: negative size");
  if (d->T > kFp8Most || d->K > kFp8Most || d->N > kFp8Most) return fail(TK_ERR_UNSUPPORTED, "tk_fp8_block_wgrad: sizes up to %d (got %d x %d x %d)", kFp8Most, d->T, d->K, d->N);
  if (d->dy_dtype != TK_BF16 && d->dy_dtype != TK_F16) return fail(TK_ERR_UNSUPPORTED, "tk_fp8_block_wgrad: dy must be bf16 or fp16 (dtype %d)", d->dy_dtype);
  if (d->y_dtype != TK_F32 && d->y_dtype != TK_BF16 && d->y_dtype != TK_F16) return fail(TK_ERR_UNSUPPORTED, "tk_fp8_block_wgrad: the gradient is fp32, bf16 or fp16 (dtype %d)", d->y_dtype);
  if (d->slice_sizes ? !d->slice_offs : d->n_slices > 1) return fail(TK_ERR_INVALID, "tk_fp8_block_wgrad: slices need their sizes and offsets");
  if (d->n_slices == 0 || d->K == 0 || d->N == 0) return TK_OK;
  if (!d->y || (d->T > 0 && (!d->x || !d->x_scale || !d->dy))) return fail(TK_ERR_INVALID, "tk_fp8_block_wgrad: null operand");
  p = WgradParams{};
  p.parts = 1;
  p.x = d->x, p.x_t = d->x_stride_t, p.xs = d->x_scale, p.xs_t = d->xs_stride_t, p.xs_k = d->xs_stride_k;
  p.dy = static_cast<const uint16_t*>(d->dy), p.dy_t = d->dy_stride_t;
  p.slice_sizes = d->slice_sizes, p.slice_offs = d->slice_offs, p.n_slices = d->n_slices;
  p.T = d->T, p.K = d->K, p.N = d->N;
  p.y = static_cast<uint8_t*>(d->y), p.y_e = d->y_stride_e, p.y_k = d->y_stride_k;
  p.pow2 = d->pow2_scales;
  // Lines that begin at sixteen-byte boundaries and do not overlap (a line's last piece is read whole: its end lies in the sixteen bytes that hold the line's), and offsets
  // within a stage of 64 rows that fit a buffer resource.
  const int64_t limit = (int64_t)1 << 31;
  if (((reinterpret_cast<uintptr_t>(p.x) | (uint64_t)p.x_t) & 15) == 0 && ((reinterpret_cast<uintptr_t>(p.dy) | (uint64_t)(p.dy_t * 2)) & 15) == 0 && p.x_t >= p.K && p.dy_t >= p.N &&
      p.xs_t >= 0 && p.xs_k >= 0 && 64 * p.x_t < limit && 128 * p.dy_t < limit && (64 * p.xs_t + 2 * p.xs_k) * 4 < limit) {
    if (d->workspace) p.parts = wgrad_parts(p.T, p.K, p.N, p.n_slices);
    if (p.parts > 1 && reinterpret_cast<uintptr_t>(d->workspace) % 16) return fail(TK_ERR_INVALID, "tk_fp8_block_wgrad: the workspace is not 16-byte aligned");
    tile = p.parts == 1 && cdiv(p.K, 256) * cdiv(p.N, 256) * p.n_slices >= 2 * cus ? 256 : 128;
  } else {
    tile = 64;
  }
  return TK_OK;
}

}  // namespace
}  // namespace tk

using namespace tk;

extern "C" int64_t tk_fp8_block_wgrad_workspace_bytes(int32_t T, int32_t K, int32_t N, int32_t n_slices) {
  if (T < 0 || K < 0 || N < 0 || n_slices < 0) return -1;
  const int64_t parts = wgrad_parts(T, K, N, n_slices);
  return parts > 1 ? parts * n_slices * K * (cdiv(N, 4) * 4) * 4 : 0;
}

extern "C" int32_t tk_fp8_block_wgrad(const tk_fp8_wgrad_desc* d, tk_stream_t stream) {
  WgradParams p;
  int32_t tile;
  if (const int32_t rc = plan(d, device_cu_count(), p, tile)) return rc;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (tile == 0) return TK_OK;
  if (tile == 64) return launch_any(p, d->dy_dtype, d->y_dtype, st);
  if (tile == 256) return launch_tiles<256>(p, d->dy_dtype, d->y_dtype, st);
  if (p.parts == 1) return launch_tiles<128>(p, d->dy_dtype, d->y_dtype, st);
  WgradParams q = p;
  const int64_t pitch = cdiv(p.N, 4) * 4;
  q.y = static_cast<uint8_t*>(d->workspace), q.y_e = p.K * pitch, q.y_k = pitch;
  if (const int32_t rc = launch_tiles<128>(q, d->dy_dtype, TK_F32, st)) return rc;
  const int64_t blocks = cdiv(p.n_slices * p.K * (pitch / 4), 256);
  auto join = [&](auto kern) {
    hipLaunchKernelGGL(kern, dim3((unsigned)(blocks < 2048 ? blocks : 2048)), dim3(256), 0, st, static_cast<const float*>(d->workspace), p.parts, (int64_t)p.n_slices, (int64_t)p.K,
                       (int64_t)p.N, pitch, static_cast<void*>(p.y), p.y_e, p.y_k);
  };
  d->y_dtype == TK_F32 ? join(fp8_wgrad_join_kernel<TK_F32>) : d->y_dtype == TK_BF16 ? join(fp8_wgrad_join_kernel<TK_BF16>) : join(fp8_wgrad_join_kernel<TK_F16>);
  return check_launch("fp8_wgrad_join_kernel");
}

extern "C" int32_t tk_host_fp8_block_wgrad_kernel(const tk_fp8_wgrad_desc* d, int32_t cus, int32_t* tile, int32_t* parts) {
  if (!tile || !parts || cus <= 0) return fail(TK_ERR_INVALID, "tk_host_fp8_block_wgrad_kernel: bad argument");
  WgradParams p = {};
  const int32_t rc = plan(d, cus, p, *tile);
  *parts = *tile ? p.parts : 0;
  return rc;
}
