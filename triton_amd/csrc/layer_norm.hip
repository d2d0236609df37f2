// Layer norm of rows, forward and backward.  Both move each element of the rows once a pass and are bound by that; what the kernels below
// arrange is that a row stays in registers between its reductions and its results, and that the sums over rows stay in registers over many
// rows.
//
// Times in the comments are medians over replays of a captured graph of a few calls on the same buffers, so that what fits the last-level
// cache (256 MB) may come from it; where two ways stand side by side, both were timed on one card when the choice between them was made.
#include "row_math.h"

namespace tk {
namespace {

// VE elements of a weight of any type from column c on, `fill` from column C on and without a weight.
template <int VE>
__device__ __forceinline__ void load_weights(const void* p, int dtype, int c, int C, float fill, float (&out)[VE]) {
  if (!p || c + VE > C) {
#pragma unroll
    for (int e = 0; e < VE; ++e) out[e] = p && c + e < C ? load_any(p, dtype, c + e) : fill;
  } else if (dtype == TK_F32) {
#pragma unroll
    for (int q = 0; q < VE / 4; ++q) {
      const row_u32x4 v = RowType<TK_F32>::load_vec(p, c + 4 * q);
#pragma unroll
      for (int e = 0; e < 4; ++e) out[4 * q + e] = bits_f32(v[e]);
    }
  } else {
    typedef uint32_t words __attribute__((ext_vector_type(VE / 2)));
    typedef words words_at2 __attribute__((aligned(2)));
    const words v = *reinterpret_cast<const words_at2*>(static_cast<const uint16_t*>(p) + c);
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      const uint32_t h = e & 1 ? v[e >> 1] >> 16 : v[e >> 1] & 0xFFFFu;
      out[e] = dtype == TK_BF16 ? bits_f32(h << 16) : f16_bits_to_f32((uint16_t)h);
    }
  }
}

// The sum over the TPR lanes that share a row, in each of them; from 256 lanes on through `buf` (a float a wave) and one barrier.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* buf) {
  if constexpr (TPR >= 256) return block_sum<TPR>(v, buf);
  if constexpr (TPR == 64) return wave_sum_f32(v);
  int x = __builtin_bit_cast(int, v);
#define TK_STEP(ctrl) x = __builtin_bit_cast(int, __builtin_bit_cast(float, x) + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, x, ctrl, 0xF, 0xF, false)));
  TK_STEP(TK_DPP_QUAD_XOR1)
  TK_STEP(TK_DPP_QUAD_XOR2)
  TK_STEP(TK_DPP_ROW_HALF_MIRROR)
  if constexpr (TPR >= 16) TK_STEP(TK_DPP_ROW_MIRROR)
#undef TK_STEP
  v = __builtin_bit_cast(float, x);
  if constexpr (TPR >= 32) v += __shfl_xor(v, 16);
  return v;
}

// Between two passes over a row's registers: without it the compiler keeps the first pass' 32-bit elements (and what else of it the second
// one could use) beside the packed ones, at up to four times the registers.
template <int N>
__device__ __forceinline__ void once_more(row_u32x4 (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(v[i]));
}

// s / C, rounded once: the mean of equal elements whose sum is exact is that element, and their distances from it are zero.
__device__ __forceinline__ float mean_of(float s, float C, float inv_c) {
  const float q = s * inv_c;
  return fmaf(fmaf(-q, C, s), inv_c, q);
}

constexpr int block_of(int tpr) { return tpr < 256 ? 256 : tpr; }

// The sums of two numbers over the TPR lanes that share a row, in each of them; from 256 lanes on through `buf` (a pair a wave) and one
// barrier.
template <int TPR>
__device__ __forceinline__ void row_sums(float& a, float& b, float2* buf) {
  if constexpr (TPR < 256) {
    a = row_sum<TPR>(a, nullptr);
    b = row_sum<TPR>(b, nullptr);
  } else {
    a = wave_sum_f32(a);
    b = wave_sum_f32(b);
    if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = make_float2(a, b);
    __syncthreads();
    a = buf[0].x;
    b = buf[0].y;
#pragma unroll
    for (int w = 1; w < TPR / 64; ++w) {
      a += buf[w].x;
      b += buf[w].y;
    }
  }
}

// A mean that comes from one sum is off by that sum's roundings, 2^-24 mean|x| for each number added: nothing beside the deviation as a
// rule, but as much as the deviation or more where that is small against the mean (a row of 12345.678 alone: off by 8e-3, where eps stands
// for a deviation of 3e-3).  Rows whose mean is beyond four deviations therefore look at their distances d = x - mu again, s1 = sum d and
// s2 = sum d^2: s1 has roundings of the distances' size, so that the mean is off by its own rounding in the end, and
// mean(d^2) - mean(d)^2 is the variance while the rest is small against the deviation.  Where it is not, the distances are taken once more,
// from the better mean: a row of equal elements then has that element as its mean, distances of zero and no variance.
// For all rows the same costs up to 11 % of the time (65000 x 500 bf16 28.8 us, 32.2); for these rows alone 1 % where there are none.
__device__ __forceinline__ bool beside_large_mean(float mu, float var) { return mu * mu > 16.f * var; }
struct Spread {
  float rest, var;
  bool again;
  __device__ __forceinline__ Spread(float mean_d, float mean_d2) {
    rest = mean_d;
    again = rest * rest > 0.0625f * mean_d2;
    var = fmaxf(mean_d2 - rest * rest, 0.f);
  }
};

// What the reductions of a row's statistics write in LDS: a place of its own for each, so that one barrier a reduction will do.
template <int WAVES>
struct StatisticsLds {
  float sum[WAVES], scaled[WAVES], squares[WAVES];
  float2 spread[2][WAVES];
};

// One row's mean and reciprocal deviation from its registers (TPR lanes a row, NV vectors of 16 bytes a lane, the first FULL of them within
// any row that comes here): the mean first, then the distances from it.  `lds`: not used below 256 lanes a row.
template <int DT, int TPR, int NV, int FULL>
__device__ __forceinline__ void row_statistics(row_u32x4 (&raw)[NV], int lane, int C, float inv_c, float eps, StatisticsLds<16>* lds,
                                               float* mean, float* rstd) {
  typedef RowType<DT> R;
  constexpr int VE = R::VE;
  const auto sum = [&](float scale) {
    float s = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int e = 0; e < VE; ++e) s += R::element(raw[v], e) * scale;
    return s;
  };
  float mu = mean_of(row_sum<TPR>(sum(1.f), lds ? lds->sum : nullptr), (float)C, inv_c);
  once_more(raw);
  if constexpr (DT != TK_F16)  // (whose sums are not that large)
    if (!(fabsf(mu) < __builtin_inff())) {  // (the sum, but perhaps not the mean, is beyond 32 bits)
      mu = mean_of(row_sum<TPR>(sum(0x1p-32f), lds ? lds->scaled : nullptr), (float)C, inv_c) * 0x1p32f;
      once_more(raw);
    }
  float s = 0.f;
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      const float d = R::element(raw[v], e) - mu;
      s = fmaf(d, v < FULL || (v * TPR + lane) * VE + e < C ? d : 0.f, s);
    }
  float var = row_sum<TPR>(s, lds ? lds->squares : nullptr) * inv_c;
  once_more(raw);
  if (beside_large_mean(mu, var))
    for (int turn = 0; turn < 2; ++turn) {
      float s1 = 0.f, s2 = 0.f;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int here = v < FULL ? VE : R::left((v * TPR + lane) * VE, C);
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          const float x = R::element(raw[v], e) - mu, d = v < FULL || e < here ? x : 0.f;
          s1 += d;
          s2 = fmaf(d, d, s2);
        }
        __builtin_amdgcn_sched_barrier(0);  // (a vector after the other: all distances at once take up to 90 registers more)
      }
      row_sums<TPR>(s1, s2, lds ? lds->spread[turn] : nullptr);
      once_more(raw);
      const Spread r(mean_of(s1, (float)C, inv_c), s2 * inv_c);
      mu += r.rest;
      var = r.var;
      if (!r.again) break;
    }
  *mean = mu;
  *rstd = 1.0f / sqrtf(var + eps);
}

// A row's vectors, and what is to be done with them before they are used: elements behind the row's end are zero then.  (Rows shorter than
// a vector come element by element.)
template <int DT, int TPR, int NV, int FULL>
__device__ __forceinline__ void load_row(const void* x, int64_t at, int lane, int C, row_u32x4 (&raw)[NV]) {
  typedef RowType<DT> R;
  const void* row = static_cast<const char*>(x) + at * R::BYTES;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int i = (v * TPR + lane) * R::VE;
    raw[v] = v < FULL ? R::load_vec(row, i) : TPR == 8 && C < R::VE ? R::load_vec_to(row, i, C, 0u) : R::load_last(row, i, C);
  }
}
template <int DT, int TPR, int NV, int FULL>
__device__ __forceinline__ void place_row(int lane, int C, row_u32x4 (&raw)[NV]) {
  typedef RowType<DT> R;
#pragma unroll
  for (int v = FULL; v < NV; ++v)
    if (!(TPR == 8 && C < R::VE)) raw[v] = R::last(raw[v], (v * TPR + lane) * R::VE, C);
}

// A row a group of TPR lanes.  The weights are requested with the row, so that its latency covers theirs.
template <int DT, int TPR, int NV, int FULL>
__global__ __launch_bounds__(block_of(TPR)) void layer_norm_kernel(const void* x, int64_t M, int C, int64_t sx, const void* w, int wt, const void* b, int bt,
                                                                   float eps, void* y, int64_t sy, float* mean, float* rstd, int64_t m0) {
  typedef RowType<DT> R;
  constexpr int VE = R::VE, ROWS = block_of(TPR) / TPR;
  __shared__ StatisticsLds<16> lds;
  const int lane = (int)threadIdx.x % TPR;
  const int64_t m = m0 + (int64_t)blockIdx.x * ROWS + threadIdx.x / TPR;
  if (m >= M) return;  // (lanes that share a row leave together)
  row_u32x4 raw[NV];
  load_row<DT, TPR, NV, FULL>(x, m * sx, lane, C, raw);
  float wv[NV][VE], bv[NV][VE], mu, r;
  const auto weights = [&](int v) {
    load_weights<VE>(w, wt, (v * TPR + lane) * VE, C, 1.f, wv[v]);
    load_weights<VE>(b, bt, (v * TPR + lane) * VE, C, 0.f, bv[v]);
  };
  constexpr bool EARLY = NV * VE <= 16;  // (beyond that their registers cost more rows at a time than their latency: 8192 x 8192 bf16 65 us, 56)
  if (EARLY)
#pragma unroll
    for (int v = 0; v < NV; ++v) weights(v);
  place_row<DT, TPR, NV, FULL>(lane, C, raw);
  row_statistics<DT, TPR, NV, FULL>(raw, lane, C, 1.0f / (float)C, eps, TPR >= 256 ? &lds : nullptr, &mu, &r);
  void* out = static_cast<char*>(y) + m * sy * R::BYTES;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    float o[VE];
    if (!EARLY) weights(v);
#pragma unroll
    for (int e = 0; e < VE; ++e) o[e] = fmaf((R::element(raw[v], e) - mu) * r, wv[v][e], bv[v][e]);
    if (v < FULL)
      R::store_vec(out, (v * TPR + lane) * VE, R::pack(o));
    else
      R::store_vec_to(out, (v * TPR + lane) * VE, C, R::pack(o));
  }
  if (lane == 0 && mean) {
    mean[m] = mu;
    rstd[m] = r;
  }
}

// Many rows (16384 x 2880 bf16 34.0 us, 5.5 TB/s both ways, 135168 x 128 16.4 us, 4.2): workgroups of four waves that stay, the weights
// read once each, into registers (up to 16 elements a lane) or LDS; a group's next rows are requested before the present ones are summed.
// AT rows a group at a time, so that short rows keep as many bytes under way as long ones.
template <int DT, int TPR, int NV, int FULL>
__global__ __launch_bounds__(256) void layer_norm_many_kernel(const void* x, int64_t M, int C, int64_t sx, const void* w, int wt, const void* b, int bt,
                                                              float eps, void* y, int64_t sy, float* mean, float* rstd) {
  typedef RowType<DT> R;
  constexpr int VE = R::VE, GROUPS = 256 / TPR, AT = NV == 1 ? 2 : 1;
  constexpr bool IN_LDS = NV * VE > 16;
  __shared__ row_u32x4 wl[IN_LDS ? 2 : 1][IN_LDS ? NV : 1][VE / 4][IN_LDS ? TPR : 1];
  const int lane = (int)threadIdx.x % TPR;
  const float inv_c = 1.0f / (float)C;
  float wv[IN_LDS ? 1 : NV][VE], bv[IN_LDS ? 1 : NV][VE];
  if constexpr (IN_LDS) {
    for (int i = threadIdx.x; i < 2 * NV * TPR; i += 256) {
      const int which = i / (NV * TPR), j = i % (NV * TPR);
      float o[VE];
      load_weights<VE>(which ? b : w, which ? bt : wt, j * VE, C, which ? 0.f : 1.f, o);
#pragma unroll
      for (int q = 0; q < VE / 4; ++q)
        wl[which][j / TPR][q][j % TPR] = row_u32x4{f32_bits(o[4 * q]), f32_bits(o[4 * q + 1]), f32_bits(o[4 * q + 2]), f32_bits(o[4 * q + 3])};
    }
    __syncthreads();
  } else {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      load_weights<VE>(w, wt, (v * TPR + lane) * VE, C, 1.f, wv[v]);
      load_weights<VE>(b, bt, (v * TPR + lane) * VE, C, 0.f, bv[v]);
    }
  }
  const int64_t step = (int64_t)gridDim.x * GROUPS * AT;
  int64_t m = ((int64_t)blockIdx.x * GROUPS + threadIdx.x / TPR) * AT;
  if (m >= M) return;  // (lanes that share a row leave together)
  row_u32x4 next[AT][NV];
#pragma unroll
  for (int i = 0; i < AT; ++i) load_row<DT, TPR, NV, FULL>(x, (m + i < M ? m + i : M - 1) * sx, lane, C, next[i]);
  for (; m < M; m += step) {
    row_u32x4 raw[AT][NV];
#pragma unroll
    for (int i = 0; i < AT; ++i) {
#pragma unroll
      for (int v = 0; v < NV; ++v) raw[i][v] = next[i][v];
      if (m + step < M) load_row<DT, TPR, NV, FULL>(x, (m + step + i < M ? m + step + i : M - 1) * sx, lane, C, next[i]);
    }
    __builtin_amdgcn_sched_barrier(0);  // (the requests first)
#pragma unroll
    for (int i = 0; i < AT; ++i) {
      float mu, r;
      place_row<DT, TPR, NV, FULL>(lane, C, raw[i]);
      row_statistics<DT, TPR, NV, FULL>(raw[i], lane, C, inv_c, eps, nullptr, &mu, &r);
      if (m + i >= M) break;
      void* out = static_cast<char*>(y) + (m + i) * sy * R::BYTES;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        float o[VE];
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          const float we = IN_LDS ? bits_f32(wl[0][IN_LDS ? v : 0][e / 4][IN_LDS ? lane : 0][e % 4]) : wv[IN_LDS ? 0 : v][e];
          const float be = IN_LDS ? bits_f32(wl[IN_LDS ? 1 : 0][IN_LDS ? v : 0][e / 4][IN_LDS ? lane : 0][e % 4]) : bv[IN_LDS ? 0 : v][e];
          o[e] = fmaf((R::element(raw[i][v], e) - mu) * r, we, be);
        }
        if (v < FULL)
          R::store_vec(out, (v * TPR + lane) * VE, R::pack(o));
        else
          R::store_vec_to(out, (v * TPR + lane) * VE, C, R::pack(o));
        if (IN_LDS) __builtin_amdgcn_sched_barrier(0);
      }
      if (lane == 0 && mean) {
        mean[m + i] = mu;
        rstd[m + i] = r;
      }
    }
  }
}

// The gradients (16384 x 2880 bf16 66 us, 4.3 TB/s, with the sums' launch).  Workgroups stay for many rows: a lane's columns are the same
// in each of them, so that their sums over rows stay in registers (`SUMS`), are joined over the workgroup's rows in LDS, and leave as one
// row of partial sums a workgroup (parts [2][gridDim.x][C]), which layer_norm_sums_kernel adds in their order.  The weight lies in LDS in
// 32 bits, in the order in which lanes take it.
template <int DT, int TPR, int NV, int FULL, int BLOCK, bool SUMS>
__global__ __launch_bounds__(BLOCK) void layer_norm_backward_kernel(const void* dy, int64_t sdy, const void* x, int64_t M, int C, int64_t sx, const void* w,
                                                                    int wt, const float* mean, const float* rstd, void* dx, int64_t sdx, float* parts) {
  typedef RowType<DT> R;
  constexpr int VE = R::VE, ROWS = BLOCK / TPR, WIDTH = NV * TPR * VE, WPR = TPR / 64;
  // The next row is requested before the present one is summed, where there are registers for both (us without and with: 16384 x 2880 bf16
  // 76.8, 65.6, x 4096 98.7, 92.4, 135168 x 128 31.7, 29.8).
  constexpr bool AHEAD = NV * VE <= 32;
  __shared__ float buf[2][2][16];
  __shared__ row_u32x4 wl[NV][VE / 4][TPR];
  const int lane = (int)threadIdx.x % TPR, group = (int)threadIdx.x / TPR;
  const float inv_c = 1.0f / (float)C;
  for (int i = threadIdx.x; i < NV * TPR; i += BLOCK) {
    float o[VE];
    load_weights<VE>(w, wt, i * VE, C, 1.f, o);
#pragma unroll
    for (int q = 0; q < VE / 4; ++q) wl[i / TPR][q][i % TPR] = row_u32x4{f32_bits(o[4 * q]), f32_bits(o[4 * q + 1]), f32_bits(o[4 * q + 2]), f32_bits(o[4 * q + 3])};
  }
  __syncthreads();
  float dw[SUMS ? NV : 1][VE], db[SUMS ? NV : 1][VE];
  if constexpr (SUMS)
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int e = 0; e < VE; ++e) dw[v][e] = db[v][e] = 0.f;
  row_u32x4 xn[AHEAD ? NV : 1], gn[AHEAD ? NV : 1];
  float mu_n = 0.f, r_n = 0.f;
  // (groups of a workgroup go through the loop together: those without a row take the last one and count it as nothing)
  const auto fetch = [&](int64_t m, row_u32x4* xv, row_u32x4* gv, float* mu, float* r) {
    const int64_t at = m < M ? m : M - 1;
    row_u32x4(&xa)[NV] = *reinterpret_cast<row_u32x4(*)[NV]>(xv);
    row_u32x4(&ga)[NV] = *reinterpret_cast<row_u32x4(*)[NV]>(gv);
    load_row<DT, TPR, NV, FULL>(x, at * sx, lane, C, xa);
    load_row<DT, TPR, NV, FULL>(dy, at * sdy, lane, C, ga);
    *mu = mean[at];
    *r = rstd[at];
  };
  const int64_t first = (int64_t)blockIdx.x * ROWS + group, step = (int64_t)gridDim.x * ROWS;
  if constexpr (AHEAD) fetch(first, xn, gn, &mu_n, &r_n);
  int turn = 0;
  for (int64_t m = first; m - group < M; m += step, turn ^= 1) {
    row_u32x4 xv[NV], gv[NV];
    float mu, r;
    if constexpr (AHEAD) {
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        xv[v] = xn[v];
        gv[v] = gn[v];
      }
      mu = mu_n;
      r = r_n;
      if (m - group + step < M) fetch(m + step, xn, gn, &mu_n, &r_n);
      __builtin_amdgcn_sched_barrier(0);  // (the requests first)
    } else {
      fetch(m, xv, gv, &mu, &r);
    }
    place_row<DT, TPR, NV, FULL>(lane, C, xv);
    place_row<DT, TPR, NV, FULL>(lane, C, gv);
    if (m >= M)
#pragma unroll
      for (int v = 0; v < NV; ++v) gv[v] = row_u32x4{0, 0, 0, 0};
    float sg = 0.f, sgh = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int here = v < FULL ? VE : R::left((v * TPR + lane) * VE, C);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        // (behind the last column there is no x: of large equal ones (0 - mean) rstd may be infinite where their own h is zero)
        const float g0 = R::element(gv[v], e), h = v < FULL || e < here ? (R::element(xv[v], e) - mu) * r : 0.f, g = g0 * bits_f32(wl[v][e / 4][lane][e % 4]);
        sg += g;
        sgh = fmaf(g, h, sgh);
        if constexpr (SUMS) {
          dw[v][e] = fmaf(g0, h, dw[v][e]);
          db[v][e] += g0;
          asm volatile("" : "+v"(dw[v][e]), "+v"(db[v][e]));  // (here, and not when the row is done: both factors would have to be kept)
        }
      }
      __builtin_amdgcn_sched_barrier(0);  // (a vector after the other: all of them at once would not fit the registers)
    }
    if constexpr (TPR > 64) {
      sg = wave_sum_f32(sg);
      sgh = wave_sum_f32(sgh);
      if ((threadIdx.x & 63) == 0) {
        buf[turn][0][threadIdx.x >> 6] = sg;
        buf[turn][1][threadIdx.x >> 6] = sgh;
      }
      __syncthreads();
      sg = sgh = 0.f;
#pragma unroll
      for (int i = 0; i < WPR; ++i) {
        sg += buf[turn][0][group * WPR + i];
        sgh += buf[turn][1][group * WPR + i];
      }
    } else {
      sg = row_sum<TPR>(sg, nullptr);
      sgh = row_sum<TPR>(sgh, nullptr);
    }
    if (!dx || m >= M) continue;
    once_more(xv);
    once_more(gv);
    asm volatile("" ::: "memory");  // (the weight comes from LDS once more, too)
    const float mg = sg * inv_c, mgh = sgh * inv_c;
    void* out = static_cast<char*>(dx) + m * sdx * R::BYTES;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float o[VE];
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const float h = (R::element(xv[v], e) - mu) * r, g = R::element(gv[v], e) * bits_f32(wl[v][e / 4][lane][e % 4]);
        o[e] = (fmaf(-h, mgh, g) - mg) * r;
      }
      if (v < FULL)
        R::store_vec(out, (v * TPR + lane) * VE, R::pack(o));
      else
        R::store_vec_to(out, (v * TPR + lane) * VE, C, R::pack(o));
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  if constexpr (SUMS) {
    // rows that share a wave, then the waves one after the other
    float* sums = reinterpret_cast<float*>(wl);  // WIDTH floats, one of the two sums at a time
    static_assert(sizeof(wl) == WIDTH * 4, "the sums take the weight's place");
#pragma unroll
    for (int which = 0; which < 2; ++which) {
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          float a = which ? db[v][e] : dw[v][e];
          if constexpr (TPR < 64)
#pragma unroll
            for (int d = TPR; d < 64; d *= 2) a += __shfl_xor(a, d);
          (which ? db : dw)[v][e] = a;
        }
      const int leader = (int)threadIdx.x % (TPR < 64 ? 64 : TPR);  // lanes that hold the sums of a wave (or of the workgroup's only row)
      for (int i = 0; i < (TPR >= 64 ? ROWS : BLOCK / 64); ++i) {
        __syncthreads();
        if ((int)threadIdx.x / (TPR < 64 ? 64 : TPR) == i && leader < TPR)
#pragma unroll
          for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int e = 0; e < VE; ++e) {
              float* to = sums + (v * VE + e) * TPR + lane;
              *to = (i ? *to : 0.f) + (which ? db[v][e] : dw[v][e]);
            }
      }
      __syncthreads();
      float* out = parts + ((int64_t)which * gridDim.x + blockIdx.x) * C;
      for (int c = threadIdx.x; c < C; c += BLOCK) {
        const int j = c / VE;
        out[c] = sums[((j / TPR) * VE + c % VE) * TPR + j % TPR];
      }
    }
  }
}

// The partial sums' sums: 16 columns a workgroup, four lanes a row of 64 bytes, 64 rows at a time and eight such requested together; then
// over the lanes and waves that hold the same columns.
__global__ __launch_bounds__(256) void layer_norm_sums_kernel(const float* parts, int n, int C, void* dw, int wt, void* db, int bt, int c0) {
  __shared__ float acc[4][16];
  const int first = c0 + (int)blockIdx.x * 16, c = first + (int)(threadIdx.x & 3) * 4;
  void* out = blockIdx.y ? db : dw;
  if (!out) return;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  const float* p = parts + (int64_t)blockIdx.y * n * C;
  for (int i0 = threadIdx.x >> 2; i0 < n; i0 += 512) {
    row_u32x4 v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = i0 + u * 64 < n ? RowType<TK_F32>::load_vec_to(p + (int64_t)(i0 + u * 64) * C, c, C, 0u) : row_u32x4{0, 0, 0, 0};
#pragma unroll
    for (int u = 0; u < 8; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[e] += bits_f32(v[u][e]);
  }
#pragma unroll
  for (int d = 4; d < 64; d *= 2)
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] += __shfl_xor(s[e], d);
  if ((threadIdx.x & 63) < 4)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[threadIdx.x >> 6][(threadIdx.x & 3) * 4 + e] = s[e];
  __syncthreads();
  if (threadIdx.x < 16 && first + (int)threadIdx.x < C)
    store_any(out, blockIdx.y ? bt : wt, first + (int)threadIdx.x, (acc[0][threadIdx.x] + acc[1][threadIdx.x]) + (acc[2][threadIdx.x] + acc[3][threadIdx.x]));
}

// ---- rows of any length: read once for each step ----------------------------------------------------------------

// A thread's sums of N numbers over the columns of a row that are its own: add(column, sums).  Sums of 64, of 64 such and of these, so that
// rows of 2^24 columns add no more than 64 numbers one after the other, and rows of 2^30 1024 (one sum for all of them: 4 million).
template <int N, class F>
__device__ __forceinline__ void long_sums(int64_t C, float (&out)[N], F&& add) {
  constexpr int64_t STEP = 256, FEW = STEP * 64, MANY = FEW * 64;
#pragma unroll
  for (int i = 0; i < N; ++i) out[i] = 0.f;
  for (int64_t c0 = threadIdx.x; c0 < C; c0 += MANY) {
    float many[N] = {};
    for (int64_t c1 = c0; c1 < C && c1 < c0 + MANY; c1 += FEW) {
      float few[N] = {};
      const int64_t end = C < c1 + FEW ? C : c1 + FEW;
      for (int64_t c = c1; c < end; c += STEP) add(c, few);
#pragma unroll
      for (int i = 0; i < N; ++i) many[i] += few[i];
    }
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] += many[i];
  }
}

template <int DT>
__global__ __launch_bounds__(256) void layer_norm_long_kernel(const void* x, int64_t M, int64_t C, int64_t sx, const void* w, int wt, const void* b, int bt,
                                                              float eps, void* y, int64_t sy, float* mean, float* rstd) {
  __shared__ StatisticsLds<4> lds;
  for (int64_t m = blockIdx.x; m < M; m += gridDim.x) {
    const auto element = [&](int64_t c) { return RowType<DT>::load(x, m * sx + c); };
    float s[1], d[2];
    long_sums(C, s, [&](int64_t c, float (&o)[1]) { o[0] += element(c); });
    float mu = block_sum<256>(s[0], lds.sum) / (float)C;
    if (!(fabsf(mu) < __builtin_inff())) {
      long_sums(C, s, [&](int64_t c, float (&o)[1]) { o[0] += element(c) * 0x1p-32f; });
      mu = block_sum<256>(s[0], lds.scaled) / (float)C * 0x1p32f;
    }
    long_sums(C, s, [&](int64_t c, float (&o)[1]) { o[0] = fmaf(element(c) - mu, element(c) - mu, o[0]); });
    float var = block_sum<256>(s[0], lds.squares) / (float)C;
    if (beside_large_mean(mu, var))
      for (int turn = 0; turn < 2; ++turn) {
        long_sums(C, d, [&](int64_t c, float (&o)[2]) {
          const float x = element(c) - mu;
          o[0] += x;
          o[1] = fmaf(x, x, o[1]);
        });
        row_sums<256>(d[0], d[1], lds.spread[turn]);
        const Spread spread(d[0] / (float)C, d[1] / (float)C);
        mu += spread.rest;
        var = spread.var;
        if (!spread.again) break;
      }
    const float r = 1.0f / sqrtf(var + eps);
    for (int64_t c = threadIdx.x; c < C; c += 256) {
      const float h = (element(c) - mu) * r;
      RowType<DT>::store(y, m * sy + c, fmaf(h, w ? load_any(w, wt, c) : 1.0f, b ? load_any(b, bt, c) : 0.0f));
    }
    if (threadIdx.x == 0 && mean) {
      mean[m] = mu;
      rstd[m] = r;
    }
  }
}

template <int DT>
__global__ __launch_bounds__(256) void layer_norm_dx_long_kernel(const void* dy, int64_t sdy, const void* x, int64_t M, int64_t C, int64_t sx, const void* w,
                                                                 int wt, const float* mean, const float* rstd, void* dx, int64_t sdx) {
  __shared__ float buf[2][4];
  for (int64_t m = blockIdx.x; m < M; m += gridDim.x) {
    const float mu = mean[m], r = rstd[m];
    float sums[2];
    long_sums(C, sums, [&](int64_t c, float (&o)[2]) {
      const float g = RowType<DT>::load(dy, m * sdy + c) * (w ? load_any(w, wt, c) : 1.0f);
      o[0] += g;
      o[1] = fmaf(g, (RowType<DT>::load(x, m * sx + c) - mu) * r, o[1]);
    });
    const float sg = block_sum<256>(sums[0], buf[0]) / (float)C, sgh = block_sum<256>(sums[1], buf[1]) / (float)C;
    for (int64_t c = threadIdx.x; c < C; c += 256) {
      const float g = RowType<DT>::load(dy, m * sdy + c) * (w ? load_any(w, wt, c) : 1.0f), h = (RowType<DT>::load(x, m * sx + c) - mu) * r;
      RowType<DT>::store(dx, m * sdx + c, (g - sg - h * sgh) * r);
    }
  }
}

// Row blockIdx.y of the partial sums [2][gridDim.y][C].
template <int DT>
__global__ __launch_bounds__(256) void layer_norm_parts_long_kernel(const void* dy, int64_t sdy, const void* x, int64_t M, int64_t C, int64_t sx,
                                                                    const float* mean, const float* rstd, float* parts) {
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= C) return;
  float dw = 0.f, db = 0.f;
  for (int64_t m = blockIdx.y; m < M; m += gridDim.y) {
    const float g = RowType<DT>::load(dy, m * sdy + c);
    dw = fmaf(g, (RowType<DT>::load(x, m * sx + c) - mean[m]) * rstd[m], dw);
    db += g;
  }
  parts[blockIdx.y * C + c] = dw;
  parts[(gridDim.y + blockIdx.y) * C + c] = db;
}

constexpr int64_t MAX_COLS = 1 << 30;
constexpr int64_t LONG_PARTS = 128;  // partial rows of rows beyond 16384 columns
// Lanes a workgroup of the backward pass, and the most workgroups, each of which leaves a row of partial sums: eight waves a CU carry long
// rows, short ones want more (us at 256, 512, 768, 1024 workgroups: 65000 x 500 bf16 86, 59, 49, 50; 135168 x 128 43, 32, 29, 30; 32768 x
// 1024 64, 48, 49, 50; rows shared by two waves, workgroups of eight: 16384 x 4096 85, 94, 104, 113).
constexpr int backward_block(int tpr) { return tpr == 128 ? 512 : block_of(tpr); }
constexpr int backward_parts(int tpr, int nv) { return nv == 1 ? 768 : tpr == 128 ? 256 : 512; }
// Rows from this many on go through workgroups that stay; fewer have a workgroup each (16 x 2880 bf16 4.0 us, by waves 6.4; 1024 x 2880
// 6.7, 9.4; 4096 x 2880 14.4, by workgroups 17.9).
constexpr int64_t MANY_ROWS = 2048;
// such workgroups, at most (16384 x 4096 bf16 with 1024, 2048, 4096: 53.6, 54.5, 51.2 us; 65000 x 500 fp16 42.0, 35.5, 36.0)
constexpr int64_t STAYING = 2048;
unsigned rows_grid(int64_t rows) { return (unsigned)(rows < 1 << 20 ? rows : 1 << 20); }

struct Forward {
  const void* x;
  int64_t M, C, sx;
  const void* w;
  int wt;
  const void* b;
  int bt;
  float eps;
  void* y;
  int64_t sy;
  float *mean, *rstd;
  hipStream_t s;
  template <int DT, int TPR, int NV, int FULL>
  void run() const {
    if constexpr (TPR <= 64) {
      if (NV > 1 || M >= MANY_ROWS) {
        const int64_t wgs = cdiv(M, 256 / TPR * (NV == 1 ? 2 : 1));
        hipLaunchKernelGGL((layer_norm_many_kernel<DT, TPR, NV, FULL>), dim3((unsigned)(wgs < STAYING ? wgs : STAYING)), dim3(256), 0, s, x, M, (int)C, sx, w, wt, b, bt, eps,
                           y, sy, mean, rstd);
        return;
      }
    }
    if constexpr (TPR > 64 || NV == 1) {
      constexpr int64_t rows = block_of(TPR) / TPR, most = 1 << 21;  // (workgroups of a launch: 2^32 threads are its limit)
      for (int64_t m0 = 0; m0 < M; m0 += most * rows)
        hipLaunchKernelGGL((layer_norm_kernel<DT, TPR, NV, FULL>), dim3((unsigned)(cdiv(M - m0, rows) < most ? cdiv(M - m0, rows) : most)), dim3(block_of(TPR)), 0, s, x,
                           M, (int)C, sx, w, wt, b, bt, eps, y, sy, mean, rstd, m0);
    }
  }
};

struct Backward {
  const void* dy;
  int64_t sdy;
  const void* x;
  int64_t M, C, sx;
  const void* w;
  int wt;
  const float *mean, *rstd;
  void* dx;
  int64_t sdx;
  void *dw, *db;
  int bt;
  float* parts;
  hipStream_t s;
  template <int DT, int TPR, int NV, int FULL>
  void run() const {
    constexpr int BLOCK = backward_block(TPR), PARTS = backward_parts(TPR, NV);
    const int64_t wgs = cdiv(M, BLOCK / TPR);
    const bool sums = dw || db;
    const int n = (int)(sums ? (wgs < PARTS ? wgs : PARTS) : wgs < 2048 ? wgs : 2048);
    if (n && sums)
      hipLaunchKernelGGL((layer_norm_backward_kernel<DT, TPR, NV, FULL, BLOCK, true>), dim3(n), dim3(BLOCK), 0, s, dy, sdy, x, M, (int)C, sx, w, wt, mean, rstd, dx,
                         sdx, parts);
    else if (n)
      hipLaunchKernelGGL((layer_norm_backward_kernel<DT, TPR, NV, FULL, BLOCK, false>), dim3(n), dim3(BLOCK), 0, s, dy, sdy, x, M, (int)C, sx, w, wt, mean, rstd, dx,
                         sdx, nullptr);
    if (sums) join(n);
  }
  void join(int n) const {
    constexpr int64_t most = 1 << 27;  // columns of a launch: sixteen threads each, of which 2^32 are its limit
    for (int64_t c0 = 0; c0 < C; c0 += most)
      hipLaunchKernelGGL(layer_norm_sums_kernel, dim3((unsigned)cdiv(C - c0 < most ? C - c0 : most, 16), 2), dim3(256), 0, s, parts, n, (int)C, dw, wt, db, bt, (int)c0);
  }
};

// Lanes a row, vectors a lane and how many of these are full for rows of C columns: part of a wave up to 32 vectors, a wave up to 32
// elements a lane (forward 64), two waves up to 32 (backward, whose sums take two registers an element), then a workgroup of 256 up to 32
// and one of 1024 up to 16.  False: longer ones.
template <int DT, bool BACKWARD, class Op>
bool by_length(const Op& op, int64_t C) {
  constexpr int VE = RowType<DT>::VE;
  const int64_t vecs = cdiv(C, VE);
#define TK_LN(tpr, nv, full)               \
  if (vecs <= (int64_t)tpr * nv) {         \
    op.template run<DT, tpr, nv, full>(); \
    return true;                           \
  }
  TK_LN(8, 1, 0) TK_LN(16, 1, 0) TK_LN(32, 1, 0) TK_LN(64, 1, 0) TK_LN(64, 2, 1) TK_LN(64, 3, 2) TK_LN(64, 4, 3)
  if constexpr (BACKWARD && DT != TK_F32) {
    TK_LN(128, 3, 2) TK_LN(128, 4, 3)
  } else {
    TK_LN(64, 6, 4) TK_LN(64, 8, 6)
  }
  if constexpr (BACKWARD && DT == TK_F32) {
    TK_LN(128, 6, 4) TK_LN(128, 8, 6)
  } else if constexpr (DT == TK_F32) {
    TK_LN(64, 12, 8) TK_LN(64, 16, 12)
  }
  if constexpr (DT == TK_F32) {
    TK_LN(256, 8, 4) TK_LN(1024, 4, 2)
  } else {
    TK_LN(256, 4, 2) TK_LN(1024, 2, 1)
  }
#undef TK_LN
  return false;
}

template <int DT>
void forward(const Forward& f) {
  const int64_t vecs = cdiv(f.C, RowType<DT>::VE);
  if (f.M < MANY_ROWS && vecs > 64 && vecs <= 1024) {  // few rows: a workgroup a row
    if (vecs <= 256)
      f.run<DT, 256, 1, 0>();
    else if (vecs <= 512)
      f.run<DT, 256, 2, 1>();
    else
      f.run<DT, 256, 4, 2>();
    return;
  }
  if (!by_length<DT, false>(f, f.C))
    hipLaunchKernelGGL(layer_norm_long_kernel<DT>, dim3(rows_grid(f.M)), dim3(256), 0, f.s, f.x, f.M, f.C, f.sx, f.w, f.wt, f.b, f.bt, f.eps, f.y, f.sy, f.mean, f.rstd);
}

template <int DT>
void backward(const Backward& b) {
  if (by_length<DT, true>(b, b.C)) return;
  if (b.dx && b.M)
    hipLaunchKernelGGL(layer_norm_dx_long_kernel<DT>, dim3(rows_grid(b.M)), dim3(256), 0, b.s, b.dy, b.sdy, b.x, b.M, b.C, b.sx, b.w, b.wt, b.mean, b.rstd, b.dx, b.sdx);
  if (!b.dw && !b.db) return;
  const int n = (int)(b.M < LONG_PARTS ? b.M : LONG_PARTS);
  if (n)
    hipLaunchKernelGGL(layer_norm_parts_long_kernel<DT>, dim3((unsigned)cdiv(b.C, 256), n), dim3(256), 0, b.s, b.dy, b.sdy, b.x, b.M, b.C, b.sx, b.mean, b.rstd,
                       b.parts);
  b.join(n);
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
  if (!x || !y || !mean != !rstd) return fail(TK_ERR_INVALID, "tk_layer_norm: null pointer");
  const Forward f = {x, n_rows, n_cols, stride_xm, weight, weight_dtype, bias, bias_dtype, eps, y, stride_ym, mean, rstd, static_cast<hipStream_t>(stream)};
  (dtype == TK_F32 ? forward<TK_F32> : dtype == TK_BF16 ? forward<TK_BF16> : forward<TK_F16>)(f);
  return check_launch("layer_norm_kernel");
}

extern "C" int64_t tk_layer_norm_backward_workspace_bytes(int64_t n_rows, int64_t n_cols) {
  const int64_t parts = n_cols <= 512 ? 768 : n_cols <= 16384 ? 512 : LONG_PARTS;  // (a bound for each type)
  return n_rows > 0 && n_cols > 0 ? 2 * (n_rows < parts ? n_rows : parts) * n_cols * 4 : 0;
}

extern "C" int32_t tk_layer_norm_backward(const void* dy, int64_t stride_dym, const void* x, int32_t dtype, int64_t n_rows, int64_t n_cols,
                                          int64_t stride_xm, const void* weight, int32_t weight_dtype, const float* mean, const float* rstd, void* dx,
                                          int64_t stride_dxm, void* dweight, void* dbias, int32_t bias_dtype, void* workspace, tk_stream_t stream) {
  if (n_rows < 0 || n_cols <= 0 || n_cols > MAX_COLS)
    return fail(TK_ERR_INVALID, "tk_layer_norm_backward: bad sizes %lld x %lld", (long long)n_rows, (long long)n_cols);
  if (!is_row_dtype(dtype) || ((weight || dweight) && !is_row_dtype(weight_dtype)) || (dbias && !is_row_dtype(bias_dtype)))
    return fail(TK_ERR_UNSUPPORTED, "tk_layer_norm_backward: fp32, bf16 and fp16 only");
  if (n_rows && (!dy || !x || !mean || !rstd)) return fail(TK_ERR_INVALID, "tk_layer_norm_backward: null pointer");
  if (n_rows && (dweight || dbias) && !workspace) return fail(TK_ERR_INVALID, "tk_layer_norm_backward: the sums over rows need a workspace");
  const Backward b = {dy,   stride_dym, x,  n_rows,     n_cols,  stride_xm, weight,    weight_dtype,
                      mean, rstd,       dx, stride_dxm, dweight, dbias,     bias_dtype, static_cast<float*>(workspace), static_cast<hipStream_t>(stream)};
  (dtype == TK_F32 ? backward<TK_F32> : dtype == TK_BF16 ? backward<TK_BF16> : backward<TK_F16>)(b);
  return check_launch("layer_norm_backward_kernel");
}
