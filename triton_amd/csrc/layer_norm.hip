// Layer norm of rows, forward and backward.  Both move each element of the rows once a pass and are bound by that; what the kernels
// below arrange is that a row stays in registers between its reductions and its results, and that the sums over rows stay
// in registers over many rows.
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

// Between two passes over a row's registers: without it the compiler keeps the first pass' 32-bit elements (and what else of it the second one
// could use) beside the packed ones, at up to four times the registers.
template <int N>
__device__ __forceinline__ void once_more(row_u32x4 (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(v[i]));
}

constexpr int block_of(int tpr) { return tpr < 256 ? 256 : tpr; }

// TPR lanes a row, NV vectors of 16 bytes a lane, FULL of which lie within any row that comes here: the row is read once, into registers; mean, then the sum of squares around it.
template <int DT, int TPR, int NV, int FULL>
__global__ __launch_bounds__(block_of(TPR)) void layer_norm_kernel(const void* x, int64_t M, int C, int64_t sx, const void* w, int wt, const void* b, int bt,
                                                                   float eps, void* y, int64_t sy, float* mean, float* rstd, int64_t m0) {
  typedef RowType<DT> R;
  constexpr int VE = R::VE, ROWS = block_of(TPR) / TPR;
  __shared__ float buf[2][16];
  const int lane = (int)threadIdx.x % TPR;
  const float inv_c = 1.0f / (float)C;
  const int64_t m = m0 + (int64_t)blockIdx.x * ROWS + threadIdx.x / TPR;
  if (m >= M) return;  // (lanes that share a row leave together)
  const char* row = static_cast<const char*>(x) + m * sx * R::BYTES;
  row_u32x4 raw[NV];
  float s = 0.f;
#pragma unroll
  for (int v = 0; v < NV; ++v) raw[v] = v < FULL ? R::load_vec(row, (v * TPR + lane) * VE) : R::load_vec_to(row, (v * TPR + lane) * VE, C, 0u);
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int e = 0; e < VE; ++e) s += R::element(raw[v], e);
  const float mu = row_sum<TPR>(s, buf[0]) * inv_c;
  once_more(raw);
  s = 0.f;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const bool full = v < FULL;
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      const float d = R::element(raw[v], e) - mu;
      s = fmaf(d, full || (v * TPR + lane) * VE + e < C ? d : 0.f, s);
    }
  }
  const float r = 1.0f / sqrtf(row_sum<TPR>(s, buf[1]) * inv_c + eps);
  once_more(raw);
  void* out = static_cast<char*>(y) + m * sy * R::BYTES;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int c = (v * TPR + lane) * VE;
    float wv[VE], bv[VE], o[VE];
    load_weights<VE>(w, wt, c, C, 1.f, wv);
    load_weights<VE>(b, bt, c, C, 0.f, bv);
#pragma unroll
    for (int e = 0; e < VE; ++e) o[e] = fmaf((R::element(raw[v], e) - mu) * r, wv[e], bv[e]);
    if (v < FULL)
      R::store_vec(out, c, R::pack(o));
    else
      R::store_vec_to(out, c, C, R::pack(o));
  }
  if (lane == 0 && mean) {
    mean[m] = mu;
    rstd[m] = r;
  }
}

// The gradients.  Workgroups stay for many rows: a lane's columns are the same in each of them, so that their sums over rows stay in
// registers (`SUMS`), are joined over the workgroup's rows in LDS, and leave as one row of partial sums a workgroup (parts [2][gridDim.x][C]),
// which layer_norm_sums_kernel adds in their order.  The weight lies in LDS in 32 bits, in the order in which lanes take it.
template <int DT, int TPR, int NV, int FULL, bool SUMS>
__global__ __launch_bounds__(block_of(TPR)) void layer_norm_backward_kernel(const void* dy, int64_t sdy, const void* x, int64_t M, int C, int64_t sx,
                                                                            const void* w, int wt, const float* mean, const float* rstd, void* dx,
                                                                            int64_t sdx, float* parts) {
  typedef RowType<DT> R;
  constexpr int VE = R::VE, BLOCK = block_of(TPR), ROWS = BLOCK / TPR, WIDTH = NV * TPR * VE;
  __shared__ float buf[2][2][16];
  __shared__ row_u32x4 wl[NV][VE / 4][TPR];
  const int lane = (int)threadIdx.x % TPR;
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
  int turn = 0;
  for (int64_t m = (int64_t)blockIdx.x * ROWS + threadIdx.x / TPR; m < M; m += (int64_t)gridDim.x * ROWS, turn ^= 1) {
    const char *xr = static_cast<const char*>(x) + m * sx * R::BYTES, *gr = static_cast<const char*>(dy) + m * sdy * R::BYTES;
    row_u32x4 xv[NV], gv[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * TPR + lane) * VE;
      const bool full = v < FULL;
      xv[v] = full ? R::load_vec(xr, c) : R::load_vec_to(xr, c, C, 0u);
      gv[v] = full ? R::load_vec(gr, c) : R::load_vec_to(gr, c, C, 0u);
    }
    const float mu = mean[m], r = rstd[m];
    float sg = 0.f, sgh = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        // (behind the last column dy is zero, and h is finite where the row's is)
        const float g0 = R::element(gv[v], e), h = (R::element(xv[v], e) - mu) * r, g = g0 * bits_f32(wl[v][e / 4][lane][e % 4]);
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
    if constexpr (TPR >= 256) {
      sg = wave_sum_f32(sg);
      sgh = wave_sum_f32(sgh);
      if ((threadIdx.x & 63) == 0) {
        buf[turn][0][threadIdx.x >> 6] = sg;
        buf[turn][1][threadIdx.x >> 6] = sgh;
      }
      __syncthreads();
      sg = sgh = 0.f;
#pragma unroll
      for (int i = 0; i < TPR / 64; ++i) {
        sg += buf[turn][0][i];
        sgh += buf[turn][1][i];
      }
    } else {
      sg = row_sum<TPR>(sg, nullptr);
      sgh = row_sum<TPR>(sgh, nullptr);
    }
    if (!dx) continue;
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

// The partial sums' sums: 32 columns a workgroup, eight lanes a row of 128 bytes, 32 rows at a time; then the rows' sums in their order.
__global__ __launch_bounds__(256) void layer_norm_sums_kernel(const float* parts, int n, int C, void* dw, int wt, void* db, int bt) {
  __shared__ float acc[32][33];
  const int c = (int)blockIdx.x * 32 + (int)(threadIdx.x & 7) * 4;
  void* out = blockIdx.y ? db : dw;
  if (!out) return;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  const float* p = parts + (int64_t)blockIdx.y * n * C;
  for (int i = threadIdx.x >> 3; i < n; i += 32) {
    const row_u32x4 v = RowType<TK_F32>::load_vec_to(p + (int64_t)i * C, c, C, 0u);
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] += bits_f32(v[e]);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) acc[threadIdx.x >> 3][(threadIdx.x & 7) * 4 + e] = s[e];
  __syncthreads();
  if (threadIdx.x < 32 && (int)blockIdx.x * 32 + (int)threadIdx.x < C) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) t += acc[i][threadIdx.x];
    store_any(out, blockIdx.y ? bt : wt, (int)blockIdx.x * 32 + threadIdx.x, t);
  }
}

// ---- rows of any length: read once for each step ----------------------------------------------------------------

template <int DT>
__global__ __launch_bounds__(256) void layer_norm_long_kernel(const void* x, int64_t M, int64_t C, int64_t sx, const void* w, int wt, const void* b, int bt,
                                                              float eps, void* y, int64_t sy, float* mean, float* rstd) {
  __shared__ float buf[2][4];
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
constexpr int MAX_PARTS = 512;  // rows of partial sums: two workgroups a CU
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
    constexpr int64_t rows = block_of(TPR) / TPR, most = 1 << 21;  // (workgroups of a launch: 2^32 threads are its limit)
    for (int64_t m0 = 0; m0 < M; m0 += most * rows)
      hipLaunchKernelGGL((layer_norm_kernel<DT, TPR, NV, FULL>), dim3((unsigned)(cdiv(M - m0, rows) < most ? cdiv(M - m0, rows) : most)), dim3(block_of(TPR)), 0, s, x, M,
                         (int)C, sx, w, wt, b, bt, eps, y, sy, mean, rstd, m0);
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
    const int64_t wgs = cdiv(M, block_of(TPR) / TPR);
    const bool sums = dw || db;
    const int n = (int)(sums ? (wgs < MAX_PARTS ? wgs : MAX_PARTS) : wgs < 2048 ? wgs : 2048);
    if (n && sums)
      hipLaunchKernelGGL((layer_norm_backward_kernel<DT, TPR, NV, FULL, true>), dim3(n), dim3(block_of(TPR)), 0, s, dy, sdy, x, M, (int)C, sx, w, wt, mean, rstd, dx,
                         sdx, parts);
    else if (n)
      hipLaunchKernelGGL((layer_norm_backward_kernel<DT, TPR, NV, FULL, false>), dim3(n), dim3(block_of(TPR)), 0, s, dy, sdy, x, M, (int)C, sx, w, wt, mean, rstd, dx,
                         sdx, nullptr);
    if (sums) join(n);
  }
  void join(int n) const {
    hipLaunchKernelGGL(layer_norm_sums_kernel, dim3((unsigned)cdiv(C, 32), 2), dim3(256), 0, s, parts, n, (int)C, dw, wt, db, bt);
  }
};

// Lanes a row and vectors a lane for rows of C columns: part of a wave up to 32 vectors, a wave up to 64 elements a lane, then a workgroup
// of 256 up to 32 and one of 1024 up to 16 a lane.  False: longer ones.
template <int DT, class Op>
bool by_length(const Op& op, int64_t C) {
  constexpr int VE = RowType<DT>::VE;
  const int64_t vecs = cdiv(C, VE);
#define TK_LN(tpr, nv, full)               \
  if (vecs <= (int64_t)tpr * nv) {         \
    op.template run<DT, tpr, nv, full>(); \
    return true;                           \
  }
  TK_LN(8, 1, 0) TK_LN(16, 1, 0) TK_LN(32, 1, 0) TK_LN(64, 1, 0) TK_LN(64, 2, 1) TK_LN(64, 3, 2) TK_LN(64, 4, 3) TK_LN(64, 6, 4) TK_LN(64, 8, 6)
  if constexpr (DT == TK_F32) {
    TK_LN(64, 12, 8) TK_LN(64, 16, 12) TK_LN(256, 8, 4) TK_LN(1024, 4, 2)
  } else {
    TK_LN(256, 4, 2) TK_LN(1024, 2, 1)
  }
#undef TK_LN
  return false;
}

template <int DT>
void forward(const Forward& f) {
  if (!by_length<DT>(f, f.C))
    hipLaunchKernelGGL(layer_norm_long_kernel<DT>, dim3(rows_grid(f.M)), dim3(256), 0, f.s, f.x, f.M, f.C, f.sx, f.w, f.wt, f.b, f.bt, f.eps, f.y, f.sy, f.mean, f.rstd);
}

template <int DT>
void backward(const Backward& b) {
  if (by_length<DT>(b, b.C)) return;
  if (b.dx && b.M)
    hipLaunchKernelGGL(layer_norm_dx_long_kernel<DT>, dim3(rows_grid(b.M)), dim3(256), 0, b.s, b.dy, b.sdy, b.x, b.M, b.C, b.sx, b.w, b.wt, b.mean, b.rstd, b.dx, b.sdx);
  if (!b.dw && !b.db) return;
  const int n = (int)(b.M < 128 ? b.M : 128);
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
  return n_rows > 0 && n_cols > 0 ? 2 * (n_rows < MAX_PARTS ? n_rows : MAX_PARTS) * n_cols * 4 : 0;
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
