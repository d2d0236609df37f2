// Pieces shared by the kernels of e4m3 matrices with one fp32 scale for each block of 128 (fp8_quant.hip, fp8_gemm*.hip, fp8_wgrad.hip).
#pragma once
#include "gemm_common.h"

namespace tk {

struct Fp8GemmParams {
  const uint8_t* x;
  int64_t x_stride_m;
  const float* xs;
  int64_t xs_m, xs_k;
  const uint8_t* w;
  int64_t w_e, w_n;
  const float* ws;
  int64_t ws_e, ws_k, ws_n;
  const void* bias;
  int64_t bias_e;
  int32_t bias_is_f32;
  const int32_t* gather;
  const int32_t* scatter;
  int32_t scatter_len;
  const void* gammas;
  int32_t gammas_is_f32;
  const int32_t* slice_sizes;
  const int32_t* slice_offs;
  const int32_t* block_sched;
  int32_t n_slices, grid_m, grid_n;
  int32_t M, N, K;
  void* y;
  int64_t y_stride_m;
  float alpha, limit;  // (limit: +inf without one)
  int32_t zero_rest;
  int32_t pow2;      // all scales are powers of two (fp8_scale's)
  uint32_t x_bytes;  // with gather: the extent of x for a buffer resource
};

// 16-bit results, up to kDmaSlices slices, operands as fp8_tiles_run (fp8_gemm.hip) wants them; tile = 256 or 128
int32_t fp8_gemm_launch_tiles(const Fp8GemmParams& p, int tile, int yt, bool swiglu, hipStream_t st);
int32_t fp8_gemm_launch_ring(const Fp8GemmParams& p, int yt, bool swiglu, hipStream_t st);  // operands as for the tiles, any number of slices
int32_t fp8_gemm_launch_few(const Fp8GemmParams& p, bool aligned, int yt, bool swiglu, hipStream_t st);

namespace {

constexpr int kFp8Block = 128;
constexpr int kFp8Most = 0x7FFFFF00;  // of a size: with a tile more it is still a number of 32 bits

// c + the product of 16 columns of w and 16 rows of x over a block of 128: lane l holds 32 consecutive k, from (l >> 4) * 32 on, of column / row l & 15.  The
// scales are e8m0 bytes, the exponents of powers of two as fp32 numbers have them.
__device__ __forceinline__ f32x4_t mfma_block(i32x8_t w, i32x8_t x, f32x4_t c, uint32_t w_exp = 0x7F7F7F7Fu, uint32_t x_exp = 0x7F7F7F7Fu) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, c, 0, 0, 0, (int)w_exp, 0, (int)x_exp);
}

// The same product from the values' exact 16-bit form, for fp32 results: the e4m3 instructions add eight products at a time and drop what of one lies below 2^-13
// of the power of two in the largest of them, always towards zero.  Eight products are off by up to 7 * 2^-13 of the largest one; nothing bounds that by the result, which may be
// small beside it.  A choice for results of 16 bits, at twice the rate of the 16-bit instructions and without conversions.  Relative error against 64 bits (root mean square; in brackets what the
// result's rounding alone makes), K 1024: normal operands bf16 1.66e-3 (1.66e-3), fp16 2.09e-4 (2.08e-4); one sign, magnitudes over fourteen powers of two, bf16 1.63e-3 (1.62e-3), fp16
// 2.17e-4 (2.03e-4), on the average 7.6e-5 too small; sums that cancel to a sixteenth (K 128) bf16 1.67e-3 (1.65e-3), fp16 2.79e-4 (2.10e-4).
__device__ __forceinline__ f32x4_t mfma_block_exact(i32x8_t w, i32x8_t x, f32x4_t c) {
#pragma unroll
  for (int t = 0; t < 4; ++t) {  // (eight of the lane's k each: any order does that is the same for both)
    bf16x8_t a, b;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const bf16x2_t a0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[2 * t + i], 1.0f, false), a1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[2 * t + i], 1.0f, true);
      const bf16x2_t b0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[2 * t + i], 1.0f, false), b1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[2 * t + i], 1.0f, true);
      a[4 * i] = a0[0], a[4 * i + 1] = a0[1], a[4 * i + 2] = a1[0], a[4 * i + 3] = a1[1];
      b[4 * i] = b0[0], b[4 * i + 1] = b0[1], b[4 * i + 2] = b1[0], b[4 * i + 3] = b1[1];
    }
    c = Frag<16>::mma(a, b, c);
  }
  return c;
}

// sixteen bytes at `k` of a row of K, whatever its address; zeros past K and without a row
__device__ __forceinline__ u32x4_t load_piece(const uint8_t* row, int k, int K) {
  u32x4_t v = {0, 0, 0, 0};
  if (!row || k >= K) return v;
  if (k + 16 <= K) {
    __builtin_memcpy(&v, row + k, 16);
  } else if (K >= 16) {  // the row's last sixteen bytes, moved down (byte by byte a row of 1000 took 3 us of its product's 9)
    uint64_t q[2];
    __builtin_memcpy(q, row + K - 16, 16);
    const int drop = 8 * (k + 16 - K);  // 8 .. 120 bits
    const uint64_t lo = drop < 64 ? q[0] >> drop | q[1] << (64 - drop) : q[1] >> (drop - 64), hi = drop < 64 ? q[1] >> drop : 0;
    v = u32x4_t{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
  } else {
    for (int i = 0; i < K - k; ++i) v[i >> 2] |= (uint32_t)row[k + i] << (i & 3) * 8;
  }
  return v;
}

// ---- scales and conversions ----------------------------------------------------------------------------------------------------------------
// The smallest power of two s >= 2^-126 with amax <= 448 s, from amax's own bits (448 = 1.75 * 2^8): no logarithm and no division, so every
// place that quantises a block has the same scale.  Zero: 1.
__device__ __forceinline__ float fp8_scale(uint32_t amax_bits) {
  if (amax_bits == 0) return 1.0f;
  const int e = (int)(amax_bits >> 23) - 8 + ((amax_bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return bits_f32((uint32_t)(e < 1 ? 1 : e) << 23);
}
// 1 / s for such a scale: a power of two between 2^-120 and 2^126
__device__ __forceinline__ float fp8_inverse(float s) { return bits_f32(0x7F000000u - f32_bits(s)); }

// the magnitude that counts for the scale: none for infinities and NaN
__device__ __forceinline__ uint32_t finite_bits(float v) {
  const uint32_t u = f32_bits(v) & 0x7FFFFFFFu;
  return u < 0x7F800000u ? u : 0u;
}
// the largest of sixteen lanes' numbers, in each of them
__device__ __forceinline__ uint32_t max16(uint32_t v) {
#define TK_STEP(ctrl)                                                                             \
  {                                                                                               \
    const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, 0xF, 0xF, false);     \
    v = o > v ? o : v;                                                                            \
  }
  TK_STEP(0xB1)   // quad_perm [1,0,3,2]
  TK_STEP(0x4E)   // quad_perm [2,3,0,1]
  TK_STEP(0x141)  // row_half_mirror
  TK_STEP(0x140)  // row_mirror
#undef TK_STEP
  return v;
}
// four numbers of at most 448 (or NaN; an infinity becomes NaN, e4m3 has none) to e4m3, nearest, ties to even
__device__ __forceinline__ uint32_t to_e4m3(float a, float b, float c, float d) {
  int o = 0;
  o = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, o, false);
  o = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, o, true);
  return (uint32_t)o;
}
__device__ __forceinline__ float no_infinity(float v) { return (f32_bits(v) & 0x7FFFFFFFu) == 0x7F800000u ? bits_f32(0x7FC00000u) : v; }
__device__ __forceinline__ void from_e4m3(uint32_t q, float* o) {
  const f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)q, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)q, true);
  o[0] = lo[0], o[1] = lo[1], o[2] = hi[0], o[3] = hi[1];
}

template <int DT>
__device__ __forceinline__ float load_elem(const void* p, int64_t i) {
  if constexpr (DT == TK_F32) return static_cast<const float*>(p)[i];
  if constexpr (DT == TK_BF16) return bf16_bits_to_f32(static_cast<const uint16_t*>(p)[i]);
  return f16_bits_to_f32(static_cast<const uint16_t*>(p)[i]);
}
template <int DT>
__device__ __forceinline__ void store_elem(void* p, int64_t i, float v) {
  if constexpr (DT == TK_F32)
    static_cast<float*>(p)[i] = v;
  else if constexpr (DT == TK_BF16)
    static_cast<uint16_t*>(p)[i] = f32_to_bf16_bits(v);
  else
    static_cast<uint16_t*>(p)[i] = f32_to_f16_bits(v);
}
// N (4 or 8) consecutive elements at any element's address: wide loads and stores need no alignment here, but those that cross cache lines take two
template <class V>
__device__ __forceinline__ V load_wide(const void* p) {
  V v;
  __builtin_memcpy(&v, p, sizeof(V));
  return v;
}
template <class V>
__device__ __forceinline__ void store_wide(void* p, V v) {
  __builtin_memcpy(p, &v, sizeof(V));
}
template <int DT, int N>
__device__ __forceinline__ void load_vec(const void* p, int64_t i, float* v) {
  if constexpr (DT == TK_F32) {
#pragma unroll
    for (int c = 0; c < N; c += 4) {
      const f32x4_t t = load_wide<f32x4_t>(static_cast<const float*>(p) + i + c);
#pragma unroll
      for (int k = 0; k < 4; ++k) v[c + k] = t[k];
    }
  } else {
    typedef uint32_t words_t __attribute__((ext_vector_type(N / 2)));
    const words_t w = load_wide<words_t>(static_cast<const uint16_t*>(p) + i);
#pragma unroll
    for (int k = 0; k < N / 2; ++k) {
      if constexpr (DT == TK_BF16) {
        v[2 * k] = bits_f32(w[k] << 16), v[2 * k + 1] = bits_f32(w[k] & 0xFFFF0000u);
      } else {
        const f16x2_t h = __builtin_bit_cast(f16x2_t, (uint32_t)w[k]);
        v[2 * k] = (float)h[0], v[2 * k + 1] = (float)h[1];
      }
    }
  }
}
template <int DT, int N>
__device__ __forceinline__ void store_vec(void* p, int64_t i, const float* v) {
  if constexpr (DT == TK_F32) {
#pragma unroll
    for (int c = 0; c < N; c += 4) store_wide(static_cast<float*>(p) + i + c, f32x4_t{v[c], v[c + 1], v[c + 2], v[c + 3]});
  } else {
    typedef uint32_t words_t __attribute__((ext_vector_type(N / 2)));
    words_t w;
#pragma unroll
    for (int k = 0; k < N / 2; ++k) w[k] = pack_out2<DT == TK_F16>(v[2 * k], v[2 * k + 1]);
    store_wide(static_cast<uint16_t*>(p) + i, w);
  }
}

// ---- swiglu ----------------------------------------------------------------------------------------------------------------------------------
// sigma(x) = 1 / (1 + exp(-x)) as the product u v, and 1 - sigma.  With t = exp(-|x| / 2) nothing overflows, sigma and 1 - sigma have no difference in them, and
// (y u) v is good as long as y sigma is a normal number, where exp(-|x|) itself no longer is.  For results of 16 bits the hardware's exp2 and reciprocal (1 ulp
// each) of a once rounded x log2(e): off by |x| 2^-24, next to 2^-9 of the result's rounding.  For fp32 results (EXACT) that product is kept in two parts and the
// reciprocal is a division.
struct Sigmoid {
  float u, v, rest;
};
template <bool EXACT>
__device__ __forceinline__ Sigmoid sigmoid_of(float x) {
  const float ax = fabsf(x), hi = ax * -1.44269504088896340736f;
  float t = __builtin_amdgcn_exp2f(hi * 0.5f);
  if constexpr (EXACT) {
    const float lo = fmaf(ax, -1.44269504088896340736f, -hi) - ax * 1.92596299112661746887e-8f;  // (log2(e) less its fp32)
    if (hi > -512.0f) t = fmaf(t, lo * 0.346573590279972654709f, t);
  }
  const float e = t * t, d = 1.0f + e, r = EXACT ? 1.0f / d : __builtin_amdgcn_rcpf(d);
  const bool neg = x < 0.f;
  return Sigmoid{neg ? t : 1.0f, neg ? t * r : r, neg ? r : e * r};
}
// (comparisons that keep NaN, as torch's clamp does)
__device__ __forceinline__ float at_most(float v, float m) { return v > m ? m : v; }
__device__ __forceinline__ float at_least(float v, float m) { return v < m ? m : v; }

template <bool EXACT>
__device__ __forceinline__ float swiglu_of(float gate, float lin, float alpha, float limit) {
  gate = at_most(gate, limit);
  lin = at_least(at_most(lin, limit), -limit);
  const Sigmoid q = sigmoid_of<EXACT>(alpha * gate);
  const float s = gate * q.u * q.v;
  return fmaf(s, lin, s);
}

// ---- the product's epilogue ------------------------------------------------------------------------------------------------------------------
// rows behind the last slice
template <int YT, bool SWIGLU>
__device__ __forceinline__ void fp8_zero_rest(const Fp8GemmParams& p) {
  if (!p.zero_rest || !p.slice_sizes) return;
  const int cols = SWIGLU ? p.N / 2 : p.N;
  for (int64_t r = (int64_t)p.slice_offs[p.n_slices] + blockIdx.x; r < p.M; r += gridDim.x)
    for (int c = threadIdx.x; c < cols; c += blockDim.x) store_elem<YT>(p.y, r * p.y_stride_m + c, 0.f);
}

// acc[f][j] = 16 x 16 fragment of output columns ncol0 + f * 16 .. and rows off_m + (j * WM + mw) * 16 .. of the slice, as the MFMA leaves it with the
// weights as its first operand: register i of lane l is column (l >> 4) * 4 + i of row l & 15.  n_end: the first column that the tile does not have.
template <int YT, bool SWIGLU, int WM, int MFW, int NFW>
__device__ __forceinline__ void fp8_epilogue(const Fp8GemmParams& p, f32x4_t (&acc)[NFW][MFW], int expert, int off_m, int start_m, int eM, int ncol0, int n_end,
                                             int mw, int lane) {
  static_assert(NFW % 2 == 0, "fragments go in pairs");
  const int lr = lane & 15, g4 = lane >> 4;
  float gam[MFW];
  int dst[MFW];
#pragma unroll
  for (int j = 0; j < MFW; ++j) {
    const int row = off_m + (j * WM + mw) * 16 + lr, r = start_m + (row < eM ? row : eM - 1);
    dst[j] = r;
    if (p.scatter) dst[j] = r < p.scatter_len ? p.scatter[r] : -1;
    if (row >= eM) dst[j] = -1;
    gam[j] = p.gammas ? load_scalar(p.gammas, r, p.gammas_is_f32) : 1.0f;
  }
#pragma unroll
  for (int f = 0; f < NFW; f += 2) {
    // after the exchange of the odd groups of sixteen lanes of the first fragment with the even ones of the second a lane has eight consecutive columns
    const int n0 = ncol0 + f * 16 + (g4 & 1) * 16 + (g4 >> 1) * 8;
    float b[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] = p.bias && n0 + i < n_end ? load_scalar(p.bias, expert * p.bias_e + n0 + i, p.bias_is_f32) : 0.f;
#pragma unroll
    for (int j = 0; j < MFW; ++j) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const auto s = __builtin_amdgcn_permlane16_swap(f32_bits(acc[f][j][i]), f32_bits(acc[f + 1][j][i]), false, false);
        v[i] = bits_f32(s[0]) + b[i];
        v[4 + i] = bits_f32(s[1]) + b[4 + i];
      }
      if (dst[j] < 0) continue;
      const int64_t row = (int64_t)dst[j] * p.y_stride_m;
      if constexpr (SWIGLU) {
        float o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = swiglu_of<YT == TK_F32>(v[2 * i], v[2 * i + 1], p.alpha, p.limit) * gam[j];
        if (n0 + 8 <= n_end) {
          store_vec<YT, 4>(p.y, row + n0 / 2, o);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (n0 + 2 * i < n_end) store_elem<YT>(p.y, row + n0 / 2 + i, o[i]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= gam[j];
        if (n0 + 8 <= n_end) {
          store_vec<YT, 8>(p.y, row + n0, v);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (n0 + i < n_end) store_elem<YT>(p.y, row + n0 + i, v[i]);
        }
      }
    }
  }
}

}  // namespace
}  // namespace tk
