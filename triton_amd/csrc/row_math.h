// Pieces that the row operators share (layer norm, operators over a vocabulary): typed element access and sums over a workgroup.
#pragma once
#include "common.h"
#include "route_common.h"

namespace tk {

typedef uint32_t row_u32x4 __attribute__((ext_vector_type(4)));
typedef row_u32x4 row_u32x4_at2 __attribute__((aligned(2)));  // sixteen bytes at the address of any element

template <int DT>
struct RowType {
  static constexpr int BYTES = DT == TK_F32 ? 4 : 2;
  static __device__ __forceinline__ float load(const void* p, int64_t i) {
    if constexpr (DT == TK_F32) return static_cast<const float*>(p)[i];
    if constexpr (DT == TK_BF16) return bf16_bits_to_f32(static_cast<const uint16_t*>(p)[i]);
    return f16_bits_to_f32(static_cast<const uint16_t*>(p)[i]);
  }
  static __device__ __forceinline__ void store(void* p, int64_t i, float v) {
    if constexpr (DT == TK_F32)
      static_cast<float*>(p)[i] = v;
    else if constexpr (DT == TK_BF16)
      static_cast<uint16_t*>(p)[i] = f32_to_bf16_bits(v);
    else
      static_cast<uint16_t*>(p)[i] = f32_to_f16_bits(v);
  }

  // Sixteen bytes of a row: VE elements.  Rows of an odd number of 16-bit elements begin at any even address; the memory pipe takes such
  // addresses in one instruction.
  static constexpr int VE = 16 / BYTES;
  static constexpr uint32_t NEG_INF_BITS = DT == TK_F32 ? 0xFF800000u : DT == TK_BF16 ? 0xFF80FF80u : 0xFC00FC00u;  // a dword of -inf
  static __device__ __forceinline__ row_u32x4 load_vec(const void* p, int64_t i) {
    return *reinterpret_cast<const row_u32x4_at2*>(static_cast<const char*>(p) + i * BYTES);
  }
  // The same with the hint that the elements are not looked at again.
  static __device__ __forceinline__ row_u32x4 load_vec_once(const void* p, int64_t i) {
    return __builtin_nontemporal_load(reinterpret_cast<const row_u32x4_at2*>(static_cast<const char*>(p) + i * BYTES));
  }
  static __device__ __forceinline__ void store_vec_once(void* p, int64_t i, row_u32x4 v) {
    __builtin_nontemporal_store(v, reinterpret_cast<row_u32x4_at2*>(static_cast<char*>(p) + i * BYTES));
  }
  // What is left of a row from element i on; opaque, since the compiler would keep a mask for each element of each vector over a loop
  // over rows, at a hundred registers.
  static __device__ __forceinline__ int left(int i, int end) {
    int n = end - i;
    asm volatile("" : "+v"(n));
    return n;
  }
  // The same where the elements in front of `begin` and from `end` on are not there: they read as `fill` (a dword of it), and nothing there
  // is touched.  Pairs of 16-bit elements are requested together, from the nearest element that there is, and chosen afterwards: one by one
  // under their conditions, each waits for the one that it shares a register with, up to seven memory latencies in a row at the end of each
  // row.
  static __device__ __forceinline__ row_u32x4 load_vec_in(const void* p, int i, int begin, int end, uint32_t fill) {
    const int n = left(i, end), skip = begin - i;
    if (skip <= 0 && n >= VE) return load_vec(p, i);
    row_u32x4 v = {fill, fill, fill, fill};
    if constexpr (DT == TK_F32) {
#pragma unroll
      for (int e = 0; e < VE; ++e)
        if (e >= skip && e < n) v[e] = static_cast<const uint32_t*>(p)[i + e];
    } else if (n > 0 && skip < VE) {
      uint32_t x[VE];
#pragma unroll
      for (int e = 0; e < VE; ++e) x[e] = static_cast<const uint16_t*>(p)[i + (e < skip ? skip : e < n ? e : n - 1)];
#pragma unroll
      for (int e = 0; e < VE; ++e) x[e] = e >= skip && e < n ? x[e] : fill & 0xFFFFu;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = x[2 * e] | x[2 * e + 1] << 16;
    }
    return v;
  }
  static __device__ __forceinline__ row_u32x4 load_vec_to(const void* p, int i, int end, uint32_t fill) { return load_vec_in(p, i, i, end, fill); }
  // A row's last vectors without a branch, for rows of at least VE elements: load_last() takes the sixteen bytes that end with the row
  // where those from i on pass its end, and last() moves them to their places, with zeros behind.  The move may wait until the vector is
  // used.
  static __device__ __forceinline__ row_u32x4 load_last(const void* p, int i, int end) { return load_vec(p, i < end - VE ? i : end - VE); }
  static __device__ __forceinline__ row_u32x4 last(row_u32x4 v, int i, int end) {
    const int n = left(i, end), drop = n >= VE ? 0 : n <= 0 ? 128 : (VE - n) * (8 * BYTES);
    uint64_t lo = (uint64_t)v[1] << 32 | v[0], hi = (uint64_t)v[3] << 32 | v[2];
    const bool half = drop >= 64;
    const int s = drop & 63;
    lo = half ? hi : lo;
    hi = half ? 0 : hi;
    const uint64_t carry = s ? hi << (64 - s) : 0;
    lo = drop >= 128 ? 0 : lo >> s | carry;
    hi = hi >> s;
    return row_u32x4{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
  }
  static __device__ __forceinline__ float element(row_u32x4 v, int e) {
    if constexpr (DT == TK_F32) return bits_f32(v[e]);
    if constexpr (DT == TK_BF16) return bits_f32(e & 1 ? v[e >> 1] & 0xFFFF0000u : v[e >> 1] << 16);
    return f16_bits_to_f32((uint16_t)(e & 1 ? v[e >> 1] >> 16 : v[e >> 1]));
  }
  // Results rounded to nearest even.
  static __device__ __forceinline__ row_u32x4 pack(const float (&x)[VE]) {
    row_u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == TK_F32)
        v[i] = f32_bits(x[i]);
      else if constexpr (DT == TK_BF16)
        v[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t{x[2 * i], x[2 * i + 1]}), bf16x2_t));
      else
        v[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t{x[2 * i], x[2 * i + 1]}), f16x2_t));
    }
    return v;
  }
  static __device__ __forceinline__ void store_vec(void* p, int64_t i, row_u32x4 v) {
    *reinterpret_cast<row_u32x4_at2*>(static_cast<char*>(p) + i * BYTES) = v;
  }
  static __device__ __forceinline__ void store_vec_to(void* p, int i, int end, row_u32x4 v) {
    const int n = left(i, end);
    if (n >= VE) return store_vec(p, i, v);
#pragma unroll
    for (int e = 0; e < VE; ++e)
      if (e < n) {
        if constexpr (DT == TK_F32)
          static_cast<uint32_t*>(p)[i + e] = v[e];
        else
          static_cast<uint16_t*>(p)[i + e] = (uint16_t)(e & 1 ? v[e >> 1] >> 16 : v[e >> 1]);
      }
  }
};

// An element of a type that is only known at run time (weights, of which there are few).
__device__ __forceinline__ float load_any(const void* p, int dtype, int64_t i) {
  if (dtype == TK_F32) return RowType<TK_F32>::load(p, i);
  return dtype == TK_BF16 ? RowType<TK_BF16>::load(p, i) : RowType<TK_F16>::load(p, i);
}
__device__ __forceinline__ void store_any(void* p, int dtype, int64_t i, float v) {
  if (dtype == TK_F32)
    RowType<TK_F32>::store(p, i, v);
  else if (dtype == TK_BF16)
    RowType<TK_BF16>::store(p, i, v);
  else
    RowType<TK_F16>::store(p, i, v);
}

inline bool is_row_dtype(int32_t t) { return t == TK_F32 || t == TK_BF16 || t == TK_F16; }

__device__ __forceinline__ float wave_max_f32(float v) {
  int x = __builtin_bit_cast(int, v);
#define TK_STEP(ctrl) x = __builtin_bit_cast(int, fmaxf(__builtin_bit_cast(float, x), __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, x, ctrl, 0xF, 0xF, false))));
  TK_ROW16(TK_STEP)
#undef TK_STEP
  const float a = __builtin_bit_cast(float, __builtin_amdgcn_readlane(x, 0)), b = __builtin_bit_cast(float, __builtin_amdgcn_readlane(x, 16));
  const float c = __builtin_bit_cast(float, __builtin_amdgcn_readlane(x, 32)), d = __builtin_bit_cast(float, __builtin_amdgcn_readlane(x, 48));
  return fmaxf(fmaxf(a, b), fmaxf(c, d));
}

// Over a workgroup of THREADS, in every lane: the waves' results by lane exchanges, then through `buf` (THREADS / 64 floats of LDS, not in
// use by anything in front of the call).  One barrier; the caller puts another one in front of the next use of `buf`.
template <int THREADS>
__device__ __forceinline__ float block_sum(float v, float* buf) {
  v = wave_sum_f32(v);
  if constexpr (THREADS == 64) return v;
  if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = buf[0];
#pragma unroll
  for (int w = 1; w < THREADS / 64; ++w) s += buf[w];
  return s;
}
template <int THREADS>
__device__ __forceinline__ float block_max(float v, float* buf) {
  v = wave_max_f32(v);
  if constexpr (THREADS == 64) return v;
  if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = buf[0];
#pragma unroll
  for (int w = 1; w < THREADS / 64; ++w) s = fmaxf(s, buf[w]);
  return s;
}

}  // namespace tk
