// Pieces that the row operators share (layer norm, operators over a vocabulary): typed element access and sums over a workgroup.
#pragma once
#include "common.h"

namespace tk {

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

// The sum over a workgroup of THREADS, in every lane; `buf`: THREADS floats of LDS.  Begins and ends with a barrier.
template <int THREADS>
__device__ __forceinline__ float block_sum(float v, float* buf) {
  __syncthreads();
  buf[threadIdx.x] = v;
  __syncthreads();
#pragma unroll
  for (int d = THREADS / 2; d; d >>= 1) {
    if ((int)threadIdx.x < d) buf[threadIdx.x] += buf[threadIdx.x + d];
    __syncthreads();
  }
  const float s = buf[0];
  __syncthreads();
  return s;
}

}  // namespace tk
