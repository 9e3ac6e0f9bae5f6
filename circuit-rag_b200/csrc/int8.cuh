// What the 8-bit row kernels share: the row types, 16-byte vectors of a row, and
// the checks of the C entries.
#pragma once

#include <cstdint>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/circuit_ops.h"
#include "common.cuh"
#include "index_internal.h"

namespace cb {
namespace i8 {

// ---------------------------------------------------------------- row types
template <typename T>
struct RowType;  // V: elements of a 16-byte vector
template <>
struct RowType<float> {
  static constexpr int V = 4;
  __device__ static float get(float x) { return x; }
  __device__ static float put(float x) { return x; }
};
template <>
struct RowType<__half> {
  static constexpr int V = 8;
  __device__ static float get(__half x) { return __half2float(x); }
  __device__ static __half put(float x) { return __float2half_rn(x); }
};
template <>
struct RowType<__nv_bfloat16> {
  static constexpr int V = 8;
  __device__ static float get(__nv_bfloat16 x) { return __bfloat162float(x); }
  __device__ static __nv_bfloat16 put(float x) { return __float2bfloat16_rn(x); }
};

template <typename T>
union Vec {
  uint4 raw;
  T e[RowType<T>::V];
};

// Elements [c, c + V) of a row of d elements: one 16-byte access where the row
// allows it, else one access an element; zeros past the row's end.
template <typename T>
__device__ __forceinline__ Vec<T> load_vec(const T* row, int c, int d, bool wide) {
  constexpr int V = RowType<T>::V;
  Vec<T> v;
  v.raw = make_uint4(0, 0, 0, 0);
  if (wide && c + V <= d) {
    v.raw = *reinterpret_cast<const uint4*>(row + c);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (c + i < d) v.e[i] = row[c + i];
  }
  return v;
}
template <typename T>
__device__ __forceinline__ void store_vec(T* row, int c, int d, bool wide, const Vec<T>& v) {
  constexpr int V = RowType<T>::V;
  if (wide && c + V <= d) {
    *reinterpret_cast<uint4*>(row + c) = v.raw;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (c + i < d) row[c + i] = v.e[i];
  }
}

// ---------------------------------------------------------------- host side
inline int bad(const char* msg) {
  try {
    cb::set_error(msg);
  } catch (...) {
  }
  return CIRCUIT_ERR_ARG;
}
inline int check(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return CIRCUIT_OK;
  try {
    cb::cuda_ok(e, what);
  } catch (...) {
  }
  return CIRCUIT_ERR_CUDA;
}
inline bool on16(const void* p, int64_t stride_bytes) {
  return ((reinterpret_cast<uintptr_t>(p) | (uintptr_t)stride_bytes) & 15) == 0;
}
inline int type_bytes(int dtype) { return dtype == CIRCUIT_F32 ? 4 : dtype == CIRCUIT_F16 || dtype == CIRCUIT_BF16 ? 2 : 0; }

}  // namespace i8
}  // namespace cb
