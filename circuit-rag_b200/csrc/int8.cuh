// What the 8-bit row kernels share: the row types, 16-byte vectors of a row, and
// the checks of the C entries.
#pragma once

#include <cstdint>
#include <cstring>

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
  using Pair = __half2;
  static constexpr int V = 8;
  __device__ static float get(__half x) { return __half2float(x); }
  __device__ static __half put(float x) { return __float2half_rn(x); }
};
template <>
struct RowType<__nv_bfloat16> {
  using Pair = __nv_bfloat162;
  static constexpr int V = 8;
  __device__ static float get(__nv_bfloat16 x) { return __bfloat162float(x); }
  __device__ static __nv_bfloat16 put(float x) { return __float2bfloat16_rn(x); }
};

// The larger magnitude, keeping a NaN (fmaxf would drop it); its sign is the product of
// the operands' signs: the caller takes the magnitude at the end.
__device__ __forceinline__ float max_abs_nan(float m, float x) {
  float r;
  asm("max.NaN.xorsign.abs.f32 %0, %1, %2;" : "=f"(r) : "f"(m), "f"(x));
  return r;
}

// a += b, each sum rounded once to the row's type (pairs of 16-bit values in one instruction).
template <typename T, int E>
__device__ __forceinline__ void add_to(T (&a)[E], const T (&b)[E]) {
  if constexpr (sizeof(T) == 4 || E == 1) {
#pragma unroll
    for (int i = 0; i < E; ++i) a[i] = RowType<T>::put(RowType<T>::get(a[i]) + RowType<T>::get(b[i]));
  } else {
    using P = typename RowType<T>::Pair;
#pragma unroll
    for (int i = 0; i < E; i += 2) {
      const P s = __hadd2_rn(P{a[i], a[i + 1]}, P{b[i], b[i + 1]});
      a[i] = s.x;
      a[i + 1] = s.y;
    }
  }
}
// |top| = max(|top|, |v|), a NaN stays.
template <typename T, int E>
__device__ __forceinline__ void raise_top(float& top, const T (&v)[E]) {
  if constexpr (sizeof(T) == 4 || E == 1) {
#pragma unroll
    for (int i = 0; i < E; ++i) top = max_abs_nan(top, RowType<T>::get(v[i]));
  } else {
    using P = typename RowType<T>::Pair;
    P m = __habs2(P{v[0], v[1]});
#pragma unroll
    for (int i = 2; i < E; i += 2) m = __hmax2_nan(m, __habs2(P{v[i], v[i + 1]}));
    top = max_abs_nan(max_abs_nan(top, RowType<T>::get(m.x)), RowType<T>::get(m.y));
  }
}

// A word of BYTES bytes.
template <int BYTES>
struct Word;
template <> struct Word<16> { using type = uint4; };
template <> struct Word<8> { using type = uint2; };
template <> struct Word<4> { using type = uint32_t; };
template <> struct Word<2> { using type = uint16_t; };
template <> struct Word<1> { using type = uint8_t; };

// E elements of a row held by one thread, loaded and stored as one word: rows are
// of whole words on their alignment.
template <typename T, int E>
struct Vec {
  using W = typename Word<E * (int)sizeof(T)>::type;
  T e[E];
  // elements [c, c + E) of a row of d; zeros past its end
  __device__ __forceinline__ static Vec load(const T* row, int c, int d) {
    W word{};
    if (c < d) word = *reinterpret_cast<const W*>(row + c);
    Vec v;
    memcpy(&v, &word, sizeof(W));
    return v;
  }
  __device__ __forceinline__ void store(T* row, int c, int d) const {
    if (c >= d) return;
    W word;
    memcpy(&word, this, sizeof(W));
    *reinterpret_cast<W*>(row + c) = word;
  }
  // not zero if an element is not zero
  __device__ __forceinline__ uint32_t bits() const {
    uint32_t words[(sizeof(W) + 3) / 4] = {}, all = 0;
    memcpy(words, this, sizeof(W));
#pragma unroll
    for (uint32_t w : words) all |= w;
    return all;
  }
};

// ---------------------------------------------------------------- host side
// Launches a kernel that may start while the one before it on the stream still runs:
// each of these kernels first waits for that one's completion (griddep_wait, before
// any access to memory) and only then lets the next one start early, so that no more
// than two of a chain overlap.  They read global memory by ordinary loads: a load by the
// non-coherent path asks for data that no one writes while the kernel lives, and the
// one before still writes when these start.  What is saved is the launch and the set-up, one to
// two microseconds a kernel (a pass of one query against 2M rows: 128 -> 120 us).
template <typename... Params, typename... Args>
inline cudaError_t launch(void (*kernel)(Params...), dim3 grid, int threads, int smem, int cluster, cudaStream_t st,
                          Args... args) {
  cudaLaunchAttribute attrs[2]{};
  attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = 1;
  attrs[1].id = cudaLaunchAttributeClusterDimension;
  attrs[1].val.clusterDim.x = (unsigned)cluster;
  attrs[1].val.clusterDim.y = attrs[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cfg.attrs = attrs;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}
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
